// Host check of the channels-last operators: do two pitched matrices share memory?
#pragma once

#include <cstdint>

namespace s2 {

// `rows` rows of `width` bytes, `pitch` bytes apart.
struct PitchedSpan {
    const void *ptr;
    long long rows, width, pitch;
};

inline PitchedSpan bytes_at(const void *p, long long n) { return {p, 1, n, n}; }

// Whether the `n` bytes from `at` share any with a's rows.
inline bool meets(const PitchedSpan &a, __int128 at, __int128 n)
{
    const __int128 pa = reinterpret_cast<uintptr_t>(a.ptr), past = at - pa - a.width;  // the first row that ends behind `at`
    const __int128 row = past < 0 || a.rows == 1 ? 0 : past / a.pitch + 1;
    return row < a.rows && pa + row * a.pitch < at + n && at < pa + row * a.pitch + a.width;
}

// True when a and b may share bytes. Single rows are told apart exactly, equal pitches by columns (two column
// ranges of one wider buffer do not overlap); else their whole extents are compared.
inline bool may_overlap(const PitchedSpan &a, const PitchedSpan &b)
{
    if (!a.ptr || !b.ptr || a.rows <= 0 || b.rows <= 0) return false;
    const __int128 pa = reinterpret_cast<uintptr_t>(a.ptr), pb = reinterpret_cast<uintptr_t>(b.ptr);
    const __int128 ea = pa + static_cast<__int128>(a.rows - 1) * a.pitch + a.width;
    const __int128 eb = pb + static_cast<__int128>(b.rows - 1) * b.pitch + b.width;
    if (ea <= pb || eb <= pa) return false;
    if (b.rows == 1) return meets(a, pb, b.width);
    if (a.rows == 1) return meets(b, pa, a.width);
    if (a.pitch == b.pitch && a.pitch > 0) {
        __int128 off = (pb - pa) % a.pitch;
        if (off < 0) off += a.pitch;
        if (off >= a.width && off + b.width <= a.pitch) return false;
    }
    return true;
}

}  // namespace s2
