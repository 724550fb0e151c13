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

// True when a and b may share bytes. Equal pitches are told apart by columns (two column
// ranges of one wider buffer do not overlap); else their whole extents are compared.
inline bool may_overlap(const PitchedSpan &a, const PitchedSpan &b)
{
    if (!a.ptr || !b.ptr || a.rows <= 0 || b.rows <= 0) return false;
    const __int128 pa = reinterpret_cast<uintptr_t>(a.ptr), pb = reinterpret_cast<uintptr_t>(b.ptr);
    const __int128 ea = pa + static_cast<__int128>(a.rows - 1) * a.pitch + a.width;
    const __int128 eb = pb + static_cast<__int128>(b.rows - 1) * b.pitch + b.width;
    if (ea <= pb || eb <= pa) return false;
    if (a.pitch == b.pitch && a.pitch > 0) {
        __int128 off = (pb - pa) % a.pitch;
        if (off < 0) off += a.pitch;
        if (off >= a.width && off + b.width <= a.pitch) return false;
    }
    return true;
}

}  // namespace s2
