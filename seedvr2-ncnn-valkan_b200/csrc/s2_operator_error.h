// The error word of channels-last operator calls that bring none of their own.
#pragma once

#include <cstdint>

namespace s2 {

// The current device's word; NULL where there is none to be had (no time-out is then reported).
int32_t *operator_error_word();

}  // namespace s2
