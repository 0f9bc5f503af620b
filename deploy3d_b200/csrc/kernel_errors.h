// What the kernels with bounded waits share: the limit that d3d_debug_set_wait_limit sets, and the error words of those besides
// SPConvMM's, read and cleared by d3d_debug_take_kernel_error.
#pragma once
#include <stdint.h>

namespace d3d {
uint32_t wait_limit();  // cycles
int take_int8_linear_error(int* code);
}  // namespace d3d
