// Error words of the kernels with bounded waits besides SPConvMM's: read and cleared by d3d_debug_take_kernel_error.
#pragma once

namespace d3d {
int take_int8_linear_error(int* code);
}  // namespace d3d
