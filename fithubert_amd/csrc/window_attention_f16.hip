// The window attention's kernels for IEEE half (a translation unit per element type: they compile side by side).
#include "window_attention.cuh"

WIN_INSTANCE(f16, f16)
