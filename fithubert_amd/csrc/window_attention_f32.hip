// The window attention's kernels for fp32 (a translation unit per element type: they compile side by side).
#include "window_attention.cuh"

WIN_INSTANCE(f32, float)
