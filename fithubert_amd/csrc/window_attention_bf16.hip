// The window attention's kernels for bf16 (a translation unit per element type: they compile side by side).
#include "window_attention.cuh"

WIN_INSTANCE(bf16, bf16)
