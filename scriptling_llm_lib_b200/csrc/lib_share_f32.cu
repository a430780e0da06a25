// Attention over shared pages, 32-bit elements.
#include "share_kernels.cuh"
#define ELEM float
#define FN(name) sllm_##name##_f32
#include "share_launchers.inc"
