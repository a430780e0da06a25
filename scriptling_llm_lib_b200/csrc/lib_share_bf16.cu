// Attention over shared pages, bfloat16 elements: the widths that the tcgen05 form does not take, and the joining of partial results.
#include "share_kernels.cuh"
#define ELEM bf16
#define FN(name) sllm_##name##_bf16
#include "share_launchers.inc"
