// Sparse attention, fp16 models (paged_attention.hip).
#define GLLM_PAGED_F16 1
#define GLLM_PAGED_SPARSE 1
#include "paged_attention.hip"
