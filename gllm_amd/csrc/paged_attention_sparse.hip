// Sparse attention, bf16 models (paged_attention.hip).
#define GLLM_PAGED_SPARSE 1
#include "paged_attention.hip"
