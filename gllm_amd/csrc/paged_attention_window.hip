// Sliding windows, bf16 models (paged_attention.hip).
#define GLLM_PAGED_WINDOW 1
#include "paged_attention.hip"
