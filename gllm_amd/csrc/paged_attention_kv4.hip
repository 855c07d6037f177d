// 4-bit KV cache, bf16 models (paged_attention.hip).
#define GLLM_PAGED_KV4 1
#include "paged_attention.hip"
