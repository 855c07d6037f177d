// Shared prefixes, bf16 models (paged_attention.hip).
#define GLLM_PAGED_PREFIX 1
#include "paged_attention.hip"
