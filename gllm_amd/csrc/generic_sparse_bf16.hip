// Sparse attention on the generic kernel, bf16 models (generic_attention.hip).
#define GLLM_GENERIC_QT __bf16
#define GLLM_GENERIC_LAUNCH launch_sparse_generic_bf16
#define GLLM_GENERIC_SPARSE 1
#include "generic_attention.hip"
