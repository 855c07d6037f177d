// Sparse attention on the generic kernel, fp32 models (generic_attention.hip).
#define GLLM_GENERIC_QT float
#define GLLM_GENERIC_LAUNCH launch_sparse_generic_f32
#define GLLM_GENERIC_SPARSE 1
#include "generic_attention.hip"
