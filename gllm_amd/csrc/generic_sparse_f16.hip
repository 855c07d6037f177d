// Sparse attention on the generic kernel, fp16 models (generic_attention.hip).
#define GLLM_GENERIC_QT _Float16
#define GLLM_GENERIC_LAUNCH launch_sparse_generic_f16
#define GLLM_GENERIC_SPARSE 1
#include "generic_attention.hip"
