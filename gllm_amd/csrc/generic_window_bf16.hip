// Generic attention with a sliding window, bf16 models (generic_attention.hip).
#define GLLM_GENERIC_QT __bf16
#define GLLM_GENERIC_LAUNCH launch_window_bf16
#define GLLM_GENERIC_WINDOW 1
#include "generic_attention.hip"
