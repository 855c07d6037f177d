// Generic attention with a sliding window, f32 models (generic_attention.hip).
#define GLLM_GENERIC_QT float
#define GLLM_GENERIC_LAUNCH launch_window_f32
#define GLLM_GENERIC_WINDOW 1
#include "generic_attention.hip"
