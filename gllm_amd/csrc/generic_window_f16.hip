// Generic attention with a sliding window, f16 models (generic_attention.hip).
#define GLLM_GENERIC_QT _Float16
#define GLLM_GENERIC_LAUNCH launch_window_f16
#define GLLM_GENERIC_WINDOW 1
#include "generic_attention.hip"
