#include "pattn_prompt.h"
void pa_prompt_e4m3(const pa_args &a, bool uniform, hipStream_t st) { pa_prompt<MLLM_E4M3, false>(a, uniform, st); }
