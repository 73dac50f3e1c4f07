#include "pattn_prompt.h"
void pa_prompt_wide_f16(const pa_args &a, bool uniform, hipStream_t st) { pa_prompt<MLLM_F16, true>(a, uniform, st); }
