#include "pattn_prompt.h"
void pa_prompt_wide_bf16(const pa_args &a, bool uniform, hipStream_t st) { pa_prompt<MLLM_BF16, true>(a, uniform, st); }
