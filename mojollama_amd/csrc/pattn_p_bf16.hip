#include "pattn_prompt.h"
void pa_prompt_bf16(const pa_args &a, bool uniform, hipStream_t st) { pa_prompt<MLLM_BF16, false>(a, uniform, st); }
