#include "pattn_decode.h"
void pa_decode_bf16(const pa_args &a, bool wide, bool uniform, hipStream_t st) { pa_decode<MLLM_BF16>(a, wide, uniform, st); }
