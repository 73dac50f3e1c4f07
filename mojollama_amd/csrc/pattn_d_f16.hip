#include "pattn_decode.h"
void pa_decode_f16(const pa_args &a, bool wide, bool uniform, hipStream_t st) { pa_decode<MLLM_F16>(a, wide, uniform, st); }
