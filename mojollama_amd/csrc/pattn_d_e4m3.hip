#include "pattn_decode.h"
void pa_decode_e4m3(const pa_args &a, bool wide, bool uniform, hipStream_t st) { pa_decode<MLLM_E4M3>(a, wide, uniform, st); }
