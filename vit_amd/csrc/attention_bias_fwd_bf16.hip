// bfloat16 instances of attention_bias_fwd.h (a source file each, so that they compile side by side).
#include "attention_bias_fwd.h"

int vitk_abias_fwd_bf16(const abias::Args& a, hipStream_t st) { return fwd_dispatch<bf16_t>(a, st); }
