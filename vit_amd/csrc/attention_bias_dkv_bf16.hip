// bfloat16 instances of attention_bias_dkv.h (a source file each, so that they compile side by side).
#include "attention_bias_dkv.h"

int vitk_abias_dkv_bf16(const abias::Args& a, hipStream_t st) { return dkv_dispatch<bf16_t>(a, st); }
