// float32 instances of attention_bias_dq.h (a source file each, so that they compile side by side).
#include "attention_bias_dq.h"

int vitk_abias_dq_f32(const abias::Args& a, bool sums, hipStream_t st) { return dq_dispatch<float>(a, sums, st); }
