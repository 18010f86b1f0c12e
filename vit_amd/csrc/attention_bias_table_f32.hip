// float32 instances of attention_bias_table.h (a source file each, so that they compile side by side).
#include "attention_bias_table.h"

int vitk_abias_table_f32(const abias::Args& a, const abias::TablePlan& p, float* sums, hipStream_t st) { return table_dispatch<float>(a, p, sums, st); }
