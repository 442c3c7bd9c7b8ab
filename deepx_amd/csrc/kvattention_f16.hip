// kvattention_f16.hip — the attention kernels (kvattention.hpp) for f16 rows
#include "kvattention.hpp"

int dxh::kvattention_f16(const AttArgs &a, bool i8, hipStream_t st) { return i8 ? kvattention_launch<f16_t, CodeI8>(a, st) : kvattention_launch<f16_t, CodeE4M3>(a, st); }
