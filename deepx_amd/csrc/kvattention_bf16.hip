// kvattention_bf16.hip — the attention kernels (kvattention.hpp) for bf16 rows
#include "kvattention.hpp"

int dxh::kvattention_bf16(const AttArgs &a, bool i8, hipStream_t st) { return i8 ? kvattention_launch<bf16_t, CodeI8>(a, st) : kvattention_launch<bf16_t, CodeE4M3>(a, st); }
