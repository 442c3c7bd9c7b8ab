// kvattention_f32.hip — the attention kernels (kvattention.hpp) for f32 rows
#include "kvattention.hpp"

int dxh::kvattention_f32(const AttArgs &a, bool i8, hipStream_t st) { return i8 ? kvattention_launch<float, CodeI8>(a, st) : kvattention_launch<float, CodeE4M3>(a, st); }
