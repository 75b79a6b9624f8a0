// float16 instances of the long-sequence attention kernels
#include "long_attention.h"

#include "long_attention_impl.inc"

int la_run_f16(const LaP& p, int what, hipStream_t st) { return la_run<_Float16>(p, what, st); }
