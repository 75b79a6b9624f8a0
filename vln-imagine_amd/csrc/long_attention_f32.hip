// float32 instances of the long-sequence attention kernels (v_mfma_f32_32x32x2_f32: exact products, the parity path); a file of their own
// because the three types together are the slowest source to compile.
#include "long_attention.h"

#include "long_attention_impl.inc"

int la_run_f32(const LaP& p, int what, hipStream_t st) { return la_run<float>(p, what, st); }
