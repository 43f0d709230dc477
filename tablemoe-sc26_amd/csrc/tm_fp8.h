// Internal entry points of the 8-bit kernels shared between translation units
// (hidden from the shared object's symbol table).
#pragma once

#include "tm_common.h"

// tm_fp8_quantize_rows on checked arguments.
__attribute__((visibility("hidden"))) int tm_internal_fp8_rows(int32_t dtype, const void *x, int64_t n, int64_t k,
                                                               int64_t ld_x, void *q, int64_t ld_q, float *scale,
                                                               int64_t ld_s, hipStream_t s);
