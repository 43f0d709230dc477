// Internal entry points of the 8-bit kernels shared between translation units
// (hidden from the shared object's symbol table).
#pragma once

#include "tm_common.h"

// What tm_internal_fp8_rows writes: e4m3 values; the same values as bf16; bf16
// values q * s without scales.
enum { kFp8Rows8 = 0, kFp8Rows16, kFp8RowsScaled };

// tm_fp8_quantize_rows on checked arguments (row stride of q in elements).
__attribute__((visibility("hidden"))) int tm_internal_fp8_rows(int32_t dtype, const void *x, int64_t n, int64_t k,
                                                               int64_t ld_x, void *q, int64_t ld_q, float *scale,
                                                               int64_t ld_s, int out, hipStream_t s);
// e4m3 rows (16-byte aligned, k a multiple of 8) as bf16.
__attribute__((visibility("hidden"))) int tm_internal_fp8_widen(const void *q, int64_t n, int64_t k, int64_t ld_q,
                                                                void *out, int64_t ld_o, hipStream_t s);
