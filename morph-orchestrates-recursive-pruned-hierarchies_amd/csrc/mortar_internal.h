// Shared declarations of libmortar_hip.so (host side).
#ifndef MORTAR_INTERNAL_H
#define MORTAR_INTERNAL_H

#include "../../include/mortar_hip.h"

// Records the calling thread's error message and returns `code`.
int mortar_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

int mortar_check_bcsr_host(const int32_t *row_ptr, const int16_t *col, int32_t Rb, int32_t Cb);

// The kernels address the octet stream with 32-bit byte offsets (1 KiB of 4-bit codes per octet): refuses larger matrices.
// Cb and seg_cb are positive.
__attribute__((visibility("hidden"))) int mortar_check_octets(const mortar_bcsr_t *W);

// Plain product on the +-1 / 0 codes alone, unrounded: y32[m, :] = sum over the kept blocks of codes . x[m, :] in fp32
// (the one-scale kernels with the scale left out).  Returns MORTAR_NO_KERNEL when the pack has no such kernel for M rows.
__attribute__((visibility("hidden"))) int mortar_spmm_codes_f32(const mortar_bcsr_t *W, const int32_t *sched, const uint16_t *x,
                                                                 int64_t M, int64_t ldx, float *y32, int64_t ldy, void *stream);

// qv[m, :] = x[m, :] W^T + bias for few tokens (bias may be null): K shared by the waves of a workgroup.  The caller has checked
// the shapes: d_in % 8 == 0, d_in <= 2048, d_out % 4 == 0, all pointers and rows 16-byte aligned.  xn [M, d_in], M <= 16: the rows of x
// are RMS-normalised first (norm_w may be null) and written there as well.
__attribute__((visibility("hidden"))) int mortar_router_project_skinny(const uint16_t *x, int64_t M, int32_t d_in, int64_t ldx, const float *wq,
                                                                       int32_t d_out, const float *bias, float *qv, int64_t ldq, void *stream,
                                                                       const uint16_t *norm_w = nullptr, float eps = 0.f, uint16_t *xn = nullptr);

// Tile (index into DENSE_TILES) and number of K ranges of a dense product C [M, N] of `steps` K steps (64 16-bit values, 128 e4m3 values).
struct MortarDensePlan {
    int tile, splits;
};
enum { MORTAR_PLAN_PLAIN, MORTAR_PLAN_SWIGLU, MORTAR_PLAN_SWIGLU_KEEP, MORTAR_PLAN_SWIGLU_BWD, MORTAR_PLAN_E4M3 };
__attribute__((visibility("hidden"))) MortarDensePlan mortar_dense_plan(int64_t M, int64_t N, int64_t steps, int form);
// Whether an e4m3 product is the few-rows kernel's.
__attribute__((visibility("hidden"))) bool mortar_fp8_few_rows(int64_t M, int64_t N, int64_t K);
// c = the sum of the fp32 slabs [M, N] of the K ranges, in their order, rounded to `type` (bf16, fp16).
__attribute__((visibility("hidden"))) int mortar_dense_join(const float *slabs, int splits, int64_t M, int64_t N, int32_t type, void *c, int64_t ldc, void *stream);

#endif
