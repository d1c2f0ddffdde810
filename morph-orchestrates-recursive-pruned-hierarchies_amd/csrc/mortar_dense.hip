// The SwiGLU MLP of a block that is not carved: dense products in bf16 or fp16, forward and backward.
//
// Forward:   g = x Wg^T, u = x Wu^T, h = silu(g) u  in one kernel (DENSE_SWIGLU),  y = h Wd^T.
// Backward:  dh = dy Wd with the SwiGLU derivative in its epilogue (DENSE_SWIGLU_BWD): d_up = dh silu(g),
//            d_gate = dh u (s + silu(g) (1 - s)), s = sigmoid(g), and h once more, so that only g and u are kept from the
//            forward;  dx = dgu Wgu,  dWgu = dgu^T x,  dWd = dy^T h.
// Sums, silu and its derivative are fp32.  Rounded to 16 bits are what goes through memory as an operand of a matrix product
// (h, dgu) and the results; h and the derivatives are formed from the unrounded sums of their own kernel, and from g and u as
// kept, in 24 bits.
#include <hip/hip_runtime.h>

#include "mortar_dense_core.h"
#include "mortar_internal.h"

namespace {

int launch_error(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// ---- tile products ---------------------------------------------------------------------------------------------------

using Plan = MortarDensePlan;

// Which tile, and in how many K ranges, from the estimated cycles of the busiest CU: what a step of a tile takes with the chip full (measured,
// at the 2 GHz that the chip runs under this load; workgroups that share a CU share its matrix cores), and no less than the way of
// its copies; a tile's start and end; for K ranges a pass over their fp32 slabs and a launch.
Plan plan_tiles(int64_t M, int64_t N, int64_t K, bool swiglu, bool may_split) {
    constexpr double step_cycles[DENSE_N_TILES] = {2900, 2230, 1770, 920, 440}, way[DENSE_N_TILES] = {1500, 1500, 1000, 1500, 700};
    constexpr double ends = 5000, slab_byte = 2 * 0.0005, launch = 8000;
    const int64_t steps = (K + 63) / 64;
    Plan best{0, 1};
    double best_t = 1e300;
    for (int c = 0; c < DENSE_N_TILES; ++c) {
        const int64_t bn = swiglu ? DENSE_TILES[c].bn / 2 : DENSE_TILES[c].bn, bm = DENSE_TILES[c].bm;
        const int64_t tiles = ((N + bn - 1) / bn) * ((M + bm - 1) / bm);
        for (int s = 1; s <= 16; s *= 2) {
            if (s > 1 && (!may_split || steps / s < 4)) break;
            const int64_t wgs = (tiles * s + 255) / 256, both = wgs < DENSE_TILES[c].per_cu ? wgs : DENSE_TILES[c].per_cu;
            const double rounds = (double)wgs / both, per_step = both * step_cycles[c] > way[c] ? both * step_cycles[c] : way[c];
            double t = rounds * ((double)((steps + s - 1) / s) * per_step + ends);
            if (s > 1) t += launch + slab_byte * s * M * N * 4;
            if (t < best_t) {
                best_t = t;
                best = Plan{c, s};
            }
        }
    }
    return best;
}

// Adds the slabs of the K ranges in their order.
template <DenseType T>
__global__ __launch_bounds__(256) void dense_join_kernel(const float *slabs, int splits, int64_t M, int64_t N, uint16_t *c, int64_t ldc) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = N >> 3;
    if (i >= M * per) return;
    const int64_t m = i / per, n = (i - m * per) * 8;
    const f32x4_t *p = reinterpret_cast<const f32x4_t *>(slabs + m * N + n);
    f32x4_t lo = p[0], hi = p[1];
    for (int s = 1; s < splits; ++s) {
        p += M * N / 4;
        lo += p[0];
        hi += p[1];
    }
    const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    *reinterpret_cast<u32x4_t *>(c + m * ldc + n) = dense_pack8<T>(v);
}

// One plain product into 16-bit C, over K ranges where the plan has them.
template <DenseType T, bool PC, bool QC>
int run_plain(DenseArgs a, float *ws, hipStream_t st, const char *what) {
    const Plan p = plan_tiles(a.M, a.N, a.K, false, true);
    a.steps = (a.K + 63) / 64;
    a.splits = p.splits;
    if (p.splits == 1) return dense_launch<T, DENSE_STORE, PC, QC>(a, p.tile, st, what);
    if (!ws) return mortar_fail(MORTAR_ERR_ARG, "%s: this shape needs a workspace", what);
    DenseArgs b = a;
    b.c = ws;
    const int rc = dense_launch<T, DENSE_PARTIAL, PC, QC>(b, p.tile, st, what);
    if (rc) return rc;
    return mortar_dense_join(ws, p.splits, a.M, a.N, T == DENSE_F16 ? MORTAR_FP16 : MORTAR_BF16, a.c, a.ldc, st);
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// Up to 64 rows the weights are the traffic: a workgroup owns 16 rows of W (with SWIGLU the 16 gate rows and their up rows),
// its waves take K in turns of 64 values and read W straight into the matrix cores' operand registers, U turns (2 U loads per
// row set) in flight; the waves' sums meet in LDS.
constexpr int FEW_ROWS = 64;

__device__ __forceinline__ u32x4_t buffer_read(__amdgpu_buffer_rsrc_t buf, uint32_t off) {
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(buf, off, 0, 0));
}

template <DenseType T, bool SWIGLU, int MT, int NW, int U>
__global__ __launch_bounds__(NW * 64) void dense_few_kernel(const DenseArgs a) {
    constexpr int RS = SWIGLU ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) f32x4_t part[];          // [wave][row set][token tile][lane]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int n0 = blockIdx.x * 16;
    const auto whole = [](const void *p) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, DENSE_OUTSIDE, 0x00020000); };
    __amdgpu_buffer_rsrc_t wb[RS], xb = whole(a.q);
    uint32_t wo, xo[MT];
#pragma unroll
    for (int s = 0; s < RS; ++s) wb[s] = whole(static_cast<const char *>(a.p) + ((int64_t)n0 + (int64_t)s * a.N) * a.ldp);
    wo = n0 + r < a.N ? (uint32_t)(r * a.ldp) + g * 16 : DENSE_OUTSIDE;
#pragma unroll
    for (int t = 0; t < MT; ++t) xo[t] = t * 16 + r < a.M ? (uint32_t)((t * 16 + r) * a.ldq) + g * 16 : DENSE_OUTSIDE;

    f32x4_t acc[RS][MT];
#pragma unroll
    for (int s = 0; s < RS; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[s][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int turns = (a.K + 63) / 64;
    for (int c0 = wave; c0 < turns; c0 += NW * U) {
        u32x4_t w[U][2][RS], x[U][2][MT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int kb = (c0 + u * NW) * 128 + h * 64;               // bytes into the rows
                const bool in = kb + g * 16 < a.K * 2;
#pragma unroll
                for (int s = 0; s < RS; ++s) w[u][h][s] = buffer_read(wb[s], in ? wo + kb : DENSE_OUTSIDE);
#pragma unroll
                for (int t = 0; t < MT; ++t) x[u][h][t] = buffer_read(xb, in ? xo[t] + kb : DENSE_OUTSIDE);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int s = 0; s < RS; ++s)
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[s][t] = dense_mfma<T>(w[u][h][s], x[u][h][t], acc[s][t]);
    }
#pragma unroll
    for (int s = 0; s < RS; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) part[((wave * RS + s) * MT + t) * 64 + lane] = acc[s][t];
    __syncthreads();
    if (wave >= MT) return;
    f32x4_t sum[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        sum[s] = part[(s * MT + wave) * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) sum[s] += part[((w * RS + s) * MT + wave) * 64 + lane];
    }
    const int64_t m = wave * 16 + r;
    const int n = n0 + 4 * g;
    if (m >= a.M || n >= a.N) return;
    const auto put = [&](void *c, int64_t at, f32x4_t v) {
        *reinterpret_cast<u32x2_t *>(static_cast<uint16_t *>(c) + at) = u32x2_t{dense_pack2<T>(v[0], v[1]), dense_pack2<T>(v[2], v[3])};
    };
    if constexpr (SWIGLU) {
        f32x4_t h;
#pragma unroll
        for (int v = 0; v < 4; ++v) h[v] = sum[0][v] * dense_sigmoid(sum[0][v]) * sum[RS - 1][v];
        put(a.c, m * a.ldc + n, h);
        if (a.gu) {
            const auto keep = [&](int64_t at, f32x4_t v) {
                const uint32_t b0 = dense_round24(v[0]), b1 = dense_round24(v[1]), b2 = dense_round24(v[2]), b3 = dense_round24(v[3]);
                *reinterpret_cast<u32x2_t *>(a.gu + at) = u32x2_t{dense_hi2(b0, b1), dense_hi2(b2, b3)};
                *reinterpret_cast<uint32_t *>(a.gul + at) = dense_lo4(b0, b1, b2, b3);
            };
            keep(m * 2 * a.N + n, sum[0]);
            keep(m * 2 * a.N + a.N + n, sum[RS - 1]);
        }
    } else {
        put(a.c, m * a.ldc + n, sum[0]);
    }
}

template <DenseType T, bool SWIGLU, int MT, int NW, int U>
int launch_few_form(const DenseArgs &a, hipStream_t st, const char *what) {
    const auto kern = dense_few_kernel<T, SWIGLU, MT, NW, U>;
    constexpr int smem = NW * (SWIGLU ? 2 : 1) * MT * 1024;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    hipLaunchKernelGGL(kern, dim3((unsigned)((a.N + 15) / 16)), dim3(NW * 64), smem, st, a);
    return launch_error(what);
}
template <DenseType T, bool SWIGLU>
int launch_few(const DenseArgs &a, hipStream_t st, const char *what) {
    if (a.M <= 16) return launch_few_form<T, SWIGLU, 1, 16, 2>(a, st, what);
    if (a.M <= 32) return launch_few_form<T, SWIGLU, 2, 16, 2>(a, st, what);
    return launch_few_form<T, SWIGLU, 4, 16, 1>(a, st, what);
}

// ---- checks ----------------------------------------------------------------------------------------------------------

// A [rows, cols] matrix of 16-bit values as the kernels read it: 16-byte rows, and 512 rows or 2 * rows2 of them within 2 GiB of each other.
int check_matrix(const char *what, const char *name, const void *p, int64_t rows, int64_t cols, int64_t ld) {
    if (!p) return mortar_fail(MORTAR_ERR_ARG, "%s: %s is null", what, name);
    if (cols % 8 || ld % 8 || ld < cols || (reinterpret_cast<uintptr_t>(p) & 15))
        return mortar_fail(MORTAR_ERR_ARG, "%s: %s needs rows of a multiple of 8 values on 16-byte addresses", what, name);
    if (rows >= INT32_MAX / 2 || cols >= INT32_MAX / 4) return mortar_fail(MORTAR_ERR_LIMIT, "%s: %s is too large", what, name);
    if (256 * ld * 2 >= (int64_t)DENSE_OUTSIDE) return mortar_fail(MORTAR_ERR_LIMIT, "%s: the rows of %s are too far apart", what, name);
    return MORTAR_OK;
}
int check_type(const char *what, int32_t type) {
    return type == MORTAR_BF16 || type == MORTAR_FP16 ? MORTAR_OK : mortar_fail(MORTAR_ERR_ARG, "%s: bf16 or fp16", what);
}
#define CHECK(...) do { const int rc_ = (__VA_ARGS__); if (rc_) return rc_; } while (0)

}  // namespace

MortarDensePlan mortar_dense_plan(int64_t M, int64_t N, int64_t K, int swiglu, int may_split) { return plan_tiles(M, N, K, swiglu, may_split); }

int mortar_dense_join(const float *slabs, int splits, int64_t M, int64_t N, int32_t type, void *c, int64_t ldc, void *stream) {
    const int64_t n = M * (N / 8);
    if ((n + 255) / 256 >= INT32_MAX) return mortar_fail(MORTAR_ERR_LIMIT, "dense: too many results");
    const auto kern = type == MORTAR_FP16 ? dense_join_kernel<DENSE_F16> : dense_join_kernel<DENSE_BF16>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), slabs, splits, M, N,
                       static_cast<uint16_t *>(c), ldc);
    return launch_error("dense");
}

extern "C" int64_t mortar_dense_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const Plan p = plan_tiles(M, N, K, false, true);
    return p.splits > 1 ? p.splits * M * N * 4 : 0;
}

extern "C" int mortar_dense_gateup_swiglu(const void *x, int64_t M, int32_t d, int64_t ldx, const void *w, int64_t ldw, int32_t f, int32_t type,
                                          void *h, int64_t ldh, void *gu, void *stream) {
    const char *what = "dense_gateup_swiglu";
    if (M < 0 || d <= 0 || f <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    CHECK(check_type(what, type));
    if (M == 0) return MORTAR_OK;
    CHECK(check_matrix(what, "x", x, M, d, ldx));
    CHECK(check_matrix(what, "w", w, 2 * (int64_t)f, d, ldw));
    CHECK(check_matrix(what, "h", h, M, f, ldh));
    if (gu) CHECK(check_matrix(what, "gu", gu, M, 2 * (int64_t)f, 2 * (int64_t)f));
    if ((f + (int64_t)256) * ldw * 2 >= (int64_t)DENSE_OUTSIDE) return mortar_fail(MORTAR_ERR_LIMIT, "%s: w is too large", what);
    DenseArgs a{};
    a.p = w; a.ldp = ldw * 2; a.q = x; a.ldq = ldx * 2;
    a.M = (int32_t)M; a.N = f; a.K = d;
    a.c = h; a.ldc = ldh;
    if (gu) a.gu = static_cast<uint16_t *>(gu), a.gul = static_cast<uint8_t *>(gu) + M * 4 * f;
    a.steps = (d + 63) / 64; a.splits = 1;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (M <= FEW_ROWS) return type == MORTAR_BF16 ? launch_few<DENSE_BF16, true>(a, st, what) : launch_few<DENSE_F16, true>(a, st, what);
    const Plan p = plan_tiles(M, f, d, true, false);
    return type == MORTAR_BF16 ? dense_launch<DENSE_BF16, DENSE_SWIGLU, false, false>(a, p.tile, st, what)
                               : dense_launch<DENSE_F16, DENSE_SWIGLU, false, false>(a, p.tile, st, what);
}

extern "C" int mortar_dense_linear(const void *x, int64_t M, int32_t K, int64_t ldx, const void *w, int64_t ldw, int32_t N, int32_t type, void *y,
                                   int64_t ldy, float *workspace, void *stream) {
    const char *what = "dense_linear";
    if (M < 0 || K <= 0 || N <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    CHECK(check_type(what, type));
    if (M == 0) return MORTAR_OK;
    CHECK(check_matrix(what, "x", x, M, K, ldx));
    CHECK(check_matrix(what, "w", w, N, K, ldw));
    CHECK(check_matrix(what, "y", y, M, N, ldy));
    DenseArgs a{};
    a.p = w; a.ldp = ldw * 2; a.q = x; a.ldq = ldx * 2;
    a.M = (int32_t)M; a.N = N; a.K = K;
    a.c = y; a.ldc = ldy;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (M <= FEW_ROWS) return type == MORTAR_BF16 ? launch_few<DENSE_BF16, false>(a, st, what) : launch_few<DENSE_F16, false>(a, st, what);
    return type == MORTAR_BF16 ? run_plain<DENSE_BF16, false, false>(a, workspace, st, what) : run_plain<DENSE_F16, false, false>(a, workspace, st, what);
}

extern "C" int mortar_dense_linear_dx(const void *dy, int64_t M, int32_t K, int64_t lddy, const void *w, int64_t ldw, int32_t N, int32_t type,
                                      void *dx, int64_t lddx, float *workspace, void *stream) {
    const char *what = "dense_linear_dx";
    if (M < 0 || K <= 0 || N <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    CHECK(check_type(what, type));
    if (M == 0) return MORTAR_OK;
    CHECK(check_matrix(what, "dy", dy, M, K, lddy));
    CHECK(check_matrix(what, "w", w, K, N, ldw));
    CHECK(check_matrix(what, "dx", dx, M, N, lddx));
    DenseArgs a{};
    a.p = w; a.ldp = ldw * 2; a.q = dy; a.ldq = lddy * 2;
    a.M = (int32_t)M; a.N = N; a.K = K;
    a.c = dx; a.ldc = lddx;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return type == MORTAR_BF16 ? run_plain<DENSE_BF16, true, false>(a, workspace, st, what) : run_plain<DENSE_F16, true, false>(a, workspace, st, what);
}

extern "C" int mortar_dense_linear_dw(const void *dy, int64_t M, int32_t n_out, int64_t lddy, const void *x, int64_t ldx, int32_t n_in, int32_t type,
                                      void *dw, int64_t lddw, float *workspace, void *stream) {
    const char *what = "dense_linear_dw";
    if (M <= 0 || n_out <= 0 || n_in <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    CHECK(check_type(what, type));
    CHECK(check_matrix(what, "dy", dy, M, n_out, lddy));
    CHECK(check_matrix(what, "x", x, M, n_in, ldx));
    CHECK(check_matrix(what, "dw", dw, n_out, n_in, lddw));
    DenseArgs a{};
    a.p = x; a.ldp = ldx * 2; a.q = dy; a.ldq = lddy * 2;
    a.M = n_out; a.N = n_in; a.K = (int32_t)M;
    a.c = dw; a.ldc = lddw;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return type == MORTAR_BF16 ? run_plain<DENSE_BF16, true, true>(a, workspace, st, what) : run_plain<DENSE_F16, true, true>(a, workspace, st, what);
}

extern "C" int mortar_dense_swiglu_bwd(const void *dy, int64_t M, int32_t d, int64_t lddy, const void *w, int64_t ldw, int32_t f, int32_t type,
                                       const void *gu, void *dgu, int64_t lddgu, void *h, int64_t ldh, void *stream) {
    const char *what = "dense_swiglu_bwd";
    if (M < 0 || d <= 0 || f <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    CHECK(check_type(what, type));
    if (M == 0) return MORTAR_OK;
    CHECK(check_matrix(what, "dy", dy, M, d, lddy));
    CHECK(check_matrix(what, "w", w, d, f, ldw));
    CHECK(check_matrix(what, "gu", gu, M, 2 * (int64_t)f, 2 * (int64_t)f));
    CHECK(check_matrix(what, "dgu", dgu, M, 2 * (int64_t)f, lddgu));
    if (h) CHECK(check_matrix(what, "h", h, M, f, ldh));
    DenseArgs a{};
    a.p = w; a.ldp = ldw * 2; a.q = dy; a.ldq = lddy * 2;
    a.M = (int32_t)M; a.N = f; a.K = d;
    a.c = dgu; a.ldc = lddgu; a.h = h; a.ldh = ldh;
    a.gu = static_cast<uint16_t *>(const_cast<void *>(gu)); a.gul = static_cast<uint8_t *>(const_cast<void *>(gu)) + M * 4 * f;
    a.steps = (d + 63) / 64; a.splits = 1;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const Plan p = plan_tiles(M, f, d, false, false);
    return type == MORTAR_BF16 ? dense_launch<DENSE_BF16, DENSE_SWIGLU_BWD, true, false>(a, p.tile, st, what)
                               : dense_launch<DENSE_F16, DENSE_SWIGLU_BWD, true, false>(a, p.tile, st, what);
}
