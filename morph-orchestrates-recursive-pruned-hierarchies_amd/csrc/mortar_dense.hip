// The SwiGLU MLP of a block that is not carved: dense products in bf16 or fp16, forward and backward.
//
// Forward:   g = x Wg^T, u = x Wu^T, h = silu(g) u  in one kernel (DENSE_SWIGLU),  y = h Wd^T.
// Backward:  dh = dy Wd with the SwiGLU derivative in its epilogue (DENSE_SWIGLU_BWD): d_up = dh silu(g),
//            d_gate = dh u (s + silu(g) (1 - s)), s = sigmoid(g), and h once more, so that only g and u are kept from the
//            forward;  dx = dgu Wgu,  dWgu = dgu^T x,  dWd = dy^T h.
// Sums, silu and its derivative are fp32.  Rounded to 16 bits are what goes through memory as an operand of a matrix product
// (h, dgu) and the results; h and the derivatives are formed from the unrounded sums of their own kernel, and from g and u as
// kept, in 24 bits.
//
// Measured at 4096 rows, 2048 and 5632 wide, bf16: g, u, h 146 to 150 us (1.3 PFLOP/s), with g and u kept 184 (the 138 MB are written between
// products, at 5 TB/s), y 83 to 91 (1.1), the derivative 151 alone and 167 behind the forward (138 MB read, 138 written), dWd 97, dWgu 185, dx
// 162 + 16 for the join of its K ranges (1.0 to 1.1).  The library's product of 4096 x 2048 x 11264 takes 163 (1.16).
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

// Which tile, and in how many K ranges: the smallest estimate of
//   launch + rounds of workgroups * (steps * time of a step + end of a tile + its output bytes at a CU's share of the memory)
// with, for K ranges, a second launch and the slabs' way out and back.  The times are those of the kernels as they are, fitted to 16-bit
// products of 100 to 16384 rows and widths of 88 to 11264, the operands in the caches and in none of them (geometric mean of the two).  Over 396 others
// the choice is 0.8 % slower than the best tile and number of ranges on average, 15 % at worst; the best number of ranges of the fourth tile
// alone 12 %, of the first 45 % on average.  The backward of SwiGLU reads as much as it writes: above 6 M values a byte is dearer by
// TIMES_BWD, most in the large tiles, where the values on their way do not fit the registers.  Of 494 such products (1 to 20000 rows, widths 64 to 11264)
// the choice is 0.3 % slower than the best tile on average, of the 139 above the line 0.4 % and 11 % at worst; with one price it is 2.6 %, 8.8 %
// and 31 %.  (16384 rows, 768 and 2048 wide: 161, 153, 140 and 146 us in the first four tiles; 4096 rows, 2048 and 5632: 192, 152, 149 and 158.)
struct TileTimes {
    double step, step_alone, end;      // us; a step of one of several workgroups on a CU, of a workgroup alone there
};
constexpr TileTimes TIMES_16[DENSE_N_TILES] = {{1.31, 1.31, 0.1}, {1.10, 1.10, 0.1}, {0.84, 0.84, 0.65}, {1.06, 0.68, 0.44}, {0.46, 0.26, 1.0}};
// e4m3 (from DENSE_E4M3_FIRST on): from 4096 x 2048 x 11264, 4096 x 8192 x 4096 and 8192^3.  Over 470 products of 33 to 9000 rows the choice is 2.3 % slower
// than the best tile and number of ranges on average (33 to 128 rows 1.5, 129 to 2399 3.2, above 0.9), 41 % at worst.
constexpr TileTimes TIMES_8[DENSE_N_TILES] = {{}, {1.48, 1.48, 10.8}, {1.19, 1.19, 3.8}, {1.28, 0.75, 0.3}, {0.6, 0.33, 1.2}};
constexpr double TIMES_BWD[DENSE_N_TILES] = {2.1, 1.8, 1.2, 1.2, 1.2};

Plan plan_tiles(int64_t M, int64_t N, int64_t steps, int form) {
    constexpr double byte = 3.7e-5, launch = 4.8, join = 2.0, slab_byte = 2.4e-7;
    constexpr int ranges[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16};
    const TileTimes *times = form == MORTAR_PLAN_E4M3 ? TIMES_8 : TIMES_16;
    const bool swiglu = form == MORTAR_PLAN_SWIGLU || form == MORTAR_PLAN_SWIGLU_KEEP, plain = form == MORTAR_PLAN_PLAIN || form == MORTAR_PLAN_E4M3;
    const int out = form == MORTAR_PLAN_SWIGLU_BWD ? 12 : form == MORTAR_PLAN_SWIGLU_KEEP ? 8 : 2;
    Plan best{0, 1};
    double best_t = 1e300;
    for (int c = form == MORTAR_PLAN_E4M3 ? DENSE_E4M3_FIRST : 0; c < DENSE_N_TILES; ++c) {
        const int64_t bn = swiglu ? DENSE_TILES[c].bn / 2 : DENSE_TILES[c].bn, bm = DENSE_TILES[c].bm;
        const int64_t tiles = ((N + bn - 1) / bn) * ((M + bm - 1) / bm);
        for (const int s : ranges) {
            if (s > 1 && (!plain || steps / s < 4)) break;
            const int64_t wgs = (tiles * s + 255) / 256, both = wgs < DENSE_TILES[c].per_cu ? wgs : DENSE_TILES[c].per_cu;
            const double each = byte * (form == MORTAR_PLAN_SWIGLU_BWD && M * N > 6 << 20 ? TIMES_BWD[c] : 1);
            const double step = both == DENSE_TILES[c].per_cu ? times[c].step : times[c].step_alone;
            double t = launch + (double)wgs / both * ((double)((steps + s - 1) / s) * step + times[c].end + both * each * bn * bm * (s > 1 ? 4 : out));
            if (s > 1) t += join + slab_byte * s * M * N * 4;
            if (t < best_t) {
                best_t = t;
                best = Plan{c, s};
            }
        }
    }
    return best;
}

// Adds the slabs of the K ranges in their order, up to eight loads in flight.
template <DenseType T>
__global__ __launch_bounds__(256) void dense_join_kernel(const float *slabs, int splits, int64_t M, int64_t N, uint16_t *c, int64_t ldc) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = N >> 2;
    if (i >= M * per) return;
    const int64_t m = i / per, n = (i - m * per) * 4, slab = M * N / 4;
    const f32x4_t *p = reinterpret_cast<const f32x4_t *>(slabs + m * N + n);
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; s += 8) {
        f32x4_t v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = p[(s + k < splits ? s + k : s) * slab];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s + k < splits) sum += v[k];
    }
    *reinterpret_cast<u32x2_t *>(c + m * ldc + n) = u32x2_t{dense_pack2<T>(sum[0], sum[1]), dense_pack2<T>(sum[2], sum[3])};
}

// One plain product into 16-bit C, over K ranges where the plan has them.
template <DenseType T, bool PC, bool QC>
int run_plain(DenseArgs a, float *ws, hipStream_t st, const char *what) {
    a.steps = (a.K + 63) / 64;
    const Plan p = plan_tiles(a.M, a.N, a.steps, MORTAR_PLAN_PLAIN);
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
// Up to 8 rows the weights are the traffic, and the launch.  A workgroup owns 8 rows of W (with SWIGLU 8 gate rows and their up rows); the
// matrix instruction's 16 rows and 16 columns hold two halves of K side by side, so that two of the four quarters of its result
// are sums and the others are not used (with 16 rows per workgroup instead, `down` of 2048 rows keeps half of the chip).  W goes
// straight into the operand registers, U turns of 64 values per half and wave in flight, while x is staged in LDS (read as
// operands from memory it costs as many load cycles as W); the waves' and halves' sums meet there.  2048 / 5632, weights in no cache:
// gate_up 10.2 us at one row and 11.7 at eight, down 5.9 and 7.7, where plain reads of the weights take 9.3 and 4.8 and the 64 x 64
// tile 13.1 and 9.6 (its rows are then free up to 64).
constexpr int FEW_ROWS = MORTAR_DENSE_FEW_ROWS, FEW_LDS = 96 * 1024;

// x rows in LDS: two halves of whole turns, and 16 bytes so that the rows start on different banks.
constexpr int64_t few_pitch(int64_t K) { return ((K + 63) / 64 + 1) / 2 * 256 + 16; }

template <DenseType T, bool SWIGLU, int NW, int U>
__global__ __launch_bounds__(NW * 64) void dense_few_kernel(const DenseArgs a) {
    constexpr int RS = SWIGLU ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    f32x4_t *part = reinterpret_cast<f32x4_t *>(smem);                      // [wave][row set][lane]
    unsigned char *xs = smem + NW * RS * 1024;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int n0 = blockIdx.x * 8, turns = (((a.K + 63) >> 6) + 1) >> 1, half = (r >> 3) * turns * 128;       // (half: bytes in front of it)
    const int pitch = turns * 256 + 16;
    __amdgpu_buffer_rsrc_t wb[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s)
        wb[s] = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(static_cast<const char *>(a.p) + ((int64_t)n0 + (int64_t)s * a.N) * a.ldp), 0, DENSE_OUTSIDE, 0x00020000);
    const uint32_t wo = (uint32_t)((r & 7) * a.ldp) + half + g * 16;
    const int left = a.K * 2 - half - g * 16;                               // bytes of the row behind this lane's first unit
    const unsigned char *xl = xs + min(r & 7, a.M - 1) * pitch + half + g * 16;

    f32x4_t acc[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s) acc[s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int c0 = wave; c0 < turns || c0 == wave; c0 += NW * U) {
        u32x4_t w[U][2][RS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * NW < turns ? c0 + u * NW : 0;            // (beyond the end: not used)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int s = 0; s < RS; ++s)
                    w[u][h][s] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(wb[s], c * 128 + h * 64 < left ? wo : DENSE_OUTSIDE, c * 128 + h * 64, 0));
        }
        if (c0 == wave) {                                                   // every wave once
            const int units = turns * 16;
            for (int i = threadIdx.x; i < a.M * units; i += NW * 64) {
                const int m = i / units, u = i - m * units;
                u32x4_t v = {0, 0, 0, 0};
                if (u * 8 < a.K) v = *reinterpret_cast<const u32x4_t *>(static_cast<const char *>(a.q) + m * a.ldq + u * 16);
                *reinterpret_cast<u32x4_t *>(xs + m * pitch + u * 16) = v;
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * NW < turns)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4_t x = *reinterpret_cast<const u32x4_t *>(xl + (c0 + u * NW) * 128 + h * 64);
#pragma unroll
                    for (int s = 0; s < RS; ++s) acc[s] = dense_mfma<T>(w[u][h][s], x, acc[s]);
                }
    }
#pragma unroll
    for (int s = 0; s < RS; ++s) part[(wave * RS + s) * 64 + lane] = acc[s];
    __syncthreads();
    if (wave || g > 1 || r >= a.M) return;                                  // lane: token r, features 4 g .. 4 g + 3
    f32x4_t sum[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        sum[s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) sum[s] += part[(w * RS + s) * 64 + lane] + part[(w * RS + s) * 64 + lane + 40];       // + 40: the other half of K
    }
    const int64_t m = r;
    const int n = n0 + 4 * g;
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

bool few_rows(int64_t M, int64_t N, int64_t K) { return M <= FEW_ROWS && M * few_pitch(K) <= FEW_LDS && N <= 1 << 24; }        // (a grid has 2^32 threads at most)

template <DenseType T, bool SWIGLU, int NW, int U>
int launch_few_form(const DenseArgs &a, hipStream_t st, const char *what) {
    const auto kern = dense_few_kernel<T, SWIGLU, NW, U>;
    constexpr int sums = NW * (SWIGLU ? 2 : 1) * 1024;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, sums + FEW_LDS);
    if (e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.N / 8)), dim3(NW * 64), sums + a.M * few_pitch(a.K), st, a);
    return launch_error(what);
}
template <DenseType T, bool SWIGLU>
int launch_few(const DenseArgs &a, hipStream_t st, const char *what) {
    if constexpr (SWIGLU) return launch_few_form<T, true, 8, 2>(a, st, what);
    else return launch_few_form<T, false, 16, 3>(a, st, what);
}

// ---- checks ----------------------------------------------------------------------------------------------------------

// A [rows, cols] matrix of 16-bit values as the kernels read it: 16-byte rows, 256 of which lie within 2 GiB (DENSE_OUTSIDE: a tile is addressed in 32 bits).
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

MortarDensePlan mortar_dense_plan(int64_t M, int64_t N, int64_t steps, int form) { return plan_tiles(M, N, steps, form); }

int mortar_dense_join(const float *slabs, int splits, int64_t M, int64_t N, int32_t type, void *c, int64_t ldc, void *stream) {
    const int64_t n = M * (N / 4);
    if ((n + 255) / 256 >= INT32_MAX) return mortar_fail(MORTAR_ERR_LIMIT, "dense: too many results");
    const auto kern = type == MORTAR_FP16 ? dense_join_kernel<DENSE_F16> : dense_join_kernel<DENSE_BF16>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), slabs, splits, M, N,
                       static_cast<uint16_t *>(c), ldc);
    return launch_error("dense");
}

extern "C" int64_t mortar_dense_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const Plan p = plan_tiles(M, N, (K + 63) / 64, MORTAR_PLAN_PLAIN);
    return p.splits > 1 ? p.splits * M * N * 4 : 0;
}

extern "C" int mortar_dense_form_host(int32_t kind, int64_t M, int64_t N, int64_t K, int32_t *tile_n, int32_t *tile_m, int32_t *ranges) {
    if (kind < 0 || kind > 5 || M <= 0 || N <= 0 || K <= 0 || !tile_n || !tile_m || !ranges) return mortar_fail(MORTAR_ERR_ARG, "dense_form: bad argument");
    constexpr int forms[] = {MORTAR_PLAN_PLAIN, MORTAR_PLAN_PLAIN, MORTAR_PLAN_SWIGLU, MORTAR_PLAN_SWIGLU_KEEP, MORTAR_PLAN_SWIGLU_BWD, MORTAR_PLAN_E4M3};
    const bool few = kind == 5 ? mortar_fp8_few_rows(M, N, K) : kind != 1 && kind != 4 && few_rows(M, N, K);
    const Plan p = few ? Plan{0, 1} : plan_tiles(M, N, kind == 5 ? (K + 127) / 128 : (K + 63) / 64, forms[kind]);
    *tile_n = few ? 0 : DENSE_TILES[p.tile].bn;
    *tile_m = few ? 0 : DENSE_TILES[p.tile].bm;
    *ranges = p.splits;
    return MORTAR_OK;
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
    if (few_rows(M, a.N, a.K)) return type == MORTAR_BF16 ? launch_few<DENSE_BF16, true>(a, st, what) : launch_few<DENSE_F16, true>(a, st, what);
    const Plan p = plan_tiles(M, f, a.steps, gu ? MORTAR_PLAN_SWIGLU_KEEP : MORTAR_PLAN_SWIGLU);
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
    if (few_rows(M, a.N, a.K)) return type == MORTAR_BF16 ? launch_few<DENSE_BF16, false>(a, st, what) : launch_few<DENSE_F16, false>(a, st, what);
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
    const Plan p = plan_tiles(M, f, a.steps, MORTAR_PLAN_SWIGLU_BWD);
    return type == MORTAR_BF16 ? dense_launch<DENSE_BF16, DENSE_SWIGLU_BWD, true, false>(a, p.tile, st, what)
                               : dense_launch<DENSE_F16, DENSE_SWIGLU_BWD, true, false>(a, p.tile, st, what);
}
