// Dense layers served in 4 bits: y = x W^T, W = (c - z) s with 4-bit codes c, one scale s and zero point z per row and group of 32, 64 or 128 K.
//   y[m, n] = sum_g s[n, g] ( sum_{k in g} x[m, k] (16 + c[n, k]) - (16 + z[n, g]) sum_{k in g} x[m, k] )
// 16 + c is exact in bf16 and in fp16: a code's four bits are the upper mantissa bits behind the exponent of 16, so that two weights are made
// by one shift and one and-or, and go into the matrix cores beside x as it is.  The sums of a group come out of them unscaled and enter the fp32 result with one
// multiply-add: W is never rounded.  (W in 16 bits instead would cost as much again as the rounding of y.)  What the 16 adds is a few times the
// codes' own size in sums of 24 bits.  It is taken off as a sum of its own, and what the two round differently is left: little beside what the group's weights
// give, but not where they all are 0 (pruned ones, whose scale need not be small).  Such a group gives 0 exactly here:
//   few rows   both sums run through the same instructions in the same order, with 24 in place of a weight of 0, which the code 8 is; with zero points the
//              weights are 24 + (c - z) / 2: half a code, added to the bits of the row's 24 - z / 2 instead of set in those of 16.  Zero points beyond 15,
//              which no code reaches, count as 15, and (z - 15) / 2 sums of x are taken off besides.
//   many rows  a subtraction more per result and group takes 3 to 15 % longer, looking at the codes beside the products 3 to 17 %: the launch in front reads
//              them instead (1 to 2 us for 23 million weights) and gives groups of zeros the scale 0.
// The codes of a word lie so that one shift brings a pair of neighbours into its two halves.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mortar_dense_core.h"
#include "mortar_internal.h"

namespace {

// Rows of x in LDS: whole chunks, and 16 bytes so that they start on different banks.
__host__ __device__ constexpr int int4_pitch(int K) { return (K + 127) / 128 * 256 + 16; }

struct Int4Args {
    const void *x;
    int64_t ldx;                         // bytes
    const uint32_t *c;
    int64_t ldc;                         // bytes
    const void *s;
    int64_t s_n, s_g;                    // values
    const uint8_t *z;
    int64_t z_n, z_g;
    uint16_t *y;
    int64_t ldy;
    int32_t M, N, K, groups, K_used;     // K_used: codes behind it are not looked at, x is 0 there
    const float *xs, *st, *zt;           // tiles: sums of x [groups][Mp], scales and 16 + z [groups][Np]
    int32_t Mp, Np, tiles_n, tiles_m, splits;
    float *slabs;                        // more than one K range: their fp32 sums [splits][M][Np]
};

// Eight weights 16 + c, or with Z 24 + (c - z) / 2, of a word in the order of K: one shift and one and-or for two.  (The constants are kept in registers: as literals, of
// which an instruction takes one, the and and the or are two instructions.)
template <DenseType T, bool Z>
struct Int4Unpack {
    static constexpr bool H = T == DENSE_F16;
    static constexpr uint32_t BASE = H ? 0x4C004C00u : 0x41804180u, HALF = H ? 0x00200020u : 0x00040004u;       // 16, and what 1/2 adds to it
    uint32_t mask = HALF * (Z ? 15 : 30), one = BASE;
    __device__ __forceinline__ Int4Unpack() { asm("" : "+s"(mask), "+v"(one)); }
    // Z: base is that of the row's zero point
    __device__ __forceinline__ u32x4_t operator()(uint32_t w, uint32_t base) const {
        if constexpr (Z && H) return u32x4_t{(w << 5 & mask) + base, (w << 1 & mask) + base, (w >> 3 & mask) + base, (w >> 7 & mask) + base};
        else if constexpr (Z) return u32x4_t{(w << 2 & mask) + base, (w >> 2 & mask) + base, (w >> 6 & mask) + base, (w >> 10 & mask) + base};
        else if constexpr (H) return u32x4_t{(w << 6 & mask) | one, (w << 2 & mask) | one, (w >> 2 & mask) | one, (w >> 6 & mask) | one};
        else return u32x4_t{(w << 3 & mask) | one, (w >> 1 & mask) | one, (w >> 5 & mask) | one, (w >> 9 & mask) | one};
    }
    // 24 - z / 2 (zero points beyond 15 count as 15): what a code adds to, and never beyond 31.5.
    static __device__ __forceinline__ uint32_t base(uint32_t z) { return (16 - min(z, 15u)) * HALF + BASE; }
    // What a weight of 0 is among them: 24, eight times.
    static __device__ __forceinline__ u32x4_t zeros() {
        constexpr uint32_t v = H ? 0x4E004E00u : 0x41C041C0u;
        return u32x4_t{v, v, v, v};
    }
};
// What is taken off of 24 sum x: all of it, and (z - 15) / 2 sums of x for zero points beyond 15.
__device__ __forceinline__ float int4_factor(uint32_t z) { return __builtin_fmaf((float)(max(z, 15u) - 15), -1.0f / 48.0f, -1.0f); }
template <DenseType T, int S>
__device__ __forceinline__ float int4_scale(const void *s, int64_t i) {
    if constexpr (S == 4) return static_cast<const float *>(s)[i];
    else if constexpr (T == DENSE_F16) return (float)static_cast<const _Float16 *>(s)[i];
    else return bf16_to_f32(static_cast<const uint16_t *>(s)[i]);
}

// The values of a row's groups from those that its four lanes hold, one each (two groups: one for two lanes).
template <int GPC, typename V>
__device__ __forceinline__ void int4_share(V v, V (&all)[GPC]) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    if constexpr (GPC == 1) {
        all[0] = v;
    } else {
        const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);            // lanes of q 0, 1 and of q 2, 3, twice each
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t w = h[i];
            if constexpr (GPC == 2) {
                all[i] = __builtin_bit_cast(V, w);
            } else {
                const auto l = __builtin_amdgcn_permlane16_swap(w, w, false, false);
                all[2 * i] = __builtin_bit_cast(V, (uint32_t)l[0]);
                all[2 * i + 1] = __builtin_bit_cast(V, (uint32_t)l[1]);
            }
        }
    }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// 16 F rows of W and 16 MX of x per workgroup, chunks of 128 K dealt to its waves, a lane's 16 bytes of codes straight into registers: their traffic is what
// bounds these calls, from about 20 MB on: one row of 8192 -> 8192 8.7 us (34 MB, 3.9 TB/s; the library's bf16 product 22.1), of 2048 -> 11264 4.8 (12 MB;
// 10.6), the rest of which is the launch and one load behind the other.  The matrix cores take x as rows and W as columns, so that a lane's results belong to one row of W: one scale per
// lane and group.  What is taken off comes from one more product, with 24.
// Groups of 128 with x in LDS: lane (n, q) multiplies the words it loaded, K 32 q + 8 t + {0..7} in product t.  Smaller groups must not meet in a product, and x from memory
// comes in whole pieces of 64 bytes: the four lanes of a row exchange their words first, so that product t is K 32 t + 8 q + {0..7} (48 rows of 5640 -> 2048 9.1 -> 8.5 us).
// XL: x goes through LDS, where the rows of a fragment that are not there cost nothing and all loads are whole rows; otherwise it is read as operands from memory.
template <DenseType T, int G, int S, bool Z, int F, int MX, int NW, bool XL>
__global__ __launch_bounds__(NW * 64) void int4_few_kernel(const Int4Args a) {
    constexpr int GPC = 128 / G, PER = 4 / GPC;                 // groups of a chunk, products of a group
    constexpr bool AS_LOADED = G == 128 && XL;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    f32x4_t *part = reinterpret_cast<f32x4_t *>(smem);          // [wave][tile][lane]
    unsigned char *xs = smem + NW * F * MX * 1024;                   // XL: rows of x, whole chunks
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, r = lane & 15;
    const int n0 = blockIdx.x * (16 * F), m0 = blockIdx.y * (16 * MX), rows = min(a.M - m0, 16 * MX);
    const int chunks = (a.K + 127) >> 7, words = (a.K + 31) >> 5 << 4, pitch = int4_pitch(a.K);       // (words: bytes of a row of codes)
    const auto whole = [](const void *p) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, DENSE_OUTSIDE, 0x00020000); };
    const auto read = [](__amdgpu_buffer_rsrc_t b, uint32_t off) { return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0)); };
    const char *x0 = static_cast<const char *>(a.x) + (int64_t)m0 * a.ldx;
    const __amdgpu_buffer_rsrc_t cb = whole(reinterpret_cast<const char *>(a.c) + (int64_t)n0 * a.ldc), xb = whole(x0);
    uint32_t co[F];
    int64_t n[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        co[f] = n0 + f * 16 + r < a.N ? (uint32_t)((f * 16 + r) * a.ldc) + q * 16 : DENSE_OUTSIDE;
        n[f] = min(n0 + f * 16 + r, a.N - 1);
    }
    uint32_t xo[MX];                                            // (results of rows behind the last one are not used)
#pragma unroll
    for (int j = 0; j < MX; ++j) xo[j] = (uint32_t)min(j * 16 + r, rows - 1) * (XL ? (uint32_t)pitch : (uint32_t)a.ldx);
    const Int4Unpack<T, Z> unpack;
    const u32x4_t zeros = unpack.zeros();
    f32x4_t acc[F][MX];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int j = 0; j < MX; ++j) acc[f][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int c = wave; c < chunks || (XL && c == wave); c += NW) {
        u32x4_t w[F], x[MX][4];
        float s1[F];                                            // of the lane's own group of the chunk: K 32 q on
        uint32_t z1[F];
#pragma unroll
        for (int f = 0; f < F; ++f) w[f] = read(cb, c * 64 + q * 16 < words ? co[f] + c * 64 : DENSE_OUTSIDE);
        const int own = min(c * GPC + q * GPC / 4, a.groups - 1);
#pragma unroll
        for (int f = 0; f < F; ++f) {
            s1[f] = int4_scale<T, S>(a.s, n[f] * a.s_n + own * a.s_g) * (Z ? 2.0f : 1.0f);
            if constexpr (Z) z1[f] = a.z[n[f] * a.z_n + own * a.z_g];
        }
        __builtin_amdgcn_sched_barrier(0);                       // (x behind the codes and scales: 13 rows of 8192 -> 8192 14.6 -> 13.2 us)
        const auto x_at = [&](int p) { return c * 128 + (AS_LOADED ? q * 32 + p * 8 : p * 32 + q * 8); };
        if constexpr (XL) {
            if (c == wave) {                                     // every wave once
                const int units = chunks * 16;
                for (int i = threadIdx.x; i < rows * units; i += NW * 64) {
                    const int m = i / units, u = i - m * units;
                    u32x4_t v = {0, 0, 0, 0};
                    if (u * 8 < a.K) v = *reinterpret_cast<const u32x4_t *>(x0 + m * a.ldx + u * 16);
                    *reinterpret_cast<u32x4_t *>(xs + m * pitch + u * 16) = v;
                }
                __syncthreads();
            }
            if (c >= chunks) break;
#pragma unroll
            for (int p = 0; p < 4; ++p) x[0][p] = *reinterpret_cast<const u32x4_t *>(xs + xo[0] + 2 * x_at(p));
        } else {
#pragma unroll
            for (int j = 0; j < MX; ++j)
#pragma unroll
                for (int p = 0; p < 4; ++p) x[j][p] = read(xb, x_at(p) < a.K ? xo[j] + 2 * x_at(p) : DENSE_OUTSIDE);
        }
        float s[F][GPC];
        uint32_t z[F][GPC];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            int4_share<GPC>(s1[f], s[f]);
            if constexpr (Z) int4_share<GPC>(z1[f], z[f]);
        }
        if constexpr (!AS_LOADED) {                              // word p of lane q <-> word q of lane p
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const u32x4_t v = w[f];
                const auto l0 = __builtin_amdgcn_permlane16_swap(v[0], v[1], false, false), l1 = __builtin_amdgcn_permlane16_swap(v[2], v[3], false, false);
                const auto h0 = __builtin_amdgcn_permlane32_swap(l0[0], l1[0], false, false), h1 = __builtin_amdgcn_permlane32_swap(l0[1], l1[1], false, false);
                w[f] = u32x4_t{h0[0], h1[0], h0[1], h1[1]};
            }
        }
#pragma unroll
        for (int i = 0; i < GPC; ++i) {
            if (c * GPC + i >= a.groups) break;
            f32x4_t d[F][MX], e[MX];
            uint32_t base[F];
#pragma unroll
            for (int f = 0; f < F; ++f) base[f] = Z ? unpack.base(z[f][i]) : 0u;
#pragma unroll
            for (int j = 0; j < MX; ++j) {
                e[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < F; ++f) d[f][j] = e[j];
            }
#pragma unroll
            for (int p = i * PER; p < (i + 1) * PER; ++p) {
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    const uint32_t word = w[f][p];
                    const u32x4_t u = unpack(word, base[f]);
#pragma unroll
                    for (int j = 0; j < MX; ++j) d[f][j] = dense_mfma<T>(x[j][p], u, d[f][j]);
                }
#pragma unroll
                for (int j = 0; j < MX; ++j) e[j] = dense_mfma<T>(x[j][p], zeros, e[j]);
            }
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const float factor = Z ? int4_factor(z[f][i]) : -1.0f;
#pragma unroll
                for (int j = 0; j < MX; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[f][j][v] = __builtin_fmaf(s[f][i], __builtin_fmaf(factor, e[j][v], d[f][j][v]), acc[f][j][v]);
            }
        }
    }
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int j = 0; j < MX; ++j) part[(wave * F * MX + f * MX + j) * 64 + lane] = acc[f][j];
    __syncthreads();
    if (wave >= F * MX) return;
    f32x4_t sum = part[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum += part[(w * F * MX + wave) * 64 + lane];
    const int at = n0 + wave / MX * 16 + r, row = wave % MX * 16 + 4 * q;
    if (at >= a.N) return;
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (row + v < rows) a.y[(int64_t)(m0 + row + v) * a.ldy + at] = (uint16_t)dense_pack2<T>(sum[v], 0.f);
}

// ---- many rows -------------------------------------------------------------------------------------------------------
// Which codes of a word count whose first value has `left` to the last one.
__device__ __forceinline__ uint32_t int4_counted(int left) {
    const int v = min(max(left, 0), 8);
    return ((1u << 4 * ((v + 1) >> 1)) - 1) | ((1u << 4 * (v >> 1)) - 1) << 16;
}
// Whether all codes of group g of row n are z.
__device__ __forceinline__ bool int4_all_zero(const Int4Args &a, int64_t n, int g, int group, uint32_t z) {
    const u32x4_t *c = reinterpret_cast<const u32x4_t *>(reinterpret_cast<const char *>(a.c) + n * a.ldc + (int64_t)g * (group / 2));
    const int units = min(group, a.K - g * group + 31) / 32;      // 16 bytes of codes
    u32x4_t w[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) w[p] = c[min(p, units - 1)];
    uint32_t other = z > 15;
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p < units) other |= (w[p][j] ^ z * 0x11111111u) & int4_counted(a.K_used - (g * group + p * 32 + j * 8));
    return !other;
}

constexpr int INT4_ROWS = 16;                                    // of W that a wave looks through (4: 8192 -> 8192 in groups of 32 85 -> 101 us)
// What a tile needs of the groups, laid out so that its pieces are whole 16-byte units: sums of x times -1 or, without zero points, -24 [groups][Mp], scales and 16 + z [groups][Np], zeros beyond M,
// N and the last group.  The scale is times 0 where all codes are the zero point.  A wave takes 16 rows of W and 64 units of 32 K, one per lane, of whose codes it reads whole
// rows, all 16 at once; only where a group's codes are all the same they are compared with its zero point.
template <DenseType T, int S, int G, bool Z>
__global__ __launch_bounds__(256) void int4_prepare_kernel(const Int4Args a, int groups, float *xs, float *st, float *zt, unsigned n_blocks) {
    constexpr int group = G;
    if (blockIdx.x >= n_blocks) {                                // sums of x, behind the codes, which take longer: 8 values per thread, the lanes of a group side by side
        const int per = group / 8;
        const int64_t i = ((int64_t)(blockIdx.x - n_blocks) * 256 + threadIdx.x) / per, m = i / groups;
        const int g = (int)(i - m * groups), lane = threadIdx.x & (per - 1), k = g * group + lane * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (m < a.M && k < a.K) dense_unpack8<T>(*reinterpret_cast<const u32x4_t *>(static_cast<const char *>(a.x) + m * a.ldx + (int64_t)k * 2), v);
        float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        const auto add = [&](uint32_t other) { sum += __builtin_bit_cast(float, other); };
        if (per > 8) add(mortar_row_xor<8>(__builtin_bit_cast(uint32_t, sum)));
        if (per > 4) add(mortar_row_xor<4>(__builtin_bit_cast(uint32_t, sum)));
        add(mortar_row_xor<2>(__builtin_bit_cast(uint32_t, sum)));
        add(mortar_row_xor<1>(__builtin_bit_cast(uint32_t, sum)));
        if (lane == 0 && m < a.Mp) xs[(int64_t)g * a.Mp + m] = Z ? -sum : -24.0f * sum;
        return;
    }
    constexpr int PER = G / 32, GROUPS = 64 / PER, ROWS = INT4_ROWS, SIDE = 64 / ROWS, TURNS = GROUPS / SIDE;   // units of a group, groups of the wave, SIDE at a time
    const int lane = threadIdx.x & 63, chunks = (groups + GROUPS - 1) / GROUPS, units = (a.K + 31) >> 5;
    const int64_t task = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), block = task / chunks, n = block * ROWS + lane % ROWS;
    if (block * ROWS >= a.Np) return;
    const int g0 = (int)(task - block * chunks) * GROUPS, u = g0 * PER + lane, left = a.K_used - u * 32;
    const char *c = reinterpret_cast<const char *>(a.c) + (int64_t)min(u, units - 1) * 16;
    u32x4_t w[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) w[i] = *reinterpret_cast<const u32x4_t *>(c + min(block * ROWS + i, (int64_t)a.N - 1) * a.ldc);
    const int64_t row = min(n, (int64_t)a.N - 1);
    float s[TURNS];
    uint32_t z[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const int64_t g = min(g0 + i * SIDE + lane / ROWS, a.groups - 1);
        s[i] = int4_scale<T, S>(a.s, row * a.s_n + g * a.s_g);
        if constexpr (Z) z[i] = a.z[row * a.z_n + g * a.z_g];
    }
    uint32_t same = 0;                                           // bit i: the lane's group has one code throughout in row i
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const uint32_t first = (w[i][0] & 15) * 0x11111111u;
        uint32_t other = 0;
        if (left >= 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) other |= w[i][j] ^ first;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) other |= (w[i][j] ^ first) & int4_counted(left - j * 8);
        }
        same |= (other == 0 ? 1u : 0u) << i;
    }
#pragma unroll
    for (int d = 1; d < PER; d <<= 1) same &= __shfl_xor(same, d);
    uint32_t zeros = 0;                                          // bit i: of turn i
#pragma unroll
    for (int i = 0; i < TURNS; ++i) zeros |= (__shfl(same, (i * SIDE + lane / ROWS) * PER) >> lane % ROWS & 1) << i;
    if (zeros)
        for (int i = 0; i < TURNS; ++i) {
            const int g = min(g0 + i * SIDE + lane / ROWS, a.groups - 1);
            if ((zeros >> i & 1) && !int4_all_zero(a, row, g, G, Z ? a.z[row * a.z_n + g * a.z_g] : 8)) zeros &= ~(1u << i);
        }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const int g = g0 + i * SIDE + lane / ROWS;
        const bool on = g < a.groups && n < a.N;
        if (g >= groups) continue;
        st[(int64_t)g * a.Np + n] = on ? (zeros >> i & 1 ? s[i] * 0.f : s[i]) : 0.f;          // (NaN stays)
        if constexpr (Z) zt[(int64_t)g * a.Np + n] = on ? 16.0f + (float)z[i] : 0.f;
    }
}

// BN features x BM tokens by WN x WM waves, SPS steps of 64 K per turn through a ring of NS turns in LDS filled by asynchronous copies: x in rows of 128 bytes
// with their units permuted, codes in rows of 32 bytes, and each step's groups: scales, sums of x, 16 + z.  One barrier per turn.  A wave makes its
// weights from the codes in registers.  The first product of a group starts at -(16 + z) sum x instead of 0.
// What bounds it is the instructions that a wave issues beside the products: 128 x 128 with 32 x 128 per wave has 3 per product (4096 rows of 2048 -> 11264
// in 176 to 195 us with the launch in front; where it took 189, 64 x 64 per wave took 194, eight waves of 32 x 64 201; the library's bf16 product 149 to 160;
// groups of 64 212 to 218, of 32 248 to 263, with zero points 192, 230 and 292 at least), and the power that the chip may draw: the same on zeros takes 164 of 189.  A third turn in the ring costs more than it hides (197), and so do 32 x 32 products (204), operands read a half step ahead of them (196) and
// copies issued behind the reads.
// The ranges of a product over several of them leave fp32 sums.
template <DenseType T, int G, bool Z, int BN, int BM, int WN, int WM, int NS, int SPS>
__global__ __launch_bounds__(WN *WM * 64, 2) void int4_tile_kernel(const Int4Args a) {
    constexpr int NW = WN * WM, FN = BN / WN / 16, FM = BM / WM / 16, GPS = G == 32 ? 2 : 1;
    constexpr int X = BM * 128, C = BN * 32, GB = (BN + BM + (Z ? BN : 0)) * 4, GC = (GB + 1023) / 1024, SLOT = X + C + GPS * GC * 1024;
    constexpr int LX = X / 1024 / NW, CC = C / 1024, EXTRA = CC + GPS * GC, LE = (EXTRA + NW - 1) / NW, LEAST = (LX + EXTRA / NW) * SPS;
    static_assert(X % (1024 * NW) == 0 && C % 1024 == 0, "whole copies");
    static_assert(FN % 2 == 0, "fragments are joined in pairs");
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, r = lane & 15;
    const int wn = wave % WN, wm = wave / WN;
    const uint32_t l0 = mortar_lds_addr(lds);
    // As in the 16-bit products: workgroups of one XCD take a contiguous run of tiles, in bands of 8 along m.
    const int tiles = a.tiles_n * a.tiles_m, total = tiles * a.splits, per_xcd = (total + 7) >> 3, place = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (place >= min(total, (int)((blockIdx.x & 7) + 1) * per_xcd)) return;
    const int split = place / tiles, id = place - split * tiles;
    const int band = id / (8 * a.tiles_n), rest = id - band * 8 * a.tiles_n, bh = min(8, a.tiles_m - band * 8), tn = rest / bh;
    const int n0 = __builtin_amdgcn_readfirstlane(tn * BN), m0 = __builtin_amdgcn_readfirstlane((band * 8 + rest - tn * bh) * BM);
    const int steps = (a.K + 63) >> 6, row_bytes = (a.K + 31) >> 5 << 4;
    constexpr int WHOLE = G == 128 || SPS == 2 ? 2 : 1;          // a range begins with a group and whole turns
    const int units = (steps + WHOLE - 1) / WHOLE, begin_step = WHOLE * __builtin_amdgcn_readfirstlane(units * split / a.splits),
              end_step = min(steps, WHOLE * __builtin_amdgcn_readfirstlane(units * (split + 1) / a.splits));

    // Sources of this lane's copies: offsets that move on with the steps, and where K ends for them.
    const u32x4_t xbuf = dense_buffer(static_cast<const char *>(a.x) + (int64_t)m0 * a.ldx), cbuf = dense_buffer(reinterpret_cast<const char *>(a.c) + (int64_t)n0 * a.ldc);
    uint32_t xoff[LX], coff[LE];
    int kx;
    const int kc = (lane & 1) ^ ((lane >> 4) & 1);               // unit of a row of codes (rows 8 apart, which share banks, have theirs in opposite order)
    {
        const int u = lane & 7;
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int row = (i * NW + wave) * 8 + (lane >> 3);
            xoff[i] = m0 + row < a.M ? (uint32_t)(row * a.ldx) + (u ^ (row & 7)) * 16 : DENSE_OUTSIDE;
        }
        kx = (u ^ ((lane >> 3) & 7)) * 16;                       // (the same in all copies: their rows are 8 apart)
#pragma unroll
        for (int i = 0; i < LE; ++i) {
            const int e = i * NW + wave;                         // copies of codes, then those of the groups
            const int row = e * 32 + (lane >> 1);
            coff[i] = e < CC && n0 + row < a.N ? (uint32_t)(row * a.ldc) + kc * 16 : DENSE_OUTSIDE;
        }
    }
    const char *gsrc[LE];                                        // the lane's part of a group's piece (scales, sums, zero points): of group 0, and the
    uint32_t gpitch[LE];                                         // bytes to the next
#pragma unroll
    for (int i = 0; i < LE; ++i) {
        const int gc = i * NW + wave - CC, at = (gc < 0 ? 0 : gc % GC) * 256 + lane * 4;
        const bool sums = at >= BN && (at < BN + BM || !Z);
        gsrc[i] = reinterpret_cast<const char *>(at < BN ? a.st + n0 + at : sums ? a.xs + m0 + min(at - BN, BM - 4) : a.zt + n0 + min(at - BN - BM, BN - 4));
        gpitch[i] = (uint32_t)(sums ? a.Mp : a.Np) * 4u;
    }
    const auto copy_to = [&](auto whole, int k, uint32_t slot) __attribute__((always_inline)) {  // k: the step; beyond the last one it copies zeros; whole: all of it is inside K
        constexpr bool inside = whole.value;
        const uint32_t base = l0 + slot;
#pragma unroll
        for (int i = 0; i < LX; ++i) dense_copy(xbuf, inside || kx + k * 128 < a.K * 2 ? xoff[i] + k * 128 : DENSE_OUTSIDE, base + (i * NW + wave) * 1024);
#pragma unroll
        for (int i = 0; i < LE; ++i) {
            const int e = i * NW + wave;
            if ((i + 1) * NW <= CC || e < CC) {                  // (the first half known to the compiler)
                dense_copy(cbuf, inside || kc * 16 + k * 32 < row_bytes ? coff[i] + k * 32 : DENSE_OUTSIDE, base + X + e * 1024);
            } else if (e < EXTRA) {
                const int gc = e - CC;
                const uint32_t g = k < steps ? (G == 128 ? k >> 1 : G == 64 ? k : 2 * k + gc / GC) : 0;
                const char *src = gsrc[i] + (uint64_t)g * gpitch[i];
                mortar_load_to_lds(reinterpret_cast<const MORTAR_GLOBAL char *>(reinterpret_cast<uintptr_t>(src)), base + X + C + gc * 1024);
            }
        }
    };
    const auto copy_step = [&](int k, uint32_t slot) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SPS; ++u) {
            if ((k + SPS) * 64 <= a.K) copy_to(Const<1>{}, k + u, slot + u * SLOT);
            else copy_to(Const<0>{}, k + u, slot + u * SLOT);
        }
    };
    const uint32_t ax = l0 + dense_row_addr(wm * FM * 16, lane), ac = l0 + X + (wn * FN * 16 + r) * 32 + (r >> 3) * 16 + q * 4, ag = l0 + X + C;

    const Int4Unpack<T, false> unpack;
    f32x4_t acc[FN][FM], part[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = part[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) copy_step(begin_step + i * SPS, i * SPS * SLOT);
    uint32_t slot = 0, free_slot = (NS - 1) * SPS * SLOT;
    // first / last: the step, in slot `at`, begins / ends a group (groups of 128: two steps)
    const auto multiply = [&](uint32_t at, auto first, auto last) __attribute__((always_inline)) {
        const uint32_t ga = ag + at;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t gt = ga + (GPS == 2 ? t * GC * 1024 : 0);
            u32x4_t xf[FM], wf[FN];
#pragma unroll
            for (int i = 0; i < FN; ++i) wf[i] = unpack(*(const MORTAR_LDS uint32_t *)(uintptr_t)(((ac + at) ^ (t * 16)) + i * 512), 0);
#pragma unroll
            for (int j = 0; j < FM; ++j) xf[j] = dense_read(((ax + at) ^ (t * 64)) + j * 2048);
            const bool begin = GPS == 2 || (first.value && t == 0), end = GPS == 2 || (last.value && t == 1);
            if (begin) {
                float sx[FM];
#pragma unroll
                for (int j = 0; j < FM; ++j) sx[j] = *(const MORTAR_LDS float *)(uintptr_t)(gt + (BN + (wm * FM + j) * 16 + r) * 4);
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    f32x4_t zv = {1.f, 1.f, 1.f, 1.f};
                    if constexpr (Z) zv = *(const MORTAR_LDS f32x4_t *)(uintptr_t)(gt + (BN + BM + (wn * FN + i) * 16 + 4 * q) * 4);
#pragma unroll
                    for (int j = 0; j < FM; ++j) {
                        f32x4_t c;
#pragma unroll
                        for (int v = 0; v < 4; ++v) c[v] = Z ? zv[v] * sx[j] : sx[j];
                        part[i][j] = dense_mfma<T>(wf[i], xf[j], c);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int j = 0; j < FM; ++j) part[i][j] = dense_mfma<T>(wf[i], xf[j], part[i][j]);
            }
            if (end) {
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    const f32x4_t sv = *(const MORTAR_LDS f32x4_t *)(uintptr_t)(gt + ((wn * FN + i) * 16 + 4 * q) * 4);
#pragma unroll
                    for (int j = 0; j < FM; ++j)
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[i][j][v] = __builtin_fmaf(sv[v], part[i][j][v], acc[i][j][v]);
                }
            }
        }
    };
    // A turn: all waves meet, SPS steps are multiplied and as many copied to where the last turn's were.
    const auto meet = [&](int k) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * LEAST) : "memory");
        copy_step(k + (NS - 1) * SPS, free_slot);
    };
    const auto turned = [&] {
        free_slot = slot;
        slot = slot + SPS * SLOT == NS * SPS * SLOT ? 0u : slot + SPS * SLOT;
    };
    if constexpr (G == 128 || SPS == 2) {
        constexpr int C1 = G == 128 ? 0 : 1;
        int k = begin_step;
        for (; k + 1 < end_step; k += 2) {
            meet(k);
            multiply(slot, Const<1>{}, Const<C1>{});
            if constexpr (SPS == 1) turned(), meet(k + 1);
            multiply(slot + (SPS - 1) * SLOT, Const<C1>{}, Const<1>{});
            turned();
        }
        if (k < end_step) {
            meet(k);
            multiply(slot, Const<1>{}, Const<1>{});
        }
    } else {
        for (int k = begin_step; k < end_step; ++k) {
            meet(k);
            multiply(slot, Const<1>{}, Const<1>{});
            turned();
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (the copies of the steps behind the last)

    const bool vector = a.ldy % 8 == 0 && a.N % 8 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + (wm * FM + j) * 16 + r;
        if (m >= a.M) continue;
#pragma unroll
        for (int i = 0; i < FN; i += 2) {
            float d[8];
            dense_join8(acc[i][j], acc[i + 1][j], d);
            const int n = n0 + (wn * FN + i) * 16 + dense_lane_n(lane);
            if (n >= a.N) continue;
            if (a.splits > 1) {
                float *p = a.slabs + ((int64_t)split * a.M + m) * a.Np + n;
                *reinterpret_cast<f32x4_t *>(p) = f32x4_t{d[0], d[1], d[2], d[3]};
                *reinterpret_cast<f32x4_t *>(p + 4) = f32x4_t{d[4], d[5], d[6], d[7]};
                continue;
            }
            uint16_t *o = a.y + m * a.ldy + n;
            if (vector) {
                *reinterpret_cast<u32x4_t *>(o) = dense_pack8<T>(d);
            } else {
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    if (n + v < a.N) o[v] = (uint16_t)dense_pack2<T>(d[v], 0.f);
            }
        }
    }
}

// The slabs of the K ranges added in their order: 2.5 us and their reading, which plan() weighs against rounds of idle CUs (1738 rows of 5728 -> 869: 75 us in
// one range, 51 in several).
template <DenseType T>
__global__ __launch_bounds__(256) void int4_join_kernel(const Int4Args a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (a.N + 3) >> 2;
    if (i >= a.M * per) return;
    const int64_t m = i / per, n = (i - m * per) * 4, slab = (int64_t)a.M * a.Np;
    const float *p = a.slabs + m * a.Np + n;
    f32x4_t v[8], sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const f32x4_t *>(p + (k < a.splits ? k : 0) * slab);
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < a.splits) sum += v[k];
    uint16_t *o = a.y + m * a.ldy + n;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (n + k < a.N) o[k] = (uint16_t)dense_pack2<T>(sum[k], 0.f);
}

// Rows of x with any strides, on any address and of any length as rows of whole 16-byte units, zeros behind K: bound by the memory, a launch in front of the
// product (680 rows of 410 -> 749 9.0 us with both, with torch's padding 16).
__global__ __launch_bounds__(256) void int4_rows_kernel(const uint16_t *x, int64_t M, int32_t K, int64_t s_m, int64_t s_k, uint16_t *o) {
    const int units = (K + 7) >> 3;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / units;
    if (m >= M) return;
    const int k = (int)(i - m * units) * 8;
    const uint16_t *p = x + m * s_m + k * s_k;
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? p[j * s_k] : 0u;
    *reinterpret_cast<u32x4_t *>(o + i * 8) = u32x4_t{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
}

// ---- quantising ------------------------------------------------------------------------------------------------------
template <int TYPE>
__device__ __forceinline__ float int4_read(const void *p, int64_t i) {
    if constexpr (TYPE == MORTAR_FP32) return static_cast<const float *>(p)[i];
    else if constexpr (TYPE == MORTAR_FP16) return (float)static_cast<const _Float16 *>(p)[i];
    else return bf16_to_f32(static_cast<const uint16_t *>(p)[i]);
}
// 8 values per thread, the lanes of a group side by side (16 of them at most: within a row of lanes).  One pass, once per weight, bound by
// its loads of one value each: 23 million bf16 weights 39 us (1.5 TB/s), with zero points 41, in fp32 43.
template <int TYPE, int STYPE>
__global__ __launch_bounds__(256) void int4_quantize_kernel(const void *w, int32_t N, int32_t K, int64_t ldw, int group, uint32_t *c, int64_t ldc, void *s, int64_t s_n,
                                                            int64_t s_g, uint8_t *z, int64_t z_n, int64_t z_g) {
    const int per = group / 8, groups = (K + group - 1) / group, words = (K + 31) / 32 * 4;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / per, n = i / groups;
    if (n >= N) return;                                          // (whole groups of lanes)
    const int g = (int)(i - n * groups), lane = threadIdx.x & (per - 1), k = g * group + lane * 8;
    float v[8], lo = 0.f, hi = 0.f;
    uint32_t bad = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = k + j < K ? int4_read<TYPE>(w, n * ldw + k + j) : 0.f;
        lo = fminf(lo, v[j]);
        hi = fmaxf(hi, v[j]);
        bad |= !(__builtin_fabsf(v[j]) < __builtin_inff());
    }
    const auto join = [&](auto x) {
        constexpr int X = decltype(x)::value;
        lo = fminf(lo, __builtin_bit_cast(float, mortar_row_xor<X>(__builtin_bit_cast(uint32_t, lo))));
        hi = fmaxf(hi, __builtin_bit_cast(float, mortar_row_xor<X>(__builtin_bit_cast(uint32_t, hi))));
        bad |= mortar_row_xor<X>(bad);            // (with every lane: no shortcut)
    };
    if (per > 8) join(Const<8>{});
    if (per > 4) join(Const<4>{});
    join(Const<2>{});
    join(Const<1>{});
    float sc = z ? (hi - lo) / 15.0f : fmaxf(hi / 7.0f, lo / -8.0f);
    if (bad) sc = __builtin_nanf("");
    if constexpr (STYPE == MORTAR_FP16) sc = (float)(_Float16)sc;
    else if constexpr (STYPE == MORTAR_BF16) sc = bf16r(sc);
    if (sc == 0.f) sc = 1.0f;
    const float zero = z ? fminf(fmaxf(rintf(-lo / sc), 0.f), 15.f) : 8.0f;
    uint32_t word = 0;
    constexpr int place[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float code = k + j < K ? fminf(fmaxf(rintf(v[j] / sc) + zero, 0.f), 15.f) : 8.0f;
        word |= (uint32_t)code << 4 * place[j];
    }
    if (k / 8 < words) c[n * ldc + k / 8] = word;
    if (lane) return;
    if constexpr (STYPE == MORTAR_FP32) static_cast<float *>(s)[n * s_n + g * s_g] = sc;
    else if constexpr (STYPE == MORTAR_FP16) static_cast<_Float16 *>(s)[n * s_n + g * s_g] = (_Float16)sc;
    else static_cast<uint16_t *>(s)[n * s_n + g * s_g] = (uint16_t)bf16_bits_rne(sc);
    if (z) z[n * z_n + g * z_g] = (uint8_t)zero;
}

// ---- host side -------------------------------------------------------------------------------------------------------

int launch_error(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int64_t up128(int64_t v) { return (v + 127) / 128 * 128; }

// Which kernel: the smallest estimate, in us, from products of 9 to 4096 rows with 16 weights of 300 to 16384 rows and 512 to 8192 columns in every form (of 1334 random
// products of 1 to 4096 rows what is chosen takes 2.6 % longer than the best form, of which timing itself makes about 1).
// Few rows: workgroups of 16 x 16 F results, one round of the chip if F = 4 still gives one, with the smallest such F (16 rows of 2048 -> 11264 7.8 with F = 4 and 9.1 in
// two rounds with 2; 64 of 5632 -> 2048 11.0 with 2, 13.3 with 4 on half of the CUs; 77 of them 13.5 with 4, 17.4 in two rounds with 2), and 16 waves instead of 8 if there
// is work for them.  Where that takes several rounds, 32 rows of x share what is unpacked of W (32 rows of 2048 -> 11264 11.1 -> 9.5, 17 of 5120 -> 12288 20.3 -> 16.1,
// 256 of 5632 -> 2048 24.3 -> 18.9).  Tiles are bound by the instructions of a step, which one workgroup of a CU alone cannot issue behind each other's latencies, and need a second
// launch for the sums of x; 32 x 128 per wave pays for the sums of smaller groups, the small tile less so.
struct Int4Plan {
    int f, waves, tile, splits;  // few rows: f > 0; else index into INT4_TILES and ranges of K
    bool xl;
    int mx = 1;                  // few rows: 16 of x each
};
struct Int4Tile {
    int bn, bm;
    double alone[3], more[3];    // us of a step of 64 K with groups of 128, 64, 32: of the only workgroup of a CU, and of each of many
};
constexpr Int4Tile INT4_TILES[] = {{128, 128, {0.60, 0.78, 1.09}, {0.53, 0.58, 0.80}}, {64, 64, {0.335, 0.335, 0.43}, {0.19, 0.215, 0.285}}};
constexpr int MOST_FEW_ROWS = 4096, MOST_LDS = 160 * 1024;

// ldx: bytes between rows of x.
Int4Plan plan(int64_t M, int64_t N, int64_t K, int group, int64_t ldx) {
    const int64_t chunks = (K + 127) / 128, steps = (K + 63) / 64, n16 = (N + 15) / 16, m16 = (M + 15) / 16;
    Int4Plan p{1, 8, 0, 1, false};
    if (M <= 16) {
        // x through LDS: rows a multiple of 1 KB apart meet in the same channels when a fragment loads 16 of them at once (8 rows of 5632 -> 2048 7.2 -> 6.1 us, 8 of 5640
        // in rows of 8192 6.6 -> 6.2, 5 of 11264 -> 2048 10.1 -> 8.5, long rows at the price of one workgroup per CU).  Others are better read as operands from 3 rows on
        // (13 of 5632 in rows of 5640 7.1 -> 6.6), with groups of 128, whose words need no exchange there, from 6 on (5 of 5640 -> 2048 5.7, as operands 6.0), and of
        // 9 rows and more all where 8 waves do (13 of 2048 -> 2048 4.8 -> 4.7, but 13 of 2560 5.3 as operands, 4.9 through LDS).
        const bool apart = ldx % 1024 == 0;
        const int64_t bytes = M * int4_pitch((int)K);
        p.f = n16 >= 512 && chunks >= 32 ? 2 : 1;
        p.waves = chunks > 16 ? 16 : 8;
        p.xl = M <= 8 && (M <= (group == 128 ? 5 : 2) || apart) && bytes <= 64 * 1024;
        if (apart && chunks > 16 && (n16 + p.f - 1) / p.f <= 256) p.xl |= bytes <= MOST_LDS - p.waves * p.f * 1024;
        if (p.xl) return p;
    }
    p.f = 4;
    for (const int f : {2, 1})
        if ((n16 + f - 1) / f * m16 <= 256) p.f = f;
    const int64_t wgs = (n16 + p.f - 1) / p.f * m16;
    p.waves = wgs <= 256 && chunks > 8 ? 16 : 8;
    if (M <= 16) return p;
    const double chunk = p.f == 1 ? 0.12 : p.f == 2 ? 0.155 : 0.206;
    const auto few = [&](int64_t workgroups, double us) { return 3.3 + (double)((workgroups + 255) / 256) * (0.5 + us * (double)chunks); };
    double best = M <= MOST_FEW_ROWS ? few(wgs, chunk) : 1e300;
    const int64_t wgs32 = (n16 + 3) / 4 * ((m16 + 1) / 2);
    if (const double us = few(wgs32, wgs32 <= 256 ? 0.33 : 0.40); M <= MOST_FEW_ROWS && us < best) best = us, p = Int4Plan{4, 8, 0, 1, false, 2};
    const int64_t whole = 2, units = (steps + whole - 1) / whole;
    const int g = group == 128 ? 0 : group == 64 ? 1 : 2;
    for (int t = 0; t < 2; ++t) {
        const Int4Tile &d = INT4_TILES[t];
        const int64_t tiles = ((N + d.bn - 1) / d.bn) * ((M + d.bm - 1) / d.bm);
        for (const int splits : {1, 2, 3, 4, 6, 8}) {
            if (splits > 1 && (units * whole < 4 * splits || tiles * splits > 1024)) break;
            const int64_t per_cu = (tiles * splits + 255) / 256, each = (units + splits - 1) / splits * whole;
            double us = 7.0 + 7.8e-8 * (double)N * (double)K + (double)each * std::max(d.alone[g], d.more[g] * (double)per_cu);
            if (splits > 1) us += 3.0 + 1.2e-6 * (double)splits * (double)M * (double)up128(N);
            if (us < best) best = us, p = Int4Plan{0, 0, t, splits, false};
        }
    }
    return p;
}
int64_t groups_padded(int64_t K, int group) { return group == 32 ? (K + 63) / 64 * 2 : (K + group - 1) / group; }

template <DenseType T, int G, int S, bool Z, int F, int MX, int NW, bool XL>
int launch_few_form(const Int4Args &a, hipStream_t st, const char *what) {
    const auto kern = int4_few_kernel<T, G, S, Z, F, MX, NW, XL>;
    constexpr int sums = NW * F * MX * 1024;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, XL ? MOST_LDS : sums);
    if (e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    const dim3 grid((unsigned)((a.N + 16 * F - 1) / (16 * F)), (unsigned)((a.M + 16 * MX - 1) / (16 * MX)));
    hipLaunchKernelGGL(kern, grid, dim3(NW * 64), sums + (XL ? a.M * int4_pitch(a.K) : 0), st, a);
    return launch_error(what);
}
template <DenseType T, int G, int S, bool Z>
int launch_few(const Int4Args &a, const Int4Plan &p, hipStream_t st, const char *what) {
    if (p.xl) {
        if (p.f == 2) return launch_few_form<T, G, S, Z, 2, 1, 16, true>(a, st, what);
        return p.waves == 16 ? launch_few_form<T, G, S, Z, 1, 1, 16, true>(a, st, what) : launch_few_form<T, G, S, Z, 1, 1, 8, true>(a, st, what);
    }
    if (p.mx == 2) return launch_few_form<T, G, S, Z, 4, 2, 8, false>(a, st, what);
    if (p.waves == 16)
        return p.f == 4 ? launch_few_form<T, G, S, Z, 4, 1, 16, false>(a, st, what) : p.f == 2 ? launch_few_form<T, G, S, Z, 2, 1, 16, false>(a, st, what) : launch_few_form<T, G, S, Z, 1, 1, 16, false>(a, st, what);
    return p.f == 4 ? launch_few_form<T, G, S, Z, 4, 1, 8, false>(a, st, what) : p.f == 2 ? launch_few_form<T, G, S, Z, 2, 1, 8, false>(a, st, what) : launch_few_form<T, G, S, Z, 1, 1, 8, false>(a, st, what);
}

template <DenseType T, int G, bool Z, int BN, int BM, int WN, int WM, int NS, int SPS>
int launch_tile_form(Int4Args a, hipStream_t st, const char *what) {
    const auto kern = int4_tile_kernel<T, G, Z, BN, BM, WN, WM, NS, SPS>;
    constexpr int smem = NS * SPS * (BM * 128 + BN * 32 + (G == 32 ? 2 : 1) * (((BN + BM + (Z ? BN : 0)) * 4 + 1023) / 1024) * 1024);
    static_assert(smem * 2 <= 160 * 1024, "two workgroups per CU");
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    const int64_t tn = ((int64_t)a.N + BN - 1) / BN, tm = ((int64_t)a.M + BM - 1) / BM;
    if (tn * tm * a.splits > 1 << 22) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many tiles", what);
    a.tiles_n = (int)tn;
    a.tiles_m = (int)tm;
    hipLaunchKernelGGL(kern, dim3((unsigned)(8 * ((tn * tm * a.splits + 7) / 8))), dim3(WN * WM * 64), smem, st, a);
    return launch_error(what);
}

template <DenseType T, int G, int S, bool Z>
int launch_many(Int4Args a, const Int4Plan &p, float *ws, hipStream_t st, const char *what) {
    const int64_t groups = groups_padded(a.K, G);
    a.Mp = (int32_t)up128(a.M);
    a.Np = (int32_t)up128(a.N);
    float *xs = ws, *s = xs + groups * a.Mp, *zt = Z ? s + groups * a.Np : nullptr;
    a.xs = xs; a.st = s; a.zt = zt;
    a.splits = p.splits;
    a.slabs = s + 2 * groups * a.Np;
    const int64_t x_blocks = (groups * a.Mp * (G / 8) + 255) / 256, n_blocks = (a.Np / INT4_ROWS * ((groups * (G / 32) + 63) / 64) + 3) / 4;     // (a wave each: rows, 64 units)
    if (x_blocks + n_blocks >= 1 << 24) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many values", what);
    hipLaunchKernelGGL((int4_prepare_kernel<T, S, G, Z>), dim3((unsigned)(x_blocks + n_blocks)), dim3(256), 0, st, a, (int)groups, xs, s, zt, (unsigned)n_blocks);
    if (const int rc = launch_error(what)) return rc;
    const int rc = p.tile == 0 ? launch_tile_form<T, G, Z, 128, 128, 4, 1, 2, 1>(a, st, what) : launch_tile_form<T, G, Z, 64, 64, 2, 2, 2, 2>(a, st, what);
    if (rc || p.splits == 1) return rc;
    hipLaunchKernelGGL(int4_join_kernel<T>, dim3((unsigned)(((int64_t)a.M * ((a.N + 3) / 4) + 255) / 256)), dim3(256), 0, st, a);
    return launch_error(what);
}

template <DenseType T, int G, int S>
int launch_zeros(const Int4Args &a, float *ws, hipStream_t st, const char *what) {
    const Int4Plan p = plan(a.M, a.N, a.K, G, a.ldx);
    if (p.f) return a.z ? launch_few<T, G, S, true>(a, p, st, what) : launch_few<T, G, S, false>(a, p, st, what);
    return a.z ? launch_many<T, G, S, true>(a, p, ws, st, what) : launch_many<T, G, S, false>(a, p, ws, st, what);
}
template <DenseType T, int G>
int launch_scales(const Int4Args &a, bool s32, float *ws, hipStream_t st, const char *what) {
    return s32 ? launch_zeros<T, G, 4>(a, ws, st, what) : launch_zeros<T, G, 2>(a, ws, st, what);
}
template <DenseType T>
int launch_group(const Int4Args &a, int group, bool s32, float *ws, hipStream_t st, const char *what) {
    return group == 32 ? launch_scales<T, 32>(a, s32, ws, st, what) : group == 64 ? launch_scales<T, 64>(a, s32, ws, st, what) : launch_scales<T, 128>(a, s32, ws, st, what);
}

int check_group(const char *what, int group) {
    return group == 32 || group == 64 || group == 128 ? MORTAR_OK : mortar_fail(MORTAR_ERR_ARG, "%s: groups of 32, 64 or 128 values", what);
}
bool known(int32_t type) { return type == MORTAR_BF16 || type == MORTAR_FP16 || type == MORTAR_FP32; }
int check_codes(const char *what, const void *c, int64_t K, int64_t ldc) {
    if (!c) return mortar_fail(MORTAR_ERR_ARG, "%s: the codes are null", what);
    if (ldc % 4 || ldc < (K + 31) / 32 * 4 || (reinterpret_cast<uintptr_t>(c) & 15)) return mortar_fail(MORTAR_ERR_ARG, "%s: the codes need whole rows of 32 values on 16-byte addresses", what);
    if (128 * ldc * 4 >= (int64_t)DENSE_OUTSIDE) return mortar_fail(MORTAR_ERR_LIMIT, "%s: the rows of codes are too far apart", what);
    return MORTAR_OK;
}
#define CHECK(...) do { const int rc_ = (__VA_ARGS__); if (rc_) return rc_; } while (0)

}  // namespace

extern "C" int mortar_int4_quantize(const void *w, int32_t N, int32_t K, int64_t ldw, int32_t type, int32_t group, uint32_t *c, int64_t ldc, void *s, int32_t s_type,
                                    int64_t s_n, int64_t s_g, uint8_t *z, int64_t z_n, int64_t z_g, void *stream) {
    const char *what = "int4_quantize";
    if (N <= 0 || K <= 0 || !known(type) || !known(s_type)) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape or type", what);
    CHECK(check_group(what, group));
    CHECK(check_codes(what, c, K, ldc));
    if (!w || !s || ldw < K) return mortar_fail(MORTAR_ERR_ARG, "%s: w or s is null, or rows overlap", what);
    const int64_t threads = (int64_t)N * ((K + group - 1) / group) * (group / 8);
    if (threads >= INT64_C(1) << 32) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many values", what);
    const dim3 grid((unsigned)((threads + 255) / 256));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const auto launch = [&](auto t, auto u) {
        hipLaunchKernelGGL((int4_quantize_kernel<decltype(t)::value, decltype(u)::value>), grid, dim3(256), 0, st, w, N, K, ldw, group, c, ldc, s, s_n, s_g, z, z_n, z_g);
        return launch_error(what);
    };
    const auto scales = [&](auto t) {
        return s_type == MORTAR_FP32 ? launch(t, Const<MORTAR_FP32>{}) : s_type == MORTAR_FP16 ? launch(t, Const<MORTAR_FP16>{}) : launch(t, Const<MORTAR_BF16>{});
    };
    return type == MORTAR_FP32 ? scales(Const<MORTAR_FP32>{}) : type == MORTAR_FP16 ? scales(Const<MORTAR_FP16>{}) : scales(Const<MORTAR_BF16>{});
}

extern "C" int mortar_int4_rows(const void *x, int64_t M, int32_t K, int64_t s_m, int64_t s_k, void *out, void *stream) {
    const char *what = "int4_rows";
    if (M < 0 || K <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    if (M == 0) return MORTAR_OK;
    if (!x || !out || (reinterpret_cast<uintptr_t>(x) & 1) || (reinterpret_cast<uintptr_t>(out) & 15)) return mortar_fail(MORTAR_ERR_ARG, "%s: x or out is null or not on its address", what);
    if (K >= 1 << 28 || M >= INT64_C(1) << 32 || M * ((K + 7) / 8) >= INT64_C(1) << 32) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many values", what);
    hipLaunchKernelGGL(int4_rows_kernel, dim3((unsigned)((M * ((K + 7) / 8) + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const uint16_t *>(x), M, K,
                       s_m, s_k, static_cast<uint16_t *>(out));
    return launch_error(what);
}

extern "C" int mortar_int4_form_host(int64_t M, int64_t N, int64_t K, int32_t group, int32_t *tile_n, int32_t *tile_m, int32_t *waves, int32_t *ranges) {
    const char *what = "int4_form";
    CHECK(check_group(what, group));
    if (M <= 0 || N <= 0 || K <= 0 || !tile_n || !tile_m || !waves || !ranges) return mortar_fail(MORTAR_ERR_ARG, "%s: bad argument", what);
    const Int4Plan p = plan(M, N, K, group, 2 * K);
    *tile_n = p.f ? 16 * p.f : INT4_TILES[p.tile].bn;
    *tile_m = p.f ? 16 * p.mx : INT4_TILES[p.tile].bm;
    *waves = p.xl ? -p.waves : p.f ? p.waves : 4;
    *ranges = p.splits;
    return MORTAR_OK;
}

extern "C" int64_t mortar_int4_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t group) {
    if (M <= 0 || N <= 0 || K <= 0 || group < 32) return 0;
    const Int4Plan p = plan(M, N, K, group, 2 * K);              // (the rows' distance chooses among forms of few rows only)
    if (p.f) return 0;
    return 4 * (groups_padded(K, group) * (up128(M) + 2 * up128(N)) + (p.splits > 1 ? p.splits * M * up128(N) : 0));
}

extern "C" int mortar_int4_linear(const void *x, int64_t M, int32_t K, int64_t ldx, int32_t type, const uint32_t *c, int64_t ldc, int32_t N, int32_t group, const void *s,
                                  int32_t s_type, int64_t s_n, int64_t s_g, const uint8_t *z, int64_t z_n, int64_t z_g, void *y, int64_t ldy, void *workspace,
                                  void *stream) {
    return mortar_int4_linear_part(x, M, K, K, ldx, type, c, ldc, N, group, s, s_type, s_n, s_g, z, z_n, z_g, y, ldy, workspace, stream);
}

extern "C" int mortar_int4_linear_part(const void *x, int64_t M, int32_t K, int32_t K_used, int64_t ldx, int32_t type, const uint32_t *c, int64_t ldc, int32_t N, int32_t group,
                                       const void *s, int32_t s_type, int64_t s_n, int64_t s_g, const uint8_t *z, int64_t z_n, int64_t z_g, void *y, int64_t ldy,
                                       void *workspace, void *stream) {
    const char *what = "int4_linear";
    if (M < 0 || K <= 0 || N <= 0 || K_used > K || K_used <= K - 8) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    if (type != MORTAR_BF16 && type != MORTAR_FP16) return mortar_fail(MORTAR_ERR_ARG, "%s: bf16 or fp16", what);
    if (s_type != type && s_type != MORTAR_FP32) return mortar_fail(MORTAR_ERR_ARG, "%s: scales in the type of x or fp32", what);
    CHECK(check_group(what, group));
    if (M == 0) return MORTAR_OK;
    CHECK(check_codes(what, c, K, ldc));
    if (!x || K % 8 || ldx % 8 || (M > 1 && ldx < K) || (reinterpret_cast<uintptr_t>(x) & 15)) return mortar_fail(MORTAR_ERR_ARG, "%s: x needs rows of a multiple of 8 values on 16-byte addresses", what);
    if (!s || !y || ldy < N || (reinterpret_cast<uintptr_t>(y) & 1)) return mortar_fail(MORTAR_ERR_ARG, "%s: s or y is null, or rows of y overlap", what);
    if (s_n < 0 || s_g < 0 || z_n < 0 || z_g < 0) return mortar_fail(MORTAR_ERR_ARG, "%s: negative strides", what);
    if (128 * ldx * 2 >= (int64_t)DENSE_OUTSIDE || K >= 1 << 28) return mortar_fail(MORTAR_ERR_LIMIT, "%s: the rows of x are too far apart", what);
    if (M >= INT32_MAX / 2 || N >= 1 << 24) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many rows or columns", what);
    if (mortar_int4_workspace_bytes(M, N, K, group) && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return mortar_fail(MORTAR_ERR_ARG, "%s: this shape needs a workspace", what);
    Int4Args a{};
    a.x = x; a.ldx = ldx * 2; a.c = c; a.ldc = ldc * 4;
    a.s = s; a.s_n = s_n; a.s_g = s_g; a.z = z; a.z_n = z_n; a.z_g = z_g;
    a.y = static_cast<uint16_t *>(y); a.ldy = ldy;
    a.M = (int32_t)M; a.N = N; a.K = K; a.groups = (K + group - 1) / group; a.K_used = K_used;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    float *ws = static_cast<float *>(workspace);
    return type == MORTAR_BF16 ? launch_group<DENSE_BF16>(a, group, s_type == MORTAR_FP32, ws, st, what) : launch_group<DENSE_F16>(a, group, s_type == MORTAR_FP32, ws, st, what);
}
