// Tile kernel of the dense products (gfx950): C[m, n] = sum_k P(n, k) Q(m, k), fp32 sums, P and Q in bf16, fp16 or e4m3.
//
// P is the operand whose index runs along the rows of C in memory (the matrix core's A operand: a lane then holds four
// consecutive n of one m), Q the other one.  Either is stored K-contiguous ("rows": [n or m, k]) or K-strided ("columns":
// [k, n or m], 16-bit types only, read through the transposing LDS load), which gives the three products of a linear layer:
//   y  = x W^T    P = W  rows,     Q = x  rows
//   dx = dy W     P = W  columns,  Q = dy rows
//   dW = dy^T x   P = x  columns,  Q = dy columns
//
// A workgroup computes BN x BM of C in steps of 128 bytes of K (64 16-bit values, 128 e4m3 values).  Both operands' slices go
// from global memory into LDS by asynchronous 16-byte copies (buffer loads: rows, columns and K values outside the matrix are
// given an offset beyond the record count and arrive as zeros, so no tail is treated apart), one stage ahead of the stage that
// is multiplied.  In LDS the 16-byte units are permuted within their rows so that the operand reads are free of bank conflicts;
// the permutation is applied to the copies' source addresses, their destination being linear by construction.
#ifndef MORTAR_DENSE_CORE_H
#define MORTAR_DENSE_CORE_H

#include "mortar_device.h"

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
#define MORTAR_LDS __attribute__((address_space(3)))

enum DenseType { DENSE_BF16, DENSE_F16, DENSE_E4M3 };
enum DenseEpilogue {
    DENSE_STORE,        // C in the 16-bit type (e4m3 operands: bf16)
    DENSE_PARTIAL,      // fp32 sums of one K range into a slab of the workspace
    DENSE_SWIGLU,       // P rows are gate and up features: h = silu(g) u, and g, u themselves where asked for
    DENSE_SWIGLU_BWD    // C is dh: the derivatives of the stored g, u, and h once more
};

struct DenseArgs {
    const void *p, *q;             // operands; leading dimensions in bytes
    int64_t ldp, ldq;
    int32_t M, N, K;               // N: columns of C (DENSE_SWIGLU: d_ff); K in values
    void *c;                       // C / h (DENSE_SWIGLU) / dgu (DENSE_SWIGLU_BWD) / slabs (DENSE_PARTIAL), leading dimension in values
    int64_t ldc;
    void *gu;                      // DENSE_SWIGLU: gate_up output to store or null; DENSE_SWIGLU_BWD: the stored one
    int64_t ldgu;
    void *h;                       // DENSE_SWIGLU_BWD: h to store or null
    int64_t ldh;
    const float *sx, *sw;          // e4m3: scales of Q per (m, K block) with strides, of P per (128 n, K block)
    int64_t sx_m, sx_k, sw_n;
    int32_t tiles_n, tiles_m;
    int32_t steps, splits;         // K steps in all, and how many ranges they are cut into
};

constexpr uint32_t DENSE_OUTSIDE = 0x80000000u;      // also the record count of the buffers

template <DenseType T>
__device__ __forceinline__ f32x4_t dense_mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    if constexpr (T == DENSE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else
        return mortar_mfma(a, b, c);
}

// Two floats rounded to the 16-bit output type (nearest even), and the two values of a dword as floats.
template <DenseType T>
__device__ __forceinline__ uint32_t dense_pack2(float lo, float hi) {
    if constexpr (T == DENSE_F16) {
        const f32x2_t v = {lo, hi};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
    } else {
        return bf16_pack2(lo, hi);
    }
}
template <DenseType T>
__device__ __forceinline__ f32x2_t dense_unpack2(uint32_t w) {
    if constexpr (T == DENSE_F16) return __builtin_convertvector(__builtin_bit_cast(f16x2_t, w), f32x2_t);
    else return f32x2_t{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
}

__device__ __forceinline__ u32x4_t dense_buffer(const char *base) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    return u32x4_t{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, DENSE_OUTSIDE, 0x00020000u};
}
// 16 bytes per lane, global -> LDS at lds + 16 * lane; lanes at DENSE_OUTSIDE or beyond write zeros.
__device__ __forceinline__ void dense_copy(u32x4_t buf, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(buf) : "memory", "m0");
}

// One operand's slice of ROWS (n or m) x 128 bytes of K, copied by NW waves, L instructions each.
template <int ROWS, bool COLS, int NW, int ESIZE>
struct DenseSlice {
    static constexpr int BYTES = ROWS * 128, L = BYTES / 1024 / NW;
    static_assert(L * 1024 * NW == BYTES, "whole instructions per wave");
    static constexpr int UPR = COLS ? ROWS / 8 : 8;          // 16-byte units per LDS row
    static constexpr int RPI = 64 / UPR;                     // LDS rows per instruction
    const char *base;
    uint32_t off[L];       // of this lane's unit in the first K step
    uint32_t kpos[L];      // and where in K it lies: bytes (rows) or values (columns)
    int64_t step;          // bytes from one K step to the next

    // Permutation of a K-strided slice: 32-byte pieces (16 n, one fragment's width) of the rows that one transposing read
    // touches, 4 rows per 16 lanes at distances of 8, fall into different pieces of the 256-byte bank window.
    static __device__ __forceinline__ int piece_swz(int k) {
        if constexpr (ROWS == 64) return ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
        else return (k & 3) | ((k >> 3) & 1) << 2;
    }

    // row_of(r): row of the matrix that LDS row r of a K-contiguous slice holds, relative to `base`, or -1;
    // n_left: columns from `base` on of a K-strided one.
    template <typename RowOf>
    __device__ __forceinline__ void init(const char *b, int64_t ld, int wave, int lane, RowOf row_of, int n_left) {
        base = b;
        step = COLS ? 64 * ld : 128;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int r = (wave * L + i) * RPI + lane / UPR, u = lane % UPR;
            if constexpr (COLS) {
                const int src = ((u >> 1) ^ piece_swz(r)) << 1 | (u & 1);
                kpos[i] = r;
                off[i] = src * 8 < n_left ? (uint32_t)(r * ld) + src * 16 : DENSE_OUTSIDE;
            } else {
                const int src = u ^ (r & 7), row = row_of(r);
                kpos[i] = src * 16;
                off[i] = row >= 0 ? (uint32_t)(row * ld) + src * 16 : DENSE_OUTSIDE;
            }
        }
    }
    // Copies K step s (K values in all) to LDS address `lds` (the wave's first kilobyte is wave * L).
    __device__ __forceinline__ void copy(int s, int K, uint32_t lds) const {
        const u32x4_t buf = dense_buffer(base + s * step);
        const int left = COLS ? K - s * 64 : K * ESIZE - s * 128;
        const bool whole = left >= (COLS ? 64 : 128);
#pragma unroll
        for (int i = 0; i < L; ++i) dense_copy(buf, whole || (int)kpos[i] < left ? off[i] : DENSE_OUTSIDE, lds + i * 1024);
    }
};

// Fragment (16 rows x half a K step) of a K-contiguous slice: address of K half 0; the other half lies at ^ 64.
__device__ __forceinline__ uint32_t dense_row_addr(int row, int lane) {
    return (uint32_t)((row + (lane & 15)) * 128 + (((lane >> 4) ^ (lane & 7)) * 16));
}
__device__ __forceinline__ u32x4_t dense_read(uint32_t addr) {
    return *(const MORTAR_LDS u32x4_t *)(uintptr_t)addr;
}
// The same of a K-strided slice: K values 32 s + 8 g + 4 t + {0..3} of column (lane & 15) in half t.
template <int ROWS>
__device__ __forceinline__ uint32_t dense_col_addr(int frag, int lane) {
    const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
    return (uint32_t)(k * ROWS * 2 + (frag ^ DenseSlice<ROWS, true, 1, 2>::piece_swz(k)) * 32 + (lane & 3) * 8);
}
template <int ROWS>
__device__ __forceinline__ u32x4_t dense_read_t(uint32_t addr) {
    const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MORTAR_LDS s16x4_t *)(uintptr_t)addr);
    const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MORTAR_LDS s16x4_t *)(uintptr_t)(addr + 4 * ROWS * 2));
    const u32x2_t x = __builtin_bit_cast(u32x2_t, a), y = __builtin_bit_cast(u32x2_t, b);
    return u32x4_t{x[0], x[1], y[0], y[1]};
}

// Fragments a (columns n .. n + 15) and b (n + 16 .. n + 31) as a lane holds them, four consecutive n each, to eight
// consecutive n of one of them: those of dense_lane_n.
__device__ __forceinline__ void dense_join(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ int dense_lane_n(int lane) { return ((lane >> 4) & 1) * 16 + (lane >> 5) * 8; }
__device__ __forceinline__ void dense_join8(f32x4_t a, f32x4_t b, float (&o)[8]) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const float av = a[v], bv = b[v];        // (a bit cast of the element itself reads element 0)
        uint32_t x = __builtin_bit_cast(uint32_t, av), y = __builtin_bit_cast(uint32_t, bv);
        dense_join(x, y);
        o[v] = __builtin_bit_cast(float, x);
        o[v + 4] = __builtin_bit_cast(float, y);
    }
}
template <DenseType T>
__device__ __forceinline__ u32x4_t dense_pack8(const float (&v)[8]) {
    return u32x4_t{dense_pack2<T>(v[0], v[1]), dense_pack2<T>(v[2], v[3]), dense_pack2<T>(v[4], v[5]), dense_pack2<T>(v[6], v[7])};
}
template <DenseType T>
__device__ __forceinline__ void dense_unpack8(u32x4_t w, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2_t x = dense_unpack2<T>(w[j]);
        v[2 * j] = x[0];
        v[2 * j + 1] = x[1];
    }
}

__device__ __forceinline__ float dense_sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

template <DenseType T, DenseEpilogue E, bool PC, bool QC, int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(WN *WM * 64, WN *WM >= 8 ? 2 : 2) void dense_tile_kernel(const DenseArgs a) {
    constexpr int NW = WN * WM, FN = BN / WN / 16, FM = BM / WM / 16, ES = T == DENSE_E4M3 ? 1 : 2;
    static_assert(T != DENSE_E4M3 || (!PC && !QC), "e4m3 operands are K-contiguous");
    static_assert(FN % (E == DENSE_SWIGLU ? 4 : 2) == 0, "fragments are joined in pairs");
    constexpr int PB = BN * 128, STAGE = PB + BM * 128;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wn = wave % WN, wm = wave / WN, g = lane >> 4;

    // Workgroups of one XCD (blockIdx % 8) take a contiguous run of tiles, in bands of 8 tiles along m, so that the operands
    // which the 32 of them share at a time stay in their L2.
    const int tiles = a.tiles_n * a.tiles_m;
    const int per_xcd = (tiles * a.splits + 7) >> 3;
    const int t0 = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
    if (t0 >= tiles * a.splits) return;
    const int split = t0 / tiles, t = t0 - split * tiles;
    const int band = t / (8 * a.tiles_n), rest = t - band * 8 * a.tiles_n;
    const int bh = min(8, a.tiles_m - band * 8);
    const int tn = rest / bh, tm = band * 8 + rest - tn * bh;
    const int first = (int)((int64_t)a.steps * split / a.splits), last = (int)((int64_t)a.steps * (split + 1) / a.splits);

    // DENSE_SWIGLU: LDS rows of a wave's half are BN / WN / 2 gate features, then the same up features
    constexpr int FEAT = E == DENSE_SWIGLU ? BN / 2 : BN;
    const int n0 = tn * FEAT, m0 = tm * BM;
    DenseSlice<BN, PC, NW, ES> P;
    DenseSlice<BM, QC, NW, ES> Q;
    {
        const char *pb = static_cast<const char *>(a.p) + (PC ? (int64_t)n0 * ES : (int64_t)n0 * a.ldp);
        const int n_left = a.N - n0;
        P.init(pb, a.ldp, wave, lane, [&](int r) {
            if constexpr (E == DENSE_SWIGLU) {
                constexpr int H = BN / WN / 2;
                const int f = r / (2 * H) * H + r % H;
                return f < n_left ? f + (r / H & 1) * a.N : -1;
            } else {
                return r < n_left ? r : -1;
            }
        }, n_left);
        const char *qb = static_cast<const char *>(a.q) + (QC ? (int64_t)m0 * ES : (int64_t)m0 * a.ldq);
        const int m_left = a.M - m0;
        Q.init(qb, a.ldq, wave, lane, [&](int r) { return r < m_left ? r : -1; }, m_left);
    }
    const uint32_t l0 = mortar_lds_addr(lds), lp = l0 + wave * P.L * 1024, lq = l0 + PB + wave * Q.L * 1024;
    const auto copy = [&](int s, int stage) {
        P.copy(s, a.K, lp + stage * STAGE);
        Q.copy(s, a.K, lq + stage * STAGE);
    };

    // this lane's read addresses in stage 0
    const int fp = wn * FN, fq = wm * FM;            // first fragment of the wave
    uint32_t ap[PC ? FN : 1], aq[QC ? FM : 1];
    if constexpr (PC) {
#pragma unroll
        for (int i = 0; i < FN; ++i) ap[i] = l0 + dense_col_addr<BN>(fp + i, lane);
    } else {
        ap[0] = l0 + dense_row_addr(fp * 16, lane);
    }
    if constexpr (QC) {
#pragma unroll
        for (int j = 0; j < FM; ++j) aq[j] = l0 + PB + dense_col_addr<BM>(fq + j, lane);
    } else {
        aq[0] = l0 + PB + dense_row_addr(fq * 16, lane);
    }
    const auto read_p = [&](int i, int s, uint32_t stage) {
        if constexpr (PC) return dense_read_t<BN>(ap[i] + stage + s * 32 * BN * 2);
        else return dense_read(((ap[0] + stage) ^ (s * 64)) + i * 2048);
    };
    const auto read_q = [&](int j, int s, uint32_t stage) {
        if constexpr (QC) return dense_read_t<BM>(aq[j] + stage + s * 32 * BM * 2);
        else return dense_read(((aq[0] + stage) ^ (s * 64)) + j * 2048);
    };

    f32x4_t acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // e4m3: the scales of the next step's blocks
    float sx[FM], sw = 0.f;
    const float *sxp[FM];
    const float *swp = nullptr;
    const auto load_scales = [&](int s) {
        sw = swp[s];
#pragma unroll
        for (int j = 0; j < FM; ++j) sx[j] = sxp[j][s * a.sx_k];
    };
    if constexpr (T == DENSE_E4M3) {
        const int nb = min(n0 + fp * 16, a.N - 1) >> 7;
        swp = a.sw + nb * a.sw_n;
#pragma unroll
        for (int j = 0; j < FM; ++j) sxp[j] = a.sx + min(m0 + (fq + j) * 16 + (lane & 15), a.M - 1) * a.sx_m;
        if (first < last) load_scales(first);
    }

    if (first < last) copy(first, 0);
    for (int s = first; s < last; ++s) {
        // this step's slices have landed for every wave, and every wave has read the other stage into registers
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int cur = (s - first) & 1;
        if (s + 1 < last) copy(s + 1, cur ^ 1);
        const uint32_t stage = cur * STAGE;
        if constexpr (T == DENSE_E4M3) {
            float f[FM];
#pragma unroll
            for (int j = 0; j < FM; ++j) f[j] = sx[j] * sw;
            if (s + 1 < last) load_scales(s + 1);
            i32x8_t qf[FM];
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const u32x4_t x = read_q(j, 0, stage), y = read_q(j, 1, stage);
                qf[j] = i32x8_t{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
            }
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const u32x4_t x = read_p(i, 0, stage), y = read_p(i, 1, stage);
                const i32x8_t pf = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
#pragma unroll
                for (int j = 0; j < FM; ++j) {
                    const f32x4_t d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(pf, qf[j], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[i][j][v] = __builtin_fmaf(d[v], f[j], acc[i][j][v]);
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4_t qf[FM];
#pragma unroll
                for (int j = 0; j < FM; ++j) qf[j] = read_q(j, h, stage);
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    const u32x4_t pf = read_p(i, h, stage);
#pragma unroll
                    for (int j = 0; j < FM; ++j) acc[i][j] = dense_mfma<T>(pf, qf[j], acc[i][j]);
                }
            }
        }
    }

    // ---- epilogue: pairs of fragments joined to eight consecutive n per lane, 16-byte stores
    constexpr DenseType O = T == DENSE_E4M3 ? DENSE_BF16 : T;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + (fq + j) * 16 + (lane & 15);
        if (m >= a.M) continue;
        if constexpr (E == DENSE_SWIGLU) {
            constexpr int HF = FN / 2;
#pragma unroll
            for (int i = 0; i < HF; i += 2) {
                float gt[8], up[8], hv[8];
                dense_join8(acc[i][j], acc[i + 1][j], gt);
                dense_join8(acc[HF + i][j], acc[HF + i + 1][j], up);
#pragma unroll
                for (int v = 0; v < 8; ++v) hv[v] = gt[v] * dense_sigmoid(gt[v]) * up[v];
                const int n = n0 + wn * HF * 16 + i * 16 + dense_lane_n(lane);
                if (n < a.N) {
                    *reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(a.c) + m * a.ldc + n) = dense_pack8<O>(hv);
                    if (a.gu) {
                        uint16_t *o = static_cast<uint16_t *>(a.gu) + m * a.ldgu + n;
                        *reinterpret_cast<u32x4_t *>(o) = dense_pack8<O>(gt);
                        *reinterpret_cast<u32x4_t *>(o + a.N) = dense_pack8<O>(up);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < FN; i += 2) {
                float d[8];
                dense_join8(acc[i][j], acc[i + 1][j], d);
                const int n = n0 + (fp + i) * 16 + dense_lane_n(lane);
                if (n >= a.N) continue;
                if constexpr (E == DENSE_STORE) {
                    *reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(a.c) + m * a.ldc + n) = dense_pack8<O>(d);
                } else if constexpr (E == DENSE_PARTIAL) {
                    float *o = static_cast<float *>(a.c) + ((int64_t)split * a.M + m) * a.N + n;
                    *reinterpret_cast<f32x4_t *>(o) = f32x4_t{d[0], d[1], d[2], d[3]};
                    *reinterpret_cast<f32x4_t *>(o + 4) = f32x4_t{d[4], d[5], d[6], d[7]};
                } else {
                    const uint16_t *gu = static_cast<const uint16_t *>(a.gu) + m * a.ldgu + n;
                    float gt[8], up[8], dg[8], du[8], hv[8];
                    dense_unpack8<O>(*reinterpret_cast<const u32x4_t *>(gu), gt);
                    dense_unpack8<O>(*reinterpret_cast<const u32x4_t *>(gu + a.N), up);
#pragma unroll
                    for (int v = 0; v < 8; ++v) {
                        const float sg = dense_sigmoid(gt[v]), si = gt[v] * sg;
                        hv[v] = si * up[v];
                        du[v] = d[v] * si;
                        dg[v] = d[v] * up[v] * (sg + si * (1.0f - sg));
                    }
                    uint16_t *o = static_cast<uint16_t *>(a.c) + m * a.ldc + n;
                    *reinterpret_cast<u32x4_t *>(o) = dense_pack8<O>(dg);
                    *reinterpret_cast<u32x4_t *>(o + a.N) = dense_pack8<O>(du);
                    if (a.h) *reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(a.h) + m * a.ldh + n) = dense_pack8<O>(hv);
                }
            }
        }
    }
}

#endif
