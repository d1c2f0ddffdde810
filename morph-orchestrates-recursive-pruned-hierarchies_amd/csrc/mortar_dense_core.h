// Tile kernel of the dense products (gfx950): C[m, n] = sum_k P(n, k) Q(m, k), fp32 sums, P and Q in bf16, fp16 or e4m3.
//
// P is the operand whose index runs along the rows of C in memory (the matrix core's A operand: a lane then holds four
// consecutive n of one m), Q the other one.  Either is stored K-contiguous ("rows": [n or m, k]) or K-strided ("columns":
// [k, n or m], 16-bit types only, read through the transposing LDS load), which gives the three products of a linear layer:
//   y  = x W^T    P = W  rows,     Q = x  rows
//   dx = dy W     P = W  columns,  Q = dy rows
//   dW = dy^T x   P = x  columns,  Q = dy columns
//
// A workgroup computes BN x BM of C in steps of 128 bytes of K (64 16-bit values, 128 e4m3 values), multiplied in halves.  Both operands
// go from global memory into a ring of LDS slots by asynchronous 16-byte copies (buffer loads: rows, columns and K values outside the
// matrix are given an offset beyond the record count and arrive as zeros, so no tail is treated apart), ahead of the products.  A
// slot is a whole step where an operand is K-contiguous, since its rows then are whole 128-byte lines (in halves of lines the
// products of 4096 x 2048 x 11264 take 10 to 25 % longer), and half a step where both are K-strided: the copies are then four halves
// ahead instead of one to two (dW of 2048 x 5632 from 4096 rows in no cache: 139 -> 96 us in 256 x 256 tiles).  In LDS the 16-byte
// units are permuted within their rows so that the operand reads are free of bank conflicts; the permutation is applied to the
// copies' source addresses, their destination being linear by construction.
#ifndef MORTAR_DENSE_CORE_H
#define MORTAR_DENSE_CORE_H

#include "mortar_device.h"
#include "mortar_internal.h"

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
#define MORTAR_LDS __attribute__((address_space(3)))

enum DenseType { DENSE_BF16, DENSE_F16, DENSE_E4M3 };
enum DenseEpilogue {
    DENSE_STORE,        // C in the 16-bit type (e4m3 operands: bf16)
    DENSE_PARTIAL,      // fp32 sums of one K range into a slab of the workspace
    DENSE_SWIGLU,       // P rows are gate and up features: h = silu(g) u, and g, u themselves where asked for
    DENSE_SWIGLU_BWD,   // C is dh: the derivatives of the stored g, u, and h once more
    DENSE_STREAM        // as DENSE_STORE, past the caches
};

struct DenseArgs {
    const void *p, *q;             // operands; leading dimensions in bytes
    int64_t ldp, ldq;
    int32_t M, N, K;               // N: columns of C (DENSE_SWIGLU: d_ff); K in values
    void *c;                       // C / h (DENSE_SWIGLU) / dgu (DENSE_SWIGLU_BWD) / slabs (DENSE_PARTIAL), leading dimension in values
    int64_t ldc;
    uint16_t *gu;                  // DENSE_SWIGLU: gate_up output to store or null; DENSE_SWIGLU_BWD: the stored one.  The upper 24 bits of
    uint8_t *gul;                  // the fp32 values: 16 bits [M, 2 N] in gu, 8 bits [M, 2 N] in gul
    void *h;                       // DENSE_SWIGLU_BWD: h to store or null
    int64_t ldh;
    const float *sx, *sw;          // e4m3: scales of Q per (m, K block) with strides, of P per (128 n, K block)
    int64_t sx_m, sx_k, sw_n;      // (4 M sx_m is below 2^31)
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

// One operand's slot: ROWS (n or m) x KB bytes of K, copied by NW waves in turns of one kilobyte.
template <int ROWS, bool COLS, int NW, int ESIZE, int KB>
struct DenseSlice {
    static constexpr int BYTES = ROWS * KB, COPIES = BYTES / 1024, L = (COPIES + NW - 1) / NW, LEAST = COPIES / NW;
    static constexpr int UPR = COLS ? ROWS / 8 : KB / 16;          // 16-byte units per LDS row
    static_assert(COLS || KB == 128, "rows are whole lines");
    static constexpr bool EVEN = 64 % UPR == 0;              // a copy fills whole LDS rows
    const char *base;
    uint32_t off[L];              // of this lane's unit in the first slot
    int kpos[COLS && !EVEN ? L : 1];      // where in a slot it lies: bytes (rows: the same in all copies) or values (columns)
    int64_t step;                 // bytes from one slot to the next

    // Permutation of K-contiguous rows of eight units.
    static __device__ __forceinline__ int unit(int u, int r) { return u ^ (r & 7); }
    // Permutation of K-strided rows: 32-byte pieces (16 n, one fragment's width) of the rows that one transposing read touches, 4 rows
    // per 16 lanes at distances of 8, fall into different pieces of the 256-byte bank window.
    // (Of 192 columns the last four pieces only change places among themselves: two rows of the eight meet there.)
    static __device__ __forceinline__ int piece_swz(int k) {
        if constexpr (ROWS == 64) return ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
        else return (k & 3) | ((k >> 3) & 1) << 2;
    }
    static __device__ __forceinline__ int piece(int c, int k) { return c ^ (ROWS == 192 && c >= 8 ? piece_swz(k) & 3 : piece_swz(k)); }

    // row_of(r): row of the matrix that LDS row r of a K-contiguous slice holds, relative to `base`, or -1;
    // n_left: columns from `base` on of a K-strided one.
    template <typename RowOf>
    __device__ __forceinline__ void init(const char *b, int64_t ld, int wave, int lane, RowOf row_of, int n_left) {
        base = b;
        step = COLS ? KB / 2 * ld : KB;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int t = (i * NW + wave) * 64 + lane, r = t / UPR, u = t % UPR;
            if constexpr (COLS) {
                const int src = piece(u >> 1, r) << 1 | (u & 1);
                if (i < (int)(sizeof kpos / 4)) kpos[i] = r;
                off[i] = src * 8 < n_left ? (uint32_t)(r * ld) + src * 16 : DENSE_OUTSIDE;
            } else {
                const int src = unit(u, r), row = row_of(r);
                if (i == 0) kpos[0] = src * 16;         // (r & 7 is the lane's alone)
                off[i] = row >= 0 ? (uint32_t)(row * ld) + src * 16 : DENSE_OUTSIDE;
            }
        }
    }
    // What is left of K from slot k on, in the units of kpos.
    static __device__ __forceinline__ int left(int k, int K) { return COLS ? K - k * (KB / 2) : K * ESIZE - k * KB; }
    __device__ __forceinline__ u32x4_t buffer(int k) const { return dense_buffer(base + k * step); }
    // Copy i of a slot, all of it inside K or `left` to go, to LDS address `lds` (that of the wave's first one).
    static __device__ __forceinline__ bool has(int i, int wave) { return COPIES % NW == 0 || i * NW + wave < COPIES; }
    __device__ __forceinline__ void copy(int i, int wave, u32x4_t buf, uint32_t lds) const {
        if (has(i, wave)) dense_copy(buf, off[i], lds + i * NW * 1024);
    }
    __device__ __forceinline__ void copy(int i, int wave, u32x4_t buf, int left, uint32_t lds) const {
        const int k = COLS ? (EVEN ? kpos[0] + i * NW * (64 / UPR) : kpos[EVEN ? 0 : i]) : kpos[0];
        if (has(i, wave)) dense_copy(buf, k < left ? off[i] : DENSE_OUTSIDE, lds + i * NW * 1024);
    }
};

// Fragment (16 rows x half a K step) of a K-contiguous slice: a lane holds unit (lane >> 4) of row (lane & 15).  Address of half 0; the other
// half lies at ^ 64.
__device__ __forceinline__ uint32_t dense_row_addr(int row, int lane) {
    return (uint32_t)((row + (lane & 15)) * 128 + (((lane >> 4) ^ (lane & 7)) * 16));
}
__device__ __forceinline__ u32x4_t dense_read(uint32_t addr) {
    return *(const MORTAR_LDS u32x4_t *)(uintptr_t)addr;
}
// The same of a K-strided slice: K values 32 h + 8 g + 4 t + {0..3} of column (lane & 15) in part t of half h.  Address of fragment `first` (a multiple of the
// power of two that is the number of the wave's fragments); fragment first + i lies at ^ (32 i).
template <int ROWS>
__device__ __forceinline__ uint32_t dense_col_addr(int first, int lane) {
    const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
    return (uint32_t)(k * ROWS * 2 + DenseSlice<ROWS, true, 1, 2, 64>::piece(first, k) * 32 + (lane & 3) * 8);
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

// The gate and up values that the backward needs are kept in the upper 24 bits of their fp32 sums, 16 bits in one array and 8 in
// another: rounded to 16 alone, they were the largest part of the gradients' error (root mean square 3.5e-3 of the bf16 gradients
// instead of 2.4e-3, of which 1.7e-3 is their own rounding).  One byte more per value is 2 % of a training step.
__device__ __forceinline__ uint32_t dense_round24(float f) { return __builtin_bit_cast(uint32_t, f) + 0x80u; }       // (a NaN of the matrix cores has zeros there)
__device__ __forceinline__ uint32_t dense_hi2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t dense_lo4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0501u), __builtin_amdgcn_perm(b, a, 0x0c0c0501u), 0x05040100u);
}
__device__ __forceinline__ void dense_store24(uint16_t *hi, uint8_t *lo, int64_t at, const float (&v)[8]) {
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = dense_round24(v[j]);
    *reinterpret_cast<u32x4_t *>(hi + at) = u32x4_t{dense_hi2(u[0], u[1]), dense_hi2(u[2], u[3]), dense_hi2(u[4], u[5]), dense_hi2(u[6], u[7])};
    *reinterpret_cast<u32x2_t *>(lo + at) = u32x2_t{dense_lo4(u[0], u[1], u[2], u[3]), dense_lo4(u[4], u[5], u[6], u[7])};
}
struct Dense24 {                                     // eight of them as they are stored
    u32x4_t h;
    u32x2_t l;
};
__device__ __forceinline__ Dense24 dense_load24(const uint16_t *hi, const uint8_t *lo, int64_t at) {
    return {*reinterpret_cast<const u32x4_t *>(hi + at), *reinterpret_cast<const u32x2_t *>(lo + at)};
}
__device__ __forceinline__ void dense_values24(const Dense24 &x, float (&v)[8]) {
    constexpr uint32_t pick[4] = {0x0504000cu, 0x0706010cu, 0x0504020cu, 0x0706030cu};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t hw = x.h[j >> 1], lw = x.l[j >> 2];
        v[j] = __builtin_bit_cast(float, __builtin_amdgcn_perm(hw, lw, pick[j & 3]));
    }
}

__device__ __forceinline__ float dense_sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

template <int V>
struct Const {
    static constexpr int value = V;
};

constexpr int dense_slot_bytes(bool pc, bool qc) { return pc && qc ? 64 : 128; }

template <DenseType T, DenseEpilogue E, bool PC, bool QC, int BN, int BM, int WN, int WM, int NS>
__global__ __launch_bounds__(WN *WM * 64, 2) void dense_tile_kernel(const DenseArgs a) {
    constexpr int NW = WN * WM, FN = BN / WN / 16, FM = BM / WM / 16, ES = T == DENSE_E4M3 ? 1 : 2;
    static_assert(T != DENSE_E4M3 || (!PC && !QC), "e4m3 operands are K-contiguous");
    static_assert(FN % (E == DENSE_SWIGLU ? 4 : 2) == 0, "fragments are joined in pairs");
    static_assert((FN & (FN - 1)) == 0, "K-strided fragments of P are found by xor");
    constexpr int KB = dense_slot_bytes(PC, QC), PER_STEP = 128 / KB;       // slots per step
    using SliceP = DenseSlice<BN, PC, NW, ES, KB>;
    using SliceQ = DenseSlice<BM, QC, NW, ES, KB>;
    constexpr int SLOT = SliceP::BYTES + SliceQ::BYTES, RING = NS * SLOT, LEAST = SliceP::LEAST + SliceQ::LEAST;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wn = wave % WN, wm = wave / WN;
    const int fp = wn * FN, fq = wm * FM;            // first fragments of the wave
    const uint32_t l0 = mortar_lds_addr(lds), lp = l0 + wave * 1024, lq = l0 + SliceP::BYTES + wave * 1024;
    const uint32_t ap = l0 + (PC ? dense_col_addr<BN>(fp, lane) : dense_row_addr(fp * 16, lane));
    constexpr bool XQ = (FM & (FM - 1)) == 0;        // K-strided fragments of Q are found by xor, too, if their number is a power of two
    uint32_t aq[QC && !XQ ? FM : 1];
#pragma unroll
    for (int j = 0; j < (int)(sizeof aq / 4); ++j) aq[j] = l0 + SliceP::BYTES + (QC ? dense_col_addr<BM>(fq + j, lane) : dense_row_addr(fq * 16, lane));
    const auto read_p = [&](int i, int h, uint32_t slot) {
        if constexpr (PC) return dense_read_t<BN>(((ap + slot) ^ (i * 32)) + h * 32 * BN * 2);
        else return dense_read(((ap + slot) ^ (h * 64)) + i * 2048);
    };
    const auto read_q = [&](int j, int h, uint32_t slot) {
        if constexpr (QC) return dense_read_t<BM>((XQ ? (aq[0] + slot) ^ (j * 32) : aq[XQ ? 0 : j] + slot) + h * 32 * BM * 2);
        else return dense_read(((aq[0] + slot) ^ (h * 64)) + j * 2048);
    };

    // Workgroups of one XCD (blockIdx % 8) walk over a contiguous run of tiles, in bands of 8 tiles along m, so that the operands
    // which the 32 of them share at a time stay in their L2.
    const int tiles = a.tiles_n * a.tiles_m, total = tiles * a.splits;
    const int xcd = blockIdx.x & 7, stride = gridDim.x >> 3, per_xcd = (total + 7) >> 3;
    const int end = min(total, (xcd + 1) * per_xcd);
    constexpr int FEAT = E == DENSE_SWIGLU ? BN / 2 : BN;
    struct Tile {
        int n0, m0, split, first, last;
    };
    const auto tile_of = [&](int id) {
        Tile r;
        r.split = id / tiles;
        const int t = id - r.split * tiles, band = t / (8 * a.tiles_n), rest = t - band * 8 * a.tiles_n;
        const int bh = min(8, a.tiles_m - band * 8), tn = rest / bh;
        r.n0 = tn * FEAT;
        r.m0 = (band * 8 + rest - tn * bh) * BM;
        r.first = a.steps * r.split / a.splits;
        r.last = a.steps * (r.split + 1) / a.splits;
        return r;
    };
    SliceP P;
    SliceQ Q;
    const auto aim = [&](const Tile &t) {
        const char *pb = static_cast<const char *>(a.p) + (PC ? (int64_t)t.n0 * ES : (int64_t)t.n0 * a.ldp);
        const int n_left = a.N - t.n0;
        P.init(pb, a.ldp, wave, lane, [&](int r) {
            if constexpr (E == DENSE_SWIGLU) {       // LDS rows of a wave's half are BN / WN / 2 gate features, then the same up features
                constexpr int H = BN / WN / 2;
                const int f = r / (2 * H) * H + r % H;
                return f < n_left ? f + (r / H & 1) * a.N : -1;
            } else {
                return r < n_left ? r : -1;
            }
        }, n_left);
        const char *qb = static_cast<const char *>(a.q) + (QC ? (int64_t)t.m0 * ES : (int64_t)t.m0 * a.ldq);
        const int m_left = a.M - t.m0;
        Q.init(qb, a.ldq, wave, lane, [&](int r) { return r < m_left ? r : -1; }, m_left);
    };
    // Copies run NS slots ahead of the products over the slots of this workgroup's tiles, one behind the other: slot `ahead` of the
    // tile `aim_id` is the next to be copied.
    const auto behind = [](uint32_t slot) { return slot + SLOT == RING ? 0u : slot + SLOT; };
    int id = xcd * per_xcd + (int)(blockIdx.x >> 3);
    if (id >= end) return;
    int aim_id = id, ahead, ahead_last;
    const auto aim_at = [&](int which) {
        const Tile t = tile_of(which);
        aim(t);
        ahead = PER_STEP * t.first;
        ahead_last = PER_STEP * t.last;
    };
    const auto advance = [&] {
        if (++ahead == ahead_last && (aim_id += stride) < end) aim_at(aim_id);
    };
    const auto copying = [&] { return aim_id < end; };
    // Copy q of the wave's for slot k, all of it inside K (plain) or with the tails looked after.
    const auto copy = [&](auto plain, int q, int k, u32x4_t pb, u32x4_t qb, uint32_t slot) {
        if constexpr (plain.value) {
            if (q < SliceP::L) P.copy(q, wave, pb, lp + slot);
            else Q.copy(q - SliceP::L, wave, qb, lq + slot);
        } else {
            if (q < SliceP::L) P.copy(q, wave, pb, P.left(k, a.K), lp + slot);
            else Q.copy(q - SliceP::L, wave, qb, Q.left(k, a.K), lq + slot);
        }
    };
    constexpr int COPIES = SliceP::L + SliceQ::L;
    // Waits until this wave's copies of a slot have landed and every wave is here, all its LDS reads done.  `newer` slots were copied
    // behind that one if there still is one to be copied: then their copies may be on their way.
    const auto meet = [&](auto newer, auto plain) {
        if (plain.value || (newer.value > 0 && copying())) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(newer.value * LEAST) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    aim_at(id);
    uint32_t slot = 0;                               // of the values that are multiplied next
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if (copying()) {
            const u32x4_t pb = P.buffer(ahead), qb = Q.buffer(ahead);
#pragma unroll
            for (int q = 0; q < COPIES; ++q) copy(Const<0>{}, q, ahead, pb, qb, i * SLOT);
            advance();
        }
    [[maybe_unused]] u32x4_t pf[T == DENSE_E4M3 ? 1 : 2][FN], qf[T == DENSE_E4M3 ? 1 : 2][FM];
    meet(Const<NS - 1>{}, Const<0>{});
    if constexpr (T != DENSE_E4M3) {
#pragma unroll
        for (int j = 0; j < FM; ++j) qf[0][j] = read_q(j, 0, slot);
#pragma unroll
        for (int i = 0; i < FN; ++i) pf[0][i] = read_p(i, 0, slot);
        if constexpr (PER_STEP == 2) meet(Const<NS - 2>{}, Const<0>{});
    }
    for (;;) {
    f32x4_t acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const Tile cur = tile_of(id);
    const int n0 = cur.n0, m0 = cur.m0;
    id += stride;
    const bool more = id < end;

    int s = cur.first;
    const int plain_end = cur.last - 1 - (NS + PER_STEP - 1) / PER_STEP;     // up to here a step's copies are of whole slots of this tile

    if constexpr (T == DENSE_E4M3) {
        // One matrix instruction is a step deep: FN groups of FM products, scaled and added a group later.  Fragments of P are read two groups
        // ahead, those of Q behind their last use; all waves meet two groups before the end, when the step is in registers.
        const int nb = min(n0 + fp * 16, a.N - 1) >> 7;
        const float *swp = a.sw + nb * a.sw_n;
        uint32_t sxo[FM];                             // bytes
        float sx[FM], sw;                             // the scales of the next step
#pragma unroll
        for (int j = 0; j < FM; ++j) sxo[j] = (uint32_t)(min(m0 + (fq + j) * 16 + (lane & 15), a.M - 1) * (int)a.sx_m) * 4;
        const auto load_scales = [&](int k) {
            sw = swp[k];
            const char *row = reinterpret_cast<const char *>(a.sx + k * a.sx_k);
#pragma unroll
            for (int j = 0; j < FM; ++j) sx[j] = *reinterpret_cast<const float *>(row + sxo[j]);
        };
        float sum[FN][FM][4];                         // (single floats: as vectors they are copied about)
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) sum[i][j][v] = 0.f;
        const auto whole = [](u32x4_t x, u32x4_t y) { return i32x8_t{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]}; };
        i32x8_t p8[FN], q8[FM];
        load_scales(s);
#pragma unroll
        for (int j = 0; j < FM; ++j) q8[j] = whole(read_q(j, 0, slot), read_q(j, 1, slot));
#pragma unroll
        for (int i = 0; i < 2; ++i) p8[i] = whole(read_p(i, 0, slot), read_p(i, 1, slot));
        constexpr int MEET = FN - 2;
        const auto step = [&](auto on, auto plain, int k, int scales) {          // as below; scales: the step whose scales are loaded
            float f[FM];
#pragma unroll
            for (int j = 0; j < FM; ++j) f[j] = sx[j] * sw;
            if constexpr (on.value) load_scales(scales);
            f32x4_t d[2][FM];
            const auto add = [&](int i, int j) {
#pragma unroll
                for (int v = 0; v < 4; ++v) sum[i][j][v] = __builtin_fmaf(d[i & 1][j][v], f[j], sum[i][j][v]);
            };
            const uint32_t next = behind(slot);
            constexpr int EACH = (COPIES + FN - MEET - 1) / (FN - MEET);
            bool go = true;
            u32x4_t pb{}, qb{};
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                if (i == MEET) {                      // the step is in registers, or will be without its slot
                    meet(Const<NS - 2>{}, plain);
                    if constexpr (!plain.value) k = ahead, go = copying();
                    pb = P.buffer(k), qb = Q.buffer(k);
                }
                if (i + 2 < FN) p8[i + 2] = whole(read_p(i + 2, 0, slot), read_p(i + 2, 1, slot));
                else if constexpr (on.value) p8[i + 2 - FN] = whole(read_p(i + 2 - FN, 0, next), read_p(i + 2 - FN, 1, next));
                if (i >= MEET && go) {
#pragma unroll
                    for (int q = (i - MEET) * EACH; q < (i - MEET + 1) * EACH && q < COPIES; ++q) copy(plain, q, k, pb, qb, slot);
                }
#pragma unroll
                for (int j = 0; j < FM; ++j) {
                    d[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p8[i], q8[j], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
                    if (i) add(i - 1, j);
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (on.value)
                        if (i == FN - 1) q8[j] = whole(read_q(j, 0, next), read_q(j, 1, next));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < FM; ++j) add(FN - 1, j);
            __builtin_amdgcn_sched_barrier(0);
            if (!plain.value && go) advance();
            slot = next;
        };
        if (s < plain_end) {
            for (; s < plain_end; ++s) step(Const<1>{}, Const<1>{}, s + NS, s + 1);
            ahead = s + NS;
        }
        for (; s + 1 < cur.last; ++s) step(Const<1>{}, Const<0>{}, 0, s + 1);
        step(Const<0>{}, Const<0>{}, 0, 0);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = f32x4_t{sum[i][j][0], sum[i][j][1], sum[i][j][2], sum[i][j][3]};
    } else {
        // While the matrix cores work on one half the next one is read from LDS into the other set of registers.  Behind the half that read the
        // last of a slot all waves meet: that slot is then in registers everywhere and copied over next, and the slot behind it has landed.
        // The reads of a group of FM products: the fragments of Q first, then those of P, each behind the products that free a register for it.
        constexpr int EACH = (COPIES + FN - 1) / FN;
        constexpr auto reads = [](int groups) { return groups == 0 ? 0 : groups == FN ? FM + FN : FM + (3 * (groups - 1) / 2 < FN ? 3 * (groups - 1) / 2 : FN); };
        // set: of the registers that are multiplied, the half of the step; on: there is a next half; plain: the copies are of a whole slot of
        // this tile, k the one due
        const auto half = [&](auto set, bool on, auto plain, int k) {
            constexpr bool LAST = PER_STEP == 2 || set.value == 1;        // of its slot: that is free, the next half is in the next one
            const uint32_t next = LAST ? behind(slot) : slot;
            constexpr int h = PER_STEP == 2 ? 0 : 1 - set.value;
            if constexpr (!plain.value) k = ahead;
            const bool go = LAST && (plain.value || copying());
            const u32x4_t pb = P.buffer(k), qb = Q.buffer(k);
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                if (on) {
#pragma unroll
                    for (int q = reads(i); q < reads(i + 1); ++q) {
                        if (q < FM) qf[1 - set.value][q] = read_q(q, h, next);
                        else pf[1 - set.value][q - FM] = read_p(q - FM, h, next);
                    }
                }
                if (go) {
#pragma unroll
                    for (int q = i * EACH; q < (i + 1) * EACH && q < COPIES; ++q) copy(plain, q, k, pb, qb, slot);
                }
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[i][j] = dense_mfma<T>(pf[set.value][i], qf[set.value][j], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!plain.value && go) advance();
            if constexpr (PER_STEP == 2 || set.value == 0) meet(Const<NS - 2>{}, plain);
            slot = next;
        };
        if (s < plain_end) {
            for (; s < plain_end; ++s) {
                half(Const<0>{}, true, Const<1>{}, PER_STEP * s + NS);
                half(Const<1>{}, true, Const<1>{}, PER_STEP * (s + 1) - 1 + NS);
            }
            ahead = PER_STEP * s + NS;
        }
        for (; s < cur.last; ++s) {
            half(Const<0>{}, true, Const<0>{}, 0);
            half(Const<1>{}, more || s + 1 < cur.last, Const<0>{}, 0);
        }
    }

    // ---- epilogue: pairs of fragments joined to eight consecutive n per lane, 16-byte stores
    constexpr DenseType O = T == DENSE_E4M3 ? DENSE_BF16 : T;
    if constexpr (E == DENSE_SWIGLU_BWD) {
        // The gate and up values of a pair of fragments are loaded AHEAD pairs early, since loads wait for the stores before them: 4096 rows,
        // 2048 and 5632 wide 160 -> 151 us in 256 x 192.  A wave of the 64 x 64 tile has two pairs, whose loads the compiler puts first.
        constexpr int PAIRS = FN / 2, ITEMS = FM * PAIRS, AHEAD = FM == 1 ? 0 : FM * FN >= 32 ? 1 : 2, HELD = AHEAD ? AHEAD : 1;
        Dense24 kept[HELD][2];
        const auto row = [&](int q) { return m0 + (fq + q / PAIRS) * 16 + (lane & 15); };
        const auto column = [&](int q) { return n0 + (fp + q % PAIRS * 2) * 16 + dense_lane_n(lane); };
        const auto fetch = [&](int q) {
            const int n = column(q);
            const int64_t at = (int64_t)min(row(q), a.M - 1) * 2 * a.N + (n < a.N ? n : 0);
            kept[q % HELD][0] = dense_load24(a.gu, a.gul, at);
            kept[q % HELD][1] = dense_load24(a.gu, a.gul, at + a.N);
        };
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) fetch(q);
#pragma unroll
        for (int q = 0; q < ITEMS; ++q) {
            float d[8], gt[8], up[8], dg[8], du[8], hv[8];
            if (AHEAD == 0) fetch(q);
            dense_values24(kept[q % HELD][0], gt);
            dense_values24(kept[q % HELD][1], up);
            dense_join8(acc[q % PAIRS * 2][q / PAIRS], acc[q % PAIRS * 2 + 1][q / PAIRS], d);
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                const float sg = dense_sigmoid(gt[v]), si = gt[v] * sg;
                hv[v] = si * up[v];
                du[v] = d[v] * si;
                dg[v] = d[v] * up[v] * (sg + si * (1.0f - sg));
            }
            if (AHEAD && q + AHEAD < ITEMS) fetch(q + AHEAD);
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
            const int64_t m = row(q);
            const int n = column(q);
            if (m < a.M && n < a.N) {
                uint16_t *o = static_cast<uint16_t *>(a.c) + m * a.ldc + n;
                *reinterpret_cast<u32x4_t *>(o) = dense_pack8<O>(dg);
                *reinterpret_cast<u32x4_t *>(o + a.N) = dense_pack8<O>(du);
                if (a.h) *reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(a.h) + m * a.ldh + n) = dense_pack8<O>(hv);
            }
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
        }
    } else {
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
                        const int64_t at = m * 2 * a.N + n;
                        dense_store24(a.gu, a.gul, at, gt);
                        dense_store24(a.gu, a.gul, at + a.N, up);
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
                } else if constexpr (E == DENSE_STREAM) {
                    __builtin_nontemporal_store(dense_pack8<O>(d), reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(a.c) + m * a.ldc + n));
                } else if constexpr (E == DENSE_PARTIAL) {
                    float *o = static_cast<float *>(a.c) + ((int64_t)cur.split * a.M + m) * a.N + n;
                    *reinterpret_cast<f32x4_t *>(o) = f32x4_t{d[0], d[1], d[2], d[3]};
                    *reinterpret_cast<f32x4_t *>(o + 4) = f32x4_t{d[4], d[5], d[6], d[7]};
                }
            }
        }
    }
    }
    if (!more) return;
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------

// The tiles: BN x BM of C by WN x WM waves, LDS steps (slots: twice as many halves, and one more where they fit), workgroups per CU.  The larger the tile the fewer bytes go through the L1 for a
// product (64 per cycle and CU is what it takes: at the full matrix rate 256 x 256 would keep it half busy, 256 x 128 three quarters); the smaller ones
// are for matrices that do not fill the chip with large ones.
struct DenseTile {
    int bn, bm, wn, wm, steps, halves, per_cu;
};
constexpr DenseTile DENSE_TILES[] = {{256, 256, 2, 4, 2, 5, 1}, {256, 192, 2, 4, 2, 5, 1}, {256, 128, 4, 2, 3, 6, 1}, {128, 128, 2, 2, 2, 5, 2}, {64, 64, 1, 4, 4, 10, 2}};
constexpr int DENSE_N_TILES = sizeof DENSE_TILES / sizeof DENSE_TILES[0];
// The first tile of the e4m3 products: 256 x 256 does not fit the registers beside the unscaled sums (4096 x 2048 x 11264 in 320 us, where
// 256 x 192, 256 x 128 and 128 x 128 take 138, 137 and 121).
constexpr int DENSE_E4M3_FIRST = 1;

template <DenseType T, DenseEpilogue E, bool PC, bool QC, int I = 0>
int dense_launch(DenseArgs a, int tile, hipStream_t st, const char *what) {
    if constexpr (T == DENSE_E4M3 && I < DENSE_E4M3_FIRST) return dense_launch<T, E, PC, QC, DENSE_E4M3_FIRST>(a, tile, st, what);
    else {
    if constexpr (I + 1 < DENSE_N_TILES)
        if (tile != I) return dense_launch<T, E, PC, QC, I + 1>(a, tile, st, what);
    constexpr DenseTile D = DENSE_TILES[I];
    constexpr int kb = dense_slot_bytes(PC, QC), slots = kb == 64 ? D.halves : D.steps;
    const auto kern = dense_tile_kernel<T, E, PC, QC, D.bn, D.bm, D.wn, D.wm, slots>;
    constexpr int smem = slots * (D.bn + D.bm) * kb, feat = E == DENSE_SWIGLU ? D.bn / 2 : D.bn;
    static_assert(smem * D.per_cu <= 160 * 1024, "LDS");
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    const int64_t tn = ((int64_t)a.N + feat - 1) / feat, tm = ((int64_t)a.M + D.bm - 1) / D.bm, total = tn * tm * a.splits;
    if (total > (1 << 30)) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many tiles", what);
    a.tiles_n = (int)tn;
    a.tiles_m = (int)tm;
    const int64_t per_xcd = (total + 7) / 8, room = 32 * D.per_cu;
    hipLaunchKernelGGL(kern, dim3((unsigned)(8 * (per_xcd < room ? per_xcd : room))), dim3(D.wn * D.wm * 64), smem, st, a);
    const hipError_t l = hipGetLastError();
    return l == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(l));
    }
}

#endif
