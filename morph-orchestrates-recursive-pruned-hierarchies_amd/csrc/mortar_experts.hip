// Tokens sorted by expert and back.  A token n has k slots, each with the number of an expert or empty (any number outside 0 .. E - 1):
//   sort       position[n, j] = row of slot (n, j) when all N k slots are sorted by expert, in the order of the slots within one (a stable counting
//              sort), the empty ones behind all others; token[row] = n; offsets[e] = the first row of expert e, offsets[E] = the full rows
//   dispatch   xs[position[n, j]] = x[n], zeros in the rows of empty slots;     backward: dx[n] = sum_j dxs[position[n, j]] over full slots
//   combine    y[n] = sum_j w[n, j] ys[position[n, j]] over full slots
//              backward: dys[position[n, j]] = w[n, j] dy[n] (zeros for empty slots),  dw[n, j] = <dy[n], ys[position[n, j]]> (0 for empty ones)
// Positions are a permutation of the rows, so every row is written by exactly one wave and no atomics are needed: sums run over a token's slots in
// their order, in fp32, and are rounded once.  Rows of empty slots are not read.  What bounds all but the sort is the memory.
// A position that is none of the rows takes its slot out of the order; the row that it had is then named by no slot.  With the tokens of the rows at hand a wave
// looks whether its row is, and makes it zeros otherwise.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mortar_device.h"
#include "mortar_internal.h"

namespace {

constexpr int MOST_EXPERTS = 1024, MOST_SLOTS = (1 << 26) - 4;  // (a wave per slot, four per workgroup: a grid has fewer than 2^32 threads)

int launch_error(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// ---- sort ------------------------------------------------------------------------------------------------------------
// Workgroups of 16 waves, each with a run of slots: first they count the slots per expert, then each of them adds up what lies in front of its own (the
// experts in front, the runs in front) and places its slots.  A wave owns 64 HELD consecutive slots and keeps their experts in registers; the counts of a
// run are kept per wave, so that the order within a run needs nothing of other waves but their counts, and within 64 slots it is found with one
// ballot per bit of the expert's number.  Few slots are one workgroup's, in one launch.  Both launches are chains of latencies: ids, counts, sums.
// Measured: up to 4096 slots 2.7 us, 32768 slots of 64 experts 4.7 + 4.7 behind other work, 3.2 + 5.2 of 16.
constexpr int SORT_WAVES = 16, SORT_THREADS = SORT_WAVES * 64, SORT_ALONE = 4096, SORT_BLOCKS = 64;

template <typename ID>
struct Slots {
    const ID *ids;
    int64_t n;
    int experts;
};

// The experts of this wave's slots, from `at` on (-1: no slot), and counts[e] of them: one row of `counts` per wave, in LDS and zeroed here.
template <typename ID, int HELD>
__device__ __forceinline__ void count_run(const Slots<ID> &s, int64_t at, int (&key)[HELD], int *counts) {
    const int keys = s.experts + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    ID id[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) id[h] = at + h * 64 + lane < s.n ? s.ids[at + h * 64 + lane] : 0;
    for (int i = lane; i < keys; i += 64) counts[wave * keys + i] = 0;          // (a wave's row is its own)
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        key[h] = at + h * 64 + lane < s.n ? (id[h] >= 0 && id[h] < s.experts ? (int)id[h] : s.experts) : -1;
        if (key[h] >= 0) atomicAdd(&counts[wave * keys + key[h]], 1);
    }
    __syncthreads();
}

// totals [expert][run]: those of one expert lie together, where a thread reads them.
template <typename ID, int HELD>
__global__ __launch_bounds__(SORT_THREADS) void expert_count_kernel(const Slots<ID> s, int32_t *totals) {
    extern __shared__ int counts[];
    const int keys = s.experts + 1;
    int key[HELD];
    count_run(s, ((int64_t)blockIdx.x * SORT_WAVES + (threadIdx.x >> 6)) * 64 * HELD, key, counts);
    for (int e = threadIdx.x; e < keys; e += SORT_THREADS) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) sum += counts[w * keys + e];
        totals[(int64_t)e * gridDim.x + blockIdx.x] = sum;
    }
}

// Exclusive sums of v over the workgroup's threads.
__device__ __forceinline__ int scan_workgroup(int v, int *part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) base += w < wave ? part[w] : 0;
    return base + sum - v;
}

// ALONE: one workgroup has all slots and no totals of others.
template <typename ID, int HELD, bool ALONE>
__global__ __launch_bounds__(SORT_THREADS) void expert_place_kernel(const Slots<ID> s, uint32_t slots_per_token, const int32_t *totals, int32_t *position, int32_t *token,
                                                                    int32_t *offsets) {
    extern __shared__ int counts[];
    __shared__ int part[2][SORT_WAVES];
    const int keys = s.experts + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t at = ((int64_t)blockIdx.x * SORT_WAVES + wave) * 64 * HELD;
    int all[2] = {0, 0}, mine[2] = {0, 0};               // of experts threadIdx.x and (the one key beyond 1024) threadIdx.x + 1024
    if constexpr (!ALONE) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = threadIdx.x + k * SORT_THREADS;
            if (e >= keys) continue;
            const int32_t *t = totals + (int64_t)e * gridDim.x;
            const int runs = gridDim.x, own = blockIdx.x;
            for (int b = 0; b < runs; b += 16) {         // (sixteen loads on their way)
                int c[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) c[i] = t[min(b + i, runs - 1)];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    mine[k] += b + i < own ? c[i] : 0;
                    all[k] += b + i < runs ? c[i] : 0;
                }
            }
        }
    }
    int key[HELD];
    count_run(s, at, key, counts);
    // Rows in front of this workgroup's slots of an expert, and from them those of each wave: in place of the counts.
    int before = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int e = threadIdx.x + k * SORT_THREADS;
        if (k * SORT_THREADS >= keys) break;
        int c[SORT_WAVES];
        if (e < keys) {
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                c[w] = counts[w * keys + e];
                if (ALONE) all[k] += c[w];
            }
        }
        const int front = before + scan_workgroup(all[k], part[k]);
        if (e < keys) {
            int row = front + mine[k];
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                counts[w * keys + e] = row;
                row += c[w];
            }
            if (blockIdx.x == 0) offsets[e] = front;
        }
        if (k == 0) {
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) before += part[0][w];
        }
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(s.experts);
    int *next = counts + wave * keys;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int64_t i = at + h * 64 + lane;
        const bool on = key[h] >= 0;
        uint64_t same = __ballot(on);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(key[h] >> b & 1);
            same &= key[h] >> b & 1 ? set : ~set;
        }
        const int rank = __popcll(same & ((UINT64_C(1) << lane) - 1));
        int row = 0;
        if (on) row = __hip_atomic_load(next + key[h], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) + rank;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (on && same >> lane == 1) __hip_atomic_store(next + key[h], row + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);      // the last lane of its expert
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (on) {
            position[i] = row;
            token[row] = (int32_t)((uint32_t)i / slots_per_token);
        }
    }
}

// Slots that a lane holds: a power of two, so that there are at most SORT_BLOCKS runs up to 2^20 slots.
int held_of(int64_t n) {
    for (const int held : {2, 4, 8})
        if (n <= (int64_t)SORT_BLOCKS * SORT_THREADS * held) return held;
    return 16;
}

template <typename ID, int HELD>
int sort_held(const Slots<ID> &s, int slots_per_token, int32_t *position, int32_t *token, int32_t *offsets, int32_t *totals, hipStream_t st, const char *what) {
    const int smem = (s.experts + 1) * SORT_WAVES * 4;
    const auto room = [&](const void *kern) {
        return smem <= 64 * 1024 ? hipSuccess : hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (MOST_EXPERTS + 1) * SORT_WAVES * 4);
    };
    if (s.n <= SORT_ALONE) {
        const auto kern = expert_place_kernel<ID, HELD, true>;
        if (const hipError_t e = room(reinterpret_cast<const void *>(kern)); e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
        hipLaunchKernelGGL(kern, dim3(1), dim3(SORT_THREADS), smem, st, s, (uint32_t)slots_per_token, nullptr, position, token, offsets);
        return launch_error(what);
    }
    const unsigned blocks = (unsigned)((s.n + SORT_THREADS * HELD - 1) / (SORT_THREADS * HELD));
    const auto count = expert_count_kernel<ID, HELD>;
    const auto place = expert_place_kernel<ID, HELD, false>;
    for (const void *kern : {reinterpret_cast<const void *>(count), reinterpret_cast<const void *>(place)})
        if (const hipError_t e = room(kern); e != hipSuccess) return mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    hipLaunchKernelGGL(count, dim3(blocks), dim3(SORT_THREADS), smem, st, s, totals);
    if (const int rc = launch_error(what)) return rc;
    hipLaunchKernelGGL(place, dim3(blocks), dim3(SORT_THREADS), smem, st, s, (uint32_t)slots_per_token, totals, position, token, offsets);
    return launch_error(what);
}
template <typename ID>
int sort(const Slots<ID> &s, int slots_per_token, int32_t *position, int32_t *token, int32_t *offsets, int32_t *totals, hipStream_t st, const char *what) {
    if (s.n <= SORT_ALONE) return s.n <= 1024 ? sort_held<ID, 1>(s, slots_per_token, position, token, offsets, totals, st, what) : sort_held<ID, 4>(s, slots_per_token, position, token, offsets, totals, st, what);
    switch (held_of(s.n)) {
        case 2: return sort_held<ID, 2>(s, slots_per_token, position, token, offsets, totals, st, what);
        case 4: return sort_held<ID, 4>(s, slots_per_token, position, token, offsets, totals, st, what);
        case 8: return sort_held<ID, 8>(s, slots_per_token, position, token, offsets, totals, st, what);
        default: return sort_held<ID, 16>(s, slots_per_token, position, token, offsets, totals, st, what);
    }
}

// ---- rows ------------------------------------------------------------------------------------------------------------
// Rows are read and written in 16-byte units on whatever addresses they lie (odd widths: multiples of 2 bytes), what is left behind the last whole one
// value by value.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
template <bool STREAM>
__device__ __forceinline__ void put16(char *p, u32x4_any_t w) {
    if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any_t *>(p));
    else *reinterpret_cast<u32x4_any_t *>(p) = w;
}

template <int TYPE>
struct Row {
    static constexpr int UNIT = TYPE == MORTAR_FP32 ? 4 : 8, SIZE = 16 / UNIT;
    static __device__ __forceinline__ u32x4_t load(const char *p) { return *reinterpret_cast<const u32x4_any_t *>(p); }
    static __device__ __forceinline__ void store(char *p, u32x4_t w) { *reinterpret_cast<u32x4_any_t *>(p) = w; }
    static __device__ __forceinline__ void unpack(u32x4_t w, float (&v)[UNIT]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t d = w[j];
            if constexpr (TYPE == MORTAR_FP32) {
                v[j] = __builtin_bit_cast(float, d);
            } else if constexpr (TYPE == MORTAR_FP16) {
                const f32x2_t f = __builtin_convertvector(__builtin_bit_cast(f16x2_t, d), f32x2_t);
                v[2 * j] = f[0], v[2 * j + 1] = f[1];
            } else {
                v[2 * j] = __builtin_bit_cast(float, d << 16);
                v[2 * j + 1] = __builtin_bit_cast(float, d & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ u32x4_t pack(const float (&v)[UNIT]) {
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == MORTAR_FP32) w[j] = __builtin_bit_cast(uint32_t, v[j]);
            else if constexpr (TYPE == MORTAR_FP16) w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * j], v[2 * j + 1]}, f16x2_t));
            else w[j] = bf16_pack2(v[2 * j], v[2 * j + 1]);
        }
        return w;
    }
    static __device__ __forceinline__ float one(const char *p) {
        if constexpr (TYPE == MORTAR_FP32) return *reinterpret_cast<const float *>(p);
        else if constexpr (TYPE == MORTAR_FP16) return (float)*reinterpret_cast<const _Float16 *>(p);
        else return bf16_to_f32(*reinterpret_cast<const uint16_t *>(p));
    }
    static __device__ __forceinline__ void put(char *p, float v) {
        if constexpr (TYPE == MORTAR_FP32) *reinterpret_cast<float *>(p) = v;
        else if constexpr (TYPE == MORTAR_FP16) *reinterpret_cast<_Float16 *>(p) = (_Float16)v;
        else *reinterpret_cast<uint16_t *>(p) = (uint16_t)bf16_bits_rne(v);
    }
};

struct RowArgs {
    const char *x;               // rows per token (dispatch: x, combine backward: dy), ldx bytes apart
    const char *ys;              // rows per slot, d values apart
    char *out;                   // dispatch: xs, combine: y, combine backward: dys or null
    char *dw;                    // combine backward: gradients of the weights or null
    const char *w;               // weights [N, k], or null for 1
    const int32_t *position, *full, *token;      // token: of each row, or null
    int64_t ldx, slots;          // slots: N k
    int32_t k, d, w_type;
};

__device__ __forceinline__ float read_weight(const RowArgs &a, int64_t i) {
    if (!a.w) return 1.0f;
    return a.w_type == MORTAR_FP32 ? Row<MORTAR_FP32>::one(a.w + i * 4) : a.w_type == MORTAR_FP16 ? Row<MORTAR_FP16>::one(a.w + i * 2) : Row<MORTAR_BF16>::one(a.w + i * 2);
}

// Whether one of its token's slots names row i.  The loads are on their way while the wave does something else: begin, then named.
struct Named {
    int64_t first;               // slot of the token, below a.slots if there is one
    int32_t position;
    __device__ __forceinline__ void begin(const RowArgs &a, uint32_t i, int lane) {
        first = a.token ? (int64_t)(uint32_t)a.token[i] * a.k : a.slots;
        position = -1;
        if (first < a.slots && lane < a.k) position = a.position[first + lane];
    }
    __device__ __forceinline__ bool named(const RowArgs &a, uint32_t i, int lane) const {
        bool is = __ballot(position == (int)i) != 0;
        if (first < a.slots)
            for (int j = 64; j < a.k; j += 64) is |= __ballot(j + lane < a.k && a.position[first + min(j + lane, a.k - 1)] == (int)i) != 0;
        return is;
    }
};
// Row i as zeros.
template <int SIZE>
__device__ __forceinline__ void clear_row(const RowArgs &a, uint32_t i, int lane) {
    const int bytes = a.d * SIZE, units = bytes / 16, at = units * 16 + lane * SIZE;
    char *dst = a.out + (int64_t)i * bytes;
    for (int u = lane; u < units; u += 64) *reinterpret_cast<u32x4_any_t *>(dst + u * 16) = u32x4_any_t{0, 0, 0, 0};
    if (at >= bytes) return;
    if constexpr (SIZE == 4) *reinterpret_cast<uint32_t *>(dst + at) = 0u;
    else *reinterpret_cast<uint16_t *>(dst + at) = 0;
}

// A wave per slot; the rows of a token are read by neighbouring waves and come out of the caches but once.  Bound by the rows written: 4096 tokens, 8 slots
// of 2048 bf16 values 28 to 29 us (151 MB with the reads, 5.3 TB/s), 16384 tokens, 2 of 768 15 (75 MB, 5.0; 20 between the launches of a backward pass); rows of 1999
// values, on odd addresses, take 1.7 times as long (50 us), small launches of them more (5105 of them 9.1, 2.7 TB/s).
template <int SIZE, bool STREAM>
__global__ __launch_bounds__(256) void expert_dispatch_kernel(const RowArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t i = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (i >= a.slots) return;
    const int row = a.position[i];
    const bool live = row < *a.full;
    Named own;
    own.begin(a, i, lane);
    if ((uint32_t)row < (uint32_t)a.slots) {
        const char *src = a.x + i / (uint32_t)a.k * a.ldx;
        char *dst = a.out + (int64_t)row * a.d * SIZE;
        const int bytes = a.d * SIZE, units = bytes / 16;
        int u = lane;
        for (; u + 192 < units; u += 256) {
            u32x4_t v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = live ? *reinterpret_cast<const u32x4_any_t *>(src + (u + q * 64) * 16) : u32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < 4; ++q) put16<STREAM>(dst + (u + q * 64) * 16, v[q]);
        }
        for (; u < units; u += 64) put16<STREAM>(dst + u * 16, live ? *reinterpret_cast<const u32x4_any_t *>(src + u * 16) : u32x4_any_t{0, 0, 0, 0});
        const int at = units * 16 + lane * SIZE;
        if (at < bytes) {
            if constexpr (SIZE == 4) *reinterpret_cast<uint32_t *>(dst + at) = live ? *reinterpret_cast<const uint32_t *>(src + at) : 0u;
            else *reinterpret_cast<uint16_t *>(dst + at) = live ? *reinterpret_cast<const uint16_t *>(src + at) : (uint16_t)0;
        }
    }
    if (a.token && !own.named(a, i, lane)) clear_row<SIZE>(a, i, lane);
}

// A wave per TOKENS consecutive tokens and 64 units of their rows, the rows of eight slots on their way at a time: with few slots per token one token alone
// leaves too little on the way (two slots of 768 values: 16384 tokens in 20 us, 14 with four tokens).  The wave's lanes hold the positions and weights of its slots.
// Bound by the rows read: 4096 tokens, 8 slots of 2048 bf16 values 34 us (151 MB, 4.5 TB/s), of 1999 45, without weights (the gradient of the dispatch) behind other
// work 46 and 64.
constexpr int NO_WEIGHT = 3;
template <int TYPE, int WTYPE, int TOKENS>
__global__ __launch_bounds__(256) void expert_combine_kernel(const RowArgs a, int parts) {
    using R = Row<TYPE>;
    constexpr int J = 8 / TOKENS;                        // slots of a token at a time
    const int lane = threadIdx.x & 63;
    const uint32_t task = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), group = task / (uint32_t)parts;
    const int64_t first = (int64_t)group * TOKENS * a.k;  // slot
    if (first >= a.slots) return;
    const int unit = (int)(task - group * parts) * 64 + lane, left = a.d - unit * R::UNIT;
    const int64_t pitch = (int64_t)a.d * R::SIZE, in = (int64_t)unit * 16;
    const uint32_t full = min((uint32_t)*a.full, (uint32_t)a.slots);
    const int mine = (int)min((int64_t)(TOKENS * a.k), a.slots - first);
    float sum[TOKENS][R::UNIT];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t)
#pragma unroll
        for (int v = 0; v < R::UNIT; ++v) sum[t][v] = 0.f;
    for (int s0 = 0; s0 < (TOKENS > 1 ? 1 : a.k); s0 += 64) {        // (several tokens: 8 slots in all)
        int position = -1;
        float weight = 1.0f;
        if (s0 + lane < mine) {
            position = a.position[first + s0 + lane];
            if constexpr (WTYPE != NO_WEIGHT) weight = Row<WTYPE>::one(a.w + (first + s0 + lane) * (16 / Row<WTYPE>::UNIT));
        }
        const int slots = TOKENS > 1 ? a.k : min(64, a.k - s0);
        for (int j0 = 0; j0 < slots; j0 += J) {
            u32x4_t v[TOKENS][J];
            uint32_t row[TOKENS][J];
            float w[TOKENS][J];
#pragma unroll
            for (int t = 0; t < TOKENS; ++t)
#pragma unroll
                for (int q = 0; q < J; ++q) {
                    const int from = t * a.k + j0 + q;
                    row[t][q] = j0 + q < slots ? (uint32_t)__builtin_amdgcn_readlane(position, from) : UINT32_MAX;
                    w[t][q] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), from & 63));
                }
            if (left >= R::UNIT) {
#pragma unroll
                for (int t = 0; t < TOKENS; ++t)
#pragma unroll
                    for (int q = 0; q < J; ++q)
                        if (row[t][q] < full) v[t][q] = R::load(a.ys + row[t][q] * pitch + in);
#pragma unroll
                for (int t = 0; t < TOKENS; ++t)
#pragma unroll
                    for (int q = 0; q < J; ++q)
                        if (row[t][q] < full) {
                            float f[R::UNIT];
                            R::unpack(v[t][q], f);
#pragma unroll
                            for (int u = 0; u < R::UNIT; ++u) sum[t][u] = __builtin_fmaf(w[t][q], f[u], sum[t][u]);
                        }
            } else {
#pragma unroll
                for (int t = 0; t < TOKENS; ++t)
                    for (int q = 0; q < J; ++q)
                        if (row[t][q] < full) {
#pragma unroll
                            for (int u = 0; u < R::UNIT; ++u)
                                if (u < left) sum[t][u] = __builtin_fmaf(w[t][q], R::one(a.ys + row[t][q] * pitch + in + u * R::SIZE), sum[t][u]);
                        }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
        if (t * a.k >= mine) break;
        char *dst = a.out + ((int64_t)group * TOKENS + t) * pitch + in;
        if (left >= R::UNIT) {
            R::store(dst, R::pack(sum[t]));
        } else {
#pragma unroll
            for (int u = 0; u < R::UNIT; ++u)
                if (u < left) R::put(dst + u * R::SIZE, sum[t][u]);
        }
    }
}

template <int TYPE, int WTYPE>
int launch_combine(const RowArgs &a, hipStream_t st, const char *what) {
    const int per = 64 * Row<TYPE>::UNIT, parts = (a.d + per - 1) / per, tokens = a.k <= 2 ? 4 : a.k <= 4 ? 2 : 1;
    const int64_t N = a.slots / a.k, groups = ((N + tokens - 1) / tokens * parts + 3) / 4;
    if (groups >= 1 << 24) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many values", what);
    const auto kern = tokens == 4 ? expert_combine_kernel<TYPE, WTYPE, 4> : tokens == 2 ? expert_combine_kernel<TYPE, WTYPE, 2> : expert_combine_kernel<TYPE, WTYPE, 1>;
    hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, st, a, parts);
    return launch_error(what);
}
template <int TYPE>
int launch_combine_weights(const RowArgs &a, hipStream_t st, const char *what) {
    if (!a.w) return launch_combine<TYPE, NO_WEIGHT>(a, st, what);
    return a.w_type == MORTAR_FP32 ? launch_combine<TYPE, MORTAR_FP32>(a, st, what) : a.w_type == MORTAR_FP16 ? launch_combine<TYPE, MORTAR_FP16>(a, st, what) : launch_combine<TYPE, MORTAR_BF16>(a, st, what);
}

// A wave per slot: its row of dys, and the dot product over the row.  Bound by both: 4096 tokens, 8 slots of 2048 bf16 values 54 us (285 MB, 5.3 TB/s), of 1999 66.
template <int TYPE, bool STREAM>
__global__ __launch_bounds__(256) void expert_combine_bwd_kernel(const RowArgs a) {
    using R = Row<TYPE>;
    const int lane = threadIdx.x & 63;
    const uint32_t i = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (i >= a.slots) return;
    const int row = a.position[i];
    const int32_t full = *a.full;
    Named own;
    own.begin(a, i, lane);
    float dot = 0.f;                                       // (a slot whose position is none of the rows: as an empty one)
    if ((uint32_t)row < (uint32_t)a.slots) {
        const bool live = row < full;
        const float w = live ? read_weight(a, i) : 0.f;
        const char *dy = a.x + i / (uint32_t)a.k * a.ldx;
        const int64_t at_row = (int64_t)row * a.d * R::SIZE;
        const int units = a.d / R::UNIT;
        for (int u = lane; u < units; u += 64) {
            float g[R::UNIT], f[R::UNIT];
#pragma unroll
            for (int t = 0; t < R::UNIT; ++t) g[t] = f[t] = 0.f;
            if (live) {
                const u32x4_t gw = R::load(dy + (int64_t)u * 16);
                if (a.dw) R::unpack(R::load(a.ys + at_row + (int64_t)u * 16), f);
                R::unpack(gw, g);
#pragma unroll
                for (int t = 0; t < R::UNIT; ++t) dot = __builtin_fmaf(g[t], f[t], dot);
            }
            if (a.out) {
#pragma unroll
                for (int t = 0; t < R::UNIT; ++t) g[t] = live ? g[t] * w : 0.f;
                put16<STREAM>(a.out + at_row + (int64_t)u * 16, R::pack(g));
            }
        }
        const int last = units * R::UNIT + lane;
        if (last < a.d) {
            const float g = live ? R::one(dy + (int64_t)last * R::SIZE) : 0.f;
            if (live && a.dw) dot = __builtin_fmaf(g, R::one(a.ys + at_row + (int64_t)last * R::SIZE), dot);
            if (a.out) R::put(a.out + at_row + (int64_t)last * R::SIZE, live ? g * w : 0.f);
        }
    }
    if (a.out && a.token && !own.named(a, i, lane)) clear_row<R::SIZE>(a, i, lane);
    if (!a.dw) return;
    dot = mortar_wave_sum(dot);
    if (lane) return;
    if (a.w_type == MORTAR_FP32) Row<MORTAR_FP32>::put(a.dw + i * 4, dot);
    else if (a.w_type == MORTAR_FP16) Row<MORTAR_FP16>::put(a.dw + i * 2, dot);
    else Row<MORTAR_BF16>::put(a.dw + i * 2, dot);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows by slot that the memory-side cache (256 MB) cannot hold for whoever reads them next are stored past it: 268 MB of fp32 dispatched in 63 -> 51 us (54 with the look at the
// rows' slots).
// Smaller ones gain little (134 MB 26.4 -> 25.7) and are read from there; rows on odd addresses lose (35 -> 43).
bool past_caches(const RowArgs &a, int32_t type) {
    const int64_t row = (int64_t)a.d * (type == MORTAR_FP32 ? 4 : 2);
    return a.slots * row > 256 << 20 && row % 16 == 0 && aligned16(a.out);
}

bool known(int32_t type) { return type == MORTAR_BF16 || type == MORTAR_FP16 || type == MORTAR_FP32; }

int check_rows(const char *what, int64_t N, int32_t k, int32_t d, int32_t type) {
    if (N < 0 || k <= 0 || d <= 0 || !known(type)) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape or type", what);
    if (d >= 1 << 28 || N > MOST_SLOTS || N * k > MOST_SLOTS) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many slots or values", what);
    return MORTAR_OK;
}
int check_pointer(const char *what, const char *name, const void *p, int32_t type) {
    if (!p) return mortar_fail(MORTAR_ERR_ARG, "%s: %s is null", what, name);
    return reinterpret_cast<uintptr_t>(p) % (type == MORTAR_FP32 ? 4 : 2) ? mortar_fail(MORTAR_ERR_ARG, "%s: %s is not on an address of its type", what, name) : MORTAR_OK;
}
#define CHECK(...) do { const int rc_ = (__VA_ARGS__); if (rc_) return rc_; } while (0)

}  // namespace

extern "C" int64_t mortar_expert_sort_workspace_bytes(int64_t slots, int32_t n_experts) {
    if (slots <= SORT_ALONE || n_experts <= 0) return 0;
    const int64_t run = SORT_THREADS * held_of(slots);
    return 4 * ((slots + run - 1) / run) * (n_experts + 1);
}

extern "C" int mortar_expert_sort(const void *ids, int32_t ids_64, int64_t N, int32_t k, int32_t n_experts, int32_t *position, int32_t *token, int32_t *offsets,
                                  void *workspace, void *stream) {
    const char *what = "expert_sort";
    CHECK(check_rows(what, N, k, 1, MORTAR_FP32));
    if (n_experts <= 0) return mortar_fail(MORTAR_ERR_ARG, "%s: no experts", what);
    if (n_experts > MOST_EXPERTS) return mortar_fail(MORTAR_ERR_LIMIT, "%s: more than %d experts", what, MOST_EXPERTS);
    const int64_t n = N * k;
    if (!offsets || (n && (!ids || !position || !token)) || (mortar_expert_sort_workspace_bytes(n, n_experts) && !workspace))
        return mortar_fail(MORTAR_ERR_ARG, "%s: a pointer is null", what);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    int32_t *totals = static_cast<int32_t *>(workspace);
    if (ids_64) return sort(Slots<int64_t>{static_cast<const int64_t *>(ids), n, n_experts}, k, position, token, offsets, totals, st, what);
    return sort(Slots<int32_t>{static_cast<const int32_t *>(ids), n, n_experts}, k, position, token, offsets, totals, st, what);
}

extern "C" int mortar_expert_dispatch(const void *x, int64_t N, int32_t d, int64_t ldx, int32_t type, int32_t k, const int32_t *position, const int32_t *full, void *xs,
                                      void *stream) {
    return mortar_expert_dispatch_rows(x, N, d, ldx, type, k, position, full, nullptr, xs, stream);
}

extern "C" int mortar_expert_dispatch_rows(const void *x, int64_t N, int32_t d, int64_t ldx, int32_t type, int32_t k, const int32_t *position, const int32_t *full,
                                           const int32_t *token, void *xs, void *stream) {
    const char *what = "expert_dispatch";
    CHECK(check_rows(what, N, k, d, type));
    if (N == 0) return MORTAR_OK;
    CHECK(check_pointer(what, "x", x, type));
    CHECK(check_pointer(what, "xs", xs, type));
    CHECK(check_pointer(what, "position", position, MORTAR_FP32));
    CHECK(check_pointer(what, "full", full, MORTAR_FP32));
    if (token) CHECK(check_pointer(what, "token", token, MORTAR_FP32));
    RowArgs a{};
    a.x = static_cast<const char *>(x); a.ldx = ldx * (type == MORTAR_FP32 ? 4 : 2);
    a.out = static_cast<char *>(xs); a.position = position; a.full = full; a.token = token;
    a.slots = N * k; a.k = k; a.d = d;
    const dim3 grid((unsigned)((a.slots + 3) / 4));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool past = past_caches(a, type);
    const auto kern = type == MORTAR_FP32 ? (past ? expert_dispatch_kernel<4, true> : expert_dispatch_kernel<4, false>) : (past ? expert_dispatch_kernel<2, true> : expert_dispatch_kernel<2, false>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a);
    return launch_error(what);
}

extern "C" int mortar_expert_combine(const void *ys, int64_t N, int32_t d, int32_t type, int32_t k, const int32_t *position, const int32_t *full, const void *weights,
                                     int32_t w_type, void *y, void *stream) {
    const char *what = "expert_combine";
    CHECK(check_rows(what, N, k, d, type));
    if (N == 0) return MORTAR_OK;
    CHECK(check_pointer(what, "ys", ys, type));
    CHECK(check_pointer(what, "y", y, type));
    CHECK(check_pointer(what, "position", position, MORTAR_FP32));
    CHECK(check_pointer(what, "full", full, MORTAR_FP32));
    if (weights && !known(w_type)) return mortar_fail(MORTAR_ERR_ARG, "%s: bad type of the weights", what);
    if (weights) CHECK(check_pointer(what, "weights", weights, w_type));
    RowArgs a{};
    a.ys = static_cast<const char *>(ys); a.out = static_cast<char *>(y); a.w = static_cast<const char *>(weights); a.w_type = w_type;
    a.position = position; a.full = full; a.slots = N * k; a.k = k; a.d = d;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return type == MORTAR_FP32 ? launch_combine_weights<MORTAR_FP32>(a, st, what) : type == MORTAR_FP16 ? launch_combine_weights<MORTAR_FP16>(a, st, what) : launch_combine_weights<MORTAR_BF16>(a, st, what);
}

extern "C" int mortar_expert_combine_bwd(const void *dy, int64_t lddy, const void *ys, int64_t N, int32_t d, int32_t type, int32_t k, const int32_t *position,
                                         const int32_t *full, const void *weights, int32_t w_type, void *dys, void *dw, void *stream) {
    return mortar_expert_combine_bwd_rows(dy, lddy, ys, N, d, type, k, position, full, nullptr, weights, w_type, dys, dw, stream);
}

extern "C" int mortar_expert_combine_bwd_rows(const void *dy, int64_t lddy, const void *ys, int64_t N, int32_t d, int32_t type, int32_t k, const int32_t *position,
                                              const int32_t *full, const int32_t *token, const void *weights, int32_t w_type, void *dys, void *dw, void *stream) {
    const char *what = "expert_combine_bwd";
    CHECK(check_rows(what, N, k, d, type));
    if (N == 0 || (!dys && !dw)) return MORTAR_OK;
    CHECK(check_pointer(what, "dy", dy, type));
    CHECK(check_pointer(what, "position", position, MORTAR_FP32));
    CHECK(check_pointer(what, "full", full, MORTAR_FP32));
    if (token) CHECK(check_pointer(what, "token", token, MORTAR_FP32));
    if (dys) CHECK(check_pointer(what, "dys", dys, type));
    if ((weights || dw) && !known(w_type)) return mortar_fail(MORTAR_ERR_ARG, "%s: bad type of the weights", what);
    if (weights) CHECK(check_pointer(what, "weights", weights, w_type));
    if (dw) CHECK(check_pointer(what, "dw", dw, w_type));
    if (dw) CHECK(check_pointer(what, "ys", ys, type));
    RowArgs a{};
    a.x = static_cast<const char *>(dy); a.ldx = lddy * (type == MORTAR_FP32 ? 4 : 2);
    a.ys = static_cast<const char *>(ys); a.out = static_cast<char *>(dys); a.dw = static_cast<char *>(dw);
    a.w = static_cast<const char *>(weights); a.w_type = w_type;
    a.position = position; a.full = full; a.token = token; a.slots = N * k; a.k = k; a.d = d;
    const dim3 grid((unsigned)((a.slots + 3) / 4));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool past = past_caches(a, type);
    const auto pick = [&](auto plain, auto streaming) { return past ? streaming : plain; };
    const auto kern = type == MORTAR_FP32   ? pick(expert_combine_bwd_kernel<MORTAR_FP32, false>, expert_combine_bwd_kernel<MORTAR_FP32, true>)
                      : type == MORTAR_FP16 ? pick(expert_combine_bwd_kernel<MORTAR_FP16, false>, expert_combine_bwd_kernel<MORTAR_FP16, true>)
                                            : pick(expert_combine_bwd_kernel<MORTAR_BF16, false>, expert_combine_bwd_kernel<MORTAR_BF16, true>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a);
    return launch_error(what);
}
