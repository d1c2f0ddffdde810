// The norm over the gradients of many tensors and the gradients clipped to it:
//   n = (sum g^2)^(1/2) or max |g|,   c = min(1, max_norm / (n + 1e-6)),   out = g c
// What bounds it is the memory: every gradient is read once for the norm and once more for its product, and the product written.  Squares
// and their sums are 64 bits: the sum of any finite gradients is then finite and right (fp32 squares overflow from 1.8e19 on and vanish
// below 1e-23), and the two conversions and multiply-adds per value are still less than the memory takes.  The product is fp32, rounded once.
//
// A launch takes the table of up to 128 tensors as its argument, so nothing is copied to the device and a captured launch keeps what it needs.  Tensors
// are cut into chunks of 16 KB that no two tensors share, a workgroup takes every n-th chunk and leaves one partial sum in a slot of its own; the
// slots are added in a fixed order, so that a call gives the same bits every time.  Neighbouring workgroups take neighbouring chunks (a run of chunks for each
// instead: 51 -> 55 us for 86 MB).
// Measured, norm and product: 86 MB of gradients 14 + 28 us (6.1 TB/s, the product's reads partly from the caches), 400 MB 194 (6.2 TB/s),
// 2.4 MB two launches of 4; 500 tensors of 10 MB in all 8 launches of 4, which the host takes 90 us to prepare.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <memory>
#include <new>

#include "mortar_device.h"
#include "mortar_internal.h"

namespace {

constexpr int TENSORS = 128;             // of a launch: the table fits a kernel's 4 KB of arguments
constexpr int CHUNK_BYTES = 16384;       // of gradients
constexpr int MOST_WORKGROUPS = 1024;    // 4 per CU: 400 MB in 194 us, with 8 in 194, with 32 in 209
constexpr int MOST_SLOTS = 2048;         // that every workgroup of the clipping adds for itself: of 2200, 284 MB, 149 us that way and 148 with one launch for it

struct Table {
    const void *src[TENSORS];
    void *dst[TENSORS];
    int64_t size[TENSORS];               // values, and << 48 the type of the gradients, and << 52 of the results (a table of bytes would be read by scalar
                                         // loads from addresses whose parts are no multiples of 4, and those lose their lower bits)
    int32_t first[TENSORS + 1];          // chunks in front of each tensor's; all of them behind the last
    int32_t count;
};
static_assert(sizeof(Table) <= 4000, "a kernel's arguments");
constexpr int64_t SIZE_MASK = (INT64_C(1) << 48) - 1;

// Gradients are parts of flat buffers: their addresses need not be multiples of 16.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

template <int TYPE>
struct Values {
    static constexpr int UNIT = TYPE == MORTAR_FP32 ? 4 : 8;       // values of 16 bytes
    static constexpr int SIZE = 16 / UNIT;
    static __device__ __forceinline__ void unpack(u32x4_t w, float (&v)[UNIT]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == MORTAR_FP32) {
                v[j] = __builtin_bit_cast(f32x4_t, w)[j];
            } else if constexpr (TYPE == MORTAR_FP16) {
                const uint32_t d = w[j];
                const f32x2_t f = __builtin_convertvector(__builtin_bit_cast(f16x2_t, d), f32x2_t);
                v[2 * j] = f[0], v[2 * j + 1] = f[1];
            } else {
                v[2 * j] = __builtin_bit_cast(float, w[j] << 16);
                v[2 * j + 1] = __builtin_bit_cast(float, w[j] & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ float one(const void *p, int64_t i) {
        if constexpr (TYPE == MORTAR_FP32) return static_cast<const float *>(p)[i];
        else if constexpr (TYPE == MORTAR_FP16) return (float)static_cast<const _Float16 *>(p)[i];
        else return bf16_to_f32(static_cast<const uint16_t *>(p)[i]);
    }
    static __device__ __forceinline__ u32x4_t load(const void *p, int64_t unit) { return static_cast<const u32x4_any_t *>(p)[unit]; }
    // A unit of values in this type.
    static __device__ __forceinline__ u32x4_t pack(const float (&v)[UNIT]) {
        if constexpr (TYPE == MORTAR_FP32) {
            return __builtin_bit_cast(u32x4_t, f32x4_t{v[0], v[1], v[2], v[3]});
        } else {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (TYPE == MORTAR_FP16) w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * j], v[2 * j + 1]}, f16x2_t));
                else w[j] = bf16_pack2(v[2 * j], v[2 * j + 1]);
            }
            return w;
        }
    }
    static __device__ __forceinline__ void put(void *p, int64_t i, float v) {
        if constexpr (TYPE == MORTAR_FP32) static_cast<float *>(p)[i] = v;
        else if constexpr (TYPE == MORTAR_FP16) static_cast<_Float16 *>(p)[i] = (_Float16)v;
        else static_cast<uint16_t *>(p)[i] = (uint16_t)bf16_bits_rne(v);
    }
};

// The chunks of a workgroup, every gridDim.x-th one, from the last to the first with `back`: f(tensor, its types, first value, values).  All of it is the same for all
// lanes.  A lane keeps two of the table's counts, and a chunk's tensor is found with two ballots (reading the table from its front took the
// 500 odd tensors of a call 3 us a launch).
template <typename F>
__device__ __forceinline__ void each_chunk(const Table &t, bool back, F f) {
    const int all = t.first[TENSORS], lane = threadIdx.x & 63;
    const int f0 = t.first[lane + 1], f1 = t.first[lane + 65];
    for (int k = blockIdx.x; k < all; k += gridDim.x) {
        const int c = back ? all - 1 - k : k;
        const int i = __popcll(__ballot(f0 <= c)) + __popcll(__ballot(f1 <= c));
        const int64_t size = t.size[i];
        const int types = (int)(size >> 48);
        const int64_t per = CHUNK_BYTES / ((types & 15) == MORTAR_FP32 ? 4 : 2), at = (c - t.first[i]) * per, left = (size & SIZE_MASK) - at;
        f(i, types, at, (int)(left < per ? left : per));
    }
}

// ---- norm ------------------------------------------------------------------------------------------------------------
// A slot is 8 bytes: the sum of squares in 64 bits, or the bits of the largest |g| (as an integer, so that NaN is the largest).

struct Square {
    double s = 0.0;
    __device__ __forceinline__ void take(float v) { s = __builtin_fma((double)v, (double)v, s); }
    __device__ __forceinline__ void join(uint64_t other) { s += __builtin_bit_cast(double, other); }
    __device__ __forceinline__ uint64_t bits() const { return __builtin_bit_cast(uint64_t, s); }
    __device__ __forceinline__ void wave() { s = mortar_wave_sum(s); }
    __device__ __forceinline__ double norm() const { return __builtin_sqrt(s); }
};
struct Largest {
    uint32_t m = 0;
    __device__ __forceinline__ void take(float v) { m = max(m, __builtin_bit_cast(uint32_t, v) & 0x7fffffffu); }
    __device__ __forceinline__ void join(uint64_t other) { m = max(m, (uint32_t)other); }
    __device__ __forceinline__ uint64_t bits() const { return m; }
    __device__ __forceinline__ void wave() { m = mortar_wave_reduce(m, [](uint32_t a, uint32_t b) { return max(a, b); }); }
    __device__ __forceinline__ double norm() const { return (double)__builtin_bit_cast(float, m); }
};

// Of the 256 threads; thread 0 has it.
template <typename R>
__device__ __forceinline__ void join_workgroup(R &r) {
    __shared__ uint64_t part[4];
    r.wave();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r.bits();
    __syncthreads();
    if (threadIdx.x == 0) {
        r = R{};
        for (int w = 0; w < 4; ++w) r.join(part[w]);
    }
}

template <typename R, int TYPE>
__device__ __forceinline__ void take_chunk(R (&r)[2], const void *base, int64_t at, int n) {
    using V = Values<TYPE>;
    const char *p = static_cast<const char *>(base) + at * V::SIZE;
    const int units = n / V::UNIT;
    if (n == CHUNK_BYTES / V::SIZE) {
        u32x4_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = V::load(p, k * 256 + threadIdx.x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[V::UNIT];
            V::unpack(w[k], v);
#pragma unroll
            for (int j = 0; j < V::UNIT; ++j) r[j & 1].take(v[j]);
        }
    } else {
        for (int u = threadIdx.x; u < units; u += 256) {
            float v[V::UNIT];
            V::unpack(V::load(p, u), v);
#pragma unroll
            for (int j = 0; j < V::UNIT; ++j) r[j & 1].take(v[j]);
        }
        const int i = units * V::UNIT + threadIdx.x;
        if (i < n) r[0].take(V::one(p, i));
    }
}

template <typename R>
__global__ __launch_bounds__(256) void grad_norm_kernel(const Table t, uint64_t *slots) {
    R r[2];
    each_chunk(t, false, [&](int i, int types, int64_t at, int n) {
        const int type = types & 15;
        if (type == MORTAR_BF16) take_chunk<R, MORTAR_BF16>(r, t.src[i], at, n);
        else if (type == MORTAR_FP16) take_chunk<R, MORTAR_FP16>(r, t.src[i], at, n);
        else take_chunk<R, MORTAR_FP32>(r, t.src[i], at, n);
    });
    r[0].join(r[1].bits());
    join_workgroup(r[0]);
    if (threadIdx.x == 0) slots[blockIdx.x] = r[0].bits();
}

// All slots by one workgroup: the norm.
template <typename R>
__device__ __forceinline__ double join_slots(const uint64_t *slots, int count) {
    __shared__ double norm;
    R r;
    for (int i = threadIdx.x; i < count; i += 256) r.join(slots[i]);
    join_workgroup(r);
    if (threadIdx.x == 0) norm = r.norm();
    __syncthreads();
    return norm;
}
// The norm, and (not null) the slot that all of them make.
template <typename R>
__global__ __launch_bounds__(256) void grad_join_kernel(const uint64_t *slots, int count, float *norm_out, uint64_t *joined) {
    R r;
    for (int i = threadIdx.x; i < count; i += 256) r.join(slots[i]);
    join_workgroup(r);
    if (threadIdx.x) return;
    if (norm_out) *norm_out = (float)r.norm();
    if (joined) *joined = r.bits();
}

// ---- clipping --------------------------------------------------------------------------------------------------------

template <int TYPE, int OUT, bool STREAM>
__device__ __forceinline__ void scale_chunk(const void *base, void *out, int64_t at, int n, float c) {
    using V = Values<TYPE>;
    using O = Values<OUT>;
    const char *p = static_cast<const char *>(base) + at * V::SIZE;
    char *q = static_cast<char *>(out) + at * O::SIZE;
    const int units = n / V::UNIT;
    const auto store = [&](int u, u32x4_t w) {
        float v[V::UNIT];
        V::unpack(w, v);
#pragma unroll
        for (int k = 0; k < V::UNIT / O::UNIT; ++k) {
            float f[O::UNIT];
#pragma unroll
            for (int j = 0; j < O::UNIT; ++j) f[j] = v[k * O::UNIT + j] * c;
            u32x4_any_t *to = reinterpret_cast<u32x4_any_t *>(q) + u * (V::UNIT / O::UNIT) + k;
            if constexpr (STREAM) __builtin_nontemporal_store((u32x4_any_t)O::pack(f), to);
            else *to = O::pack(f);
        }
    };
    if (n == CHUNK_BYTES / V::SIZE) {
        u32x4_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = V::load(p, k * 256 + threadIdx.x);
#pragma unroll
        for (int k = 0; k < 4; ++k) store(k * 256 + threadIdx.x, w[k]);
    } else {
        for (int u = threadIdx.x; u < units; u += 256) store(u, V::load(p, u));
        const int i = units * V::UNIT + threadIdx.x;
        if (i < n) O::put(q, i, V::one(p, i) * c);
    }
}

// Every workgroup adds the slots for itself: a launch less than with a kernel that does it once.  The chunks are taken in the opposite order, those
// first that the norm read last and the caches still hold.  STREAM: results that the L2s cannot hold go past the caches, which keep the gradients then
// (86 MB 51 -> 40 us with the norm; 400 MB 227 -> 194, all of that by the order).
template <typename R, bool STREAM>
__global__ __launch_bounds__(256) void grad_clip_kernel(const Table t, const uint64_t *slots, int count, double max_norm, float *norm_out) {
    const double n = join_slots<R>(slots, count);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)n;
    double ratio = max_norm / (n + 1e-6);
    if (ratio > 1.0) ratio = 1.0;                        // (NaN stays)
    const float c = (float)ratio;
    each_chunk(t, true, [&](int i, int types, int64_t at, int n) {
        if (c == 1.0f && t.dst[i] == t.src[i]) return;   // in place, and nothing changes
        switch (types) {
            case MORTAR_BF16 | MORTAR_BF16 << 4: scale_chunk<MORTAR_BF16, MORTAR_BF16, STREAM>(t.src[i], t.dst[i], at, n, c); break;
            case MORTAR_FP16 | MORTAR_FP16 << 4: scale_chunk<MORTAR_FP16, MORTAR_FP16, STREAM>(t.src[i], t.dst[i], at, n, c); break;
            case MORTAR_BF16 | MORTAR_FP32 << 4: scale_chunk<MORTAR_BF16, MORTAR_FP32, STREAM>(t.src[i], t.dst[i], at, n, c); break;
            case MORTAR_FP16 | MORTAR_FP32 << 4: scale_chunk<MORTAR_FP16, MORTAR_FP32, STREAM>(t.src[i], t.dst[i], at, n, c); break;
            default: scale_chunk<MORTAR_FP32, MORTAR_FP32, STREAM>(t.src[i], t.dst[i], at, n, c);
        }
    });
}

// ---- host side -------------------------------------------------------------------------------------------------------

int launch_error(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int size_of(int32_t type) { return type == MORTAR_FP32 ? 4 : 2; }

int check(const char *what, const mortar_grad_t *g, int64_t count, bool clip) {
    if (count < 0 || (count && !g)) return mortar_fail(MORTAR_ERR_ARG, "%s: bad list", what);
    for (int64_t i = 0; i < count; ++i) {
        const auto bad = [&](int32_t t) { return t != MORTAR_BF16 && t != MORTAR_FP16 && t != MORTAR_FP32; };
        if (g[i].n < 0 || bad(g[i].type)) return mortar_fail(MORTAR_ERR_ARG, "%s: tensor %lld: bad size or type", what, (long long)i);
        if (g[i].n >= INT64_C(1) << 40) return mortar_fail(MORTAR_ERR_LIMIT, "%s: tensor %lld is too large", what, (long long)i);
        if (g[i].n && (!g[i].src || reinterpret_cast<uintptr_t>(g[i].src) % size_of(g[i].type)))
            return mortar_fail(MORTAR_ERR_ARG, "%s: tensor %lld is null or not on an address of its type", what, (long long)i);
        if (!clip) continue;
        if (bad(g[i].out_type) || (g[i].out_type != g[i].type && g[i].out_type != MORTAR_FP32))
            return mortar_fail(MORTAR_ERR_ARG, "%s: tensor %lld: the result has its type or fp32", what, (long long)i);
        if (g[i].n && (!g[i].dst || reinterpret_cast<uintptr_t>(g[i].dst) % size_of(g[i].out_type)))
            return mortar_fail(MORTAR_ERR_ARG, "%s: result %lld is null or not on an address of its type", what, (long long)i);
    }
    return MORTAR_OK;
}

// The next launch's table from tensor `at` on: returns the tensor behind it.
int64_t fill(Table &t, const mortar_grad_t *g, int64_t count, int64_t at) {
    t.count = 0;
    t.first[0] = 0;
    for (; at < count && t.count < TENSORS; ++at) {
        if (!g[at].n) continue;
        const int64_t chunks = (g[at].n * size_of(g[at].type) + CHUNK_BYTES - 1) / CHUNK_BYTES;
        if (t.first[t.count] + chunks > INT32_MAX) break;            // (one tensor alone has 2^28 at most)
        const int i = t.count++;
        t.src[i] = g[at].src;
        t.dst[i] = g[at].dst;
        t.size[i] = g[at].n | (int64_t)(g[at].type | (g[at].out_type & 15) << 4) << 48;
        t.first[i + 1] = t.first[i] + (int32_t)chunks;
    }
    std::fill(t.first + t.count + 1, t.first + TENSORS + 1, t.first[t.count]);
    return at;
}
int workgroups(const Table &t) { return std::min(t.first[t.count], MOST_WORKGROUPS); }

// Slots of all launches of the norm, and (not null) how many launches.
int64_t slots_of(const mortar_grad_t *g, int64_t count, int64_t *launches = nullptr) {
    Table t;
    int64_t all = 0, n = 0;
    for (int64_t at = 0; at < count; ++n) {
        at = fill(t, g, count, at);
        all += workgroups(t);
    }
    if (launches) *launches = n;
    return all;
}

template <typename R>
int run(const mortar_grad_t *g, int64_t count, bool clip, double max_norm, float *norm, uint64_t *slots, hipStream_t st, const char *what) {
    Table t;
    int64_t used = 0, bytes = 0, launches = 0;
    if (slots_of(g, count, &launches) >= INT32_MAX) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many tensors", what);
    const std::unique_ptr<int64_t[]> starts(new (std::nothrow) int64_t[launches + 1]);        // first tensor of each launch
    if (!starts) return mortar_fail(MORTAR_ERR_LIMIT, "%s: no memory for the list of launches", what);
    for (int64_t at = 0, k = 0; at < count;) {
        starts[k++] = at;
        at = fill(t, g, count, at);
        if (!t.count) continue;
        hipLaunchKernelGGL(grad_norm_kernel<R>, dim3(workgroups(t)), dim3(256), 0, st, t, slots + used);
        used += workgroups(t);
        if (const int rc = launch_error(what)) return rc;
    }
    if (!clip || !used || used > MOST_SLOTS) {
        uint64_t *joined = clip && used ? slots + used : nullptr;
        hipLaunchKernelGGL(grad_join_kernel<R>, dim3(1), dim3(256), 0, st, slots, (int)used, norm, joined);
        if (const int rc = launch_error(what)) return rc;
        if (!joined) return MORTAR_OK;
        slots = joined, used = 1, norm = nullptr;
    }
    for (int64_t i = 0; i < count; ++i) bytes += g[i].n * size_of(g[i].out_type);
    const auto kern = bytes > 32 << 20 ? grad_clip_kernel<R, true> : grad_clip_kernel<R, false>;
    for (int64_t k = launches; k-- > 0;) {
        fill(t, g, count, starts[k]);
        if (!t.count) continue;
        hipLaunchKernelGGL(kern, dim3(workgroups(t)), dim3(256), 0, st, t, slots, (int)used, max_norm, norm);
        norm = nullptr;
        if (const int rc = launch_error(what)) return rc;
    }
    return MORTAR_OK;
}

int grad(const mortar_grad_t *g, int64_t count, bool clip, int32_t largest, double max_norm, float *norm, void *workspace, void *stream, const char *what) {
    if (const int rc = check(what, g, count, clip)) return rc;
    if (!norm || (slots_of(g, count) && !workspace)) return mortar_fail(MORTAR_ERR_ARG, "%s: norm or workspace is null", what);
    if (clip && !(max_norm >= 0)) return mortar_fail(MORTAR_ERR_ARG, "%s: max_norm is negative or NaN", what);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    uint64_t *slots = static_cast<uint64_t *>(workspace);
    return largest ? run<Largest>(g, count, clip, max_norm, norm, slots, st, what) : run<Square>(g, count, clip, max_norm, norm, slots, st, what);
}

}  // namespace

extern "C" int64_t mortar_grad_workspace_bytes(const mortar_grad_t *grads, int64_t count) {
    if (const int rc = check("grad_workspace", grads, count, false)) return rc;
    return 8 * (slots_of(grads, count) + 1);
}
extern "C" int mortar_grad_norm(const mortar_grad_t *grads, int64_t count, int32_t largest, float *norm, void *workspace, void *stream) {
    return grad(grads, count, false, largest, 0.0, norm, workspace, stream, "grad_norm");
}
extern "C" int mortar_grad_clip(const mortar_grad_t *grads, int64_t count, int32_t largest, double max_norm, float *norm, void *workspace, void *stream) {
    return grad(grads, count, true, largest, max_norm, norm, workspace, stream, "grad_clip");
}
