// LayerNorm over the last dimension with its gradients.
//   y  = (x - mu) r w + b,  mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = r (g - mean(g) - z mean(g z)),  z = (x - mu) r,  g = dy w
//   dw = sum over rows of dy z,  db = sum over rows of dy
// All of it in fp32 on the values as loaded (the variance from the centred values in registers, no E[x^2] - mu^2), results rounded
// once.  Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx; a row stays in registers between its sums
// and its result.  A row belongs to one wavefront (up to 4 KB, or 512 single values) or to the four of a workgroup; workgroups walk over rows, w
// and b in registers, and the backward adds dw and db of its rows there: one fp32 slab per workgroup, added in order by a second
// kernel, so that results do not depend on timing.
// Measured, forward / backward / join of the slabs: 16384 x 2048 bf16 23 / 35 / 4 us (134 and 201 MB: 5.8 TB/s, where a large copy reaches
// 5.0), 16384 x 768 fp32 17 / 25 / 4, 1021 x 1999 fp16 (no row is aligned: single values) 6 / 10 / 4.  The next row is loaded before the
// sums of the present one (without that the backward of the first took 43), the weights behind the first row and all at once (one by
// one its forward took 26), the slabs by 32 threads per column (9).
#include <hip/hip_runtime.h>

#include "mortar_dense_core.h"
#include "mortar_internal.h"

namespace {

enum { LN_BF16, LN_F16, LN_F32 };

template <int T>
struct Elem {
    using type = uint16_t;
};
template <>
struct Elem<LN_F32> {
    using type = float;
};
template <int T>
__device__ __forceinline__ float to_float(typename Elem<T>::type v) {
    if constexpr (T == LN_F32) return v;
    else if constexpr (T == LN_F16) return (float)__builtin_bit_cast(_Float16, v);
    else return bf16_to_f32(v);
}
template <int T>
__device__ __forceinline__ typename Elem<T>::type from_float(float v) {
    if constexpr (T == LN_F32) return v;
    else if constexpr (T == LN_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    else return (uint16_t)bf16_bits_rne(v);
}
// VEC consecutive values as they lie in memory: 16 bytes or one value.
template <int T, int VEC>
struct Raw {
    u32x4_t w;
    __device__ __forceinline__ void read(const typename Elem<T>::type *p) { w = *reinterpret_cast<const u32x4_t *>(p); }
    __device__ __forceinline__ void clear() { w = u32x4_t{0, 0, 0, 0}; }
    __device__ __forceinline__ void values(float (&v)[VEC]) const {
        if constexpr (T == LN_F32) {
            const f32x4_t f = __builtin_bit_cast(f32x4_t, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = f[j];
        } else {
            dense_unpack8<T == LN_F16 ? DENSE_F16 : DENSE_BF16>(w, v);
        }
    }
};
template <int T>
struct Raw<T, 1> {
    typename Elem<T>::type e;
    __device__ __forceinline__ void read(const typename Elem<T>::type *p) { e = *p; }
    __device__ __forceinline__ void clear() { e = 0; }
    __device__ __forceinline__ void values(float (&v)[1]) const { v[0] = to_float<T>(e); }
};
template <>
struct Raw<LN_F32, 8> {                           // fp32 weights beside eight 16-bit values
    Raw<LN_F32, 4> a, b;
    __device__ __forceinline__ void read(const float *p) { a.read(p), b.read(p + 4); }
    __device__ __forceinline__ void clear() { a.clear(), b.clear(); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        float lo[4], hi[4];
        a.values(lo), b.values(hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lo[j], v[j + 4] = hi[j];
    }
};
template <int T, int VEC>
__device__ __forceinline__ void store(typename Elem<T>::type *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        *p = from_float<T>(v[0]);
    } else if constexpr (T == LN_F32) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) *reinterpret_cast<f32x4_t *>(p + i) = f32x4_t{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
        static_assert(VEC == 8, "16 bytes");
        *reinterpret_cast<u32x4_t *>(p) = dense_pack8<T == LN_F16 ? DENSE_F16 : DENSE_BF16>(v);
    }
}

struct LnArgs {
    const void *x, *dy, *w, *b;
    void *y;                      // y, or dx (null: not wanted)
    float *mean, *rstd;           // forward: may be null
    float *slabs;                 // backward: [workgroups][2][d], null: no dw, db
    int64_t M, ldx, lddy, ldy;
    int32_t d;
    float eps;
};

// Sum over the TPR threads of a row (a wavefront, or the workgroup of four; `turn` alternates so that one barrier suffices).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (&sm)[2][4], int &turn) {
    v = mortar_wave_sum(v);
    if constexpr (TPR > 64) {
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) sm[turn][threadIdx.x >> 6] = v;
        __syncthreads();
        v = (sm[turn][0] + sm[turn][1]) + (sm[turn][2] + sm[turn][3]);
    }
    return v;
}

template <int T, int WT, int VEC, int PER, int TPR>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const LnArgs a) {
    using E = typename Elem<T>::type;
    using W = typename Elem<WT>::type;
    __shared__ float sm[2][4];
    int turn = 0;
    const int t = threadIdx.x % TPR, d = a.d;
    constexpr int RPW = 256 / TPR;
    const float inv_d = 1.0f / (float)d;
    Raw<T, VEC> raw[PER];                         // the row after the one that is worked on is on its way
    const auto fetch = [&](int64_t m) {
        const E *x = static_cast<const E *>(a.x) + m * a.ldx;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * TPR + t) * VEC;
            raw[i].clear();
            if (c < d) raw[i].read(x + c);
        }
    };
    const int64_t first = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR, step = (int64_t)gridDim.x * RPW;
    if (first < a.M) fetch(first);
    float w[PER][VEC], b[PER][VEC];
    {
        Raw<WT, VEC> rw[PER], rb[PER];            // all of them on their way at once
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * TPR + t) * VEC;
            rw[i].clear(), rb[i].clear();
            if (c < d && a.w) rw[i].read(static_cast<const W *>(a.w) + c);
            if (c < d && a.b) rb[i].read(static_cast<const W *>(a.b) + c);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            rw[i].values(w[i]), rb[i].values(b[i]);
            if (!a.w)
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[i][j] = 1.f;
        }
    }
    for (int64_t m = first; m < a.M; m += step) {
        float v[PER][VEC], s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) raw[i].values(v[i]);
        if (m + step < a.M) fetch(m + step);
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += v[i][j];
        const float mu = row_sum<TPR>(s, sm, turn) * inv_d;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool in = (i * TPR + t) * VEC < d;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] = in ? v[i][j] - mu : 0.f;
                s = __builtin_fmaf(v[i][j], v[i][j], s);
            }
        }
        const float r = 1.0f / sqrtf(row_sum<TPR>(s, sm, turn) * inv_d + a.eps);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * TPR + t) * VEC;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = __builtin_fmaf(v[i][j] * r, w[i][j], b[i][j]);
            if (c < d) store<T, VEC>(static_cast<E *>(a.y) + m * a.ldy + c, o);
        }
        if (t == 0 && a.mean) a.mean[m] = mu, a.rstd[m] = r;
    }
}

template <int T, int WT, int VEC, int PER, int TPR, bool PARAMS>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const LnArgs a) {
    using E = typename Elem<T>::type;
    using W = typename Elem<WT>::type;
    __shared__ float sm[2][2][4];
    int turn = 0, turn2 = 0;
    const int t = threadIdx.x % TPR, d = a.d;
    constexpr int RPW = 256 / TPR;
    const float inv_d = 1.0f / (float)d;
    Raw<T, VEC> rx[PER], rdy[PER];                // the row after the one that is worked on is on its way
    float mu_next = 0.f, r_next = 0.f;
    const auto fetch = [&](int64_t m) {
        const E *x = static_cast<const E *>(a.x) + m * a.ldx, *dy = static_cast<const E *>(a.dy) + m * a.lddy;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * TPR + t) * VEC;
            rx[i].clear(), rdy[i].clear();
            if (c < d) rx[i].read(x + c), rdy[i].read(dy + c);
        }
        mu_next = a.mean[m], r_next = a.rstd[m];
    };
    const int64_t first = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR, step = (int64_t)gridDim.x * RPW;
    if (first < a.M) fetch(first);
    float w[PER][VEC], dw[PARAMS ? PER : 1][VEC], db[PARAMS ? PER : 1][VEC];
    {
        Raw<WT, VEC> rw[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * TPR + t) * VEC;
            rw[i].clear();
            if (c < d && a.w) rw[i].read(static_cast<const W *>(a.w) + c);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            rw[i].values(w[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (!a.w) w[i][j] = 1.f;
                if constexpr (PARAMS) dw[i][j] = 0.f, db[i][j] = 0.f;
            }
        }
    }
    for (int64_t m = first; m < a.M; m += step) {
        float z[PER][VEC], g[PER][VEC];
#pragma unroll
        for (int i = 0; i < PER; ++i) rx[i].values(z[i]), rdy[i].values(g[i]);
        const float mu = mu_next, r = r_next;
        if (m + step < a.M) fetch(m + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float mean = (i * TPR + t) * VEC < d ? mu : 0.f;        // beyond the row z = 0, also where mu r is not finite
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                z[i][j] = (z[i][j] - mean) * r;
                if constexpr (PARAMS) {
                    dw[i][j] = __builtin_fmaf(g[i][j], z[i][j], dw[i][j]);
                    db[i][j] += g[i][j];
                }
                g[i][j] *= w[i][j];
                s1 += g[i][j];
                s2 = __builtin_fmaf(g[i][j], z[i][j], s2);
            }
        }
        if (!a.y) continue;
        s1 = row_sum<TPR>(s1, sm[0], turn) * inv_d;
        s2 = row_sum<TPR>(s2, sm[1], turn2) * inv_d;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (i * TPR + t) * VEC;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = r * (g[i][j] - s1 - z[i][j] * s2);
            if (c < d) store<T, VEC>(static_cast<E *>(a.y) + m * a.ldy + c, o);
        }
    }
    if constexpr (PARAMS) {
        float *out = a.slabs + (int64_t)blockIdx.x * 2 * d;
        if constexpr (TPR == 64) {            // the rows of the four waves: added through LDS in their order
            __shared__ float part[4][64 * VEC];
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < VEC; ++j) part[threadIdx.x >> 6][t * VEC + j] = p ? db[i][j] : dw[i][j];
                    __syncthreads();
                    for (int q = threadIdx.x; q < 64 * VEC; q += 256) {
                        const int c = i * 64 * VEC + q;
                        if (c < d) out[p * d + c] = (part[0][q] + part[1][q]) + (part[2][q] + part[3][q]);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int c = (i * TPR + t) * VEC + j;
                    if (c < d) out[c] = dw[i][j], out[d + c] = db[i][j];
                }
        }
    }
}

// Rows too long for registers: a workgroup per row that reads it again for every sum (from L2), and column sums on their own.
template <int T, int WT>
__global__ __launch_bounds__(256) void ln_fwd_long_kernel(const LnArgs a) {
    using E = typename Elem<T>::type;
    using W = typename Elem<WT>::type;
    __shared__ float sm[2][4];
    int turn = 0;
    const int64_t m = blockIdx.x;
    const E *x = static_cast<const E *>(a.x) + m * a.ldx;
    const float inv_d = 1.0f / (float)a.d;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.d; c += 256) s += to_float<T>(x[c]);
    const float mu = row_sum<256>(s, sm, turn) * inv_d;
    s = 0.f;
    for (int c = threadIdx.x; c < a.d; c += 256) {
        const float v = to_float<T>(x[c]) - mu;
        s = __builtin_fmaf(v, v, s);
    }
    const float r = 1.0f / sqrtf(row_sum<256>(s, sm, turn) * inv_d + a.eps);
    for (int c = threadIdx.x; c < a.d; c += 256) {
        const float w = a.w ? to_float<WT>(static_cast<const W *>(a.w)[c]) : 1.f, b = a.b ? to_float<WT>(static_cast<const W *>(a.b)[c]) : 0.f;
        static_cast<E *>(a.y)[m * a.ldy + c] = from_float<T>(__builtin_fmaf((to_float<T>(x[c]) - mu) * r, w, b));
    }
    if (threadIdx.x == 0 && a.mean) a.mean[m] = mu, a.rstd[m] = r;
}
template <int T, int WT>
__global__ __launch_bounds__(256) void ln_dx_long_kernel(const LnArgs a) {
    using E = typename Elem<T>::type;
    using W = typename Elem<WT>::type;
    __shared__ float sm[2][4];
    int turn = 0;
    const int64_t m = blockIdx.x;
    const E *x = static_cast<const E *>(a.x) + m * a.ldx, *dy = static_cast<const E *>(a.dy) + m * a.lddy;
    const float inv_d = 1.0f / (float)a.d, mu = a.mean[m], r = a.rstd[m];
    const auto grad = [&](int c) { return to_float<T>(dy[c]) * (a.w ? to_float<WT>(static_cast<const W *>(a.w)[c]) : 1.f); };
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.d; c += 256) {
        const float g = grad(c);
        s1 += g;
        s2 = __builtin_fmaf(g, (to_float<T>(x[c]) - mu) * r, s2);
    }
    s1 = row_sum<256>(s1, sm, turn) * inv_d;
    s2 = row_sum<256>(s2, sm, turn) * inv_d;
    for (int c = threadIdx.x; c < a.d; c += 256)
        static_cast<E *>(a.y)[m * a.ldy + c] = from_float<T>(r * (grad(c) - s1 - (to_float<T>(x[c]) - mu) * r * s2));
}
template <int T>
__global__ __launch_bounds__(256) void ln_columns_long_kernel(const LnArgs a, int groups) {
    using E = typename Elem<T>::type;
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.d) return;
    float dw = 0.f, db = 0.f;
    for (int64_t m = blockIdx.y; m < a.M; m += groups) {
        const float g = to_float<T>(static_cast<const E *>(a.dy)[m * a.lddy + c]);
        dw = __builtin_fmaf(g, (to_float<T>(static_cast<const E *>(a.x)[m * a.ldx + c]) - a.mean[m]) * a.rstd[m], dw);
        db += g;
    }
    float *out = a.slabs + (int64_t)blockIdx.y * 2 * a.d;
    out[c] = dw;
    out[a.d + c] = db;
}

// dw, db from the slabs: 32 columns per workgroup, 32 runs of slabs side by side, added in a fixed order.
template <int WT>
__global__ __launch_bounds__(1024) void ln_join_kernel(const float *slabs, int n, int d, void *dw, void *db) {
    using W = typename Elem<WT>::type;
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const float *p = slabs + (int64_t)blockIdx.y * d + min(c, d - 1);
    float s = 0.f;
    for (int i = run; i < n; i += 32 * 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = p[(int64_t)min(i + k * 32, n - 1) * 2 * d];
#pragma unroll
        for (int k = 0; k < 8; ++k) s += i + k * 32 < n ? v[k] : 0.f;
    }
    part[run][lane] = s;
    __syncthreads();
    if (run || c >= d) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) s += part[i][lane];
    W *out = static_cast<W *>(blockIdx.y ? db : dw);
    if (out) out[c] = from_float<WT>(s);
}

// ---- launches --------------------------------------------------------------------------------------------------------

// Threads per row and vectors per thread for rows of d values, vec of them at a time; 0: too long for registers.
struct Form {
    int vec, tpr, per;
};
Form form_of(int32_t d, int type, bool vectors) {
    const int vec = vectors ? (type == LN_F32 ? 4 : 8) : 1;
    const int units = (d + vec - 1) / vec, one = vectors ? 4 : 8, most = vectors ? 8 : 32;
    if (units <= 64 * one) {
        int per = one;
        while (per > 1 && units <= 64 * (per / 2)) per /= 2;
        return Form{vec, 64, per};
    }
    for (int per = 2; per <= most; per *= 2)
        if (units <= 256 * per) return Form{vec, 256, per};
    return Form{vec, 0, 0};
}

constexpr int MAX_SLABS = 512;
int64_t slabs_of(int64_t M) {
    const int64_t n = (M + 3) / 4;
    return n < MAX_SLABS ? n : MAX_SLABS;
}

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int T, int WT, int VEC, int PER, int TPR>
void launch_rows(const LnArgs &a, bool bwd, hipStream_t st) {
    const int64_t rows = 256 / TPR, all = (a.M + rows - 1) / rows;
    if (!bwd) {
        hipLaunchKernelGGL((ln_fwd_kernel<T, WT, VEC, PER, TPR>), dim3((unsigned)(all < 2048 ? all : 2048)), dim3(256), 0, st, a);
    } else if (a.slabs) {
        hipLaunchKernelGGL((ln_bwd_kernel<T, WT, VEC, PER, TPR, true>), dim3((unsigned)slabs_of(a.M)), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((ln_bwd_kernel<T, WT, VEC, PER, TPR, false>), dim3((unsigned)(all < 2048 ? all : 2048)), dim3(256), 0, st, a);
    }
}

template <int T, int WT>
void launch_norm(const LnArgs &a, bool bwd, bool vectors, hipStream_t st) {
    constexpr int V = T == LN_F32 ? 4 : 8;
    const Form f = form_of(a.d, T, vectors);
    if (!f.tpr) {
        const int64_t n = slabs_of(a.M);
        if (!bwd) hipLaunchKernelGGL((ln_fwd_long_kernel<T, WT>), dim3((unsigned)a.M), dim3(256), 0, st, a);
        if (bwd && a.y) hipLaunchKernelGGL((ln_dx_long_kernel<T, WT>), dim3((unsigned)a.M), dim3(256), 0, st, a);
        if (bwd && a.slabs) hipLaunchKernelGGL((ln_columns_long_kernel<T>), dim3((unsigned)((a.d + 255) / 256), (unsigned)n), dim3(256), 0, st, a, (int)n);
    } else if (vectors && f.tpr == 64) {
        if (f.per == 1) launch_rows<T, WT, V, 1, 64>(a, bwd, st);
        else if (f.per == 2) launch_rows<T, WT, V, 2, 64>(a, bwd, st);
        else launch_rows<T, WT, V, 4, 64>(a, bwd, st);
    } else if (vectors) {
        if (f.per == 2) launch_rows<T, WT, V, 2, 256>(a, bwd, st);
        else if (f.per == 4) launch_rows<T, WT, V, 4, 256>(a, bwd, st);
        else launch_rows<T, WT, V, 8, 256>(a, bwd, st);
    } else if (f.tpr == 64) {
        if (f.per == 1) launch_rows<T, WT, 1, 1, 64>(a, bwd, st);
        else if (f.per == 2) launch_rows<T, WT, 1, 2, 64>(a, bwd, st);
        else if (f.per == 4) launch_rows<T, WT, 1, 4, 64>(a, bwd, st);
        else launch_rows<T, WT, 1, 8, 64>(a, bwd, st);
    } else {
        if (f.per <= 4) launch_rows<T, WT, 1, 4, 256>(a, bwd, st);
        else if (f.per == 8) launch_rows<T, WT, 1, 8, 256>(a, bwd, st);
        else if (f.per == 16) launch_rows<T, WT, 1, 16, 256>(a, bwd, st);
        else launch_rows<T, WT, 1, 32, 256>(a, bwd, st);
    }
}

void launch_typed(const LnArgs &a, int type, int w_fp32, bool bwd, bool vectors, hipStream_t st) {
    if (type == LN_F32) launch_norm<LN_F32, LN_F32>(a, bwd, vectors, st);
    else if (type == LN_BF16 && w_fp32) launch_norm<LN_BF16, LN_F32>(a, bwd, vectors, st);
    else if (type == LN_BF16) launch_norm<LN_BF16, LN_BF16>(a, bwd, vectors, st);
    else if (w_fp32) launch_norm<LN_F16, LN_F32>(a, bwd, vectors, st);
    else launch_norm<LN_F16, LN_F16>(a, bwd, vectors, st);
}

int check_rows(const char *what, int64_t M, int32_t d, int32_t type, int64_t ld0, int64_t ld1, int64_t ld2) {
    if (M < 0 || d <= 0 || ld0 < d || ld1 < d || ld2 < d) return mortar_fail(MORTAR_ERR_ARG, "%s: bad shape", what);
    if (type != LN_BF16 && type != LN_F16 && type != LN_F32) return mortar_fail(MORTAR_ERR_ARG, "%s: bf16, fp16 or fp32", what);
    if (M >= INT32_MAX || d > (1 << 30)) return mortar_fail(MORTAR_ERR_LIMIT, "%s: too many rows or columns", what);
    return MORTAR_OK;
}

}  // namespace

extern "C" int mortar_layernorm(const void *x, int64_t M, int32_t d, int64_t ldx, int32_t type, const void *w, const void *b, int32_t w_fp32, float eps,
                                void *y, int64_t ldy, float *mean, float *rstd, void *stream) {
    const int rc = check_rows("layernorm", M, d, type, ldx, ldy, ldy);
    if (rc) return rc;
    if (M == 0) return MORTAR_OK;
    if (!x || !y || !mean != !rstd) return mortar_fail(MORTAR_ERR_ARG, "layernorm: null pointer");
    LnArgs a{};
    a.x = x; a.w = w; a.b = b; a.y = y; a.mean = mean; a.rstd = rstd;
    a.M = M; a.ldx = ldx; a.ldy = ldy; a.d = d; a.eps = eps;
    const int v = type == LN_F32 ? 4 : 8;
    const bool vectors = d % v == 0 && ldx % v == 0 && ldy % v == 0 && aligned(x) && aligned(y) && aligned(w) && aligned(b);
    launch_typed(a, type, w_fp32, false, vectors, static_cast<hipStream_t>(stream));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "layernorm: %s", hipGetErrorString(e));
}

extern "C" int64_t mortar_layernorm_workspace_bytes(int64_t M, int32_t d) { return M > 0 && d > 0 ? slabs_of(M) * 2 * d * 4 : 0; }

extern "C" int mortar_layernorm_bwd(const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t M, int32_t d, int32_t type, const void *w,
                                    int32_t w_fp32, const float *mean, const float *rstd, void *dx, int64_t lddx, void *dw, void *db,
                                    float *workspace, void *stream) {
    const int rc = check_rows("layernorm_bwd", M, d, type, ldx, lddy, dx ? lddx : d);
    if (rc) return rc;
    if (M == 0) return mortar_fail(MORTAR_ERR_ARG, "layernorm_bwd: no rows");
    const bool params = dw || db;
    if (!x || !dy || !mean || !rstd || (params && !workspace)) return mortar_fail(MORTAR_ERR_ARG, "layernorm_bwd: null pointer");
    if (!dx && !params) return MORTAR_OK;
    LnArgs a{};
    a.x = x; a.dy = dy; a.w = w; a.y = dx; a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.slabs = params ? workspace : nullptr;
    a.M = M; a.ldx = ldx; a.lddy = lddy; a.ldy = lddx; a.d = d;
    const int v = type == LN_F32 ? 4 : 8;
    const bool vectors = d % v == 0 && ldx % v == 0 && lddy % v == 0 && aligned(x) && aligned(dy) && aligned(w) && (!dx || (lddx % v == 0 && aligned(dx)));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    launch_typed(a, type, w_fp32, true, vectors, st);
    if (params) {
        const dim3 grid((unsigned)((d + 31) / 32), 2);
        const int n = (int)slabs_of(M);
        if (type == LN_F32 || w_fp32) hipLaunchKernelGGL((ln_join_kernel<LN_F32>), grid, dim3(1024), 0, st, workspace, n, d, dw, db);
        else if (type == LN_BF16) hipLaunchKernelGGL((ln_join_kernel<LN_BF16>), grid, dim3(1024), 0, st, workspace, n, d, dw, db);
        else hipLaunchKernelGGL((ln_join_kernel<LN_F16>), grid, dim3(1024), 0, st, workspace, n, d, dw, db);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MORTAR_OK : mortar_fail(MORTAR_ERR_HIP, "layernorm_bwd: %s", hipGetErrorString(e));
}
