// Log-probabilities of given tokens under a model's logits, and the two losses that train on them: the clipped policy loss with a
// KL term and the loss of paired log ratios.  For every token (row) with logits z[V], target a, temperature tau:
//   c = max z,   s = sum_j exp((z_j - c) / tau),   lp = (z_a - c) / tau - log s,   p_j = exp((z_j - c) / tau) / s
//   d lp / d z_j = (1[j = a] - p_j) / tau
// Everything is bound by the bytes of the logits (65536 of them per token), so a row's maximum and sum are taken in one pass
// (the sum is rescaled when the maximum grows), and where the gradient needs nothing but the row itself (policy loss) the row is
// read again right behind that, out of the L2 cache (rows in flight: two 512-thread blocks per SM, 39 MB of bf16 rows of 65536).
// Rows that the mask leaves out, or whose target is no token, are not read: their log-probability and gradient are zero
// whatever the logits hold.
// The difference z - c is formed before it is scaled, so that it is exact near the maximum and does not overflow for logits at the
// end of the type's range; a row of -inf has no distribution and gives NaN.
// The reference has no trainer (its trainer files are empty); these operators stand beside the next-token loss.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "wkv6_internal.h"

namespace wkv6 {

namespace {

struct Rows {
    const void *z;
    const int64_t *targets;
    const uint8_t *mask;
    int64_t rows, seq_stride, row_stride;
    int T, V;
    float k;         // log2(e) / tau
    float inv_tau;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (a + b) * c per component, two instructions for the pair
__device__ __forceinline__ float2 add_mul(float2 a, float b, float c) {
    unsigned long long x, y, w;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(b));
    asm("mov.b64 %0, {%1, %1};" : "=l"(w) : "f"(c));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(w));
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}

// Sixteen bytes of logits as fp32 pairs and back (each value rounded once, to nearest).
template <typename T> struct Vec;

template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4 &v, float2 (&f)[4]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 put(const float2 (&f)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[i].x, f[i].y);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float max(const uint4 &v) {
        const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&v);
        const float2 f = __bfloat1622float2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ __nv_bfloat16 one(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ float get1(__nv_bfloat16 x) { return __bfloat162float(x); }
};

template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4 &v, float2 (&f)[4]) {
        const __half2 *p = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __half22float2(p[i]);
    }
    static __device__ __forceinline__ uint4 put(const float2 (&f)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float max(const uint4 &v) {
        const __half2 *p = reinterpret_cast<const __half2 *>(&v);
        const float2 f = __half22float2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
        return fmaxf(f.x, f.y);
    }
    static __device__ __forceinline__ __half one(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ float get1(__half x) { return __half2float(x); }
};

template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4 &v, float2 (&f)[2]) {
        f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ uint4 put(const float2 (&f)[2]) {
        return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    }
    static __device__ __forceinline__ float max(const uint4 &v) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static __device__ __forceinline__ float one(float x) { return x; }
    static __device__ __forceinline__ float get1(float x) { return x; }
};

// Values in front of the first 16-byte boundary at or behind p (at most n).
template <typename T>
__device__ __forceinline__ int head_of(const T *p, int n) {
    const int h = (int)((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T));
    return h < n ? h : n;
}

// (maximum, sum of exp2((z - maximum) k)) of two parts of a row; the same bits whichever part comes first, so that all lanes of an
// exchange end with one result
__device__ __forceinline__ void merge(float &mx, float &sum, float mx2, float sum2, float k) {
    const float m = fmaxf(mx, mx2);
    sum = __fadd_rn(__fmul_rn(sum, ex2((mx - m) * k)), __fmul_rn(sum2, ex2((mx2 - m) * k)));
    mx = m;
}

// This thread's share (every THREADS-th vector) of a row.  The maximum starts at the lowest finite value and not at -inf: a part
// that holds nothing but -inf then adds zeros.
template <typename T, int THREADS>
__device__ __forceinline__ void row_part(const T *z, int V, int tid, float k, float &mx, float &sum) {
    constexpr int N = Vec<T>::N, U = 4;
    mx = -FLT_MAX;
    sum = 0.f;
    const int head = head_of(z, V), vecs = (V - head) / N;
    const uint4 *v = reinterpret_cast<const uint4 *>(z + head);
    for (int i0 = tid; i0 < vecs; i0 += THREADS * U) {
        uint4 q[U];
        float m = mx;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * THREADS < vecs) q[u] = __ldg(v + i0 + u * THREADS);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * THREADS < vecs) m = fmaxf(m, Vec<T>::max(q[u]));
        sum *= ex2((mx - m) * k);
        mx = m;
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * THREADS < vecs) {
                float2 f[N / 2];
                Vec<T>::get(q[u], f);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float2 d = add_mul(f[e], -mx, k);
                    s2.x += ex2(d.x);
                    s2.y += ex2(d.y);
                }
            }
        }
        sum += s2.x + s2.y;
    }
    const int tail = head + vecs * N, loose = head + V - tail;      // values outside the vectors: fewer than two vectors' worth
    for (int i = tid; i < loose; i += THREADS) {
        const float x = Vec<T>::get1(z[i < head ? i : tail + i - head]), m = fmaxf(mx, x);
        sum = sum * ex2((mx - m) * k) + ex2((x - m) * k);
        mx = m;
    }
}

// g_j = c (1[j = a] - p_j) over the vectors of the gradient row from `first` on, every `step`-th.  The logits' row may lie at
// another offset from the 16-byte boundaries than the gradient's: its values are then loaded one by one.  (Products and sums are
// kept apart, so that both kernels that come here give the same bits.)
template <typename T>
__device__ __forceinline__ void row_gradient(const T *z, T *g, int V, int target, float mx, float inv_sum, float k, float c, int first, int step) {
    constexpr int N = Vec<T>::N, U = 2;
    const int head = head_of(g, V), vecs = (V - head) / N;
    const bool same = head_of(z, V) == head;
    const float neg = -c * inv_sum;
    for (int i0 = first; i0 < vecs; i0 += step * U) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * step;
            if (i < vecs) {
                if (same) {
                    q[u] = __ldg(reinterpret_cast<const uint4 *>(z + head) + i);
                } else {
                    T x[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) x[e] = z[head + (int64_t)i * N + e];
                    memcpy(&q[u], x, 16);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * step;
            if (i < vecs) {
                float2 f[N / 2];
                Vec<T>::get(q[u], f);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float2 d = add_mul(f[e], -mx, k);
                    f[e] = make_float2(__fmul_rn(ex2(d.x), neg), __fmul_rn(ex2(d.y), neg));
                }
                const int at = target - head - i * N;
                if (at >= 0 && at < N) {
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        if (at == 2 * e) f[e].x = __fadd_rn(f[e].x, c);
                        if (at == 2 * e + 1) f[e].y = __fadd_rn(f[e].y, c);
                    }
                }
                reinterpret_cast<uint4 *>(g + head)[i] = Vec<T>::put(f);
            }
        }
    }
    const int tail = head + vecs * N, loose = head + V - tail;
    for (int i = first; i < loose; i += step) {
        const int j = i < head ? i : tail + i - head;
        float x = __fmul_rn(ex2((Vec<T>::get1(z[j]) - mx) * k), neg);
        if (j == target) x = __fadd_rn(x, c);
        g[j] = Vec<T>::one(x);
    }
}

template <typename T>
__device__ __forceinline__ void row_zero(T *g, int V, int first, int step) {
    constexpr int N = Vec<T>::N;
    const int head = head_of(g, V), vecs = (V - head) / N, tail = head + vecs * N, loose = head + V - tail;
    for (int i = first; i < vecs; i += step) reinterpret_cast<uint4 *>(g + head)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = first; i < loose; i += step) g[i < head ? i : tail + i - head] = Vec<T>::one(0.f);
}

template <typename T>
__device__ __forceinline__ const T *row_of(const Rows &a, int64_t row) {
    return static_cast<const T *>(a.z) + (row / a.T) * a.seq_stride + (row % a.T) * a.row_stride;
}

// The row's target, or -1 where the row does not count.
__device__ __forceinline__ int target_of(const Rows &a, int64_t row) {
    const int64_t t = a.targets[row];
    return (a.mask == nullptr || a.mask[row]) && t >= 0 && t < a.V ? (int)t : -1;
}

// What the policy loss takes beside the rows.
struct Policy {
    const float *advantages, *old_lp, *ref_lp;
    float low, high, kl, scale;
    int reduction;
    const int *counts;       // live rows of each part
    int parts;
    float *row_loss;
    unsigned *done;
    float *loss;
};

constexpr int kCountRows = 1024;    // rows of a part where tokens are counted over all sequences
constexpr int kRowThreads = 512, kWarpRows = 8;

// The last block to finish adds up the rows, in an order that does not depend on which block that is.
__device__ __forceinline__ void total_loss(const Policy &q, int64_t rows) {
    __shared__ double part[32];
    __shared__ bool last;
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(q.done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) x += (double)__ldcg(q.row_loss + i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < (int)blockDim.x / 32; ++i) x += part[i];
        *q.loss = (float)x;
    }
}

// THREADS = 512: a block per row; 32: a warp per row (rows of a few KB, where a block's reduction would cost more than its row).
// POLICY: the loss and, with g, the gradient behind the log-probabilities.
template <typename T, int THREADS, bool POLICY>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpRows : THREADS, THREADS == 32 ? 4 : 2)
token_rows_kernel(const Rows a, float *__restrict__ lp_out, float2 *__restrict__ stat, const Policy q, float *__restrict__ coefficient,
                  T *__restrict__ g) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = THREADS == 32 ? lane : threadIdx.x;
    const int64_t row = THREADS == 32 ? (int64_t)blockIdx.x * kWarpRows + warp : blockIdx.x;
    if (THREADS != 32 || row < a.rows) {
        const int target = target_of(a, row);
        float lp = 0.f, c = 0.f, loss = 0.f, mx = 0.f, inv_sum = 0.f;
        const T *z = row_of<T>(a, row);
        if (target >= 0) {
            float adv = 0.f, old = 0.f, ref = 0.f;
            int n = 0;
            if constexpr (POLICY) {       // requested before the row
                adv = q.advantages[row];
                old = q.old_lp[row];
                if (q.ref_lp != nullptr) ref = q.ref_lp[row];
                if (q.reduction == WKV6_MEAN)
                    for (int i = lane; i < q.parts; i += 32) n += q.counts[i];
                else if (q.reduction == WKV6_SEQUENCE_MEAN)
                    n = q.counts[row / a.T];
            }
            float sum;
            const float zt = Vec<T>::get1(z[target]);
            row_part<T, THREADS>(z, a.V, tid, a.k, mx, sum);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, mx, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
                merge(mx, sum, m2, s2, a.k);
            }
            if constexpr (THREADS != 32) {
                __shared__ float2 part[THREADS / 32];
                if (lane == 0) part[warp] = make_float2(mx, sum);
                __syncthreads();
                const float2 p = part[lane % (THREADS / 32)];
                mx = p.x;
                sum = p.y;
#pragma unroll
                for (int o = THREADS / 64; o > 0; o >>= 1) {
                    const float m2 = __shfl_xor_sync(0xffffffffu, mx, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
                    merge(mx, sum, m2, s2, a.k);
                }
            }
            inv_sum = 1.f / sum;
            lp = (zt - mx) * a.inv_tau - logf(sum);
            if constexpr (POLICY) {
                float w = q.scale;
                if (q.reduction == WKV6_MEAN) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
                    w = q.scale / (float)n;
                } else if (q.reduction == WKV6_SEQUENCE_MEAN) {
                    w = q.scale / ((float)n * (float)(a.rows / a.T));
                }
                // comparisons written so that a NaN ratio is not clipped away
                const float rho = expf(lp - old), free = rho * adv;
                const float clipped = (rho < q.low ? q.low : rho > q.high ? q.high : rho) * adv;
                const bool open = !(free > clipped);
                loss = open ? -free : -clipped;
                c = open ? -free : 0.f;
                if (q.ref_lp != nullptr) {     // exp(d) - d - 1 is d^2 / 2 for small d: taken from exp(d) - 1
                    const float d = ref - lp, e = expm1f(d);
                    loss += q.kl * (e - d);
                    c -= q.kl * e;
                }
                loss *= w;
                c *= w;
            }
        }
        if (tid == 0) {
            lp_out[row] = lp;
            if (stat != nullptr) stat[row] = make_float2(mx, inv_sum);
            if constexpr (POLICY) {
                q.row_loss[row] = loss;
                coefficient[row] = c;
            }
        }
        if constexpr (POLICY) {
            if (g != nullptr) {
                T *gr = g + row * a.V;
                if (c != 0.f)                  // NaN included
                    row_gradient(z, gr, a.V, target, mx, inv_sum, a.k, c * a.inv_tau, tid, THREADS);
                else
                    row_zero(gr, a.V, tid, THREADS);
            }
        }
    }
    if constexpr (POLICY) {
        if (THREADS == 32) __syncthreads();
        total_loss(q, a.rows);
    }
}

// Gradient of the logits from the rows' statistics and one coefficient per row, or per sequence:
//   g = coefficient (*factor) (1[j = a] - p_j) / tau
// A block takes a part of a row (blockIdx.y), so that few long rows fill the GPU too.  `unless_one`: nothing is done where *factor
// is 1 (the gradient is there already).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpRows : THREADS, THREADS == 32 ? 4 : 3)
token_gradient_kernel(const Rows a, const float2 *__restrict__ stat, const float *__restrict__ coefficient, int per_sequence,
                      const float *__restrict__ factor, int unless_one, T *__restrict__ g) {
    const float f = factor != nullptr ? *factor : 1.f;
    if (unless_one && f == 1.f) return;
    const int64_t row = THREADS == 32 ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    const int first = THREADS == 32 ? threadIdx.x & 31 : blockIdx.y * THREADS + threadIdx.x, step = THREADS == 32 ? 32 : THREADS * gridDim.y;
    const int target = target_of(a, row);
    const float c = target < 0 ? 0.f : coefficient[per_sequence ? row / a.T : row] * f * a.inv_tau;
    T *gr = g + row * a.V;
    if (c != 0.f) {
        const float2 s = stat[row];
        row_gradient(row_of<T>(a, row), gr, a.V, target, s.x, s.y, a.k, c, first, step);
    } else {
        row_zero(gr, a.V, first, step);
    }
}

// Live rows of every part: a sequence, or kCountRows rows of the whole where only their total is wanted.
__global__ void __launch_bounds__(256) count_rows_kernel(const Rows a, int64_t part_rows, int *__restrict__ counts, unsigned *__restrict__ done) {
    __shared__ int part[8];
    if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0u;
    const int64_t first = blockIdx.x * part_rows, end = first + part_rows < a.rows ? first + part_rows : a.rows;
    int n = 0;
    for (int64_t i = first + threadIdx.x; i < end; i += 256) n += target_of(a, i) >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) n += part[i];
        counts[blockIdx.x] = n;
    }
}

// log-probability of every sequence: its live rows' sum (in 64 bits: thousands of terms, of which only the difference to a
// reference matters) or mean.  A block per sequence.
__global__ void __launch_bounds__(256) sequence_sum_kernel(const Rows a, const float *__restrict__ lp, int average, float *__restrict__ seq,
                                                           double *__restrict__ seq64, int *__restrict__ count) {
    __shared__ double part[8];
    __shared__ int live[8];
    const int64_t first = (int64_t)blockIdx.x * a.T;
    double x = 0.0;
    int n = 0;
    for (int i = threadIdx.x; i < a.T; i += 256) {
        if (target_of(a, first + i) >= 0) {
            x += (double)lp[first + i];
            ++n;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = x;
        live[threadIdx.x >> 5] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) {
            x += part[i];
            n += live[i];
        }
        if (average && n > 1) x /= n;
        seq64[blockIdx.x] = x;
        seq[blockIdx.x] = (float)x;
        count[blockIdx.x] = n;
    }
}

// One block: margin, loss and slope of every pair, their mean in a fixed order.
__global__ void __launch_bounds__(256) preference_pairs_kernel(int pairs, const double *__restrict__ seq64, const int *__restrict__ count,
                                                               const float *__restrict__ ref, double beta, double smoothing, double margin,
                                                               int average, double scale, float *__restrict__ coefficient,
                                                               float *__restrict__ loss) {
    __shared__ double part[8];
    double total = 0.0;
    for (int i = threadIdx.x; i < pairs; i += 256) {
        const int j = i + pairs;
        double over = seq64[i] - seq64[j];
        if (ref != nullptr) over -= (double)ref[i] - (double)ref[j];
        const double d = beta * over - margin, tail = log1p(exp(-fabs(d)));
        total += (1.0 - smoothing) * (tail + fmax(-d, 0.0));           // a NaN reaches the sum through the tail
        if (smoothing != 0.0) total += smoothing * (tail + fmax(d, 0.0));
        const double slope = -beta * (1.0 - smoothing - 1.0 / (1.0 + exp(-d))) * (scale / pairs);
        coefficient[i] = (float)(slope / (average && count[i] > 1 ? count[i] : 1));
        coefficient[j] = (float)(-slope / (average && count[j] > 1 ? count[j] : 1));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) total += part[i];
        *loss = (float)(total * (scale / pairs));
    }
}

// A warp per row up to this many bytes of logits, a block above.
constexpr int64_t kWarpRowBytes = 4096;

int rows_of(const wkv6_token_logits *p, Rows *a, const char *what, bool need_logits) {
    if (p == nullptr) return fail(WKV6_ERR_INVALID, "%s: NULL argument", what);
    if (p->S < 0 || p->T < 0 || p->V < 1) return fail(WKV6_ERR_INVALID, "%s: S=%d T=%d V=%d", what, p->S, p->T, p->V);
    if (p->dtype != WKV6_BF16 && p->dtype != WKV6_F16 && p->dtype != WKV6_F32) return fail(WKV6_ERR_INVALID, "%s: unknown dtype code", what);
    if (!(p->temperature > 0.f) || std::isinf(p->temperature)) return fail(WKV6_ERR_INVALID, "%s: temperature must be positive and finite", what);
    a->rows = (int64_t)p->S * p->T;
    if (a->rows > 2147483647LL) return fail(WKV6_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", what);
    a->T = p->T;
    a->V = p->V;
    a->row_stride = p->row_stride ? p->row_stride : p->V;
    a->seq_stride = p->seq_stride ? p->seq_stride : p->T * a->row_stride;
    if (a->row_stride < 0 || a->seq_stride < 0) return fail(WKV6_ERR_INVALID, "%s: negative strides", what);
    if (a->rows > 0 && ((need_logits && p->logits == nullptr) || p->targets == nullptr)) return fail(WKV6_ERR_INVALID, "%s: NULL argument", what);
    if (reinterpret_cast<uintptr_t>(p->logits) % dtype_size(p->dtype)) return fail(WKV6_ERR_INVALID, "%s: misaligned logits", what);
    a->z = p->logits;
    a->targets = p->targets;
    a->mask = p->mask;
    a->k = (float)(1.4426950408889634 / (double)p->temperature);
    a->inv_tau = (float)(1.0 / (double)p->temperature);
    return WKV6_OK;
}

bool warp_rows(const wkv6_token_logits *p) { return (int64_t)p->V * (int64_t)dtype_size(p->dtype) <= kWarpRowBytes; }

template <bool POLICY>
int launch_rows(const wkv6_token_logits *p, const Rows &a, float *lp, float2 *stat, const Policy &q, float *coefficient, void *g,
                cudaStream_t st) {
    const bool warp = warp_rows(p);
    const unsigned grid = (unsigned)(warp ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows);
#define LAUNCH(T)                                                                                                                   \
    if (warp) token_rows_kernel<T, 32, POLICY><<<grid, 32 * kWarpRows, 0, st>>>(a, lp, stat, q, coefficient, static_cast<T *>(g)); \
    else token_rows_kernel<T, kRowThreads, POLICY><<<grid, kRowThreads, 0, st>>>(a, lp, stat, q, coefficient, static_cast<T *>(g))
    switch (p->dtype) {
        case WKV6_BF16: LAUNCH(__nv_bfloat16); break;
        case WKV6_F16: LAUNCH(__half); break;
        default: LAUNCH(float); break;
    }
#undef LAUNCH
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? WKV6_OK : cuda_fail(e, "token_rows_kernel launch");
}

int64_t count_parts(int64_t S, int64_t T, int reduction) {
    return reduction == WKV6_SEQUENCE_MEAN ? S : (S * T + kCountRows - 1) / kCountRows;
}

}  // namespace

}  // namespace wkv6

using namespace wkv6;

extern "C" int wkv6_token_log_probs(const wkv6_token_logits *p, float *log_probs, float *stat, void *stream) {
    Rows a;
    if (const int rc = rows_of(p, &a, "wkv6_token_log_probs", true)) return rc;
    if (a.rows == 0) return WKV6_OK;
    if (log_probs == nullptr) return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs: NULL argument");
    if (reinterpret_cast<uintptr_t>(stat) % 8) return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs: stat must be 8-byte aligned");
    return launch_rows<false>(p, a, log_probs, reinterpret_cast<float2 *>(stat), Policy{}, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int wkv6_token_log_probs_backward(const wkv6_token_logits *p, const float *stat, const float *coefficient, int32_t per_sequence,
                                             const float *factor, int32_t unless_one, void *g, void *stream) {
    Rows a;
    if (const int rc = rows_of(p, &a, "wkv6_token_log_probs_backward", true)) return rc;
    if (a.rows == 0) return WKV6_OK;
    if (!stat || !coefficient || !g || (unless_one && !factor)) return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs_backward: NULL argument");
    if (!aligned16(g) || reinterpret_cast<uintptr_t>(stat) % 8)
        return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs_backward: the gradient must be 16-byte aligned, stat 8-byte");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool warp = warp_rows(p);
    constexpr int threads = 256;
    // parts of at least two vectors a thread, as many as four blocks per SM need
    const int64_t want = (4LL * sm_count() + a.rows - 1) / a.rows, most = (int64_t)a.V * (int64_t)dtype_size(p->dtype) / (threads * 32) + 1;
    const dim3 grid((unsigned)(warp ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows), (unsigned)(warp ? 1 : want < most ? want : most));
    const float2 *s = reinterpret_cast<const float2 *>(stat);
#define LAUNCH(T)                                                                                                                            \
    if (warp) token_gradient_kernel<T, 32><<<grid, 32 * kWarpRows, 0, st>>>(a, s, coefficient, per_sequence, factor, unless_one, static_cast<T *>(g)); \
    else token_gradient_kernel<T, threads><<<grid, threads, 0, st>>>(a, s, coefficient, per_sequence, factor, unless_one, static_cast<T *>(g))
    switch (p->dtype) {
        case WKV6_BF16: LAUNCH(__nv_bfloat16); break;
        case WKV6_F16: LAUNCH(__half); break;
        default: LAUNCH(float); break;
    }
#undef LAUNCH
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? WKV6_OK : cuda_fail(e, "token_gradient_kernel launch");
}

extern "C" size_t wkv6_policy_loss_workspace_bytes(int32_t S, int32_t T, int32_t reduction) {
    if (S <= 0 || T <= 0) return 0;
    return 16 + (size_t)((int64_t)S * T) * 4 + (size_t)count_parts(S, T, reduction) * 4;
}

extern "C" int wkv6_policy_loss(const wkv6_token_logits *p, const wkv6_policy *c, float *loss, float *log_probs, float *stat,
                                float *coefficient, void *g, void *workspace, size_t workspace_bytes, void *stream) {
    Rows a;
    if (const int rc = rows_of(p, &a, "wkv6_policy_loss", true)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c == nullptr || loss == nullptr) return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: NULL argument");
    if (c->reduction != WKV6_MEAN && c->reduction != WKV6_SEQUENCE_MEAN && c->reduction != WKV6_SUM)
        return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: unknown reduction");
    if (a.rows == 0) {
        const cudaError_t e = cudaMemsetAsync(loss, 0, sizeof(float), st);
        return e == cudaSuccess ? WKV6_OK : cuda_fail(e, "cudaMemsetAsync");
    }
    if (!c->advantages || !c->old_log_probs || !log_probs || !coefficient || !workspace)
        return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: NULL argument");
    if (!aligned16(g) || reinterpret_cast<uintptr_t>(stat) % 8 || !aligned16(workspace))
        return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: the gradient and the workspace must be 16-byte aligned, stat 8-byte");
    if (workspace_bytes < wkv6_policy_loss_workspace_bytes(p->S, p->T, c->reduction))
        return fail(WKV6_ERR_WORKSPACE, "wkv6_policy_loss: workspace of %zu bytes, %zu are needed", workspace_bytes,
                    wkv6_policy_loss_workspace_bytes(p->S, p->T, c->reduction));
    Policy q{};
    q.advantages = c->advantages;
    q.old_lp = c->old_log_probs;
    q.ref_lp = c->kl_coef != 0.0 ? c->ref_log_probs : nullptr;
    if (c->kl_coef != 0.0 && c->ref_log_probs == nullptr) return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: a KL term needs ref_log_probs");
    q.low = (float)(1.0 - c->clip_low);
    q.high = (float)(1.0 + c->clip_high);
    q.kl = (float)c->kl_coef;
    q.scale = (float)c->scale;
    q.reduction = c->reduction;
    q.done = static_cast<unsigned *>(workspace);
    q.row_loss = reinterpret_cast<float *>(static_cast<char *>(workspace) + 16);
    int *counts = reinterpret_cast<int *>(q.row_loss + a.rows);
    q.counts = counts;
    q.parts = (int)count_parts(p->S, p->T, c->reduction);
    q.loss = loss;
    count_rows_kernel<<<q.parts, 256, 0, st>>>(a, c->reduction == WKV6_SEQUENCE_MEAN ? p->T : kCountRows, counts, q.done);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "count_rows_kernel launch");
    return launch_rows<true>(p, a, log_probs, reinterpret_cast<float2 *>(stat), q, coefficient, g, st);
}

extern "C" size_t wkv6_preference_loss_workspace_bytes(int32_t S) { return S > 0 ? (size_t)S * 12 : 0; }

extern "C" int wkv6_preference_loss(const wkv6_token_logits *p, const float *log_probs, const wkv6_preference *c, float *loss,
                                    float *sequence_log_probs, float *coefficient, void *workspace, size_t workspace_bytes, void *stream) {
    Rows a;
    if (const int rc = rows_of(p, &a, "wkv6_preference_loss", false)) return rc;
    if (p->S % 2) return fail(WKV6_ERR_INVALID, "wkv6_preference_loss: S=%d sequences are no pairs", p->S);
    if (c == nullptr || loss == nullptr) return fail(WKV6_ERR_INVALID, "wkv6_preference_loss: NULL argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->S == 0) {
        const cudaError_t e = cudaMemsetAsync(loss, 0, sizeof(float), st);
        return e == cudaSuccess ? WKV6_OK : cuda_fail(e, "cudaMemsetAsync");
    }
    if (!sequence_log_probs || !coefficient || !workspace || (a.rows && !log_probs))
        return fail(WKV6_ERR_INVALID, "wkv6_preference_loss: NULL argument");
    if (reinterpret_cast<uintptr_t>(workspace) % 8) return fail(WKV6_ERR_INVALID, "wkv6_preference_loss: the workspace must be 8-byte aligned");
    if (workspace_bytes < wkv6_preference_loss_workspace_bytes(p->S))
        return fail(WKV6_ERR_WORKSPACE, "wkv6_preference_loss: workspace of %zu bytes, %zu are needed", workspace_bytes,
                    wkv6_preference_loss_workspace_bytes(p->S));
    double *seq64 = static_cast<double *>(workspace);
    int *count = reinterpret_cast<int *>(seq64 + p->S);
    sequence_sum_kernel<<<p->S, 256, 0, st>>>(a, log_probs, c->average, sequence_log_probs, seq64, count);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "sequence_sum_kernel launch");
    preference_pairs_kernel<<<1, 256, 0, st>>>(p->S / 2, seq64, count, c->ref_log_probs, c->beta, c->label_smoothing, c->margin, c->average,
                                               c->scale, coefficient, loss);
    e = cudaGetLastError();
    return e == cudaSuccess ? WKV6_OK : cuda_fail(e, "preference_pairs_kernel launch");
}
