// Log-probabilities of given tokens under a model's logits, and the two losses that train on them: the clipped policy loss with a
// KL term and the loss of paired log ratios.  For every token (row) with logits z[V], target a, temperature tau, k = log2(e) / tau:
//   c = k max z,   s = sum_j 2^(k z_j - c),   lp = (k z_a - c - log2 s) ln 2,   p_j = 2^(k z_j - c) / s
//   d lp / d z_j = (1[j = a] - p_j) / tau
// Everything is bound by the bytes of the logits (65536 of them per token) and next by instructions: at the copy bandwidth a bf16
// logit has to be done with in 11 (it takes 6.4 forward, 15 with the gradient behind it, for which there is twice the time).  A row's
// maximum and sum are taken in one pass (the sum is rescaled when the maximum grows), and where the gradient needs nothing but the row
// itself (policy loss) the row is gone through again right behind that, from its end to its start: the end is still in registers, the
// start in shared memory, the middle in the L2 cache.  A block of 256 threads has a row, four of them are on an SM: with 512 threads all warps of an SM compute or wait
// at once (rows of 65536 bf16: 82 us instead of 72 for 2968 of them), with 128 the rows under way do not fit the L2 cache (policy loss of
// 8192 such rows 418 us instead of 373), and rows that blocks claim and request ahead through shared memory took 92 us: more instructions, nothing gained.
// Measured, 6000 rows of 65536 bf16, all of them counting: log-probabilities 121 us = 6.48 TB/s (99 % of the copy bandwidth), their
// gradient 249 us = 6.31 TB/s, the policy loss with its gradient 281 us = 5.6 TB/s: what its second pass takes from the L2 cache is
// lost there for 9 % of the rows (20 % without the part in shared memory, and 286 us).
// Rows that the mask leaves out, or whose target is no token, are not read: their log-probability and gradient are zero
// whatever the logits hold.
// k z - c is one multiply-add: c is rounded, but it is the same c everywhere in a part of a row, and what it is off by, as a power of two,
// is a factor of that part's sum that the next rescaling takes off again.  It has to stay a harmless one: below |c| = 2^24 it is at most 2^(1/2).
// Rows with a maximum beyond that (|z| / tau above 1.16e7) take a second way (`wide`), which subtracts the maximum before the scaling;
// smaller logits among ordinary ones (fills of -1e10 and the like) lie below the maximum that every part starts with, and add zeros.
// A row of -inf has no distribution and gives NaN.
// The reference has no trainer (its trainer files are empty); these operators stand beside the next-token loss.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>

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
    float low;       // where a part's maximum starts; rows whose maximum is not between low and -low take the wide way
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (a - b) k, by way of half the difference: that of two values at the ends of the range does not overflow, and k may be small.  (Written
// as separate operations, and the loop over a row that takes this way not unrolled: with fmaf and unrolled the rows that never come here
// lost 0.06 us of 5.08, 16 rows of 65536 bf16, and calls in a row 0.25 of 6.45.)
__device__ __forceinline__ float apart(float a, float b, float k) { return __fmul_rn(__fsub_rn(a * 0.5f, b * 0.5f), k) * 2.f; }

// Sixteen bytes of logits as fp32 pairs and back (each value rounded once, to nearest).
template <typename T> struct Vec;

template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t kNone = 0xff80ff80u;      // -inf throughout
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
    static constexpr uint32_t kNone = 0xfc00fc00u;
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
    static constexpr uint32_t kNone = 0xff800000u;
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

__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// What a part of a row has come to: its maximum (not below Rows::low, so that parts of nothing but -inf or large fills add zeros), c = k max,
// and the sum.
struct Part {
    float mx, c, sum;
};

// Takes U vectors into a part, or the first `have` of them.
template <typename T, int U>
__device__ __forceinline__ void take(const uint4 (&q)[U], float k, Part &r, int have = U) {
    constexpr int N = Vec<T>::N;
    float m = r.mx;
#pragma unroll
    for (int u = 0; u < U; ++u) m = fmaxf(m, Vec<T>::max(q[u]));
    const float c = __fmul_rn(m, k);       // not to be contracted with a sum: c stands for itself, rounded, everywhere
    const float scale = ex2(r.c - c);
    float sum0 = 0.f, sum1 = 0.f;      // not the whole sum: next to a large term in it, each of hundreds of small ones would be rounded
    r.mx = m;
    r.c = c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u >= have) break;
        float2 f[N / 2];
        Vec<T>::get(q[u], f);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            sum0 += ex2(fmaf(f[e].x, k, -c));
            sum1 += ex2(fmaf(f[e].y, k, -c));
        }
    }
    r.sum = fmaf(r.sum, scale, sum0 + sum1);
}

// g (1[j = a] - p_j) of a vector of logits: neg = -g / sum, `at` = a's place in the vector.  (Products and sums are kept apart, so that all
// kernels that come here give the same bits.)  WIDE: c is the maximum itself.
template <typename T, bool WIDE>
__device__ __forceinline__ float gradient_of(float z, float k, float c, float neg) {
    return __fmul_rn(ex2(WIDE ? apart(z, c, k) : fmaf(z, k, -c)), neg);
}
template <typename T, bool WIDE>
__device__ __forceinline__ uint4 gradient_of(const uint4 &q, int at, float k, float c, float neg, float g) {
    constexpr int N = Vec<T>::N;
    float2 f[N / 2];
    Vec<T>::get(q, f);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) f[e] = make_float2(gradient_of<T, WIDE>(f[e].x, k, c, neg), gradient_of<T, WIDE>(f[e].y, k, c, neg));
    if (at >= 0) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            if (at == 2 * e) f[e].x = __fadd_rn(f[e].x, g);
            if (at == 2 * e + 1) f[e].y = __fadd_rn(f[e].y, g);
        }
    }
    return Vec<T>::put(f);
}

// A row's vectors, and its values outside them: fewer than two vectors' worth, in front (head) and behind (from tail on).
struct Cut {
    int head, vecs, tail, loose;
    __device__ __forceinline__ int at(int i) const { return i < head ? i : tail + i - head; }
};
template <typename T>
__device__ __forceinline__ Cut cut_of(const T *p, int V) {
    Cut l;
    l.head = head_of(p, V);
    l.vecs = (V - l.head) / Vec<T>::N;
    l.tail = l.head + l.vecs * Vec<T>::N;
    l.loose = l.head + V - l.tail;
    return l;
}

template <typename T>
__device__ __forceinline__ void take_loose(const T *z, const Cut &l, int first, int step, float k, Part &r) {
    for (int i = first; i < l.loose; i += step) {
        const float x = Vec<T>::get1(z[l.at(i)]), m = fmaxf(r.mx, x), c = __fmul_rn(m, k);
        r.sum = r.sum * ex2(r.c - c) + ex2(fmaf(x, k, -c));
        r.mx = m;
        r.c = c;
    }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void gradient_loose(const T *z, T *out, const Cut &l, int target, float k, float c, float neg, float g, int first, int step) {
    for (int i = first; i < l.loose; i += step) {
        const int j = l.at(i);
        float x = gradient_of<T, WIDE>(Vec<T>::get1(z[j]), k, c, neg);
        if (j == target) x = __fadd_rn(x, g);
        out[j] = Vec<T>::one(x);
    }
}

constexpr int kU = 4;         // vectors that a thread requests at once, while it computes on as many

// Logits that are read once leave no line in the first-level cache; KEEP (the row will be read again): nor do the others, but with that
// hint they also leave the second-level cache early (policy loss of 8192 rows of 65536 bf16: 402 us instead of 373).
template <bool KEEP>
__device__ __forceinline__ uint4 load16(const uint4 *p) {
    if (KEEP) return __ldg(p);
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// A thread's vectors of a row (v[0], v[THREADS], ...), kU at a time.
template <typename T, int THREADS>
struct Share {
    const uint4 *v;
    int count;
    __device__ __forceinline__ Share(const uint4 *vectors, int n, int tid) : v(vectors + tid), count((n - tid + THREADS - 1) / THREADS) {}
    __device__ __forceinline__ int batches() const { return (count + kU - 1) / kU; }
    // Vectors that do not exist come as -inf: no maximum.
    template <bool KEEP>
    __device__ __forceinline__ void load(int b, uint4 (&q)[kU]) const {
        const uint4 *p = v + (int64_t)b * (kU * THREADS);
        if ((b + 1) * kU <= count) {
#pragma unroll
            for (int u = 0; u < kU; ++u) q[u] = load16<KEEP>(p + u * THREADS);
        } else {
            const uint32_t none = Vec<T>::kNone;
#pragma unroll
            for (int u = 0; u < kU; ++u) q[u] = b * kU + u < count ? load16<KEEP>(p + u * THREADS) : make_uint4(none, none, none, none);
        }
    }
};

// Two batches of a share: one is computed on while the other one travels.
struct Batches {
    uint4 even[kU], odd[kU];
};

// A thread's first batches of a row in shared memory, for a gradient right behind the row's sum (N = 0: none).  own: the thread's place,
// which no other thread looks at.
template <int THREADS, int N>
struct Stash {
    uint4 *own;       // NULL where no gradient follows
    __device__ __forceinline__ void put(int b, const uint4 (&q)[kU]) const {
        if constexpr (N > 0) {
            if (own != nullptr && b < N) {
#pragma unroll
                for (int u = 0; u < kU; ++u) own[(b * kU + u) * THREADS] = q[u];
            }
        }
    }
    __device__ __forceinline__ bool get(int b, uint4 (&q)[kU]) const {
        if constexpr (N > 0) {
            if (b < N) {
#pragma unroll
                for (int u = 0; u < kU; ++u) q[u] = own[(b * kU + u) * THREADS];
                return true;
            }
        }
        return false;
    }
};

// Maximum and sum over a thread's share of a row.  The last batch stays in x.odd, the one before it in x.even, and of those before them
// the first ones in the stash.
template <typename T, int THREADS, bool KEEP, int N>
__device__ __forceinline__ void row_part(const Share<T, THREADS> &w, float k, Part &r, Batches &x, const Stash<THREADS, N> &stash) {
    const int n = w.batches();
    int b = n & 1;
    if (b) w.template load<KEEP>(0, x.odd);
    if (n > b) w.template load<KEEP>(b, x.even);
    if (b) {
        stash.put(0, x.odd);
        take<T, kU>(x.odd, k, r, w.count);          // where it is the only one, not all of it need be there
    }
    for (; b + 2 < n; b += 2) {
        w.template load<KEEP>(b + 1, x.odd);
        stash.put(b, x.even);
        take<T, kU>(x.even, k, r);
        w.template load<KEEP>(b + 2, x.even);
        stash.put(b + 1, x.odd);
        take<T, kU>(x.odd, k, r);
    }
    if (b < n) {
        w.template load<KEEP>(b + 1, x.odd);
        take<T, kU>(x.even, k, r);
        take<T, kU>(x.odd, k, r, w.count - (n - 1) * kU);
    }
}

// What row_part leaves, for a gradient that has no sum in front of it.
template <typename T, int THREADS>
__device__ __forceinline__ void last_batches(const Share<T, THREADS> &w, Batches &x) {
    const int n = w.batches();
    if (n > 0) w.template load<false>(n - 1, x.odd);
    if (n > 1) w.template load<false>(n - 2, x.even);
}

// The gradient over a thread's share of a row, into out[0], out[THREADS], ..., from the end to the start: the end is in registers, what is
// before it was read last, and the start is in the stash.  own = the number of the thread's vector that holds the target (at place `at`), or -1.  STREAM: the gradient
// is not to displace rows that are waiting for theirs in the second-level cache (381 us instead of 373 otherwise).
template <typename T, int THREADS, bool STREAM, int N>
__device__ __forceinline__ void row_gradient(const Share<T, THREADS> &w, Batches &x, const Stash<THREADS, N> &stash, uint4 *out, int own, int at, float k, float c, float neg, float g) {
    auto put = [&](int b, const uint4 (&q)[kU]) {
        uint4 *p = out + (int64_t)b * (kU * THREADS);
        const bool whole = (b + 1) * kU <= w.count;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (whole || b * kU + u < w.count) {
                const uint4 y = gradient_of<T, false>(q[u], b * kU + u == own ? at : -1, k, c, neg, g);
                if (STREAM) __stcs(p + u * THREADS, y);
                else p[u * THREADS] = y;
            }
        }
    };
    int b = w.batches() - 1;
    for (; b >= 1; b -= 2) {
        put(b, x.odd);
        if (b >= 2 && !stash.get(b - 2, x.odd)) w.template load<false>(b - 2, x.odd);
        put(b - 1, x.even);
        if (b >= 3 && !stash.get(b - 3, x.even)) w.template load<false>(b - 3, x.even);
    }
    if (b == 0) put(0, x.odd);
}

// The same for the wide way, and for logits that lie at another offset from the 16-byte boundaries than the gradient (their values are
// loaded one by one).
template <typename T, bool WIDE>
__device__ __forceinline__ void row_gradient_direct(const T *z, T *out, const Cut &l, int target, float k, float c, float neg, float g, int first, int step) {
    constexpr int N = Vec<T>::N, U = 2;
    const bool same = (reinterpret_cast<uintptr_t>(z) - reinterpret_cast<uintptr_t>(out)) % 16 == 0;
    const int at = target - l.head, own = at < 0 ? -1 : at / N;
    for (int i0 = first; i0 < l.vecs; i0 += step * U) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * step;
            if (i < l.vecs) {
                if (same) {
                    q[u] = __ldg(reinterpret_cast<const uint4 *>(z + l.head) + i);
                } else {
                    T x[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) x[e] = z[l.head + (int64_t)i * N + e];
                    memcpy(&q[u], x, 16);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * step;
            if (i < l.vecs) reinterpret_cast<uint4 *>(out + l.head)[i] = gradient_of<T, WIDE>(q[u], i == own ? at % N : -1, k, c, neg, g);
        }
    }
    gradient_loose<T, WIDE>(z, out, l, target, k, c, neg, g, first, step);
}

// Maximum and sum of 2^((z - maximum) k) over a thread's part of a row that takes the wide way.
template <typename T>
__device__ __forceinline__ void row_part_wide(const T *z, int V, int first, int step, float k, float &mx, float &sum) {
    mx = -FLT_MAX;
    sum = 0.f;
#pragma unroll 1
    for (int i = first; i < V; i += step) {
        const float x = Vec<T>::get1(z[i]), m = fmaxf(mx, x);
        sum = sum * ex2(apart(mx, m, k)) + ex2(apart(x, m, k));
        mx = m;
    }
}

// (c, sum) of a row from those of its threads, whose sums are of powers 2^(... - k c).  Every thread gets the same bits.
template <int THREADS, int TURN>
__device__ __forceinline__ void gather(float &c, float &sum, float k) {
    const float m = warp_max(c);
    sum = warp_sum(sum * ex2(apart(c, m, k)));
    c = m;
    if constexpr (THREADS != 32) {
        __shared__ float2 part[THREADS / 32];
        const int lane = threadIdx.x & 31;
        if (lane == 0) part[threadIdx.x >> 5] = make_float2(c, sum);
        __syncthreads();
        const float2 p = lane < THREADS / 32 ? part[lane] : make_float2(c, 0.f);
        c = warp_max(p.x);
        sum = warp_sum(p.y * ex2(apart(p.x, c, k)));
    }
}

template <typename T>
__device__ __forceinline__ void row_zero(T *g, const Cut &l, int first, int step) {
    for (int i = first; i < l.vecs; i += step) reinterpret_cast<uint4 *>(g + l.head)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = first; i < l.loose; i += step) g[l.at(i)] = Vec<T>::one(0.f);
}

template <typename T>
__device__ __forceinline__ const T *row_of(const Rows &a, int64_t row) {
    const uint32_t s = (uint32_t)row / (uint32_t)a.T, t = (uint32_t)row - s * (uint32_t)a.T;      // there are fewer than 2^31 rows
    return static_cast<const T *>(a.z) + s * a.seq_stride + t * a.row_stride;
}

// The row's target, or -1 where the row does not count.
__device__ __forceinline__ int target_of(const Rows &a, int64_t row) {
    const int64_t t = a.targets[row];
    const uint8_t counts = a.mask != nullptr ? a.mask[row] : 1;      // on its way together with the target
    return counts && t >= 0 && t < a.V ? (int)t : -1;
}

// What the policy loss takes beside the rows.
struct Policy {
    const float *advantages, *old_lp, *ref_lp;
    int64_t adv_seq, adv_row;      // strides of the advantages
    float low, high, kl, scale;
    int reduction;
    const int *counts;       // live rows of each part
    int parts;
    double *row_loss;        // of each block
    unsigned *done;
    float *loss;
};

// Rows of a part where tokens are counted over all sequences: at most 64 parts, which every row adds up.
__host__ __device__ constexpr int64_t count_rows(int64_t rows) { return rows > 64 * 1024 ? (rows + 63) / 64 : 1024; }
constexpr int kWarpRows = 8;

// The last block to draw a number behind its loss adds up all blocks', in an order that does not depend on which block that is.
// Thread 0 draws it while the gradient is still to be written.
__device__ __forceinline__ void draw_number(const Policy &q, bool &last) {
    __threadfence();
    last = atomicAdd(q.done, 1u) == gridDim.x - 1;
}
__device__ __forceinline__ void total_loss(const Policy &q, const bool &last) {
    __shared__ double part[32];
    __syncthreads();
    if (!last) return;
    __threadfence();
    double x = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += blockDim.x) x += __ldcg(q.row_loss + i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < (int)blockDim.x / 32; ++i) x += part[i];
        *q.loss = (float)x;
    }
}

constexpr int kRowThreads = 256;     // of a long row
__host__ __device__ constexpr int row_blocks(int threads) { return 1024 / (threads == 32 ? 32 * kWarpRows : threads); }   // per SM

// The policy loss of long rows keeps the first batches of a row in shared memory for the gradient: less is read from the L2 cache again,
// and less of the rows under way has to last there.  Two batches (32 KB a block) of four blocks per SM, in fp32, which has fewer
// instructions per byte to hide, three batches of three blocks: 6000 rows of 65536 bf16 281 us (287 without; 286 with three blocks of three
// batches; 320 with four, which leave the first-level cache too little for the loads under way), of 32768 fp32 261 us (291 without, 279
// with four blocks of two).  Rows of a warp or of 128 threads: nothing gained (16384 bf16: 97 us either way), short ones lose by it.
template <typename T, int THREADS, bool POLICY>
struct LongRows {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr int kStash = POLICY && THREADS == kRowThreads ? (kWide ? 3 : 2) : 0;
    static constexpr int kBlocks = kStash > 0 && kWide ? 3 : row_blocks(THREADS);
    static constexpr int kBytes = kStash * kU * 16 * THREADS;
};

// What a row's loss takes beside its log-probability, requested before the row.
struct Terms {
    float adv = 0.f, old = 0.f, ref = 0.f;
    int n = 0;
};
__device__ __forceinline__ Terms terms_of(const Rows &a, const Policy &q, int64_t row) {
    Terms t;
    const uint32_t s = (uint32_t)row / (uint32_t)a.T;
    t.adv = q.advantages[s * q.adv_seq + ((uint32_t)row - s * (uint32_t)a.T) * q.adv_row];
    t.old = q.old_lp[row];
    if (q.ref_lp != nullptr) t.ref = q.ref_lp[row];
    if (q.reduction == WKV6_MEAN)
        for (int i = threadIdx.x & 31; i < q.parts; i += 32) t.n += q.counts[i];
    else if (q.reduction == WKV6_SEQUENCE_MEAN)
        t.n = q.counts[s];
    return t;
}

// Loss of a row and its derivative by the row's log-probability.
__device__ __forceinline__ float2 loss_of(const Rows &a, const Policy &q, Terms t, float lp) {
    float w = q.scale;
    if (q.reduction == WKV6_MEAN) {
        t.n = __reduce_add_sync(0xffffffffu, t.n);
        w = q.scale / (float)t.n;
    } else if (q.reduction == WKV6_SEQUENCE_MEAN) {
        w = q.scale / ((float)t.n * (float)((uint32_t)a.rows / (uint32_t)a.T));
    }
    // comparisons written so that a NaN ratio is not clipped away
    const float rho = expf(lp - t.old), free = rho * t.adv;
    const float clipped = (rho < q.low ? q.low : rho > q.high ? q.high : rho) * t.adv;
    const bool open = !(free > clipped);
    float loss = open ? -free : -clipped, slope = open ? -free : 0.f;
    if (q.ref_lp != nullptr) {     // exp(d) - d - 1 is d^2 / 2 for small d: taken from exp(d) - 1
        const float d = t.ref - lp, e = expm1f(d);
        loss += q.kl * (e - d);
        slope -= q.kl * e;
    }
    return make_float2(loss * w, slope * w);
}

// A log-probability that rounding has lifted above 0; a NaN stays.
__device__ __forceinline__ float at_most_zero(float x) { return x > 0.f ? 0.f : x; }

// From the threads' parts of a row to its log-probability: r becomes the row's (c and sum), `wide` says how.
template <typename T, int THREADS>
__device__ __forceinline__ float finish_row(const Rows &a, const T *z, float zt, int tid, Part &r, bool &wide) {
    gather<THREADS, 0>(r.c, r.sum, 1.f);
    const float end = -__fmul_rn(a.low, a.k);      // 2^24; the same in all threads; a NaN in the sum stays what it is
    wide = !(r.c > -end && r.c < end);
    if (wide) {
        row_part_wide(z, a.V, tid, THREADS, a.k, r.c, r.sum);
        gather<THREADS, 1>(r.c, r.sum, a.k);
        return at_most_zero(apart(zt, r.c, a.inv_tau) - logf(r.sum));
    }
    const float below = fmaf(zt, a.k, -r.c);
    if (below == -INFINITY) return zt * a.inv_tau + (r.sum - r.sum);      // the type's lowest value: its product with log2(e) leaves fp32, the rest is lost in it
    // The logarithm's whole part is taken off first, which is exact or nearly so: only a part in [0, 1) is off by its rounding.  (r.sum is
    // at least about 2^(-1/2); the last term is 0, or NaN where the sum is.)
    const uint32_t bits = __float_as_uint(r.sum);
    const float whole = (float)((int)(bits >> 23) - 127), part = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
    return at_most_zero(((below - whole) - log2f(part)) * 0.69314718055994531f + (r.sum - r.sum));
}

// THREADS = 32: a warp per row, several to a block (rows of a few KB, where a block's reduction would cost more than its row);
// otherwise a block per row.  POLICY: the loss and, with g, the gradient behind the log-probabilities.
template <typename T, int THREADS, bool POLICY>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpRows : THREADS, LongRows<T, THREADS, POLICY>::kBlocks)
token_rows_kernel(const Rows a, float *__restrict__ lp_out, float2 *__restrict__ stat, const Policy q, float *__restrict__ coefficient,
                  T *__restrict__ g) {
    __shared__ bool last;
    __shared__ double of_warp[kWarpRows];
    const int tid = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = THREADS == 32 ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
    if (THREADS != 32 || row < a.rows) {
        const int target = target_of(a, row);
        const T *z = row_of<T>(a, row);
        const Cut l = cut_of(z, a.V);
        const Share<T, THREADS> share(reinterpret_cast<const uint4 *>(z + l.head), l.vecs, tid);
        float lp = 0.f, inv_sum = 0.f;
        float2 loss = make_float2(0.f, 0.f);
        Part r{a.low, __fmul_rn(a.low, a.k), 0.f};
        bool wide = false;
        Batches x;
        extern __shared__ uint4 stashed[];
        const Stash<THREADS, LongRows<T, THREADS, POLICY>::kStash> stash{g != nullptr ? stashed + tid : nullptr};
        Terms t;
        if constexpr (POLICY) t = terms_of(a, q, row);
        if (target >= 0) {
            const float zt = Vec<T>::get1(z[target]);
            row_part<T, THREADS, POLICY>(share, a.k, r, x, stash);
            take_loose(z, l, tid, THREADS, a.k, r);
            lp = finish_row<T, THREADS>(a, z, zt, tid, r, wide);
            inv_sum = 1.f / r.sum;
            if constexpr (POLICY) loss = loss_of(a, q, t, lp);
        }
        if (tid == 0) {
            lp_out[row] = lp;
            if (stat != nullptr) stat[row] = make_float2(r.c, wide ? -inv_sum : inv_sum);
            if constexpr (POLICY) {
                coefficient[row] = loss.y;
                if (THREADS != 32) {
                    q.row_loss[row] = loss.x;
                    draw_number(q, last);
                } else {
                    of_warp[threadIdx.x >> 5] = loss.x;
                }
            }
        }
        if constexpr (POLICY) {
            if (g != nullptr) {
                T *gr = g + row * a.V;
                const float gc = loss.y * a.inv_tau, neg = -gc * inv_sum;
                if (loss.y == 0.f) {                 // a NaN is not
                    row_zero(gr, cut_of(gr, a.V), tid, THREADS);
                } else if (wide) {
                    row_gradient_direct<T, true>(z, gr, cut_of(gr, a.V), target, a.k, r.c, neg, gc, tid, THREADS);
                } else if ((reinterpret_cast<uintptr_t>(z) - reinterpret_cast<uintptr_t>(gr)) % 16 == 0) {
                    const int at = target - l.head, vec = at / Vec<T>::N, own = at >= 0 && vec % THREADS == tid ? vec / THREADS : -1;
                    row_gradient<T, THREADS, true>(share, x, stash, reinterpret_cast<uint4 *>(gr + l.head) + tid, own, at % Vec<T>::N, a.k, r.c, neg, gc);
                    gradient_loose<T, false>(z, gr, l, target, a.k, r.c, neg, gc, tid, THREADS);
                } else {
                    row_gradient_direct<T, false>(z, gr, cut_of(gr, a.V), target, a.k, r.c, neg, gc, tid, THREADS);
                }
            }
        }
    }
    if constexpr (POLICY) {
        if constexpr (THREADS == 32) {
            __syncthreads();
            if (threadIdx.x == 0) {
                double x = 0.0;
                for (int i = 0; i < kWarpRows; ++i)
                    if (blockIdx.x * (int64_t)kWarpRows + i < a.rows) x += of_warp[i];
                q.row_loss[blockIdx.x] = x;
                draw_number(q, last);
            }
        }
        total_loss(q, last);
    }
}

// Gradient of the logits from the rows' statistics and one coefficient per row, or per sequence:
//   g = coefficient (*factor) (1[j = a] - p_j) / tau
// A block takes a part of a row (blockIdx.y), so that few long rows fill the GPU too.  `unless_one`: nothing is done where *factor
// is 1 (the gradient is there already).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpRows : THREADS, row_blocks(THREADS))
token_gradient_kernel(const Rows a, const float2 *__restrict__ stat, const float *__restrict__ coefficient, int per_sequence,
                      const float *__restrict__ factor, int unless_one, T *__restrict__ g) {
    const int64_t row = THREADS == 32 ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    // everything small is requested at once
    const float f = factor != nullptr ? *factor : 1.f, per_row = coefficient[per_sequence ? (uint32_t)row / (uint32_t)a.T : row];
    const float2 s = stat[row];
    const int target = target_of(a, row);
    if (unless_one && f == 1.f) return;
    const int tid = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x, first = blockIdx.y * THREADS + tid, step = THREADS * gridDim.y;
    const float gc = target < 0 ? 0.f : per_row * f * a.inv_tau;
    const T *z = row_of<T>(a, row);
    T *gr = g + row * a.V;
    const Cut l = cut_of(gr, a.V);
    if (gc == 0.f) {
        row_zero(gr, l, first, step);
        return;
    }
    if (signbit(s.y)) {
        row_gradient_direct<T, true>(z, gr, l, target, a.k, s.x, gc * s.y, gc, first, step);
    } else if ((reinterpret_cast<uintptr_t>(z) - reinterpret_cast<uintptr_t>(gr)) % 16 == 0) {
        const int each = (l.vecs + gridDim.y - 1) / gridDim.y, begin = each * blockIdx.y, n = min(each, l.vecs - begin);
        if (n > 0) {
            const int at = target - l.head, vec = at / Vec<T>::N - begin;
            const int own = at >= 0 && vec >= 0 && vec < n && vec % THREADS == tid ? vec / THREADS : -1;
            const Share<T, THREADS> share(reinterpret_cast<const uint4 *>(z + l.head) + begin, n, tid);
            Batches x;
            last_batches(share, x);
            row_gradient<T, THREADS, false>(share, x, Stash<THREADS, 0>{nullptr}, reinterpret_cast<uint4 *>(gr + l.head) + begin + tid, own, at % Vec<T>::N, a.k, s.x, -gc * s.y, gc);
        }
        gradient_loose<T, false>(z, gr, l, target, a.k, s.x, -gc * s.y, gc, first, step);
    } else {
        row_gradient_direct<T, false>(z, gr, l, target, a.k, s.x, -gc * s.y, gc, first, step);
    }
}

// Live rows of every part: a sequence, or count_rows() rows of the whole where only their total is wanted.
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

// What the preference loss takes beside the rows.
struct Pairs {
    const float *lp, *ref;
    double beta, smoothing, margin, scale;
    int S, average;
    float *seq;          // log-probability of every sequence
    double *seq64;
    int *count;          // of its live rows
    float *coefficient, *loss;
};

// Log-probability of a sequence: its live rows' sum (in 64 bits: thousands of terms, of which only the difference to a
// reference matters) or mean, by WARPS warps.
template <int WARPS>
__device__ __forceinline__ void sum_sequence(const Rows &a, const Pairs &q, int s) {
    constexpr int THREADS = WARPS * 32, U = 8;
    const int64_t first = (int64_t)s * a.T;
    const int lane = threadIdx.x & 31, tid = WARPS == 1 ? lane : threadIdx.x;
    double x = 0.0;
    int n = 0;
    for (int64_t i0 = tid; i0 < a.T; i0 += THREADS * U) {
        float lp[U];
        int target[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {      // requested together: those behind the end ask for the last one again
            const int64_t at = i0 + u * THREADS, i = at < a.T ? at : a.T - 1;
            lp[u] = q.lp[first + i];
            target[u] = target_of(a, first + i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool live = target[u] >= 0 && i0 + u * THREADS < a.T;
            x += live ? (double)lp[u] : 0.0;
            n += live;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    n = __reduce_add_sync(0xffffffffu, n);
    if constexpr (WARPS > 1) {
        __shared__ double part[WARPS];
        __shared__ int live[WARPS];
        if (lane == 0) {
            part[threadIdx.x >> 5] = x;
            live[threadIdx.x >> 5] = n;
        }
        __syncthreads();
        if (threadIdx.x == 0)
            for (int i = 1; i < WARPS; ++i) {
                x += part[i];
                n += live[i];
            }
    }
    if (tid == 0) {
        if (q.average && n > 1) x /= n;
        q.seq64[s] = x;
        q.seq[s] = (float)x;
        q.count[s] = n;
    }
}

// One block: margin, loss and slope of every pair, their mean in a fixed order.
constexpr int kPairThreads = 256;
__device__ __forceinline__ void all_pairs(const Pairs &q) {
    __shared__ double part[kPairThreads / 32];
    const int pairs = q.S / 2;
    double total = 0.0;
    if (threadIdx.x < kPairThreads) {
        for (int i = threadIdx.x; i < pairs; i += kPairThreads) {
            const int j = i + pairs;
            double over = q.seq64[i] - q.seq64[j];
            if (q.ref != nullptr) over -= (double)q.ref[i] - (double)q.ref[j];
            const double d = q.beta * over - q.margin, tail = log1p(exp(-fabs(d)));
            total += (1.0 - q.smoothing) * (tail + fmax(-d, 0.0));           // a NaN reaches the sum through the tail
            if (q.smoothing != 0.0) total += q.smoothing * (tail + fmax(d, 0.0));
            const double slope = -q.beta * (1.0 - q.smoothing - 1.0 / (1.0 + exp(-d))) * (q.scale / pairs);
            q.coefficient[i] = (float)(slope / (q.average && q.count[i] > 1 ? q.count[i] : 1));
            q.coefficient[j] = (float)(-slope / (q.average && q.count[j] > 1 ? q.count[j] : 1));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kPairThreads / 32; ++i) total += part[i];
        *q.loss = (float)(total * (q.scale / pairs));
    }
}

// Few tokens: everything in one block, a warp per sequence, which saves a launch (3 us of the host).
constexpr int kOneBlock = 1024;
__global__ void __launch_bounds__(kOneBlock) preference_kernel(const Rows a, const Pairs q) {
    for (int s = threadIdx.x >> 5; s < q.S; s += kOneBlock / 32) sum_sequence<1>(a, q, s);
    __syncthreads();
    all_pairs(q);
}

// Many tokens: a block per sequence, then the pairs.
__global__ void __launch_bounds__(256) sequence_sum_kernel(const Rows a, const Pairs q) { sum_sequence<8>(a, q, blockIdx.x); }
__global__ void __launch_bounds__(kPairThreads) preference_pairs_kernel(const Pairs q) { all_pairs(q); }

// Threads of a row by the bytes of its logits.  A warp saves the block's barriers: up to 16 KB forward (100 M bf16 logits in rows of 8192:
// policy loss 103 us, 116 with 128 threads; in rows of 12000: 108 and 105), up to 8 KB for the gradient alone (rows of 4096: 69 and 77 us; of
// 8192: 71 and 65) - where there are rows enough for 32 warps on every SM, otherwise up to 4 KB.  128 threads up to 32 KB (rows of 16384:
// 100 us, 107 with 256; of 32768: 97 and 95).
int row_threads(const wkv6_token_logits *p, bool gradient) {
    const int64_t n = (int64_t)p->V * (int64_t)dtype_size(p->dtype), rows = (int64_t)p->S * p->T;
    const int64_t warp = rows < 32 * (int64_t)sm_count() ? 4096 : gradient ? 8192 : 16384;
    return n <= warp ? 32 : n <= 32768 ? 128 : kRowThreads;
}

// f(std::integral_constant<int, THREADS>, T *) for the call's type and row size
template <typename F>
int dispatch(const wkv6_token_logits *p, bool gradient, F f) {
    const int threads = row_threads(p, gradient);
    auto typed = [&](auto *t) {
        if (threads == 32) return f(std::integral_constant<int, 32>{}, t);
        if (threads == 128) return f(std::integral_constant<int, 128>{}, t);
        return f(std::integral_constant<int, kRowThreads>{}, t);
    };
    if (p->dtype == WKV6_BF16) return typed(static_cast<__nv_bfloat16 *>(nullptr));
    if (p->dtype == WKV6_F16) return typed(static_cast<__half *>(nullptr));
    return typed(static_cast<float *>(nullptr));
}

int rows_of(const wkv6_token_logits *p, Rows *a, const char *what, bool need_logits) {
    if (p == nullptr) return fail(WKV6_ERR_INVALID, "%s: NULL argument", what);
    if (p->S < 0 || p->T < 0 || p->V < 1) return fail(WKV6_ERR_INVALID, "%s: S=%d T=%d V=%d", what, p->S, p->T, p->V);
    if (p->dtype != WKV6_BF16 && p->dtype != WKV6_F16 && p->dtype != WKV6_F32) return fail(WKV6_ERR_INVALID, "%s: unknown dtype code", what);
    if (!(p->temperature >= 1e-30f) || std::isinf(p->temperature)) return fail(WKV6_ERR_INVALID, "%s: temperature must be at least 1e-30 and finite", what);
    a->rows = (int64_t)p->S * p->T;
    if (a->rows > 2147483647LL) return fail(WKV6_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", what);
    if (p->V > 1 << 30) return fail(WKV6_ERR_UNSUPPORTED, "%s: V=%d, at most 2^30", what, p->V);
    a->T = p->T;
    a->V = p->V;
    a->row_stride = p->row_stride ? p->row_stride : p->V;
    a->seq_stride = p->seq_stride ? p->seq_stride : p->T * a->row_stride;
    if (a->row_stride < 0 || a->seq_stride < 0) return fail(WKV6_ERR_INVALID, "%s: negative strides", what);
    if (a->rows > 0 && ((need_logits && p->logits == nullptr) || p->targets == nullptr)) return fail(WKV6_ERR_INVALID, "%s: NULL argument", what);
    if (reinterpret_cast<uintptr_t>(p->logits) % dtype_size(p->dtype)) return fail(WKV6_ERR_INVALID, "%s: misaligned logits", what);
    if (!aligned(8, {p->targets})) return fail(WKV6_ERR_INVALID, "%s: misaligned targets", what);
    a->z = p->logits;
    a->targets = p->targets;
    a->mask = p->mask;
    a->k = (float)(1.4426950408889634 / (double)p->temperature);
    a->inv_tau = (float)(1.0 / (double)p->temperature);
    a->low = -(float)std::min(16777216.0 / (double)a->k, (double)FLT_MAX / 4.0);      // |c| < 2^24, see the top; no infinity for a tiny k
    return WKV6_OK;
}

template <bool POLICY>
int launch_rows(const wkv6_token_logits *p, const Rows &a, float *lp, float2 *stat, const Policy &q, float *coefficient, void *g,
                cudaStream_t st) {
    return dispatch(p, false, [&](auto size, auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int threads = size.value;
        const unsigned grid = (unsigned)(threads == 32 ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows);
        const auto kernel = token_rows_kernel<T, threads, POLICY>;
        const int stash = g != nullptr ? LongRows<T, threads, POLICY>::kBytes : 0;
        if (stash >= 47 * 1024)      // with what the kernel declares, more than a launch may have unasked
            if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, stash); e != cudaSuccess)
                return cuda_fail(e, "cudaFuncSetAttribute");
        kernel<<<grid, threads == 32 ? 32 * kWarpRows : threads, stash, st>>>(a, lp, stat, q, coefficient, static_cast<T *>(g));
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? (int)WKV6_OK : cuda_fail(e, "token_rows_kernel launch");
    });
}

int64_t count_parts(int64_t S, int64_t T, int reduction) {
    return reduction == WKV6_SEQUENCE_MEAN ? S : (S * T + count_rows(S * T) - 1) / count_rows(S * T);
}

}  // namespace

}  // namespace wkv6

using namespace wkv6;

extern "C" int wkv6_token_log_probs(const wkv6_token_logits *p, float *log_probs, float *stat, void *stream) {
    Rows a;
    if (const int rc = rows_of(p, &a, "wkv6_token_log_probs", true)) return rc;
    if (a.rows == 0) return WKV6_OK;
    if (log_probs == nullptr) return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs: NULL argument");
    if (!aligned(8, {stat}) || !aligned(4, {log_probs})) return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs: stat must be 8-byte aligned, log_probs 4-byte");
    return launch_rows<false>(p, a, log_probs, reinterpret_cast<float2 *>(stat), Policy{}, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int wkv6_token_log_probs_backward(const wkv6_token_logits *p, const float *stat, const float *coefficient, int32_t per_sequence,
                                             const float *factor, int32_t unless_one, void *g, void *stream) {
    Rows a;
    if (const int rc = rows_of(p, &a, "wkv6_token_log_probs_backward", true)) return rc;
    if (a.rows == 0) return WKV6_OK;
    if (!stat || !coefficient || !g || (unless_one && !factor)) return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs_backward: NULL argument");
    if (!aligned16(g) || !aligned(8, {stat}) || !aligned(4, {coefficient, factor}))
        return fail(WKV6_ERR_INVALID, "wkv6_token_log_probs_backward: the gradient must be 16-byte aligned, stat 8-byte, other values 4-byte");
    return dispatch(p, true, [&](auto size, auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int threads = size.value;
        // parts of at least one stage, as many as it takes to give every SM its blocks
        const int64_t want = ((int64_t)row_blocks(threads) * sm_count() + a.rows - 1) / a.rows;
        const int64_t most = (int64_t)p->V * (int64_t)sizeof(T) / (threads * kU * 16) + 1;
        const dim3 grid((unsigned)(threads == 32 ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows), (unsigned)(threads == 32 ? 1 : want < most ? want : most));
        token_gradient_kernel<T, threads><<<grid, threads == 32 ? 32 * kWarpRows : threads, 0, static_cast<cudaStream_t>(stream)>>>(
            a, reinterpret_cast<const float2 *>(stat), coefficient, per_sequence, factor, unless_one, static_cast<T *>(g));
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? (int)WKV6_OK : cuda_fail(e, "token_gradient_kernel launch");
    });
}

extern "C" uint64_t wkv6_capture_id(void *stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id) != cudaSuccess) {
        cudaGetLastError();      // the legacy stream next to a capture: it is not part of it
        return 0;
    }
    return status == cudaStreamCaptureStatusNone ? 0 : id;
}

extern "C" size_t wkv6_policy_loss_workspace_bytes(int32_t S, int32_t T, int32_t reduction) {
    if (S <= 0 || T <= 0) return 0;
    return 16 + (size_t)((int64_t)S * T) * 8 + (size_t)count_parts(S, T, reduction) * 4;
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
    if (!aligned16(g) || !aligned(8, {stat}) || !aligned16(workspace) ||
        !aligned(4, {loss, log_probs, coefficient, c->advantages, c->old_log_probs, c->ref_log_probs}))
        return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: the gradient and the workspace must be 16-byte aligned, stat 8-byte, other values 4-byte");
    if (workspace_bytes < wkv6_policy_loss_workspace_bytes(p->S, p->T, c->reduction))
        return fail(WKV6_ERR_WORKSPACE, "wkv6_policy_loss: workspace of %zu bytes, %zu are needed", workspace_bytes,
                    wkv6_policy_loss_workspace_bytes(p->S, p->T, c->reduction));
    Policy q{};
    if (c->advantage_seq_stride < 0 || c->advantage_row_stride < 0) return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: negative strides");
    q.advantages = c->advantages;
    q.adv_seq = c->advantage_seq_stride;
    q.adv_row = c->advantage_row_stride;
    q.old_lp = c->old_log_probs;
    q.ref_lp = c->kl_coef != 0.0 ? c->ref_log_probs : nullptr;
    if (c->kl_coef != 0.0 && c->ref_log_probs == nullptr) return fail(WKV6_ERR_INVALID, "wkv6_policy_loss: a KL term needs ref_log_probs");
    q.low = (float)(1.0 - c->clip_low);
    q.high = (float)(1.0 + c->clip_high);
    q.kl = (float)c->kl_coef;
    q.scale = (float)c->scale;
    q.reduction = c->reduction;
    q.done = static_cast<unsigned *>(workspace);
    q.row_loss = reinterpret_cast<double *>(static_cast<char *>(workspace) + 16);
    int *counts = reinterpret_cast<int *>(q.row_loss + a.rows);
    q.counts = counts;
    q.parts = (int)count_parts(p->S, p->T, c->reduction);
    q.loss = loss;
    count_rows_kernel<<<q.parts, 256, 0, st>>>(a, c->reduction == WKV6_SEQUENCE_MEAN ? p->T : count_rows(a.rows), counts, q.done);
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
    if (!aligned(8, {workspace}) || !aligned(4, {log_probs, c->ref_log_probs, loss, sequence_log_probs, coefficient}))
        return fail(WKV6_ERR_INVALID, "wkv6_preference_loss: the workspace must be 8-byte aligned, other values 4-byte");
    if (workspace_bytes < wkv6_preference_loss_workspace_bytes(p->S))
        return fail(WKV6_ERR_WORKSPACE, "wkv6_preference_loss: workspace of %zu bytes, %zu are needed", workspace_bytes,
                    wkv6_preference_loss_workspace_bytes(p->S));
    Pairs q{};
    q.lp = log_probs;
    q.ref = c->ref_log_probs;
    q.beta = c->beta;
    q.smoothing = c->label_smoothing;
    q.margin = c->margin;
    q.scale = c->scale;
    q.S = p->S;
    q.average = c->average;
    q.seq = sequence_log_probs;
    q.seq64 = static_cast<double *>(workspace);
    q.count = reinterpret_cast<int *>(q.seq64 + p->S);
    q.coefficient = coefficient;
    q.loss = loss;
    // One block against two launches.  A training call of few rows' bytes is bound by the host, which the second launch costs 2 us: forward and
    // gradient of 32 x 700 tokens, V = 259, 62.7 us and 64.6, 32 x 1024 62.7 and 64.3, 2 x 65 62.7 and 64.0.  What the rule gives up is device
    // time where the host waits or a graph is replayed: 32 x 700 33.1 us and 29.9, 8 x 1024 18.0 and 16.1, 32 x 1024 45.4 and 40.7, while up to
    // 4096 tokens there is nothing to give up (8 x 512 12.9 and 12.9, 32 x 128 12.9 and 12.7, 2 x 65 of 65536 bf16 16.6 and 17.4).
    if (p->S <= 32 && p->T <= 1024) {
        preference_kernel<<<1, kOneBlock, 0, st>>>(a, q);
    } else {
        sequence_sum_kernel<<<p->S, 256, 0, st>>>(a, q);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "sequence_sum_kernel launch");
        preference_pairs_kernel<<<1, kPairThreads, 0, st>>>(q);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? WKV6_OK : cuda_fail(e, "preference_pairs_kernel launch");
}
