// AdamW over many tensors at once (include/wkv6_b200.h gives the formulas), states in fp32 or in blocks of 256 e4m3 codes with a scale.
//
// A bf16 value with fp32 states moves 22 bytes, with 8-bit states 10.06.  The first is bound by HBM: 379 M values (two layers, embedding
// and head of the 1.6B shape) in 1328 us, 96 % of the copy bandwidth.  The second is bound by instructions: 896 us, 65 % of it, at 64.6
// instructions per value (at the copy bandwidth there is time for 55): random bits, two square roots' and two conversions' worth of
// work per value, and moments that keep the bits of elementary operations.
// The tensors of a model differ in size by four orders of magnitude, so they are cut into chunks and the blocks of one launch share all
// chunks; a chunk's tensor is found in a table that travels in the launch's arguments (no copy to the device, nothing to
// keep alive, and a captured launch holds its own).  A thread has eight neighbouring values, a warp the 256 of a block of codes, whose
// largest value is one warp reduction.  The next chunk's values are requested before this one's are computed.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "wkv6_internal.h"

namespace wkv6 {

namespace {

// Two blocks per SM: with the next chunk's values in registers a thread needs 112 to 118 of them.  Measured for 379 M bf16 values: fp32
// states 1328 us (three blocks 1519, four 1602); 8 bits 896 us with 16 values per thread and chunk (eight: 1017; not requested ahead: 983).
constexpr int kThreads = 256, kPerThread = 8, kGroupValues = kThreads * kPerThread, kBlock = 256, kBlocksPerSm = 2;
__host__ __device__ constexpr int groups(int bits) { return bits == 8 ? 2 : 1; }     // of eight values per thread and chunk

struct Entry {
    void *p;
    const void *g;
    void *m, *v;
    float *m_scale, *v_scale;
    int64_t n;
    uint32_t index;
    uint32_t first_chunk;     // of the launch
};

// Arguments of one launch: up to 32764 bytes.
template <int CAP>
struct Table {
    Entry e[CAP];
    int count;
    uint32_t chunks;
    uint32_t seed_key;
    int64_t step;
    const int64_t *step_device;
    const float *lr_device, *grad_scale;
    double lr, beta1, beta2, eps, weight_decay;
    float step_size, inv_root2;    // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), where both are known to the host
};

// A bijection of 32-bit words that stirs their bits (multipliers: the fractional parts of the square roots of 2 and 3).
__host__ __device__ __forceinline__ uint32_t stir(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// beta^t in double by squaring: 1 - beta^t loses nothing for beta near 1.
__host__ __device__ inline double power(double beta, int64_t t) {
    double r = 1.0;
    for (; t > 0; t >>= 1, beta *= beta)
        if (t & 1) r *= beta;
    return r;
}

// Products and sums of the moments are rounded one by one, so that they have the bits of the formulas' elementary operations: a
// moment in 8 bits that lies next to a border then never falls on its other side, and the scales of blocks do not drift apart from
// those of another implementation.  (In pairs, mul.rn.f32x2 and add.rn.f32x2, ptxas contracts them into multiply-adds all the same,
// and the moves that form the pairs cost what they save.)
__device__ __forceinline__ float blend(float old, float keep, float add, float share) { return __fadd_rn(__fmul_rn(old, keep), __fmul_rn(add, share)); }

__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float root_near(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The square root rounded to nearest, for x >= 2^-100: Newton's step on the residual x - s^2, which a fused multiply-add gives
// exactly (P. Markstein, IBM J. Res. Dev. 34, 1990).  Compared with sqrtf for all 2^24 values in [1, 4): no difference.
__device__ __forceinline__ float root_exact(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    const float s = __fmul_rn(x, y);
    return __fmaf_rn(__fmaf_rn(-s, s, x), __fmul_rn(y, 0.5f), s);
}

// Largest and smallest of three; a NaN among them stays.
__device__ __forceinline__ float largest(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ float smallest(float a, float b, float c) {
    float y;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

using Eight = float[8];

__device__ __forceinline__ float largest(const Eight &f) {
    return largest(largest(f[0], f[1], f[2]), largest(f[3], f[4], f[5]), largest(f[6], f[7], f[7]));
}

__device__ __forceinline__ float smallest(const Eight &f) {
    return smallest(smallest(f[0], f[1], f[2]), smallest(f[3], f[4], f[5]), smallest(f[6], f[7], f[7]));
}

// Eight neighbouring values as they lie in memory.
template <typename T>
struct Raw {
    uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw<T> load8(const T *p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}

__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16> &r, Eight &f) {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ void unpack(const Raw<float> &r, Eight &f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(r.w[i].x);
        f[4 * i + 1] = __uint_as_float(r.w[i].y);
        f[4 * i + 2] = __uint_as_float(r.w[i].z);
        f[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
}

__device__ __forceinline__ void store8(float *p, const Eight &f) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// What eight values of a tensor need from memory.
template <typename T, int BITS>
struct Group {
    Raw<T> p, g;
    Raw<float> m, v;
};
template <typename T>
struct Group<T, 8> {
    Raw<T> p, g;
    uint2 m, v;
    float m_scale, v_scale;
};

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }

// fp32 to bf16 (in the upper half of the word): 16 random bits are added below the last kept one, which carries into it with the
// probability that keeps the mean.  x must not be a NaN: the sum would carry it into the sign.
__device__ __forceinline__ uint32_t up_or_down(float x, uint32_t random) { return __float_as_uint(x) + ((random ^ (random >> 16)) & 0xffffu); }

// q >= 0 in units of the block's scale onto the e4m3 grid in the same way; never from above zero to zero, which would divide the next
// update by eps alone.
__device__ __forceinline__ float grid_normal(float q, uint32_t random) {
    return __uint_as_float(((random >> 16) * 16u + __float_as_uint(q)) & 0xfff00000u);
}
__device__ __forceinline__ float grid_any(float q, uint32_t random) {
    const float tiny = fmaxf(floorf(fmaf(q, 512.f, (float)(random >> 16) * 0x1p-16f)), 1.f) * (1.f / 512.f);
    return q >= 0x1p-6f ? grid_normal(q, random) : q > 0.f ? tiny : 0.f;
}

__device__ __forceinline__ void decode8(uint2 codes, float scale, Eight &f) {
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        __half2 h[2];
        uint32_t *u = reinterpret_cast<uint32_t *>(h);
        asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(u[0]), "=r"(u[1]) : "r"(w[i]));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 x = __half22float2(h[j]);
            f[4 * i + 2 * j] = __fmul_rn(x.x, scale);
            f[4 * i + 2 * j + 1] = __fmul_rn(x.y, scale);
        }
    }
}

__device__ __forceinline__ uint2 encode8(const Eight &f) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        asm("{\n.reg .b16 a, b;\ncvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\nmov.b32 %0, {a, b};\n}"
            : "=r"(w[i]) : "f"(f[4 * i]), "f"(f[4 * i + 1]), "f"(f[4 * i + 2]), "f"(f[4 * i + 3]));
    return make_uint2(w[0], w[1]);
}

// Largest magnitude of the warp's 256 values, compared as bits: a NaN is larger than all others and stays.
__device__ __forceinline__ float block_top(float top) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu));
}

// A block's scale and the factor onto multiples of it.  Blocks below 2^-100 are zeros: their scale would leave the normal numbers.
__device__ __forceinline__ float2 block_scale(float top) {
    if (top < 0x1p-100f) top = 0.f;
    return make_float2(top * (1.f / 448.f), top > 0.f ? __frcp_rn(top) * 448.f : 0.f);
}

template <typename T, int BITS, bool STOCHASTIC, int CAP>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) adamw_kernel(const __grid_constant__ Table<CAP> a) {
    constexpr int G = groups(BITS);
    __shared__ float shared[2];
    float step_size = a.step_size, inv_root2 = a.inv_root2;
    float decay = (float)(1.0 - a.lr * a.weight_decay);
    int64_t t = a.step;
    if (a.step_device != nullptr || a.lr_device != nullptr) {
        const double lr = a.lr_device != nullptr ? (double)*a.lr_device : a.lr;
        if (a.step_device != nullptr) t = max((long long)*a.step_device, 1ll);
        if (threadIdx.x == 0) {
            shared[0] = (float)(lr / (1.0 - power(a.beta1, t)));
            shared[1] = (float)(1.0 / sqrt(1.0 - power(a.beta2, t)));
        }
        __syncthreads();
        step_size = shared[0];
        inv_root2 = shared[1];
        decay = (float)(1.0 - lr * a.weight_decay);
    }
    const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2), eps = (float)a.eps;
    const bool scaled = a.grad_scale != nullptr;
    const float gs = scaled ? *a.grad_scale : 1.f;
    const uint32_t step_key = stir((uint32_t)t ^ a.seed_key);
    const int lane = threadIdx.x & 31;

    // a contiguous range of chunks: its first tensor by bisection, the next ones are the neighbours
    uint32_t chunk = (uint32_t)((uint64_t)a.chunks * blockIdx.x / gridDim.x);
    const uint32_t chunk_end = (uint32_t)((uint64_t)a.chunks * (blockIdx.x + 1) / gridDim.x);
    int at = 0;
    for (int bound = a.count; bound - at > 1;) {
        const int mid = (at + bound) >> 1;
        if (a.e[mid].first_chunk <= chunk) at = mid; else bound = mid;
    }
    // this thread's first value of a chunk; `whole`: the chunk can be moved as vectors
    struct Place {
        int k;
        int64_t i;
        bool whole;
    };
    auto locate = [&]() {
        while (at + 1 < a.count && a.e[at + 1].first_chunk <= chunk) ++at;
        const Entry &e = a.e[at];
        const int64_t start = (int64_t)(chunk - e.first_chunk) * (G * kGroupValues);
        const bool aligned = ((reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g)) & 15) == 0 &&
                             ((reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v)) & (BITS == 32 ? 15 : 7)) == 0;
        return Place{at, start + threadIdx.x * kPerThread, aligned && start + G * kGroupValues <= e.n};
    };
    auto fetch = [&](const Entry &e, int64_t i, Group<T, BITS> &d) {
        d.p = load8(static_cast<const T *>(e.p) + i);
        d.g = load8(static_cast<const T *>(e.g) + i);
        if constexpr (BITS == 32) {
            d.m = load8(static_cast<const float *>(e.m) + i);
            d.v = load8(static_cast<const float *>(e.v) + i);
        } else {
            d.m = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(e.m) + i);
            d.v = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(e.v) + i);
            d.m_scale = e.m_scale[(uint64_t)i / kBlock];
            d.v_scale = e.v_scale[(uint64_t)i / kBlock];
        }
    };
    // The step of eight values: x, m, v in, x, m and v (8 bits: codes) out; random: what rounds them (see stir()).
    auto update = [&](const Entry &e, int64_t i, Eight &x, Eight &g, Eight &m, Eight &v, uint32_t (&random)[8], uint2 &mc, uint2 &vc) {
        Eight r;
        if (scaled) {
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = __fmul_rn(g[j], gs);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (BITS == 8) v[j] = __fmul_rn(v[j], v[j]);
            m[j] = blend(m[j], b1, g[j], c1);
            v[j] = blend(v[j], b2, __fmul_rn(g[j], g[j]), c2);
            r[j] = BITS == 8 ? root_exact(v[j]) : root_near(v[j]);
        }
        if constexpr (STOCHASTIC || BITS == 8) {
            // stir(i ^ key) but for its last step, which is left to each use; eight neighbours differ in three bits of the first word
            const uint32_t high = (uint32_t)((uint64_t)i >> 32), key = stir(e.index ^ step_key);
            uint32_t word = (uint32_t)i ^ (high ? stir(key + high) : key);
            word ^= word >> 16;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t w = (word ^ j) * 0x6A09E667u;
                w ^= w >> 15;
                random[j] = w * 0xBB67AE85u;
            }
        }
        if constexpr (BITS == 8) {
            const float2 ms = block_scale(block_top(largest(largest(m), -smallest(m), 0.f)));
            float2 vs = block_scale(block_top(largest(r)));
            Eight q;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(r[j], vs.y);
            // Rare: a value whose code is below the normal ones (under 1 / 28672 of its block's largest), zeros, or roots of values under
            // 2^-100.  One test for the warp; a NaN fails it.
            if (__all_sync(0xffffffffu, smallest(q) >= 0x1p-6f && vs.x >= 0x1p-40f)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = grid_normal(q[j], random[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j] = __fsqrt_rn(v[j]);
                vs = block_scale(block_top(largest(r)));
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = grid_any(__fmul_rn(r[j], vs.y), random[j]);
            }
            vc = encode8(q);
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(m[j], ms.y);
            mc = encode8(q);
            if (lane == 0) {
                e.m_scale[(uint64_t)i / kBlock] = ms.x;
                e.v_scale[(uint64_t)i / kBlock] = vs.x;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(m[j] * -step_size, reciprocal(fmaf(r[j], inv_root2, eps)), x[j] * decay);
    };

    // the next chunk's values travel while this one's are computed
    Place next{};
    Group<T, BITS> ahead[G];
    auto advance = [&]() {
        next = locate();
        if (next.whole) {
#pragma unroll
            for (int u = 0; u < G; ++u) fetch(a.e[next.k], next.i + u * kGroupValues, ahead[u]);
        }
    };
    if (chunk < chunk_end) advance();
    while (chunk < chunk_end) {
        const Place now = next;
        Group<T, BITS> d[G];
#pragma unroll
        for (int u = 0; u < G; ++u) d[u] = ahead[u];
        if (++chunk < chunk_end) advance();
        const Entry &e = a.e[now.k];
        if (now.whole) {
#pragma unroll
            for (int u = 0; u < G; ++u) {
                const int64_t i = now.i + u * kGroupValues;
                Eight x, g, m, v;
                uint32_t random[8];
                uint2 mc, vc;
                unpack(d[u].p, x);
                unpack(d[u].g, g);
                if constexpr (BITS == 32) {
                    unpack(d[u].m, m);
                    unpack(d[u].v, v);
                } else {
                    decode8(d[u].m, d[u].m_scale, m);
                    decode8(d[u].v, d[u].v_scale, v);
                }
                update(e, i, x, g, m, v, random, mc, vc);
                if constexpr (sizeof(T) == 2) {
                    uint32_t w[4];
                    const float most = largest(x);
                    if (STOCHASTIC && most == most) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = __byte_perm(up_or_down(x[2 * j], random[2 * j]), up_or_down(x[2 * j + 1], random[2 * j + 1]), 0x7632);
                    } else {               // to nearest; or a NaN among the values
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
                            w[j] = *reinterpret_cast<const uint32_t *>(&h);
                            if (STOCHASTIC) {
                                if (x[2 * j] == x[2 * j]) w[j] = __byte_perm(up_or_down(x[2 * j], random[2 * j]), w[j], 0x7632);
                                if (x[2 * j + 1] == x[2 * j + 1]) w[j] = __byte_perm(w[j], up_or_down(x[2 * j + 1], random[2 * j + 1]), 0x7610);
                            }
                        }
                    }
                    *reinterpret_cast<uint4 *>(static_cast<T *>(e.p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    store8(static_cast<float *>(e.p) + i, x);
                }
                if constexpr (BITS == 32) {
                    store8(static_cast<float *>(e.m) + i, m);
                    store8(static_cast<float *>(e.v) + i, v);
                } else {
                    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(e.m) + i) = mc;
                    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(e.v) + i) = vc;
                }
            }
            continue;
        }
        // the end of a tensor, or one that does not start at a vector's boundary: value by value
#pragma unroll 1
        for (int u = 0; u < G; ++u) {
            const int64_t i = now.i + u * kGroupValues, n = e.n;
            if (i - lane * kPerThread >= n) break;             // the warp as a whole
            const int have = i + kPerThread <= n ? kPerThread : i < n ? (int)(n - i) : 0;
            T *p = static_cast<T *>(e.p);
            const T *gp = static_cast<const T *>(e.g);
            Eight x, g, m, v;
            uint32_t random[8];
            uint2 mc = make_uint2(0u, 0u), vc = make_uint2(0u, 0u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = j < have;
                x[j] = in ? value(p[i + j]) : 0.f;
                g[j] = in ? value(gp[i + j]) : 0.f;
                if constexpr (BITS == 32) {
                    m[j] = in ? static_cast<const float *>(e.m)[i + j] : 0.f;
                    v[j] = in ? static_cast<const float *>(e.v)[i + j] : 0.f;
                } else if (in) {
                    (j < 4 ? mc.x : mc.y) |= (uint32_t)static_cast<const uint8_t *>(e.m)[i + j] << (8 * (j % 4));
                    (j < 4 ? vc.x : vc.y) |= (uint32_t)static_cast<const uint8_t *>(e.v)[i + j] << (8 * (j % 4));
                }
            }
            if constexpr (BITS == 8) {
                decode8(mc, e.m_scale[(uint64_t)i / kBlock], m);
                decode8(vc, e.v_scale[(uint64_t)i / kBlock], v);
                __syncwarp();                                  // all have read the scales before one writes the new ones
            }
            update(e, i, x, g, m, v, random, mc, vc);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j < have) {
                    if constexpr (sizeof(T) == 2)
                        p[i + j] = STOCHASTIC && x[j] == x[j] ? __ushort_as_bfloat16((unsigned short)(up_or_down(x[j], random[j]) >> 16)) : __float2bfloat16_rn(x[j]);
                    else
                        p[i + j] = x[j];
                    if constexpr (BITS == 32) {
                        static_cast<float *>(e.m)[i + j] = m[j];
                        static_cast<float *>(e.v)[i + j] = v[j];
                    } else {
                        static_cast<uint8_t *>(e.m)[i + j] = (uint8_t)((j < 4 ? mc.x : mc.y) >> (8 * (j % 4)));
                        static_cast<uint8_t *>(e.v)[i + j] = (uint8_t)((j < 4 ? vc.x : vc.y) >> (8 * (j % 4)));
                    }
                }
            }
        }
    }
}

// Tensors of one launch: what fits into the 32764 bytes of arguments, or a small table where that is enough: its launch is cheaper (calls
// of 16 tensors of 1000 values 6 us, 8 with the large table; of 54 tensors 12.2 and 14.2; a replayed launch takes 5.1 and 5.6 us either way).
constexpr int kTensors = 500, kFewTensors = 56;

template <typename T, int BITS, bool STOCHASTIC, int CAP>
int launch(const wkv6_adamw &c, int64_t count, const wkv6_adamw_tensor *ts, cudaStream_t st) {
    static_assert(sizeof(Table<CAP>) <= 32764, "arguments of a launch");
    Table<CAP> a;
    a.step = c.step;
    a.step_device = c.step_device;
    a.lr_device = c.lr_device;
    a.grad_scale = c.grad_scale;
    a.lr = c.lr;
    a.beta1 = c.beta1;
    a.beta2 = c.beta2;
    a.eps = c.eps;
    a.weight_decay = c.weight_decay;
    a.seed_key = stir((uint32_t)c.seed);
    a.step_size = (float)(c.lr / (1.0 - power(c.beta1, c.step)));
    a.inv_root2 = (float)(1.0 / sqrt(1.0 - power(c.beta2, c.step)));
    constexpr int chunk_values = groups(BITS) * kGroupValues;
    int64_t i = 0;
    while (i < count) {
        a.count = 0;
        int64_t chunks = 0;
        for (; i < count && a.count < CAP; ++i) {
            if (ts[i].n == 0) continue;
            const int64_t more = (ts[i].n + chunk_values - 1) / chunk_values;
            if (chunks + more > 0x7fffffffLL) {
                if (a.count == 0) return fail(WKV6_ERR_UNSUPPORTED, "wkv6_adamw_step: tensor of %lld values", (long long)ts[i].n);
                break;
            }
            a.e[a.count++] = Entry{ts[i].p, ts[i].g, ts[i].m, ts[i].v, ts[i].m_scale, ts[i].v_scale, ts[i].n, (uint32_t)ts[i].index, (uint32_t)chunks};
            chunks += more;
        }
        if (a.count == 0) break;
        a.chunks = (uint32_t)chunks;
        const int64_t most = (int64_t)kBlocksPerSm * sm_count();
        adamw_kernel<T, BITS, STOCHASTIC, CAP><<<(unsigned)std::min(chunks, most), kThreads, 0, st>>>(a);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "adamw_kernel launch");
    }
    return WKV6_OK;
}

template <typename T, int BITS, bool STOCHASTIC>
int launch_sized(const wkv6_adamw &c, int64_t count, const wkv6_adamw_tensor *ts, cudaStream_t st) {
    return count <= kFewTensors ? launch<T, BITS, STOCHASTIC, kFewTensors>(c, count, ts, st) : launch<T, BITS, STOCHASTIC, kTensors>(c, count, ts, st);
}

}  // namespace

}  // namespace wkv6

using namespace wkv6;

extern "C" int wkv6_adamw_step(const wkv6_adamw *c, int64_t count, const wkv6_adamw_tensor *ts, void *stream) {
    if (c == nullptr || count < 0 || (count > 0 && ts == nullptr)) return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: NULL argument");
    if (c->dtype != WKV6_BF16 && c->dtype != WKV6_F32) return fail(WKV6_ERR_UNSUPPORTED, "wkv6_adamw_step: parameters must be bf16 or fp32");
    if (c->state_bits != 8 && c->state_bits != 32) return fail(WKV6_ERR_UNSUPPORTED, "wkv6_adamw_step: states of %d bits", c->state_bits);
    if (c->step_device == nullptr && c->step < 1) return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: step must be at least 1");
    if (!(c->beta1 >= 0.0 && c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0)) return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: betas must lie in [0, 1)");
    if (!(c->eps == 0.0 || (c->eps >= (double)FLT_MIN && c->eps <= (double)FLT_MAX)))      // a subnormal one would be zero in reciprocal()
        return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: eps must be 0 or a normal fp32 number, not %g", c->eps);
    // without gradients a code falls only if beta1 of it is beyond the border to its lower neighbour, which is at 17/18 of a code 1.125 2^n
    if (c->state_bits == 8 && c->beta1 > 0.94) return fail(WKV6_ERR_UNSUPPORTED, "wkv6_adamw_step: beta1 = %g, at most 0.94 with states of 8 bits", c->beta1);
    if (!aligned(8, {c->step_device}) || !aligned(4, {c->lr_device, c->grad_scale}))
        return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: values on the device must be aligned to their size");
    const size_t e = dtype_size(c->dtype), es = c->state_bits == 32 ? 4 : 1;
    for (int64_t i = 0; i < count; ++i) {
        const wkv6_adamw_tensor &t = ts[i];
        if (t.n < 0 || t.index < 0 || t.index > 0x7fffffffLL) return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: tensor %lld: n=%lld index=%lld", (long long)i, (long long)t.n, (long long)t.index);
        if (t.n == 0) continue;
        if (!t.p || !t.g || !t.m || !t.v || (c->state_bits == 8 && (!t.m_scale || !t.v_scale)))
            return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: tensor %lld: NULL pointer", (long long)i);
        const uintptr_t pg = reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g), mv = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
        const uintptr_t sc = c->state_bits == 8 ? reinterpret_cast<uintptr_t>(t.m_scale) | reinterpret_cast<uintptr_t>(t.v_scale) : 0;
        if (pg % e || mv % es || sc % 4) return fail(WKV6_ERR_INVALID, "wkv6_adamw_step: tensor %lld: misaligned pointer", (long long)i);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->dtype == WKV6_F32)
        return c->state_bits == 32 ? launch_sized<float, 32, false>(*c, count, ts, st) : launch_sized<float, 8, false>(*c, count, ts, st);
    if (c->stochastic)
        return c->state_bits == 32 ? launch_sized<__nv_bfloat16, 32, true>(*c, count, ts, st) : launch_sized<__nv_bfloat16, 8, true>(*c, count, ts, st);
    return c->state_bits == 32 ? launch_sized<__nv_bfloat16, 32, false>(*c, count, ts, st) : launch_sized<__nv_bfloat16, 8, false>(*c, count, ts, st);
}
