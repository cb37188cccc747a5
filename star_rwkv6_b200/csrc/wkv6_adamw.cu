// AdamW over many tensors at once (include/wkv6_b200.h gives the formulas), states in fp32 or in blocks of 256 e4m3 codes with a scale.
//
// Bound by HBM: a bf16 value with fp32 states moves 22 bytes, with 8-bit states 10.06, for about twenty operations.  The tensors of a
// model differ in size by four orders of magnitude, so they are cut into chunks of 4096 values and the blocks of one launch walk all
// chunks; a chunk's tensor is found by bisection in a table that travels in the launch's arguments (no copy to the device, nothing to
// keep alive, and a captured launch holds its own).  A thread has eight neighbouring values, a warp the 256 of a block of codes, whose
// largest value is one warp reduction.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "wkv6_internal.h"

namespace wkv6 {

namespace {

constexpr int kThreads = 256, kChunk = 4096, kPerThread = 8, kBlock = 256;

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

__device__ __forceinline__ float root(float x) {
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
}

__device__ __forceinline__ void store8(float *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }

// fp32 to bf16: to nearest, or with 16 random bits added below the last kept one and then dropped.
template <bool STOCHASTIC>
__device__ __forceinline__ __nv_bfloat16 narrow(float x, uint32_t random) {
    if (!STOCHASTIC || x != x) return __float2bfloat16_rn(x);       // the sum would carry a NaN into the sign
    return __ushort_as_bfloat16((unsigned short)((__float_as_uint(x) + (random & 0xffffu)) >> 16));
}

// q >= 0 in units of the block's scale onto the e4m3 grid, up or down by 16 random bits; never from above zero to zero, which would
// divide the next update by eps alone.
__device__ __forceinline__ float grid8(float q, uint32_t random) {
    const float normal = __uint_as_float((__float_as_uint(q) + ((random >> 16) << 4)) & 0xfff00000u);
    const float tiny = fmaxf(floorf(fmaf(q, 512.f, (float)(random >> 16) * 0x1p-16f)), 1.f) * (1.f / 512.f);
    return q >= 0x1p-6f ? normal : q > 0.f ? tiny : 0.f;
}

__device__ __forceinline__ void decode8(uint64_t codes, float scale, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * i)), __NV_E4M3);
        const float2 x = __half22float2(__half2(h));
        f[2 * i] = x.x * scale;
        f[2 * i + 1] = x.y * scale;
    }
}

__device__ __forceinline__ uint64_t encode8(const float (&f)[8]) {
    uint64_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        codes |= (uint64_t)__nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3) << (16 * i);
    return codes;
}

// Largest magnitude of the warp's 256 values, compared as bits: a NaN is larger than all others and stays.
__device__ __forceinline__ float block_top(const float (&f)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}

// A block's scale and the factor onto multiples of it.  Blocks below 2^-100 are zeros: their scale would leave the normal numbers.
__device__ __forceinline__ float2 block_scale(float top) {
    if (top < 0x1p-100f) top = 0.f;
    return make_float2(top * (1.f / 448.f), top > 0.f ? 448.f / top : 0.f);
}

template <typename T, int BITS, bool STOCHASTIC, int CAP>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ Table<CAP> a) {
    __shared__ float shared[2];
    float step_size = a.step_size, inv_root2 = a.inv_root2;
    float decay = (float)(1.0 - a.lr * a.weight_decay);
    int64_t t = a.step;
    if (a.step_device != nullptr || a.lr_device != nullptr) {
        const double lr = a.lr_device != nullptr ? (double)*a.lr_device : a.lr;
        if (a.step_device != nullptr) t = *a.step_device;
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
    const float gs = a.grad_scale != nullptr ? *a.grad_scale : 1.f;
    const uint32_t step_key = stir((uint32_t)t ^ a.seed_key);
    const int lane = threadIdx.x & 31;
    for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
        int k = 0, end = a.count;
        while (end - k > 1) {
            const int mid = (k + end) >> 1;
            if (a.e[mid].first_chunk <= chunk) k = mid; else end = mid;
        }
        const Entry &e = a.e[k];
        const int64_t n = e.n, start = (int64_t)(chunk - e.first_chunk) * kChunk;
        const uint32_t key = stir(e.index ^ step_key);
        T *p = static_cast<T *>(e.p);
        const T *g = static_cast<const T *>(e.g);
        const bool aligned = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & 15) == 0 &&
                             ((reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v)) & (BITS == 32 ? 15 : 7)) == 0;
#pragma unroll
        for (int it = 0; it < kChunk / (kThreads * kPerThread); ++it) {
            const int64_t i = start + it * (kThreads * kPerThread) + threadIdx.x * kPerThread;
            const int64_t block = i / kBlock;                 // of this warp
            if (i - lane * kPerThread >= n) break;            // the warp as a whole
            const bool whole = aligned && i + kPerThread <= n;
            const int have = i + kPerThread <= n ? kPerThread : i < n ? (int)(n - i) : 0;
            float x[8], gr[8], m[8], v[8];
            if (whole) {
                load8(p + i, x);
                load8(g + i, gr);
                if constexpr (BITS == 32) {
                    load8(static_cast<const float *>(e.m) + i, m);
                    load8(static_cast<const float *>(e.v) + i, v);
                } else {
                    decode8(*reinterpret_cast<const uint64_t *>(static_cast<const uint8_t *>(e.m) + i), e.m_scale[block], m);
                    decode8(*reinterpret_cast<const uint64_t *>(static_cast<const uint8_t *>(e.v) + i), e.v_scale[block], v);
                }
            } else {
                uint64_t mc = 0, vc = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool in = j < have;
                    x[j] = in ? value(p[i + j]) : 0.f;
                    gr[j] = in ? value(g[i + j]) : 0.f;
                    if constexpr (BITS == 32) {
                        m[j] = in ? static_cast<const float *>(e.m)[i + j] : 0.f;
                        v[j] = in ? static_cast<const float *>(e.v)[i + j] : 0.f;
                    } else if (in) {
                        mc |= (uint64_t)static_cast<const uint8_t *>(e.m)[i + j] << (8 * j);
                        vc |= (uint64_t)static_cast<const uint8_t *>(e.v)[i + j] << (8 * j);
                    }
                }
                if constexpr (BITS == 8) {
                    decode8(mc, e.m_scale[block], m);
                    decode8(vc, e.v_scale[block], v);
                }
            }
            const uint32_t high = (uint32_t)((uint64_t)i >> 32);
            const uint32_t place = high ? stir(key + high) : key;      // eight neighbours share the upper word
            uint32_t random[8];
            float r[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (STOCHASTIC || BITS == 8) random[j] = stir(((uint32_t)i + j) ^ place);
                if constexpr (BITS == 8) v[j] *= v[j];
                const float gj = gr[j] * gs;
                m[j] = fmaf(gj, c1, m[j] * b1);
                v[j] = fmaf(gj * gj, c2, v[j] * b2);
                r[j] = root(v[j]);
                x[j] = x[j] * decay - __fdividef(m[j] * step_size, fmaf(r[j], inv_root2, eps));
            }
            uint64_t mc = 0, vc = 0;
            if constexpr (BITS == 8) {
                const float2 ms = block_scale(block_top(m)), vs = block_scale(block_top(r));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    m[j] = ms.y > 0.f ? m[j] * ms.y : 0.f;
                    r[j] = grid8(r[j] * vs.y, random[j]);
                }
                mc = encode8(m);
                vc = encode8(r);
                if (lane == 0) {
                    e.m_scale[block] = ms.x;
                    e.v_scale[block] = vs.x;
                }
            }
            if (whole) {
                if constexpr (sizeof(T) == 2) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const __nv_bfloat162 h(narrow<STOCHASTIC>(x[2 * j], random[2 * j]), narrow<STOCHASTIC>(x[2 * j + 1], random[2 * j + 1]));
                        w[j] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    *reinterpret_cast<uint4 *>(p + i) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    store8(p + i, x);
                }
                if constexpr (BITS == 32) {
                    store8(static_cast<float *>(e.m) + i, m);
                    store8(static_cast<float *>(e.v) + i, v);
                } else {
                    *reinterpret_cast<uint64_t *>(static_cast<uint8_t *>(e.m) + i) = mc;
                    *reinterpret_cast<uint64_t *>(static_cast<uint8_t *>(e.v) + i) = vc;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j < have) {
                        if constexpr (sizeof(T) == 2) p[i + j] = narrow<STOCHASTIC>(x[j], random[j]); else p[i + j] = x[j];
                        if constexpr (BITS == 32) {
                            static_cast<float *>(e.m)[i + j] = m[j];
                            static_cast<float *>(e.v)[i + j] = v[j];
                        } else {
                            static_cast<uint8_t *>(e.m)[i + j] = (uint8_t)(mc >> (8 * j));
                            static_cast<uint8_t *>(e.v)[i + j] = (uint8_t)(vc >> (8 * j));
                        }
                    }
                }
            }
        }
    }
}

// Tensors of one launch: what fits into the 32764 bytes of arguments, or a small table where that is enough (its launch is cheaper).
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
    int64_t i = 0;
    while (i < count) {
        a.count = 0;
        int64_t chunks = 0;
        for (; i < count && a.count < CAP; ++i) {
            if (ts[i].n == 0) continue;
            const int64_t more = (ts[i].n + kChunk - 1) / kChunk;
            if (chunks + more > 0x7fffffffLL) {
                if (a.count == 0) return fail(WKV6_ERR_UNSUPPORTED, "wkv6_adamw_step: tensor of %lld values", (long long)ts[i].n);
                break;
            }
            a.e[a.count++] = Entry{ts[i].p, ts[i].g, ts[i].m, ts[i].v, ts[i].m_scale, ts[i].v_scale, ts[i].n, (uint32_t)ts[i].index, (uint32_t)chunks};
            chunks += more;
        }
        if (a.count == 0) break;
        a.chunks = (uint32_t)chunks;
        const int64_t most = 4LL * sm_count();
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
