// AdamW over many tensors.  Per element, in this order and with every product and sum rounded to fp32 by itself (no contraction: what is
// held in 8 bits changes with the last bit, and a plain evaluation of the same formulas then holds the same bits):
//   g = grad * grad_scale;  m = m beta1 + g (1 - beta1);  v = v beta2 + (g g)(1 - beta2);  r = sqrt(v)
//   p = p decay - (m / (r inv_root + eps)) step_size
// Bound: HBM.  32-bit moments: 28 bytes a parameter in fp32 (p, g, m, v read; p, m, v written); 8-bit moments: 16, 10 in bf16.
// 21 M parameters in 141 tensors: 107 us with 32 bits (5.5 TB/s, above what HBM gives: part of it stays in the last-level cache), 75 with 8; 200 M in bf16
// with 8 bits: 510 us (3.9 TB/s, and some 75 vector instructions an element).
//
// 8-bit moments.  m and r = sqrt(v) (half the decades of v) are held as e4m3 values of x / scale, scale = the largest |x| of 256
// consecutive elements / 448.  Rounding to nearest would freeze them: beta2 = 0.999 moves v by 0.1 % a step and half a step of e4m3 is
// 6 %.  So a value is rounded down or up with the probability of its remainder, from 16 bits of a hash of (salt, step, element): the means of m and
// r move as in 32 bits.  The mean of v = r^2 does not: rounding spreads r, and v is above its true mean by that variance -- under 0.5 % where gradients
// keep their size; where an element's fall against its block's largest, by the logarithm of the fall / 16 to / 8 (tenfold, over 1500 steps: 7 %).
// r > 0 is never held as 0 -- its next step would divide by eps.
// One wave owns a block of 256: four elements a lane, the block's maximum through lane exchanges, no LDS.
#include <math.h>

#include "seq.h"

namespace {

constexpr int kBatch = 52;       // tensors per launch: 52 x 64 bytes of the 4 KB of kernel arguments
constexpr int kChunk = 4096;     // elements per workgroup: 16 blocks of 256, four per wave
constexpr int kThreads = 256;
constexpr long kMostChunks = (1L << 24) - 1;       // of one launch: fewer than 2^32 threads
constexpr int kBlock = 256;
constexpr float kTop = 448.0f;   // the largest e4m3 value

struct Table {
    fsc_adamw_tensor t[kBatch];
    int chunk_start[kBatch + 1];
    int n;
};
struct Hyper {
    float decay, step_size, inv_root, step;
    float beta1, rest1, beta2, rest2, eps, grad_scale;
    const float* dev;            // non-null: the first four come from device memory
};
static_assert(sizeof(Table) + sizeof(Hyper) <= 4096, "kernel arguments");

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x9E3779B9u;
    x = (x ^ (x >> 15)) * 0xB7E15163u;
    return x ^ (x >> 16);
}

// 1 / x for x in the normal range: the estimate (1 ulp) and one correction, rounded correctly (but for x of all ones, where it is 1 ulp off); a
// quarter of the instructions of a division that scales its operands.
__device__ __forceinline__ float reciprocal(float x) {
    const float y = __builtin_amdgcn_rcpf(x);
    return fmaf(fmaf(-x, y, 1.0f), y, y);
}

// scale and 448 / top of a block (0 and 0 where the scale would be below the normal numbers: the block is held as zeros)
struct BlockScale {
    float scale, inverse;
    __device__ explicit BlockScale(float top) {
#pragma clang fp contract(off)
        scale = top * (1.0f / kTop);
        const bool dead = scale < 1.17549435e-38f;
        inverse = dead ? 0.f : reciprocal(top) * kTop;
        scale = dead ? 0.f : scale;
    }
};

// e4m3 pattern of x * inverse, rounded down or up by the 16 random bits.  Normal values: adding them below the three mantissa bits
// carries with the probability of the remainder; below 2^-6 the values are multiples of 2^-9.  FINITE: nothing in the block is NaN or infinite.
template <bool POSITIVE, bool FINITE>
__device__ __forceinline__ uint32_t held(float x, float inverse, uint32_t bits16) {
#pragma clang fp contract(off)
    const float y = x * inverse, size = fabsf(y);
    const uint32_t pattern = __float_as_uint(size);
    const uint32_t normal = ((pattern + (bits16 << 4)) >> 20) - (120u << 3);
    const uint32_t small = (uint32_t)(size * 512.0f + (float)bits16 * 0x1p-16f);
    uint32_t code = size >= 0x1p-6f ? normal : small;
    code = code > 0x7Eu ? 0x7Eu : code;
    if (POSITIVE) code = code == 0 && y > 0.f ? 1 : code;
    else code |= (__float_as_uint(y) >> 24) & 0x80u;
    return FINITE || pattern < 0x7F800000u ? code : 0x7Fu;
}

// The value of a pattern: sign, four exponent bits (bias 7), three mantissa bits; 0x7F and 0xFF are NaN.
__device__ __forceinline__ float e4m3_value(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

// The largest pattern of the wave's (non-negative) values, in every lane: they order as integers do, and integers need no canonical form.
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
    return v > w ? v : w;
}
__device__ __forceinline__ float wave_top(float value) {
    uint32_t v = max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(__float_as_uint(value)))));
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t r0 = rows[0], r1 = rows[1];
    v = r0 > r1 ? r0 : r1;
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t h0 = halves[0], h1 = halves[1];
    return __uint_as_float(h0 > h1 ? h0 : h1);
}

// What a lane has of a block of 256: four consecutive elements, the held ones as they lie in memory.
template <typename T, int BITS>
struct Four {
    fsc::Pack<T, 4> p, g;
    fsc::Pack<float, 4> m, v;            // BITS == 32
    uint32_t w0, w1;                     // BITS == 8
    float s0, s1;
};

// The step on one block.  ALL: every lane has its four elements and wide accesses are aligned; else `have` of them, one by one.
template <typename T, int BITS, bool ALL>
__device__ __forceinline__ void load_four(const fsc_adamw_tensor& t, long block, int lane, int have, Four<T, BITS>& f) {
    const long e = block + 4 * lane;
    const T* p = reinterpret_cast<const T*>(t.param) + e;
    const T* g = reinterpret_cast<const T*>(t.grad) + e;
    if constexpr (ALL) {
        f.p = fsc::load_pack<T, 4>(p);
        f.g = fsc::load_pack<T, 4>(g);
        if constexpr (BITS == 32) {
            f.m = fsc::load_pack<float, 4>(reinterpret_cast<const float*>(t.state0) + e);
            f.v = fsc::load_pack<float, 4>(reinterpret_cast<const float*>(t.state1) + e);
        } else {
            f.w0 = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(t.state0) + e);
            f.w1 = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(t.state1) + e);
        }
    } else {
        f = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= have) break;
            f.p.v[i] = p[i];
            f.g.v[i] = g[i];
            if constexpr (BITS == 32) {
                f.m.v[i] = reinterpret_cast<const float*>(t.state0)[e + i];
                f.v.v[i] = reinterpret_cast<const float*>(t.state1)[e + i];
            } else {
                f.w0 |= (uint32_t)reinterpret_cast<const uint8_t*>(t.state0)[e + i] << (8 * i);
                f.w1 |= (uint32_t)reinterpret_cast<const uint8_t*>(t.state1)[e + i] << (8 * i);
            }
        }
    }
    if constexpr (BITS == 8) {
        f.s0 = t.scale0[block / kBlock];
        f.s1 = t.scale1[block / kBlock];
    }
}

template <bool FINITE>
__device__ __forceinline__ void hold_four(const float (&m)[4], const float (&r)[4], const BlockScale& b0, const BlockScale& b1, uint32_t e, uint32_t key,
                                          uint32_t& w0, uint32_t& w1) {
    w0 = w1 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bits = mix32((e + i) ^ key);
        w0 |= held<false, FINITE>(m[i], b0.inverse, bits >> 16) << (8 * i);
        w1 |= held<true, FINITE>(r[i], b1.inverse, bits & 0xFFFFu) << (8 * i);
    }
}

template <typename T, int BITS, bool ALL>
__device__ __forceinline__ void step_four(const fsc_adamw_tensor& t, const Hyper& h, uint32_t key, long block, int lane, int have, const Four<T, BITS>& f) {
#pragma clang fp contract(off)
    const long e = block + 4 * lane;
    float m[4], v[4], r[4];
    fsc::Pack<T, 4> out;
    float top0 = 0.f, top1 = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BITS == 32) {
            m[i] = f.m.v[i];
            v[i] = f.v.v[i];
        } else {
            m[i] = e4m3_value((f.w0 >> (8 * i)) & 0xFF) * f.s0;
            const float held_r = e4m3_value((f.w1 >> (8 * i)) & 0xFF) * f.s1;
            v[i] = held_r * held_r;
        }
        const float g = (float)f.g.v[i] * h.grad_scale;
        m[i] = m[i] * h.beta1 + g * h.rest1;
        v[i] = v[i] * h.beta2 + (g * g) * h.rest2;
        r[i] = sqrtf(v[i]);
        out.v[i] = (T)((float)f.p.v[i] * h.decay - (m[i] / (r[i] * h.inv_root + h.eps)) * h.step_size);
        if (ALL || i < have) {
            top0 = fmaxf(top0, fabsf(m[i]));
            top1 = fmaxf(top1, r[i]);
        }
    }
    T* p = reinterpret_cast<T*>(t.param) + e;
    if constexpr (ALL) {
        fsc::store_pack<T, 4>(p, out);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < have) p[i] = out.v[i];
    }
    if constexpr (BITS == 32) {
        float* m_out = reinterpret_cast<float*>(t.state0) + e;
        float* v_out = reinterpret_cast<float*>(t.state1) + e;
        fsc::store_row<4>(m_out, ALL, have, m);
        fsc::store_row<4>(v_out, ALL, have, v);
    } else {
        // (a sum is NaN or infinite where a term is; fmaxf drops NaN)
        const float sum = (m[0] + m[1]) + (m[2] + m[3]) + ((r[0] + r[1]) + (r[2] + r[3]));
        uint32_t w0, w1;
        BlockScale b0(0.f), b1(0.f);
        if (__builtin_amdgcn_ballot_w64(!(fabsf(sum) < INFINITY)) == 0) {
            b0 = BlockScale(wave_top(top0));
            b1 = BlockScale(wave_top(top1));
            hold_four<true>(m, r, b0, b1, (uint32_t)e, key, w0, w1);
        } else {                                             // something is not finite: it stays out of the maxima and is held as NaN
            top0 = top1 = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                top0 = fmaxf(top0, fabsf(m[i]) < INFINITY && i < have ? fabsf(m[i]) : 0.f);
                top1 = fmaxf(top1, r[i] < INFINITY && i < have ? r[i] : 0.f);
            }
            b0 = BlockScale(wave_top(top0));
            b1 = BlockScale(wave_top(top1));
            hold_four<false>(m, r, b0, b1, (uint32_t)e, key, w0, w1);
        }
        uint8_t* c0 = reinterpret_cast<uint8_t*>(t.state0) + e;
        uint8_t* c1 = reinterpret_cast<uint8_t*>(t.state1) + e;
        if constexpr (ALL) {
            *reinterpret_cast<uint32_t*>(c0) = w0;
            *reinterpret_cast<uint32_t*>(c1) = w1;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= have) break;
                c0[i] = (uint8_t)(w0 >> (8 * i));
                c1[i] = (uint8_t)(w1 >> (8 * i));
            }
        }
        if (lane == 0) {
            t.scale0[block / kBlock] = b0.scale;
            t.scale1[block / kBlock] = b1.scale;
        }
    }
}

template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table tb, Hyper h) {
    if (h.dev != nullptr) {
        h.decay = h.dev[0];
        h.step_size = h.dev[1];
        h.inv_root = h.dev[2];
        h.step = h.dev[3];
    }
    int lo = 0, hi = tb.n - 1;                               // the last tensor that begins at or before this chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int)blockIdx.x >= tb.chunk_start[mid]) lo = mid; else hi = mid - 1;
    }
    const fsc_adamw_tensor t = tb.t[lo];
    const long base = (long)((int)blockIdx.x - tb.chunk_start[lo]) * kChunk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr size_t kStateAlign = BITS == 32 ? 16 : 4;
    const bool wide = (((size_t)t.param | (size_t)t.grad) & (4 * sizeof(T) - 1)) == 0 &&
                      (((size_t)t.state0 | (size_t)t.state1) & (kStateAlign - 1)) == 0;
    uint32_t key = 0;
    if constexpr (BITS == 8) {
        key = mix32(mix32((uint32_t)t.salt) + (uint32_t)h.step);
        if (base >> 32) key = mix32(key + (uint32_t)(base >> 32));
    }
    constexpr int kTurns = kChunk / (4 * kThreads), kWaves = kThreads / 64;
    if (wide && base + kChunk <= t.count) {                  // a whole chunk: the loads of its four blocks are in flight together
        Four<T, BITS> f[kTurns];
#pragma unroll
        for (int it = 0; it < kTurns; ++it) load_four<T, BITS, true>(t, base + (it * kWaves + wave) * kBlock, lane, 4, f[it]);
#pragma unroll
        for (int it = 0; it < kTurns; ++it) step_four<T, BITS, true>(t, h, key, base + (it * kWaves + wave) * kBlock, lane, 4, f[it]);
        return;
    }
    for (int it = 0; it < kTurns; ++it) {
        const long block = base + (it * kWaves + wave) * kBlock;
        if (block >= t.count) return;                        // (a wave's blocks ascend)
        Four<T, BITS> f;
        if (wide && block + kBlock <= t.count) {
            load_four<T, BITS, true>(t, block, lane, 4, f);
            step_four<T, BITS, true>(t, h, key, block, lane, 4, f);
        } else {
            const long left = t.count - block - 4 * lane;
            const int have = left <= 0 ? 0 : left < 4 ? (int)left : 4;
            load_four<T, BITS, false>(t, block, lane, have, f);
            step_four<T, BITS, false>(t, h, key, block, lane, have, f);
        }
    }
}

}  // namespace

extern "C" {

void fsc_adamw_step_factors(double lr, double beta1, double beta2, double weight_decay, long step, float* out4_host) {
    out4_host[0] = (float)(1.0 - lr * weight_decay);
    out4_host[1] = (float)(lr / (1.0 - pow(beta1, (double)step)));
    out4_host[2] = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    out4_host[3] = (float)(step & 0xFFFFFF);
}

int fsc_adamw_step(const fsc_adamw_tensor* tensors_host, int n_tensors, int dtype, int state_bits, const float* factors4,
                   const float* factors4_dev, double beta1, double beta2, float eps, float grad_scale, fsc_stream_t stream) {
    FSC_CHECK_ARG(tensors_host && n_tensors > 0 && (factors4 != nullptr) != (factors4_dev != nullptr), "fsc_adamw_step: bad arguments");
    FSC_CHECK_ARG(fsc::dtype_ok(dtype), "fsc_adamw_step: dtype %d", dtype);
    FSC_CHECK_ARG(state_bits == 32 || state_bits == 8, "fsc_adamw_step: state_bits %d (32 or 8)", state_bits);
    for (int i = 0; i < n_tensors; ++i) {
        const fsc_adamw_tensor& t = tensors_host[i];
        FSC_CHECK_ARG(t.count >= 0, "fsc_adamw_step: tensor %d has %ld elements", i, t.count);
        FSC_CHECK_ARG(t.count == 0 || (t.param && t.grad && t.state0 && t.state1), "fsc_adamw_step: tensor %d has null pointers", i);
        FSC_CHECK_ARG(t.count == 0 || state_bits == 32 || (t.scale0 && t.scale1), "fsc_adamw_step: tensor %d misses its scales", i);
        FSC_CHECK_ARG(t.count <= kChunk * kMostChunks, "fsc_adamw_step: tensor %d is too large", i);
    }
    Hyper h{};
    if (factors4 != nullptr) {
        h.decay = factors4[0];
        h.step_size = factors4[1];
        h.inv_root = factors4[2];
        h.step = factors4[3];
    }
    h.beta1 = (float)beta1;
    h.rest1 = (float)(1.0 - beta1);
    h.beta2 = (float)beta2;
    h.rest2 = (float)(1.0 - beta2);
    h.eps = eps;
    h.grad_scale = grad_scale;
    h.dev = factors4_dev;
    hipStream_t st = fsc::as_stream(stream);
    int next = 0;
    while (next < n_tensors) {
        Table tb{};
        long chunks = 0;
        while (next < n_tensors && tb.n < kBatch) {
            const fsc_adamw_tensor& t = tensors_host[next];
            const long more = (t.count + kChunk - 1) / kChunk;
            if (tb.n > 0 && chunks + more > kMostChunks) break;
            ++next;
            if (more == 0) continue;
            tb.t[tb.n] = t;
            tb.chunk_start[tb.n++] = (int)chunks;
            chunks += more;
        }
        if (tb.n == 0) continue;
        tb.chunk_start[tb.n] = (int)chunks;
        auto launch = [&](auto type) {
            using T = decltype(type);
            if (state_bits == 32) hipLaunchKernelGGL((adamw_kernel<T, 32>), dim3((unsigned)chunks), dim3(kThreads), 0, st, tb, h);
            else hipLaunchKernelGGL((adamw_kernel<T, 8>), dim3((unsigned)chunks), dim3(kThreads), 0, st, tb, h);
        };
        FSC_WITH_DTYPE(dtype, launch);
        FSC_LAUNCH_CHECK("fsc_adamw_step");
    }
    return 0;
}

}  // extern "C"
