// What the sequence kernels and the decoupled optimizer share: activations in three types, reductions over neighbouring lanes.
#pragma once
#include "common.h"

namespace fsc {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V consecutive values as one load or store (the caller has checked that the address is a multiple of their size)
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// The same bytes as one integer word: a wide access must not look like the narrow ones beside it, or the two paths are merged into narrow ones.
template <int N> struct Word;
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    const auto w = *reinterpret_cast<const typename Word<sizeof(T) * V>::type*>(p);
    return __builtin_bit_cast(Pack<T, V>, w);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    *reinterpret_cast<typename Word<sizeof(T) * V>::type*>(p) = __builtin_bit_cast(typename Word<sizeof(T) * V>::type, v);
}

// V consecutive values on their way from memory, as the 32-bit words that hold them; converted where they are used.  (Held as values, those of a
// wide load would be taken apart where the wide and the narrow path meet, right behind the load, and so would wait for it there.)
template <typename T, int V>
struct Raw {
    uint32_t w[(V * sizeof(T) + 3) / 4];
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) {
            const uint32_t word = w[i];
            return __builtin_bit_cast(float, word);
        } else {
            const uint16_t half = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
            return (float)__builtin_bit_cast(T, half);
        }
    }
    __device__ __forceinline__ void wide(const T* p) {
        const auto word = *reinterpret_cast<const typename Word<sizeof(T) * V>::type*>(p);
        if constexpr (sizeof(T) * V < 4) w[0] = word;
        else *this = __builtin_bit_cast(Raw, word);
    }
    // Waits for the load here.  Loads and stores are counted together, in order: in front of stores, a load is not held up by them.
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 4); ++i) asm volatile("" : "+v"(w[i]));
    }
    // from(i): the address of the i-th value
    template <typename From>
    __device__ __forceinline__ void narrow(From from) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 4); ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = *reinterpret_cast<const uint32_t*>(from(i));
            } else {
                w[i] = *reinterpret_cast<const uint16_t*>(from(2 * i));
                if (2 * i + 1 < V) w[i] |= (uint32_t)*reinterpret_cast<const uint16_t*>(from(2 * i + 1)) << 16;
            }
        }
        arrived();
    }
};

// V consecutive values at `p` as floats: one wide load where `wide`, else one by one and only the first `have` (the others are 0).
template <int V, typename T>
__device__ __forceinline__ void load_row(const T* p, bool wide, int have, float (&out)[V]) {
    if (wide) {
        const Pack<T, V> w = load_pack<T, V>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)w.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = i < have ? (float)p[i] : 0.f;
    }
}
template <int V, typename T>
__device__ __forceinline__ void store_row(T* p, bool wide, int have, const float (&in)[V]) {
    if (wide) {
        Pack<T, V> w;
#pragma unroll
        for (int i = 0; i < V; ++i) w.v[i] = (T)in[i];
        store_pack<T, V>(p, w);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < have) p[i] = (T)in[i];
    }
}

// A neighbour's value within a row of 16 lanes, in the adder's own operand fetch.  CTRL: 0xB1 lane ^ 1, 0x4E lane ^ 2, 0x141 mirrored
// within 8 (with equal quads: lane ^ 4), 0x140 mirrored within 16 (with equal eights: lane ^ 8), 0x124 / 0x128 turned by 4 / 8 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// The value is there from here on: sums that nothing reads for a while are otherwise put off, with all their terms kept in registers until
// then, and lane exchanges end up under a mask, where they cannot be part of the addition.
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// ... of an array; in front of a loop: what was loaded there is waited for there, not at its first use inside, behind the loop's own loads.
template <int N>
__device__ __forceinline__ void pin_all(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) pin(v[i]);
}

// The sum over aligned groups of L <= 16 lanes, in every lane of the group.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    if constexpr (L >= 2) v += dpp<0xB1>(v);
    if constexpr (L >= 4) v += dpp<0x4E>(v);
    if constexpr (L >= 8) v += dpp<0x141>(v);
    if constexpr (L >= 16) v += dpp<0x140>(v);
    return v;
}

// Lanes 32..63 of `a` change places with lanes 0..31 of `b` (swap32), the odd rows of 16 of `a` with the even rows of `b` (swap16):
// a + b is then the halfway sum of both, `a`'s in the lower half or the even rows, `b`'s in the others.
__device__ __forceinline__ void swap32(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned first = r[0], second = r[1];      // (out of the vector first: a bit cast of its element reads element 0)
    a = __builtin_bit_cast(float, first);
    b = __builtin_bit_cast(float, second);
}
__device__ __forceinline__ void swap16(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned first = r[0], second = r[1];      // (out of the vector first: a bit cast of its element reads element 0)
    a = __builtin_bit_cast(float, first);
    b = __builtin_bit_cast(float, second);
}

inline size_t dtype_bytes(int dtype) { return dtype == FSC_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == FSC_DTYPE_F32 || dtype == FSC_DTYPE_BF16 || dtype == FSC_DTYPE_F16; }
// whether p is a multiple of `bytes`, a power of two
inline bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

}  // namespace fsc

// `run(T())` with the activation type that `dtype` names
#define FSC_WITH_DTYPE(dtype, run)                                                                                              \
    ((dtype) == FSC_DTYPE_F32 ? run(float()) : (dtype) == FSC_DTYPE_BF16 ? run(fsc::bf16_t()) : run(fsc::f16_t()))
