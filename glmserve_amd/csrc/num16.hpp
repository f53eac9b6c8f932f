// The two 16-bit number types of the ragged products (grouped.hip, lora.hip):
// fragments, matrix instructions, conversions, and loads of 8 consecutive values.
#pragma once

#include "common.hpp"

namespace glmmoe {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// The same vectors at any address of their elements: the memory pipeline takes them there.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Data type codes of the C entries (GLMMOE_F32 / BF16 / F16).
constexpr int kF32 = 0, kBf16 = 1, kF16 = 2;

struct Bf16 {
    static constexpr int code = kBf16;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) { return pack_bf16x2(a, b); }
    static __device__ __forceinline__ float up(uint32_t h) { return bf16_to_f32(h & 0xffffu); }
};

struct F16 {
    static constexpr int code = kF16;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    // Round to nearest even, as the hardware conversion does.
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
    }
    static __device__ __forceinline__ float up(uint32_t h) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    }
};

// 8 values k .. k + 7 of a row, all inside it.
__device__ __forceinline__ u32x4 load8(const uint16_t* row, int k) {
    return *reinterpret_cast<const u32x4_any*>(row + k);
}

// The same of a row of K values, with zeros from K on. ask8: the eight that end at K instead, where the row ends
// before k + 8 (a row of fewer has them one by one); fit8 makes of them what was asked for. Loads and
// their use stay apart so, without a branch between them.
__device__ __forceinline__ u32x4 ask8(const uint16_t* row, int k, int K) {
    if (K >= 8) return load8(row, min(k, K - 8));
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < K) v[i / 2] |= (uint32_t)row[i] << (16 * (i & 1));
    return v;
}
__device__ __forceinline__ u32x4 fit8(u32x4 v, int k, int K) {
    const int over = min(max(k - max(K - 8, 0), 0), 8);      // values before k; K < 8: k is a multiple of 8
    uint64_t lo = v[0] | (uint64_t)v[1] << 32, hi = v[2] | (uint64_t)v[3] << 32;
    if (over & 4) lo = hi, hi = 0;
    const int sh = (over & 3) * 16;
    lo = sh ? lo >> sh | hi << (64 - sh) : lo;
    hi >>= sh;
    if (over == 8) lo = 0, hi = 0;
    return (u32x4){(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}
__device__ __forceinline__ u32x4 load8_tail(const uint16_t* row, int k, int K) { return fit8(ask8(row, k, K), k, K); }

// 16 bytes of zeros in memory, for copies of what lies past a row's end.
static __device__ const u32x4 kZero16 = {0u, 0u, 0u, 0u};

// 64 lanes x 16 B from memory to LDS at base + 16 * lane, without the compiler's knowledge: it
// would have every LDS read wait for all of them.
// NT: read once, not worth a place in L2.
template <bool NT = false>
__device__ __forceinline__ void copy16(const void* g, uint32_t lds) {
    if constexpr (NT)
        asm volatile("s_mov_b32 m0, %1\n s_nop 0\n global_load_lds_dwordx4 %0, off nt"
                     :: "v"(g), "s"(lds) : "memory");
    else
        asm volatile("s_mov_b32 m0, %1\n s_nop 0\n global_load_lds_dwordx4 %0, off"
                     :: "v"(g), "s"(lds) : "memory");
}

// Four consecutive outputs of a row from element `at` on, of which cnt are inside it.
template <class T, bool F32>
__device__ __forceinline__ void store4(void* y, long at, f32x4 v, int cnt) {
    if constexpr (F32) {
        float* p = static_cast<float*>(y) + at;
        if (cnt >= 4) {
            *reinterpret_cast<f32x4_any*>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < cnt) p[i] = v[i];
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(y) + at;
        const u32x2 w = {T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
        if (cnt >= 4) {
            *reinterpret_cast<u32x2_any*>(p) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < cnt) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

}  // namespace glmmoe
