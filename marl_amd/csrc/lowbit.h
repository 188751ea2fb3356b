// What the low-bit passes share (mx_kernels.hip, act_kernels.hip): loads of float32 / bfloat16 / float16 rows at any
// element alignment, absolute maxima as integers, and the power-of-two scale of a block of 32 values.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/marl_amd.h"

namespace oc {

int set_error(int code, const std::string& msg);  // capi.hip

constexpr int LB_BLOCK = 32;  // values that share a scale

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// The same vectors at the alignment a row of odd length leaves them with; the hardware's loads and stores take them whole.
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a1 __attribute__((aligned(1)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef uint32_t u32_a1 __attribute__((aligned(1)));

static inline size_t lb_blocks(int64_t cols) { return (size_t)((cols + LB_BLOCK - 1) / LB_BLOCK); }
static inline size_t lb_type_bytes(int type) { return type == MARL_F32 ? 4 : 2; }

__device__ __forceinline__ float bits_f(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t f_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ float half_lo(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }
__device__ __forceinline__ float half_hi(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16)); }

template <int TYPE>
__device__ __forceinline__ float load_one(const void* p, int64_t at) {
    if constexpr (TYPE == MARL_F32) return static_cast<const float*>(p)[at];
    const uint16_t u = static_cast<const uint16_t*>(p)[at];
    if constexpr (TYPE == MARL_BF16) return bits_f((uint32_t)u << 16);
    return (float)__builtin_bit_cast(_Float16, u);
}

// What is read once and is larger than this cannot have stayed in the 256 MiB last-level cache whole, and would push out of
// it what the next pass reads: it is read with the non-temporal hint.  Compressing 131072 x 512 float32 values and reading
// the codes back: 108 us with it, 146 without.
constexpr size_t LB_NT_BYTES = (size_t)64 << 20;

// 8 values from element `at` on; those at or behind element `end` read as 0 and are not touched in memory
template <int TYPE, bool NT = false>
__device__ __forceinline__ void load_eight(const void* p, int64_t at, int64_t end, float (&v)[8]) {
    if (at + 8 <= end) {
        if constexpr (TYPE == MARL_F32) {
            const float* f = static_cast<const float*>(p) + at;
            const f32x4_a4 *p0 = reinterpret_cast<const f32x4_a4*>(f), *p1 = reinterpret_cast<const f32x4_a4*>(f + 4);
            const f32x4 a = NT ? __builtin_nontemporal_load(p0) : *p0, b = NT ? __builtin_nontemporal_load(p1) : *p1;
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const u32x4_a2* p0 = reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(p) + at);
            const u32x4 u = NT ? __builtin_nontemporal_load(p0) : *p0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (TYPE == MARL_BF16) {
                    v[2 * k] = bits_f(u[k] << 16);
                    v[2 * k + 1] = bits_f(u[k] & 0xFFFF0000u);
                } else {
                    v[2 * k] = half_lo(u[k]);
                    v[2 * k + 1] = half_hi(u[k]);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = at + k < end ? load_one<TYPE>(p, at + k) : 0.0f;
}

// Largest |v| as an unsigned integer: float order for numbers, infinity above them, NaNs above infinity.
__device__ __forceinline__ uint32_t abs_top(const float (&v)[8]) {
    uint32_t t = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) t = max(t, f_bits(v[k]) & 0x7FFFFFFFu);
    return t;
}

// maximum over the four lanes of an aligned quad (two DPP moves)
__device__ __forceinline__ uint32_t quad_max(uint32_t t) {
    t = max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, 0xB1, 0xF, 0xF, true));  // quad_perm 1,0,3,2
    return max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, 0x4E, 0xF, 0xF, true));  // quad_perm 2,3,0,1
}

// value of a scale byte: 2^(byte - 127), NaN for 255 (and the denormal 2^-127 for 0)
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return bits_f(max(byte << 23 | (byte == 255u ? 0x00400000u : 0u), 0x00400000u));
}

template <int TYPE>
__device__ __forceinline__ uint16_t to_half_type(float v) {
    if constexpr (TYPE == MARL_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    return __builtin_bit_cast(uint16_t, (_Float16)v);
}

template <int TYPE>
__device__ __forceinline__ void store_eight(void* p, int64_t at, int64_t end, const float (&v)[8]) {
    if constexpr (TYPE == MARL_F32) {
        float* f = static_cast<float*>(p) + at;
        if (at + 8 <= end) {
            *reinterpret_cast<f32x4_a4*>(f) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_a4*>(f + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (at + k < end) f[k] = v[k];
        }
    } else {
        uint16_t* h = static_cast<uint16_t*>(p) + at;
        if (at + 8 <= end) {
            u32x4 u;
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = (uint32_t)to_half_type<TYPE>(v[2 * k]) | ((uint32_t)to_half_type<TYPE>(v[2 * k + 1]) << 16);
            *reinterpret_cast<u32x4_a2*>(h) = u;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (at + k < end) h[k] = to_half_type<TYPE>(v[k]);
        }
    }
}

// Passes over [rows][blocks of 32] have four lanes per block and one thread number for them all, so a call holds at most
// 2^30 - 64 blocks (a launch, whole workgroups of 256, holds fewer than 2^32 threads).  `thread` to row, block of the row, and quarter of the block:
__device__ __forceinline__ void split_block(uint32_t thread, uint32_t per_row, int64_t& row, int& b, int& quarter) {
    const uint32_t block = thread >> 2, r = block / per_row;
    row = r;
    b = (int)(block - r * per_row);
    quarter = (int)(thread & 3);
}
static inline bool too_many_blocks(int64_t rows, int64_t cols) {
    return rows >= ((int64_t)1 << 30) || (uint64_t)rows * lb_blocks(cols) > ((uint64_t)1 << 30) - 64;
}
static inline uint32_t block_grid(int64_t rows, int64_t cols) {  // workgroups of 256 threads
    return (uint32_t)(((uint64_t)rows * lb_blocks(cols) * 4 + 255) / 256);
}

}  // namespace oc
