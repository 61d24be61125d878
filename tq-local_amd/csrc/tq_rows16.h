// tq_rows16.h -- 16-bit matrix-core products over rows of 128 elements in LDS, shared by the prompts' attention and that over packed tiles (gfx950).
//
// A row is 256 bytes, its 16-byte chunk c at slot c ^ swizzle(token): the low four bits of the token with the bits 0-1 on top, so
// that the 16 rows of an operand's read, and the 4 x 2 rows that ds_read_b64_tr_b16 turns around, meet every bank once.

#pragma once

#include "tq_common.h"

namespace tqr {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
union Frag {
    uint32_t u[4];
    uint4 q;
    s16x4 t[2];
    bf16x8 b;
    f16x8 f;
};

__device__ __forceinline__ f32x16 mfma_f16(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.f, b.f, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_bf16(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.b, b.b, c, 0, 0, 0);
}
// two fp32 values, nearest even
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const f32x2 p = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, f16x2));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const f32x2 p = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
// 2^x (v_exp_f32, 1 ulp; 2^-inf = 0)
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int swizzle(int token) { return ((token & 3) << 2) | ((token >> 2) & 3); }

// 16 bytes a lane from memory to LDS, and the wait for them
__device__ __forceinline__ void load_lds16(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)g,
                                     (__attribute__((address_space(3))) uint32_t*)l, 16, 0, 0);
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ s16x4 read_tr(const uint8_t* l) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)l);
}
// Byte offset of what a lane gives ds_read_b64_tr_b16 for dims 32 d + (0..31) of the tokens 8 e + 4 h + (0..3) of 16 rows: 16 lanes
// read 4 tokens x 16 dims, and each ends with one dim's 4 tokens.
__device__ __forceinline__ int value_offset(int d, int e, int lane) {
    const int tok = 8 * e + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    return tok * 256 + ((chunk ^ swizzle(tok)) << 4) + 8 * (lane & 1);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace tqr
