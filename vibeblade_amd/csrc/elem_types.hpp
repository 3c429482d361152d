// Element types of activations (fp32, fp16, bf16) for the ops that take each.
#pragma once

#include "vb_common.hpp"

namespace vb {

enum : int32_t { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };

inline bool elem_type(int32_t t) { return t == ELEM_F32 || t == ELEM_F16 || t == ELEM_BF16; }
inline int64_t elem_bytes(int32_t t) { return t == ELEM_F32 ? 4 : 2; }

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }

// To the nearest bf16, ties to even; NaN stays NaN (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t f32_bf16x2(float lo, float hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
__device__ __forceinline__ uint16_t f32_bf16(float v) { return static_cast<uint16_t>(f32_bf16x2(v, 0.f)); }

// Element i of a tensor of a type known at run time (the same in every lane).
__device__ __forceinline__ float elem_ld(const void* p, int64_t i, int type) {
    return type == ELEM_F32 ? static_cast<const float*>(p)[i]
         : type == ELEM_F16 ? static_cast<float>(static_cast<const _Float16*>(p)[i])
                            : bf16_f32(static_cast<const uint16_t*>(p)[i]);
}

__device__ __forceinline__ void elem_st(void* p, int64_t i, int type, float v) {
    if (type == ELEM_F32) static_cast<float*>(p)[i] = v;
    else if (type == ELEM_F16) static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
    else static_cast<uint16_t*>(p)[i] = f32_bf16(v);
}

}  // namespace vb
