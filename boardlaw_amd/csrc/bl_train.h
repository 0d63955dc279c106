// bl_train.h -- device helpers shared by the learner-step operators (bl_logprobs.hip, bl_norm.hip, bl_ortho.hip): element types and
// their vector accesses, reductions over 16 lanes and over a wave, the exponential.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "../../include/boardlaw_amd.h"
#include "bl_dispatch.h"

namespace bltrain {

typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T, int N> using vec = typename VecOf<T, N>::type;

// VEC consecutive elements as floats; `p` is aligned to VEC elements (VEC == 1: to one)
template <typename T, int VEC> __device__ __forceinline__ void load(const T* p, float (&o)[VEC]) {
    if constexpr (VEC == 1) o[0] = (float)p[0];
    else if constexpr (VEC * sizeof(T) <= 16) {
        const vec<T, VEC> v = *(const vec<T, VEC>*)p;
#pragma unroll
        for (int i = 0; i < VEC; i++) o[i] = (float)v[i];
    } else {
        constexpr int H = 16 / sizeof(T);
#pragma unroll
        for (int b = 0; b < VEC; b += H) {
            const vec<T, H> v = *(const vec<T, H>*)(p + b);
#pragma unroll
            for (int i = 0; i < H; i++) o[b + i] = (float)v[i];
        }
    }
}
// ... and back, each rounded once, to nearest even
template <typename T, int VEC> __device__ __forceinline__ void store(T* p, const float (&o)[VEC]) {
    if constexpr (VEC == 1) p[0] = (T)o[0];
    else if constexpr (VEC * sizeof(T) <= 16) {
        vec<T, VEC> v;
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = (T)o[i];
        *(vec<T, VEC>*)p = v;
    } else {
        constexpr int H = 16 / sizeof(T);
#pragma unroll
        for (int b = 0; b < VEC; b += H) {
            vec<T, H> v;
#pragma unroll
            for (int i = 0; i < H; i++) v[i] = (T)o[b + i];
            *(vec<T, H>*)(p + b) = v;
        }
    }
}

// ---- reductions: every lane of the group gets the result; fixed order, so the same inputs give the same bits ----
template <int CTRL> __device__ __forceinline__ int ror(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
template <int CTRL> __device__ __forceinline__ float ror(float v) { return __builtin_bit_cast(float, ror<CTRL>(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ float lane_f(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ unsigned lane_u(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }

struct Sum { static __device__ __forceinline__ float f(float a, float b) { return a + b; } };
struct Max { static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); } };
// G = 4: a quad; G = 16: one DPP row; G = 32: two, through a shuffle; G = 64: the wave (row rotations, then the four rows' values through scalar registers)
template <int G, typename Op> __device__ __forceinline__ float reduce(float v) {
    if constexpr (G == 4) { v = Op::f(v, ror<0xb1>(v)); return Op::f(v, ror<0x4e>(v)); }
    v = Op::f(v, ror<0x128>(v)); v = Op::f(v, ror<0x124>(v)); v = Op::f(v, ror<0x122>(v)); v = Op::f(v, ror<0x121>(v));
    if constexpr (G == 32) v = Op::f(v, __shfl_xor(v, 16));
    if constexpr (G == 64) v = Op::f(Op::f(lane_f(v, 0), lane_f(v, 16)), Op::f(lane_f(v, 32), lane_f(v, 48)));
    return v;
}
template <int G> __device__ __forceinline__ unsigned reduce_max_u(unsigned v) {
    v = max(v, (unsigned)ror<0x128>((int)v)); v = max(v, (unsigned)ror<0x124>((int)v));
    v = max(v, (unsigned)ror<0x122>((int)v)); v = max(v, (unsigned)ror<0x121>((int)v));
    if constexpr (G == 32) v = max(v, (unsigned)__shfl_xor((int)v, 16));
    if constexpr (G == 64) v = max(max(lane_u(v, 0), lane_u(v, 16)), max(lane_u(v, 32), lane_u(v, 48)));
    return v;
}

// e^x for x <= 0 as one v_exp_f32: its argument x * log2(e) is rounded once, so the relative error is |x| 2^-24 and an ulp -- what the
// rounding of x = (logit - maximum) itself costs.  e^-inf = 0, NaN stays.
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

}  // namespace bltrain
