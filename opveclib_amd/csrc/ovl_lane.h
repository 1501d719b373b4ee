// What the hand-written state space and norm kernels need of the device beyond plain C++: element types, the
// hardware's exponential, logarithm and reciprocal, and moves between the lanes of a wavefront.  A host build of the
// kernels replaces this file as a whole.
//
// Lane moves are executed by all 64 lanes of a wavefront together.  A wavefront is four rows of sixteen lanes, a row
// four quads of four.
#ifndef OVL_LANE_H_
#define OVL_LANE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ovl_lane {

typedef _Float16 f16;
typedef __bf16 bf16;

// float <-> element type; to a narrower type with one rounding to nearest, ties to even
template <typename T> __device__ __forceinline__ float widen(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T narrow(float x) { return (T)x; }

// Four values, each already within the range of the format, as e4m3 bytes (nearest, ties to even); byte 0 is a.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, packed, true);
    return (uint32_t)packed;
}

// 2^x, log2(x), 1/x and 1/sqrt(x) of the hardware, each within one unit in the last place; results in the subnormal
// range are zero.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float rsq_(float x) { return __builtin_amdgcn_rsqf(x); }

template <int CTRL>
__device__ __forceinline__ float dpp_(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// The value of lane K of the own quad.
template <int K> __device__ __forceinline__ float quad_from(float x) { return dpp_<K * 0x55>(x); }
// The value of the lane whose number differs in bit 0, resp. bit 1.
__device__ __forceinline__ float quad_xor1(float x) { return dpp_<0xB1>(x); }
__device__ __forceinline__ float quad_xor2(float x) { return dpp_<0x4E>(x); }
// The value N lanes down (lane + N) or up (lane - N) the own row, zero outside of it, or N lanes round it (lane - N).
template <int N> __device__ __forceinline__ float row_down(float x) { return dpp_<0x100 + N>(x); }
template <int N> __device__ __forceinline__ float row_up(float x) { return dpp_<0x110 + N>(x); }
template <int N> __device__ __forceinline__ float row_round(float x) { return dpp_<0x120 + N>(x); }

// The upper half of the wavefront of `a` changes places with the lower half of `b`.
__device__ __forceinline__ void swap_halves(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                                    false, false);
    a = __builtin_bit_cast(float, (uint32_t)r[0]);
    b = __builtin_bit_cast(float, (uint32_t)r[1]);
}
// Rows 1 and 3 of `a` change places with rows 0 and 2 of `b`.
__device__ __forceinline__ void swap_rows(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                                    false, false);
    a = __builtin_bit_cast(float, (uint32_t)r[0]);
    b = __builtin_bit_cast(float, (uint32_t)r[1]);
}

}  // namespace ovl_lane

#endif  // OVL_LANE_H_
