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

// A kernel that is to keep at least n wavefronts on a SIMD: 512 / n registers for each lane.
#define OVL_LANE_WAVES(n) __attribute__((amdgpu_waves_per_eu(n)))

namespace ovl_lane {

// Work items of one launch: HIP takes fewer than 2^32.
constexpr uint64_t MOST_WORK_ITEMS = 0xffffffff;

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

// max(x, 0) in one instruction; 0 for NaN.
__device__ __forceinline__ float positive(float x) { return __builtin_amdgcn_fmed3f(x, 0.0f, __builtin_inff()); }

// The value is in a register at this point of the program: its computation does not move behind it.
template <typename X> __device__ __forceinline__ void keep(X& x) { asm volatile("" : "+v"(x)); }
// A number that the whole wavefront shares, as one of which the compiler knows nothing more: what is made of it is made here
// and not kept from earlier.
__device__ __forceinline__ uint32_t anew(uint32_t x) {
    asm volatile("" : "+s"(x));
    return x;
}

// A number that is the same in all lanes of a wavefront, as one that the compiler knows to be.
__device__ __forceinline__ uint32_t wavefront(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// What the lanes of a wavefront wrote to LDS before is what they read after: no other wavefront is waited for.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Memory from an address that the whole wavefront shares: accesses add a lane's 32-bit offset and one that the wavefront
// shares, both in bytes, inside the instruction.  No bounds are set: the offsets have to stay inside the tensor.
struct region {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ explicit region(const void* base)
        : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0xffffffff, 0x00020000)) {}
    template <typename T> __device__ __forceinline__ T load(uint32_t own, uint32_t shared) const {
        if constexpr (sizeof(T) == 2)
            return __builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rsrc, own, shared, 0));
        else
            return __builtin_bit_cast(T, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rsrc, own, shared, 0));
    }
    template <typename T> __device__ __forceinline__ void store(T x, uint32_t own, uint32_t shared) const {
        if constexpr (sizeof(T) == 2)
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), rsrc, own, shared, 0);
        else
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), rsrc, own, shared, 0);
    }
};

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

// A value per lane of a row of sixteen lanes, for all lanes of the row: at(n) is lane n's, taken by the instruction that
// uses it.  n is constant once the loops around it are unrolled.
struct row_values {
    float own;
    __device__ __forceinline__ explicit row_values(float x) : own(x) {}
    __device__ __forceinline__ float at(uint32_t n) const {
        switch (n) {
            case 0: return dpp_<0x150>(own);
            case 1: return dpp_<0x151>(own);
            case 2: return dpp_<0x152>(own);
            case 3: return dpp_<0x153>(own);
            case 4: return dpp_<0x154>(own);
            case 5: return dpp_<0x155>(own);
            case 6: return dpp_<0x156>(own);
            case 7: return dpp_<0x157>(own);
            case 8: return dpp_<0x158>(own);
            case 9: return dpp_<0x159>(own);
            case 10: return dpp_<0x15a>(own);
            case 11: return dpp_<0x15b>(own);
            case 12: return dpp_<0x15c>(own);
            case 13: return dpp_<0x15d>(own);
            case 14: return dpp_<0x15e>(own);
            default: return dpp_<0x15f>(own);
        }
    }
};

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
