// Test infrastructure: stands in for opveclib_amd/csrc/ovl_lane.h when the state space and norm kernels are compiled for
// the host (see ovl_device.h in this directory): the element types in software, the hardware's exponential, logarithm and
// reciprocals from the host C library, and the lane moves through the table that the threads of a wavefront share.
#ifndef OVL_LANE_H_
#define OVL_LANE_H_

#include "ovl_device.h"

static inline uint32_t min(uint32_t a, uint32_t b) { return a < b ? a : b; }
static inline uint32_t max(uint32_t a, uint32_t b) { return a > b ? a : b; }

#define OVL_LANE_WAVES(n)

namespace ovl_lane {

// few, so that calls that take several launches are tried
constexpr uint64_t MOST_WORK_ITEMS = 2048;

struct bf16 { uint16_t bits; };
struct f16 { uint16_t bits; };

static inline uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }
static inline float float_of(uint32_t x) { return __builtin_bit_cast(float, x); }

template <typename T> static inline float widen(T x);
template <> inline float widen<float>(float x) { return x; }
template <> inline float widen<bf16>(bf16 x) { return float_of((uint32_t)x.bits << 16); }
template <> inline float widen<f16>(f16 x) {
    const uint32_t sign = (uint32_t)(x.bits & 0x8000u) << 16, exponent = (x.bits >> 10) & 31u, fraction = x.bits & 1023u;
    if (exponent == 31u) return float_of(sign | 0x7f800000u | (fraction << 13));
    const float magnitude = exponent == 0u ? ldexpf((float)fraction, -24) : ldexpf((float)(fraction + 1024u), (int)exponent - 25);
    return sign ? -magnitude : magnitude;
}

template <typename T> static inline T narrow(float x);
template <> inline float narrow<float>(float x) { return x; }
template <> inline bf16 narrow<bf16>(float x) {
    const uint32_t b = bits_of(x);
    if (x != x) return bf16{(uint16_t)((b >> 16) | 0x40u)};
    return bf16{(uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16)};
}
template <> inline f16 narrow<f16>(float x) {
    const uint16_t sign = (uint16_t)((bits_of(x) >> 16) & 0x8000u);
    const float a = fabsf(x);
    if (x != x) return f16{(uint16_t)(sign | 0x7e00u)};
    if (a >= 65520.0f) return f16{(uint16_t)(sign | 0x7c00u)};
    if (a < 0x1p-14f) return f16{(uint16_t)(sign | (uint16_t)nearbyintf(ldexpf(a, 24)))};
    int e;
    const float m = frexpf(a, &e);                                   // a = m 2^e, m in [0.5, 1)
    uint32_t units = (uint32_t)nearbyintf(ldexpf(m, 11));             // 1024 .. 2048
    return f16{(uint16_t)(sign | (((uint32_t)(e + 14) << 10) + (units - 1024u)))};
}

static inline uint32_t e4m3(float x) {
    const uint32_t sign = (bits_of(x) >> 24) & 0x80u;
    const float a = fabsf(x);
    if (x != x) return sign | 0x7fu;
    if (a < 0x1p-6f) return sign | (uint32_t)nearbyintf(ldexpf(a, 9));
    int e;
    const float m = frexpf(a, &e);
    const uint32_t units = (uint32_t)nearbyintf(ldexpf(m, 4));        // 8 .. 16
    const uint32_t code = ((uint32_t)(e + 6) << 3) + (units - 8u);
    return sign | (code > 0x7eu ? 0x7eu : code);
}
static inline uint32_t e4m3x4(float a, float b, float c, float d) {
    return e4m3(a) | (e4m3(b) << 8) | (e4m3(c) << 16) | (e4m3(d) << 24);
}

static inline float exp2_(float x) { return exp2f(x); }
static inline float log2_(float x) { return log2f(x); }
static inline float rcp_(float x) { return 1.0f / x; }
static inline float rsq_(float x) { return 1.0f / sqrtf(x); }

static inline float positive(float x) { return x > 0.0f ? x : 0.0f; }
template <typename X> static inline void keep(X&) {}
static inline uint32_t anew(uint32_t x) { return x; }

static inline uint32_t wavefront(uint32_t x) { return x; }

static inline void wave_sync() { pthread_barrier_wait(&ovl_emulated_wave_barrier[threadIdx.x / 64u]); }

struct region {
    char* base;
    explicit region(const void* base_) : base(const_cast<char*>(static_cast<const char*>(base_))) {}
    template <typename T> T load(uint32_t own, uint32_t shared) const { return *reinterpret_cast<const T*>(base + own + (uint64_t)shared); }
    template <typename T> void store(T x, uint32_t own, uint32_t shared) const { *reinterpret_cast<T*>(base + own + (uint64_t)shared) = x; }
};

// The value `from` names, by lane; zero where it is negative.
template <typename F> static inline float move(float x, F from) {
    const uint32_t t = threadIdx.x, wave = t / 64u, lane = t % 64u;
    ovl_emulated_lane_values[t] = bits_of(x);
    pthread_barrier_wait(&ovl_emulated_wave_barrier[wave]);
    const int source = from((int)lane);
    const float result = source < 0 ? 0.0f : float_of((uint32_t)ovl_emulated_lane_values[wave * 64u + (uint32_t)source]);
    pthread_barrier_wait(&ovl_emulated_wave_barrier[wave]);
    return result;
}

template <int K> static inline float quad_from(float x) { return move(x, [](int l) { return (l & ~3) + K; }); }
static inline float quad_xor1(float x) { return move(x, [](int l) { return l ^ 1; }); }
static inline float quad_xor2(float x) { return move(x, [](int l) { return l ^ 2; }); }
template <int N> static inline float row_down(float x) { return move(x, [](int l) { return (l & 15) + N < 16 ? l + N : -1; }); }
template <int N> static inline float row_up(float x) { return move(x, [](int l) { return (l & 15) >= N ? l - N : -1; }); }
template <int N> static inline float row_round(float x) {
    return move(x, [](int l) { return (l & ~15) + ((l + 16 - N) & 15); });
}

struct row_values {
    float all[16];
    explicit row_values(float x) {
        const uint32_t t = threadIdx.x, wave = t / 64u;
        ovl_emulated_lane_values[t] = bits_of(x);
        pthread_barrier_wait(&ovl_emulated_wave_barrier[wave]);
        for (uint32_t n = 0; n < 16u; ++n) all[n] = float_of((uint32_t)ovl_emulated_lane_values[t / 16u * 16u + n]);
        pthread_barrier_wait(&ovl_emulated_wave_barrier[wave]);
    }
    float at(uint32_t n) const { return all[n]; }
};

static inline void swap_halves(float& a, float& b) {
    const uint32_t lane = threadIdx.x % 64u;
    const float other = move(b, [](int l) { return l ^ 32; });       // for the upper half of a
    const float mine = move(a, [](int l) { return l ^ 32; });        // for the lower half of b
    if (lane >= 32u) a = other; else b = mine;
}
static inline void swap_rows(float& a, float& b) {
    const uint32_t lane = threadIdx.x % 64u;
    const float other = move(b, [](int l) { return l ^ 16; });
    const float mine = move(a, [](int l) { return l ^ 16; });
    if (lane & 16u) a = other; else b = mine;
}

}  // namespace ovl_lane

#endif  // OVL_LANE_H_
