// Root-mean-square norm of rows for gfx950 behind the C ABI of include/ovl_norm.h: with the residual's addition, with an
// 8-bit output and its scales, and the gradient.
//
// Mathematics.  s = x + residual as stored, rstd = 1 / sqrt(mean s^2 + eps), y = s rstd w.  With t = dy w and n = s rstd
// the gradient is ds = rstd (t - n mean(t n)) + dsummed, dw = sum over rows of dy n.
//
// Work layout: LANES lanes share a row (a wavefront, four or sixteen of them) and hold all of it in registers, HELD
// vectors of eight columns per lane, so everything is read once and written once: the kernels are bound by memory.  The
// statistics of a row are one exchange between its wavefronts, the largest result for a scale that spans the row another
// (4096 rows of 20000 columns in bf16 with the residual: 155 us with the second, else 149).  Rows need not start on vector
// boundaries: the vectors are accessed with the alignment of an element, a row's last, partial vector element by element.
//
// Measured: 16384 rows of 8192 columns in bf16 with the residual's addition, to 8 bits with a scale per 128 columns, 175 us
// (939 MB, 5.4 TB/s, what a large copy reaches); 8192 rows of 4096 in bf16 with float32 sums, forward 74 us (5.4 TB/s),
// backward 105 us (5.1 TB/s) and 5 us for the weights' sums; 5 rows of 4096 to 8 bits 4.0 us (latency).
#include <math.h>
#include <stdint.h>
#include <string>
#include <type_traits>

#include "ovl_lane.h"
#include "ovl_norm.h"

#define OVL_OK 0
#define OVL_EHIP 4
#define OVL_EINVAL 6

using ovl_lane::bf16;
using ovl_lane::f16;
using ovl_lane::narrow;
using ovl_lane::widen;

namespace {

constexpr int VEC = 8;
constexpr float E4M3_MAX = 448.0f;

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) pack { T v[VEC]; };

// Eight columns from `c` on of a row, zero past its end.
template <typename T>
__device__ __forceinline__ pack<T> load_raw(const T* row, uint32_t c, uint32_t columns) {
    if (c + VEC <= columns) return *reinterpret_cast<const pack<T>*>(row + c);
    pack<T> raw;
#pragma unroll
    for (int i = 0; i < VEC; ++i) raw.v[i] = c + i < columns ? row[c + i] : narrow<T>(0.0f);
    return raw;
}

template <typename T>
__device__ __forceinline__ void widen_vec(float (&to)[VEC], const pack<T>& raw) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) to[i] = widen<T>(raw.v[i]);
}

template <typename T>
__device__ __forceinline__ void load_vec(float (&to)[VEC], const T* row, uint32_t c, uint32_t columns) {
    widen_vec<T>(to, load_raw<T>(row, c, columns));
}

template <typename T>
__device__ __forceinline__ void store_vec(const float (&x)[VEC], T* row, uint32_t c, uint32_t columns) {
    if (c + VEC <= columns) {
        pack<T> out;
#pragma unroll
        for (int i = 0; i < VEC; ++i) out.v[i] = narrow<T>(x[i]);
        *reinterpret_cast<pack<T>*>(row + c) = out;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < columns) row[c + i] = narrow<T>(x[i]);
    }
}

// The weights are float32 or of the rows' type.
template <typename T>
__device__ __forceinline__ void load_weights(float (&to)[VEC], const void* weight, bool wide, uint32_t c, uint32_t columns) {
    if (wide) load_vec<float>(to, static_cast<const float*>(weight), c, columns);
    else load_vec<T>(to, static_cast<const T*>(weight), c, columns);
}

struct add_op { __device__ static __forceinline__ float of(float a, float b) { return a + b; } };
struct max_op { __device__ static __forceinline__ float of(float a, float b) { return fmaxf(a, b); } };

// Over the sixteen lanes of a row of lanes, resp. over the wavefront; every lane receives the result.
template <typename OP> __device__ __forceinline__ float row_all(float x) {
    x = OP::of(x, ovl_lane::row_round<8>(x));
    x = OP::of(x, ovl_lane::row_round<4>(x));
    x = OP::of(x, ovl_lane::row_round<2>(x));
    return OP::of(x, ovl_lane::row_round<1>(x));
}
template <typename OP> __device__ __forceinline__ float wave_all(float x) {
    x = row_all<OP>(x);
    float a = x, b = x;
    ovl_lane::swap_rows(a, b);
    x = OP::of(a, b);
    a = x;
    b = x;
    ovl_lane::swap_halves(a, b);
    return OP::of(a, b);
}

// Over all lanes of a row of the matrix; every lane receives the result.  `lds`, a number per wavefront, is not read again
// before the next barrier after this call, so two calls need a barrier, or two places, between them.
template <int LANES, typename OP>
__device__ __forceinline__ float across(float x, float* lds) {
    x = wave_all<OP>(x);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        if ((threadIdx.x & 63u) == 0u) lds[threadIdx.x / 64u] = x;
        __syncthreads();
        x = lds[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) x = OP::of(x, lds[i]);
    }
    return x;
}

// Two sums at a time, in the same way.
template <int LANES>
__device__ __forceinline__ void across(float& first, float& second, float (*lds)[2]) {
    first = wave_all<add_op>(first);
    second = wave_all<add_op>(second);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        const uint32_t wave = threadIdx.x / 64u;
        if ((threadIdx.x & 63u) == 0u) { lds[wave][0] = first; lds[wave][1] = second; }
        __syncthreads();
        first = lds[0][0];
        second = lds[0][1];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) { first += lds[i][0]; second += lds[i][1]; }
    }
}

struct norm_args {
    uint32_t rows, columns;
    float eps, over_columns;
    const void *x, *residual, *weight;
    int64_t x_stride, residual_stride;
    int32_t wide_weight;
};

// R: the type of the residual and of s.  QUANTIZED: q and scales instead of y; GROUPED: a scale for each 128 columns
// (which are the 16 lanes of one row of lanes), else one for the row.
template <typename T, typename R, int LANES, int HELD, bool QUANTIZED, bool GROUPED>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256)
norm_forward_kernel(norm_args p, T* y, R* summed, uint8_t* q, float* scales) {
    constexpr uint32_t PER = LANES > 256 ? 1 : 256 / LANES;     // rows of a workgroup
    __shared__ float lds[2][LANES / 64];
    const uint32_t lane = threadIdx.x % LANES;
    const uint64_t row = (uint64_t)blockIdx.x * PER + threadIdx.x / LANES;
    if (row >= p.rows) return;              // with more than one row per workgroup there is no barrier
    const T* x = static_cast<const T*>(p.x) + (int64_t)row * p.x_stride;
    float s[HELD][VEC];
#pragma unroll
    for (int h = 0; h < HELD; ++h) load_vec<T>(s[h], x, (h * LANES + lane) * VEC, p.columns);
    if (p.residual != nullptr) {
        const R* residual = static_cast<const R*>(p.residual) + (int64_t)row * p.residual_stride;
        R* to = summed + row * p.columns;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const uint32_t c = (h * LANES + lane) * VEC;
            float more[VEC];
            load_vec<R>(more, residual, c, p.columns);
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[h][i] = widen<R>(narrow<R>(s[h][i] + more[i]));
            store_vec<R>(s[h], to, c, p.columns);
        }
    }
    float squares = 0.0f;
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < VEC; ++i) squares = fmaf(s[h][i], s[h][i], squares);
    float w[HELD][VEC];
#pragma unroll
    for (int h = 0; h < HELD; ++h) load_weights<T>(w[h], p.weight, p.wide_weight, (h * LANES + lane) * VEC, p.columns);
    squares = across<LANES, add_op>(squares, lds[0]);
    const float rstd = ovl_lane::rsq_(fmaf(squares, p.over_columns, p.eps));
    if constexpr (!QUANTIZED) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            float out[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) out[i] = s[h][i] * rstd * w[h][i];
            store_vec<T>(out, y + row * p.columns, (h * LANES + lane) * VEC, p.columns);
        }
        return;
    }
    float row_top = 0.0f;                   // s becomes y
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            s[h][i] = s[h][i] * rstd * w[h][i];
            if (!GROUPED) row_top = fmaxf(row_top, fabsf(s[h][i]));
        }
    // The smallest scale is the smallest normal number: the last bits of one below would not be there.  y is divided by it: a
    // product with a rounded reciprocal would move values in the middle of two e4m3 numbers, so the reciprocal is carried to
    // twice the precision, which makes the product the rounded quotient, but for the last bit of one in a million.  Its first
    // part is too small by more than its error, so that the second is positive and zeros keep their sign; the second is
    // subnormal for the largest scales, where the eight bits that it has left suffice.
    float scale, high, low;
    auto scale_by = [&](float top) {
        scale = top > 0.0f ? fmaxf(top / E4M3_MAX, 0x1p-126f) : 1.0f;
        high = ovl_lane::rcp_(scale) * (1.0f - 0x1p-22f);
        low = scale <= 0x1.fffffep+127f ? fmaf(-high, scale, 1.0f) * high : 0.0f;
    };
    if (!GROUPED) {
        scale_by(across<LANES, max_op>(row_top, lds[1]));
        if (lane == 0u) scales[row] = scale;
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const uint32_t c = (h * LANES + lane) * VEC;
        if (GROUPED) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) top = fmaxf(top, fabsf(s[h][i]));
            scale_by(row_all<max_op>(top));
            const uint32_t group = c / 128u, groups = (p.columns + 127u) / 128u;
            if ((lane & 15u) == 0u && group < groups) scales[row * groups + group] = scale;
        }
        float out[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = fmaf(s[h][i], high, s[h][i] * low);
        struct __attribute__((packed, aligned(1))) bytes { uint32_t v[2]; } packed;
        packed.v[0] = ovl_lane::e4m3x4(out[0], out[1], out[2], out[3]);
        packed.v[1] = ovl_lane::e4m3x4(out[4], out[5], out[6], out[7]);
        uint8_t* to = q + row * p.columns + c;
        if (c + VEC <= p.columns) *reinterpret_cast<bytes*>(to) = packed;
        else
#pragma unroll
            for (uint32_t i = 0; i < VEC; ++i)
                if (c + i < p.columns) to[i] = (uint8_t)(packed.v[i / 4u] >> (8u * (i % 4u)));
    }
}

struct norm_gradient_args {
    const void *d_y, *d_summed;
    int64_t d_y_stride, d_summed_stride;
    void *d_x, *d_residual;
    float* part;                            // [rows of parts][columns]
};

// A team of LANES lanes takes rows `team`, team + teams, ... and keeps its sums for the weights in registers.
template <typename T, typename R, int LANES, int HELD>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256)
norm_backward_kernel(norm_args p, norm_gradient_args g, uint32_t teams) {
    constexpr uint32_t PER = LANES > 256 ? 1 : 256 / LANES;
    __shared__ float lds[2][LANES / 64][2];
    const uint32_t lane = threadIdx.x % LANES;
    const uint32_t team = blockIdx.x * PER + threadIdx.x / LANES;
    if (team >= teams) return;              // with more than one team per workgroup there is no barrier
    float dw[HELD][VEC];
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[h][i] = 0.0f;
    // a row's inputs are read one row ahead where there are registers for it (8192 rows of 4096 columns, bf16 with float32
    // sums: 106 us, else 113).  A team of 1024 lanes has 128 registers for each and does not read ahead (4096 rows of 16384:
    // 208 us, 342 with rows ahead in scratch memory); with four vectors per lane it reads a row twice, the second time from
    // the L2, and holds no inputs in between (2048 rows of 32768: 284 us, 3.8 TB/s, 424 with them in scratch memory; 9 to 13
    // registers of each lane still go there).
    constexpr bool AHEAD = HELD <= 2 && LANES <= 256, LEAN = HELD > 2 && LANES > 256;
    float w[HELD][VEC];
    if (!LEAN)
#pragma unroll
        for (int h = 0; h < HELD; ++h) load_weights<T>(w[h], p.weight, p.wide_weight, (h * LANES + lane) * VEC, p.columns);
    struct inputs { pack<R> s[HELD]; pack<T> d_y[HELD]; pack<R> d_summed[HELD]; };
    auto fetch = [&](inputs& to, uint64_t row) {
        const R* s = static_cast<const R*>(p.x) + (int64_t)row * p.x_stride;
        const T* d_y = static_cast<const T*>(g.d_y) + (int64_t)row * g.d_y_stride;
        const R* d_summed = static_cast<const R*>(g.d_summed) + (int64_t)row * g.d_summed_stride;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const uint32_t c = (h * LANES + lane) * VEC;
            to.s[h] = load_raw<R>(s, c, p.columns);
            to.d_y[h] = load_raw<T>(d_y, c, p.columns);
            if (!LEAN && g.d_summed != nullptr) to.d_summed[h] = load_raw<R>(d_summed, c, p.columns);
        }
    };
    float n[HELD][VEC], t[HELD][VEC];
    auto again = [&](int h, uint64_t row) {
        uint32_t c = (h * LANES + lane) * VEC;
        ovl_lane::keep(c);                  // else the addresses of all its vectors are kept over the rows, in scratch memory
        load_vec<R>(n[h], static_cast<const R*>(p.x) + (int64_t)row * p.x_stride, c, p.columns);
        load_vec<T>(t[h], static_cast<const T*>(g.d_y) + (int64_t)row * g.d_y_stride, c, p.columns);
        load_weights<T>(w[h], p.weight, p.wide_weight, c, p.columns);
    };
    uint32_t turn = 0;
    inputs now, next;
    if (AHEAD) fetch(next, team);
    for (uint64_t row = team; row < p.rows; row += teams, turn ^= 1u) {
        if (AHEAD) {
            now = next;
            if (row + teams < p.rows) fetch(next, row + teams);
        } else if (!LEAN) {
            fetch(now, row);
        }
        // one exchange for both: rstd comes from the sum of s^2, and mean(t n) = rstd mean(t s)
        float squares = 0.0f, dot = 0.0f;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (LEAN) {
                again(h, row);
            } else {
                widen_vec<R>(n[h], now.s[h]);
                widen_vec<T>(t[h], now.d_y[h]);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                squares = fmaf(n[h][i], n[h][i], squares);
                dot = fmaf(t[h][i] * w[h][i], n[h][i], dot);
            }
            if (LEAN) __builtin_amdgcn_sched_barrier(0);
        }
        across<LANES>(squares, dot, lds[turn]);
        const float rstd = ovl_lane::rsq_(fmaf(squares, p.over_columns, p.eps));
        const float mean = dot * rstd * p.over_columns;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            uint32_t c = (h * LANES + lane) * VEC;
            float out[VEC];
            if (LEAN) {
                again(h, row);
                ovl_lane::keep(c);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float unit = n[h][i] * rstd;
                dw[h][i] = fmaf(t[h][i], unit, dw[h][i]);
                out[i] = rstd * fmaf(-mean, unit, t[h][i] * w[h][i]);
            }
            if (g.d_summed != nullptr) {
                float more[VEC];
                if (LEAN) load_vec<R>(more, static_cast<const R*>(g.d_summed) + (int64_t)row * g.d_summed_stride, c, p.columns);
                else widen_vec<R>(more, now.d_summed[h]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) out[i] += more[i];
            }
            if (g.d_x != nullptr) store_vec<T>(out, static_cast<T*>(g.d_x) + row * p.columns, c, p.columns);
            if (g.d_residual != nullptr) store_vec<R>(out, static_cast<R*>(g.d_residual) + row * p.columns, c, p.columns);
            if (LEAN) __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        store_vec<float>(dw[h], g.part + (uint64_t)team * p.columns, (h * LANES + lane) * VEC, p.columns);
}

// Adds the teams' parts up: 64 columns per workgroup, sixteen wavefronts share the parts, in a fixed order.
constexpr uint32_t SHARES = 16;
template <typename W>
__global__ void __launch_bounds__(64 * SHARES)
norm_sum_kernel(const float* part, uint32_t columns, uint32_t teams, W* d_weight) {
    __shared__ float lds[SHARES][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u, c = blockIdx.x * 64u + lane;
    float sum = 0.0f;
    if (c < columns)
#pragma unroll 8
        for (uint32_t k = wave; k < teams; k += SHARES) sum += part[(uint64_t)k * columns + c];
    lds[wave][lane] = sum;
    __syncthreads();
    if (wave == 0u && c < columns) {
#pragma unroll
        for (uint32_t i = 1; i < SHARES; ++i) sum += lds[i][lane];
        d_weight[c] = narrow<W>(sum);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------

thread_local std::string g_last_error;

int fail(const std::string& detail) {
    g_last_error = detail;
    return OVL_EINVAL;
}

int after_launch(const char* who) {
    const hipError_t err = hipPeekAtLastError();
    if (err != hipSuccess) {
        (void)hipGetLastError();
        g_last_error = std::string(who) + ": " + hipGetErrorString(err);
        return OVL_EHIP;
    }
    return OVL_OK;
}

bool known(int32_t dtype) { return dtype == OVL_NORM_FLOAT16 || dtype == OVL_NORM_FLOAT32 || dtype == OVL_NORM_BFLOAT16; }

int check(const char* who, const ovl_norm* p) {
    const std::string name(who);
    if (p == nullptr) return fail(name + ": null norm");
    if (p->rows == 0 || p->columns == 0) return fail(name + ": sizes must be positive");
    if (p->columns > 32768u) return fail(name + ": at most 32768 columns");
    if (!known(p->dtype)) return fail(name + ": unknown element type");
    if (p->residual_dtype != p->dtype && p->residual_dtype != OVL_NORM_FLOAT32) return fail(name + ": the residual must be of the rows' type or float32");
    if (p->weight_dtype != p->dtype && p->weight_dtype != OVL_NORM_FLOAT32) return fail(name + ": the weight must be of the rows' type or float32");
    if (p->x == nullptr || p->weight == nullptr) return fail(name + ": null tensor");
    return OVL_OK;
}

norm_args make_args(const ovl_norm* p) {
    return norm_args{p->rows, p->columns, p->eps, 1.0f / (float)p->columns, p->x, p->residual, p->weight, p->x_stride,
                     p->residual_stride, p->weight_dtype == OVL_NORM_FLOAT32 ? 1 : 0};
}

// Lanes per row and vectors per lane: a wavefront up to 2048 columns, four up to 8192, sixteen up to 32768, at most four
// vectors of eight columns per lane.
template <typename F> void by_columns(uint32_t columns, F&& call) {
    const uint32_t vectors = (columns + VEC - 1) / VEC;
#define OVL_NORM_HELD(LANES)                                                                                                   \
    {                                                                                                                         \
        const uint32_t held = (vectors + LANES - 1) / LANES;                                                                  \
        if (held <= 1) call(std::integral_constant<int, LANES>(), std::integral_constant<int, 1>());                          \
        else if (held <= 2) call(std::integral_constant<int, LANES>(), std::integral_constant<int, 2>());                     \
        else call(std::integral_constant<int, LANES>(), std::integral_constant<int, 4>());                                    \
    }
    if (vectors <= 4 * 64) OVL_NORM_HELD(64)
    else if (vectors <= 4 * 256) OVL_NORM_HELD(256)
    else OVL_NORM_HELD(1024)
#undef OVL_NORM_HELD
}

template <typename F> void by_types(const ovl_norm* p, F&& call) {
    const bool wide = p->residual_dtype == OVL_NORM_FLOAT32;
    switch (p->dtype) {
        case OVL_NORM_FLOAT32: call(float(), float()); break;
        case OVL_NORM_FLOAT16: if (wide) call(f16(), float()); else call(f16(), f16()); break;
        default: if (wide) call(bf16(), float()); else call(bf16(), bf16()); break;
    }
}

// Calls launch(first row, rows, workgroups) for pieces of the matrix that one launch can take: a row of up to 2048 columns
// is 64 work items, so 2^26 rows are too many.
template <typename F> void by_pieces(uint32_t rows, uint32_t threads, uint32_t per_workgroup, F&& launch) {
    const uint64_t most = ovl_lane::MOST_WORK_ITEMS / threads * per_workgroup;
    for (uint64_t first = 0; first < rows; first += most) {
        const uint32_t here = (uint32_t)(rows - first < most ? rows - first : most);
        launch(first, here, (here + per_workgroup - 1) / per_workgroup);
    }
}

// The arguments of the rows from `first` on.
norm_args piece_of(const ovl_norm* p, uint64_t first, uint32_t rows) {
    norm_args args = make_args(p);
    args.rows = rows;
    const int64_t size = p->dtype == OVL_NORM_FLOAT32 ? 4 : 2, residual_size = p->residual_dtype == OVL_NORM_FLOAT32 ? 4 : 2;
    args.x = static_cast<const char*>(p->x) + (int64_t)first * p->x_stride * size;
    if (p->residual != nullptr) args.residual = static_cast<const char*>(p->residual) + (int64_t)first * p->residual_stride * residual_size;
    return args;
}

template <int LANES> constexpr uint32_t threads_of() { return LANES > 256 ? LANES : 256; }

// Teams of the backward pass: two workgroups per compute unit (of 1024 lanes one); a team's part of the weight gradient
// is written and read once, so few rows get few teams.  Twice as many: 108 us for 103 at 8192 rows of 4096 columns (bf16
// with float32 sums), 125 for 112 at 32768 of 1000, but 63 for 71 at 65536 of 512 all in bf16.
uint32_t teams_for(const ovl_norm* p) {
    const uint32_t most = p->columns <= 2048u ? 2048u : p->columns <= 8192u ? 512u : 256u;
    const uint32_t few = (uint32_t)((p->rows + 3ull) / 4u);
    return few < most ? few : most;
}

}  // namespace

extern "C" {

const char* ovl_norm_last_error(void) { return g_last_error.c_str(); }

int ovl_norm_forward(const ovl_norm* p, void* y, void* summed, void* hip_stream) {
    const int rc = check("ovl_norm_forward", p);
    if (rc != OVL_OK) return rc;
    if (y == nullptr || (p->residual != nullptr && summed == nullptr)) return fail("ovl_norm_forward: null tensor");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    by_types(p, [&](auto t, auto r) {
        typedef decltype(t) T;
        typedef decltype(r) R;
        by_columns(p->columns, [&](auto lanes, auto held) {
            constexpr int LANES = decltype(lanes)::value, HELD = decltype(held)::value;
            constexpr uint32_t THREADS = threads_of<LANES>(), PER = THREADS / LANES;
            by_pieces(p->rows, THREADS, PER, [&](uint64_t first, uint32_t rows, uint32_t workgroups) {
                const norm_args args = piece_of(p, first, rows);
                T* to = static_cast<T*>(y) + first * p->columns;
                R* sum = summed != nullptr ? static_cast<R*>(summed) + first * p->columns : nullptr;
                hipLaunchKernelGGL((norm_forward_kernel<T, R, LANES, HELD, false, false>), dim3(workgroups), dim3(THREADS), 0,
                                   stream, args, to, sum, static_cast<uint8_t*>(nullptr), static_cast<float*>(nullptr));
            });
        });
    });
    return after_launch("ovl_norm_forward");
}

int ovl_norm_forward_quantized(const ovl_norm* p, uint32_t group_columns, void* q, float* scales, void* summed,
                               void* hip_stream) {
    const int rc = check("ovl_norm_forward_quantized", p);
    if (rc != OVL_OK) return rc;
    if (group_columns != 0u && group_columns != 128u)
        return fail("ovl_norm_forward_quantized: a scale spans the row or 128 columns");
    if (q == nullptr || scales == nullptr || (p->residual != nullptr && summed == nullptr))
        return fail("ovl_norm_forward_quantized: null tensor");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    const uint64_t groups = group_columns != 0u ? (p->columns + 127u) / 128u : 1u;
    by_types(p, [&](auto t, auto r) {
        typedef decltype(t) T;
        typedef decltype(r) R;
        by_columns(p->columns, [&](auto lanes, auto held) {
            constexpr int LANES = decltype(lanes)::value, HELD = decltype(held)::value;
            constexpr uint32_t THREADS = threads_of<LANES>(), PER = THREADS / LANES;
            by_pieces(p->rows, THREADS, PER, [&](uint64_t first, uint32_t rows, uint32_t workgroups) {
                const norm_args args = piece_of(p, first, rows);
                R* sum = summed != nullptr ? static_cast<R*>(summed) + first * p->columns : nullptr;
                uint8_t* to = static_cast<uint8_t*>(q) + first * p->columns;
                float* to_scales = scales + first * groups;
                const dim3 grid(workgroups);
                if (group_columns != 0u)
                    hipLaunchKernelGGL((norm_forward_kernel<T, R, LANES, HELD, true, true>), grid, dim3(THREADS), 0, stream, args,
                                       static_cast<T*>(nullptr), sum, to, to_scales);
                else
                    hipLaunchKernelGGL((norm_forward_kernel<T, R, LANES, HELD, true, false>), grid, dim3(THREADS), 0, stream, args,
                                       static_cast<T*>(nullptr), sum, to, to_scales);
            });
        });
    });
    return after_launch("ovl_norm_forward_quantized");
}

uint64_t ovl_norm_workspace_bytes(const ovl_norm* p) {
    if (check("ovl_norm_workspace_bytes", p) != OVL_OK) return 0;
    return (uint64_t)teams_for(p) * p->columns * sizeof(float);
}

int ovl_norm_backward(const ovl_norm* p, const void* d_y, int64_t d_y_stride, const void* d_summed,
                      int64_t d_summed_stride, void* d_x, void* d_residual, void* d_weight, void* workspace,
                      uint64_t workspace_bytes, void* hip_stream) {
    const int rc = check("ovl_norm_backward", p);
    if (rc != OVL_OK) return rc;
    if (d_y == nullptr || d_weight == nullptr) return fail("ovl_norm_backward: null tensor");
    const uint32_t teams = teams_for(p);
    if (workspace == nullptr || workspace_bytes < (uint64_t)teams * p->columns * sizeof(float) ||
        (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0)
        return fail("ovl_norm_backward: workspace too small or not 4-byte aligned");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    const norm_args args = make_args(p);
    norm_gradient_args g{d_y, d_summed, d_y_stride, d_summed_stride, d_x, d_residual, static_cast<float*>(workspace)};
    by_types(p, [&](auto t, auto r) {
        typedef decltype(t) T;
        typedef decltype(r) R;
        by_columns(p->columns, [&](auto lanes, auto held) {
            constexpr int LANES = decltype(lanes)::value, HELD = decltype(held)::value;
            constexpr uint32_t THREADS = threads_of<LANES>(), PER = THREADS / LANES;
            hipLaunchKernelGGL((norm_backward_kernel<T, R, LANES, HELD>), dim3((teams + PER - 1) / PER), dim3(THREADS), 0,
                               stream, args, g, teams);
        });
        const dim3 grid((p->columns + 63u) / 64u);
        if (p->weight_dtype == OVL_NORM_FLOAT32)
            hipLaunchKernelGGL((norm_sum_kernel<float>), grid, dim3(64 * SHARES), 0, stream, static_cast<const float*>(workspace),
                               p->columns, teams, static_cast<float*>(d_weight));
        else
            hipLaunchKernelGGL((norm_sum_kernel<T>), grid, dim3(64 * SHARES), 0, stream, static_cast<const float*>(workspace),
                               p->columns, teams, static_cast<T*>(d_weight));
    });
    return after_launch("ovl_norm_backward");
}

}  // extern "C"
