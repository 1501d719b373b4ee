// Short causal convolution for gfx950 behind the C ABI of include/ovl_ssm.h: forward, backward, one-token step; the error
// text of the library.
//
// Every channel has its own `width` (1 to 4) taps: pre[t] = bias + sum w[k] line[t + k], line = the kept tokens and then
// the sequence, y = pre sigmoid(pre) or pre.  With d = the gradient of pre, dx[t] = sum w[k] d[t + width - 1 - k] and
// dw[k] = sum over t of d[t] line[t + k].
//
// Work layout: a lane owns VEC neighbouring channels (16 bytes where sizes and addresses allow it) and walks along tokens
// with the last inputs in registers, so every input is loaded once but for the few tokens before a walk's first.  All of
// it is bound by memory: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx.  Measured
// on 4 sequences of 4096 tokens, 8192 channels, width 4, bf16 (x a half of a projection): forward 97 to 102 us, 5.3 to 5.5
// TB/s, as much as a large copy reaches; backward 176 to 210 us, 3.9 to 4.6 TB/s; one token of 64 sequences of 4096 channels 3.8 us.
#include <math.h>

#include "ovl_lane.h"
#include "ovl_ssm_host.h"

namespace ovl_ssm {

namespace { thread_local std::string g_last_error; }

int fail(int code, const std::string& detail) {
    g_last_error = detail;
    return code;
}

int after_launch(const char* who) {
    const hipError_t err = hipPeekAtLastError();
    if (err != hipSuccess) {
        (void)hipGetLastError();
        return fail(OVL_SSM_EHIP, std::string(who) + ": " + hipGetErrorString(err));
    }
    return OVL_SSM_OK;
}

}  // namespace ovl_ssm

using ovl_lane::bf16;
using ovl_lane::f16;
using ovl_lane::narrow;
using ovl_lane::widen;

namespace {

constexpr uint32_t THREADS = 256;
constexpr float LOG2E = 0x1.715476p+0f;

template <typename T> struct sequence { const T* data; int64_t batch_stride, token_stride; };

template <typename T> struct conv_args {
    uint32_t batch, length, channels;
    int32_t  silu;
    sequence<T> x, kept;
    const void *weight, *bias;
    bool own_weights;                       // weight and bias are T, else float32
    const int32_t* lengths;
};

// VEC elements moved as one access; their address is a multiple of their size.
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) pack { T v[VEC]; };

template <typename T, int VEC>
__device__ __forceinline__ pack<T, VEC> load_pack(const T* at) { return *reinterpret_cast<const pack<T, VEC>*>(at); }

template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* to, const float (&x)[VEC]) {
    pack<T, VEC> out;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out.v[i] = narrow<T>(x[i]);
    *reinterpret_cast<pack<T, VEC>*>(to) = out;
}

__device__ __forceinline__ float sigmoid_(float x) { return ovl_lane::rcp_(1.0f + ovl_lane::exp2_(-x * LOG2E)); }

template <typename T>
__device__ __forceinline__ uint32_t end_of(const conv_args<T>& p, uint32_t b) {
    if (p.lengths == nullptr) return p.length;
    const int32_t n = p.lengths[b];
    return n < 0 ? 0u : min((uint32_t)n, p.length);
}

// Row `at` of the line before the sequence: at = -(width - 1) .. -1 are the kept tokens.
template <typename T, int W, int VEC>
__device__ __forceinline__ void load_line(float (&to)[VEC], const conv_args<T>& p, uint32_t b, uint32_t c, int64_t at) {
    if (at >= 0 || p.kept.data != nullptr) {
        const T* from = at >= 0 ? p.x.data + (int64_t)b * p.x.batch_stride + at * p.x.token_stride + c
                                : p.kept.data + (int64_t)b * p.kept.batch_stride + (at + W - 1) * p.kept.token_stride + c;
        const pack<T, VEC> raw = load_pack<T, VEC>(from);
#pragma unroll
        for (int i = 0; i < VEC; ++i) to[i] = widen<T>(raw.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) to[i] = 0.0f;
    }
}

// COUNT neighbours at an address that is a multiple of their size only.
template <typename E, int COUNT> struct __attribute__((packed, aligned(sizeof(E)))) neighbours { E v[COUNT]; };

template <int W, int VEC, typename E>
__device__ __forceinline__ void load_taps_as(float (&w)[W][VEC], float (&bias)[VEC], const E* weight, const E* b, uint32_t c) {
    const neighbours<E, VEC * W> taps = *reinterpret_cast<const neighbours<E, VEC * W>*>(weight + (uint64_t)c * W);
    neighbours<E, VEC> more = {};
    if (b != nullptr) more = *reinterpret_cast<const neighbours<E, VEC>*>(b + c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][i] = widen<E>(taps.v[i * W + k]);
        bias[i] = b != nullptr ? widen<E>(more.v[i]) : 0.0f;
    }
}

template <typename T, int W, int VEC>
__device__ __forceinline__ void load_taps(float (&w)[W][VEC], float (&bias)[VEC], const conv_args<T>& p, uint32_t c) {
    if (p.own_weights)
        load_taps_as(w, bias, static_cast<const T*>(p.weight), static_cast<const T*>(p.bias), c);
    else
        load_taps_as(w, bias, static_cast<const float*>(p.weight), static_cast<const float*>(p.bias), c);
}

// A lane walks along `slice_tokens` tokens of VEC channels, STEP of them loaded ahead; lanes run along the channels first.
// (All of a slice of 16 tokens loaded at once, without a walk: 120 us where this takes 97; slices of 8 tokens 166.)
template <typename T, int W, int VEC>
__global__ void __launch_bounds__(THREADS)
conv_forward_kernel(conv_args<T> p, uint32_t vectors, uint32_t slices, uint32_t slice_tokens, T* y, T* last) {
    constexpr uint32_t STEP = 8;
    const uint64_t id = (uint64_t)blockIdx.x * THREADS + threadIdx.x;
    if (id >= (uint64_t)p.batch * slices * vectors) return;
    const uint32_t c = (uint32_t)(id % vectors) * VEC;
    const uint64_t rest = id / vectors;
    const uint32_t slice = (uint32_t)(rest % slices), b = (uint32_t)(rest / slices);
    const uint32_t t0 = slice * slice_tokens, end = end_of(p, b), t1 = min(t0 + slice_tokens, p.length), stop = min(t1, end);
    T* to = y + ((uint64_t)b * p.length + t0) * p.channels + c;
    uint32_t t = t0;
    if (t0 < end) {
        float w[W][VEC], bias[VEC], line[W][VEC];           // line: the W inputs of the present token, oldest first
        load_taps<T>(w, bias, p, c);
        const T* base = p.x.data + (int64_t)b * p.x.batch_stride + c;
        pack<T, VEC> next[STEP];
        // tokens behind the slice are read as its last one and not used
        auto fetch = [&](uint32_t from) {
#pragma unroll
            for (uint32_t i = 0; i < STEP; ++i)
                next[i] = load_pack<T, VEC>(base + (int64_t)min(from + i, stop - 1u) * p.x.token_stride);
        };
        fetch(t0);
#pragma unroll
        for (int k = 1; k < W; ++k) load_line<T, W, VEC>(line[k], p, b, c, (int64_t)t0 - W + k);
        for (; t < stop; t += STEP) {
            pack<T, VEC> now[STEP];
#pragma unroll
            for (uint32_t i = 0; i < STEP; ++i) now[i] = next[i];
            if (t + STEP < stop) fetch(t + STEP);
#pragma unroll
            for (uint32_t i = 0; i < STEP; ++i) {
                float out[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
#pragma unroll
                    for (int k = 0; k + 1 < W; ++k) line[k][v] = line[k + 1][v];
                    line[W - 1][v] = widen<T>(now[i].v[v]);
                    float pre = bias[v];
#pragma unroll
                    for (int k = 0; k < W; ++k) pre = fmaf(w[k][v], line[k][v], pre);
                    if (p.silu) pre *= sigmoid_(pre);
                    out[v] = pre;
                }
                if (t + i < stop) store_pack<T, VEC>(to + (uint64_t)i * p.channels, out);
            }
            to += (uint64_t)STEP * p.channels;
        }
    }
    if (stop < t1) {                        // behind the sequence the outputs are zero
        float zero[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) zero[v] = 0.0f;
        for (t = max(t0, end); t < t1; ++t) store_pack<T, VEC>(y + ((uint64_t)b * p.length + t) * p.channels + c, zero);
    }
    if (slice == 0u) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) {
            float row[VEC];
            load_line<T, W, VEC>(row, p, b, c, (int64_t)end - (W - 1) + k);
            store_pack<T, VEC>(last + ((uint64_t)b * (W - 1) + k) * p.channels + c, row);
        }
    }
}

template <typename T> struct conv_gradient_args {
    sequence<T> d_y, d_last;
    T *d_x, *d_kept;
    float* part;                            // [slices of the grid][channels][W + 1]
};

// A workgroup holds `lanes` vectors of channels side by side (a power of two) and THREADS / lanes slices of the tokens; a
// slice is a run of tokens of one sequence.  Each lane walks its slice and W - 1 tokens further (whose gradients reach
// back into it), four tokens of loads ahead; the sums for the taps and the bias stay in registers, are added up over
// the workgroup's slices through LDS and leave as one part per workgroup.
template <typename T, int W, int VEC>
__global__ void __launch_bounds__(THREADS)
conv_backward_kernel(conv_args<T> p, conv_gradient_args<T> g, uint32_t vectors, uint32_t lanes, uint32_t columns,
                     uint32_t slices, uint32_t slice_tokens) {
    constexpr int STEP = 4, SUMS = W + 1;
    __shared__ float lds[THREADS * VEC];
    const uint32_t column = blockIdx.x % columns, row = blockIdx.x / columns, per_group = THREADS / lanes;
    const uint32_t vector = column * lanes + threadIdx.x % lanes;
    const uint64_t slice = (uint64_t)row * per_group + threadIdx.x / lanes;
    const bool active = vector < vectors && slice < (uint64_t)p.batch * slices;
    float dw[W][VEC], db[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        db[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][v] = 0.0f;
    }
    const uint32_t c = vector * VEC;
    if (active) {
        const uint32_t b = (uint32_t)(slice / slices), t0 = (uint32_t)(slice % slices) * slice_tokens;
        const uint32_t end = end_of(p, b), t1 = min(t0 + slice_tokens, p.length);
        float w[W][VEC], bias[VEC], line[W][VEC], d[W][VEC];
        load_taps<T>(w, bias, p, c);
        const T* x_base = p.x.data + (int64_t)b * p.x.batch_stride + c;
        const T* dy_base = g.d_y.data + (int64_t)b * g.d_y.batch_stride + c;
#pragma unroll
        for (int k = 0; k < W; ++k) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) { line[k][v] = 0.0f; d[k][v] = 0.0f; }
            if (k >= 1 && t0 < end) load_line<T, W, VEC>(line[k], p, b, c, (int64_t)t0 - W + k);
        }
        // position t of the walk makes d[t] and with it dx[t - (W - 1)]
        const uint32_t stop = t1 + W - 1;
        const uint32_t safe = end > 0u ? end - 1u : 0u;
        pack<T, VEC> x_next[STEP], dy_next[STEP];
        auto fetch = [&](uint32_t t) {
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                x_next[i] = load_pack<T, VEC>(x_base + (int64_t)min(t + i, safe) * p.x.token_stride);
                dy_next[i] = load_pack<T, VEC>(dy_base + (int64_t)min(t + i, safe) * g.d_y.token_stride);
            }
        };
        fetch(t0);
        for (uint32_t base = t0; base < stop; base += STEP) {
            pack<T, VEC> x_now[STEP], dy_now[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) { x_now[i] = x_next[i]; dy_now[i] = dy_next[i]; }
            if (base + STEP < stop) fetch(base + STEP);
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                const uint32_t t = base + i;
                const bool token = t < end;
                float dx[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
#pragma unroll
                    for (int k = 0; k + 1 < W; ++k) { line[k][v] = line[k + 1][v]; d[k][v] = d[k + 1][v]; }
                    line[W - 1][v] = token ? widen<T>(x_now[i].v[v]) : 0.0f;
                    float up = token ? widen<T>(dy_now[i].v[v]) : 0.0f;
                    if (p.silu) {
                        float pre = bias[v];
#pragma unroll
                        for (int k = 0; k < W; ++k) pre = fmaf(w[k][v], line[k][v], pre);
                        const float s = sigmoid_(pre);
                        // (a token behind the sequence has up = 0; its pre may be anything finite or not)
                        up = token ? up * s * fmaf(pre, 1.0f - s, 1.0f) : 0.0f;
                    }
                    d[W - 1][v] = up;
                    dx[v] = 0.0f;
#pragma unroll
                    for (int k = 0; k < W; ++k) dx[v] = fmaf(w[k][v], d[W - 1 - k][v], dx[v]);
                    if (token) {
                        const float mine = t < t1 ? up : 0.0f;          // the sums of a token belong to its own slice
                        db[v] += mine;
#pragma unroll
                        for (int k = 0; k < W; ++k) dw[k][v] = fmaf(mine, line[k][v], dw[k][v]);
                    }
                }
                const int64_t at = (int64_t)t - (W - 1);        // dx[at]
                if (at >= (int64_t)end)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) dx[v] = 0.0f;
                if (t < stop && at >= (t0 == 0u ? -(int64_t)(W - 1) : (int64_t)t0)) {
                    const int64_t from_last = at - ((int64_t)end - (W - 1));
                    if (W > 1 && g.d_last.data != nullptr && from_last >= 0 && from_last < W - 1) {
                        const pack<T, VEC> more = load_pack<T, VEC>(g.d_last.data + (int64_t)b * g.d_last.batch_stride +
                                                                    from_last * g.d_last.token_stride + c);
#pragma unroll
                        for (int v = 0; v < VEC; ++v) dx[v] += widen<T>(more.v[v]);
                    }
                    if (at >= 0) store_pack<T, VEC>(g.d_x + ((uint64_t)b * p.length + at) * p.channels + c, dx);
                    else if (g.d_kept != nullptr)
                        store_pack<T, VEC>(g.d_kept + ((uint64_t)b * (W - 1) + at + W - 1) * p.channels + c, dx);
                }
            }
        }
    }
    // the workgroup's sums, one tap at a time
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; ++v) lds[threadIdx.x * VEC + v] = k < W ? dw[k < W ? k : 0][v] : db[v];
        __syncthreads();
        for (uint32_t at = threadIdx.x; at < lanes * VEC; at += THREADS) {
            float sum = 0.0f;
            for (uint32_t s = 0; s < per_group; ++s) sum += lds[s * lanes * VEC + at];
            const uint32_t channel = column * lanes * VEC + at;
            if (channel < p.channels) g.part[((uint64_t)k * (gridDim.x / columns) + row) * p.channels + channel] = sum;
        }
    }
}

// Adds the parts up (k = W: the bias), in a fixed order: a workgroup for a tap of 64 channels, whose sixteen wavefronts
// share the rows of parts, of which many short sequences make many.
constexpr uint32_t SHARES = 16;
template <int W>
__global__ void __launch_bounds__(64 * SHARES)
conv_sum_kernel(const float* part, uint32_t channels, uint32_t columns, uint32_t rows, float* d_weight, float* d_bias) {
    __shared__ float lds[SHARES][64];
    const uint32_t lane = threadIdx.x & 63u, share = ovl_lane::wavefront(threadIdx.x / 64u), k = blockIdx.x / columns;
    const uint32_t channel = blockIdx.x % columns * 64u + lane;
    float sum = 0.0f;
    if (channel < channels)
#pragma unroll 8
        for (uint32_t r = share; r < rows; r += SHARES) sum += part[((uint64_t)k * rows + r) * channels + channel];
    lds[share][lane] = sum;
    __syncthreads();
    if (share != 0u || channel >= channels) return;
#pragma unroll
    for (uint32_t i = 1; i < SHARES; ++i) sum += lds[i][lane];
    if (k < W) d_weight[(uint64_t)channel * W + k] = sum;
    else if (d_bias != nullptr) d_bias[channel] = sum;
}

// One token of every sequence: a lane takes VEC channels.
template <typename T, int W, int VEC>
__global__ void __launch_bounds__(THREADS)
conv_step_kernel(conv_args<T> p, uint32_t vectors, T* kept, T* y) {
    const uint64_t id = (uint64_t)blockIdx.x * THREADS + threadIdx.x;
    if (id >= (uint64_t)p.batch * vectors) return;
    const uint32_t c = (uint32_t)(id % vectors) * VEC, b = (uint32_t)(id / vectors);
    float w[W][VEC], bias[VEC];
    load_taps<T>(w, bias, p, c);
    T* own = kept + (int64_t)b * p.kept.batch_stride + c;
    pack<T, VEC> line[W];
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) line[k] = load_pack<T, VEC>(own + k * p.kept.token_stride);
    line[W - 1] = load_pack<T, VEC>(p.x.data + (int64_t)b * p.x.batch_stride + c);
    float out[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float pre = bias[v];
#pragma unroll
        for (int k = 0; k < W; ++k) pre = fmaf(w[k][v], widen<T>(line[k].v[v]), pre);
        if (p.silu) pre *= sigmoid_(pre);
        out[v] = pre;
    }
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) *reinterpret_cast<pack<T, VEC>*>(own + k * p.kept.token_stride) = line[k + 1];
    store_pack<T, VEC>(y + (uint64_t)b * p.channels + c, out);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------

using ovl_ssm::after_launch;
using ovl_ssm::fail;
using ovl_ssm::launchable;

uint32_t size_of(int32_t dtype) { return dtype == OVL_SSM_FLOAT32 ? 4u : 2u; }

int check(const char* who, const ovl_ssm_conv* s, bool token) {
    const std::string name(who);
    if (s == nullptr) return fail(OVL_SSM_EINVAL, name + ": null convolution");
    if (s->batch == 0 || s->length == 0 || s->channels == 0) return fail(OVL_SSM_EINVAL, name + ": sizes must be positive");
    if (s->width < 1u || s->width > 4u) return fail(OVL_SSM_EINVAL, name + ": width must be 1 to 4");
    if (s->dtype != OVL_SSM_FLOAT16 && s->dtype != OVL_SSM_FLOAT32 && s->dtype != OVL_SSM_BFLOAT16)
        return fail(OVL_SSM_EINVAL, name + ": unknown element type");
    if (s->x.data == nullptr || s->weight == nullptr) return fail(OVL_SSM_EINVAL, name + ": null tensor");
    if (token && (s->length != 1u || s->lengths != nullptr))
        return fail(OVL_SSM_EINVAL, name + ": a step takes one token of every sequence");
    if (s->length > (1u << 30)) return fail(OVL_SSM_EINVAL, name + ": length must be at most 2^30");
    if (s->channels > (1u << 31)) return fail(OVL_SSM_EINVAL, name + ": at most 2^31 channels");
    if ((uint64_t)s->batch * s->length > ((1ull << 31) - 1) * THREADS / s->channels)
        return fail(OVL_SSM_EINVAL, name + ": too many elements for one launch");
    return OVL_SSM_OK;
}

// Whether a lane for `vec` channels of every sequence can be launched (the forward pass has more only where that is few).
int check_lanes(const char* who, const ovl_ssm_conv* s, uint32_t vec) {
    if (launchable(((uint64_t)s->batch * (s->channels / vec) + THREADS - 1) / THREADS, THREADS)) return OVL_SSM_OK;
    return fail(OVL_SSM_EINVAL, std::string(who) + ": too many elements for one launch");
}

// The widest access (in elements, at most 16 bytes) that the channel count, the strides and the addresses allow.
struct width_finder {
    uint64_t bits;                          // every byte offset that must be a multiple of the access
    explicit width_finder(uint64_t row_bytes) : bits(row_bytes) {}
    void take(const void* p) { bits |= reinterpret_cast<uintptr_t>(p); }
    void take(const ovl_ssm_sequence& s, uint32_t size) {
        if (s.data == nullptr) return;
        take(s.data);
        bits |= (uint64_t)s.batch_stride * size | (uint64_t)s.token_stride * size;
    }
    uint32_t elements(uint32_t size) const {
        uint32_t bytes = 16;
        while (bytes > size && (bits & (bytes - 1u)) != 0) bytes /= 2;
        return bytes / size;
    }
};

template <typename T>
conv_args<T> make_args(const ovl_ssm_conv* s) {
    auto seq = [](const ovl_ssm_sequence& v) {
        return sequence<T>{static_cast<const T*>(v.data), v.batch_stride, v.token_stride};
    };
    return conv_args<T>{s->batch, s->length, s->channels, s->silu, seq(s->x), seq(s->kept), s->weight, s->bias,
                        s->own_weights != 0, s->lengths};
}

template <typename T, int W, int VEC>
void forward(const ovl_ssm_conv* s, T* y, T* last, hipStream_t stream) {
    const uint32_t vectors = s->channels / VEC;
    // so many tokens per lane that there are three wavefronts per SIMD, but at least 4 tokens (two: 137 us where these take
    // 97 to 105; six: 109)
    constexpr uint64_t WANTED = 64 * 3 * 1024;              // lanes
    const uint64_t strands = (uint64_t)s->batch * vectors, most = (s->length + 3u) / 4u;
    uint64_t slices = WANTED / strands;
    slices = slices < 1 ? 1 : slices > most ? most : slices;
    const uint32_t slice_tokens = (uint32_t)((s->length + slices - 1) / slices);
    slices = (s->length + slice_tokens - 1u) / slice_tokens;
    const uint64_t all = strands * slices;
    hipLaunchKernelGGL((conv_forward_kernel<T, W, VEC>), dim3((uint32_t)((all + THREADS - 1) / THREADS)), dim3(THREADS), 0, stream,
                       make_args<T>(s), vectors, (uint32_t)slices, slice_tokens, y, last);
}

// How the backward pass cuts the work: a grid of `columns` by `rows` workgroups.
struct cut { uint32_t vectors, lanes, columns, slices, slice_tokens, rows; };
cut cut_for(const ovl_ssm_conv* s, uint32_t vec) {
    // workgroups: as many as are resident with the 230 registers of the widest variant, two per compute unit (768 take
    // 226 us where these take 180, 2048 take 236, since one behind the others is waited for, and write more parts)
    constexpr uint64_t WANTED = 512;
    cut k;
    k.vectors = s->channels / vec;
    k.lanes = 64;
    while (k.lanes > 8u && k.lanes / 2u >= k.vectors) k.lanes /= 2u;
    k.columns = (k.vectors + k.lanes - 1u) / k.lanes;
    const uint64_t per_group = THREADS / k.lanes;
    uint64_t slices = (WANTED * per_group + (uint64_t)k.columns * s->batch - 1) / ((uint64_t)k.columns * s->batch);
    const uint64_t most = (s->length + 15u) / 16u;          // at least 16 tokens each
    slices = slices < 1 ? 1 : slices > most ? most : slices;
    k.slice_tokens = (uint32_t)((s->length + slices - 1) / slices);
    k.slices = (s->length + k.slice_tokens - 1u) / k.slice_tokens;
    k.rows = (uint32_t)(((uint64_t)s->batch * k.slices + per_group - 1) / per_group);
    return k;
}

// Workgroups of conv_sum_kernel for a tap.
uint32_t sum_columns(const ovl_ssm_conv* s) { return s->channels / 64u + (s->channels % 64u != 0u); }

template <typename T, int W, int VEC>
void backward(const ovl_ssm_conv* s, const ovl_ssm_sequence* d_y, const ovl_ssm_sequence* d_last, T* d_x, T* d_kept,
              float* d_weight, float* d_bias, float* part, hipStream_t stream) {
    const cut k = cut_for(s, VEC);
    conv_gradient_args<T> g;
    g.d_y = sequence<T>{static_cast<const T*>(d_y->data), d_y->batch_stride, d_y->token_stride};
    g.d_last = sequence<T>{nullptr, 0, 0};
    if (d_last != nullptr) g.d_last = sequence<T>{static_cast<const T*>(d_last->data), d_last->batch_stride, d_last->token_stride};
    g.d_x = d_x;
    g.d_kept = d_kept;
    g.part = part;
    hipLaunchKernelGGL((conv_backward_kernel<T, W, VEC>), dim3(k.columns * k.rows), dim3(THREADS), 0, stream, make_args<T>(s), g,
                       k.vectors, k.lanes, k.columns, k.slices, k.slice_tokens);
    const uint32_t columns = sum_columns(s);
    hipLaunchKernelGGL((conv_sum_kernel<W>), dim3(columns * (W + 1)), dim3(64 * SHARES), 0, stream, part, s->channels, columns,
                       k.rows, d_weight, d_bias);
}

template <typename T, int W, int VEC>
void step(const ovl_ssm_conv* s, T* y, hipStream_t stream) {
    const uint32_t vectors = s->channels / VEC;
    const uint64_t all = (uint64_t)s->batch * vectors;
    const conv_args<T> args = make_args<T>(s);
    hipLaunchKernelGGL((conv_step_kernel<T, W, VEC>), dim3((uint32_t)((all + THREADS - 1) / THREADS)), dim3(THREADS), 0, stream,
                       args, vectors, const_cast<T*>(args.kept.data), y);
}

// Calls F<T, W, VEC>(...) for the element type, the number of taps and the width of an access.
#define OVL_SSM_BY_VEC(F, T, W, ...)                                        \
    switch (vec) {                                                          \
        case 8u: if constexpr (sizeof(T) == 2) F<T, W, 8>(__VA_ARGS__); break; \
        case 4u: F<T, W, 4>(__VA_ARGS__); break;                            \
        case 2u: F<T, W, 2>(__VA_ARGS__); break;                            \
        default: F<T, W, 1>(__VA_ARGS__); break;                            \
    }
#define OVL_SSM_BY_WIDTH(F, T, ...)                                         \
    switch (s->width) {                                                     \
        case 1u: OVL_SSM_BY_VEC(F, T, 1, __VA_ARGS__) break;                \
        case 2u: OVL_SSM_BY_VEC(F, T, 2, __VA_ARGS__) break;                \
        case 3u: OVL_SSM_BY_VEC(F, T, 3, __VA_ARGS__) break;                \
        default: OVL_SSM_BY_VEC(F, T, 4, __VA_ARGS__) break;                \
    }

}  // namespace

extern "C" {

const char* ovl_ssm_last_error(void) { return ovl_ssm::g_last_error.c_str(); }

int ovl_ssm_conv_forward(const ovl_ssm_conv* s, void* y, void* last, void* hip_stream) {
    const int rc = check("ovl_ssm_conv_forward", s, false);
    if (rc != OVL_SSM_OK) return rc;
    if (y == nullptr || (last == nullptr && s->width > 1u)) return fail(OVL_SSM_EINVAL, "ovl_ssm_conv_forward: null tensor");
    const uint32_t size = size_of(s->dtype);
    width_finder f((uint64_t)s->channels * size);
    f.take(s->x, size);
    f.take(s->kept, size);
    f.take(y);
    f.take(last);
    const uint32_t vec = f.elements(size);
    if (const int few = check_lanes("ovl_ssm_conv_forward", s, vec)) return few;
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    switch (s->dtype) {
        case OVL_SSM_FLOAT32: OVL_SSM_BY_WIDTH(forward, float, s, static_cast<float*>(y), static_cast<float*>(last), stream) break;
        case OVL_SSM_FLOAT16: OVL_SSM_BY_WIDTH(forward, f16, s, static_cast<f16*>(y), static_cast<f16*>(last), stream) break;
        default: OVL_SSM_BY_WIDTH(forward, bf16, s, static_cast<bf16*>(y), static_cast<bf16*>(last), stream) break;
    }
    return after_launch("ovl_ssm_conv_forward");
}

uint64_t ovl_ssm_conv_workspace_bytes(const ovl_ssm_conv* s) {
    if (check("ovl_ssm_conv_workspace_bytes", s, false) != OVL_SSM_OK) return 0;
    if (!launchable(sum_columns(s) * (s->width + 1ull), 64 * SHARES)) return 0;
    uint64_t most = 0;                      // whatever access the backward pass will find
    for (uint32_t vec = 16u / size_of(s->dtype); vec >= 1u; vec /= 2u) {
        if (s->channels % vec != 0u) continue;
        const uint64_t need = (uint64_t)cut_for(s, vec).rows * s->channels * (s->width + 1u) * sizeof(float);
        most = need > most ? need : most;
    }
    return most;
}

int ovl_ssm_conv_backward(const ovl_ssm_conv* s, const ovl_ssm_sequence* d_y, const ovl_ssm_sequence* d_last, void* d_x,
                          void* d_kept, float* d_weight, float* d_bias, void* workspace, uint64_t workspace_bytes,
                          void* hip_stream) {
    const int rc = check("ovl_ssm_conv_backward", s, false);
    if (rc != OVL_SSM_OK) return rc;
    if (d_y == nullptr || d_y->data == nullptr || d_x == nullptr || d_weight == nullptr)
        return fail(OVL_SSM_EINVAL, "ovl_ssm_conv_backward: null tensor");
    const uint32_t size = size_of(s->dtype);
    width_finder f((uint64_t)s->channels * size);
    f.take(s->x, size);
    f.take(s->kept, size);
    f.take(*d_y, size);
    if (d_last != nullptr) f.take(*d_last, size);
    f.take(d_x);
    f.take(d_kept);
    const uint32_t vec = f.elements(size);
    const cut k = cut_for(s, vec);
    if (!launchable(sum_columns(s) * (s->width + 1ull), 64 * SHARES) || !launchable((uint64_t)k.columns * k.rows, THREADS))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_conv_backward: too many elements for one launch");
    if (workspace == nullptr || workspace_bytes < ovl_ssm_conv_workspace_bytes(s) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_conv_backward: workspace too small or not 4-byte aligned");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    float* part = static_cast<float*>(workspace);
    switch (s->dtype) {
        case OVL_SSM_FLOAT32: OVL_SSM_BY_WIDTH(backward, float, s, d_y, d_last, static_cast<float*>(d_x), static_cast<float*>(d_kept), d_weight, d_bias, part, stream) break;
        case OVL_SSM_FLOAT16: OVL_SSM_BY_WIDTH(backward, f16, s, d_y, d_last, static_cast<f16*>(d_x), static_cast<f16*>(d_kept), d_weight, d_bias, part, stream) break;
        default: OVL_SSM_BY_WIDTH(backward, bf16, s, d_y, d_last, static_cast<bf16*>(d_x), static_cast<bf16*>(d_kept), d_weight, d_bias, part, stream) break;
    }
    return after_launch("ovl_ssm_conv_backward");
}

int ovl_ssm_conv_step(const ovl_ssm_conv* s, void* y, void* hip_stream) {
    const int rc = check("ovl_ssm_conv_step", s, true);
    if (rc != OVL_SSM_OK) return rc;
    if (y == nullptr || (s->kept.data == nullptr && s->width > 1u)) return fail(OVL_SSM_EINVAL, "ovl_ssm_conv_step: null tensor");
    const uint32_t size = size_of(s->dtype);
    width_finder f((uint64_t)s->channels * size);
    f.take(s->x, size);
    f.take(s->kept, size);
    f.take(y);
    const uint32_t vec = f.elements(size);
    if (const int few = check_lanes("ovl_ssm_conv_step", s, vec)) return few;
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    switch (s->dtype) {
        case OVL_SSM_FLOAT32: OVL_SSM_BY_WIDTH(step, float, s, static_cast<float*>(y), stream) break;
        case OVL_SSM_FLOAT16: OVL_SSM_BY_WIDTH(step, f16, s, static_cast<f16*>(y), stream) break;
        default: OVL_SSM_BY_WIDTH(step, bf16, s, static_cast<bf16*>(y), stream) break;
    }
    return after_launch("ovl_ssm_conv_step");
}

}  // extern "C"
