// Selective state space scan for gfx950 behind the C ABI of include/ovl_ssm.h: forward, backward, one-token step.
//
// Mathematics.  Every (sequence, channel, state entry) is a linear recurrence of its own, h[t] = a[t] h[t-1] + b[t] with
// a[t] = exp(dt[t] A) and b[t] = dt[t] u[t] B[t]; the output sums over the state entries, y[t] = sum C[t] h[t].  The
// gradient is the same recurrence from the other end: g[t] = C[t] dy[t] + r[t+1], r[t] = a[t] g[t].
//
// Bound.  Per state entry and token: one multiplication and one exponential (two issue slots) for the decay, one
// multiplication and two fused multiply-adds: 24 clocks of a SIMD per 64 entries, measured; at 16 state entries that is
// more than what the loads and stores take, so the vector ALU bounds the scan, and a SIMD needs two wavefronts or more (one
// alone issues an instruction in 6.3 clocks, several together one in 4.3).
//
// Splitting the length.  A sequence is sequential; few channels leave SIMDs idle.  Then the tokens are split into chunks:
// one pass computes every chunk's effect on a zero state (the decay of a chunk needs only the sum of its dt), a small
// kernel joins the chunks' states, and the full pass starts every chunk from its true state.  The price is a second
// evaluation of every decay, so the split is made only where it pays (chunks_for below).
//
// Work layouts.  Where a lane needs nothing but its channel (the forward pass, and the pass over the gradient's chunks) it
// holds all entries of the channel's state, up to 64, in registers: a wavefront owns 64 neighbouring channels of one group
// and a chunk, nothing is summed across lanes, and there is no barrier.  B and C, the same for the whole wavefront, come
// from the lanes of a row as operands of the consuming instructions and through a part of LDS of its own.  Addresses are
// scalar with 32 bits per lane.  (With a quad per channel the forward pass of 4 sequences of 2048 tokens, 4096 channels of
// 16 entries in bf16 took 373 us without a split, now it takes 248 with both passes and the join.)
// The backward pass holds states and decays of several tokens, and sums over channels: a quad owns a channel and its
// lanes a quarter of the state each; what depends on (token, channel) only is done once for four tokens in the four lanes
// and handed round with lane moves; sums over the state end in an exchange that leaves every lane with its own token.
#include <math.h>

#include "ovl_lane.h"
#include "ovl_ssm_host.h"

using ovl_lane::bf16;
using ovl_lane::f16;
using ovl_lane::narrow;
using ovl_lane::widen;

namespace {

constexpr uint32_t TILE = 16;               // tokens per tile; states are kept for the backward pass once per tile
constexpr uint32_t QUADS = TILE / 4;        // groups of four tokens
constexpr uint32_t WAVES = 4;
constexpr uint32_t THREADS = 64 * WAVES;
constexpr uint32_t BLOCK = 64;              // channels of a workgroup
constexpr uint32_t STEP = 8;                // tokens that a lane with a channel of its own takes at a time

constexpr float LOG2E = 0x1.715476p+0f, LN2 = 0x1.62e43p-1f;

template <typename T> struct sequence { const T* data; int64_t batch_stride, token_stride; };
template <typename T> struct vectors { const T* data; int64_t batch_stride, token_stride, group_stride; };

template <typename T> struct scan_args {
    uint32_t batch, length, channels, state, groups;
    uint32_t per_group, blocks;             // channels per group, workgroups per group
    uint32_t tiles, chunks, chunk_tiles;    // tiles of the length, chunks, tiles per chunk
    int32_t  softplus;
    sequence<T> u, delta, z;
    vectors<T> B, C;
    const float *A, *D, *delta_bias, *entering;
    const int32_t* lengths;
};

// Where a workgroup works: sequence, group, block of channels, chunk.
struct place {
    uint32_t b, g, block, chunk;
    uint32_t q, channel;                    // lane of its channel's team; channel (clamped to a valid one)
    bool active;                            // whether the channel is one of the group's
    uint32_t first, last;                   // tiles
    uint32_t end;                           // first token behind the sequence
};

// TEAM: lanes per channel.  `unit` counts blocks of channels first, so that neighbouring units read the same B and C.
template <uint32_t TEAM, typename T>
__device__ __forceinline__ place find_place(const scan_args<T>& p, uint32_t unit, uint32_t lane, uint32_t chunk_base, uint32_t chunks) {
    place w;
    uint32_t id = unit;
    w.block = id % p.blocks;
    id /= p.blocks;
    w.g = id % p.groups;
    id /= p.groups;
    w.chunk = chunk_base + id % chunks;
    w.b = id / chunks;
    w.q = lane % TEAM;
    uint32_t c = w.block * BLOCK + lane / TEAM;
    w.active = c < p.per_group;
    c = w.active ? c : p.per_group - 1u;
    w.channel = w.g * p.per_group + c;
    w.first = w.chunk * p.chunk_tiles;
    w.last = min(w.first + p.chunk_tiles, p.tiles);
    w.end = p.length;
    if (p.lengths != nullptr) {
        const int32_t n = p.lengths[w.b];
        w.end = n < 0 ? 0u : min((uint32_t)n, p.length);
    }
    return w;
}

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x|; what 1 + e rounds away is put back, so that the result keeps its
// relative precision where it is small (time steps of 0.001 are ordinary).  The product |x| log2(e) is carried to twice
// the precision for the same reason.
__device__ __forceinline__ float softplus_(float x) {
    const float ax = fabsf(x);
    const float p = -ax * LOG2E;
    const float low = fmaf(-ax, LOG2E, -p);
    float e = ovl_lane::exp2_(p);
    e = ax < 100.0f ? fmaf(e * LN2, low, e) : e;
    const float w = 1.0f + e;
    const float lost = e - (w - 1.0f);      // to be divided by w; it matters only where w is nearly one
    const float log1p = fmaf(ovl_lane::log2_(w), LN2, lost);
    return ovl_lane::positive(x) + log1p;
}

__device__ __forceinline__ float sigmoid_(float x) { return ovl_lane::rcp_(1.0f + ovl_lane::exp2_(-x * LOG2E)); }

// A in powers of two.  One without bound counts as the largest number: tokens behind the sequence have dt = 0 and change
// nothing, while 0 times infinity would be NaN.
__device__ __forceinline__ float rate_(float a) {
    constexpr float MOST = 0x1.fffffep+127f;
    const float r = a * LOG2E;
    return r < -MOST ? -MOST : r > MOST ? MOST : r;
}

// A sequence tensor as a lane reads it: N tokens of its channel, PACE tokens apart, of a tile of N * PACE tokens.  The
// tile's address and the tokens' offsets are the same for the whole wavefront and stay in scalar registers; a lane adds 32
// bits of its own (the host has checked that they suffice).  The offsets are made anew for every tile: kept, those of all
// tensors would not fit the scalar registers, and their places in vector registers cost wavefronts.
template <typename T, uint32_t N, uint32_t PACE> struct reader {
    const T* tile;
    uint32_t token_bytes, own;
    __device__ __forceinline__ reader(const sequence<T>& s, const place& w, uint32_t t0)
        : tile(s.data + (int64_t)w.b * s.batch_stride + (int64_t)t0 * s.token_stride),
          token_bytes((uint32_t)s.token_stride * (uint32_t)sizeof(T)),
          own(w.q * token_bytes + w.channel * (uint32_t)sizeof(T)) {}
    __device__ __forceinline__ void load(T (&to)[N]) const {
        const ovl_lane::region r(tile);
        const uint32_t pace = ovl_lane::anew(token_bytes) * PACE;
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) to[j] = r.template load<T>(own, j * pace);
    }
    // Only `left` tokens (at least one) are there: those behind are read as the last; the values are not used.
    __device__ __forceinline__ void load_some(T (&to)[N], uint32_t left, uint32_t first) const {
        const ovl_lane::region r(tile);
        const uint32_t bytes = ovl_lane::anew(token_bytes);
#pragma unroll
        for (uint32_t j = 0; j < N; ++j)
            to[j] = r.template load<T>(own + (min(PACE * j + first, left - 1u) - first) * bytes, 0u);
    }
    // DIRECTION 1 or -1
    template <int DIRECTION> __device__ __forceinline__ void move() {
        const char* at = reinterpret_cast<const char*>(tile);
        const uint64_t bytes = N * PACE * (uint64_t)token_bytes;
        tile = reinterpret_cast<const T*>(DIRECTION > 0 ? at + bytes : at - bytes);
    }
};

// Where a lane writes dense output sequences; several outputs of one shape share it.
template <typename T, uint32_t N, uint32_t PACE> struct writer {
    uint64_t tile;                          // in bytes
    uint32_t token_bytes, own;
    __device__ __forceinline__ writer(const place& w, uint32_t length, uint32_t channels, uint32_t t0)
        : tile(((uint64_t)w.b * length + t0) * channels * sizeof(T)), token_bytes(channels * (uint32_t)sizeof(T)),
          own(w.q * token_bytes + w.channel * (uint32_t)sizeof(T)) {}
    __device__ __forceinline__ void store(T* to, const T (&x)[N]) const {
        const ovl_lane::region r(reinterpret_cast<char*>(to) + tile);
        const uint32_t pace = ovl_lane::anew(token_bytes) * PACE;
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) r.template store<T>(x[j], own, j * pace);
    }
    // the first `left` tokens of the tile
    __device__ __forceinline__ void store_some(T* to, const T (&x)[N], uint32_t left, uint32_t first) const {
        const ovl_lane::region r(reinterpret_cast<char*>(to) + tile);
        const uint32_t pace = ovl_lane::anew(token_bytes) * PACE;
#pragma unroll
        for (uint32_t j = 0; j < N; ++j)
            if (PACE * j + first < left) r.template store<T>(x[j], own, j * pace);
    }
    template <int DIRECTION> __device__ __forceinline__ void move() { tile += DIRECTION * (int64_t)(N * PACE) * token_bytes; }
};

// The elements of a tile of B or C that this thread takes to LDS: TOKENS tokens of NP entries, from entry `first` on.
template <typename T, uint32_t NP, uint32_t TOKENS, uint32_t LANES> struct vector_stage {
    static constexpr uint32_t ALL = TOKENS * NP, PER = (ALL + LANES - 1) / LANES;
    const T* tile;
    uint32_t token_bytes, own[PER];
    uint32_t lane;
    T raw[PER];
    __device__ __forceinline__ vector_stage(const vectors<T>& v, const place& w, uint32_t lane_, uint32_t t0, uint32_t n, uint32_t first = 0u)
        : tile(v.data + (int64_t)w.b * v.batch_stride + (int64_t)w.g * v.group_stride + (int64_t)t0 * v.token_stride),
          token_bytes((uint32_t)v.token_stride * (uint32_t)sizeof(T)), lane(lane_) {
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t at = (lane + i * LANES) % ALL;
            own[i] = at / NP * token_bytes + min(first + at % NP, n - 1u) * (uint32_t)sizeof(T);
        }
    }
    __device__ __forceinline__ void load() {
        const ovl_lane::region r(tile);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) raw[i] = r.template load<T>(own[i], 0u);
    }
    __device__ __forceinline__ void load_some(uint32_t left) {
        const ovl_lane::region r(tile);
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t token = (lane + i * LANES) % ALL / NP;
            raw[i] = r.template load<T>(own[i] - (token < left ? 0u : (token - left + 1u) * token_bytes), 0u);
        }
    }
    // Entries past the state (`n` from the first on are in it) and tokens behind the sequence (`tokens` of the tile's are in
    // it) become zero: they then add nothing anywhere.
    __device__ __forceinline__ void store(float* lds, uint32_t tokens, uint32_t n) const {
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t at = lane + i * LANES;
            if (ALL % LANES == 0u || at < ALL) lds[at] = (at % NP < n && at / NP < tokens) ? widen<T>(raw[i]) : 0.0f;
        }
    }
    template <int DIRECTION> __device__ __forceinline__ void move() {
        const char* at = reinterpret_cast<const char*>(tile);
        const uint64_t bytes = TOKENS * (uint64_t)token_bytes;
        tile = reinterpret_cast<const T*>(DIRECTION > 0 ? at + bytes : at - bytes);
    }
};

// Values that are to be in registers here: the compiler would otherwise move what they are made of, and the waiting for
// its loads, behind the loads of the next tile.
template <uint32_t N> __device__ __forceinline__ void settle(float (&v)[N]) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) ovl_lane::keep(v[i]);
}

// States that kernels hand to each other: padded to NP entries, four neighbouring entries of a channel side by side, then
// the channels, so that a wavefront's accesses are dense.  S entries from entry `first` on.
template <int S>
__device__ __forceinline__ uint32_t state_offset(uint32_t first, uint32_t channel, uint32_t channels) {
    return (first / 4u * channels + channel) * 4u + first % 4u;
}
template <int S>
__device__ __forceinline__ void load_states(float (&h)[S], const float* from, uint32_t first, uint32_t channel, uint32_t channels) {
    constexpr int WIDE = S >= 4 ? 4 : S;
    typedef float vec __attribute__((ext_vector_type(WIDE)));
#pragma unroll
    for (int i = 0; i < S; i += WIDE) {
        const vec v = *reinterpret_cast<const vec*>(from + state_offset<S>(first + i, channel, channels));
#pragma unroll
        for (int k = 0; k < WIDE; ++k) h[i + k] = v[k];
    }
}
template <int S>
__device__ __forceinline__ void store_states(const float (&h)[S], float* to, uint32_t first, uint32_t channel, uint32_t channels) {
    constexpr int WIDE = S >= 4 ? 4 : S;
    typedef float vec __attribute__((ext_vector_type(WIDE)));
#pragma unroll
    for (int i = 0; i < S; i += WIDE) {
        vec v;
#pragma unroll
        for (int k = 0; k < WIDE; ++k) v[k] = h[i + k];
        *reinterpret_cast<vec*>(to + state_offset<S>(first + i, channel, channels)) = v;
    }
}

// S entries of a [.., state] tensor for the lane's part of the state, zero past the end.
template <int S>
__device__ __forceinline__ void load_entries(float (&h)[S], const float* row, uint32_t q, uint32_t n) {
    if ((q + 1u) * S <= n) {
        struct __attribute__((packed, aligned(4))) whole { float v[S]; };
        const whole w = *reinterpret_cast<const whole*>(row + q * S);
#pragma unroll
        for (int s = 0; s < S; ++s) h[s] = w.v[s];
        return;
    }
#pragma unroll
    for (uint32_t s = 0; s < S; ++s) {
        const uint32_t at = q * S + s;
        h[s] = at < n ? row[at] : 0.0f;
    }
}
template <int S>
__device__ __forceinline__ void store_entries(const float (&h)[S], float* row, uint32_t q, uint32_t n) {
#pragma unroll
    for (uint32_t s = 0; s < S; ++s) {
        const uint32_t at = q * S + s;
        if (at < n) row[at] = h[s];
    }
}

__device__ __forceinline__ float quad_sum(float x) {
    x += ovl_lane::quad_xor1(x);
    return x + ovl_lane::quad_xor2(x);
}

// Four values per lane, one for each token of the quad: lane q receives the sum over the quad of value q.
__device__ __forceinline__ float quad_scatter_sum(const float (&v)[4], uint32_t q) {
    const bool odd = q & 1u, high = q & 2u;
    const float low = (odd ? v[1] : v[0]) + ovl_lane::quad_xor1(odd ? v[0] : v[1]);
    const float up = (odd ? v[3] : v[2]) + ovl_lane::quad_xor1(odd ? v[2] : v[3]);
    return (high ? up : low) + ovl_lane::quad_xor2(high ? low : up);
}

// quad_from with a number that is constant once the loops around it are unrolled
__device__ __forceinline__ float quad_pick(float x, int k) {
    switch (k) {
        case 0: return ovl_lane::quad_from<0>(x);
        case 1: return ovl_lane::quad_from<1>(x);
        case 2: return ovl_lane::quad_from<2>(x);
        default: return ovl_lane::quad_from<3>(x);
    }
}

// The vectors B or C of the tokens of a step for kernels with a channel per lane, where every lane needs all S entries.
// Lane l of every row of sixteen holds entries l, l + 16, ..., and instructions take their operand from the lane of their
// row that has it: nothing is copied, no LDS is read (sixteen registers loaded from LDS per token and vector, as broadcasts,
// cost more than a tenth of the time).
template <typename T, int S> struct vectors_of_step {
    static constexpr uint32_t HELD = S <= 16 ? 1 : S / 16, IN_ROW = S < 16 ? S : 16;
    const T* step;
    uint32_t token_bytes, own[HELD], real;  // byte offsets; which of the lane's entries there are
    T raw[STEP][HELD];
    float now[STEP][HELD];
    __device__ __forceinline__ vectors_of_step(const vectors<T>& v, const place& w, uint32_t lane, uint32_t t0, uint32_t n)
        : step(v.data + (int64_t)w.b * v.batch_stride + (int64_t)w.g * v.group_stride + (int64_t)t0 * v.token_stride),
          token_bytes((uint32_t)v.token_stride * (uint32_t)sizeof(T)), real(0u) {
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i) {
            const uint32_t entry = lane % 16u + 16u * i;
            own[i] = min(entry, n - 1u) * (uint32_t)sizeof(T);
            real |= entry < n ? 1u << i : 0u;
        }
    }
    __device__ __forceinline__ void load() {
        const ovl_lane::region r(step);
        const uint32_t bytes = ovl_lane::anew(token_bytes);
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j)
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) raw[j][i] = r.template load<T>(own[i], j * bytes);
    }
    // Only `left` tokens (at least one) are there: those behind are read as the last.
    __device__ __forceinline__ void load_some(uint32_t left) {
        const ovl_lane::region r(step);
        const uint32_t bytes = ovl_lane::anew(token_bytes);
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j)
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) raw[j][i] = r.template load<T>(own[i], min(j, left - 1u) * bytes);
    }
    // The loaded ones become the present ones.  Entries past the state and tokens behind the sequence (`tokens` of the step's
    // are in it) become zero: they then add nothing anywhere.
    __device__ __forceinline__ void take(uint32_t tokens) {
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j)
#pragma unroll
            for (uint32_t i = 0; i < HELD; ++i) {
                now[j][i] = (real >> i & 1u) != 0u ? widen<T>(raw[j][i]) : 0.0f;
                ovl_lane::keep(now[j][i]);
            }
        if (tokens < STEP)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j)
#pragma unroll
                for (uint32_t i = 0; i < HELD; ++i) now[j][i] = j < tokens ? now[j][i] : 0.0f;
    }
    __device__ __forceinline__ void move() {        // to the next step
        step = reinterpret_cast<const T*>(reinterpret_cast<const char*>(step) + STEP * (uint64_t)token_bytes);
    }
};

// The vectors of TOKENS tokens in LDS, S entries each, read in pieces of up to 16 entries one piece ahead of their use: an
// LDS read takes about as long as a dozen instructions.  BACKWARD: the tokens from the last.  All indexes are constants
// once the loops are unrolled.
template <int S, uint32_t TOKENS, bool BACKWARD> struct vector_queue {
    static constexpr uint32_t WIDE = S < 16 ? S : 16, PIECES = S / WIDE;
    const float* lds;
    float held[2][WIDE];
    __device__ __forceinline__ explicit vector_queue(const float* lds_) : lds(lds_) {}
    __device__ __forceinline__ void read(uint32_t piece) {
        const uint32_t token = BACKWARD ? TOKENS - 1u - piece / PIECES : piece / PIECES;
#pragma unroll
        for (uint32_t e = 0; e < WIDE; ++e) held[piece & 1u][e] = lds[token * S + piece % PIECES * WIDE + e];
    }
    __device__ __forceinline__ void begin() { read(0u); }
    __device__ __forceinline__ void next(uint32_t j, uint32_t i) {
        if (j * PIECES + i + 1u < TOKENS * PIECES) read(j * PIECES + i + 1u);
    }
    __device__ __forceinline__ float get(uint32_t j, uint32_t i, uint32_t e) const { return held[(j * PIECES + i) & 1u][e]; }
};

// ---------------------------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------------------------

// S entries (all of a state, padded) in the lane of their channel: nothing has to be summed across lanes.  A wavefront owns
// 64 channels and a chunk and takes STEP tokens at a time, the next ones' loads in flight.  The four wavefronts of a
// workgroup have nothing to do with each other; they are one workgroup so that every SIMD of a compute unit gets one.
// 4 sequences of 2048 tokens, 4096 channels of 16 entries, bf16: full pass with kept states 143 us, pass over states only
// 97 us, where the recurrence's instructions alone take 82 (with the output) and 64 us; the rest is softplus, the gate,
// conversions and addresses, once per token and channel.  One sequence of 8192 tokens, 2048 channels: 71 and 51 us.
// OUTPUT: the full pass (y, the last state, the kept states).  Otherwise only states: the chunk's own effect on a zero
// state (`local`, `dt_sum`), or the kept states.
template <typename T, int S, bool OUTPUT>
__global__ void __launch_bounds__(THREADS)
scan_forward_kernel(scan_args<T> p, uint32_t units, uint32_t chunks, T* y, float* last, float* saved, const float* entry, float* local,
                    float* dt_sum) {
    typedef reader<T, STEP, 1> reads;
    // B is taken from the lanes of a row, where it costs nothing as the factor of a product; C, a factor of a fused
    // multiply-add, which has no such form, comes through a part of the LDS that is the wavefront's own
    __shared__ __attribute__((aligned(16))) float lds_vectors[WAVES][OUTPUT ? 2 : 1][OUTPUT ? STEP * S : 4];
    const uint32_t lane = threadIdx.x % 64u, wave = ovl_lane::wavefront(threadIdx.x / 64u), unit = blockIdx.x * WAVES + wave;
    if (unit >= units) return;              // there is no barrier
    float (*lds_C)[OUTPUT ? STEP * S : 4] = lds_vectors[wave];
    const place w = find_place<1>(p, unit, lane, 0u, chunks);
    const uint64_t chunk_row = ((uint64_t)w.b * p.chunks + w.chunk) * p.channels;
    const uint64_t state_row = (uint64_t)w.b * p.channels + w.channel;

    float h[S], A2[S];
    load_entries(A2, p.A + (uint64_t)w.channel * p.state, 0u, p.state);
#pragma unroll
    for (int s = 0; s < S; ++s) { A2[s] = rate_(A2[s]); h[s] = 0.0f; }
    if (entry != nullptr) load_states(h, entry + chunk_row * S, 0u, w.channel, p.channels);
    else if (local == nullptr && p.entering != nullptr) load_entries(h, p.entering + state_row * p.state, 0u, p.state);
    const float bias = p.delta_bias != nullptr ? p.delta_bias[w.channel] : 0.0f;
    const float skip = OUTPUT && p.D != nullptr ? p.D[w.channel] : 0.0f;
    const bool gate = OUTPUT && p.z.data != nullptr;
    float dt_total = 0.0f;

    // tokens from `start` on; those of the sequence end before `stop`
    const uint32_t start = w.first * TILE, stop = max(start, min(w.last * TILE, w.end)), behind = min(w.last * TILE, p.length);
    reads u_from(p.u, w, start), delta_from(p.delta, w, start), z_from(p.z, w, start);
    writer<T, STEP, 1> out_at(w, p.length, p.channels, start);
    vectors_of_step<T, S> B(p.B, w, lane, start, p.state);
    vector_stage<T, S, STEP, 64> C(p.C, w, lane, start, p.state);
    float* kept = saved + ((uint64_t)w.b * p.tiles + w.first) * p.channels * S;
    T u_next[STEP], delta_next[STEP], z_next[STEP], done[STEP];
    auto fetch = [&](uint32_t left) {
        if (left >= STEP) {
            u_from.load(u_next);
            delta_from.load(delta_next);
            if (gate) z_from.load(z_next);
            B.load();
            if (OUTPUT) C.load();
        } else {
            u_from.load_some(u_next, left, 0u);
            delta_from.load_some(delta_next, left, 0u);
            if (gate) z_from.load_some(z_next, left, 0u);
            B.load_some(left);
            if (OUTPUT) C.load_some(left);
        }
        u_from.template move<1>();
        delta_from.template move<1>();
        z_from.template move<1>();
        B.move();
        C.template move<1>();
    };
    if (start < stop) fetch(p.length - start);

    uint32_t t0 = start;
    for (uint32_t turn = 0; t0 < stop; t0 += STEP, turn ^= 1u) {
        const uint32_t tokens = stop - t0;
        B.take(tokens);
        if (OUTPUT) C.store(lds_C[turn], tokens, p.state);
        float u[STEP], dt[STEP], z[STEP], out[STEP];
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j) {
            u[j] = widen<T>(u_next[j]);
            dt[j] = widen<T>(delta_next[j]) + bias;
            z[j] = 0.0f;
        }
        if (gate)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) z[j] = widen<T>(z_next[j]);
        settle(u);
        settle(dt);
        settle(z);
        if (OUTPUT) ovl_lane::wave_sync();
        // Stores stand here, in front of the next loads: loads are waited for in the order of all memory accesses, so
        // stores behind them would be waited for as well, right after they were issued.
        if (OUTPUT && t0 > start) {
            out_at.store(y, done);
            out_at.template move<1>();
        }
        if (saved != nullptr && t0 % TILE == 0u) {
            store_states(h, kept, 0u, w.channel, p.channels);
            kept += (uint64_t)p.channels * S;
        }
        if (tokens > STEP) fetch(p.length - t0 - STEP);
        if (p.softplus)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) dt[j] = softplus_(dt[j]);
        if (tokens < STEP)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) {
                dt[j] = j < tokens ? dt[j] : 0.0f;
                u[j] = j < tokens ? u[j] : 0.0f;
            }
        // C of the next token is on its way from LDS while the present one is worked on
        vector_queue<S, STEP, false> C_queue(lds_C[OUTPUT ? turn : 0u]);
        if (OUTPUT) C_queue.begin();
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j) {
            const float x = dt[j] * u[j];
            if (!OUTPUT) dt_total += dt[j];
            float sum = skip * u[j];
#pragma unroll
            for (uint32_t i = 0; i < B.HELD; ++i) {
                const ovl_lane::row_values B_row(B.now[j][i]);
                if (OUTPUT) C_queue.next(j, i);
#pragma unroll
                for (uint32_t e = 0; e < B.IN_ROW; ++e) {
                    const uint32_t s = 16u * i + e;
                    const float a = ovl_lane::exp2_(dt[j] * A2[s]);
                    h[s] = fmaf(a, h[s], B_row.at(e) * x);
                    if (OUTPUT) sum = fmaf(C_queue.get(j, i, e), h[s], sum);
                }
                if (OUTPUT) __builtin_amdgcn_sched_barrier(0);
            }
            out[j] = sum;
        }
        if (OUTPUT) {
            if (gate)
#pragma unroll
                for (uint32_t j = 0; j < STEP; ++j) out[j] *= z[j] * sigmoid_(z[j]);
            if (tokens < STEP)
#pragma unroll
                for (uint32_t j = 0; j < STEP; ++j) out[j] = j < tokens ? out[j] : 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) done[j] = narrow<T>(out[j]);
        }
    }
    if (OUTPUT) {
        if (start < stop) {                 // the last step's outputs
            out_at.store_some(y, done, behind - (t0 - STEP), 0u);
            out_at.template move<1>();
        }
        T none[STEP];                       // behind the sequence the outputs are zero
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j) none[j] = narrow<T>(0.0f);
        for (; t0 < behind; t0 += STEP) {
            out_at.store_some(y, none, behind - t0, 0u);
            out_at.template move<1>();
        }
    }
    if (OUTPUT && w.chunk + 1u == p.chunks) store_entries(h, last + state_row * p.state, 0u, p.state);
    if (!OUTPUT && local != nullptr) {
        store_states(h, local + chunk_row * S, 0u, w.channel, p.channels);
        dt_sum[chunk_row + w.channel] = dt_total;
    }
}

// Joins the chunks: in place of each chunk's own effect `local` the state that enters it.  A thread takes AHEAD chunks of a
// (sequence, channel, state entry) in a row, which it reads before any is overwritten, and `walkers` threads (a power of
// two) stand behind one another: each makes one step (decay, effect) of its chunks, the states between them are joined
// through LDS, and each hands its own state on.  So 128 chunks are one trip of 16 walkers, where a thread alone would wait
// for memory 16 times (128 chunks of 2048 channels of 16 entries: 19.6 us alone, 9.2 with 16 walkers).  REVERSE: the gradient's recurrence, which
// enters chunks from their ends.
constexpr uint32_t AHEAD = 8, MOST_WALKERS = 16;
constexpr uint32_t join_ids(uint32_t walkers) { return walkers < 4u ? THREADS / walkers : 64u; }

template <bool REVERSE>
__global__ void __launch_bounds__(64 * MOST_WALKERS)
scan_join_kernel(const float* A, const float* start, float* local, const float* dt_sum, uint32_t batch, uint32_t channels,
                 uint32_t state, uint32_t padded, uint32_t chunks, uint32_t walkers) {
    __shared__ float lds_step[2][64 * MOST_WALKERS];
    const uint32_t ids = join_ids(walkers), column = threadIdx.x % ids;
    const uint32_t walker = ovl_lane::wavefront(threadIdx.x / 64u) * 64u / ids;
    const uint64_t row_size = (uint64_t)channels * padded, all = batch * row_size;
    // threads behind the last entry repeat it, but do not write
    const uint64_t wanted = (uint64_t)blockIdx.x * ids + column, id = wanted < all ? wanted : all - 1u;
    // the place inside a chunk's states (state_offset above), and what it stands for
    const uint32_t b = (uint32_t)(id / row_size), in = (uint32_t)(id % row_size);
    const uint32_t channel = in / 4u % channels, n = in / 4u / channels * 4u + in % 4u;
    const uint64_t row = (uint64_t)b * channels + channel;
    const bool real = n < state;
    const float A2 = real ? rate_(A[(uint64_t)channel * state + n]) : 0.0f;
    float h = real && start != nullptr ? start[row * state + n] : 0.0f;
    for (uint32_t trip = 0; trip < chunks; trip += walkers * AHEAD) {
        const uint32_t base = trip + walker * AHEAD;
        float own[AHEAD], decay[AHEAD];
        uint64_t at[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t step = min(base + i, chunks - 1u);
            const uint32_t chunk = REVERSE ? chunks - 1u - step : step;
            at[i] = (uint64_t)b * chunks + chunk;
            // the last chunk of the walk has no effect to pass on (and none was computed)
            const bool passes = step + 1u < chunks;
            own[i] = passes ? local[at[i] * row_size + in] : 0.0f;
            decay[i] = passes ? dt_sum[at[i] * channels + channel] : 0.0f;
        }
        float effect = 0.0f, factor = 1.0f;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            decay[i] = ovl_lane::exp2_(decay[i] * A2);
            effect = fmaf(decay[i], effect, own[i]);
            factor *= decay[i];
        }
        if (walkers > 1u) {
            lds_step[0][threadIdx.x] = factor;
            lds_step[1][threadIdx.x] = effect;
            __syncthreads();                // also: every chunk of the trip has been read
        }
        float mine = h;
        for (uint32_t before = 0; before < walker; ++before)
            mine = fmaf(lds_step[0][before * ids + column], mine, lds_step[1][before * ids + column]);
        if (walkers > 1u) {
            for (uint32_t other = 0; other < walkers; ++other)
                h = fmaf(lds_step[0][other * ids + column], h, lds_step[1][other * ids + column]);
            __syncthreads();
        } else {
            h = fmaf(factor, h, effect);
        }
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            if (base + i < chunks) {
                if (wanted < all) local[at[i] * row_size + in] = mine;
                mine = fmaf(decay[i], mine, own[i]);
            }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------------------------------

template <typename T> struct gradient_args {
    sequence<T> d_y;
    const float* d_last;
    T *d_u, *d_delta, *d_z;
    float* d_entering;
    // parts that a later kernel sums: dB and dC per block of channels, dA, dD and d_bias per sequence and chunk
    float *vector_part, *A_part, *D_part, *bias_part;
    uint32_t padded, slices;                // entries of a state as it is kept; slices of it that are worked on in turn
};

// The effect of a chunk on a zero gradient entering at its end: r = a (C dy + r), tokens walked from the last.  Lanes as in
// the forward pass.
template <typename T, int S>
__global__ void __launch_bounds__(THREADS)
scan_gradient_local_kernel(scan_args<T> p, uint32_t units, sequence<T> d_y, float* local, float* dt_sum) {
    typedef reader<T, STEP, 1> reads;
    __shared__ __attribute__((aligned(16))) float lds_vectors[WAVES][2][STEP * S];
    const uint32_t lane = threadIdx.x % 64u, wave = ovl_lane::wavefront(threadIdx.x / 64u), unit = blockIdx.x * WAVES + wave;
    if (unit >= units) return;              // there is no barrier
    float (*lds_C)[STEP * S] = lds_vectors[wave];
    const place w = find_place<1>(p, unit, lane, 1u, p.chunks - 1u);       // nothing enters from the first chunk
    const uint64_t chunk_row = ((uint64_t)w.b * p.chunks + w.chunk) * p.channels;
    float r[S], A2[S];
    load_entries(A2, p.A + (uint64_t)w.channel * p.state, 0u, p.state);
#pragma unroll
    for (int s = 0; s < S; ++s) { A2[s] = rate_(A2[s]); r[s] = 0.0f; }
    const float bias = p.delta_bias != nullptr ? p.delta_bias[w.channel] : 0.0f;
    const bool gate = p.z.data != nullptr;
    float dt_total = 0.0f;

    const uint32_t start = w.first * TILE, stop = max(start, min(w.last * TILE, w.end));
    const uint32_t steps = (stop - start + STEP - 1u) / STEP, t_last = start + (max(steps, 1u) - 1u) * STEP;
    reads delta_from(p.delta, w, t_last), z_from(p.z, w, t_last), dy_from(d_y, w, t_last);
    vector_stage<T, S, STEP, 64> C_next(p.C, w, lane, t_last, p.state);
    T delta_next[STEP], z_next[STEP], dy_next[STEP];
    auto fetch = [&](uint32_t left) {
        if (left >= STEP) {
            delta_from.load(delta_next);
            dy_from.load(dy_next);
            if (gate) z_from.load(z_next);
            C_next.load();
        } else {
            delta_from.load_some(delta_next, left, 0u);
            dy_from.load_some(dy_next, left, 0u);
            if (gate) z_from.load_some(z_next, left, 0u);
            C_next.load_some(left);
        }
        delta_from.template move<-1>();
        dy_from.template move<-1>();
        z_from.template move<-1>();
        C_next.template move<-1>();
    };
    if (steps > 0u) fetch(p.length - t_last);
    for (uint32_t step = steps; step-- > 0u;) {
        const uint32_t t0 = start + step * STEP, tokens = stop - t0, turn = step & 1u;
        C_next.store(lds_C[turn], tokens, p.state);
        float dt[STEP], d[STEP], z[STEP];
#pragma unroll
        for (uint32_t j = 0; j < STEP; ++j) {
            dt[j] = widen<T>(delta_next[j]) + bias;
            d[j] = widen<T>(dy_next[j]);
            z[j] = 0.0f;
        }
        if (gate)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) z[j] = widen<T>(z_next[j]);
        settle(dt);
        settle(d);
        settle(z);
        ovl_lane::wave_sync();
        if (step > 0u) fetch(STEP);
        if (p.softplus)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) dt[j] = softplus_(dt[j]);
        if (gate)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) d[j] *= z[j] * sigmoid_(z[j]);
        if (tokens < STEP)
#pragma unroll
            for (uint32_t j = 0; j < STEP; ++j) {
                dt[j] = j < tokens ? dt[j] : 0.0f;
                d[j] = j < tokens ? d[j] : 0.0f;
            }
        vector_queue<S, STEP, true> C_queue(lds_C[turn]);
        C_queue.begin();
#pragma unroll
        for (uint32_t k = 0; k < STEP; ++k) {
            const uint32_t j = STEP - 1u - k;
            dt_total += dt[j];
#pragma unroll
            for (uint32_t i = 0; i < C_queue.PIECES; ++i) {
                C_queue.next(k, i);
#pragma unroll
                for (uint32_t e = 0; e < C_queue.WIDE; ++e) {
                    const uint32_t s = i * C_queue.WIDE + e;
                    r[s] = ovl_lane::exp2_(dt[j] * A2[s]) * fmaf(d[j], C_queue.get(k, i, e), r[s]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    store_states(r, local + chunk_row * S, 0u, w.channel, p.channels);
    dt_sum[chunk_row + w.channel] = dt_total;
}

// Sums over the 16 channels of a wavefront (the quads) of 2 S values per lane and token, four tokens together.  Within a
// row every addition halves the number of values a lane holds: afterwards quad i of a row holds entries
// m + (S / 2) (i & 1) of the first (i < 2) or second set; the rows then trade tokens: row r ends with token r.
template <int S> struct channel_sums {
    static constexpr int KEPT = S / 2;
    float kept[KEPT][4];
    __device__ __forceinline__ void add(const float (&first)[S], const float (&second)[S], int k, uint32_t lane) {
        const bool far = lane & 8u, odd = lane & 4u;
        float v[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const float a = first[s] + ovl_lane::row_round<8>(first[s]), b = second[s] + ovl_lane::row_round<8>(second[s]);
            v[s] = far ? b : a;
        }
#pragma unroll
        for (int m = 0; m < KEPT; ++m) {
            const float a = v[m] + ovl_lane::row_down<4>(v[m]), b = v[m + KEPT] + ovl_lane::row_up<4>(v[m + KEPT]);
            kept[m][k] = odd ? b : a;
        }
    }
    // Writes the sums to lds [2][TILE][NP] for the four tokens from `t`.
    __device__ __forceinline__ void put(float* lds, uint32_t t, uint32_t lane) {
        constexpr uint32_t NP = 4 * S;
        const uint32_t row = lane / 16u, quad = (lane / 4u) & 3u, q = lane & 3u;
#pragma unroll
        for (int m = 0; m < KEPT; ++m) {
            float a = kept[m][0], b = kept[m][1], c = kept[m][2], d = kept[m][3];
            ovl_lane::swap_halves(a, c);
            ovl_lane::swap_halves(b, d);
            float even = a + c, odd = b + d;
            ovl_lane::swap_rows(even, odd);
            const uint32_t s = m + KEPT * (quad & 1u);
            lds[((quad >> 1) * TILE + t + row) * NP + q * S + s] = even + odd;
        }
    }
};

// The gradient, tile by tile from the last: the tile's states are computed again from the one kept before it, then the
// recurrence runs backwards through them.  A quad owns a channel, a lane S of its entries; a workgroup owns 64 channels of
// one group, so that its part of dB and dC, [2][token][entry], is a sum over its lanes and wavefronts.  B and C are in LDS
// as float32, one barrier per tile for them and one for the sums.
//
// Bound by the vector ALU: 26 instructions per token and 64 entries (14 of the recurrences, 4.5 of the sums over channels,
// 2 of the states computed twice, the rest per token and channel), and the vector ALU is busy for 380 of the 465 us
// that 4 sequences of 2048 tokens, 4096 channels of 16 entries in bf16 take.
//
// SLICED: states of more than 16 entries are taken 16 at a time, tile by tile, and what a lane keeps of the other slices is
// in LDS: with 8 or 16 entries in a lane only one wavefront fits a SIMD, or none without spilling (2048 channels of 32
// entries 781 us and 620 in slices, of 64 entries 3289 and 1141; of 16 entries 320).
template <typename T, int S, bool GATE, bool SLICED>
__global__ void __launch_bounds__(THREADS) OVL_LANE_WAVES(2)
scan_backward_kernel(scan_args<T> p, gradient_args<T> g, const float* saved, const float* entry) {
    constexpr uint32_t NP = 4 * S, MOST_SLICES = SLICED ? 4 : 1;
    // tokens whose states and decays are held in registers at a time
    constexpr uint32_t SUB = S <= 2 ? 16 : 8, SUBS = TILE / SUB;
    __shared__ __attribute__((aligned(16))) float lds_B[TILE * NP];
    __shared__ __attribute__((aligned(16))) float lds_C[TILE * NP];
    __shared__ float lds_sums[WAVES][2 * TILE * NP];
    // what a lane keeps of the slices it is not working on: r and dA; of a tile's slices before: y and its gradients
    __shared__ float lds_r[MOST_SLICES][S][SLICED ? THREADS : 1], lds_dA[MOST_SLICES][S][SLICED ? THREADS : 1];
    __shared__ float lds_before[3][QUADS][SLICED ? THREADS : 1];
    const place w = find_place<4>(p, blockIdx.x, threadIdx.x, 0u, p.chunks);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u, slices = SLICED ? g.slices : 1u;
    const uint32_t padded = SLICED ? g.padded : NP;
    const uint64_t chunk_row = ((uint64_t)w.b * p.chunks + w.chunk) * p.channels;
    const uint64_t state_row = (uint64_t)w.b * p.channels + w.channel;
    const float* A_row = p.A + (uint64_t)w.channel * p.state;

    float r[S], A2[S], dA[S];
    auto load_A2 = [&](uint32_t slice) {
        load_entries(A2, A_row, slice * 4u + w.q, p.state);
#pragma unroll
        for (int s = 0; s < S; ++s) A2[s] = rate_(A2[s]);
    };
    for (uint32_t slice = 0; slice < slices; ++slice) {
#pragma unroll
        for (int s = 0; s < S; ++s) { r[s] = 0.0f; dA[s] = 0.0f; }
        if (entry != nullptr) load_states(r, entry + chunk_row * padded, (slice * 4u + w.q) * S, w.channel, p.channels);
        else if (g.d_last != nullptr) load_entries(r, g.d_last + state_row * p.state, slice * 4u + w.q, p.state);
        if (SLICED)
#pragma unroll
            for (int s = 0; s < S; ++s) { lds_r[slice][s][threadIdx.x] = r[s]; lds_dA[slice][s][threadIdx.x] = 0.0f; }
    }
    if (!SLICED) load_A2(0u);
    const float bias = p.delta_bias != nullptr ? p.delta_bias[w.channel] : 0.0f;
    const float skip = p.D != nullptr ? p.D[w.channel] : 0.0f;
    float dD = 0.0f, dbias = 0.0f;

    const uint32_t stop = max(w.first, min(w.last, (w.end + TILE - 1u) / TILE)), start = (max(stop, 1u) - 1u) * TILE;
    typedef reader<T, QUADS, 4> reads;
    typedef writer<T, QUADS, 4> writes;
    typedef vector_stage<T, NP, TILE, THREADS> stage;
    reads u_from(p.u, w, start), delta_from(p.delta, w, start), z_from(p.z, w, start), dy_from(g.d_y, w, start);
    writes out_at(w, p.length, p.channels, start);
    stage B_all(p.B, w, threadIdx.x, start, p.state), C_all(p.C, w, threadIdx.x, start, p.state);
    const float* kept = saved + ((uint64_t)w.b * p.tiles + start / TILE) * p.channels * padded;
    float* const part = g.vector_part + (((uint64_t)w.g * p.blocks + w.block) * p.batch + w.b) * p.length * (2u * p.state);

    // behind the sequence all gradients are zero
    for (uint32_t t = stop * TILE + threadIdx.x / BLOCK; t < min(w.last * TILE, p.length); t += THREADS / BLOCK) {
        const uint32_t c = w.block * BLOCK + threadIdx.x % BLOCK;
        if (c < p.per_group) {
            const uint64_t at = ((uint64_t)w.b * p.length + t) * p.channels + w.g * p.per_group + c;
            g.d_u[at] = narrow<T>(0.0f);
            g.d_delta[at] = narrow<T>(0.0f);
            if (GATE) g.d_z[at] = narrow<T>(0.0f);
        }
        for (uint32_t n = threadIdx.x % BLOCK; n < 2u * p.state; n += BLOCK) part[(uint64_t)t * 2u * p.state + n] = 0.0f;
    }

    for (uint32_t tile = stop; tile-- > w.first;) {
        const uint32_t t0 = tile * TILE, left = p.length - t0, tokens = w.end - t0;
        T u_raw[QUADS], delta_raw[QUADS], z_raw[QUADS], dy_raw[QUADS], du_done[QUADS], ddelta_done[QUADS], dz_done[QUADS];
        float h_first[S];
        // Loaded here and not a tile ahead: the registers for that cost the second wavefront of a SIMD, which hides more
        // (261 registers and one wavefront: 690 us, 247 and two: 500 us for 4 x 2048 tokens of 4096 channels).
        if (left >= TILE) {
            u_from.load(u_raw);
            delta_from.load(delta_raw);
            dy_from.load(dy_raw);
            if (GATE) z_from.load(z_raw);
            if (!SLICED) {
                B_all.load();
                C_all.load();
            }
        } else {
            u_from.load_some(u_raw, left, w.q);
            delta_from.load_some(delta_raw, left, w.q);
            dy_from.load_some(dy_raw, left, w.q);
            if (GATE) z_from.load_some(z_raw, left, w.q);
            if (!SLICED) {
                B_all.load_some(left);
                C_all.load_some(left);
            }
        }
        if (!SLICED) {
            load_states(h_first, kept, w.q * S, w.channel, p.channels);
            B_all.store(lds_B, tokens, p.state);
            C_all.store(lds_C, tokens, p.state);
        }
        float u[QUADS], dt[QUADS], x[QUADS], d[QUADS];
        float slope[QUADS], gate_slope[QUADS];              // d dt / d delta; d z is gate_slope times y
#pragma unroll
        for (uint32_t j = 0; j < QUADS; ++j) {
            // lanes without a channel of their own add nothing to any sum
            u[j] = w.active ? widen<T>(u_raw[j]) : 0.0f;
            dt[j] = widen<T>(delta_raw[j]) + bias;
            d[j] = w.active ? widen<T>(dy_raw[j]) : 0.0f;
            gate_slope[j] = GATE ? widen<T>(z_raw[j]) : 0.0f;
        }
        // also lets every wavefront finish reading lds_sums of the tile before
        if (!SLICED) __syncthreads();
        if (tokens < TILE)
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) {
                u[j] = 4u * j + w.q < tokens ? u[j] : 0.0f;
                d[j] = 4u * j + w.q < tokens ? d[j] : 0.0f;
                gate_slope[j] = 4u * j + w.q < tokens ? gate_slope[j] : 0.0f;
            }
        if (GATE)
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) {
                const float z = gate_slope[j], s = sigmoid_(z), d_out = d[j];
                d[j] = d_out * z * s;
                gate_slope[j] = d_out * s * fmaf(z, 1.0f - s, 1.0f);
            }
#pragma unroll
        for (uint32_t j = 0; j < QUADS; ++j) slope[j] = 1.0f;
        if (p.softplus)
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) {
                slope[j] = sigmoid_(dt[j]);
                dt[j] = softplus_(dt[j]);
            }
        if (tokens < TILE)
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) dt[j] = 4u * j + w.q < tokens ? dt[j] : 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < QUADS; ++j) {
            x[j] = dt[j] * u[j];
            dD = fmaf(d[j], u[j], dD);
        }

        for (uint32_t slice = 0; slice < slices; ++slice) {
            const uint32_t first = slice * NP;
            if (SLICED) {
                stage B_stage(p.B, w, threadIdx.x, t0, p.state, first), C_stage(p.C, w, threadIdx.x, t0, p.state, first);
                if (left >= TILE) {
                    B_stage.load();
                    C_stage.load();
                } else {
                    B_stage.load_some(left);
                    C_stage.load_some(left);
                }
                load_states(h_first, kept, (slice * 4u + w.q) * S, w.channel, p.channels);
                load_A2(slice);
                B_stage.store(lds_B, tokens, p.state - first);
                C_stage.store(lds_C, tokens, p.state - first);
#pragma unroll
                for (int s = 0; s < S; ++s) { r[s] = lds_r[slice][s][threadIdx.x]; dA[s] = lds_dA[slice][s][threadIdx.x]; }
                // also lets every wavefront finish reading lds_sums of the slice before
                __syncthreads();
            }
            float h[SUBS][S];
#pragma unroll
            for (int s = 0; s < S; ++s) h[0][s] = h_first[s];
            // the states that enter the later parts of the tile
#pragma unroll
            for (uint32_t part_of = 0; part_of + 1u < SUBS; ++part_of) {
#pragma unroll
                for (int s = 0; s < S; ++s) h[part_of + 1u][s] = h[part_of][s];
#pragma unroll
                for (uint32_t i = 0; i < SUB; ++i) {
                    const uint32_t at = part_of * SUB + i;
                    const float* Bt = lds_B + at * NP + w.q * S;
                    const float dt_k = quad_pick(dt[at / 4u], at & 3u), x_k = quad_pick(x[at / 4u], at & 3u);
#pragma unroll
                    for (int s = 0; s < S; ++s)
                        h[part_of + 1u][s] = fmaf(ovl_lane::exp2_(dt_k * A2[s]), h[part_of + 1u][s], x_k * Bt[s]);
                    if (at % 4u == 3u) __builtin_amdgcn_sched_barrier(0);
                }
            }

            float dA_tile[S];
#pragma unroll
            for (int s = 0; s < S; ++s) dA_tile[s] = 0.0f;
#pragma unroll
            for (uint32_t back = 0; back < SUBS; ++back) {
                const uint32_t part_of = SUBS - 1u - back;
                float a[SUB][S], state[SUB + 1u][S], y[SUB / 4u];
#pragma unroll
                for (int s = 0; s < S; ++s) state[0][s] = h[part_of][s];
#pragma unroll
                for (uint32_t i = 0; i < SUB; i += 4u) {
                    const uint32_t j = part_of * (SUB / 4u) + i / 4u;
                    float sums[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float* Bt = lds_B + (4u * j + k) * NP + w.q * S;
                        const float* Ct = lds_C + (4u * j + k) * NP + w.q * S;
                        const float dt_k = quad_pick(dt[j], k), x_k = quad_pick(x[j], k);
                        sums[k] = 0.0f;
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            a[i + k][s] = ovl_lane::exp2_(dt_k * A2[s]);
                            state[i + k + 1][s] = fmaf(a[i + k][s], state[i + k][s], x_k * Bt[s]);
                            if (GATE) sums[k] = fmaf(Ct[s], state[i + k + 1][s], sums[k]);
                        }
                    }
                    y[i / 4u] = GATE ? quad_scatter_sum(sums, w.q) : 0.0f;
                    // (keeps the scheduler from loading B and C of all tokens at once)
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (uint32_t step = 0; step < SUB; step += 4u) {
                    const uint32_t i = SUB - 4u - step, j = part_of * (SUB / 4u) + i / 4u;
                    channel_sums<S> sums;
                    float dx[4], through[4];
#pragma unroll
                    for (int k = 3; k >= 0; --k) {
                        const float* Bt = lds_B + (4u * j + k) * NP + w.q * S;
                        const float* Ct = lds_C + (4u * j + k) * NP + w.q * S;
                        const float dt_k = quad_pick(dt[j], k), x_k = quad_pick(x[j], k), d_k = quad_pick(d[j], k);
                        float dB[S], dC[S];
                        dx[k] = 0.0f;
                        through[k] = 0.0f;
#pragma unroll
                        for (int s = 0; s < S; ++s) {
                            const float grad = fmaf(d_k, Ct[s], r[s]);
                            dx[k] = fmaf(grad, Bt[s], dx[k]);
                            dB[s] = grad * x_k;
                            dC[s] = d_k * state[i + k + 1][s];
                            r[s] = grad * a[i + k][s];
                            const float moved = r[s] * state[i + k][s];
                            dA_tile[s] = fmaf(dt_k, moved, dA_tile[s]);
                            through[k] = fmaf(moved, A2[s], through[k]);
                        }
                        sums.add(dB, dC, k, lane);
                    }
                    sums.put(lds_sums[wave], 4u * j, lane);
                    float d_x = quad_scatter_sum(dx, w.q), d_through = quad_scatter_sum(through, w.q), out = y[i / 4u];
                    if (SLICED && slice > 0u) {
                        d_x += lds_before[0][j][threadIdx.x];
                        d_through += lds_before[1][j][threadIdx.x];
                        if (GATE) out += lds_before[2][j][threadIdx.x];
                    }
                    if (SLICED && slice + 1u < slices) {
                        lds_before[0][j][threadIdx.x] = d_x;
                        lds_before[1][j][threadIdx.x] = d_through;
                        if (GATE) lds_before[2][j][threadIdx.x] = out;
                    } else {
                        float d_dt = fmaf(d_x, u[j], LN2 * d_through) * slope[j];
                        if (tokens < TILE) d_dt = 4u * j + w.q < tokens ? d_dt : 0.0f;
                        dbias += d_dt;
                        du_done[j] = narrow<T>(fmaf(d_x, dt[j], skip * d[j]));
                        ddelta_done[j] = narrow<T>(d_dt);
                        if (GATE) dz_done[j] = narrow<T>(gate_slope[j] * fmaf(skip, u[j], out));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int s = 0; s < S; ++s) dA[s] += dA_tile[s];
            if (SLICED)
#pragma unroll
                for (int s = 0; s < S; ++s) { lds_r[slice][s][threadIdx.x] = r[s]; lds_dA[slice][s][threadIdx.x] = dA[s]; }

            // the four wavefronts' sums, as [token][B entries, C entries]
            auto sum_up = [&] {
                __syncthreads();
                for (uint32_t at = threadIdx.x; at < 2u * TILE * NP; at += THREADS) {
                    const uint32_t set = at / (TILE * NP), t = at / NP % TILE, n = first + at % NP;
                    float sum = 0.0f;
#pragma unroll
                    for (uint32_t v = 0; v < WAVES; ++v) sum += lds_sums[v][at];
                    if (n < p.state && t < left) part[(uint64_t)(t0 + t) * 2u * p.state + set * p.state + n] = t < tokens ? sum : 0.0f;
                }
            };
            if (SLICED && slice + 1u < slices) {
                sum_up();
                continue;
            }
            if (tokens < TILE)
#pragma unroll
                for (uint32_t j = 0; j < QUADS; ++j) {
                    du_done[j] = 4u * j + w.q < tokens ? du_done[j] : narrow<T>(0.0f);
                    if (GATE) dz_done[j] = 4u * j + w.q < tokens ? dz_done[j] : narrow<T>(0.0f);
                }
            if (!w.active) {
            } else if (left >= TILE) {
                out_at.store(g.d_u, du_done);
                out_at.store(g.d_delta, ddelta_done);
                if (GATE) out_at.store(g.d_z, dz_done);
            } else {
                out_at.store_some(g.d_u, du_done, left, w.q);
                out_at.store_some(g.d_delta, ddelta_done, left, w.q);
                if (GATE) out_at.store_some(g.d_z, dz_done, left, w.q);
            }
            sum_up();
        }
        u_from.template move<-1>();
        delta_from.template move<-1>();
        dy_from.template move<-1>();
        z_from.template move<-1>();
        B_all.template move<-1>();
        C_all.template move<-1>();
        out_at.template move<-1>();
        kept -= (uint64_t)p.channels * padded;
    }
    if (w.active)
        for (uint32_t slice = 0; slice < slices; ++slice) {
            if (SLICED)
#pragma unroll
                for (int s = 0; s < S; ++s) { r[s] = lds_r[slice][s][threadIdx.x]; dA[s] = lds_dA[slice][s][threadIdx.x]; }
            store_states(dA, g.A_part + chunk_row * padded, (slice * 4u + w.q) * S, w.channel, p.channels);
            if (w.chunk == 0u && g.d_entering != nullptr) store_entries(r, g.d_entering + state_row * p.state, slice * 4u + w.q, p.state);
        }
    dD = quad_sum(dD);
    dbias = quad_sum(dbias);
    if (w.active && w.q == 0u) {
        g.D_part[chunk_row + w.channel] = dD;
        g.bias_part[chunk_row + w.channel] = dbias;
    }
}

// Sums the parts of dB and dC over the blocks of a group, one thread per result, and of dA, dD and d_bias over sequences
// and chunks, of which there may be thousands: there the sixteen wavefronts of a workgroup share the parts of 64 results
// that lie side by side.  The order of the additions is fixed.
constexpr uint32_t SHARES = 16;
template <typename T>
__global__ void __launch_bounds__(64 * SHARES)
scan_gradient_sum_kernel(const float* vector_part, const float* A_part, const float* D_part, const float* bias_part,
                         uint32_t batch, uint32_t length, uint32_t channels, uint32_t state, uint32_t padded,
                         uint32_t groups, uint32_t blocks, uint32_t rows, uint32_t vector_groups,
                         T* d_B, T* d_C, float* d_A, float* d_D, float* d_bias) {
    __shared__ float lds_sums[SHARES][64];
    const uint64_t per_block = (uint64_t)batch * length * 2u * state;
    if (blockIdx.x < vector_groups) {
        const uint64_t id = (uint64_t)blockIdx.x * (64u * SHARES) + threadIdx.x;
        if (id >= per_block * groups) return;
        const uint32_t g = (uint32_t)(id / per_block);
        const uint64_t in = id % per_block;
        const float* from = vector_part + (uint64_t)g * blocks * per_block + in;
        float sum = 0.0f;
#pragma unroll 8
        for (uint32_t k = 0; k < blocks; ++k) sum += from[k * per_block];
        const uint32_t n = (uint32_t)(in % (2u * state));
        const uint64_t token = in / (2u * state);
        T* to = n < state ? d_B : d_C;
        to[(token * groups + g) * state + (n < state ? n : n - state)] = narrow<T>(sum);
        return;
    }
    // dA in the order of its parts (state_offset above), then dD, then d_bias
    const uint32_t lane = threadIdx.x & 63u, share = ovl_lane::wavefront(threadIdx.x / 64u), entries = channels * padded;
    const uint32_t id = (blockIdx.x - vector_groups) * 64u + lane, channel = id < entries ? id / 4u % channels : (id - entries) % channels;
    const bool in_A = id < entries, in_D = !in_A && id < entries + channels;
    const uint32_t n = id / 4u / channels * 4u + id % 4u;       // of dA
    float* to = in_A ? (n < state ? d_A + (uint64_t)channel * state + n : nullptr)
                     : in_D ? (d_D != nullptr ? d_D + channel : nullptr)
                            : (d_bias != nullptr && id < entries + 2u * channels ? d_bias + channel : nullptr);
    float sum = 0.0f;
    if (to != nullptr) {
        const float* from = in_A ? A_part + id : (in_D ? D_part : bias_part) + channel;
        const uint64_t pace = in_A ? entries : channels;
#pragma unroll 8
        for (uint32_t k = share; k < rows; k += SHARES) sum += from[k * pace];
    }
    lds_sums[share][lane] = sum;
    __syncthreads();
    if (share != 0u || to == nullptr) return;
#pragma unroll
    for (uint32_t i = 1; i < SHARES; ++i) sum += lds_sums[i][lane];
    *to = sum;
}

// ---------------------------------------------------------------------------------------------------------------------
// one token
// ---------------------------------------------------------------------------------------------------------------------

// The recurrence once: a quad per (sequence, channel), a workgroup for 64 channels of a sequence.  Bound by reading and
// writing the state: 96 sequences of 4096 channels, 16 entries, bf16: 54 MB in 12.6 us, 4.3 TB/s (the same
// states again at once, which are still in the caches: 11.0 us); 2 of 1024: 3.0 us.
// WHOLE: a lane's S entries are all there, and accessed as vectors of 16 (S = 2: 8) aligned bytes.
template <typename T, int S, bool WHOLE>
__global__ void __launch_bounds__(THREADS)
scan_step_kernel(scan_args<T> p, uint32_t per_sequence, float* state, int64_t state_stride, T* y) {
    const uint32_t b = blockIdx.x / per_sequence, q = threadIdx.x & 3u;
    const uint32_t wanted = (blockIdx.x - b * per_sequence) * BLOCK + threadIdx.x / 4u;
    const bool active = wanted < p.channels;
    const uint32_t channel = min(wanted, p.channels - 1u);
    float* own = state + (int64_t)b * state_stride + (uint64_t)channel * p.state;
    const float* A = p.A + (uint64_t)channel * p.state;
    const uint32_t group = channel / p.per_group;
    const T* B = p.B.data + (int64_t)b * p.B.batch_stride + (int64_t)group * p.B.group_stride;
    const T* C = p.C.data + (int64_t)b * p.C.batch_stride + (int64_t)group * p.C.group_stride;
    float h[S], A_row[S], B_row[S], C_row[S];
    if constexpr (WHOLE) {
        typedef float vec __attribute__((ext_vector_type(S >= 4 ? 4 : S)));
        constexpr int PIECES = S >= 4 ? S / 4 : 1, WIDE = S >= 4 ? 4 : S;
        struct __attribute__((packed, aligned(sizeof(T)))) entries { T v[S]; };
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const vec v = *reinterpret_cast<const vec*>(own + q * S + i * WIDE);
            const vec a = *reinterpret_cast<const vec*>(A + q * S + i * WIDE);
#pragma unroll
            for (int k = 0; k < WIDE; ++k) { h[i * WIDE + k] = v[k]; A_row[i * WIDE + k] = a[k]; }
        }
        const entries b_row = *reinterpret_cast<const entries*>(B + q * S), c_row = *reinterpret_cast<const entries*>(C + q * S);
#pragma unroll
        for (int s = 0; s < S; ++s) { B_row[s] = widen<T>(b_row.v[s]); C_row[s] = widen<T>(c_row.v[s]); }
    } else {
        load_entries(h, own, q, p.state);
        load_entries(A_row, A, q, p.state);
#pragma unroll
        for (uint32_t s = 0; s < S; ++s) {
            const uint32_t at = min(q * S + s, p.state - 1u);
            B_row[s] = q * S + s < p.state ? widen<T>(B[at]) : 0.0f;
            C_row[s] = q * S + s < p.state ? widen<T>(C[at]) : 0.0f;
        }
    }
    const float u = widen<T>(p.u.data[(int64_t)b * p.u.batch_stride + channel]);
    float dt = widen<T>(p.delta.data[(int64_t)b * p.delta.batch_stride + channel]);
    const bool gate = p.z.data != nullptr;
    const float z = gate ? widen<T>(p.z.data[(int64_t)b * p.z.batch_stride + channel]) : 0.0f;
    if (p.delta_bias != nullptr) dt += p.delta_bias[channel];
    if (p.softplus) dt = softplus_(dt);
    const float x = dt * u;
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        h[s] = fmaf(ovl_lane::exp2_(dt * (A_row[s] * LOG2E)), h[s], x * B_row[s]);
        sum = fmaf(C_row[s], h[s], sum);
    }
    sum = quad_sum(sum);
    if (p.D != nullptr) sum = fmaf(p.D[channel], u, sum);
    if (gate) sum *= z * sigmoid_(z);
    if (!active) return;
    if constexpr (WHOLE) {
        typedef float vec __attribute__((ext_vector_type(S >= 4 ? 4 : S)));
        constexpr int PIECES = S >= 4 ? S / 4 : 1, WIDE = S >= 4 ? 4 : S;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            vec v;
#pragma unroll
            for (int k = 0; k < WIDE; ++k) v[k] = h[i * WIDE + k];
            *reinterpret_cast<vec*>(own + q * S + i * WIDE) = v;
        }
    } else {
        store_entries(h, own, q, p.state);
    }
    if (q == 0u) y[(uint64_t)b * p.channels + channel] = narrow<T>(sum);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------

using ovl_ssm::after_launch;
using ovl_ssm::fail;
using ovl_ssm::launchable;
using ovl_ssm::round_up;

// State entries per lane of a quad: the smallest variant that holds the state.
uint32_t entries_of(uint32_t state) { return state <= 8u ? 2u : state <= 16u ? 4u : state <= 32u ? 8u : 16u; }

struct plan {
    uint32_t per_group, blocks, tiles, chunks, chunk_tiles, entries;
    uint64_t strands;                       // 64 channels of a sequence: a wavefront, in the backward pass a workgroup
};

enum class direction { forward, backward, token };

// Into how many chunks the length is split, where the split pays for its second evaluation of the decays: into so many that
// the passes with a channel per lane have 4096 wavefronts, four for each SIMD.  Not all of them are resident together in every
// variant: with 8, 16, 32, 64 entries the full pass has registers for 4, 3, 2, 1 wavefronts on a SIMD, the forward pass over
// states for 6, 4, 3, 1, the gradient's for 5, 4, 3, 2; the others start as these end.  4096 channels of 16 entries, bf16:
//   forward    below 1024 strands (one wavefront per SIMD without a split): 12 sequences of 2048 tokens, 768 strands, take
//              694 us split and 761 else, 16 sequences 813 split and 768 else
//   backward   below 512, since a strand is four wavefronts of its main kernel: 4 sequences, 256 strands, take 598 us split
//              and 735 else, 8 sequences 1139 split and 996 else
// Fewer than six tiles are not worth two more launches (64 tokens of 64 channels of 8 entries: 21 us split, 17 else), but a
// chunk may be a single tile (3 sequences of 333 tokens, 650 channels of 8 entries in float32: 20 us, with four tiles 45).
void chunks_for(plan& p, direction of) {
    const uint64_t enough = of == direction::backward ? 512 : 1024, wanted = (4096 + p.strands - 1) / p.strands;
    p.chunks = p.strands < enough && p.tiles >= 6u ? (uint32_t)(wanted < p.tiles ? wanted : p.tiles) : 1u;
    p.chunk_tiles = (p.tiles + p.chunks - 1u) / p.chunks;
    p.chunks = (p.tiles + p.chunk_tiles - 1u) / p.chunk_tiles;
}

// Workgroups of the kernel that sums the gradients' parts: for dB and dC, and for the parameters.
struct sum_grid { uint64_t vector_groups, rest; };
sum_grid sum_grid_of(const ovl_ssm_scan* s, const plan& p) {
    const uint64_t vector_all = (uint64_t)s->groups * s->batch * s->length * 2u * s->state;
    return {(vector_all + 64u * SHARES - 1u) / (64u * SHARES), ((uint64_t)s->channels * (4u * p.entries + 2u) + 63u) / 64u};
}

// Checks a scan, and plans it.
int check(const char* who, const ovl_ssm_scan* s, direction of, plan& p) {
    const bool token = of == direction::token;
    const std::string name(who);
    if (s == nullptr) return fail(OVL_SSM_EINVAL, name + ": null scan");
    if (s->batch == 0 || s->length == 0 || s->channels == 0 || s->state == 0 || s->groups == 0)
        return fail(OVL_SSM_EINVAL, name + ": sizes must be positive");
    if (s->state > 64u) return fail(OVL_SSM_EINVAL, name + ": at most 64 state entries per channel");
    if (s->channels % s->groups != 0u) return fail(OVL_SSM_EINVAL, name + ": groups must divide channels");
    if (s->dtype != OVL_SSM_FLOAT16 && s->dtype != OVL_SSM_FLOAT32 && s->dtype != OVL_SSM_BFLOAT16)
        return fail(OVL_SSM_EINVAL, name + ": unknown element type");
    if (s->u.data == nullptr || s->delta.data == nullptr || s->B.data == nullptr || s->C.data == nullptr || s->A == nullptr)
        return fail(OVL_SSM_EINVAL, name + ": null tensor");
    if (token && (s->length != 1u || s->lengths != nullptr))
        return fail(OVL_SSM_EINVAL, name + ": a step takes one token of every sequence");
    if (s->length > (1u << 30)) return fail(OVL_SSM_EINVAL, name + ": length must be at most 2^30");
    // a lane's offset inside a tile has 32 bits
    if (s->channels > (1u << 22)) return fail(OVL_SSM_EINVAL, name + ": at most 2^22 channels");
    for (const int64_t stride : {s->u.token_stride, s->delta.token_stride, s->z.token_stride, s->B.token_stride, s->C.token_stride})
        if (!token && s->length > 1u && (stride < 0 || stride > OVL_SSM_MAX_TOKEN_STRIDE))
            return fail(OVL_SSM_EINVAL, name + ": token strides must be 0 to 2^25 elements");
    p.entries = entries_of(s->state);
    p.per_group = s->channels / s->groups;
    p.blocks = (p.per_group + BLOCK - 1u) / BLOCK;
    p.tiles = (s->length + TILE - 1u) / TILE;
    p.strands = (uint64_t)s->batch * s->groups * p.blocks;
    chunks_for(p, of);
    // all launches of the call; the forward pass has four strands to a workgroup, and its join, where the length is split,
    // few entries
    bool fits = (uint64_t)s->batch * s->length <= (1ull << 38) / ((uint64_t)s->groups * 2u * s->state);
    if (of == direction::forward) fits = fits && launchable((p.strands * p.chunks + WAVES - 1) / WAVES, THREADS);
    if (of == direction::backward) {
        const sum_grid sums = sum_grid_of(s, p);
        fits = fits && launchable(p.strands * p.chunks, THREADS) && launchable(sums.vector_groups + sums.rest, 64u * SHARES);
    }
    if (token) fits = fits && launchable((uint64_t)s->batch * ((s->channels + BLOCK - 1u) / BLOCK), THREADS);
    if (!fits) return fail(OVL_SSM_EINVAL, name + ": too many elements for one launch");
    return OVL_SSM_OK;
}

template <typename T>
scan_args<T> make_args(const ovl_ssm_scan* s, const plan& p) {
    auto seq = [](const ovl_ssm_sequence& v) {
        return sequence<T>{static_cast<const T*>(v.data), v.batch_stride, v.token_stride};
    };
    auto vec = [](const ovl_ssm_vectors& v) {
        return vectors<T>{static_cast<const T*>(v.data), v.batch_stride, v.token_stride, v.group_stride};
    };
    return scan_args<T>{s->batch, s->length, s->channels, s->state, s->groups, p.per_group, p.blocks, p.tiles, p.chunks,
                        p.chunk_tiles, s->softplus, seq(s->u), seq(s->delta), seq(s->z), vec(s->B), vec(s->C), s->A, s->D,
                        s->delta_bias, s->entering, s->lengths};
}

// Scratch memory, in floats: the chunks' states and sums of dt; for the backward pass also the parts of the gradients.
struct layout {
    uint64_t local, dt_sum, vector_part, A_part, D_part, bias_part, all;
};
layout lay_out(const ovl_ssm_scan* s, const plan& p, bool backward) {
    layout at;
    const uint64_t rows = (uint64_t)s->batch * p.chunks * s->channels, padded = 4u * p.entries;
    uint64_t next = 0;
    auto take = [&](uint64_t n) { const uint64_t here = next; next += round_up(n, 64); return here; };
    at.local = take(p.chunks > 1u ? rows * padded : 0);
    at.dt_sum = take(p.chunks > 1u ? rows : 0);
    at.vector_part = take(backward ? (uint64_t)s->groups * p.blocks * s->batch * s->length * 2u * s->state : 0);
    at.A_part = take(backward ? rows * padded : 0);
    at.D_part = take(backward ? rows : 0);
    at.bias_part = take(backward ? rows : 0);
    at.all = next;
    return at;
}

template <bool REVERSE>
void join(const ovl_ssm_scan* s, const plan& p, const float* start, float* local, const float* dt_sum, hipStream_t stream) {
    const uint64_t all = (uint64_t)s->batch * s->channels * 4u * p.entries;
    uint32_t walkers = 1;
    while (walkers < MOST_WALKERS && walkers * AHEAD < p.chunks) walkers *= 2u;
    const uint32_t ids = join_ids(walkers);
    hipLaunchKernelGGL((scan_join_kernel<REVERSE>), dim3((uint32_t)((all + ids - 1) / ids)), dim3(ids * walkers), 0, stream,
                       s->A, start, local, dt_sum, s->batch, s->channels, s->state, 4u * p.entries, p.chunks, walkers);
}

// Workgroups of kernels whose wavefronts take a unit each.
dim3 groups_of(uint64_t units) { return dim3((uint32_t)((units + WAVES - 1) / WAVES)); }

// ENTRIES: state entries per lane of a quad; a lane with a channel of its own holds four times as many.
template <typename T, int ENTRIES>
void forward(const ovl_ssm_scan* s, const plan& p, T* y, float* last, float* saved, float* scratch, hipStream_t stream) {
    constexpr int S = 4 * ENTRIES;
    const scan_args<T> args = make_args<T>(s, p);
    const layout at = lay_out(s, p, false);
    const float* entry = nullptr;
    if (p.chunks > 1u) {
        float* local = scratch + at.local;
        float* dt_sum = scratch + at.dt_sum;
        hipLaunchKernelGGL((scan_forward_kernel<T, S, false>), groups_of(p.strands * (p.chunks - 1u)), dim3(THREADS), 0,
                           stream, args, (uint32_t)(p.strands * (p.chunks - 1u)), p.chunks - 1u, static_cast<T*>(nullptr), static_cast<float*>(nullptr),
                           static_cast<float*>(nullptr), static_cast<const float*>(nullptr), local, dt_sum);
        join<false>(s, p, s->entering, local, dt_sum, stream);
        entry = local;
    }
    const uint32_t units = (uint32_t)(p.strands * p.chunks);
    if (y != nullptr)
        hipLaunchKernelGGL((scan_forward_kernel<T, S, true>), groups_of(units), dim3(THREADS), 0, stream, args, units, p.chunks, y, last, saved,
                           entry, static_cast<float*>(nullptr), static_cast<float*>(nullptr));
    else
        hipLaunchKernelGGL((scan_forward_kernel<T, S, false>), groups_of(units), dim3(THREADS), 0, stream, args, units, p.chunks, y, last, saved,
                           entry, static_cast<float*>(nullptr), static_cast<float*>(nullptr));
}

template <typename T, int S>
void backward(const ovl_ssm_scan* s, const plan& p, const float* saved, const ovl_ssm_scan_gradients* g, float* scratch,
              hipStream_t stream) {
    const scan_args<T> args = make_args<T>(s, p);
    const layout at = lay_out(s, p, true);
    gradient_args<T> to;
    to.d_y = sequence<T>{static_cast<const T*>(g->d_y.data), g->d_y.batch_stride, g->d_y.token_stride};
    to.d_last = g->d_last;
    to.d_u = static_cast<T*>(g->d_u);
    to.d_delta = static_cast<T*>(g->d_delta);
    to.d_z = static_cast<T*>(g->d_z);
    to.d_entering = g->d_entering;
    to.vector_part = scratch + at.vector_part;
    to.A_part = scratch + at.A_part;
    to.D_part = scratch + at.D_part;
    to.bias_part = scratch + at.bias_part;
    const float* entry = nullptr;
    if (p.chunks > 1u) {
        float* local = scratch + at.local;
        float* dt_sum = scratch + at.dt_sum;
        hipLaunchKernelGGL((scan_gradient_local_kernel<T, 4 * S>), groups_of(p.strands * (p.chunks - 1u)), dim3(THREADS), 0,
                           stream, args, (uint32_t)(p.strands * (p.chunks - 1u)), to.d_y, local, dt_sum);
        join<true>(s, p, g->d_last, local, dt_sum, stream);
        entry = local;
    }
    const dim3 grid((uint32_t)(p.strands * p.chunks));
    constexpr bool SLICED = S > 4;
    constexpr int HELD = SLICED ? 4 : S;
    to.padded = 4u * p.entries;
    to.slices = (s->state + 4u * HELD - 1u) / (4u * HELD);
    if (s->z.data != nullptr)
        hipLaunchKernelGGL((scan_backward_kernel<T, HELD, true, SLICED>), grid, dim3(THREADS), 0, stream, args, to, saved, entry);
    else
        hipLaunchKernelGGL((scan_backward_kernel<T, HELD, false, SLICED>), grid, dim3(THREADS), 0, stream, args, to, saved, entry);
    const sum_grid sums = sum_grid_of(s, p);
    const uint32_t vector_groups = (uint32_t)sums.vector_groups;
    hipLaunchKernelGGL((scan_gradient_sum_kernel<T>), dim3((uint32_t)(sums.vector_groups + sums.rest)), dim3(64u * SHARES), 0, stream, to.vector_part,
                       to.A_part, to.D_part, to.bias_part, s->batch, s->length, s->channels, s->state, 4u * p.entries,
                       s->groups, p.blocks, s->batch * p.chunks, vector_groups, static_cast<T*>(g->d_B),
                       static_cast<T*>(g->d_C), g->d_A, g->d_D, g->d_delta_bias);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int S>
void step(const ovl_ssm_scan* s, const plan& p, float* h, int64_t stride, T* y, hipStream_t stream) {
    const scan_args<T> args = make_args<T>(s, p);
    const uint32_t per_sequence = (s->channels + BLOCK - 1u) / BLOCK;
    const dim3 grid(s->batch * per_sequence);
    const bool whole = s->state == 4u * S && aligned16(h) && aligned16(s->A) && stride % 4 == 0;
    if (whole) hipLaunchKernelGGL((scan_step_kernel<T, S, true>), grid, dim3(THREADS), 0, stream, args, per_sequence, h, stride, y);
    else hipLaunchKernelGGL((scan_step_kernel<T, S, false>), grid, dim3(THREADS), 0, stream, args, per_sequence, h, stride, y);
}

// Calls F<T, S>(...) for the scan's element type and state.
#define OVL_SSM_BY_STATE(F, T, ...)                          \
    switch (p.entries) {                                     \
        case 2u: F<T, 2>(__VA_ARGS__); break;                \
        case 4u: F<T, 4>(__VA_ARGS__); break;                \
        case 8u: F<T, 8>(__VA_ARGS__); break;                \
        default: F<T, 16>(__VA_ARGS__); break;               \
    }

}  // namespace

extern "C" {

uint64_t ovl_ssm_scan_workspace_bytes(const ovl_ssm_scan* s, int32_t backward_pass) {
    plan p;
    if (check("ovl_ssm_scan_workspace_bytes", s, backward_pass != 0 ? direction::backward : direction::forward, p) != OVL_SSM_OK) return 0;
    return lay_out(s, p, backward_pass != 0).all * sizeof(float);
}

uint64_t ovl_ssm_scan_saved_bytes(const ovl_ssm_scan* s) {
    plan p;
    if (check("ovl_ssm_scan_saved_bytes", s, direction::forward, p) != OVL_SSM_OK) return 0;
    return (uint64_t)s->batch * p.tiles * s->channels * 4u * p.entries * sizeof(float);
}

int ovl_ssm_scan_forward(const ovl_ssm_scan* s, void* y, float* last, float* saved, void* workspace,
                         uint64_t workspace_bytes, void* hip_stream) {
    plan p;
    const int rc = check("ovl_ssm_scan_forward", s, direction::forward, p);
    if (rc != OVL_SSM_OK) return rc;
    if ((y == nullptr) != (last == nullptr) || (y == nullptr && saved == nullptr))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_scan_forward: y and last go together; without them saved is needed");
    const uint64_t need = lay_out(s, p, false).all * sizeof(float);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_scan_forward: workspace too small or not 16-byte aligned");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    float* scratch = static_cast<float*>(workspace);
    switch (s->dtype) {
        case OVL_SSM_FLOAT32: OVL_SSM_BY_STATE(forward, float, s, p, static_cast<float*>(y), last, saved, scratch, stream) break;
        case OVL_SSM_FLOAT16: OVL_SSM_BY_STATE(forward, f16, s, p, static_cast<f16*>(y), last, saved, scratch, stream) break;
        default: OVL_SSM_BY_STATE(forward, bf16, s, p, static_cast<bf16*>(y), last, saved, scratch, stream) break;
    }
    return after_launch("ovl_ssm_scan_forward");
}

int ovl_ssm_scan_backward(const ovl_ssm_scan* s, const float* saved, const ovl_ssm_scan_gradients* g, void* workspace,
                          uint64_t workspace_bytes, void* hip_stream) {
    plan p;
    const int rc = check("ovl_ssm_scan_backward", s, direction::backward, p);
    if (rc != OVL_SSM_OK) return rc;
    if (g == nullptr || saved == nullptr || g->d_y.data == nullptr || g->d_u == nullptr || g->d_delta == nullptr ||
        g->d_B == nullptr || g->d_C == nullptr || g->d_A == nullptr || (s->z.data != nullptr && g->d_z == nullptr))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_scan_backward: null tensor");
    if (s->length > 1u && (g->d_y.token_stride < 0 || g->d_y.token_stride > OVL_SSM_MAX_TOKEN_STRIDE))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_scan_backward: token strides must be 0 to 2^25 elements");
    if (workspace == nullptr || workspace_bytes < lay_out(s, p, true).all * sizeof(float) || !aligned16(workspace))
        return fail(OVL_SSM_EINVAL, "ovl_ssm_scan_backward: workspace too small or not 16-byte aligned");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    float* scratch = static_cast<float*>(workspace);
    switch (s->dtype) {
        case OVL_SSM_FLOAT32: OVL_SSM_BY_STATE(backward, float, s, p, saved, g, scratch, stream) break;
        case OVL_SSM_FLOAT16: OVL_SSM_BY_STATE(backward, f16, s, p, saved, g, scratch, stream) break;
        default: OVL_SSM_BY_STATE(backward, bf16, s, p, saved, g, scratch, stream) break;
    }
    return after_launch("ovl_ssm_scan_backward");
}

int ovl_ssm_scan_step(const ovl_ssm_scan* s, float* h, int64_t h_batch_stride, void* y, void* hip_stream) {
    plan p;
    const int rc = check("ovl_ssm_scan_step", s, direction::token, p);
    if (rc != OVL_SSM_OK) return rc;
    if (h == nullptr || y == nullptr) return fail(OVL_SSM_EINVAL, "ovl_ssm_scan_step: null tensor");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    switch (s->dtype) {
        case OVL_SSM_FLOAT32: OVL_SSM_BY_STATE(step, float, s, p, h, h_batch_stride, static_cast<float*>(y), stream) break;
        case OVL_SSM_FLOAT16: OVL_SSM_BY_STATE(step, f16, s, p, h, h_batch_stride, static_cast<f16*>(y), stream) break;
        default: OVL_SSM_BY_STATE(step, bf16, s, p, h, h_batch_stride, static_cast<bf16*>(y), stream) break;
    }
    return after_launch("ovl_ssm_scan_step");
}

}  // extern "C"
