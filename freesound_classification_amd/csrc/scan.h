// What the forward and the backward of the selective scan share: the split of the work, the staging of a tile of frames.
//
// The recurrence is independent for every (sequence, channel, state) and serial in time; per element it costs an exponential and a few
// multiply-adds, so it is bound by the vector ALU and its transcendental rate, not by HBM (S = 16: 64 states' work for the 8 bytes of a
// channel's frame).  A workgroup of four waves owns the CB channels of a block and walks tiles of 16 frames:
//   * elementwise: thread = (frame, E neighbouring channels).  softplus, delta u, silu once a (frame, channel) instead of once a state;
//     rows are read with wide loads along the channels, the next tile's while this one is worked on;
//   * scan: L lanes share a channel, each holds NS of its states in registers.  delta / delta u come from LDS four frames at a time
//     ([channel][frame]), B / C a row a frame; the sum over the states is NS multiply-adds and log2 L lane exchanges.
// Where sequences x channel blocks do not fill the card, time is cut into segments: a first launch computes each segment's end from zero
// (and the sum of its delta: exp(A sum) is the segment's decay), the main launch joins the ends in front of its own segment.
// Measured with 16 states, bf16, ragged: 2 x 16384 frames of 2048 channels 255 us + 177 for the ends (9 vector instructions an element, 5 of them the
// recurrence); 8 x 2048 of 1024 channels 72 + 49, backward 225 + 54 (19 instructions an element; h and exp(delta A) of a tile's frames take half the
// registers and leave two waves a SIMD).
#pragma once
#include "seq.h"

namespace fsc {

constexpr int kTile = 16;                // frames staged together; also the distance of the kept states
constexpr int kPad = kTile + 4;          // row of an LDS array [channel][frame]: 16-byte rows that start in different banks
constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.69314718055994530942f;      // log2 e = kLog2e + kLog2eLow

struct ScanPlan {
    int lanes, per_lane;                 // L, NS
    int channels_block;                  // CB = 256 / L
    int group_channels, group_blocks;    // channels of a group, blocks of CB channels it takes
    int blocks;                          // groups * group_blocks
    int tiles, segments;                 // of 16 frames, of the longest sequence; segments of time (each sequence's own length in equal parts)
    int wide;                            // E neighbouring channels can be read and written at once
    __host__ __device__ int padded_states() const { return lanes * per_lane; }
    __host__ __device__ long padded_channels() const { return (long)blocks * channels_block; }
};

// LDS rows and channels of a block.  An elementwise thread has E neighbouring channels (one wide load); their rows lie 16 apart, so that the 16
// threads of a frame write neighbouring rows, which start in different banks: row r is channel (r % 16) E + r / 16.
__host__ __device__ inline int channel_of(int row, int e) { return (row & 15) * e + (row >> 4); }

inline ScanPlan scan_plan(const fsc_selective_scan_args& a) {
    ScanPlan p{};
    p.lanes = a.states <= 16 ? 4 : a.states <= 32 ? 8 : 16;
    p.per_lane = a.states <= 4 ? 1 : a.states <= 8 ? 2 : 4;
    p.channels_block = 256 / p.lanes;
    p.group_channels = a.channels / a.groups;
    p.group_blocks = ceil_div(p.group_channels, p.channels_block);
    p.blocks = a.groups * p.group_blocks;
    p.tiles = ceil_div(a.length, kTile);
    // 1024 workgroups are four waves a SIMD (a long training step, 8 x 2048 frames of 1024 channels, forward + its ends | backward + its ends:
    // 512: 151 | 309 us, 1024: 122 | 275, 2048: 128 | 293).  Segments double the exponentials, so half of that is enough not to cut (a batch of 128 x
    // 53 frames of 256 channels, 512 workgroups: 19 | 40 us whole, 30 | 61 cut in two).
    const long have = (long)a.batch * p.blocks, wanted = 1024;
    p.segments = 1;
    if (have > 0 && have * 2 < wanted && p.tiles >= 4) {        // (no sequences or no channels: nothing to cut)
        long want = (wanted + have - 1) / have, most = p.tiles / 2;
        if (most > 32) most = 32;
        p.segments = (int)(want < most ? want : most);
    }
    const int e = kTile / p.lanes;
    const size_t unit = e * dtype_bytes(a.dtype);
    auto fits = [&](const void* ptr, long batch, long time) { return ptr == nullptr || (aligned(ptr, unit) && batch % e == 0 && time % e == 0); };
    p.wide = p.group_channels % e == 0 && fits(a.u, a.u_batch, a.u_time) && fits(a.dt, a.dt_batch, a.dt_time) &&
             fits(a.z, a.z_batch, a.z_time) && fits(a.dy, a.dy_batch, a.dy_time) && fits(a.y, 0, 0) && fits(a.du, 0, 0) &&
             fits(a.ddt, 0, 0) && fits(a.dz, 0, 0);
    return p;
}

// Workgroups of 256 threads that one launch takes: fewer than 2^32 threads.
constexpr long kMostBlocks = (1L << 24) - 1;

inline const char* scan_bad(const fsc_selective_scan_args* a) {
    if (a == nullptr) return "null arguments";
    if (!dtype_ok(a->dtype)) return "unknown dtype";
    if (a->batch < 0 || a->length < 0 || a->channels < 0) return "negative size";
    if (a->states < 1 || a->states > 64) return "1 to 64 states";
    if (a->groups < 1 || a->channels % a->groups != 0) return "groups do not divide the channels";
    if (a->channels > 0 && a->a_log == nullptr) return "null a_log";
    if ((long)a->batch * ((a->channels / a->groups / 16 + 1) * (long)a->groups) > 0x3FFFFFFL || a->length > 0x7FFFFFF0)
        return "batch * channels or length is too large";
    // a tile's rows are addressed by 32-bit offsets from its first
    const long strides[] = {a->u_time, a->dt_time, a->z_time, a->b_time, a->c_time, a->dy_time, a->channels};
    for (const long s : strides)
        if (s < 0 || s > (1L << 26)) return "negative time strides, or time strides or channels above 2^26";
    return nullptr;
}

__device__ __forceinline__ int scan_frames(const fsc_selective_scan_args& a, int n) {
    if (a.lengths == nullptr) return a.length;
    const int l = a.lengths[n];
    return l < 0 ? 0 : l > a.length ? a.length : l;
}

// The (k % 4)-th of four frames' sums, which is the one that a lane writes.  (By value: a choice between elements of an array puts it in memory.)
__device__ __forceinline__ float pick4(float v0, float v1, float v2, float v3, int k) {
    const float low = k & 1 ? v1 : v0, high = k & 1 ? v3 : v2;
    return k & 2 ? high : low;
}

__device__ __forceinline__ int tiles_with(int frames) { return (frames + kTile - 1) / kTile; }

__device__ __forceinline__ float sigmoid_fast(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -kLog2e));
}

// Time steps are held in units of ln 2: exp(delta A) = 2^(delta2 A), and ln 2 is folded into B where it is staged.
// delta2 = log2(1 + 2^v2) = max(v2, 0) + log2(1 + e) with e = 2^-|v2| <= 1.  What the rounding of w = 1 + e loses, c = e - (w - 1), comes back as
// c log2(e): small values keep their bits.
__device__ __forceinline__ float softplus2(float v2) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(v2)), w = 1.0f + e;
    return fmaxf(v2, 0.f) + fmaf(e - (w - 1.0f), kLog2e, __builtin_amdgcn_logf(w));
}
__device__ __forceinline__ float sigmoid2(float v2) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v2)); }

// delta2 of E channels of a frame; 0 where the frame does not exist, so that the state passes it unchanged.  (The uniform choice stands outside the
// loop: the E chains of transcendentals then run side by side.)
template <int E, typename T>
__device__ __forceinline__ void time_steps(const Raw<T, E>& dt, const float (&bias2)[E], bool soft, bool there, float (&raw)[E], float (&delta)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) delta[i] = raw[i] = fmaf(dt[i], kLog2e, bias2[i]);
    if (soft) {
#pragma unroll
        for (int i = 0; i < E; ++i) delta[i] = softplus2(raw[i]);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) delta[i] = there ? delta[i] : 0.f;
}

// Where a workgroup and its threads stand.
template <int L, int NS>
struct ScanPlace {
    static constexpr int CB = 256 / L, E = kTile / L, SP = L * NS, ROWS = SP / 16 > 0 ? SP / 16 : 1;
    int n, block, segment;       // sequence, channel block, segment of time
    int group, c0, have;         // channel group; first channel of the block, its channels that exist
    int te, ce, he;              // elementwise: frame in the tile, first channel in the block, how many of the E exist
    int ch, sg, channel;         // scan: LDS row, share of the states; channel (of the first row for lanes without one)
    int first, work_end;         // the segment's tiles: the frames of the sequence in equal parts
    int zero_first, zero_end;    // its share of the tiles behind the sequence's end, which only get zeros
    bool whole;                  // every channel of the block exists and rows are read E channels at once
    bool real;                   // the scan lane has a channel
    int row, col;                // its row of the LDS arrays [channel][frame] and first column of B's and C's: those of zeros where it has no state
    __device__ ScanPlace(const fsc_selective_scan_args& a, const ScanPlan& p, int& len) {
        // segments vary fastest but one: blocks of one sequence's segment, which read the same B and C, follow one another
        const int per = p.blocks * p.segments;
        n = blockIdx.x / per;
        const int rest = blockIdx.x % per;
        segment = rest / p.blocks;
        block = rest % p.blocks;
        group = block / p.group_blocks;
        len = scan_frames(a, n);
        const int full = (len + kTile - 1) / kTile, part = (full + p.segments - 1) / p.segments, rest_part = (p.tiles - full + p.segments - 1) / p.segments;
        first = segment * part < full ? segment * part : full;
        work_end = first + part < full ? first + part : full;
        zero_first = full + segment * rest_part < p.tiles ? full + segment * rest_part : p.tiles;
        zero_end = zero_first + rest_part < p.tiles ? zero_first + rest_part : p.tiles;
        const int in_group = (block % p.group_blocks) * CB;
        c0 = group * p.group_channels + in_group;
        have = p.group_channels - in_group < CB ? p.group_channels - in_group : CB;
        whole = p.wide && have == CB;
        te = threadIdx.x >> 4;
        ce = (threadIdx.x & 15) * E;
        he = have - ce < 0 ? 0 : have - ce < E ? have - ce : E;
        ch = threadIdx.x / L;
        sg = threadIdx.x % L;
        real = channel_of(ch, E) < have;
        channel = c0 + (real ? channel_of(ch, E) : 0);
        // (a lane without states must not meet what is not finite in its neighbours': it would carry NaN into the sums over states and channels)
        const bool on = real && sg * NS < a.states;
        row = on ? ch : CB;
        col = on ? sg * NS : SP;
    }
    // whether the lane's i-th state exists; PARTIAL: the last lane with states has fewer than NS, the others are kept at 0 element by element
    template <bool PARTIAL>
    __device__ bool has(int i, int states) const { return !PARTIAL || sg * NS + i < states; }
    // LDS row of the elementwise thread's i-th channel
    __device__ int lds_row(int i) const { return (threadIdx.x & 15) + 16 * i; }
    // element (row, state) of a B / C tile that this thread stages as its j-th
    __device__ int bc_row(int j) const { return (threadIdx.x + j * 256) / SP; }
    __device__ int bc_state(int j) const { return (threadIdx.x + j * 256) % SP; }
    __device__ bool bc_mine(int j) const { return threadIdx.x + j * 256 < kTile * SP; }
    // this block's slot among the kept states [sequence][block][tile], each CB x SP floats in scan order
    __device__ long kept(const ScanPlan& p, int tile) const {
        return ((((long)n * p.blocks + block) * p.tiles + tile) * 256 + threadIdx.x) * NS;
    }
    // ... among the partial sums of dB and dC [sequence][block][tile], each 16 x 2 x SP floats
    __device__ long rows(const ScanPlan& p, int tile) const { return (((long)n * p.blocks + block) * p.tiles + tile) * (kTile * 2 * SP); }
    // ... and among the segments' ends [sequence][segment][block]
    __device__ long end(const ScanPlan& p, int seg) const { return ((((long)n * p.segments + seg) * p.blocks + block) * 256 + threadIdx.x) * NS; }
    __device__ long end_delta(const ScanPlan& p, int seg) const { return (((long)n * p.segments + seg) * p.blocks + block) * CB + ch; }
};

// An activation as the elementwise threads read it: E channels of frame te of a tile, as they lie in memory (converted where they are used, so that
// many loads are in flight).  The address is a uniform 64-bit one and a 32-bit offset of the thread; frames behind the last are read from
// the last, channels that do not exist from the block's last (the caller leaves both out).
template <typename T, int L, int NS>
struct ScanFrames {
    using Place = ScanPlace<L, NS>;
    static constexpr int E = Place::E;
    const char* base;
    long time;
    uint32_t off;
    __device__ ScanFrames(const Place& w, const void* ptr, long batch, long time_) : time(time_ * (long)sizeof(T)) {
        base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(ptr) + w.n * batch + w.c0);
        off = (uint32_t)w.te * (uint32_t)time + w.ce * (uint32_t)sizeof(T);
    }
    __device__ __forceinline__ void fetch(const Place& w, int tile, int len, Raw<T, E>& out) const {
        const int last = len - 1 - tile * kTile;
        const char* at = base + tile * kTile * time;
        const uint32_t o = w.te <= last ? off : (uint32_t)last * (uint32_t)time + w.ce * (uint32_t)sizeof(T);
        if (w.whole) {
            out.wide(reinterpret_cast<const T*>(at + o));
        } else {
            out.narrow([&](int i) {
                const int c = w.ce + i < w.have ? w.ce + i : w.have - 1;
                return reinterpret_cast<const T*>(at + (o + (uint32_t)(c - w.ce) * (uint32_t)sizeof(T)));
            });
        }
    }
};

// One tile of B or C as this thread stages it, in the same way; rows and states that do not exist are staged as 0, the others times `unit`.
template <typename T, int L, int NS>
struct ScanRows {
    using Place = ScanPlace<L, NS>;
    static constexpr int R = Place::ROWS;
    const char* base;
    long time;
    uint32_t off[R], col[R];
    Raw<T, 1> v[R];
    __device__ ScanRows(const Place& w, const void* ptr, long batch, long time_, long group, int states) : time(time_ * (long)sizeof(T)) {
        base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(ptr) + w.n * batch + w.group * group);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            col[j] = (uint32_t)(w.bc_state(j) < states ? w.bc_state(j) : states - 1) * (uint32_t)sizeof(T);
            off[j] = (uint32_t)row(w, j) * (uint32_t)time + col[j];
        }
    }
    // (with fewer than 16 states some threads stage nothing; they read the tile's last row)
    static __device__ int row(const Place& w, int j) { return w.bc_row(j) < kTile ? w.bc_row(j) : kTile - 1; }
    __device__ __forceinline__ void fetch(const Place& w, int tile, int len) {
        const int last = len - 1 - tile * kTile;
        const char* at = base + tile * kTile * time;
#pragma unroll
        for (int j = 0; j < R; ++j)
            v[j].wide(reinterpret_cast<const T*>(at + (row(w, j) <= last ? off[j] : (uint32_t)last * (uint32_t)time + col[j])));
    }
    __device__ __forceinline__ void stage(const Place& w, float (*to)[Place::SP + NS], int tile, int len, int states, float unit) const {
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (w.bc_mine(j)) to[w.bc_row(j)][w.bc_state(j)] = tile * kTile + w.bc_row(j) < len && w.bc_state(j) < states ? v[j][0] * unit : 0.f;
    }
};

// The LDS rows and columns of zeros, for lanes without states; visible behind the next barrier.
template <int ROWS>
__device__ __forceinline__ void scan_zero_row(float (&to)[ROWS][kPad]) {
    if (threadIdx.x < kPad) to[ROWS - 1][threadIdx.x] = 0.f;
}
template <int NS, int COLUMNS>
__device__ __forceinline__ void scan_zero_columns(float (&to)[kTile][COLUMNS]) {
    if (threadIdx.x < kTile * NS) to[threadIdx.x / NS][COLUMNS - NS + threadIdx.x % NS] = 0.f;
}

// An output row (batch, length, channels) of frame te of a tile, first channel ce of the block.
template <typename T, int L, int NS>
__device__ __forceinline__ T* scan_out(const fsc_selective_scan_args& a, const ScanPlace<L, NS>& w, void* base, int tile) {
    char* at = reinterpret_cast<char*>(reinterpret_cast<T*>(base) + ((long)w.n * a.length + (long)tile * kTile) * a.channels + w.c0);
    return reinterpret_cast<T*>(at + ((uint32_t)w.te * (uint32_t)a.channels + w.ce) * (uint32_t)sizeof(T));
}

// A = -exp(a_log), kept finite (a state that forgets everything passes frames with delta = 0 unchanged all the same); NaN stays NaN.  2^(x log2 e), where
// what the product's rounding and the constant's lose -- exp2 would multiply it by the exponent -- comes back as a factor: within 1.5 units in the last
// place.  (A single frame computes an A for each state that it reads: 256 x 2048 x 64 states 56.7 us, 58.2 with the library's expf.)
__device__ __forceinline__ float rate_of(float a_log) {
    const float x = a_log > 88.72f ? 88.72f : a_log < -104.0f ? -104.0f : a_log;      // (3.39e38; 0)
    const float hi = x * kLog2e, lo = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -hi)), e = __builtin_amdgcn_exp2f(hi);
    return -fmaf(e, lo * kLn2, e);
}

// A of the lane's states, 0 for states that do not exist.
template <int L, int NS>
__device__ __forceinline__ void scan_rates(const fsc_selective_scan_args& a, const ScanPlace<L, NS>& w, float (&rate)[NS]) {
    // (all the loads first, from places that exist: a load under a condition is waited for before the next)
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = w.sg * NS + i;
        rate[i] = a.a_log[(long)w.channel * a.states + (s < a.states ? s : 0)];
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) rate[i] = w.real && w.sg * NS + i < a.states ? rate_of(rate[i]) : 0.f;
}

// A state behind a segment: what was in front of it times the segment's decay, and the segment's end from zero.  An infinity outlasts a decay that is 0
// in fp32: frame by frame it meets factors above 0.
__device__ __forceinline__ float scan_join(float h, float rate, float sum_delta, float end) {
    const float joined = fmaf(__builtin_amdgcn_exp2f(rate * sum_delta), h, end);
    return joined == joined ? joined : h + end;
}

// The lane's states of a (batch, channels, states) tensor, zeros without one.
template <int L, int NS>
__device__ __forceinline__ void scan_state(const fsc_selective_scan_args& a, const ScanPlace<L, NS>& w, const float* from, float (&h)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = 0.f;
    if (from == nullptr) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = w.sg * NS + i;
        h[i] = from[((long)w.n * a.channels + w.channel) * a.states + (s < a.states ? s : 0)];
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = w.real && w.sg * NS + i < a.states ? h[i] : 0.f;
}

// E elementwise channels of a (channels) parameter, zeros without one and where a channel does not exist.
template <int L, int NS>
__device__ __forceinline__ void scan_param(const ScanPlace<L, NS>& w, const float* from, float (&out)[ScanPlace<L, NS>::E]) {
    constexpr int E = ScanPlace<L, NS>::E;
#pragma unroll
    for (int i = 0; i < E; ++i) out[i] = 0.f;
    if (from == nullptr) return;
#pragma unroll
    for (int i = 0; i < E; ++i) out[i] = from[w.c0 + (i < w.he ? w.ce + i : 0)];
#pragma unroll
    for (int i = 0; i < E; ++i) out[i] = i < w.he ? out[i] : 0.f;
}

// fn(lanes, per_lane) with the plan's two constants as types
template <typename Fn>
void with_scan_shape(const ScanPlan& p, Fn fn) {
    if (p.lanes == 16) fn(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
    else if (p.lanes == 8) fn(std::integral_constant<int, 8>(), std::integral_constant<int, 4>());
    else if (p.per_lane == 4) fn(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
    else if (p.per_lane == 2) fn(std::integral_constant<int, 4>(), std::integral_constant<int, 2>());
    else fn(std::integral_constant<int, 4>(), std::integral_constant<int, 1>());
}

// fn(partial) with, as a type, whether some lane has fewer states than its NS
template <int NS, typename Fn>
void with_partial(int states, Fn fn) {
    if constexpr (NS > 1) {
        if (states % NS != 0) return fn(std::true_type());
    }
    fn(std::false_type());
}

}  // namespace fsc
