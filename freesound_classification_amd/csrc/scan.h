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
#pragma once
#include "seq.h"

namespace fsc {

constexpr int kTile = 16;                // frames staged together; also the distance of the kept states
constexpr int kPad = kTile + 4;          // row of an LDS array [channel][frame]: 16-byte rows that start in different banks
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct ScanPlan {
    int lanes, per_lane;                 // L, NS
    int channels_block;                  // CB = 256 / L
    int group_channels, group_blocks;    // channels of a group, blocks of CB channels it takes
    int blocks;                          // groups * group_blocks
    int tiles, segments, segment_tiles;
    int wide;                            // E neighbouring channels can be read and written at once
    __host__ __device__ int padded_states() const { return lanes * per_lane; }
    __host__ __device__ long padded_channels() const { return (long)blocks * channels_block; }
};

inline ScanPlan scan_plan(const fsc_selective_scan_args& a) {
    ScanPlan p{};
    p.lanes = a.states <= 16 ? 4 : a.states <= 32 ? 8 : 16;
    p.per_lane = a.states <= 4 ? 1 : a.states <= 8 ? 2 : 4;
    p.channels_block = 256 / p.lanes;
    p.group_channels = a.channels / a.groups;
    p.group_blocks = ceil_div(p.group_channels, p.channels_block);
    p.blocks = a.groups * p.group_blocks;
    p.tiles = ceil_div(a.length, kTile);
    const long have = (long)a.batch * p.blocks, wanted = 1024;
    p.segments = 1;
    if (have * 2 <= wanted && p.tiles >= 4) {
        long want = (wanted + have - 1) / have, most = p.tiles / 2;
        if (most > 32) most = 32;
        p.segments = (int)(want < most ? want : most);
    }
    p.segment_tiles = p.tiles > 0 ? ceil_div(p.tiles, p.segments) : 1;
    p.segments = p.tiles > 0 ? ceil_div(p.tiles, p.segment_tiles) : 1;
    const int e = kTile / p.lanes;
    const size_t unit = e * dtype_bytes(a.dtype);
    auto fits = [&](const void* ptr, long batch, long time) { return ptr == nullptr || (aligned(ptr, unit) && batch % e == 0 && time % e == 0); };
    p.wide = p.group_channels % e == 0 && fits(a.u, a.u_batch, a.u_time) && fits(a.dt, a.dt_batch, a.dt_time) &&
             fits(a.z, a.z_batch, a.z_time) && fits(a.dy, a.dy_batch, a.dy_time) && fits(a.y, 0, 0) && fits(a.du, 0, 0) &&
             fits(a.ddt, 0, 0) && fits(a.dz, 0, 0);
    return p;
}

inline const char* scan_bad(const fsc_selective_scan_args* a) {
    if (a == nullptr) return "null arguments";
    if (!dtype_ok(a->dtype)) return "unknown dtype";
    if (a->batch < 0 || a->length < 0 || a->channels < 0) return "negative size";
    if (a->states < 1 || a->states > 64) return "1 to 64 states";
    if (a->groups < 1 || a->channels % a->groups != 0) return "groups do not divide the channels";
    if (a->channels > 0 && a->a_log == nullptr) return "null a_log";
    if ((long)a->batch * ((a->channels / a->groups / 16 + 1) * (long)a->groups) > 0x3FFFFFFL || a->length > 0x7FFFFFF0)
        return "batch * channels or length is too large";
    return nullptr;
}

__device__ __forceinline__ int scan_frames(const fsc_selective_scan_args& a, int n) {
    if (a.lengths == nullptr) return a.length;
    const int l = a.lengths[n];
    return l < 0 ? 0 : l > a.length ? a.length : l;
}

__device__ __forceinline__ int tiles_with(int frames) { return (frames + kTile - 1) / kTile; }

__device__ __forceinline__ float sigmoid_fast(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -kLog2e));
}

// log(1 + e^v).  log(w) e / (w - 1) with w = 1 + e^v as rounded: what the rounding of w loses cancels, so small values keep their bits.
__device__ __forceinline__ float softplus_fast(float v) {
    const float e = __builtin_amdgcn_exp2f(v * kLog2e), w = 1.0f + e;
    const float soft = w == 1.0f ? e : __builtin_amdgcn_logf(w) * kLn2 * (e * __builtin_amdgcn_rcpf(w - 1.0f));
    return v > 20.0f ? v : soft;
}

// Where a workgroup and its threads stand.
template <int L, int NS>
struct ScanPlace {
    static constexpr int CB = 256 / L, E = kTile / L, SP = L * NS, ROWS = SP / 16 > 0 ? SP / 16 : 1;
    int n, block, segment;       // sequence, channel block, segment of time
    int group, c0, have;         // channel group; first channel of the block, its channels that exist
    int te, ce, he;              // elementwise: frame in the tile, first channel in the block, how many of the E exist
    int ch, sg, channel;         // scan: channel in the block, share of the states; channel index (clamped for lanes without one)
    bool real;                   // the scan lane has a channel
    __device__ ScanPlace(const fsc_selective_scan_args& a, const ScanPlan& p) {
        // segments vary fastest but one: blocks of one sequence's segment, which read the same B and C, follow one another
        const int per = p.blocks * p.segments;
        n = blockIdx.x / per;
        const int rest = blockIdx.x % per;
        segment = rest / p.blocks;
        block = rest % p.blocks;
        group = block / p.group_blocks;
        const int in_group = (block % p.group_blocks) * CB;
        c0 = group * p.group_channels + in_group;
        have = p.group_channels - in_group < CB ? p.group_channels - in_group : CB;
        te = threadIdx.x >> 4;
        ce = (threadIdx.x & 15) * E;
        he = have - ce < 0 ? 0 : have - ce < E ? have - ce : E;
        ch = threadIdx.x / L;
        sg = threadIdx.x % L;
        real = ch < have;
        channel = c0 + (real ? ch : 0);
    }
    // element (row, state) of a B / C tile that this thread stages as its j-th
    __device__ int bc_row(int j) const { return (threadIdx.x + j * 256) / SP; }
    __device__ int bc_state(int j) const { return (threadIdx.x + j * 256) % SP; }
    __device__ bool bc_mine(int j) const { return threadIdx.x + j * 256 < kTile * SP; }
    // this block's slot among the kept states [sequence][block][tile], each CB x SP floats in scan order
    __device__ long kept(const ScanPlan& p, int tile) const {
        return ((((long)n * p.blocks + block) * p.tiles + tile) * 256 + threadIdx.x) * NS;
    }
    // ... and among the segments' ends [sequence][segment][block]
    __device__ long end(const ScanPlan& p, int seg) const { return ((((long)n * p.segments + seg) * p.blocks + block) * 256 + threadIdx.x) * NS; }
    __device__ long end_delta(const ScanPlan& p, int seg) const { return (((long)n * p.segments + seg) * p.blocks + block) * CB + ch; }
};

// -exp(a_log) log2(e) of the lane's states: exp(delta A) = 2^(delta A2).  0 for states that do not exist.
template <int L, int NS>
__device__ __forceinline__ void scan_rates(const fsc_selective_scan_args& a, const ScanPlace<L, NS>& w, float (&a2)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = w.sg * NS + i;
        a2[i] = w.real && s < a.states ? -expf(a.a_log[(long)w.channel * a.states + s]) * kLog2e : 0.f;
    }
}

// The lane's states of a (batch, channels, states) tensor, zeros without one.
template <int L, int NS>
__device__ __forceinline__ void scan_state(const fsc_selective_scan_args& a, const ScanPlace<L, NS>& w, const float* from, float (&h)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = w.sg * NS + i;
        h[i] = from != nullptr && w.real && s < a.states ? from[((long)w.n * a.channels + w.channel) * a.states + s] : 0.f;
    }
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

}  // namespace fsc
