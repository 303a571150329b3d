// Short causal convolution along time, one filter of K <= 8 taps a channel, SiLU behind it (the sequence head's local mixing).
//   pre[t] = bias + sum_k w[k] xin[t + k],  xin = [K - 1 frames before | x];  y = silu(pre)
// Bound: HBM (two passes over the frames forward, three backward), K multiply-adds and one exponential a value.  So each thread owns four channels
// and walks a strip of frames with the filter's window in registers: every frame is read once but for the K - 1 at a strip's ends,
// neighbouring threads read neighbouring channels.  Frames are taken eight at a time, all their loads issued before the first is used.
// Backward: the strip recomputes pre (cheaper than keeping it) and runs K - 1 frames past its end; dw / db are summed in registers, over
// the block's strips through LDS, over blocks by a second launch in a fixed order: equal inputs give equal bits.
// 4 x 8191 x 2048 in bf16, ragged (80 % of the frames), x a half of a wider tensor: forward 53 us (4.6 TB/s, what a copy of this size reaches), backward 90 - 95
// + 4 (3.8 TB/s: two waves a SIMD, the window, its gradient and the filters' sums fill the registers).  128 x 53 x 256 in fp32: 6.5 and 17 us.
#include <type_traits>

#include "seq.h"

namespace {

using fsc::load_row;
using fsc::store_row;

constexpr int kThreads = 256;
constexpr int kV = 4;             // channels a thread owns (8 in 16 bits, 16 bytes as well: twice the registers, 146 us for 91 on 4 x 8191 x 2048)

__device__ __forceinline__ float sigmoid_fast(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}

struct Plan {
    int groups;        // of V channels
    int strip, strips; // frames a thread walks, strips of one sequence
    int lanes;         // threads along the channel groups (a power of two), kThreads / lanes rows (sequence, strip) a block
    int rows;          // batch * strips
    int wide;          // every row of V channels is whole and aligned
    int wide_weights;
};

__device__ __forceinline__ int frames_of(const fsc_causal_conv_args& a, int n) {
    if (a.lengths == nullptr) return a.length;
    const int l = a.lengths[n];
    return l < 0 ? 0 : l > a.length ? a.length : l;
}

// Channels c .. c + V - 1 of frame t >= -(K - 1) of sequence n: x, the frames before it, or zeros behind its end.
template <typename T, int V>
__device__ __forceinline__ void frame(const fsc_causal_conv_args& a, int n, int c, int t, int len, bool wide, int have, float (&out)[V]) {
    if (t >= 0 && t < len) {
        load_row<V>(reinterpret_cast<const T*>(a.x) + n * a.x_batch + t * a.x_time + c, wide, have, out);
    } else if (t < 0 && a.initial != nullptr) {
        load_row<V>(reinterpret_cast<const T*>(a.initial) + ((long)n * (a.taps - 1) + a.taps - 1 + t) * a.channels + c, wide, have, out);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = 0.f;
    }
}

// Channels c .. c + V - 1 of the U frames from t, 0 <= t < len, as they lie in memory: U independent loads, which nothing waits for here.  Frames behind the
// last are read from the last; the caller leaves them out.
template <typename T, int V, int U>
__device__ __forceinline__ void fetch(const void* base, long batch, long time, int n, int c, int t, int len, bool wide, int have, fsc::Raw<T, V> (&raw)[U]) {
    const int last = len - 1 - t;
    const T* p = reinterpret_cast<const T*>(base) + n * batch + t * time + c;
    if (wide) {
#pragma unroll
        for (int j = 0; j < U; ++j) raw[j].wide(p + (j < last ? j : last) * (int)time);
    } else {
#pragma unroll
        for (int j = 0; j < U; ++j) raw[j].narrow([&](int i) { return p + (j < last ? j : last) * (int)time + (i < have ? i : have - 1); });
    }
}
template <typename T, int V, int U>
__device__ __forceinline__ void convert(const fsc::Raw<T, V> (&raw)[U], float (*out)[V]) {
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) out[j][i] = raw[j][i];
}
template <typename T, int V, int U>
__device__ __forceinline__ void frames(const void* base, long batch, long time, int n, int c, int t, int len, bool wide, int have, float (*out)[V]) {
    fsc::Raw<T, V> raw[U];
    fetch<T, V, U>(base, batch, time, n, c, t, len, wide, have, raw);
    convert<T, V, U>(raw, out);
}

// The K - 1 frames in front of a strip that begins at t0: frames of x, or (t0 == 0) the given window or zeros.
template <typename T, int K, int V>
__device__ __forceinline__ void window(const fsc_causal_conv_args& a, int n, int c, int t0, int len, bool wide, int have, float (*out)[V]) {
    if constexpr (K > 1) {
        if (t0 > 0 && t0 - (K - 1) < len) {
            frames<T, V, K - 1>(a.x, a.x_batch, a.x_time, n, c, t0 - (K - 1), len, wide, have, out);
        } else if (t0 == 0 && a.initial != nullptr) {
            frames<T, V, K - 1>(a.initial, (long)(K - 1) * a.channels, a.channels, n, c, 0, K - 1, wide, have, out);
        } else {
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) out[j][i] = 0.f;
        }
    }
}

template <int K, int V>
__device__ __forceinline__ void filters(const fsc_causal_conv_args& a, const Plan& p, int c, int have, float (&w)[K][V], float (&bias)[V]) {
    static_assert(V == 4, "K quadruples of weights");
    if (p.wide_weights && have == V) {
        float flat[V * K];
        const float* from = a.weight + (long)c * K;
#pragma unroll
        for (int q = 0; q < K; ++q) {
            const fsc::Pack<float, 4> v = fsc::load_pack<float, 4>(from + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) flat[4 * q + i] = v.v[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][i] = flat[i * K + k];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][i] = i < have ? a.weight[(long)(c + i) * K + k] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = i < have && a.bias != nullptr ? a.bias[c + i] : 0.f;
}

template <typename T, int K, int V>
__global__ __launch_bounds__(kThreads, K <= 4 ? 4 : 3) void conv_fwd_kernel(fsc_causal_conv_args a, Plan p) {
    constexpr int U = 8;
    const int g = blockIdx.y * p.lanes + (threadIdx.x & (p.lanes - 1));
    const long row = (long)blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes;
    if (g >= p.groups || row >= p.rows) return;
    const int n = (int)(row / p.strips), s = (int)(row % p.strips), c = g * V;
    const int have = a.channels - c < V ? a.channels - c : V;
    const bool wide = p.wide;
    const int len = frames_of(a, n);
    if (s == 0 && a.final != nullptr) {
        for (int j = 0; j < K - 1; ++j) {
            float v[V];
            frame<T, V>(a, n, c, len - (K - 1) + j, len, wide, have, v);
            store_row<V>(reinterpret_cast<T*>(a.final) + ((long)n * (K - 1) + j) * a.channels + c, wide, have, v);
        }
    }
    float w[K][V], bias[V];
    filters<K, V>(a, p, c, have, w, bias);
    const int t0 = s * p.strip, t1 = t0 + p.strip < a.length ? t0 + p.strip : a.length;
    float x[K - 1 + U][V];
    window<T, K, V>(a, n, c, t0, len, wide, have, x);
    T* out = reinterpret_cast<T*>(a.y) + ((long)n * a.length + t0) * a.channels + c;
    for (int t = t0; t < t1; t += U) {
        if (t < len) frames<T, V, U>(a.x, a.x_batch, a.x_time, n, c, t, len, wide, have, x + K - 1);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float v = bias[i];
#pragma unroll
                for (int k = 0; k < K; ++k) v = fmaf(w[k][i], x[j + k][i], v);
                y[i] = a.silu ? v * sigmoid_fast(v) : v;
                y[i] = t + j < len ? y[i] : 0.f;
            }
            if (t + j < t1) store_row<V>(out + j * a.channels, wide, have, y);
            __builtin_amdgcn_sched_barrier(0);       // (else all the frames' sums are in registers at once: two waves fewer a SIMD)
        }
        out += (long)U * a.channels;
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) x[j][i] = x[U + j][i];
    }
}

// FINAL: a gradient of the kept frames arrives too (rare: its reads stay out of the other variant's loop).
template <typename T, int K, int V, bool FINAL>
__global__ __launch_bounds__(kThreads) void conv_bwd_kernel(fsc_causal_conv_args a, Plan p) {
    constexpr int U = K <= 4 ? 8 : 4;
    __shared__ float red[kThreads][V];
    const int lane = threadIdx.x & (p.lanes - 1), sub = threadIdx.x / p.lanes, subs = kThreads / p.lanes;
    const int g = blockIdx.y * p.lanes + lane, c = g * V;
    const bool mine = g < p.groups;
    const int have = !mine ? 0 : a.channels - c < V ? a.channels - c : V;
    const bool wide = p.wide && mine;
    float w[K][V], bias[V], dw[K][V], db[V];
    filters<K, V>(a, p, mine ? c : 0, have, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
    }
    for (long row = (long)blockIdx.x * subs + sub; mine && row < p.rows; row += (long)gridDim.x * subs) {
        const int n = (int)(row / p.strips), s = (int)(row % p.strips);
        const int len = frames_of(a, n);
        const int t0 = s * p.strip, t1 = t0 + p.strip < a.length ? t0 + p.strip : a.length;
        // (frames past the strip are summed by the next one, and none behind the end: 0 times a frame that is not finite is not 0)
        const int counted = a.dy == nullptr ? t0 : t1 < len ? t1 : len;
        float x[K - 1 + U][V], dp[K - 1 + U][V];
        window<T, K, V>(a, n, c, t0, len, wide, have, x);
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) dp[j][i] = 0.f;
        // Frame t yields d pre[t]; with it frame t - (K - 1) has its gradient.  The next U frames are on their way while these are worked on: where
        // there are two waves a SIMD, little else covers the loads (4 x 8191 x 2048 in bf16, forward and backward: 8 taps 185 us, 278 with the loads at
        // the start of their turn, which also keeps more registers; 5 taps 147 for 160; up to 4 taps as long either way)
        fsc::Raw<T, V> raw_x[U] = {}, raw_dy[U] = {};
        auto ahead = [&](int t) {
            if (t < len) {       // (behind the end the last values stay, or the zeros: what comes of them is left out)
                fetch<T, V, U>(a.x, a.x_batch, a.x_time, n, c, t, len, wide, have, raw_x);
                if (a.dy != nullptr) fetch<T, V, U>(a.dy, a.dy_batch, a.dy_time, n, c, t, len, wide, have, raw_dy);
            }
        };
        ahead(t0);
        T* out = reinterpret_cast<T*>(a.dx) + ((long)n * a.length + t0 - (K - 1)) * a.channels + c;      // of frame t - (K - 1)
        for (int t = t0; t < t1 + K - 1; t += U) {
            float dy[U][V];
            convert<T, V, U>(raw_x, x + K - 1);
            convert<T, V, U>(raw_dy, dy);
            if (t + U < t1 + K - 1) ahead(t + U);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const bool there = t + j < len && a.dy != nullptr;
                float grad[V];
#pragma unroll
                for (int i = 0; i < V; ++i) grad[i] = dy[j][i];
                if (a.silu) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float v = bias[i];
#pragma unroll
                        for (int k = 0; k < K; ++k) v = fmaf(w[k][i], x[j + k][i], v);
                        const float sig = sigmoid_fast(v);
                        grad[i] *= sig * fmaf(v, 1.0f - sig, 1.0f);
                    }
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    fsc::pin(grad[i]);               // (computed by every lane: a branch around it would cost more)
                    grad[i] = there ? grad[i] : 0.f;
                    dp[K - 1 + j][i] = grad[i];
                }
                if (t + j < counted) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        db[i] += grad[i];
                        fsc::pin(db[i]);
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            dw[k][i] = fmaf(grad[i], x[j + k][i], dw[k][i]);
                            fsc::pin(dw[k][i]);
                        }
                    }
                }
                const int at = t + j - (K - 1);
                float dx[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float v = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k) v = fmaf(w[K - 1 - k][i], dp[j + k][i], v);
                    fsc::pin(v);
                    dx[i] = at < len ? v : 0.f;
                }
                if constexpr (FINAL) {
                    const int f = at - len + K - 1;                    // among the kept frames
                    if (f >= 0 && f < K - 1 && at < t1 && (at >= t0 || s == 0)) {
                        float more[V];
                        load_row<V>(reinterpret_cast<const T*>(a.dfinal) + ((long)n * (K - 1) + f) * a.channels + c, wide, have, more);
#pragma unroll
                        for (int i = 0; i < V; ++i) dx[i] += more[i];
                    }
                }
                if (j == U - 1) {                    // (in front of this turn's last store: backward of 4 taps 90 us for 92)
#pragma unroll
                    for (int q = 0; q < U; ++q) {
                        raw_x[q].arrived();
                        raw_dy[q].arrived();
                    }
                }
                if (at >= t0 && at < t1) store_row<V>(out + j * a.channels, wide, have, dx);
                else if (at < 0 && at >= 1 - K && a.dinitial != nullptr)
                    store_row<V>(reinterpret_cast<T*>(a.dinitial) + ((long)n * (K - 1) + K - 1 + at) * a.channels + c, wide, have, dx);
                __builtin_amdgcn_sched_barrier(0);
            }
            out += (long)U * a.channels;
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[j][i] = x[U + j][i];
                    dp[j][i] = dp[U + j][i];
                }
        }
    }
    // partial sums of the block: workspace[block][K + 1][groups * V]
    float* part = reinterpret_cast<float*>(a.workspace) + (long)blockIdx.x * (K + 1) * p.groups * V;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) red[threadIdx.x][i] = k < K ? dw[k < K ? k : 0][i] : db[i];
        __syncthreads();
        if (sub == 0 && mine) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = red[lane][i];
            for (int q = 1; q < subs; ++q)
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] += red[q * p.lanes + lane][i];
#pragma unroll
            for (int i = 0; i < V; ++i) part[(long)k * p.groups * V + c + i] = v[i];
        }
    }
}

// dweight[c, k] / dbias[c]: the blocks' partial sums, 32 columns x 8 interleaved shares of the blocks
__global__ __launch_bounds__(kThreads) void conv_bwd_finish_kernel(const float* __restrict__ part, int parts, int channels, int padded, int taps,
                                                                   float* __restrict__ dweight, float* __restrict__ dbias) {
    __shared__ float red[8][32];
    const int lane = threadIdx.x & 31, share = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
    const long columns = (long)(taps + 1) * padded;
    float v[4] = {};
    if (column < columns) {
        int q = share;
        for (; q + 24 < parts; q += 32)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[(q + 8 * i) * columns + column];
        for (; q < parts; q += 8) v[0] += part[q * columns + column];
    }
    red[share][lane] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (share != 0 || column >= columns) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[i][lane];
    const int k = column / padded, c = column % padded;
    if (c >= channels) return;
    if (k < taps) dweight[(long)c * taps + k] = sum;
    else if (dbias != nullptr) dbias[c] = sum;
}

// One frame: a thread reads its window, computes, and writes the window one frame on.
template <typename T, int K, int V>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(fsc_causal_conv_args a, Plan p) {
    const int g = blockIdx.y * p.lanes + (threadIdx.x & (p.lanes - 1));
    const long n = (long)blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes;
    if (g >= p.groups || n >= a.batch) return;
    const int c = g * V;
    const int have = a.channels - c < V ? a.channels - c : V;
    const bool wide = p.wide;
    T* window = reinterpret_cast<T*>(const_cast<void*>(a.initial)) + n * (K - 1) * a.channels + c;
    float x[K][V], w[K][V], bias[V], y[V];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load_row<V>(window + (long)k * a.channels, wide, have, x[k]);
    load_row<V>(reinterpret_cast<const T*>(a.x) + n * a.x_batch + c, wide, have, x[K - 1]);
    filters<K, V>(a, p, c, have, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store_row<V>(window + (long)k * a.channels, wide, have, x[k + 1]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float v = bias[i];
#pragma unroll
        for (int k = 0; k < K; ++k) v = fmaf(w[k][i], x[k][i], v);
        y[i] = a.silu ? v * sigmoid_fast(v) : v;
    }
    store_row<V>(reinterpret_cast<T*>(a.y) + n * a.channels + c, wide, have, y);
}

// Threads wanted in flight: two waves on each of the 1024 SIMDs.  Long strips read fewer frames twice (K - 1 at each end), short ones
// fill the card.
constexpr long kWanted = 2 * 1024 * 64;
constexpr long kMostBlocks = 1L << 24;       // of one launch: 2^32 threads and more are refused

Plan plan(const fsc_causal_conv_args& a) {
    constexpr int v = kV;
    Plan p{};
    p.groups = fsc::ceil_div(a.channels, v);
    const long frames = (long)a.batch * a.length * p.groups;
    long strip = frames / kWanted / 8 * 8;
    const long least = 8, most = 64;
    strip = strip < least ? least : strip > most ? most : strip;
    p.strip = (int)strip;
    p.strips = a.length > 0 ? fsc::ceil_div(a.length, strip) : 1;
    p.lanes = 1;
    while (p.lanes < 64 && p.lanes < p.groups) p.lanes *= 2;
    p.rows = a.batch * p.strips;
    const size_t unit = v * fsc::dtype_bytes(a.dtype);
    p.wide = a.channels % v == 0 && a.x_batch % v == 0 && a.x_time % v == 0 && a.dy_batch % v == 0 && a.dy_time % v == 0 &&
             fsc::aligned(a.x, unit) && fsc::aligned(a.initial, unit) && fsc::aligned(a.y, unit) && fsc::aligned(a.final, unit) &&
             fsc::aligned(a.dy, unit) && fsc::aligned(a.dfinal, unit) && fsc::aligned(a.dx, unit) && fsc::aligned(a.dinitial, unit);
    p.wide_weights = fsc::aligned(a.weight, 16);
    return p;
}

// Blocks along the rows of the backward pass: two blocks a CU, as many as the registers let in (4 x 8191 x 2048 in bf16: 90 us; four 97, one 121),
// and no more partial sums than that.
int bwd_parts(const Plan& p) {
    if (p.groups == 0) return 1;                 // no channels: nothing is launched
    const int across = fsc::ceil_div(p.groups, p.lanes), need = fsc::ceil_div(p.rows, kThreads / p.lanes);
    const int most = fsc::ceil_div(512, across);
    return need < most ? (need > 0 ? need : 1) : most;
}

const char* bad(const fsc_causal_conv_args* a) {
    if (a == nullptr) return "null arguments";
    if (!fsc::dtype_ok(a->dtype)) return "unknown dtype";
    if (a->taps < 1 || a->taps > 8) return "1 to 8 taps";
    if (a->batch < 0 || a->length < 0 || a->channels < 0) return "negative size";
    if ((long)a->batch * (a->length / 8 + 1) > 0x7FFFFFFFL) return "batch * length is too large";
    if (a->channels > (1 << 23)) return "more than 2^23 channels";
    const long strides[] = {a->x_time, a->dy_time};
    for (const long s : strides)
        if (s < 0 || s > (1L << 26)) return "negative time strides or above 2^26";
    if (a->channels > 0 && a->weight == nullptr) return "null weight";
    return nullptr;
}

template <typename Launch>
void with_taps(int taps, Launch launch) {
    switch (taps) {
        case 1: launch(std::integral_constant<int, 1>()); break;
        case 2: launch(std::integral_constant<int, 2>()); break;
        case 3: launch(std::integral_constant<int, 3>()); break;
        case 4: launch(std::integral_constant<int, 4>()); break;
        case 5: launch(std::integral_constant<int, 5>()); break;
        case 6: launch(std::integral_constant<int, 6>()); break;
        case 7: launch(std::integral_constant<int, 7>()); break;
        default: launch(std::integral_constant<int, 8>()); break;
    }
}

}  // namespace

extern "C" {

int fsc_causal_conv_fwd(const fsc_causal_conv_args* args_host, fsc_stream_t stream) {
    const char* why = bad(args_host);
    FSC_CHECK_ARG(why == nullptr, "fsc_causal_conv_fwd: %s", why);
    const fsc_causal_conv_args& a = *args_host;
    if (a.batch == 0 || a.channels == 0 || (a.length == 0 && a.final == nullptr)) return 0;
    FSC_CHECK_ARG(a.length == 0 || (a.x && a.y), "fsc_causal_conv_fwd: null x or y");
    const Plan p = plan(a);
    const dim3 grid(fsc::ceil_div(p.rows, kThreads / p.lanes), fsc::ceil_div(p.groups, p.lanes));
    FSC_CHECK_ARG((long)grid.x * grid.y < kMostBlocks, "fsc_causal_conv_fwd: batch * length * channels is too large");
    auto typed = [&](auto type) {
        using T = decltype(type);
        with_taps(a.taps, [&](auto taps) {
            hipLaunchKernelGGL((conv_fwd_kernel<T, decltype(taps)::value, kV>), grid, dim3(kThreads), 0, fsc::as_stream(stream), a, p);
        });
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_causal_conv_fwd");
    return 0;
}

size_t fsc_causal_conv_bwd_workspace_bytes(const fsc_causal_conv_args* args_host) {
    if (bad(args_host) != nullptr) return 0;
    const fsc_causal_conv_args& a = *args_host;
    const Plan p = plan(a);
    return sizeof(float) * (size_t)bwd_parts(p) * (a.taps + 1) * p.groups * kV;
}

int fsc_causal_conv_bwd(const fsc_causal_conv_args* args_host, fsc_stream_t stream) {
    const char* why = bad(args_host);
    FSC_CHECK_ARG(why == nullptr, "fsc_causal_conv_bwd: %s", why);
    const fsc_causal_conv_args& a = *args_host;
    if (a.channels == 0) return 0;
    FSC_CHECK_ARG(a.dweight && a.workspace, "fsc_causal_conv_bwd: null dweight or workspace");
    FSC_CHECK_ARG(a.batch == 0 || a.length == 0 || (a.x && a.dx), "fsc_causal_conv_bwd: null x or dx");
    const Plan p = plan(a);
    const int parts = bwd_parts(p);
    auto typed = [&](auto type) {
        using T = decltype(type);
        const dim3 grid(parts, fsc::ceil_div(p.groups, p.lanes));
        with_taps(a.taps, [&](auto taps) {
            if (a.dfinal != nullptr) hipLaunchKernelGGL((conv_bwd_kernel<T, decltype(taps)::value, kV, true>), grid, dim3(kThreads), 0, fsc::as_stream(stream), a, p);
            else hipLaunchKernelGGL((conv_bwd_kernel<T, decltype(taps)::value, kV, false>), grid, dim3(kThreads), 0, fsc::as_stream(stream), a, p);
        });
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_causal_conv_bwd");
    const int padded = p.groups * kV;
    hipLaunchKernelGGL(conv_bwd_finish_kernel, dim3(fsc::ceil_div((long)(a.taps + 1) * padded, 32)), dim3(kThreads), 0,
                       fsc::as_stream(stream), reinterpret_cast<const float*>(a.workspace), parts, a.channels, padded, a.taps, a.dweight,
                       a.dbias);
    FSC_LAUNCH_CHECK("fsc_causal_conv_bwd (sums)");
    return 0;
}

int fsc_causal_conv_step(const fsc_causal_conv_args* args_host, fsc_stream_t stream) {
    const char* why = bad(args_host);
    FSC_CHECK_ARG(why == nullptr, "fsc_causal_conv_step: %s", why);
    const fsc_causal_conv_args& a = *args_host;
    if (a.batch == 0 || a.channels == 0) return 0;
    FSC_CHECK_ARG(a.x && a.y && (a.taps == 1 || a.initial), "fsc_causal_conv_step: null x, y or window");
    const Plan p = plan(a);
    const dim3 grid(fsc::ceil_div(a.batch, kThreads / p.lanes), fsc::ceil_div(p.groups, p.lanes));
    FSC_CHECK_ARG((long)grid.x * grid.y < kMostBlocks, "fsc_causal_conv_step: batch * channels is too large");
    auto typed = [&](auto type) {
        using T = decltype(type);
        with_taps(a.taps, [&](auto taps) {
            hipLaunchKernelGGL((conv_step_kernel<T, decltype(taps)::value, kV>), grid, dim3(kThreads), 0, fsc::as_stream(stream), a, p);
        });
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_causal_conv_step");
    return 0;
}

}  // extern "C"
