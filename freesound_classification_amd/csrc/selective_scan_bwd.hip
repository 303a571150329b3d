// Selective scan, backward (scan.h says how the work is split).  With dyy = dy silu(z), e_t = exp(delta_t A) and G_t = dL/dh_t:
//   G_t = C_t dyy_t + e_{t+1} G_{t+1}        dC_t = sum_d h_t dyy_t           dB_t = sum_d G_t delta_t u_t
//   du = delta sum_s G B + D dyy              d delta = sum_s G (A e h_{t-1} + u B)      dA = sum_{n,t} G delta e h_{t-1}
//   dz = dy (C.h + D u) silu'(z)              ddt = d delta sigmoid(dt + bias)           dD = sum dyy u,  dh_{-1} = e_0 G_0
// A tile of 16 frames starts from the state that the forward kept there: e and h_{t-1} of its frames are formed once, forwards, and stay in
// registers (2 x 16 x NS) for the way back, so an element costs one exponential and some fifteen multiply-adds.
// The sums over the channels (dB, dC) take the wave's channels by lane exchanges that halve the number of values at each turn, the
// four waves through LDS, the blocks in a second launch; dA, dD and d dt_bias are summed in registers over time and by the second launch
// over sequences and segments.  No atomics: equal inputs give equal bits.
#include <type_traits>

#include "scan.h"

namespace {

using namespace fsc;

// The workspace: segments' ends and their deltas (one segment: none), partial sums over channel blocks and over (sequence, segment).
struct Carve {
    size_t ends, end_deltas, rows, sums, bytes;      // offsets in floats
    Carve(const fsc_selective_scan_args& a, const ScanPlan& p) {
        const size_t many = (size_t)a.batch * p.segments, channels = p.padded_channels(), sp = p.padded_states();
        ends = 0;
        end_deltas = p.segments > 1 ? many * channels * sp : 0;
        rows = end_deltas + (p.segments > 1 ? many * channels : 0);
        sums = rows + (size_t)a.batch * p.blocks * p.tiles * kTile * 2 * sp;
        bytes = sizeof(float) * (sums + many * channels * (sp + 2));
    }
};

// A segment's gradient of the state in front of it, from zero behind it: G as in the main pass, nothing else.  (PARTIAL: as in the forward; 8 x 2048 x
// 1024, a training step: 22 states 641 us, 24 states 590.)
template <typename T, int L, int NS, bool PARTIAL>
__global__ __launch_bounds__(256) void scan_bwd_ends_kernel(fsc_selective_scan_args a, ScanPlan p, float* ends, float* end_deltas) {
    using Place = ScanPlace<L, NS>;
    constexpr int CB = Place::CB, E = Place::E, SP = Place::SP;
    __shared__ __align__(16) float s_delta[CB + 1][kPad], s_dyy[CB + 1][kPad], s_c[kTile][SP + NS];
    int len;
    const Place w(a, p, len);
    if (w.segment == 0) return;
    scan_zero_row(s_delta);
    scan_zero_row(s_dyy);
    scan_zero_columns<NS>(s_c);
    float rate[NS], e[NS] = {}, sum = 0.f;
    scan_rates(a, w, rate);
    float bias[E];
    scan_param(w, a.dt_bias, bias);
#pragma unroll
    for (int i = 0; i < E; ++i) bias[i] *= kLog2e;
    const ScanFrames<T, L, NS> dt_rows(w, a.dt, a.dt_batch, a.dt_time), z_rows(w, a.z, a.z_batch, a.z_time), dy_rows(w, a.dy, a.dy_batch, a.dy_time);
    ScanRows<T, L, NS> c_rows(w, a.c, a.c_batch, a.c_time, a.c_group, a.states);
    Raw<T, E> dt_next, z_next, dy_next;
    auto fetch = [&](int tile) {
        dt_rows.fetch(w, tile, len, dt_next);
        if (a.dy != nullptr) dy_rows.fetch(w, tile, len, dy_next);
        if (a.z != nullptr) z_rows.fetch(w, tile, len, z_next);
        c_rows.fetch(w, tile, len);
    };
    if (w.first < w.work_end) fetch(w.work_end - 1);
    pin_all(bias);
    for (int tile = w.work_end - 1; tile >= w.first; --tile) {
        const int t = tile * kTile + w.te;
        __syncthreads();
        float raw[E], delta[E], dyy[E];
        time_steps(dt_next, bias, a.softplus, t < len, raw, delta);
#pragma unroll
        for (int i = 0; i < E; ++i) dyy[i] = a.dy != nullptr ? dy_next[i] : 0.f;
        if (a.z != nullptr) {
#pragma unroll
            for (int i = 0; i < E; ++i) dyy[i] *= z_next[i] * sigmoid_fast(z_next[i]);
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            s_delta[w.lds_row(i)][w.te] = delta[i];
            s_dyy[w.lds_row(i)][w.te] = t < len ? dyy[i] : 0.f;
        }
        c_rows.stage(w, s_c, tile, len, a.states, 1.0f);
        __syncthreads();
        if (tile > w.first) fetch(tile - 1);
#pragma unroll
        for (int q = kTile / 4 - 1; q >= 0; --q) {
            float dl[4], dyy[4];
            load_row<4>(&s_delta[w.row][4 * q], true, 4, dl);
            load_row<4>(&s_dyy[w.row][4 * q], true, 4, dyy);
#pragma unroll
            for (int j = 3; j >= 0; --j) {
                float cc[NS];
                load_row<NS>(&s_c[4 * q + j][w.col], true, NS, cc);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    e[i] = __builtin_amdgcn_exp2f(dl[j] * rate[i]) * fmaf(cc[i], dyy[j], e[i]);
                    e[i] = w.template has<PARTIAL>(i, a.states) ? e[i] : 0.f;
                }
                sum += dl[j];
            }
        }
    }
    store_row<NS>(ends + w.end(p, w.segment), true, NS, e);
    if (w.sg == 0) end_deltas[w.end_delta(p, w.segment)] = sum;
}

// The sums of v[0 .. 2 NS) over the channels of a wave (lanes that differ above the L lanes of one channel).  On return v[0 .. kept)
// hold the sums of the values first .. first + kept - 1.
template <int L, int NS>
__device__ __forceinline__ void channel_sums(float (&v)[2 * NS]) {
    constexpr int N = 2 * NS;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        swap32(v[i], v[i + N / 2]);
        v[i] += v[i + N / 2];
    }
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            swap16(v[i], v[i + N / 4]);
            v[i] += v[i + N / 4];
        }
    } else {
        float other = v[0];
        swap16(v[0], other);
        v[0] += other;
    }
    constexpr int kept = N >= 4 ? N / 4 : 1;
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        if constexpr (L <= 8) v[i] += dpp<0x128>(v[i]);
        if constexpr (L <= 4) v[i] += dpp<0x124>(v[i]);
        pin(v[i]);
    }
}

template <typename T, int L, int NS, bool PARTIAL>
__global__ __launch_bounds__(256, 2) void scan_bwd_kernel(fsc_selective_scan_args a, ScanPlan p, Carve at) {
    using Place = ScanPlace<L, NS>;
    constexpr int CB = Place::CB, E = Place::E, SP = Place::SP;
    __shared__ __align__(16) float s_delta[CB + 1][kPad], s_du[CB + 1][kPad], s_dyy[CB + 1][kPad], s_yh[CB][kPad], s_gb[CB][kPad], s_ga[CB][kPad];
    __shared__ __align__(16) float s_sig[256][E], s_gz[256][E];       // a thread's own, out of its registers while it scans
    __shared__ __align__(16) float s_b[kTile][SP + NS], s_c[kTile][SP + NS];
    __shared__ __align__(16) float s_red[kTile][4][2][SP];
    float* ws = reinterpret_cast<float*>(a.workspace);
    int len;
    const Place w(a, p, len);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    scan_zero_row(s_delta);
    scan_zero_row(s_du);
    scan_zero_row(s_dyy);
    scan_zero_columns<NS>(s_b);
    scan_zero_columns<NS>(s_c);

    float rate[NS], e[NS], da[NS] = {};              // e: exp(delta_{t+1} A) G_{t+1}, what reaches h_t from behind
    scan_rates(a, w, rate);
    scan_state(a, w, a.dfinal, e);
#pragma unroll 4
    for (int q = p.segments - 1; q > w.segment; --q) {
        const float ds = ws[at.end_deltas + w.end_delta(p, q)];
        float more[NS];
        load_row<NS>(ws + at.ends + w.end(p, q), true, NS, more);
#pragma unroll
        for (int i = 0; i < NS; ++i) e[i] = scan_join(e[i], rate[i], ds, more[i]);
    }
    float bias[E], skip[E], dskip[E] = {}, dbias[E] = {};
    scan_param(w, a.dt_bias, bias);
    scan_param(w, a.d, skip);
#pragma unroll
    for (int i = 0; i < E; ++i) bias[i] *= kLog2e;
    const ScanFrames<T, L, NS> u_rows(w, a.u, a.u_batch, a.u_time), dt_rows(w, a.dt, a.dt_batch, a.dt_time), z_rows(w, a.z, a.z_batch, a.z_time),
        dy_rows(w, a.dy, a.dy_batch, a.dy_time);
    ScanRows<T, L, NS> b_rows(w, a.b, a.b_batch, a.b_time, a.b_group, a.states), c_rows(w, a.c, a.c_batch, a.c_time, a.c_group, a.states);
    Raw<T, E> u_next, dt_next, z_next, dy_next;
    Raw<float, NS> h_next;
    auto fetch = [&](int tile) {
        u_rows.fetch(w, tile, len, u_next);
        dt_rows.fetch(w, tile, len, dt_next);
        if (a.dy != nullptr) dy_rows.fetch(w, tile, len, dy_next);
        if (a.z != nullptr) z_rows.fetch(w, tile, len, z_next);
        b_rows.fetch(w, tile, len);
        c_rows.fetch(w, tile, len);
        h_next.wide(a.checkpoints + w.kept(p, tile));
    };
    for (int tile = w.zero_first; tile < w.zero_end; ++tile) {
        float zero[E] = {};
        if (tile * kTile + w.te < a.length) {
            store_row<E>(scan_out<T>(a, w, a.du, tile), w.whole, w.he, zero);
            store_row<E>(scan_out<T>(a, w, a.ddt, tile), w.whole, w.he, zero);
            if (a.z != nullptr) store_row<E>(scan_out<T>(a, w, a.dz, tile), w.whole, w.he, zero);
        }
        for (int j = threadIdx.x; j < kTile * 2 * SP; j += 256) ws[at.rows + w.rows(p, tile) + j] = 0.f;
    }
    if (w.first < w.work_end) fetch(w.work_end - 1);
    pin_all(e);
    pin_all(bias);
    pin_all(skip);
    for (int tile = w.work_end - 1; tile >= w.first; --tile) {
        const int t = tile * kTile + w.te, count = len - tile * kTile;
        const Raw<T, E> u_now = u_next;
        float raw[E], delta[E], dyy[E], sig[E], gz[E], h[NS], hp[kTile][NS], ex[kTile][NS];
        time_steps(dt_next, bias, a.softplus, t < len, raw, delta);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            dyy[i] = t < len && i < w.he && a.dy != nullptr ? dy_next[i] : 0.f;
            sig[i] = 1.0f;
            gz[i] = 0.f;
        }
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < E; ++i) sig[i] = sigmoid2(raw[i]);
        }
        if (a.z != nullptr) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float z = t < len ? z_next[i] : 0.f, s = sigmoid_fast(z), zs = z * s;
                gz[i] = dyy[i] * (fmaf(-zs, s, zs) + s);
                dyy[i] *= zs;
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            s_delta[w.lds_row(i)][w.te] = delta[i];
            // (a channel that does not exist must not enter the sums over channels)
            s_du[w.lds_row(i)][w.te] = t < len && i < w.he ? delta[i] * u_now[i] : 0.f;
            s_dyy[w.lds_row(i)][w.te] = dyy[i];
        }
        store_row<E>(s_sig[threadIdx.x], true, E, sig);
        store_row<E>(s_gz[threadIdx.x], true, E, gz);
        b_rows.stage(w, s_b, tile, len, a.states, kLn2);
        c_rows.stage(w, s_c, tile, len, a.states, 1.0f);
#pragma unroll
        for (int i = 0; i < NS; ++i) h[i] = h_next[i];
        __syncthreads();
        if (tile > w.first) fetch(tile - 1);
#pragma unroll
        for (int q = 0; q < kTile / 4; ++q) {
            float dl[4], du[4], y[4];
            load_row<4>(&s_delta[w.row][4 * q], true, 4, dl);
            load_row<4>(&s_du[w.row][4 * q], true, 4, du);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float b[NS], cc[NS], v = 0.f;
                load_row<NS>(&s_b[4 * q + j][w.col], true, NS, b);
                load_row<NS>(&s_c[4 * q + j][w.col], true, NS, cc);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const bool has = w.template has<PARTIAL>(i, a.states);
                    ex[4 * q + j][i] = has ? __builtin_amdgcn_exp2f(dl[j] * rate[i]) : 0.f;
                    hp[4 * q + j][i] = h[i];
                    h[i] = has ? fmaf(ex[4 * q + j][i], h[i], du[j] * b[i]) : 0.f;
                    v = fmaf(cc[i], h[i], v);
                }
                y[j] = group_sum<L>(v);
            }
            if (L == 4 || w.sg < 4) s_yh[w.ch][4 * q + (w.sg & 3)] = pick4(y[0], y[1], y[2], y[3], w.sg);
            __builtin_amdgcn_sched_barrier(0);        // (else the reads of later frames are hoisted until registers spill)
        }
#pragma unroll
        for (int q = kTile / 4 - 1; q >= 0; --q) {
            float dl[4], du[4], dyy4[4], gb4[4] = {}, ga4[4] = {};
            load_row<4>(&s_delta[w.row][4 * q], true, 4, dl);
            load_row<4>(&s_du[w.row][4 * q], true, 4, du);
            load_row<4>(&s_dyy[w.row][4 * q], true, 4, dyy4);
#pragma unroll
            for (int j = 3; j >= 0; --j) {
                const int k = 4 * q + j;
                if (k >= count) continue;             // (a frame behind the end: its delta of 0 would make NaN of an infinite state)
                float b[NS], cc[NS], v[2 * NS], gb = 0.f, ga = 0.f;
                load_row<NS>(&s_b[k][w.col], true, NS, b);
                load_row<NS>(&s_c[k][w.col], true, NS, cc);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const float g = w.template has<PARTIAL>(i, a.states) ? fmaf(cc[i], dyy4[j], e[i]) : 0.f;
                    v[i] = g * du[j];
                    v[NS + i] = h[i] * dyy4[j];
                    gb = fmaf(g, b[i], gb);
                    e[i] = ex[k][i] * g;
                    const float gx = e[i] * hp[k][i];
                    da[i] = fmaf(gx, dl[j], da[i]);
                    ga = fmaf(gx, rate[i], ga);
                    h[i] = hp[k][i];
                }
                gb4[j] = group_sum<L>(gb);
                ga4[j] = group_sum<L>(ga);
                pin(gb4[j]);
                pin(ga4[j]);
#pragma unroll
                for (int i = 0; i < NS; ++i) pin(da[i]);
                channel_sums<L, NS>(v);
                // upper half: dC, lower half: dB; even rows of 16 lanes: the first half of the states, odd rows: the second
                constexpr int kept = NS >= 2 ? NS / 2 : 1;
                const int half = lane >> 5, row = (lane >> 4) & 1;
                if ((lane & 15) < L && (NS >= 2 || row == 0)) {
                    const int s = w.sg * NS + (NS >= 2 ? row * kept : 0);
#pragma unroll
                    for (int i = 0; i < kept; ++i) s_red[k][wave][half][s + i] = v[i];
                }
            }
            if (L == 4 || w.sg < 4) {
                s_gb[w.ch][4 * q + (w.sg & 3)] = pick4(gb4[0], gb4[1], gb4[2], gb4[3], w.sg);
                s_ga[w.ch][4 * q + (w.sg & 3)] = pick4(ga4[0], ga4[1], ga4[2], ga4[3], w.sg);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        for (int j = threadIdx.x; j < kTile * 2 * SP; j += 256) {
            const int k = j / (2 * SP), rest = j % (2 * SP);
            const float* r = &s_red[k][0][0][rest];
            ws[at.rows + w.rows(p, tile) + j] = k < count ? (r[0] + r[2 * SP]) + (r[4 * SP] + r[6 * SP]) : 0.f;
        }
        if (t < a.length) {
            float du_out[E], ddt_out[E], dz_out[E];
            load_row<E>(s_sig[threadIdx.x], true, E, sig);
            load_row<E>(s_gz[threadIdx.x], true, E, gz);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int r = w.lds_row(i);
                const float u = t < len ? u_now[i] : 0.f, gb = s_gb[r][w.te], ga = s_ga[r][w.te], dyy = s_dyy[r][w.te];
                du_out[i] = fmaf(s_delta[r][w.te], gb, skip[i] * dyy);          // (B was staged times ln 2, delta over it)
                ddt_out[i] = fmaf(u * kLog2e, gb, ga) * sig[i];
                dz_out[i] = gz[i] * fmaf(skip[i], u, s_yh[r][w.te]);
                if (t >= len) du_out[i] = ddt_out[i] = dz_out[i] = 0.f;
                dskip[i] = fmaf(dyy, u, dskip[i]);
                dbias[i] += ddt_out[i];
            }
            store_row<E>(scan_out<T>(a, w, a.du, tile), w.whole, w.he, du_out);
            store_row<E>(scan_out<T>(a, w, a.ddt, tile), w.whole, w.he, ddt_out);
            if (a.z != nullptr) store_row<E>(scan_out<T>(a, w, a.dz, tile), w.whole, w.he, dz_out);
        }
        __syncthreads();
    }
    if (a.dinitial != nullptr && w.segment == 0 && w.real) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int s = w.sg * NS + i;
            if (s < a.states) a.dinitial[((long)w.n * a.channels + w.channel) * a.states + s] = e[i];
        }
    }
    // this (sequence, segment)'s share of the parameters' gradients: [dA: channels x SP | dD | d dt_bias]
    const long channels = p.padded_channels();
    float* mine = ws + at.sums + ((long)w.n * p.segments + w.segment) * channels * (SP + 2);
    store_row<NS>(mine + ((long)w.block * 256 + threadIdx.x) * NS, true, NS, da);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        s_dyy[w.lds_row(i)][w.te] = dskip[i];
        s_yh[w.lds_row(i)][w.te] = dbias[i];
    }
    __syncthreads();
    if (threadIdx.x < CB) {
        float sd = 0.f, sb = 0.f;
#pragma unroll
        for (int k = 0; k < kTile; ++k) {
            sd += s_dyy[threadIdx.x][k];
            sb += s_yh[threadIdx.x][k];
        }
        mine[channels * SP + w.block * CB + threadIdx.x] = sd;
        mine[channels * (SP + 1) + w.block * CB + threadIdx.x] = sb;
    }
}

// Joins the partial sums: the first `row_blocks` workgroups dB / dC over the channel blocks of a group, the others (32 columns x 8
// interleaved shares) the parameters' over sequences and segments.
template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_finish_kernel(fsc_selective_scan_args a, ScanPlan p, Carve at, long row_blocks) {
    const float* ws = reinterpret_cast<const float*>(a.workspace);
    const int sp = p.padded_states();
    if (blockIdx.x < row_blocks) {
        const long i = (long)blockIdx.x * 256 + threadIdx.x;         // (sequence, frame, group, state)
        if (i >= (long)a.batch * a.length * a.groups * a.states) return;
        const int s = (int)(i % a.states);
        const long r = i / a.states;
        const int g = (int)(r % a.groups);
        const long f = r / a.groups;
        const int n = (int)(f / a.length), t = (int)(f % a.length);
        const long stride = (long)p.tiles * kTile * 2 * sp;
        const float* from = ws + at.rows + ((long)n * p.blocks + (long)g * p.group_blocks) * stride + (long)t * 2 * sp + s;
        float db = 0.f, dc = 0.f;
        for (int q = 0; q < p.group_blocks; ++q) {
            db += from[q * stride];
            dc += from[q * stride + sp];
        }
        reinterpret_cast<T*>(a.db)[i] = (T)(db * kLn2);            // (summed with delta u over ln 2)
        reinterpret_cast<T*>(a.dc)[i] = (T)dc;
        return;
    }
    __shared__ float red[8][32];
    const long channels = p.padded_channels(), columns = channels * (sp + 2);
    const int k = threadIdx.x & 31, share = threadIdx.x >> 5, count = a.batch * p.segments;
    const long column = ((long)blockIdx.x - row_blocks) * 32 + k;
    float v[4] = {};
    if (column < columns) {
        const float* from = ws + at.sums + column;
        int q = share;
        for (; q + 24 < count; q += 32)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += from[(q + 8 * i) * columns];
        for (; q < count; q += 8) v[0] += from[q * columns];
    }
    red[share][k] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (share != 0 || column >= columns) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[i][k];
    const int cb = p.channels_block;
    const long slot = column < channels * sp ? column / sp : (column - channels * sp) % channels;      // padded channel
    const int block = (int)(slot / cb), in_group = (block % p.group_blocks) * cb + channel_of((int)(slot % cb), kTile / p.lanes);
    if (in_group >= p.group_channels) return;
    const long c = (long)(block / p.group_blocks) * p.group_channels + in_group;
    if (column < channels * sp) {
        const int s = (int)(column % sp);
        if (s < a.states) a.da_log[c * a.states + s] = rate_of(a.a_log[c * a.states + s]) * kLn2 * sum;         // dA / d a_log = A; delta over ln 2
    } else if (column < channels * (sp + 1)) {
        if (a.dd != nullptr) a.dd[c] = sum;
    } else if (a.ddt_bias != nullptr) {
        a.ddt_bias[c] = sum;
    }
}

}  // namespace

extern "C" {

size_t fsc_selective_scan_workspace_bytes(const fsc_selective_scan_args* args_host, int backward) {
    if (scan_bad(args_host) != nullptr) return 0;
    const ScanPlan p = scan_plan(*args_host);
    const Carve at(*args_host, p);
    return backward ? at.bytes : sizeof(float) * at.rows;
}

int fsc_selective_scan_bwd(const fsc_selective_scan_args* args_host, fsc_stream_t stream) {
    const char* why = scan_bad(args_host);
    FSC_CHECK_ARG(why == nullptr, "fsc_selective_scan_bwd: %s", why);
    const fsc_selective_scan_args& a = *args_host;
    const ScanPlan p = scan_plan(a);
    const Carve at(a, p);
    FSC_CHECK_ARG(a.channels == 0 || (a.da_log && (a.workspace || at.bytes == 0)), "fsc_selective_scan_bwd: null da_log or workspace");
    FSC_CHECK_ARG(a.batch == 0 || a.length == 0 || (a.db && a.dc && (a.channels == 0 || (a.u && a.dt && a.b && a.c && a.checkpoints && a.du && a.ddt &&
                                                                                        (a.z == nullptr || a.dz)))),
                  "fsc_selective_scan_bwd: null input or gradient");
    float* ws = reinterpret_cast<float*>(a.workspace);
    const dim3 grid((unsigned)((long)a.batch * p.blocks * p.segments));
    const long rows = ((long)a.batch * a.length * a.groups * a.states + 255) / 256;
    const long columns = (p.padded_channels() * (p.padded_states() + 2) + 31) / 32;
    FSC_CHECK_ARG((long)a.batch * p.blocks * p.segments <= kMostBlocks && rows + columns <= kMostBlocks, "fsc_selective_scan_bwd: too large");
    if (rows + columns == 0) return 0;
    auto typed = [&](auto type) {
        using T = decltype(type);
        if (a.batch > 0 && a.channels > 0)               // (without channels db and dc are still there: sums over nothing)
            with_scan_shape(p, [&](auto lanes, auto per) {
                constexpr int L = decltype(lanes)::value, NS = decltype(per)::value;
                with_partial<NS>(a.states, [&](auto partial) {
                    constexpr bool PARTIAL = decltype(partial)::value;
                    if (p.segments > 1)
                        hipLaunchKernelGGL((scan_bwd_ends_kernel<T, L, NS, PARTIAL>), grid, dim3(256), 0, as_stream(stream), a, p, ws + at.ends,
                                           ws + at.end_deltas);
                    hipLaunchKernelGGL((scan_bwd_kernel<T, L, NS, PARTIAL>), grid, dim3(256), 0, as_stream(stream), a, p, at);
                });
            });
        hipLaunchKernelGGL((scan_bwd_finish_kernel<T>), dim3((unsigned)(rows + columns)), dim3(256), 0, as_stream(stream), a, p, at, rows);
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_selective_scan_bwd");
    return 0;
}

}  // extern "C"
