// Selective scan, forward and single frames (scan.h says how the work is split).
//   h_t = exp(delta_t A) h_{t-1} + delta_t u_t B_t,   y_t = (C_t . h_t + D u_t) silu(z_t)
#include <type_traits>

#include "scan.h"

namespace {

using namespace fsc;

// One launch for both passes.  ENDS: the segments' ends from zero (states and the sum of delta) into the workspace, nothing else.  PARTIAL: a lane has
// fewer states than its NS; the others are kept at 0 by an instruction an element, since an infinite delta u times their B of 0 would be NaN, which the
// sum over the states would carry into y (2 x 16384 x 2048, 13 states: 495 us, 447 without; lanes without any state read zeros and cost nothing).
template <typename T, int L, int NS, bool ENDS, bool PARTIAL>
__global__ __launch_bounds__(256) void scan_fwd_kernel(fsc_selective_scan_args a, ScanPlan p, float* ends, float* end_deltas) {
    using Place = ScanPlace<L, NS>;
    constexpr int CB = Place::CB, E = Place::E, SP = Place::SP;
    __shared__ __align__(16) float s_delta[CB + 1][kPad], s_du[CB + 1][kPad], s_y[ENDS ? 1 : CB][kPad];
    __shared__ __align__(16) float s_b[kTile][SP + NS], s_c[ENDS ? 1 : kTile][SP + NS];
    int len;
    const Place w(a, p, len);
    if (ENDS && w.segment == p.segments - 1) return;
    scan_zero_row(s_delta);
    scan_zero_row(s_du);
    scan_zero_columns<NS>(s_b);
    if constexpr (!ENDS) scan_zero_columns<NS>(s_c);

    float rate[NS], h[NS], sum = 0.f;
    scan_rates(a, w, rate);
    scan_state(a, w, ENDS ? nullptr : a.initial, h);
    if constexpr (!ENDS) {
#pragma unroll 4
        for (int q = 0; q < w.segment; ++q) {
            const float ds = end_deltas[w.end_delta(p, q)];
            float e[NS];
            load_row<NS>(ends + w.end(p, q), true, NS, e);
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = scan_join(h[i], rate[i], ds, e[i]);
        }
    }
    float bias[E], skip[E];
    scan_param(w, a.dt_bias, bias);
    scan_param(w, ENDS ? nullptr : a.d, skip);
#pragma unroll
    for (int i = 0; i < E; ++i) bias[i] *= kLog2e;
    const ScanFrames<T, L, NS> u_rows(w, a.u, a.u_batch, a.u_time), dt_rows(w, a.dt, a.dt_batch, a.dt_time), z_rows(w, a.z, a.z_batch, a.z_time);
    ScanRows<T, L, NS> b_rows(w, a.b, a.b_batch, a.b_time, a.b_group, a.states), c_rows(w, a.c, a.c_batch, a.c_time, a.c_group, a.states);
    Raw<T, E> u_next, dt_next, z_next;
    auto fetch = [&](int tile) {
        u_rows.fetch(w, tile, len, u_next);
        dt_rows.fetch(w, tile, len, dt_next);
        if (!ENDS && a.z != nullptr) z_rows.fetch(w, tile, len, z_next);
        b_rows.fetch(w, tile, len);
        if (!ENDS) c_rows.fetch(w, tile, len);
    };
    if (w.first < w.work_end) fetch(w.first);
    pin_all(h);
    pin_all(bias);
    pin_all(skip);
    for (int tile = w.first; tile < w.work_end; ++tile) {
        const int t = tile * kTile + w.te;
        float raw[E], delta[E];
        time_steps(dt_next, bias, a.softplus, t < len, raw, delta);
        const Raw<T, E> u_now = u_next, z_now = z_next;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            s_delta[w.lds_row(i)][w.te] = delta[i];
            s_du[w.lds_row(i)][w.te] = t < len ? delta[i] * u_now[i] : 0.f;
        }
        b_rows.stage(w, s_b, tile, len, a.states, kLn2);
        if constexpr (!ENDS) c_rows.stage(w, s_c, tile, len, a.states, 1.0f);
        __syncthreads();
        if (tile + 1 < w.work_end) fetch(tile + 1);
        if (!ENDS && a.checkpoints != nullptr) store_row<NS>(a.checkpoints + w.kept(p, tile), true, NS, h);
#pragma unroll
        for (int q = 0; q < kTile / 4; ++q) {
            float dl[4], du[4], y[4];
            load_row<4>(&s_delta[w.row][4 * q], true, 4, dl);
            load_row<4>(&s_du[w.row][4 * q], true, 4, du);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float b[NS], cc[NS];
                load_row<NS>(&s_b[4 * q + j][w.col], true, NS, b);
                if constexpr (!ENDS) load_row<NS>(&s_c[4 * q + j][w.col], true, NS, cc);
                float v = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    h[i] = fmaf(__builtin_amdgcn_exp2f(dl[j] * rate[i]), h[i], du[j] * b[i]);
                    h[i] = w.template has<PARTIAL>(i, a.states) ? h[i] : 0.f;
                    if constexpr (!ENDS) v = fmaf(cc[i], h[i], v);
                }
                if constexpr (ENDS) sum += dl[j];
                else y[j] = group_sum<L>(v);
            }
            if constexpr (!ENDS) {
                if (L == 4 || w.sg < 4) s_y[w.ch][4 * q + (w.sg & 3)] = pick4(y[0], y[1], y[2], y[3], w.sg);
            }
        }
        __syncthreads();
        if constexpr (!ENDS) {
            if (t < a.length) {
                float y[E];
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] = fmaf(skip[i], u_now[i], s_y[w.lds_row(i)][w.te]);
                if (a.z != nullptr) {
#pragma unroll
                    for (int i = 0; i < E; ++i) y[i] *= z_now[i] * sigmoid_fast(z_now[i]);
                }
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] = t < len ? y[i] : 0.f;
                store_row<E>(scan_out<T>(a, w, a.y, tile), w.whole, w.he, y);
            }
        }
    }
    if constexpr (ENDS) {
        store_row<NS>(ends + w.end(p, w.segment), true, NS, h);
        if (w.sg == 0) end_deltas[w.end_delta(p, w.segment)] = sum;
    } else {
        for (int tile = w.zero_first; tile < w.zero_end; ++tile) {
            float zero[E] = {};
            if (tile * kTile + w.te < a.length) store_row<E>(scan_out<T>(a, w, a.y, tile), w.whole, w.he, zero);
        }
        if (a.final != nullptr && w.segment == p.segments - 1 && w.real) {
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int s = w.sg * NS + i;
                if (s < a.states) a.final[((long)w.n * a.channels + w.channel) * a.states + s] = h[i];
            }
        }
    }
}

// One frame.  Bound: the state, read and written once, in 16-byte accesses; L lanes a channel as in the scan.  A workgroup takes R x CB
// channels of one sequence, each thread R of them with all their loads in flight and one read of B and C.  256 sequences x 2048 channels x 64 states:
// 58 us, 4.7 TB/s; one of 256 channels: 2.8 us.
template <typename T, int L, int NS, int R>
__global__ __launch_bounds__(256) void scan_step_kernel(fsc_selective_scan_args a, int group_channels, int group_blocks, int wide) {
    constexpr int CB = 256 / L;
    const int blocks = a.groups * group_blocks;
    const long n = blockIdx.x / blocks;
    const int block = blockIdx.x % blocks, group = block / group_blocks, first = (block % group_blocks) * (CB * R);
    const int sg = threadIdx.x % L, s0 = sg * NS;
    const int have = a.states - s0 < 0 ? 0 : a.states - s0 < NS ? a.states - s0 : NS;
    const bool go = wide && have == NS;
    float b[NS], cc[NS], h[R][NS], al[R][NS], u[R], dt[R], z[R];
    int c[R];
    bool real[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int in_group = first + r * CB + threadIdx.x / L;
        real[r] = in_group < group_channels;
        c[r] = group * group_channels + (real[r] ? in_group : 0);
        const float* state = a.final + (n * a.channels + c[r]) * a.states + s0;
        const float* rate = a.a_log + (long)c[r] * a.states + s0;
        if (go) {
            const Pack<float, NS> hv = load_pack<float, NS>(state), av = load_pack<float, NS>(rate);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                h[r][i] = hv.v[i];
                al[r][i] = av.v[i];
            }
        } else {
            load_row<NS>(state, false, have, h[r]);
            load_row<NS>(rate, false, have, al[r]);
        }
        u[r] = (float)reinterpret_cast<const T*>(a.u)[n * a.u_batch + c[r]];
        dt[r] = ((float)reinterpret_cast<const T*>(a.dt)[n * a.dt_batch + c[r]] + (a.dt_bias != nullptr ? a.dt_bias[c[r]] : 0.f)) * kLog2e;
        z[r] = a.z != nullptr ? (float)reinterpret_cast<const T*>(a.z)[n * a.z_batch + c[r]] : 0.f;
    }
    load_row<NS>(reinterpret_cast<const T*>(a.b) + n * a.b_batch + group * a.b_group + s0, false, have, b);
    load_row<NS>(reinterpret_cast<const T*>(a.c) + n * a.c_batch + group * a.c_group + s0, false, have, cc);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float delta = a.softplus ? softplus2(dt[r]) : dt[r];
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) al[r][i] = rate_of(al[r][i]);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            h[r][i] = fmaf(__builtin_amdgcn_exp2f(delta * al[r][i]), h[r][i], delta * kLn2 * u[r] * b[i]);
            if (i < have) v = fmaf(cc[i], h[r][i], v);
        }
        v = group_sum<L>(v);
        if (!real[r]) continue;
        store_row<NS>(a.final + (n * a.channels + c[r]) * a.states + s0, go, have, h[r]);
        if (sg == 0) {
            if (a.d != nullptr) v = fmaf(a.d[c[r]], u[r], v);
            if (a.z != nullptr) v *= z[r] * sigmoid_fast(z[r]);
            reinterpret_cast<T*>(a.y)[n * a.channels + c[r]] = (T)v;
        }
    }
}

}  // namespace

extern "C" {

size_t fsc_selective_scan_checkpoint_bytes(const fsc_selective_scan_args* args_host) {
    if (scan_bad(args_host) != nullptr) return 0;
    const ScanPlan p = scan_plan(*args_host);
    return sizeof(float) * (size_t)args_host->batch * p.tiles * p.padded_channels() * p.padded_states();
}

int fsc_selective_scan_fwd(const fsc_selective_scan_args* args_host, fsc_stream_t stream) {
    const char* why = scan_bad(args_host);
    FSC_CHECK_ARG(why == nullptr, "fsc_selective_scan_fwd: %s", why);
    const fsc_selective_scan_args& a = *args_host;
    if (a.batch == 0 || a.channels == 0 || (a.length == 0 && a.final == nullptr)) return 0;
    FSC_CHECK_ARG(a.length == 0 || (a.u && a.dt && a.b && a.c && a.y), "fsc_selective_scan_fwd: null u, dt, b, c or y");
    const ScanPlan p = scan_plan(a);
    FSC_CHECK_ARG(p.segments == 1 || a.workspace, "fsc_selective_scan_fwd: null workspace");
    FSC_CHECK_ARG((long)a.batch * p.blocks * p.segments <= kMostBlocks, "fsc_selective_scan_fwd: batch * channels is too large");
    float* ends = reinterpret_cast<float*>(a.workspace);
    float* end_deltas = ends == nullptr ? nullptr : ends + (size_t)a.batch * p.segments * p.padded_channels() * p.padded_states();
    const dim3 grid((unsigned)((long)a.batch * p.blocks * p.segments));
    auto typed = [&](auto type) {
        using T = decltype(type);
        with_scan_shape(p, [&](auto lanes, auto per) {
            constexpr int L = decltype(lanes)::value, NS = decltype(per)::value;
            with_partial<NS>(a.states, [&](auto partial) {
                constexpr bool PARTIAL = decltype(partial)::value;
                if (p.segments > 1)
                    hipLaunchKernelGGL((scan_fwd_kernel<T, L, NS, true, PARTIAL>), grid, dim3(256), 0, as_stream(stream), a, p, ends, end_deltas);
                hipLaunchKernelGGL((scan_fwd_kernel<T, L, NS, false, PARTIAL>), grid, dim3(256), 0, as_stream(stream), a, p, ends, end_deltas);
            });
        });
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_selective_scan_fwd");
    return 0;
}

int fsc_selective_scan_step(const fsc_selective_scan_args* args_host, fsc_stream_t stream) {
    const char* why = scan_bad(args_host);
    FSC_CHECK_ARG(why == nullptr, "fsc_selective_scan_step: %s", why);
    const fsc_selective_scan_args& a = *args_host;
    if (a.batch == 0 || a.channels == 0) return 0;
    FSC_CHECK_ARG(a.u && a.dt && a.b && a.c && a.y && a.final, "fsc_selective_scan_step: null u, dt, b, c, y or state");
    const ScanPlan p = scan_plan(a);
    const int wide = a.states % p.per_lane == 0 && aligned(a.final, 4 * p.per_lane) && aligned(a.a_log, 4 * p.per_lane);
    // four channels a thread where that still leaves two workgroups a CU, else one
    const long fours = (long)a.batch * a.groups * ceil_div(p.group_channels, 4 * p.channels_block);
    const int r = fours >= 512 ? 4 : 1, group_blocks = ceil_div(p.group_channels, r * p.channels_block);
    FSC_CHECK_ARG((long)a.batch * a.groups * group_blocks <= kMostBlocks, "fsc_selective_scan_step: batch * channels is too large");
    const dim3 grid((unsigned)((long)a.batch * a.groups * group_blocks));
    auto typed = [&](auto type) {
        using T = decltype(type);
        with_scan_shape(p, [&](auto lanes, auto per) {
            constexpr int L = decltype(lanes)::value, NS = decltype(per)::value;
            if (r == 4)
                hipLaunchKernelGGL((scan_step_kernel<T, L, NS, 4>), grid, dim3(256), 0, as_stream(stream), a, p.group_channels, group_blocks, wide);
            else
                hipLaunchKernelGGL((scan_step_kernel<T, L, NS, 1>), grid, dim3(256), 0, as_stream(stream), a, p.group_channels, group_blocks, wide);
        });
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_selective_scan_step");
    return 0;
}

}  // extern "C"
