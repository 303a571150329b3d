// Selective scan, forward and single frames (scan.h says how the work is split).
//   h_t = exp(delta_t A) h_{t-1} + delta_t u_t B_t,   y_t = (C_t . h_t + D u_t) silu(z_t)
#include <type_traits>

#include "scan.h"

namespace {

using namespace fsc;

// One launch for both passes.  ENDS: the segments' ends from zero (states and the sum of delta) into the workspace, nothing else.
template <typename T, int L, int NS, bool ENDS>
__global__ __launch_bounds__(256) void scan_fwd_kernel(fsc_selective_scan_args a, ScanPlan p, float* ends, float* end_deltas) {
    using Place = ScanPlace<L, NS>;
    constexpr int CB = Place::CB, E = Place::E, SP = Place::SP, ROWS = Place::ROWS;
    __shared__ __align__(16) float s_delta[CB][kPad], s_du[CB][kPad], s_y[ENDS ? 1 : CB][kPad];
    __shared__ __align__(16) float s_b[kTile][SP], s_c[ENDS ? 1 : kTile][SP];
    const Place w(a, p);
    if (ENDS && w.segment == p.segments - 1) return;
    const int len = scan_frames(a, w.n);
    const int first = w.segment * p.segment_tiles;
    const int last = first + p.segment_tiles < p.tiles ? first + p.segment_tiles : p.tiles;

    float a2[NS], h[NS], sum = 0.f;
    scan_rates(a, w, a2);
    scan_state(a, w, ENDS ? nullptr : a.initial, h);
    if constexpr (!ENDS) {
        for (int q = 0; q < w.segment; ++q) {
            const float ds = end_deltas[w.end_delta(p, q)];
            float e[NS];
            load_row<NS>(ends + w.end(p, q), true, NS, e);
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = fmaf(__builtin_amdgcn_exp2f(a2[i] * ds), h[i], e[i]);
        }
    }
    float bias[E], skip[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        bias[i] = a.dt_bias != nullptr && i < w.he ? a.dt_bias[w.c0 + w.ce + i] : 0.f;
        skip[i] = !ENDS && a.d != nullptr && i < w.he ? a.d[w.c0 + w.ce + i] : 0.f;
    }
    const bool wide = p.wide && w.he == E;
    const long c = w.c0 + w.ce;
    float u_next[E], dt_next[E], z_next[E], b_next[ROWS], c_next[ROWS];
    auto fetch = [&](int tile) {
        const int t = tile * kTile + w.te;
        const int he = t < len ? w.he : 0;
        const bool go = wide && t < len;
        load_row<E>(reinterpret_cast<const T*>(a.u) + w.n * a.u_batch + t * a.u_time + c, go, he, u_next);
        load_row<E>(reinterpret_cast<const T*>(a.dt) + w.n * a.dt_batch + t * a.dt_time + c, go, he, dt_next);
        if (!ENDS && a.z != nullptr) load_row<E>(reinterpret_cast<const T*>(a.z) + w.n * a.z_batch + t * a.z_time + c, go, he, z_next);
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const int tr = tile * kTile + w.bc_row(j), s = w.bc_state(j);
            const bool there = w.bc_mine(j) && tr < len && s < a.states;
            b_next[j] = there ? (float)reinterpret_cast<const T*>(a.b)[w.n * a.b_batch + tr * a.b_time + w.group * a.b_group + s] : 0.f;
            if (!ENDS)
                c_next[j] = there ? (float)reinterpret_cast<const T*>(a.c)[w.n * a.c_batch + tr * a.c_time + w.group * a.c_group + s] : 0.f;
        }
    };
    const int work_end = tiles_with(len) < last ? tiles_with(len) : last;      // tiles behind it hold no frame
    if (first < work_end) fetch(first);
    for (int tile = first; tile < work_end; ++tile) {
        const int t = tile * kTile + w.te;
        float u[E], z[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            u[i] = u_next[i];
            z[i] = ENDS ? 0.f : z_next[i];
            const float raw = dt_next[i] + bias[i];
            const float delta = t < len ? (a.softplus ? softplus_fast(raw) : raw) : 0.f;
            s_delta[w.ce + i][w.te] = delta;
            s_du[w.ce + i][w.te] = delta * u[i];
        }
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (w.bc_mine(j)) {
                s_b[w.bc_row(j)][w.bc_state(j)] = b_next[j];
                if (!ENDS) s_c[w.bc_row(j)][w.bc_state(j)] = c_next[j];
            }
        __syncthreads();
        if (tile + 1 < work_end) fetch(tile + 1);
        if (!ENDS && a.checkpoints != nullptr) store_row<NS>(a.checkpoints + w.kept(p, tile), true, NS, h);
#pragma unroll
        for (int q = 0; q < kTile / 4; ++q) {
            float dl[4], du[4], y[4];
            load_row<4>(&s_delta[w.ch][4 * q], true, 4, dl);
            load_row<4>(&s_du[w.ch][4 * q], true, 4, du);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float b[NS], cc[NS];
                load_row<NS>(&s_b[4 * q + j][w.sg * NS], true, NS, b);
                if constexpr (!ENDS) load_row<NS>(&s_c[4 * q + j][w.sg * NS], true, NS, cc);
                float v = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    h[i] = fmaf(__builtin_amdgcn_exp2f(dl[j] * a2[i]), h[i], du[j] * b[i]);
                    if constexpr (!ENDS) v = fmaf(cc[i], h[i], v);
                }
                if constexpr (ENDS) sum += dl[j];
                else y[j] = group_sum<L>(v);
            }
            if constexpr (!ENDS) {
                const int k = w.sg & 3;
                const float mine = k == 0 ? y[0] : k == 1 ? y[1] : k == 2 ? y[2] : y[3];
                if (w.sg < 4) s_y[w.ch][4 * q + k] = mine;
            }
        }
        __syncthreads();
        if constexpr (!ENDS) {
            if (t < a.length) {
                float y[E];
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    float v = fmaf(skip[i], u[i], s_y[w.ce + i][w.te]);
                    if (a.z != nullptr) v *= z[i] * sigmoid_fast(z[i]);
                    y[i] = t < len ? v : 0.f;
                }
                store_row<E>(reinterpret_cast<T*>(a.y) + ((long)w.n * a.length + t) * a.channels + c, wide, w.he, y);
            }
        }
    }
    if constexpr (ENDS) {
        store_row<NS>(ends + w.end(p, w.segment), true, NS, h);
        if (w.sg == 0) end_deltas[w.end_delta(p, w.segment)] = sum;
    } else {
        for (int tile = work_end > first ? work_end : first; tile < last; ++tile) {
            const int t = tile * kTile + w.te;
            float zero[E] = {};
            if (t < a.length) store_row<E>(reinterpret_cast<T*>(a.y) + ((long)w.n * a.length + t) * a.channels + c, wide, w.he, zero);
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

// One frame.  Bound: the state, read and written once; L lanes a channel as in the scan, four states a lane in one 16-byte access.
template <typename T, int L, int NS>
__global__ __launch_bounds__(256) void scan_step_kernel(fsc_selective_scan_args a, int wide) {
    const long slot = (long)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int sg = threadIdx.x % L;
    const bool real = slot < (long)a.batch * a.channels;
    const long n = real ? slot / a.channels : 0;
    const int c = real ? (int)(slot % a.channels) : 0, group = c / (a.channels / a.groups);
    const int s0 = sg * NS, have = a.states - s0 < 0 || !real ? 0 : a.states - s0 < NS ? a.states - s0 : NS;
    float* state = a.final + (n * a.channels + c) * a.states + s0;
    float h[NS], al[NS], b[NS], cc[NS];
    const bool go = wide && have == NS;
    load_row<NS>(state, go, have, h);
    load_row<NS>(a.a_log + (long)c * a.states + s0, go, have, al);
    load_row<NS>(reinterpret_cast<const T*>(a.b) + n * a.b_batch + group * a.b_group + s0, false, have, b);
    load_row<NS>(reinterpret_cast<const T*>(a.c) + n * a.c_batch + group * a.c_group + s0, false, have, cc);
    const float u = (float)reinterpret_cast<const T*>(a.u)[n * a.u_batch + c];
    const float raw = (float)reinterpret_cast<const T*>(a.dt)[n * a.dt_batch + c] + (a.dt_bias != nullptr ? a.dt_bias[c] : 0.f);
    const float delta = a.softplus ? softplus_fast(raw) : raw;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        h[i] = fmaf(__builtin_amdgcn_exp2f(delta * (-__expf(al[i]) * kLog2e)), h[i], delta * u * b[i]);
        if (i < have) v = fmaf(cc[i], h[i], v);
    }
    store_row<NS>(state, go, have, h);
    v = group_sum<L>(v);
    if (sg == 0 && real) {
        if (a.d != nullptr) v = fmaf(a.d[c], u, v);
        if (a.z != nullptr) {
            const float z = (float)reinterpret_cast<const T*>(a.z)[n * a.z_batch + c];
            v *= z * sigmoid_fast(z);
        }
        reinterpret_cast<T*>(a.y)[slot] = (T)v;
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
    float* ends = reinterpret_cast<float*>(a.workspace);
    float* end_deltas = ends == nullptr ? nullptr : ends + (size_t)a.batch * p.segments * p.padded_channels() * p.padded_states();
    const dim3 grid((unsigned)((long)a.batch * p.blocks * p.segments));
    auto typed = [&](auto type) {
        using T = decltype(type);
        with_scan_shape(p, [&](auto lanes, auto per) {
            constexpr int L = decltype(lanes)::value, NS = decltype(per)::value;
            if (p.segments > 1)
                hipLaunchKernelGGL((scan_fwd_kernel<T, L, NS, true>), grid, dim3(256), 0, as_stream(stream), a, p, ends, end_deltas);
            hipLaunchKernelGGL((scan_fwd_kernel<T, L, NS, false>), grid, dim3(256), 0, as_stream(stream), a, p, ends, end_deltas);
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
    const long slots = (long)a.batch * a.channels;
    const dim3 grid((unsigned)ceil_div(slots, p.channels_block));
    auto typed = [&](auto type) {
        using T = decltype(type);
        with_scan_shape(p, [&](auto lanes, auto per) {
            hipLaunchKernelGGL((scan_step_kernel<T, decltype(lanes)::value, decltype(per)::value>), grid, dim3(256), 0, as_stream(stream), a,
                               wide);
        });
    };
    FSC_WITH_DTYPE(a.dtype, typed);
    FSC_LAUNCH_CHECK("fsc_selective_scan_step");
    return 0;
}

}  // extern "C"
