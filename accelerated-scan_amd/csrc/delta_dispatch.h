// Launches the gated delta rule kernels for one element type.
#ifndef ASCAN_DELTA_DISPATCH_H_
#define ASCAN_DELTA_DISPATCH_H_

#include "ascan.h"
#include "delta_backward.h"
#include "delta_step.h"
#include "dispatch.h"

namespace ascan {
namespace {

inline int delta_status(hipError_t e) {
    if (e == hipSuccess) return ASCAN_OK;
    g_last_hip_error = (int)e;
    return ASCAN_ERR_LAUNCH;
}

inline size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

// The workspace's parts: table of the blocks' gates, T, P, copies of keys and queries, and for the backward
// pass the state gradients behind every block, the rows dR and sums over heads that share their keys.
struct DeltaParts {
    size_t gates, t, p, k, q, d_states, d_rows, sums, end;
    DeltaParts(const DeltaShape& s, bool backward, size_t element) {
        const size_t entries = (size_t)s.blocks * s.heads;
        const size_t copy = (size_t)s.blocks * s.key_heads * kBlock * (s.dk <= 64 ? 64 : 128) * element;
        gates = 0;
        t = round_up(gates + entries * kGateFloats * 4);
        p = round_up(t + entries * kMatrixBytes);
        k = round_up(p + entries * kMatrixBytes);
        q = round_up(k + copy);
        d_states = round_up(q + copy);
        d_rows = round_up(d_states + (backward ? entries * s.dk * s.dv * 4 : 0));
        sums = round_up(d_rows + (backward ? (size_t)s.rows * s.heads * s.dv * 4 : 0));
        end = round_up(sums + (backward && s.heads > s.key_heads ? entries * 2 * kBlock * (s.dk <= 64 ? 64 : 128) * 4 : 0));
    }
};

template <class... P, class... A>
hipError_t delta_launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t lds, hipStream_t stream, A... args) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, stream, args...);
    return hipGetLastError();
}

template <class E, int NI, int DK>
hipError_t prepare(const DeltaShape& s, const void* q, const void* k, const void* log_gates, const void* beta,
                   char* ws, const DeltaParts& at, bool upper, hipStream_t stream) {
    using S = typename E::S;
    const auto kernel = upper ? delta_prepare<E, NI, DK, true> : delta_prepare<E, NI, DK, false>;
    return delta_launch(kernel, dim3((unsigned)s.blocks, (unsigned)s.heads), 256,
                        kPrepareBytes<NI, DK>, stream, s, static_cast<const S*>(q), static_cast<const S*>(k),
                        log_gates, beta, reinterpret_cast<float*>(ws + at.gates), ws + at.t, ws + at.p,
                        reinterpret_cast<S*>(ws + at.k), reinterpret_cast<S*>(ws + at.q));
}

constexpr int kLdsBytes = 160 * 1024;  // of a compute unit

template <class E, int NI, int NS, int DK>
int delta_forward_dk(const DeltaForward& f) {
    static_assert(kChainBytes<NI, NS, DK> <= kLdsBytes && kPrepareBytes<NI, DK> <= kLdsBytes, "fits a compute unit");
    using S = typename E::S;
    const DeltaShape& s = f.shape;
    const DeltaParts at(s, false, sizeof(S));
    if (s.blocks > 0) {
        const hipError_t e = prepare<E, NI, DK>(s, f.q, f.k, f.log_gates, f.beta, f.workspace, at, false, f.stream);
        if (e != hipSuccess) return delta_status(e);
    }
    const auto chain = f.states != nullptr ? delta_chain<E, NI, NS, DK, true> : delta_chain<E, NI, NS, DK, false>;
    return delta_status(delta_launch(
        chain, dim3((unsigned)chain_grid(s)), 768, kChainBytes<NI, NS, DK>, f.stream,
        s, reinterpret_cast<const S*>(f.workspace + at.q), reinterpret_cast<const S*>(f.workspace + at.k), static_cast<const S*>(f.v),
        reinterpret_cast<const float*>(f.workspace + at.gates), f.workspace + at.t, f.workspace + at.p, f.initial,
        static_cast<S*>(f.out), f.final, f.states, f.updates, chain_touches<NI, NS, DK>(f.states != nullptr)));
}

template <class E, int NI, int NS, int DK>
int delta_backward_dk(const DeltaBackward& f) {
    static_assert(kReverseBytes<NI, NS, DK> <= kLdsBytes && kGradientBytes<NI, NS, DK> + kGradientStatic <= kLdsBytes, "fits a compute unit");
    using S = typename E::S;
    const DeltaShape& s = f.shape;
    const DeltaParts at(s, true, sizeof(S));
    char* ws = f.workspace;
    hipError_t e = hipSuccess;
    if (s.blocks > 0) e = prepare<E, NI, DK>(s, f.q, f.k, f.log_gates, f.beta, ws, at, true, f.stream);
    if (e != hipSuccess) return delta_status(e);
    const float* gates = reinterpret_cast<const float*>(ws + at.gates);
    float* d_states = reinterpret_cast<float*>(ws + at.d_states);
    float* d_rows = reinterpret_cast<float*>(ws + at.d_rows);
    e = delta_launch(delta_reverse_chain<E, NI, NS, DK>, dim3((unsigned)chain_grid(s)), 768, kReverseBytes<NI, NS, DK>, f.stream, s, reinterpret_cast<const S*>(ws + at.q), reinterpret_cast<const S*>(ws + at.k),
                     static_cast<const S*>(f.d_out), gates, ws + at.t, ws + at.p, f.d_final, static_cast<S*>(f.d_v),
                     f.d_initial, d_states, d_rows, chain_touches<NI, NS, DK>(true));
    if (e != hipSuccess || s.blocks == 0) return delta_status(e);
    const bool shared = s.heads > s.key_heads;
    const auto kernel = shared ? delta_gradients<E, NI, NS, DK, true> : delta_gradients<E, NI, NS, DK, false>;
    float* sums = reinterpret_cast<float*>(ws + at.sums);
    e = delta_launch(kernel, dim3((unsigned)s.blocks, (unsigned)s.heads), 512, kGradientBytes<NI, NS, DK>, f.stream, s,
                     reinterpret_cast<const S*>(ws + at.q), reinterpret_cast<const S*>(ws + at.k), static_cast<const S*>(f.v),
                     static_cast<const S*>(f.d_out), gates, f.states, f.updates, static_cast<const float*>(d_states),
                     static_cast<const float*>(d_rows), static_cast<S*>(f.d_q), static_cast<S*>(f.d_k), f.d_log_gates,
                     f.d_beta, sums);
    if (e == hipSuccess && shared)
        e = delta_launch(delta_fold<E, DK>, dim3((unsigned)s.blocks, (unsigned)s.key_heads), 512, 0, f.stream, s,
                         static_cast<const float*>(sums), static_cast<S*>(f.d_q), static_cast<S*>(f.d_k));
    return delta_status(e);
}

template <class E, int Q, int N>
int delta_step_rows(const DeltaStep& p) {
    const int groups = (p.dv + 4 * Q - 1) / (4 * Q);
    return delta_status(delta_launch(delta_step<E, Q, N>, dim3((unsigned)(p.batch * p.heads * groups)), 256, 0, p.stream, p, groups));
}

// 128 columns to a workgroup, or 32 where that leaves compute units without one: the latency of one conversation's
// step is that of a workgroup's loads and stores (32 heads of 128 x 128: 10.1 us with 32 workgroups, 6.0 with 128).
template <class E>
int delta_step_any(const DeltaStep& p) {
    const bool few = p.batch * p.heads * ((p.dv + 127) / 128) < 512;
    if (p.dk <= 64) return few ? delta_step_rows<E, 8, 2>(p) : delta_step_rows<E, 32, 8>(p);
    return few ? delta_step_rows<E, 8, 4>(p) : delta_step_rows<E, 32, 16>(p);
}

}  // namespace

#define ASCAN_DEFINE_DELTA(suffix, E, NI, NS)                                                                       \
    namespace ascan {                                                                                           \
    int delta_forward_##suffix(const DeltaForward& f) {                                                         \
        return f.shape.dk <= 64 ? delta_forward_dk<E, NI, NS, 64>(f) : delta_forward_dk<E, NI, NS, 128>(f);     \
    }                                                                                                           \
    int delta_backward_##suffix(const DeltaBackward& f) {                                                       \
        return f.shape.dk <= 64 ? delta_backward_dk<E, NI, NS, 64>(f) : delta_backward_dk<E, NI, NS, 128>(f);   \
    }                                                                                                           \
    int delta_step_##suffix(const DeltaStep& p) { return delta_step_any<E>(p); }                                \
    size_t delta_workspace_##suffix(const DeltaShape& s, bool backward) { return DeltaParts(s, backward, sizeof(E::S)).end; } \
    }

}  // namespace ascan

#endif  // ASCAN_DELTA_DISPATCH_H_
