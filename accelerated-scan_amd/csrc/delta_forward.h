// Forward pass of the gated delta rule: the chain over the blocks of a sequence (delta.h).
//
// The blocks of a sequence follow each other, so what counts is the time from a state to the next: a chain of
// three products (K S0, T R, K^T U) that are too small to fill a wave's matrix unit for long.  A workgroup
// of four waves therefore takes only 16 columns of one head's state and divides the rows: wave w keeps
// state rows dk/4 w .. in its accumulators and computes tokens 16w .. 16w+15 of every block.  State, R and U
// go round through LDS in the order in which the next product reads them, with one barrier each; everything
// that comes from memory is requested one block ahead.
#ifndef ASCAN_DELTA_FORWARD_H_
#define ASCAN_DELTA_FORWARD_H_

#include "delta_prepare.h"

namespace ascan {
namespace {

// Where workgroup `id` of a chain kernel works.  Workgroups go round the eight dies one by one: the column
// groups of a head, which read the same keys, queries and matrices, are put eight apart, behind one cache.
struct ChainAt {
    int64_t sequence;
    int head, col0;
    bool there;
};
__device__ __forceinline__ ChainAt chain_at(const DeltaShape& s) {
    const int64_t groups = (s.dv + 15) / 16, id = blockIdx.x;
    const int64_t unit = id / (8 * groups) * 8 + id % 8;
    return ChainAt{unit / s.heads, (int)(unit % s.heads), (int)(id / 8 % groups) * 16, unit < s.sequences * s.heads};
}
inline int64_t chain_grid(const DeltaShape& s) { return (s.sequences * s.heads + 7) / 8 * 8 * ((s.dv + 15) / 16); }

template <int NI, int NS, int DK>
constexpr int kChainBytes = 2 * Tile<NI, DK>::kBytes + Tile<NI, 16>::kBytes + Exchange<NS, DK / 32>::kBytes +
                            3 * Exchange<NS, 2>::kBytes;

// grid chain_grid(), 256 threads.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(256) void delta_chain(DeltaShape s, const typename E::S* __restrict__ q,
                                                   const typename E::S* __restrict__ k,
                                                   const typename E::S* __restrict__ v,
                                                   const float* __restrict__ gates, const char* __restrict__ t_in,
                                                   const char* __restrict__ p_in, const float* __restrict__ initial,
                                                   typename E::S* __restrict__ out, float* __restrict__ final,
                                                   float* __restrict__ states, float* __restrict__ updates) {
    using ES = typename E::S;
    constexpr int kDepths = DK / 32, kOwn = DK / 64, kCopies = DK / 32;  // operands of a row, state tiles of a wave, loads of a thread
    extern __shared__ __align__(16) char smem[];
    const ChainAt where = chain_at(s);
    if (!where.there) return;
    const int64_t n = where.sequence;
    const int head = where.head, key_head = head / (s.heads / s.key_heads);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int col0 = where.col0, col = col0 + c;
    const bool mine = col < s.dv;
    const SequenceAt at = sequence_at(s, n);

    char* m = smem;
    Tile<NI, DK> kt[2] = {Tile<NI, DK>(m), Tile<NI, DK>(m + Tile<NI, DK>::kBytes)};
    m += 2 * Tile<NI, DK>::kBytes;
    Tile<NI, 16> vt(m);
    m += Tile<NI, 16>::kBytes;
    Exchange<NS, kDepths> xs(m);
    m += Exchange<NS, kDepths>::kBytes;
    Exchange<NS, 2> xr(m), xu(m + Exchange<NS, 2>::kBytes), xd(m + 2 * Exchange<NS, 2>::kBytes);

    fx4 S[kOwn];
    const int64_t state_at = (n * s.heads + head) * s.dk * s.dv + col;
#pragma unroll
    for (int t = 0; t < kOwn; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * (kOwn * wave + t) + 4 * g + r;
            S[t][r] = initial != nullptr && mine && row < s.dk ? initial[state_at + (int64_t)row * s.dv] : 0.0f;
        }

    // what comes from memory for the block at `first`
    Eight<E> k_raw[kCopies], v_raw, q_raw[kDepths];
    Operand<NS> tm[2], pm[2];
    fx4 beta, beta_since, until;
    float since, whole;
    const int token = 16 * wave + c;
    const auto load_kv = [&](int64_t first) {
        const int64_t row0 = at.row + first, left = at.length - first;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
            k_raw[i] = load8<E>(k + ((row0 + row) * s.key_heads + key_head) * s.dk + d, row < left && d < s.dk);
        }
        const int row = tid >> 1, d = col0 + (tid & 1) * 8;
        v_raw = load8<E>(v + ((row0 + row) * s.heads + head) * s.dv + d, tid < 128 && row < left && d < s.dv);
    };
    const auto load_q = [&](int64_t first) {
        const ES* from = q + ((at.row + first + token) * s.key_heads + key_head) * s.dk;
#pragma unroll
        for (int d = 0; d < kDepths; ++d) q_raw[d] = load_depths<E>(from, 32 * d, g, s.dk, token < at.length - first);
    };
    const auto entry_of = [&](int64_t first) { return (at.block + first / kBlock) * s.heads + head; };
    const auto load_matrix = [&](const char* from, int64_t first, Operand<NS>(&o)[2]) {
        const char* mat = from + entry_of(first) * kMatrixBytes<NS>;
        o[0] = matrix_operand<NS>(mat, pair_lower(wave, 0), lane);
        if (wave >= 2) o[1] = matrix_operand<NS>(mat, pair_lower(wave, 1), lane);
    };
    const auto gate_row = [&](int64_t first, int row) { return gates + entry_of(first) * kGateFloats + row * kBlock; };

    int64_t next = 0;
    if (at.length > 0) {
        load_kv(0);
        load_q(0);
        beta = *reinterpret_cast<const fx4*>(gate_row(0, kBeta) + 16 * wave + 4 * g);
        beta_since = *reinterpret_cast<const fx4*>(gate_row(0, kBetaSince) + 16 * wave + 4 * g);
        load_matrix(t_in, 0, tm);
        until = *reinterpret_cast<const fx4*>(gate_row(0, kUntil) + 16 * wave + 4 * g);
        load_matrix(p_in, 0, pm);
        since = gate_row(0, kSince)[token];
        whole = gate_row(0, kSince)[kBlock - 1];
    }
    for (int64_t first = 0; first < at.length; first = next) {
        next = first + kBlock;
        const int64_t ahead = next < at.length ? next : first;
        const int64_t row0 = at.row + first;
        const int length = (int)(at.length - first < kBlock ? at.length - first : kBlock);
        Tile<NI, DK>& kb = kt[(first / kBlock) & 1];

        if (states != nullptr && mine) {
            float* to = states + entry_of(first) * s.dk * s.dv + col;
#pragma unroll
            for (int t = 0; t < kOwn; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * (kOwn * wave + t) + 4 * g + r;
                    if (row < s.dk) to[(int64_t)row * s.dv] = S[t][r];
                }
        }
#pragma unroll
        for (int t = 0; t < kOwn; ++t) xs.put(kOwn * wave + t, lane, S[t]);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) kb.template put8<E>((tid + 256 * i) / (DK / 8), (tid + 256 * i) % (DK / 8) * 8, k_raw[i]);
        if (tid < 128) vt.template put8<E>(tid >> 1, (tid & 1) * 8, v_raw);
        lds_barrier();
        load_kv(ahead);

        // K S0 (rows: tokens, columns: state columns) and (Q S0)^T (rows: state columns, columns: tokens)
        fx4 u = {0, 0, 0, 0}, o = {0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < kDepths; ++d) {
            const Operand<NS> so = xs.get(d, lane);
            u = mma<NI, NS>(kb.along(token, 32 * d, g), so, u);
            o = mma<NS, NI>(so, operand_from<NI, E>(q_raw[d]), o);
        }
        load_q(ahead);
        // R = diag(beta) V - diag(beta e^c) K S0
        {
            const fx4 x = vt.tile(16 * wave, 0, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) u[r] = beta[r] * x[r] - beta_since[r] * u[r];
        }
        beta = *reinterpret_cast<const fx4*>(gate_row(ahead, kBeta) + 16 * wave + 4 * g);
        beta_since = *reinterpret_cast<const fx4*>(gate_row(ahead, kBetaSince) + 16 * wave + 4 * g);
        xr.put(wave, lane, u);
        lds_barrier();

        // U = R + T R
        u = mma<NS, NS>(tm[0], xr.get(0, lane), u);
        if (wave >= 2) u = mma<NS, NS>(tm[1], xr.get(1, lane), u);
        load_matrix(t_in, ahead, tm);
        xu.put(wave, lane, u);
        {
            fx4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = until[r] * u[r];
            xd.put(wave, lane, x);
        }
        until = *reinterpret_cast<const fx4*>(gate_row(ahead, kUntil) + 16 * wave + 4 * g);
        lds_barrier();

        // S1 = e^c[63] S0 + K^T diag(e^(c[63]-c)) U
        {
            const Operand<NS> low = xd.get(0, lane), high = xd.get(1, lane);
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t][r] *= whole;
                S[t] = mma<NI, NS>(kb.down(0, 16 * (kOwn * wave + t), lane), low, S[t]);
                S[t] = mma<NI, NS>(kb.down(32, 16 * (kOwn * wave + t), lane), high, S[t]);
            }
        }
        // out^T = scale (Q S0)^T diag(e^c) + U^T P^T
        {
            const float f = s.scale * since;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] *= f;
            o = mma<NS, NS>(xu.get(0, lane), pm[0], o);
            if (wave >= 2) o = mma<NS, NS>(xu.get(1, lane), pm[1], o);
            const int d = col0 + 4 * g;
            if (token < length && d < s.dv) store4<E>(out + ((row0 + token) * s.heads + head) * s.dv + d, o);
        }
        load_matrix(p_in, ahead, pm);
        since = gate_row(ahead, kSince)[token];
        whole = gate_row(ahead, kSince)[kBlock - 1];
        if (updates != nullptr && mine) {
            float* to = updates + ((row0 + 16 * wave + 4 * g) * s.heads + head) * s.dv + col;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * wave + 4 * g + r < length) to[(int64_t)r * s.heads * s.dv] = u[r];
        }
    }
    if (final != nullptr && mine) {
#pragma unroll
        for (int t = 0; t < kOwn; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * (kOwn * wave + t) + 4 * g + r;
                if (row < s.dk) final[state_at + (int64_t)row * s.dv] = S[t][r];
            }
    }
    // rows in front of the first and behind the last sequence are zero
    if (s.offsets != nullptr && mine) {
        const int own = 4 * wave + g;
        if (n == 0)
            for (int64_t row = own; row < offset_at(s, 0); row += 16) out[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
        if (n == s.sequences - 1)
            for (int64_t row = offset_at(s, s.sequences) + own; row < s.rows; row += 16)
                out[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
    }
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_FORWARD_H_
