// Forward pass of the gated delta rule: the chain over the blocks of a sequence (delta.h).
//
// The blocks of a sequence follow each other, so what counts is the time from a state to the next: a chain of
// three products (K S0, T R, K^T U) that are too small to fill a wave's matrix unit for long.  A workgroup
// therefore takes only 16 columns of one head's state and divides the rows: state wave w (0 to 3) keeps state rows
// dk/4 w .. in its accumulators and computes tokens 16w .. 16w+15 of every block.  State, R and U go round through LDS
// in the order in which the next product reads them, with one barrier each.  Four more waves, one beside each
// of the first on its SIMD, do what the chain does not wait for: they bring keys and values to LDS a block ahead and
// compute the outputs.
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
constexpr int kChainBytes = 2 * Tile<NI, DK>::kBytes + 2 * Tile<NI, 16>::kBytes + Exchange<NS, DK / 32>::kBytes +
                            3 * Exchange<NS, 2>::kBytes;

// grid chain_grid(), 512 threads.  KEEP: write the states in front of the blocks and the rows U.
template <class E, int NI, int NS, int DK, bool KEEP>
__global__ __launch_bounds__(512) void delta_chain(DeltaShape s, const typename E::S* __restrict__ q,
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
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const bool keeper = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8) == 0;  // a state wave
    const int col0 = where.col0, col = col0 + c;
    const bool mine = col < s.dv;
    const SequenceAt at = sequence_at(s, n);

    char* m = smem;
    m += 2 * Tile<NI, DK>::kBytes;
    char* const vt_at = m;
    m += 2 * Tile<NI, 16>::kBytes;
    Exchange<NS, kDepths> xs(m);
    m += Exchange<NS, kDepths>::kBytes;
    Exchange<NS, 2> xr(m), xu(m + Exchange<NS, 2>::kBytes), xd(m + 2 * Exchange<NS, 2>::kBytes);

    constexpr uint32_t kSize = sizeof(ES);
    const uint32_t k_step = s.key_heads * s.dk * kSize, v_step = s.heads * s.dv * kSize;
    const int64_t seq_row = uniform(at.row), seq_length = uniform(at.length), seq_block = uniform(at.block);
    const int token = 16 * wave + c;
    const auto rows_of = [&](const void* p, int64_t first, uint32_t step, int64_t at_head, uint32_t bytes) {
        const int64_t left = seq_length - first < kBlock ? seq_length - first : kBlock;
        return buffer_of(static_cast<const char*>(p) + (seq_row + first) * step + at_head, (left - 1) * (int64_t)step + bytes);
    };
    const auto entry_of = [&](int64_t first) { return (seq_block + first / kBlock) * s.heads + head; };
    const auto gates_of = [&](int64_t first) { return buffer_of(gates + entry_of(first) * kGateFloats, kGateFloats * 4); };
    // (waves 0 and 1 have one operand to a row of tiles: their second load lies outside and gives zero)
    const auto load_matrix = [&](const char* from, int64_t first, Operand<NS>(&o)[2]) {
        const Buffer b = buffer_of(from + entry_of(first) * kMatrixBytes<NS>, kMatrixBytes<NS>);
        o[0] = matrix_operand<NS>(b, pair_lower(wave, 0), lane);
        o[1] = matrix_operand<NS>(b, wave >= 2 ? pair_lower(wave, 1) : (int)(kOutside >> 12), lane);
    };
    const auto ahead_of = [&](int64_t first) { return first + kBlock < seq_length ? first + kBlock : first; };
    const auto keys_at = [&](int64_t first) { return Tile<NI, DK>(smem + ((first / kBlock) & 1) * Tile<NI, DK>::kBytes); };
    const auto values_at = [&](int64_t first) { return Tile<NI, 16>(vt_at + ((first / kBlock) & 1) * Tile<NI, 16>::kBytes); };

    // An empty sequence has no table entry to read: its state is handed through.
    if (keeper) {
        fx4 S[kOwn];
        const int64_t state_at = (n * s.heads + head) * s.dk * s.dv + col;
#pragma unroll
        for (int t = 0; t < kOwn; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = feature_row(kOwn * wave + t, g, r);
                S[t][r] = initial != nullptr && mine && row < s.dk ? initial[state_at + (int64_t)row * s.dv] : 0.0f;
            }
        const uint32_t gate_rows = (16 * wave + 4 * g) * 4;
        Operand<NS> tm[2];
        fx4 beta, beta_since, until;
        float whole;
        if (seq_length > 0) {
            const Buffer b = gates_of(0);
            beta = fetch16(b, kBeta * 256 + gate_rows);
            beta_since = fetch16(b, kBetaSince * 256 + gate_rows);
            load_matrix(t_in, 0, tm);
            until = fetch16(b, kUntil * 256 + gate_rows);
            whole = fetch4(b, kSince * 256 + (c | 63) * 4);
        }
        for (int64_t first = 0; first < seq_length; first += kBlock) {
            const int64_t ahead = ahead_of(first);
            const Buffer gb = gates_of(ahead);
            const Tile<NI, DK> kb = keys_at(first);
#pragma unroll
            for (int t = 0; t < kOwn; ++t) xs.put(kOwn * wave + t, lane, S[t]);
            lds_barrier();

            // K S0 (rows: tokens, columns: state columns)
            fx4 u = {0, 0, 0, 0}, u2 = {0, 0, 0, 0};  // (two sums: half as many products that wait for each other)
            fx4 x;
            {
                Operand<NS> so[kDepths];
                Operand<NI> ko[kDepths];
#pragma unroll
                for (int d = 0; d < kDepths; ++d) {
                    so[d] = xs.get(d, lane);
                    ko[d] = kb.along(token, 32 * d, g);
                }
                x = values_at(first).tile(16 * wave, 0, lane);
                __builtin_amdgcn_sched_barrier(0);  // all reads on their way before the first product waits for one
#pragma unroll
                for (int d = 0; d < kDepths; d += 2) {
                    u = mma<NI, NS>(ko[d], so[d], u);
                    u2 = mma<NI, NS>(ko[d + 1], so[d + 1], u2);
                }
            }
            // R = diag(beta) V - diag(beta e^c) K S0
#pragma unroll
            for (int r = 0; r < 4; ++r) u[r] = beta[r] * x[r] - beta_since[r] * (u[r] + u2[r]);
            xr.put(wave, lane, u);
            lds_barrier();

            // U = R + T R
            {
                const Operand<NS> low = xr.get(0, lane), high = xr.get(1, lane);
                if constexpr (KEEP) {  // (the state, while these come)
                    const Buffer to = buffer_of(states + entry_of(first) * s.dk * s.dv, (int64_t)s.dk * s.dv * 4);
#pragma unroll
                    for (int t = 0; t < kOwn; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            put1<ElemF32>(to, mine ? (feature_row(kOwn * wave + t, g, r) * s.dv + col) * 4 : kOutside, S[t][r]);
                }
                beta = fetch16(gb, kBeta * 256 + gate_rows);
                beta_since = fetch16(gb, kBetaSince * 256 + gate_rows);
                __builtin_amdgcn_sched_barrier(0);
                u = mma<NS, NS>(tm[0], low, u);
                if (wave >= 2) {
                    u2 = mma<NS, NS>(tm[1], high, fx4{0, 0, 0, 0});
#pragma unroll
                    for (int r = 0; r < 4; ++r) u[r] += u2[r];
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = until[r] * u[r];
            xd.put(wave, lane, x);
            xu.put(wave, lane, u);
            lds_barrier();

            // S1 = e^c[63] S0 + K^T diag(e^(c[63]-c)) U
            {
                const Operand<NS> low = xd.get(0, lane), high = xd.get(1, lane);
                Operand<NI> k_low[kOwn], k_high[kOwn];
#pragma unroll
                for (int t = 0; t < kOwn; ++t) {
                    k_low[t] = kb.down_features(0, kOwn * wave + t, lane);
                    k_high[t] = kb.down_features(32, kOwn * wave + t, lane);
                }
                load_matrix(t_in, ahead, tm);
                until = fetch16(gb, kUntil * 256 + gate_rows);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < kOwn; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[t][r] *= whole;
                    S[t] = mma<NI, NS>(k_low[t], low, S[t]);
                    S[t] = mma<NI, NS>(k_high[t], high, S[t]);
                }
            }
            whole = fetch4(gb, kSince * 256 + (c | 63) * 4);
            if constexpr (KEEP) {
                const uint32_t step = s.heads * s.dv * 4;
                const Buffer to = rows_of(updates, first, step, (int64_t)head * s.dv * 4, s.dv * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    put1<ElemF32>(to, mine ? (16 * wave + 4 * g + r) * step + col * 4 : kOutside, u[r]);
            }
        }
        if (final != nullptr && mine) {
#pragma unroll
            for (int t = 0; t < kOwn; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = feature_row(kOwn * wave + t, g, r);
                    if (row < s.dk) final[state_at + (int64_t)row * s.dv] = S[t][r];
                }
        }
    } else if (seq_length > 0) {
        Eight<E> k_raw[kCopies], v_raw, q_raw[kDepths];
        Operand<NS> pm[2];
        float since;
        const auto load_kv = [&](int64_t first) {
            const Buffer kb = rows_of(k, first, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
            const Buffer vb = rows_of(v, first, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
                k_raw[i] = fetch8<E>(kb, d < s.dk ? row * k_step + d * kSize : kOutside);
            }
            const int d = col0 + (tid & 1) * 8;  // (the upper two waves repeat what the lower two do)
            v_raw = fetch8<E>(vb, d < s.dv ? ((tid & 127) >> 1) * v_step + d * kSize : kOutside);
        };
        const auto stage_kv = [&](int64_t first) {
            const Tile<NI, DK> kb = keys_at(first);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) kb.template put8<E>((tid + 256 * i) / (DK / 8), (tid + 256 * i) % (DK / 8) * 8, k_raw[i]);
            values_at(first).template put8<E>((tid & 127) >> 1, (tid & 1) * 8, v_raw);
        };
        const auto load_q = [&](int64_t first) {
            const Buffer b = rows_of(q, first, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
#pragma unroll
            for (int d = 0; d < kDepths; ++d)
                q_raw[d] = fetch8<E>(b, 32 * d + 8 * g < s.dk ? token * k_step + (32 * d + 8 * g) * kSize : kOutside);
        };
        load_kv(0);
        load_q(0);
        load_matrix(p_in, 0, pm);
        since = fetch4(gates_of(0), kSince * 256 + token * 4);
        stage_kv(0);
        load_kv(ahead_of(0));
        for (int64_t first = 0; first < seq_length; first += kBlock) {
            const int64_t ahead = ahead_of(first);
            lds_barrier();
            // (Q S0)^T (rows: state columns, columns: tokens)
            fx4 o = {0, 0, 0, 0}, o2 = {0, 0, 0, 0};
            {
                Operand<NS> so[kDepths];
#pragma unroll
                for (int d = 0; d < kDepths; ++d) so[d] = xs.get(d, lane);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < kDepths; d += 2) {
                    o = mma<NS, NI>(so[d], operand_from<NI, E>(q_raw[d]), o);
                    o2 = mma<NS, NI>(so[d + 1], operand_from<NI, E>(q_raw[d + 1]), o2);
                }
            }
            load_q(ahead);
            lds_barrier();
            // the other tiles' readers are behind the first barrier
            if (ahead != first) stage_kv(ahead);
            load_kv(ahead_of(ahead));
            const float f = s.scale * since;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = f * (o[r] + o2[r]);
            lds_barrier();
            // out^T = scale (Q S0)^T diag(e^c) + U^T P^T
            o = mma<NS, NS>(xu.get(0, lane), pm[0], o);
            if (wave >= 2) {
                o2 = mma<NS, NS>(xu.get(1, lane), pm[1], fx4{0, 0, 0, 0});
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] += o2[r];
            }
            const int d = col0 + 4 * g;
            const Buffer to = rows_of(out, first, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize);
            put4<E>(to, d < s.dv ? token * v_step + d * kSize : kOutside, o);
            load_matrix(p_in, ahead, pm);
            since = fetch4(gates_of(ahead), kSince * 256 + token * 4);
        }
    }
    // rows in front of the first and behind the last sequence are zero
    if (s.offsets != nullptr && mine && keeper) {
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
