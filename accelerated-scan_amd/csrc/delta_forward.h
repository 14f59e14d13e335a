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

// grid chain_grid(), 256 threads.  KEEP: write the states in front of the blocks and the rows U.
template <class E, int NI, int NS, int DK, bool KEEP>
__global__ __launch_bounds__(256, 2) void delta_chain(DeltaShape s, const typename E::S* __restrict__ q,
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
            const int row = feature_row(kOwn * wave + t, g, r);
            S[t][r] = initial != nullptr && mine && row < s.dk ? initial[state_at + (int64_t)row * s.dv] : 0.0f;
        }

    constexpr uint32_t kSize = sizeof(ES);
    const uint32_t k_step = s.key_heads * s.dk * kSize, v_step = s.heads * s.dv * kSize;
    const int64_t seq_row = uniform(at.row), seq_length = uniform(at.length), seq_block = uniform(at.block);
    const int token = 16 * wave + c;

    // what comes from memory for the block at `first`
    Eight<E> k_raw[kCopies], v_raw, q_raw[kDepths];
    Operand<NS> tm[2], pm[2];
    fx4 beta, beta_since, until;
    float since, whole;
    const auto rows_of = [&](const void* p, int64_t first, uint32_t step, int64_t at_head, uint32_t bytes) {
        const int64_t left = seq_length - first < kBlock ? seq_length - first : kBlock;
        return buffer_of(static_cast<const char*>(p) + (seq_row + first) * step + at_head, (left - 1) * (int64_t)step + bytes);
    };
    const auto entry_of = [&](int64_t first) { return (seq_block + first / kBlock) * s.heads + head; };
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
    const auto load_q = [&](int64_t first) {
        const Buffer b = rows_of(q, first, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
#pragma unroll
        for (int d = 0; d < kDepths; ++d) q_raw[d] = fetch8<E>(b, 32 * d + 8 * g < s.dk ? token * k_step + (32 * d + 8 * g) * kSize : kOutside);
    };
    // (waves 0 and 1 have one operand to a row of tiles: their second load repeats the first)
    const auto load_matrix = [&](const char* from, int64_t first, Operand<NS>(&o)[2]) {
        const Buffer b = buffer_of(from + entry_of(first) * kMatrixBytes<NS>, kMatrixBytes<NS>);
        o[0] = matrix_operand<NS>(b, pair_lower(wave, 0), lane);
        o[1] = matrix_operand<NS>(b, pair_lower(wave, wave >= 2 ? 1 : 0), lane);
    };
    const auto gates_of = [&](int64_t first) { return buffer_of(gates + entry_of(first) * kGateFloats, kGateFloats * 4); };
    const uint32_t gate_rows = (16 * wave + 4 * g) * 4;

    if (seq_length > 0) {  // (an empty sequence has no table entry to read)
        load_kv(0);
        load_q(0);
        const Buffer b = gates_of(0);
        beta = fetch16(b, kBeta * 256 + gate_rows);
        beta_since = fetch16(b, kBetaSince * 256 + gate_rows);
        load_matrix(t_in, 0, tm);
        until = fetch16(b, kUntil * 256 + gate_rows);
        whole = fetch4(b, kSince * 256 + (c | 63) * 4);
    }
    // out^T = scale (Q S0)^T diag(e^c) + U^T P^T of the block at `first`: finished while the next block's first
    // product waits for its operands
    fx4 o = {0, 0, 0, 0};
    const auto finish = [&](int64_t first, const Operand<NS>& low, const Operand<NS>& high) {
        const float f = s.scale * since;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] *= f;
        o = mma<NS, NS>(low, pm[0], o);
        if (wave >= 2) {
            const fx4 more = mma<NS, NS>(high, pm[1], fx4{0, 0, 0, 0});
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] += more[r];
        }
        const int d = col0 + 4 * g;
        const Buffer to = rows_of(out, first, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize);
        put4<E>(to, d < s.dv ? token * v_step + d * kSize : kOutside, o);
    };
    for (int64_t first = 0; first < seq_length; first += kBlock) {
        const int64_t ahead = first + kBlock < seq_length ? first + kBlock : first;
        const Buffer gb = gates_of(ahead);
        const Tile<NI, DK> kb(smem + ((first / kBlock) & 1) * Tile<NI, DK>::kBytes);

        if constexpr (KEEP) {
            const Buffer to = buffer_of(states + entry_of(first) * s.dk * s.dv, (int64_t)s.dk * s.dv * 4);
#pragma unroll
            for (int t = 0; t < kOwn; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    put1<ElemF32>(to, mine ? (feature_row(kOwn * wave + t, g, r) * s.dv + col) * 4 : kOutside, S[t][r]);
        }
#pragma unroll
        for (int t = 0; t < kOwn; ++t) xs.put(kOwn * wave + t, lane, S[t]);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) kb.template put8<E>((tid + 256 * i) / (DK / 8), (tid + 256 * i) % (DK / 8) * 8, k_raw[i]);
        vt.template put8<E>((tid & 127) >> 1, (tid & 1) * 8, v_raw);
        lds_barrier();

        // K S0 (rows: tokens, columns: state columns)
        Operand<NS> so[kDepths];
        Operand<NI> ko[kDepths];
#pragma unroll
        for (int d = 0; d < kDepths; ++d) {
            so[d] = xs.get(d, lane);
            ko[d] = kb.along(token, 32 * d, g);
        }
        const Operand<NS> u_low = xu.get(0, lane), u_high = xu.get(1, lane);  // of the block before
        fx4 x = vt.tile(16 * wave, 0, lane);
        load_kv(ahead);
        __builtin_amdgcn_sched_barrier(0);  // all reads on their way before the first product waits for one
        fx4 u = {0, 0, 0, 0}, u2 = {0, 0, 0, 0};  // (two sums: half as many products that wait for each other)
#pragma unroll
        for (int d = 0; d < kDepths; d += 2) {
            u = mma<NI, NS>(ko[d], so[d], u);
            u2 = mma<NI, NS>(ko[d + 1], so[d + 1], u2);
        }
        if (first > 0) finish(first - kBlock, u_low, u_high);
        const Buffer here = gates_of(first);
        load_matrix(p_in, first, pm);
        since = fetch4(here, kSince * 256 + token * 4);
        // R = diag(beta) V - diag(beta e^c) K S0
#pragma unroll
        for (int r = 0; r < 4; ++r) u[r] = beta[r] * x[r] - beta_since[r] * (u[r] + u2[r]);
        xr.put(wave, lane, u);
        beta = fetch16(gb, kBeta * 256 + gate_rows);
        beta_since = fetch16(gb, kBetaSince * 256 + gate_rows);
        lds_barrier();

        // U = R + T R, and (Q S0)^T (rows: state columns, columns: tokens) while its operands come
        {
            const Operand<NS> low = xr.get(0, lane), high = xr.get(1, lane);
            __builtin_amdgcn_sched_barrier(0);
            o = fx4{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < kDepths; ++d) o = mma<NS, NI>(so[d], operand_from<NI, E>(q_raw[d]), o);
            u = mma<NS, NS>(tm[0], low, u);
            if (wave >= 2) {
                u2 = mma<NS, NS>(tm[1], high, fx4{0, 0, 0, 0});
#pragma unroll
                for (int r = 0; r < 4; ++r) u[r] += u2[r];
            }
        }
        load_q(ahead);
        load_matrix(t_in, ahead, tm);
        xu.put(wave, lane, u);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = until[r] * u[r];
        xd.put(wave, lane, x);
        until = fetch16(gb, kUntil * 256 + gate_rows);
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
    if (seq_length > 0) finish((seq_length - 1) / kBlock * kBlock, xu.get(0, lane), xu.get(1, lane));
    if (final != nullptr && mine) {
#pragma unroll
        for (int t = 0; t < kOwn; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = feature_row(kOwn * wave + t, g, r);
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
