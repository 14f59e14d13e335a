// Backward pass of the gated delta rule: a chain over the blocks from the last to the first for the
// gradient D of the state, then all blocks at once for everything that needs no further block.
//
//   dU = P^T dO + diag(e^(c[63]-c)) K D1,   dR = (I + T)^T dU,   dV = diag(beta) dR
//   D0 = e^c[63] D1 + Q^T diag(scale e^c) dO - K^T diag(beta e^c) dR
//   dQ = diag(scale e^c) dO S0^T + (F . dO U^T) K,               F[i][j] = scale e^(c[i]-c[j]), j <= i
//   A  = -diag(e^c) dR S0^T - (G . dR U^T) K,                    G[i][j] = e^(c[i]-c[j]), j < i
//   B  = diag(e^(c[63]-c)) U D1^T + (F . dO U^T)^T Q - (diag(beta) G . dR U^T)^T K
//   dK = diag(beta) A + B
//   dbeta[i] = dR[i].v[i] + k[i].A[i]
//   The log gate of token t lies on the way from S0 to t and later tokens, from earlier tokens to the state behind the block,
//   from earlier tokens to t and later ones, and from S0 to the state behind the block:
//     sum over i >= t of (q.dQ + beta k.A)[i], their parts from S0,   sum over j < t of k[j].(diag(e^(c[63]-c)) U D1^T)[j],
//     sum over pairs j < t <= i,   e^c[63] S0.D1
//   Of the pairs only the sums over earlier and over later partners of a token are known: the sum over j < t <= i is the
//   difference of the two summed from t on, or up to t.  Taken from the nearer end, and without the pairs of a token
//   with itself, it has the fewest terms that cancel (none for the first and the last token).
#ifndef ASCAN_DELTA_BACKWARD_H_
#define ASCAN_DELTA_BACKWARD_H_

#include "delta_forward.h"

namespace ascan {
namespace {

constexpr int kAhead = 256;   // workgroups from one to that which takes its place: one to a compute unit
// Sums over the features of a token: its partners S0, the state behind the block, earlier and later tokens; k.A.
enum { kFromState, kToState, kEarlier, kLater, kBetas, kSums };
constexpr int kColumns = 64;  // value columns that a workgroup of delta_gradients takes at a time

template <int NI, int NS, int DK>
constexpr int kReverseBytes = 3 * Tile<NI, DK>::kBytes + 2 * Tile<NI, 16>::kBytes + Exchange<NS, DK / 32>::kBytes +
                              2 * Exchange<NS, 2>::kBytes + (4 + DK / 16) * 1024 + Exchange<NS, kPairs>::kBytes + 4 * kBlock * 4;

// The chain, last block first, divided like the forward one: 16 columns of D to a workgroup; state wave w keeps rows
// dk/4 w .. of them and computes tokens 16w .. 16w+15; D, dU and -diag(beta e^c) dR go round through LDS.  Four waves
// compute what does not wait for D (P^T dO and Q^T diag(scale e^c) dO) and write what leaves the chain, four load.
// q and k: the copies that delta_prepare made.  grid chain_grid(), 768 threads.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(768) void delta_reverse_chain(
    DeltaShape s, const typename E::S* __restrict__ q, const typename E::S* __restrict__ k,
    const typename E::S* __restrict__ d_out, const float* __restrict__ gates, const char* __restrict__ t_in,
    const char* __restrict__ p_in, const float* __restrict__ d_final, typename E::S* __restrict__ d_v,
    float* __restrict__ d_initial, float* __restrict__ d_states, float* __restrict__ d_rows, bool ahead) {
    using ES = typename E::S;
    constexpr int kDepths = DK / 32, kOwn = DK / 64, kCopies = DK / 32;
    extern __shared__ __align__(16) char smem[];
    const ChainAt where = chain_at(s);
    if (!where.there) return;
    const int64_t n = where.sequence;
    const int head = where.head, key_head = head / (s.heads / s.key_heads);
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int role = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8);
    const int col0 = where.col0, col = col0 + c;
    const bool mine = col < s.dv;
    const SequenceAt at = sequence_at(s, n);

    // Keys, values' gradients: two blocks' room.  Queries are wanted between the second and the third barrier, T and the
    // gates in front of the second one only: room for one block.
    char* m = smem + 2 * Tile<NI, DK>::kBytes;
    const Tile<NI, DK> qt(m);
    m += Tile<NI, DK>::kBytes;
    char* const ot_at = m;
    m += 2 * Tile<NI, 16>::kBytes;
    Exchange<NS, kDepths> xs(m);
    m += Exchange<NS, kDepths>::kBytes;
    Exchange<NS, 2> xr(m), xu(m + Exchange<NS, 2>::kBytes);
    m += 2 * Exchange<NS, 2>::kBytes;
    fx4* const po_at = reinterpret_cast<fx4*>(m) + lane;  // accumulator tiles from wave to wave, a KiB each
    fx4* const dr_at = po_at;  // (P^T dO is read in front of the second barrier, dR written behind it)
    fx4* const qw_at = po_at + 4 * 64;
    m += (4 + DK / 16) * 1024;
    Exchange<NS, kPairs> matrix(m);
    float* const gate = reinterpret_cast<float*>(m + Exchange<NS, kPairs>::kBytes);

    constexpr uint32_t kSize = sizeof(ES);
    constexpr int kKeyBytes = kBlock * DK * kSize;
    const uint32_t v_step = s.heads * s.dv * kSize, r_step = s.heads * s.dv * 4;
    const int64_t seq_row = uniform(at.row), seq_length = uniform(at.length), seq_block = uniform(at.block);
    const int64_t last = (seq_length - 1) / kBlock;  // number of the last block
    const int token = 16 * wave + c;
    const auto rows_of = [&](const char* p, int64_t n_block, uint32_t step, uint32_t bytes) {
        const int64_t left = seq_length - n_block * kBlock;
        return buffer_of(p, n_block < 0 ? 0 : ((left < kBlock ? (int)left : kBlock) - 1) * (int)step + (int)bytes);
    };
    const auto start_of = [&](const void* p, uint32_t step, int64_t at_head) {
        return static_cast<const char*>(p) + (seq_row + last * kBlock) * step + at_head;
    };
    const int64_t entry0 = (seq_block + last) * s.heads + head;
    const int64_t gate_move = (int64_t)s.heads * kGateFloats * 4, matrix_move = (int64_t)s.heads * kMatrixBytes;
    const int64_t k_move = (int64_t)s.key_heads * kKeyBytes, v_move = (int64_t)v_step * kBlock;
    const char* gate_p = reinterpret_cast<const char*>(gates + entry0 * kGateFloats);
    const auto keys_at = [&](int64_t n_block) { return Tile<NI, DK>(smem + (n_block & 1) * Tile<NI, DK>::kBytes); };
    const auto outs_at = [&](int64_t n_block) { return Tile<NI, 16>(ot_at + (n_block & 1) * Tile<NI, 16>::kBytes); };
    const auto gate_rows = [&](int row) { return *reinterpret_cast<const fx4*>(gate + row * kBlock + 16 * wave + 4 * g); };

    if (role == 0) {
        fx4 D[kOwn];
        const int64_t state_at = (n * s.heads + head) * s.dk * s.dv + col;
#pragma unroll
        for (int t = 0; t < kOwn; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = feature_row(kOwn * wave + t, g, r);
                D[t][r] = d_final != nullptr && mine && row < s.dk ? d_final[state_at + (int64_t)row * s.dv] : 0.0f;
            }
        __builtin_amdgcn_s_setprio(3);
        Operand<NI> ko[kDepths];
        const auto read_block = [&](int64_t n_block) {
#pragma unroll
            for (int d = 0; d < kDepths; ++d) ko[d] = keys_at(n_block).along(token, 32 * d, g);
        };
        if (seq_length > 0) {
            lds_barrier();  // the last block is there
            read_block(last);
        }
        for (int64_t now = last; now >= 0 && seq_length > 0; --now) {
            const Tile<NI, DK> kb = keys_at(now);
#pragma unroll
            for (int t = 0; t < kOwn; ++t) xs.put(kOwn * wave + t, lane, D[t]);
            lds_barrier();

            // dU = diag(e^(c[63]-c)) K D1 + P^T dO
            fx4 u = {0, 0, 0, 0}, u2 = {0, 0, 0, 0};  // (two sums: half as many products that wait for each other)
            Operand<NS> tm[2];
            fx4 beta_since;
            float whole;
            {
                Operand<NS> so[kDepths];
#pragma unroll
                for (int d = 0; d < kDepths; ++d) so[d] = xs.get(d, lane);
                const fx4 po = po_at[wave * 64], until = gate_rows(kUntil);
                tm[0] = matrix.get(pair_upper(wave, wave >> 1), lane);
                tm[1] = matrix.get(pair_upper(wave, 1), lane);
                beta_since = gate_rows(kBetaSince);
                whole = gate[kSince * kBlock + kBlock - 1];
                __builtin_amdgcn_sched_barrier(0);  // all reads on their way before the first product waits for one
#pragma unroll
                for (int d = 0; d < kDepths; d += 2) {
                    u = mma<NI, NS>(ko[d], so[d], u);
                    u2 = mma<NI, NS>(ko[d + 1], so[d + 1], u2);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) u[r] = until[r] * (u[r] + u2[r]) + po[r];
            }
            xr.put(wave, lane, u);
            lds_barrier();

            // dR = dU + T^T dU; what the next products take of the keys is read on the way
            Operand<NI> k_low[kOwn], k_high[kOwn];
            {
                const Operand<NS> low = xr.get(0, lane), high = xr.get(1, lane);
#pragma unroll
                for (int t = 0; t < kOwn; ++t) {
                    k_low[t] = kb.down_features(0, kOwn * wave + t, lane);
                    k_high[t] = kb.down_features(32, kOwn * wave + t, lane);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (wave < 2) {
                    u2 = mma<NS, NS>(tm[0], low, fx4{0, 0, 0, 0});
                    u = mma<NS, NS>(tm[1], high, u);
#pragma unroll
                    for (int r = 0; r < 4; ++r) u[r] += u2[r];
                } else {
                    u = mma<NS, NS>(tm[1], high, u);
                }
            }
            {
                fx4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = -beta_since[r] * u[r];
                xu.put(wave, lane, y);
            }
            dr_at[wave * 64] = u;
            lds_barrier();

            // D0 = e^c[63] D1 + Q^T diag(scale e^c) dO - K^T diag(beta e^c) dR
            {
                const Operand<NS> low = xu.get(0, lane), high = xu.get(1, lane);
                fx4 qw[kOwn], D2[kOwn];
#pragma unroll
                for (int t = 0; t < kOwn; ++t) qw[t] = qw_at[(kOwn * wave + t) * 64];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < kOwn; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) D[t][r] *= whole;
                    D[t] = mma<NI, NS>(k_low[t], low, D[t]);
                    D2[t] = mma<NI, NS>(k_high[t], high, qw[t]);
                }
                read_block(now > 0 ? now - 1 : now);
#pragma unroll
                for (int t = 0; t < kOwn; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) D[t][r] += D2[t][r];
            }
        }
        if (seq_length > 0 && (last & 1) == 0) {  // the other waves go on by two blocks
            lds_barrier();
            lds_barrier();
            lds_barrier();
        }
        if (d_initial != nullptr && mine) {
#pragma unroll
            for (int t = 0; t < kOwn; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = feature_row(kOwn * wave + t, g, r);
                    if (row < s.dk) d_initial[state_at + (int64_t)row * s.dv] = D[t][r];
                }
        }
    } else if (role == 1 && seq_length > 0) {
        // In front of the first block loads repeat it or give zero and stores are dropped: no condition stands around them.
        fx4 p_raw[2][2][2];
        const char* p_p = p_in + entry0 * kMatrixBytes;
        char* state_p = reinterpret_cast<char*>(d_states + entry0 * s.dk * s.dv);
        const int quad = col0 + 4 * g;
        char *v_p = const_cast<char*>(start_of(d_v, v_step, (int64_t)head * s.dv * kSize));
        char *r_p = const_cast<char*>(start_of(d_rows, r_step, (int64_t)head * s.dv * 4));
        const auto load_p = [&](int64_t n_block, int set) __attribute__((always_inline)) {
            const Buffer b = buffer_of(p_p, kMatrixBytes);
            fetch_matrix(b, wave < 2, pair_upper(wave, 0), lane, p_raw[set][0]);
            fetch_matrix(b, true, pair_upper(wave, 1), lane, p_raw[set][1]);
            if (n_block > 0) p_p -= matrix_move;
        };
        const auto outputs = [&](int64_t n_block, int set) __attribute__((always_inline)) {  // P^T dO
            const Tile<NI, 16> ot = outs_at(n_block);
            fx4 po = {0, 0, 0, 0};
            if (wave < 2) po = mma<NS, NI>(operand_of<NS>(p_raw[set][0][0], p_raw[set][0][1]), ot.down(0, 0, lane), po);
            po_at[wave * 64] = mma<NS, NI>(operand_of<NS>(p_raw[set][1][0], p_raw[set][1][1]), ot.down(32, 0, lane), po);
        };
        load_p(last, 0);
        load_p(last - 1, 1);
        lds_barrier();
        outputs(last, 0);
        load_p(last - 2, 0);
        const auto block = [&](int64_t now, int other) __attribute__((always_inline)) {  // the next block's P is in `other`
            lds_barrier();
            // W = diag(scale e^c) dO as the right operand, and the state behind the block for the kernel that follows
            fx4 w[kTiles];
            const Tile<NI, 16> ot = outs_at(now);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const fx4 f = *reinterpret_cast<const fx4*>(gate + kSince * kBlock + 16 * t + 4 * g);
                w[t] = ot.tile(16 * t, 0, lane);
#pragma unroll
                for (int r = 0; r < 4; ++r) w[t][r] *= s.scale * f[r];
            }
            const float beta = gate[kBeta * kBlock + token];
            const Operand<NS> w_low = operand_of<NS>(w[0], w[1]), w_high = operand_of<NS>(w[2], w[3]);
            {
                const Buffer to = buffer_of(state_p, now >= 0 ? (int64_t)s.dk * s.dv * 4 : 0);
#pragma unroll
                for (int t = kOwn * wave; t < kOwn * wave + kOwn; ++t)
                    put4<ElemF32>(to, quad < s.dv ? (feature_row(t, c >> 2, c & 3) * s.dv + quad) * 4 : kOutside, exchanged_row(xs, t, lane));
                state_p -= (int64_t)s.heads * s.dk * s.dv * 4;
            }
            lds_barrier();
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
                fx4 qw = mma<NI, NS>(qt.down_features(0, kOwn * wave + t, lane), w_low, fx4{0, 0, 0, 0});
                qw = mma<NI, NS>(qt.down_features(32, kOwn * wave + t, lane), w_high, qw);
                qw_at[(kOwn * wave + t) * 64] = qw;
            }
            lds_barrier();
            // row `token` of dR, four columns, from the accumulators' order
            const float* from = reinterpret_cast<const float*>(dr_at - lane + wave * 64 + (c >> 2) * 16 + 4 * g) + (c & 3);
            const fx4 u = {from[0], from[4], from[8], from[12]};
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");  // the same place takes the next P^T dO
            outputs(now - 1, other);
            load_p(now - 3, other);
            put4<ElemF32>(rows_of(r_p, now, r_step, s.dv * 4), quad < s.dv ? token * r_step + quad * 4 : kOutside, u);
            put4<E>(rows_of(v_p, now, v_step, s.dv * kSize), quad < s.dv ? token * v_step + quad * kSize : kOutside,
                    fx4{beta * u[0], beta * u[1], beta * u[2], beta * u[3]});
            v_p -= v_move;
            r_p -= (int64_t)r_step * kBlock;
        };
        for (int64_t now = last; now >= 0; now -= 2) {
            block(now, 1);
            block(now - 1, 0);
        }
    } else if (seq_length > 0) {
        // Keys, queries, dO, T and gates to LDS.
        // (in registers for two blocks, or for one where two do not fit: with 114 registers in memory fp32 (2, 2048, 8 heads
        // of 128 x 128) took 192 us, with one block 132)
        constexpr int kSets = sizeof(Eight<E>) * kCopies > 64 ? 1 : 2;
        Eight<E> k_raw[kSets][kCopies], q_raw[kSets][kCopies], o_raw[kSets];
        fx4 t_raw[kSets][kPieces];
        float gate_raw[kSets];
        const int64_t copy0 = ((seq_block + last) * s.key_heads + key_head) * kBlock * DK;
        const char *k_p = reinterpret_cast<const char*>(k + copy0), *q_p = reinterpret_cast<const char*>(q + copy0);
        const char* o_p = start_of(d_out, v_step, (int64_t)head * s.dv * kSize);
        const char* t_p = t_in + entry0 * kMatrixBytes;
        const auto load_block = [&](int64_t n_block, int set) __attribute__((always_inline)) {
            const Buffer kb = buffer_of(k_p, kKeyBytes), qb = buffer_of(q_p, kKeyBytes), tb = buffer_of(t_p, kMatrixBytes);
            const Buffer ob = d_out != nullptr ? rows_of(o_p, n_block, v_step, s.dv * kSize) : buffer_of(k_p, 0);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                k_raw[set][i] = fetch8<E>(kb, (tid + 256 * i) * 8 * kSize);
                q_raw[set][i] = fetch8<E>(qb, (tid + 256 * i) * 8 * kSize);
            }
            const int d = col0 + (tid & 1) * 8;  // (the upper two waves repeat what the lower two do)
            o_raw[set] = fetch8<E>(ob, d < s.dv ? ((tid & 127) >> 1) * v_step + d * kSize : kOutside);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) t_raw[set][i] = fetch16(tb, (tid + 256 * i) * 16);
            gate_raw[set] = fetch4(buffer_of(gate_p, kGateFloats * 4), tid * 4);
            o_p -= v_move;
            if (n_block > 0) {
                k_p -= k_move;
                q_p -= k_move;
                t_p -= matrix_move;
                gate_p -= gate_move;
            }
        };
        const auto stage_block = [&](int64_t n_block, int set) __attribute__((always_inline)) {
            const Tile<NI, DK> kb = keys_at(n_block);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) kb.template put8<E>((tid + 256 * i) / (DK / 8), (tid + 256 * i) % (DK / 8) * 8, k_raw[set][i]);
            outs_at(n_block).template put8<E>((tid & 127) >> 1, (tid & 1) * 8, o_raw[set]);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) matrix.put(4 * i + wave, lane, t_raw[set][i]);
            gate[tid] = gate_raw[set];
        };
        const auto stage_queries = [&](int set) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) qt.template put8<E>((tid + 256 * i) / (DK / 8), (tid + 256 * i) % (DK / 8) * 8, q_raw[set][i]);
        };
        const int groups = (s.dv + 15) / 16, row_bytes = s.dv * (int)kSize;
        int touched = 0;
        const auto touch_block = [&](int64_t n_block) __attribute__((always_inline)) {
            asm volatile("" ::"v"(touched));
            if (ahead && n_block >= 0) {
                const int64_t back = last - n_block, rows = seq_length - n_block * kBlock < kBlock ? seq_length - n_block * kBlock : kBlock;
                const char* at_k = reinterpret_cast<const char*>(k + copy0) - back * k_move;
                const char* at_q = reinterpret_cast<const char*>(q + copy0) - back * k_move;
                const Lines lines{{at_k, at_q, t_in + entry0 * kMatrixBytes - back * matrix_move, p_in + entry0 * kMatrixBytes - back * matrix_move,
                                   start_of(d_out, v_step, (int64_t)head * s.dv * kSize) - back * v_move},
                                  {kKeyBytes / 128, kKeyBytes / 128, kMatrixBytes / 128, kMatrixBytes / 128,
                                   d_out != nullptr ? (int)rows * ((row_bytes + 127) / 128) : 0},
                                  (row_bytes + 127) / 128, (int64_t)v_step};
                touched = touch(lines, tid * groups + col0 / 16);
            }
        };
        load_block(last, 0);
        if constexpr (kSets == 2) load_block(last - 1, 1);
        stage_block(last, 0);
        stage_queries(0);
        load_block(last - kSets, 0);
        touch_block(last - 3);
        touch_block(last - 4);
        lds_barrier();
        const auto block = [&](int64_t now, int next) __attribute__((always_inline)) {
            const int other = next & (kSets - 1);
            lds_barrier();
            lds_barrier();
            stage_block(now - 1, other);  // the readers of all but the queries are behind the second barrier
            lds_barrier();
            stage_queries(other);
            load_block(now - 1 - kSets, other);
            touch_block(now - 5);
        };
        for (int64_t now = last; now >= 0; now -= 2) {
            block(now, 1);
            block(now - 1, 0);
        }
    }
    if (s.offsets != nullptr && mine && role == 0) {
        const int own = 4 * wave + g;
        if (n == 0)
            for (int64_t row = own; row < offset_at(s, 0); row += 16) d_v[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
        if (n == s.sequences - 1)
            for (int64_t row = offset_at(s, s.sequences) + own; row < s.rows; row += 16)
                d_v[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
    }
}

constexpr int kGradientStatic = 13 * 1024;  // what delta_gradients has in LDS beside the arrays below, at most

// dO, U and dR of kColumns columns in LDS.  The second pass over the columns goes back: with room for two such sets it finds
// the last two where the first pass has left them.
template <int NI, int NS>
constexpr int kRowsBytes = Tile<NI, kColumns>::kBytes + 2 * Tile<NS, kColumns>::kBytes;
template <int NI, int NS, int DK>
constexpr int kRowSets = 2 * Tile<NI, DK>::kBytes + 2 * kRowsBytes<NI, NS> + kGradientStatic <= 160 * 1024 ? 2 : 1;
template <int NI, int NS, int DK>
constexpr int kGradientShared = kRowSets<NI, NS, DK> * kRowsBytes<NI, NS> > 4 * Exchange<NS, kPairs>::kBytes
                                    ? kRowSets<NI, NS, DK> * kRowsBytes<NI, NS>
                                    : 4 * Exchange<NS, kPairs>::kBytes;
template <int NI, int NS, int DK>
constexpr int kGradientBytes = 2 * Tile<NI, DK>::kBytes + kGradientShared<NI, NS, DK>;

// A block of one head.  A wave owns 16 features of keys and queries and dk/2 of the tokens, so that each row of the two
// states is read by one wave only (or two); the 64 x 64 products of tokens with tokens are divided among the waves by
// tiles and go round through LDS.  The products have features as rows, so that a lane holds four of a token's and writes
// 8 bytes (with tokens as rows 211 us instead of 194 for the case below, when values were in two parts; the five sums of a token
// that the gates' gradients are made of, where two with terms that cancel would do, cost 15 again).
//
// What bounds it: a workgroup reads 256 KiB and has a compute unit to itself, for its registers (250).  bf16 (2, 4096, 16 heads
// of 128 x 128) takes 229 to 246 us for 0.72 GB, 2.9 to 3.1 TB/s, with LDS at work a third of the time, vector instructions
// 37 % and the matrix units 22 %; of 195 us in two parts 134 were left when nothing was read, so that loads and products overlap
// in part only.  A loop over heads or blocks around this body, to load ahead, lifts its address
// arithmetic in front, where it does not fit the registers (428 us for 218 at the time).
//
// SHARED: dQ and dK go to `sums` in fp32, to be added over the heads that share the keys (delta_fold).
// q and k: the copies that delta_prepare made.  grid (blocks, heads), 512 threads.
template <class E, int NI, int NS, int DK, bool SHARED>
__global__ __launch_bounds__(512) void delta_gradients(
    DeltaShape s, const typename E::S* __restrict__ q, const typename E::S* __restrict__ k,
    const typename E::S* __restrict__ v, const typename E::S* __restrict__ d_out, const float* __restrict__ gates,
    const float* __restrict__ states, const float* __restrict__ updates, const float* __restrict__ d_states,
    const float* __restrict__ d_rows, typename E::S* __restrict__ d_q, typename E::S* __restrict__ d_k,
    void* __restrict__ d_log_gates, void* __restrict__ d_beta, float* __restrict__ sums) {
    using ES = typename E::S;
    constexpr int kFeatures = DK / 16, kTok = DK / 32;  // tiles of features, and of tokens that a wave owns
    extern __shared__ __align__(16) char smem[];
    __shared__ __align__(16) float gate[kGateFloats];
    __shared__ float dots[8][kSums][16 * kTok];
    __shared__ float value_dots[kBlock], diagonal[kBlock], whole_terms[8];
    const int64_t block = blockIdx.x;
    const int head = blockIdx.y, share = s.heads / s.key_heads, key_head = head / share;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;

    // rows in front of the first and behind the last sequence: zero gradients, 64 rows to a workgroup
    if (s.offsets != nullptr) {
        const int64_t before = offset_at(s, 0), behind = offset_at(s, s.sequences);
        const int64_t spans[2][2] = {{0, before}, {behind, s.rows}};
        for (int i = 0; i < 2; ++i)
            for (int64_t row = spans[i][0] + block * kBlock + wave; row < spans[i][1] && row < spans[i][0] + (block + 1) * kBlock;
                 row += 8) {
                if (head % share == 0) {
                    for (int d = lane; d < s.dk; d += 64) {
                        d_q[(row * s.key_heads + key_head) * s.dk + d] = E::put(0.0f);
                        d_k[(row * s.key_heads + key_head) * s.dk + d] = E::put(0.0f);
                    }
                }
                if (lane == 0) {
                    const int64_t to = row * s.heads + head;
                    if (s.wide_gates) {
                        static_cast<float*>(d_log_gates)[to] = static_cast<float*>(d_beta)[to] = 0.0f;
                    } else {
                        static_cast<ES*>(d_log_gates)[to] = static_cast<ES*>(d_beta)[to] = E::put(0.0f);
                    }
                }
            }
    }
    const BlockAt found = block_at(s, block);
    if (found.length <= 0) return;
    const int64_t row0 = uniform(found.row), entry = block * s.heads + head;
    const int length = __builtin_amdgcn_readfirstlane(found.length);

    const Tile<NI, DK> kt(smem), qt(smem + Tile<NI, DK>::kBytes);
    char* more = smem + 2 * Tile<NI, DK>::kBytes;
    constexpr int kSets = kRowSets<NI, NS, DK>;
    const auto set_of = [&](int group) { return more + (kSets > 1 ? (group & 1) * kRowsBytes<NI, NS> : 0); };
    const auto ot_of = [&](int group) { return Tile<NI, kColumns>(set_of(group)); };
    const auto ut_of = [&](int group) { return Tile<NS, kColumns>(set_of(group) + Tile<NI, kColumns>::kBytes); };
    const auto rt_of = [&](int group) { return Tile<NS, kColumns>(set_of(group) + Tile<NI, kColumns>::kBytes + Tile<NS, kColumns>::kBytes); };
    // the products of tokens take the place of the rows once those are done with
    Exchange<NS, kPairs> f_rows(more), l_rows(more + Exchange<NS, kPairs>::kBytes), f_cols(more + 2 * Exchange<NS, kPairs>::kBytes),
        l_cols(more + 3 * Exchange<NS, kPairs>::kBytes);

    constexpr uint32_t kSize = sizeof(ES);
    const uint32_t k_step = s.key_heads * s.dk * kSize, v_step = s.heads * s.dv * kSize, r_step = s.heads * s.dv * 4;
    const auto rows_of = [&](const void* p, uint32_t step, int64_t at_head, uint32_t bytes) {
        return buffer_of(static_cast<const char*>(p) + row0 * step + at_head, (length - 1) * (int64_t)step + bytes);
    };
    const int feature0 = 16 * (wave & (kFeatures - 1)), tile0 = kFeatures == 8 ? 0 : (wave >> 2) * kTok;  // own features, first own tile of tokens
    const int groups = (s.dv + kColumns - 1) / kColumns;

    // what comes from memory for 64 value columns
    const int64_t cells = (int64_t)s.dk * s.dv;
    const Buffer ob = d_out != nullptr ? rows_of(d_out, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize) : buffer_of(k, 0);
    const Buffer vb = rows_of(v, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize);
    const Buffer ub = rows_of(updates, r_step, (int64_t)head * s.dv * 4, s.dv * 4), rb = rows_of(d_rows, r_step, (int64_t)head * s.dv * 4, s.dv * 4);
    const Buffer sb = buffer_of(states + entry * cells, cells * 4), db = buffer_of(d_states + entry * cells, cells * 4);
    Eight<E> o_raw, v_raw;
    Eight<ElemF32> u_raw, r_raw;
    fx4 s_raw[2][2], d_raw[2][2];
    const uint32_t row_at = (tid >> 3) * v_step + (tid & 7) * 8 * kSize, row_at_r = (tid >> 3) * r_step + (tid & 7) * 32;
    const uint32_t cell_at = (feature0 + c) * (uint32_t)s.dv * 4 + 32 * g;
    const auto load_rows = [&](int group) __attribute__((always_inline)) {
        const bool in = group * kColumns + (tid & 7) * 8 < s.dv;
        const uint32_t from = in ? row_at + group * kColumns * kSize : kOutside, from_r = in ? row_at_r + group * kColumns * 4 : kOutside;
        o_raw = fetch8<E>(ob, from);
        u_raw = fetch8<ElemF32>(ub, from_r);
        r_raw = fetch8<ElemF32>(rb, from_r);
    };
    const auto load_states = [&](int group) __attribute__((always_inline)) {
        const bool in_v = group * kColumns + (tid & 7) * 8 < s.dv;
        v_raw = fetch8<E>(vb, in_v ? row_at + group * kColumns * kSize : kOutside);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = group * kColumns + 32 * i + 8 * g;
            const uint32_t cell = e < s.dv ? cell_at + (group * kColumns + 32 * i) * 4 : kOutside;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s_raw[i][h] = fetch16(sb, cell + 16 * h);
                d_raw[i][h] = fetch16(db, cell + 16 * h);
            }
        }
    };
    const auto stage_rows = [&](int group) __attribute__((always_inline)) {
        ot_of(group).template put8<E>(tid >> 3, (tid & 7) * 8, o_raw);
        ut_of(group).template put8<ElemF32>(tid >> 3, (tid & 7) * 8, u_raw);
        rt_of(group).template put8<ElemF32>(tid >> 3, (tid & 7) * 8, r_raw);
    };

    {
        const int64_t copy = (block * s.key_heads + key_head) * kBlock * DK;
        const Buffer kb = buffer_of(k + copy, kBlock * DK * kSize), qb = buffer_of(q + copy, kBlock * DK * kSize);
        const Buffer gb = buffer_of(gates + entry * kGateFloats, kGateFloats * 4);
        Eight<E> k_raw[DK / 64], q_raw[DK / 64];
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) {
            k_raw[i] = fetch8<E>(kb, (tid + 512 * i) * 8 * kSize);
            q_raw[i] = fetch8<E>(qb, (tid + 512 * i) * 8 * kSize);
        }
        const float gate_raw = fetch4(gb, tid * 4);
        load_rows(0);
        load_states(0);
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) {
            const int row = (tid + 512 * i) / (DK / 8), d = (tid + 512 * i) % (DK / 8) * 8;
            kt.template put8<E>(row, d, k_raw[i]);
            qt.template put8<E>(row, d, q_raw[i]);
        }
        if (tid < kGateFloats) gate[tid] = gate_raw;
    }

    fx4 x[kTok], a[kTok], b[kTok];  // dQ, A and B: own features (rows), own tokens (columns)
    float value_dot = 0.0f, whole_term = 0.0f;
#pragma unroll
    for (int t = 0; t < kTok; ++t) x[t] = a[t] = b[t] = fx4{0, 0, 0, 0};
#pragma unroll 1
    for (int group = 0; group < groups; ++group) {
        if (kSets == 1 && group > 0) lds_barrier();  // (of two sets the last readers are behind the other's barrier)
        stage_rows(group);
#pragma unroll
        for (int i = 0; i < 8; ++i) value_dot += r_raw.v[i] * E::get(v_raw.v[i]);
        Operand<NS> so[2], dd[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            so[i] = operand_of<NS>(s_raw[i][0], s_raw[i][1]);
            dd[i] = operand_of<NS>(d_raw[i][0], d_raw[i][1]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) whole_term += s_raw[i][h][e] * d_raw[i][h][e];
        }
        lds_barrier();
        // (behind the last group the one that the products of tokens load first, or one that is not there)
        load_rows(group + 1 < groups ? group + 1 : (groups > kSets ? groups - 1 - kSets : groups));
        if (group + 1 < groups) load_states(group + 1);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < kTok; ++t) {
                const int row = 16 * (tile0 + t) + c;
                x[t] = mma<NS, NI>(so[i], ot_of(group).along(row, 32 * i, g), x[t]);
                a[t] = mma<NS, NS>(so[i], rt_of(group).along(row, 32 * i, g), a[t]);
                b[t] = mma<NS, NS>(dd[i], ut_of(group).along(row, 32 * i, g), b[t]);
            }
    }
    // Tokens against tokens, from the last group of columns back: tile `own` against all in dO U^T (waves 0 to 3) or
    // dR U^T (4 to 7), with the own tokens as columns and earlier ones as rows, and with the own tokens as columns,
    // where the other factor is U, and later ones as rows.
    const int own = wave & 3;
    const bool second = wave >= 4;
    fx4 early[kTiles], late[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) early[t] = late[t] = fx4{0, 0, 0, 0};
#pragma unroll 1
    for (int group = groups - 1; group >= 0; --group) {
        if (group < groups - kSets) {
            lds_barrier();
            stage_rows(group);
            lds_barrier();
            load_rows(group > 0 ? group - 1 : groups);
        }
        const Tile<NI, kColumns> ot = ot_of(group);
        const Tile<NS, kColumns> ut = ut_of(group), rt = rt_of(group);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Operand<NS> u = ut.along(16 * own + c, 32 * i, g);
            if (!second) {
                const Operand<NI> o = ot.along(16 * own + c, 32 * i, g);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    if (t <= own) early[t] = mma<NS, NI>(ut.along(16 * t + c, 32 * i, g), o, early[t]);
                    if (t >= own) {
                        late[t] = mma<NI, NS>(ot.along(16 * t + c, 32 * i, g), u, late[t]);
                        asm volatile("s_nop 1" : "+v"(late[t]));  // (behind the branches that follow the compiler waits too little)
                    }
                }
            } else {
                const Operand<NS> r = rt.along(16 * own + c, 32 * i, g);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    if (t <= own) early[t] = mma<NS, NS>(ut.along(16 * t + c, 32 * i, g), r, early[t]);
                    if (t >= own) {
                        late[t] = mma<NS, NS>(rt.along(16 * t + c, 32 * i, g), u, late[t]);
                        asm volatile("s_nop 1" : "+v"(late[t]));
                    }
                }
            }
        }
    }

    // No load of this block is left to come.  What the workgroup that follows on this die wants first is asked for
    // meanwhile: its states' first 64 columns, and keys and queries, which it finds in the second cache then.
    int touched[2] = {0, 0};
    {
        const int64_t follow = (int64_t)blockIdx.y * gridDim.x + blockIdx.x + kAhead;
        const int64_t its_head = follow / gridDim.x, its_block = follow % gridDim.x;
        if (its_head < s.heads) {
            const int64_t its = its_block * s.heads + its_head;
            const char* from = reinterpret_cast<const char*>((tid < 256 ? states : d_states) + its * cells);
            const int row = (tid & 255) >> 1, at = (tid & 1) * 128;
            if (row < s.dk && at < s.dv * 4) touched[0] = *reinterpret_cast<const int*>(from + (int64_t)row * s.dv * 4 + at);
            constexpr int kLines = kBlock * DK * kSize / 128;
            const int64_t copy = (its_block * s.key_heads + its_head / share) * kBlock * DK;
            if (tid < 2 * kLines)
                touched[1] = *reinterpret_cast<const int*>(reinterpret_cast<const char*>((tid < kLines ? k : q) + copy) + tid % kLines * 128);
        }
    }

    // weighted, the products of tokens go to all waves
    lds_barrier();
    {
        const int here = 16 * own + c;
        const float high = gate[kSumHigh * kBlock + here], low = gate[kSumLow * kBlock + here];
        Exchange<NS, kPairs> rows = second ? l_rows : f_rows, cols = second ? l_cols : f_cols;
        const float factor = second ? -1.0f : s.scale;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int there0 = 16 * t + 4 * g;
            const fx4 h = *reinterpret_cast<const fx4*>(gate + kSumHigh * kBlock + there0);
            const fx4 l = *reinterpret_cast<const fx4*>(gate + kSumLow * kBlock + there0);
            if (t <= (own | 1)) {
                fx4 e = {0, 0, 0, 0};
                if (t <= own) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float w = factor * exp_of((high - h[r]) + (low - l[r]));
                        e[r] = there0 + r < here ? w * early[t][r] : 0.0f;
                        if (!second && there0 + r == here) diagonal[here] = w * early[t][r];
                    }
                }
                rows.put(2 * pair_lower(own, t >> 1) + (t & 1), lane, e);
            }
            if (t >= (own & 2)) {
                fx4 e = {0, 0, 0, 0};
                if (t >= own) {
                    const fx4 beta = *reinterpret_cast<const fx4*>(gate + kBeta * kBlock + there0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float w = factor * (second ? beta[r] : 1.0f) * exp_of((h[r] - high) + (l[r] - low));
                        e[r] = there0 + r > here ? w * late[t][r] : 0.0f;
                    }
                }
                cols.put(2 * pair_upper(own, t >> 1) + (t & 1), lane, e);
            }
        }
    }
    lds_barrier();
    Operand<NI> ko[2], qo[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        ko[p] = kt.down(32 * p, feature0, lane);
        qo[p] = qt.down(32 * p, feature0, lane);
    }
    const uint32_t to0 = feature0 + 4 * g < s.dk ? (16 * tile0 + c) * k_step + (feature0 + 4 * g) * kSize : kOutside;
    const Buffer qb = rows_of(d_q, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
    const Buffer kb = rows_of(d_k, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
    float* const mine = sums + ((entry * 16 + wave) * kTok * 64 + lane) * 4;  // dK's half is 8 waves on
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
        const int tile = tile0 + t, token = 16 * tile + c;
        // factors of the parts that went through the state
        const float since = gate[kSince * kBlock + token], until = gate[kUntil * kBlock + token], beta = gate[kBeta * kBlock + token];
        const fx4 kv = kt.quad(token, feature0 + 4 * g), qv = qt.quad(token, feature0 + 4 * g);
        float sums_of[kSums] = {0, 0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[t][r] *= s.scale * since;
            a[t][r] *= -since;
            b[t][r] *= until;
            sums_of[kFromState] += qv[r] * x[t][r] + beta * (kv[r] * a[t][r]);
            sums_of[kToState] += kv[r] * b[t][r];
        }
        fx4 xi = {0, 0, 0, 0}, ai = {0, 0, 0, 0}, bi = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            if (p <= (tile >> 1)) {
                xi = mma<NI, NS>(ko[p], f_rows.get(pair_lower(tile, p), lane), xi);
                ai = mma<NI, NS>(ko[p], l_rows.get(pair_lower(tile, p), lane), ai);
            }
            if (p >= (tile >> 1)) {
                bi = mma<NI, NS>(qo[p], f_cols.get(pair_upper(tile, p), lane), bi);
                bi = mma<NI, NS>(ko[p], l_cols.get(pair_upper(tile, p), lane), bi);
            }
        }
        const float with_itself = diagonal[token];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            sums_of[kEarlier] += qv[r] * xi[r] + beta * (kv[r] * ai[r]);
            sums_of[kLater] += kv[r] * bi[r];
            a[t][r] += ai[r];
            sums_of[kBetas] += kv[r] * a[t][r];
            x[t][r] += xi[r] + with_itself * kv[r];
            b[t][r] += bi[r] + with_itself * qv[r] + beta * a[t][r];  // dK
        }
#pragma unroll
        for (int i = 0; i < kSums; ++i) {
            sums_of[i] += __shfl_xor(sums_of[i], 16);
            sums_of[i] += __shfl_xor(sums_of[i], 32);
            if (g == 0) dots[wave][i][16 * t + c] = sums_of[i];
        }
        if constexpr (SHARED) {
            *reinterpret_cast<fx4*>(mine + t * 256) = x[t];
            *reinterpret_cast<fx4*>(mine + (8 * kTok + t) * 256) = b[t];
        } else {
            put4<E>(qb, to0 + 16 * t * k_step, x[t]);
            put4<E>(kb, to0 + 16 * t * k_step, b[t]);
        }
    }
    asm volatile("" ::"v"(touched[0]), "v"(touched[1]));  // (keeps the two loads in the program)
    whole_term = tile0 == 0 ? whole_term * gate[kSince * kBlock + kBlock - 1] : 0.0f;  // a cell counts once
    whole_term = sum16(whole_term);
    whole_term += __shfl_xor(whole_term, 16);
    whole_term += __shfl_xor(whole_term, 32);
    if (lane == 0) whole_terms[wave] = whole_term;
    value_dot += __shfl_xor(value_dot, 1);
    value_dot += __shfl_xor(value_dot, 2);
    value_dot += __shfl_xor(value_dot, 4);
    if ((tid & 7) == 0) value_dots[tid >> 3] = value_dot;
    lds_barrier();
    if (wave == 0) {
        // token `lane`: over the tiles of features, then over tokens
        float sum[kSums] = {0, 0, 0, 0, 0}, whole = 0.0f;
#pragma unroll
        for (int i = 0; i < kFeatures; ++i) {
            const int w = lane / (16 * kTok) * kFeatures + i;
#pragma unroll
            for (int n = 0; n < kSums; ++n) sum[n] += dots[w][n][lane % (16 * kTok)];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) whole += whole_terms[i];
        const bool front = lane < (length + 1) / 2;
        float from = sum[kFromState], to_state = sum[kToState], pairs = front ? sum[kLater] - sum[kEarlier] : sum[kEarlier] - sum[kLater];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const float x1 = __shfl_down(from, d), x2 = __shfl_up(to_state, d), x3 = __shfl(pairs, (front ? lane - d : lane + d) & 63);
            if (lane + d < 64) from += x1;
            if (lane >= d) to_state += x2;
            if (front ? lane >= d : lane + d < 64) pairs += x3;
        }
        to_state = __shfl_up(to_state, 1);
        const float before = __shfl_up(pairs, 1);
        if (front) pairs = lane > 0 ? before : 0.0f;
        const float dc = from + pairs + whole + (lane > 0 ? to_state : 0.0f), da = sum[kBetas];
        if (lane < length) {
            const int64_t to = (row0 + lane) * s.heads + head;
            if (s.wide_gates) {
                static_cast<float*>(d_log_gates)[to] = dc;
                static_cast<float*>(d_beta)[to] = value_dots[lane] + da;
            } else {
                static_cast<ES*>(d_log_gates)[to] = E::put(dc);
                static_cast<ES*>(d_beta)[to] = E::put(value_dots[lane] + da);
            }
        }
    }
}

// dQ and dK of a block and key head: the sums of the heads that share it, in their order.
// grid (blocks, key heads), 512 threads, which hold what the ones of delta_gradients do.
template <class E, int DK>
__global__ __launch_bounds__(512) void delta_fold(DeltaShape s, const float* __restrict__ sums,
                                                  typename E::S* __restrict__ d_q, typename E::S* __restrict__ d_k) {
    constexpr int kFeatures = DK / 16, kTok = DK / 32;
    const int64_t block = blockIdx.x;
    const int key_head = blockIdx.y, share = s.heads / s.key_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const BlockAt found = block_at(s, block);
    if (found.length <= 0) return;
    const int feature = 16 * (wave & (kFeatures - 1)) + 4 * g, tile0 = kFeatures == 8 ? 0 : (wave >> 2) * kTok;
    const float* from = sums + (((block * s.heads + key_head * share) * 16 + wave) * kTok * 64 + lane) * 4;
    fx4 x[kTok], b[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) x[t] = b[t] = fx4{0, 0, 0, 0};
    for (int h = 0; h < share; ++h, from += 16 * kTok * 256) {
#pragma unroll
        for (int t = 0; t < kTok; ++t) {
            x[t] += *reinterpret_cast<const fx4*>(from + t * 256);
            b[t] += *reinterpret_cast<const fx4*>(from + (8 * kTok + t) * 256);
        }
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
        const int row = 16 * (tile0 + t) + c;
        if (row < found.length && feature < s.dk) {
            const int64_t to = ((found.row + row) * s.key_heads + key_head) * s.dk + feature;
            store4<E>(d_q + to, x[t]);
            store4<E>(d_k + to, b[t]);
        }
    }
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_BACKWARD_H_
