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
//   dc[i] = q[i].dQ[i] + beta[i] k[i].A[i] - k[i].B[i],  and c[63] also gets e^c[63] S0.D1 + sum over i of
//           k[i].(diag(e^(c[63]-c)) U D1^T)[i];  the gradient of a log gate sums dc from its token on
#ifndef ASCAN_DELTA_BACKWARD_H_
#define ASCAN_DELTA_BACKWARD_H_

#include "delta_forward.h"

namespace ascan {
namespace {

constexpr int kColumns = 64;  // value columns that a workgroup of delta_gradients takes at a time

template <int NI, int NS, int DK>
constexpr int kReverseBytes = 3 * Tile<NI, DK>::kBytes + Tile<NI, 16>::kBytes + Exchange<NS, DK / 32>::kBytes +
                              3 * Exchange<NS, 2>::kBytes;

// The chain, last block first, divided like the forward one: 16 columns of D to a workgroup, wave w keeps rows
// dk/4 w .. of them and computes tokens 16w .. 16w+15; D, dU and -diag(beta e^c) dR go round through LDS.
// grid chain_grid(), 256 threads.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(256) void delta_reverse_chain(
    DeltaShape s, const typename E::S* __restrict__ q, const typename E::S* __restrict__ k,
    const typename E::S* __restrict__ d_out, const float* __restrict__ gates, const char* __restrict__ t_in,
    const char* __restrict__ p_in, const float* __restrict__ d_final, typename E::S* __restrict__ d_v,
    float* __restrict__ d_initial, float* __restrict__ d_states, float* __restrict__ d_rows) {
    using ES = typename E::S;
    constexpr int kDepths = DK / 32, kOwn = DK / 64, kCopies = DK / 32;
    extern __shared__ __align__(16) char smem[];
    const ChainAt where = chain_at(s);
    if (!where.there) return;
    const int64_t n = where.sequence;
    const int head = where.head, key_head = head / (s.heads / s.key_heads);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int col0 = where.col0, col = col0 + c;
    const bool mine = col < s.dv;
    const SequenceAt at = sequence_at(s, n);

    // (queries are read between the second and the third barrier only: one tile is enough)
    char* m = smem + 2 * Tile<NI, DK>::kBytes;
    const Tile<NI, DK> qt(m);
    m += Tile<NI, DK>::kBytes;
    const Tile<NI, 16> ot(m);
    m += Tile<NI, 16>::kBytes;
    Exchange<NS, kDepths> xs(m);
    m += Exchange<NS, kDepths>::kBytes;
    Exchange<NS, 2> xr(m), xw(m + Exchange<NS, 2>::kBytes), xu(m + 2 * Exchange<NS, 2>::kBytes);

    fx4 D[kOwn];
    const int64_t state_at = (n * s.heads + head) * s.dk * s.dv + col;
#pragma unroll
    for (int t = 0; t < kOwn; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = feature_row(kOwn * wave + t, g, r);
            D[t][r] = d_final != nullptr && mine && row < s.dk ? d_final[state_at + (int64_t)row * s.dv] : 0.0f;
        }

    constexpr uint32_t kSize = sizeof(ES);
    const uint32_t k_step = s.key_heads * s.dk * kSize, v_step = s.heads * s.dv * kSize, r_step = s.heads * s.dv * 4;
    const int64_t seq_row = uniform(at.row), seq_length = uniform(at.length), seq_block = uniform(at.block);
    const int token = 16 * wave + c;
    const auto rows_of = [&](const void* p, int64_t first, uint32_t step, int64_t at_head, uint32_t bytes) {
        const int64_t left = seq_length - first < kBlock ? seq_length - first : kBlock;
        return buffer_of(static_cast<const char*>(p) + (seq_row + first) * step + at_head, (left - 1) * (int64_t)step + bytes);
    };
    const auto entry_of = [&](int64_t first) { return (seq_block + first / kBlock) * s.heads + head; };
    Eight<E> k_raw[kCopies], q_raw[kCopies], o_raw;
    Operand<NS> tm[2], pm[2];
    fx4 beta, beta_since, until, since;
    float whole;
    const auto load_rows = [&](int64_t first) {
        const Buffer kb = rows_of(k, first, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
        const Buffer qb = rows_of(q, first, k_step, (int64_t)key_head * s.dk * kSize, s.dk * kSize);
        const Buffer ob = d_out != nullptr ? rows_of(d_out, first, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize) : buffer_of(k, 0);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
            k_raw[i] = fetch8<E>(kb, d < s.dk ? row * k_step + d * kSize : kOutside);
            q_raw[i] = fetch8<E>(qb, d < s.dk ? row * k_step + d * kSize : kOutside);
        }
        const int d = col0 + (tid & 1) * 8;  // (the upper two waves repeat what the lower two do)
        o_raw = fetch8<E>(ob, d < s.dv ? ((tid & 127) >> 1) * v_step + d * kSize : kOutside);
    };
    // (waves 2 and 3 have one operand to a row of tiles: their first load repeats the second)
    const auto load_matrix = [&](const char* from, int64_t first, Operand<NS>(&o)[2]) {
        const Buffer b = buffer_of(from + entry_of(first) * kMatrixBytes<NS>, kMatrixBytes<NS>);
        o[0] = matrix_operand<NS>(b, pair_upper(wave, wave < 2 ? 0 : 1), lane);
        o[1] = matrix_operand<NS>(b, pair_upper(wave, 1), lane);
    };
    const auto gates_of = [&](int64_t first) { return buffer_of(gates + entry_of(first) * kGateFloats, kGateFloats * 4); };
    const uint32_t gate_rows = (16 * wave + 4 * g) * 4;

    const int64_t last = (seq_length - 1) / kBlock * kBlock;
    if (seq_length > 0) {  // (an empty sequence has no table entry to read)
        load_rows(last);
        load_matrix(p_in, last, pm);
        const Buffer b = gates_of(last);
        until = fetch16(b, kUntil * 256 + gate_rows);
        since = fetch16(b, kSince * 256 + gate_rows);
        load_matrix(t_in, last, tm);
        beta = fetch16(b, kBeta * 256 + gate_rows);
        beta_since = fetch16(b, kBetaSince * 256 + gate_rows);
        whole = fetch4(b, kSince * 256 + (c | 63) * 4);
    }
    for (int64_t first = last; first >= 0 && seq_length > 0; first -= kBlock) {
        const int64_t ahead = first > 0 ? first - kBlock : 0;
        const Buffer gb = gates_of(ahead);
        const Tile<NI, DK> kb(smem + ((first / kBlock) & 1) * Tile<NI, DK>::kBytes);
        {
            const Buffer to = buffer_of(d_states + entry_of(first) * s.dk * s.dv, (int64_t)s.dk * s.dv * 4);
#pragma unroll
            for (int t = 0; t < kOwn; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    put1<ElemF32>(to, mine ? (feature_row(kOwn * wave + t, g, r) * s.dv + col) * 4 : kOutside, D[t][r]);
        }
#pragma unroll
        for (int t = 0; t < kOwn; ++t) xs.put(kOwn * wave + t, lane, D[t]);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
            kb.template put8<E>(row, d, k_raw[i]);
            qt.template put8<E>(row, d, q_raw[i]);
        }
        ot.template put8<E>((tid & 127) >> 1, (tid & 1) * 8, o_raw);
        lds_barrier();

        // dU = diag(e^(c[63]-c)) K D1 + P^T dO
        fx4 u = {0, 0, 0, 0}, w;
        {
            Operand<NS> so[kDepths];
            Operand<NI> ko[kDepths];
#pragma unroll
            for (int d = 0; d < kDepths; ++d) {
                so[d] = xs.get(d, lane);
                ko[d] = kb.along(token, 32 * d, g);
            }
            const Operand<NI> o_low = ot.down(0, 0, lane), o_high = ot.down(32, 0, lane);
            w = ot.tile(16 * wave, 0, lane);
            load_rows(ahead);
            __builtin_amdgcn_sched_barrier(0);  // all reads on their way before the first product waits for one
            fx4 po = {0, 0, 0, 0};
            if (wave < 2) po = mma<NS, NI>(pm[0], o_low, po);
            po = mma<NS, NI>(pm[1], o_high, po);
#pragma unroll
            for (int d = 0; d < kDepths; ++d) u = mma<NI, NS>(ko[d], so[d], u);
            load_matrix(p_in, ahead, pm);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u[r] = until[r] * u[r] + po[r];
                w[r] *= s.scale * since[r];
            }
        }
        xr.put(wave, lane, u);
        xw.put(wave, lane, w);
        until = fetch16(gb, kUntil * 256 + gate_rows);
        since = fetch16(gb, kSince * 256 + gate_rows);
        lds_barrier();

        // dR = dU + T^T dU;  D0 = e^c[63] D1 + Q^T diag(scale e^c) dO while it waits
        fx4 x;
        {
            const Operand<NS> low = xr.get(0, lane), high = xr.get(1, lane), w_low = xw.get(0, lane), w_high = xw.get(1, lane);
            Operand<NI> q_low[kOwn], q_high[kOwn];
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
                q_low[t] = qt.down_features(0, kOwn * wave + t, lane);
                q_high[t] = qt.down_features(32, kOwn * wave + t, lane);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (wave < 2) u = mma<NS, NS>(tm[0], low, u);
            u = mma<NS, NS>(tm[1], high, u);
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) D[t][r] *= whole;
                D[t] = mma<NI, NS>(q_low[t], w_low, D[t]);
                D[t] = mma<NI, NS>(q_high[t], w_high, D[t]);
            }
        }
        load_matrix(t_in, ahead, tm);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = -beta_since[r] * u[r];
        xu.put(wave, lane, x);
        beta_since = fetch16(gb, kBetaSince * 256 + gate_rows);
        whole = fetch4(gb, kSince * 256 + (c | 63) * 4);
        lds_barrier();

        // D0 -= K^T diag(beta e^c) dR
        {
            const Operand<NS> low = xu.get(0, lane), high = xu.get(1, lane);
            Operand<NI> k_low[kOwn], k_high[kOwn];
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
                k_low[t] = kb.down_features(0, kOwn * wave + t, lane);
                k_high[t] = kb.down_features(32, kOwn * wave + t, lane);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
                D[t] = mma<NI, NS>(k_low[t], low, D[t]);
                D[t] = mma<NI, NS>(k_high[t], high, D[t]);
            }
        }
        {
            const Buffer to = rows_of(d_v, first, v_step, (int64_t)head * s.dv * kSize, s.dv * kSize);
            const Buffer rows = rows_of(d_rows, first, r_step, (int64_t)head * s.dv * 4, s.dv * 4);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                put1<E>(to, mine ? (16 * wave + 4 * g + r) * v_step + col * kSize : kOutside, beta[r] * u[r]);
                put1<ElemF32>(rows, mine ? (16 * wave + 4 * g + r) * r_step + col * 4 : kOutside, u[r]);
            }
        }
        beta = fetch16(gb, kBeta * 256 + gate_rows);
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
    if (s.offsets != nullptr && mine) {
        const int own = 4 * wave + g;
        if (n == 0)
            for (int64_t row = own; row < offset_at(s, 0); row += 16) d_v[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
        if (n == s.sequences - 1)
            for (int64_t row = offset_at(s, s.sequences) + own; row < s.rows; row += 16)
                d_v[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
    }
}

// Operand of 32 columns of a row-major fp32 matrix in memory: row `row`, columns col .. col + 31 below `cols`.
template <int P>
__device__ __forceinline__ Operand<P> memory_operand(const float* p, int64_t stride, int row, int rows, int col,
                                                     int cols, int g, fx4 (&raw)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int d = col + 8 * g + 4 * h;
        raw[h] = fx4{0, 0, 0, 0};
        if (row < rows && d < cols) raw[h] = *reinterpret_cast<const fx4*>(p + row * stride + d);
    }
    return operand_of<P>(raw[0], raw[1]);
}

template <int NI, int NS, int DK>
constexpr int kGradientBytes = 2 * Tile<NI, DK>::kBytes + Tile<NI, kColumns>::kBytes + 2 * Tile<NS, kColumns>::kBytes;

// A block of one key head and all value heads that share it; a wave owns 16 of the tokens.
// grid (blocks, key heads), 256 threads.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(256) void delta_gradients(
    DeltaShape s, const typename E::S* __restrict__ q, const typename E::S* __restrict__ k,
    const typename E::S* __restrict__ v, const typename E::S* __restrict__ d_out, const float* __restrict__ gates,
    const float* __restrict__ states, const float* __restrict__ updates, const float* __restrict__ d_states,
    const float* __restrict__ d_rows, typename E::S* __restrict__ d_q, typename E::S* __restrict__ d_k,
    void* __restrict__ d_log_gates, void* __restrict__ d_beta) {
    extern __shared__ __align__(16) char smem[];
    __shared__ __align__(16) float gate[kGateFloats];
    __shared__ float dc[kBlock], db[kBlock], whole_terms[4];
    const int64_t block = blockIdx.x;
    const int key_head = blockIdx.y, share = s.heads / s.key_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;

    // rows in front of the first and behind the last sequence: zero gradients, 64 rows to a workgroup
    if (s.offsets != nullptr) {
        const int64_t before = offset_at(s, 0), behind = offset_at(s, s.sequences);
        const int64_t spans[2][2] = {{0, before}, {behind, s.rows}};
        for (int i = 0; i < 2; ++i)
            for (int64_t row = spans[i][0] + block * kBlock + wave; row < spans[i][1] && row < spans[i][0] + (block + 1) * kBlock;
                 row += 4) {
                for (int d = lane; d < s.dk; d += 64) {
                    d_q[(row * s.key_heads + key_head) * s.dk + d] = E::put(0.0f);
                    d_k[(row * s.key_heads + key_head) * s.dk + d] = E::put(0.0f);
                }
                for (int h = lane; h < share; h += 64) {
                    const int64_t to = row * s.heads + key_head * share + h;
                    if (s.wide_gates) {
                        static_cast<float*>(d_log_gates)[to] = static_cast<float*>(d_beta)[to] = 0.0f;
                    } else {
                        static_cast<typename E::S*>(d_log_gates)[to] = static_cast<typename E::S*>(d_beta)[to] = E::put(0.0f);
                    }
                }
            }
    }
    const BlockAt at = block_at(s, block);
    if (at.length <= 0) return;

    Tile<NI, DK> kt(smem), qt(smem + Tile<NI, DK>::kBytes);
    char* more = smem + 2 * Tile<NI, DK>::kBytes;
    Tile<NI, kColumns> ot(more);
    Tile<NS, kColumns> ut(more + Tile<NI, kColumns>::kBytes);
    Tile<NS, kColumns> rt(more + Tile<NI, kColumns>::kBytes + Tile<NS, kColumns>::kBytes);

    for (int i = tid; i < kBlock * DK / 8; i += 256) {
        const int row = i / (DK / 8), d = i % (DK / 8) * 8;
        const bool there = row < at.length && d < s.dk;
        const int64_t from = ((at.row + row) * s.key_heads + key_head) * s.dk + d;
        kt.template put8<E>(row, d, load8<E>(k + from, there));
        qt.template put8<E>(row, d, load8<E>(q + from, there));
    }

    fx4 q_sum[DK / 16], k_sum[DK / 16];
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) q_sum[t] = k_sum[t] = fx4{0, 0, 0, 0};

    for (int h = 0; h < share; ++h) {
        const int head = key_head * share + h;
        const int64_t entry = block * s.heads + head;
        __syncthreads();
        for (int i = tid; i < kGateFloats; i += 256) gate[i] = gates[entry * kGateFloats + i];
        fx4 x[DK / 16], a[DK / 16], b[DK / 16];  // dQ, A and B of this head
        // dO U^T and dR U^T: with the wave's tokens as columns (rows: earlier tokens) and as columns of later rows
        fx4 oc[kTiles], rc[kTiles], orow[kTiles], rrow[kTiles];
        fx4 rv = {0, 0, 0, 0};
        float whole_term = 0.0f;
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) x[t] = a[t] = b[t] = fx4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < kTiles; ++t) oc[t] = rc[t] = orow[t] = rrow[t] = fx4{0, 0, 0, 0};

        for (int col0 = 0; col0 < s.dv; col0 += kColumns) {
            __syncthreads();
            for (int i = tid; i < kBlock * kColumns / 8; i += 256) {
                const int row = i / (kColumns / 8), d = i % (kColumns / 8) * 8;
                const bool there = row < at.length && col0 + d < s.dv;
                const int64_t from = ((at.row + row) * s.heads + head) * s.dv + col0 + d;
                ot.template put8<E>(row, d, load8<E>(d_out + from, there && d_out != nullptr));
                ut.template put8<ElemF32>(row, d, load8<ElemF32>(updates + from, there));
                rt.template put8<ElemF32>(row, d, load8<ElemF32>(d_rows + from, there));
            }
            __syncthreads();
            // dR . v of the wave's tokens: a token to a row of the accumulator, four columns to a lane
            {
                const int row = 16 * wave + c;
                float sum = 0.0f;
                if (row < at.length) {
                    const int64_t from = ((at.row + row) * s.heads + head) * s.dv + col0;
#pragma unroll
                    for (int d = 4 * g; d < kColumns; d += 16)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (col0 + d < s.dv) sum += d_rows[from + d + r] * E::get(v[from + d + r]);
                }
                rv[0] += sum;
            }
#pragma unroll
            for (int d = 0; d < kColumns; d += 32) {
                const Operand<NI> o = ot.along(16 * wave + c, d, g);
                const Operand<NS> u = ut.along(16 * wave + c, d, g), r = rt.along(16 * wave + c, d, g);
#pragma unroll
                for (int t = 0; t < DK / 16; ++t) {
                    fx4 raw_s[2], raw_d[2];
                    const Operand<NS> so = memory_operand<NS>(states + entry * s.dk * s.dv, s.dv, 16 * t + c, s.dk, col0 + d, s.dv, g, raw_s);
                    const Operand<NS> dd = memory_operand<NS>(d_states + entry * s.dk * s.dv, s.dv, 16 * t + c, s.dk, col0 + d, s.dv, g, raw_d);
                    x[t] = mma<NI, NS>(o, so, x[t]);
                    a[t] = mma<NS, NS>(r, so, a[t]);
                    b[t] = mma<NS, NS>(u, dd, b[t]);
                    if (t % 4 == wave) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) whole_term += raw_s[i][e] * raw_d[i][e];
                    }
                }
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    if (t <= wave) {
                        const Operand<NS> e = ut.along(16 * t + c, d, g);
                        oc[t] = mma<NS, NI>(e, o, oc[t]);
                        rc[t] = mma<NS, NS>(e, r, rc[t]);
                    }
                    if (t >= wave) {
                        orow[t] = mma<NI, NS>(ot.along(16 * t + c, d, g), u, orow[t]);
                        rrow[t] = mma<NS, NS>(rt.along(16 * t + c, d, g), u, rrow[t]);
                    }
                }
            }
        }

        // factors of the parts that went through the state
        const fx4 since = *reinterpret_cast<const fx4*>(gate + kSince * kBlock + 16 * wave + 4 * g);
        const fx4 until = *reinterpret_cast<const fx4*>(gate + kUntil * kBlock + 16 * wave + 4 * g);
        const fx4 beta = *reinterpret_cast<const fx4*>(gate + kBeta * kBlock + 16 * wave + 4 * g);
        fx4 carried = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            const fx4 kv = kt.tile(16 * wave, 16 * t, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[t][r] *= s.scale * since[r];
                a[t][r] *= -since[r];
                b[t][r] *= until[r];
                carried[r] += kv[r] * b[t][r];
            }
        }
        whole_term *= gate[kSince * kBlock + kBlock - 1];
#pragma unroll
        for (int r = 0; r < 4; ++r) whole_term += carried[r];

        // weights of pairs of tokens inside the block
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int there = 16 * t + 4 * g + r, here = 16 * wave + c;
                const float high = gate[kSumHigh * kBlock + here] - gate[kSumHigh * kBlock + there];
                const float low = gate[kSumLow * kBlock + here] - gate[kSumLow * kBlock + there];
                const float ec = there <= here ? expf(high + low) : 0.0f;    // `there` earlier than the wave's token
                const float er = there >= here ? expf(-(high + low)) : 0.0f; // `there` later
                oc[t][r] = there <= here ? s.scale * ec * oc[t][r] : 0.0f;
                rc[t][r] = there < here ? -ec * rc[t][r] : 0.0f;
                orow[t][r] = there >= here ? s.scale * er * orow[t][r] : 0.0f;
                rrow[t][r] = there > here ? -gate[kBeta * kBlock + there] * er * rrow[t][r] : 0.0f;
            }
        }
        fx4 dots_q = {0, 0, 0, 0}, dots_a = {0, 0, 0, 0}, dots_b = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const Operand<NS> o1 = operand_of<NS>(oc[2 * p], oc[2 * p + 1]), r1 = operand_of<NS>(rc[2 * p], rc[2 * p + 1]);
            const Operand<NS> o2 = operand_of<NS>(orow[2 * p], orow[2 * p + 1]), r2 = operand_of<NS>(rrow[2 * p], rrow[2 * p + 1]);
#pragma unroll
            for (int t = 0; t < DK / 16; ++t) {
                const Operand<NI> ko = kt.down(32 * p, 16 * t, lane), qo = qt.down(32 * p, 16 * t, lane);
                x[t] = mma<NS, NI>(o1, ko, x[t]);
                a[t] = mma<NS, NI>(r1, ko, a[t]);
                b[t] = mma<NS, NI>(o2, qo, b[t]);
                b[t] = mma<NS, NI>(r2, ko, b[t]);
            }
        }
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            const fx4 kv = kt.tile(16 * wave, 16 * t, lane), qv = qt.tile(16 * wave, 16 * t, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                dots_q[r] += qv[r] * x[t][r];
                dots_a[r] += kv[r] * a[t][r];
                dots_b[r] += kv[r] * b[t][r];
                q_sum[t][r] += x[t][r];
                k_sum[t][r] += beta[r] * a[t][r] + b[t][r];
            }
        }
        const float dot_v = rv[0] + __shfl_xor(rv[0], 16);
        const float token_v = dot_v + __shfl_xor(dot_v, 32);  // of token 16 wave + lane % 16
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float dq = sum16(dots_q[r]), da = sum16(dots_a[r]), dbb = sum16(dots_b[r]);
            const float vr = __shfl(token_v, 4 * g + r);
            if (c == 0) {
                dc[16 * wave + 4 * g + r] = dq + beta[r] * da - dbb;
                db[16 * wave + 4 * g + r] = vr + da;
            }
        }
        whole_term = sum16(whole_term);
        whole_term += __shfl_xor(whole_term, 16);
        whole_term += __shfl_xor(whole_term, 32);
        if (lane == 0) whole_terms[wave] = whole_term;
        __syncthreads();
        if (wave == 0) {
            float sum = dc[lane];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const float y = __shfl_down(sum, d);
                if (lane + d < 64) sum += y;
            }
            sum += whole_terms[0] + whole_terms[1] + whole_terms[2] + whole_terms[3];
            if (lane < at.length) {
                const int64_t to = (at.row + lane) * s.heads + head;
                if (s.wide_gates) {
                    static_cast<float*>(d_log_gates)[to] = sum;
                    static_cast<float*>(d_beta)[to] = db[lane];
                } else {
                    static_cast<typename E::S*>(d_log_gates)[to] = E::put(sum);
                    static_cast<typename E::S*>(d_beta)[to] = E::put(db[lane]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * wave + 4 * g + r, d = 16 * t + c;
            if (row < at.length && d < s.dk) {
                const int64_t to = ((at.row + row) * s.key_heads + key_head) * s.dk + d;
                d_q[to] = E::put(q_sum[t][r]);
                d_k[to] = E::put(k_sum[t][r]);
            }
        }
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_BACKWARD_H_
