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

constexpr int kColumns = 64;  // value columns that a workgroup takes at a time

template <int NI, int DK>
constexpr int kReverseBytes = 2 * Tile<NI, DK>::kBytes + Tile<NI, kColumns>::kBytes;

// The chain, last block first: 16 columns of D stay in a wave's accumulators.
// grid (column groups, heads, sequences), 256 threads.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(256) void delta_reverse_chain(
    DeltaShape s, const typename E::S* __restrict__ q, const typename E::S* __restrict__ k,
    const typename E::S* __restrict__ d_out, const float* __restrict__ gates, const char* __restrict__ t_in,
    const char* __restrict__ p_in, const float* __restrict__ d_final, typename E::S* __restrict__ d_v,
    float* __restrict__ d_initial, float* __restrict__ d_states, float* __restrict__ d_rows) {
    extern __shared__ __align__(16) char smem[];
    __shared__ __align__(16) float gate[4 * kBlock];
    const int64_t n = blockIdx.z;
    const int head = blockIdx.y, key_head = head / (s.heads / s.key_heads);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int col0 = blockIdx.x * kColumns, col = col0 + 16 * wave + c;
    const bool mine = col < s.dv;
    const SequenceAt at = sequence_at(s, n);

    Tile<NI, DK> kt(smem), qt(smem + Tile<NI, DK>::kBytes);
    Tile<NI, kColumns> ot(smem + 2 * Tile<NI, DK>::kBytes);

    fx4 D[DK / 16];
    const int64_t state_at = (n * s.heads + head) * s.dk * s.dv;
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = feature_row(t, g, r);
            D[t][r] = d_final != nullptr && mine && row < s.dk ? d_final[state_at + (int64_t)row * s.dv + col] : 0.0f;
        }

    for (int64_t first = (at.length - 1) / kBlock * kBlock; first >= 0 && at.length > 0; first -= kBlock) {
        const int64_t row0 = at.row + first, block = at.block + first / kBlock;
        const int length = (int)(at.length - first < kBlock ? at.length - first : kBlock);
        const int64_t entry = block * s.heads + head;
        __syncthreads();
        for (int i = tid; i < kBlock * DK / 8; i += 256) {
            const int row = i / (DK / 8), d = i % (DK / 8) * 8;
            const bool there = row < length && d < s.dk;
            const int64_t from = ((row0 + row) * s.key_heads + key_head) * s.dk + d;
            kt.template put8<E>(row, d, load8<E>(k + from, there));
            qt.template put8<E>(row, d, load8<E>(q + from, there));
        }
        for (int i = tid; i < kBlock * kColumns / 8; i += 256) {
            const int row = i / (kColumns / 8), d = i % (kColumns / 8) * 8;
            const bool there = d_out != nullptr && row < length && col0 + d < s.dv;
            ot.template put8<E>(row, d, load8<E>(d_out + ((row0 + row) * s.heads + head) * s.dv + col0 + d, there));
        }
        gate[tid] = gates[entry * kGateFloats + tid];
        __syncthreads();
        const float whole = gate[kSince * kBlock + kBlock - 1];
        const Buffer tm = buffer_of(t_in + entry * kMatrixBytes<NS>, kMatrixBytes<NS>);
        const Buffer pm = buffer_of(p_in + entry * kMatrixBytes<NS>, kMatrixBytes<NS>);

        if (mine) {
            float* to = d_states + entry * s.dk * s.dv + col;
#pragma unroll
            for (int t = 0; t < DK / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (feature_row(t, g, r) < s.dk) to[(int64_t)feature_row(t, g, r) * s.dv] = D[t][r];
        }
        // dU = diag(e^(c[63]-c)) K D1 + P^T dO
        fx4 u[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) u[m] = fx4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) {
            const Operand<NS> so = operand_of<NS>(D[2 * d], D[2 * d + 1]);
#pragma unroll
            for (int m = 0; m < kTiles; ++m) u[m] = mma<NI, NS>(kt.along(16 * m + c, 32 * d, g), so, u[m]);
        }
        const Operand<NI> o_low = ot.down(0, 16 * wave, lane), o_high = ot.down(32, 16 * wave, lane);
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const fx4 f = *reinterpret_cast<const fx4*>(gate + kUntil * kBlock + 16 * m + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) u[m][r] *= f[r];
            if (m < 2) u[m] = mma<NS, NI>(matrix_operand<NS>(pm, pair_upper(m, 0), lane), o_low, u[m]);
            u[m] = mma<NS, NI>(matrix_operand<NS>(pm, pair_upper(m, 1), lane), o_high, u[m]);
        }
        // dR = dU + T^T dU
        {
            const Operand<NS> low = operand_of<NS>(u[0], u[1]), high = operand_of<NS>(u[2], u[3]);
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                if (m < 2) u[m] = mma<NS, NS>(matrix_operand<NS>(tm, pair_upper(m, 0), lane), low, u[m]);
                u[m] = mma<NS, NS>(matrix_operand<NS>(tm, pair_upper(m, 1), lane), high, u[m]);
            }
        }
        if (mine) {
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                const fx4 b = *reinterpret_cast<const fx4*>(gate + kBeta * kBlock + 16 * m + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * m + 4 * g + r;
                    if (row < length) {
                        const int64_t to = ((row0 + row) * s.heads + head) * s.dv + col;
                        d_v[to] = E::put(b[r] * u[m][r]);
                        d_rows[to] = u[m][r];
                    }
                }
            }
        }
        // D0 = e^c[63] D1 + Q^T diag(scale e^c) dO - K^T diag(beta e^c) dR
        fx4 w[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const fx4 f = *reinterpret_cast<const fx4*>(gate + kSince * kBlock + 16 * m + 4 * g);
            const fx4 b = *reinterpret_cast<const fx4*>(gate + kBetaSince * kBlock + 16 * m + 4 * g);
            w[m] = ot.tile(16 * m, 16 * wave, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w[m][r] *= s.scale * f[r];
                u[m][r] *= -b[r];
            }
        }
        const Operand<NS> low = operand_of<NS>(u[0], u[1]), high = operand_of<NS>(u[2], u[3]);
        const Operand<NS> w_low = operand_of<NS>(w[0], w[1]), w_high = operand_of<NS>(w[2], w[3]);
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) D[t][r] *= whole;
            D[t] = mma<NI, NS>(qt.down_features(0, t, lane), w_low, D[t]);
            D[t] = mma<NI, NS>(qt.down_features(32, t, lane), w_high, D[t]);
            D[t] = mma<NI, NS>(kt.down_features(0, t, lane), low, D[t]);
            D[t] = mma<NI, NS>(kt.down_features(32, t, lane), high, D[t]);
        }
    }
    if (d_initial != nullptr && mine) {
#pragma unroll
        for (int t = 0; t < DK / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (feature_row(t, g, r) < s.dk) d_initial[state_at + (int64_t)feature_row(t, g, r) * s.dv + col] = D[t][r];
    }
    if (s.offsets != nullptr && mine) {
        if (n == 0)
            for (int64_t row = g; row < offset_at(s, 0); row += 4) d_v[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
        if (n == s.sequences - 1)
            for (int64_t row = offset_at(s, s.sequences) + g; row < s.rows; row += 4)
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
