// Forward pass of the gated delta rule: the chain over the blocks of a sequence (delta.h).
#ifndef ASCAN_DELTA_FORWARD_H_
#define ASCAN_DELTA_FORWARD_H_

#include "delta_prepare.h"

namespace ascan {
namespace {

constexpr int kColumns = 64;  // state columns of a workgroup: 16 to a wave

template <int NI, int DK>
constexpr int kChainBytes = 2 * Tile<NI, DK>::kBytes + Tile<NI, kColumns>::kBytes;

// A wave keeps 16 columns of the state in its accumulators from the first block to the last; keys, queries
// and values of a block are shared by the workgroup's waves through LDS.
// grid (column groups, heads, sequences), 256 threads.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(256) void delta_chain(DeltaShape s, const typename E::S* __restrict__ q,
                                                   const typename E::S* __restrict__ k,
                                                   const typename E::S* __restrict__ v,
                                                   const float* __restrict__ gates, const char* __restrict__ t_in,
                                                   const char* __restrict__ p_in, const float* __restrict__ initial,
                                                   typename E::S* __restrict__ out, float* __restrict__ final,
                                                   float* __restrict__ states, float* __restrict__ updates) {
    extern __shared__ __align__(16) char smem[];
    __shared__ __align__(16) float gate[4 * kBlock];
    const int64_t n = blockIdx.z;
    const int head = blockIdx.y, key_head = head / (s.heads / s.key_heads);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int col0 = blockIdx.x * kColumns, col = col0 + 16 * wave + c;
    const bool mine = col < s.dv;
    const SequenceAt at = sequence_at(s, n);

    Tile<NI, DK> kt(smem), qt(smem + Tile<NI, DK>::kBytes);
    Tile<NI, kColumns> vt(smem + 2 * Tile<NI, DK>::kBytes);

    fx4 S[DK / 16];
    const int64_t state_at = (n * s.heads + head) * s.dk * s.dv;
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * t + 4 * g + r;
            S[t][r] = initial != nullptr && mine && row < s.dk ? initial[state_at + (int64_t)row * s.dv + col] : 0.0f;
        }

    for (int64_t first = 0; first < at.length; first += kBlock) {
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
            const bool there = row < length && col0 + d < s.dv;
            vt.template put8<E>(row, d, load8<E>(v + ((row0 + row) * s.heads + head) * s.dv + col0 + d, there));
        }
        gate[tid] = gates[entry * kGateFloats + tid];  // the first four rows of the table
        __syncthreads();
        const float whole = gate[kSince * kBlock + kBlock - 1];
        const char* tm = t_in + entry * kMatrixBytes<NS>;
        const char* pm = p_in + entry * kMatrixBytes<NS>;

        if (states != nullptr && mine) {
            float* to = states + entry * s.dk * s.dv + col;
#pragma unroll
            for (int t = 0; t < DK / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * g + r < s.dk) to[(int64_t)(16 * t + 4 * g + r) * s.dv] = S[t][r];
        }

        // K S0 (rows: tokens, columns: state columns) and (Q S0)^T (rows: state columns, columns: tokens)
        fx4 u[kTiles], o[kTiles];
#pragma unroll
        for (int m = 0; m < kTiles; ++m) u[m] = o[m] = fx4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) {
            const Operand<NS> so = operand_of<NS>(S[2 * d], S[2 * d + 1]);
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                u[m] = mma<NI, NS>(kt.along(16 * m + c, 32 * d, g), so, u[m]);
                o[m] = mma<NS, NI>(so, qt.along(16 * m + c, 32 * d, g), o[m]);
            }
        }
        // R = diag(beta) V - diag(beta e^c) K S0, U = R + T R
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const fx4 b = *reinterpret_cast<const fx4*>(gate + kBeta * kBlock + 16 * m + 4 * g);
            const fx4 bs = *reinterpret_cast<const fx4*>(gate + kBetaSince * kBlock + 16 * m + 4 * g);
            const fx4 x = vt.tile(16 * m, 16 * wave, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) u[m][r] = b[r] * x[r] - bs[r] * u[m][r];
        }
        {
            const Operand<NS> low = operand_of<NS>(u[0], u[1]), high = operand_of<NS>(u[2], u[3]);
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                u[m] = mma<NS, NS>(matrix_operand<NS>(tm, pair_lower(m, 0), lane), low, u[m]);
                if (m >= 2) u[m] = mma<NS, NS>(matrix_operand<NS>(tm, pair_lower(m, 1), lane), high, u[m]);
            }
        }
        // out^T = scale (Q S0)^T diag(e^c) + U^T P^T
        {
            const Operand<NS> low = operand_of<NS>(u[0], u[1]), high = operand_of<NS>(u[2], u[3]);
#pragma unroll
            for (int m = 0; m < kTiles; ++m) {
                const float f = s.scale * gate[kSince * kBlock + 16 * m + c];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[m][r] *= f;
                o[m] = mma<NS, NS>(low, matrix_operand<NS>(pm, pair_lower(m, 0), lane), o[m]);
                if (m >= 2) o[m] = mma<NS, NS>(high, matrix_operand<NS>(pm, pair_lower(m, 1), lane), o[m]);
                const int row = 16 * m + c, d = col0 + 16 * wave + 4 * g;
                if (row < length && d < s.dv) store4<E>(out + ((row0 + row) * s.heads + head) * s.dv + d, o[m]);
            }
        }
        if (updates != nullptr && mine) {
            float* to = updates + (row0 * s.heads + head) * s.dv + col;
#pragma unroll
            for (int m = 0; m < kTiles; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * m + 4 * g + r < length) to[(int64_t)(16 * m + 4 * g + r) * s.heads * s.dv] = u[m][r];
        }
        // S1 = e^c[63] S0 + K^T diag(e^(c[63]-c)) U
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
            const fx4 f = *reinterpret_cast<const fx4*>(gate + kUntil * kBlock + 16 * m + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) u[m][r] *= f[r];
        }
        const Operand<NS> low = operand_of<NS>(u[0], u[1]), high = operand_of<NS>(u[2], u[3]);
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] *= whole;
            S[t] = mma<NI, NS>(kt.down(0, 16 * t, lane), low, S[t]);
            S[t] = mma<NI, NS>(kt.down(32, 16 * t, lane), high, S[t]);
        }
    }
    if (final != nullptr && mine) {
#pragma unroll
        for (int t = 0; t < DK / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * t + 4 * g + r < s.dk) final[state_at + (int64_t)(16 * t + 4 * g + r) * s.dv + col] = S[t][r];
    }
    // rows in front of the first and behind the last sequence are zero
    if (s.offsets != nullptr && mine) {
        if (n == 0)
            for (int64_t row = g; row < offset_at(s, 0); row += 4) out[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
        if (n == s.sequences - 1)
            for (int64_t row = offset_at(s, s.sequences) + g; row < s.rows; row += 4)
                out[(row * s.heads + head) * s.dv + col] = E::put(0.0f);
    }
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_FORWARD_H_
