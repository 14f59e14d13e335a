// Per block of 64 tokens and head: the running sums of the log gates and the triangular matrices T and P
// (delta.h), written in the order in which the chain kernels' lanes load them as operands.
#ifndef ASCAN_DELTA_PREPARE_H_
#define ASCAN_DELTA_PREPARE_H_

#include "delta.h"
#include "delta_tile.h"

namespace ascan {
namespace {

// Rows of the table of a block's gates, 64 floats each.
enum { kBeta, kBetaSince, kSince, kUntil, kSumHigh, kSumLow, kGateRows };
constexpr int kGateFloats = kGateRows * kBlock;

template <int P>
constexpr int kMatrixBytes = P == 0 ? kPairs * 64 * 8 * 4 : P * kPairs * 64 * 8 * 2;

// Where products of depth 32 stand in a triangular matrix: row tile m, depths 32 s .. 32 s + 31.
__device__ __forceinline__ constexpr int pair_lower(int m, int s) { return m < 2 ? m : 2 * m - 2 + s; }
__device__ __forceinline__ constexpr int pair_upper(int m, int s) { return m < 2 ? 2 * m + s : m + 2; }

struct BlockAt {
    int64_t row;  // first row of the block
    int length;   // tokens, 0 where the entry is unused
    int64_t sequence;
};

__device__ __forceinline__ int64_t offset_at(const DeltaShape& s, int64_t i) {
    const int64_t o = s.wide_offsets ? static_cast<const int64_t*>(s.offsets)[i] : (int64_t) static_cast<const int32_t*>(s.offsets)[i];
    return o < 0 ? 0 : (o > s.rows ? s.rows : o);  // a table that is no ascending list of rows stays inside the tensors
}

struct SequenceAt {
    int64_t row, length, block;
};
__device__ __forceinline__ SequenceAt sequence_at(const DeltaShape& s, int64_t n) {
    if (s.offsets == nullptr) return SequenceAt{n * s.tokens, s.tokens, n * ((s.tokens + kBlock - 1) / kBlock)};
    const int64_t a = offset_at(s, n), b = offset_at(s, n + 1);
    return SequenceAt{a, b > a ? b - a : 0, a / kBlock + n};
}

// The sequence and rows of table entry `block`; every lane of the wave takes part.
__device__ __forceinline__ BlockAt block_at(const DeltaShape& s, int64_t block) {
    int64_t n;
    if (s.offsets == nullptr) {
        n = block / ((s.tokens + kBlock - 1) / kBlock);
    } else {
        // first entries ascend with the sequence: count those at or before this one
        const int lane = threadIdx.x & 63;
        int64_t count = 0;
        for (int64_t i = 0; i < s.sequences; i += 64) {
            const bool before = i + lane < s.sequences && offset_at(s, i + lane) / kBlock + i + lane <= block;
            const int found = __popcll(__ballot(before));
            count += found;
            if (found < 64) break;
        }
        if (count == 0) return BlockAt{0, 0, 0};
        n = count - 1;
    }
    const SequenceAt q = sequence_at(s, n);
    const int64_t first = (block - q.block) * kBlock;
    const int64_t left = q.length - first;
    return BlockAt{q.row + first, (int)(left < 0 ? 0 : (left > kBlock ? kBlock : left)), n};
}

// A log gate as the sums take it: e^-1000 is 0 like e^-inf, but differences of sums stay defined.
__device__ __forceinline__ double gate_sum_term(float g) { return g < -1000.0f ? -1000.0 : (double)g; }

template <class E>
__device__ __forceinline__ float load_gate(const DeltaShape& s, const void* p, int64_t i) {
    return s.wide_gates ? static_cast<const float*>(p)[i] : E::get(static_cast<const typename E::S*>(p)[i]);
}

template <class E, int NI, int NS, int DK>
constexpr int kPrepareBytes = (2 * Tile<NI, DK>::kBytes > 3 * kBlock * 65 * 4 ? 2 * Tile<NI, DK>::kBytes : 3 * kBlock * 65 * 4);

// grid (blocks, heads), 256 threads.  `upper`: the transposes of T and P, for the backward pass.
template <class E, int NI, int NS, int DK>
__global__ __launch_bounds__(256) void delta_prepare(DeltaShape s, const typename E::S* __restrict__ q,
                                                     const typename E::S* __restrict__ k,
                                                     const void* __restrict__ log_gates, const void* __restrict__ beta,
                                                     float* __restrict__ gates, char* __restrict__ t_out,
                                                     char* __restrict__ p_out, bool upper) {
    extern __shared__ __align__(16) char smem[];
    __shared__ double sum[kBlock];
    __shared__ float rate[kBlock];
    const int64_t block = blockIdx.x;
    const int head = blockIdx.y, key_head = head / (s.heads / s.key_heads);
    const BlockAt at = block_at(s, block);
    if (at.length <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;

    Tile<NI, DK> kt(smem), qt(smem + Tile<NI, DK>::kBytes);
    for (int i = tid; i < kBlock * DK / 8; i += 256) {
        const int row = i / (DK / 8), col = i % (DK / 8) * 8;
        const bool there = row < at.length && col < s.dk;
        const int64_t from = ((at.row + row) * s.key_heads + key_head) * s.dk + col;
        kt.template put8<E>(row, col, load8<E>(k + from, there));
        qt.template put8<E>(row, col, load8<E>(q + from, there));
    }
    if (wave == 0) {
        const bool there = lane < at.length;
        const int64_t from = (at.row + lane) * s.heads + head;
        const float b = there ? load_gate<E>(s, beta, from) : 0.0f;
        double x = there ? gate_sum_term(load_gate<E>(s, log_gates, from)) : 0.0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double y = __shfl_up(x, d);
            if (lane >= d) x += y;
        }
        const double whole = __shfl(x, 63);
        sum[lane] = x;
        rate[lane] = b;
        float* to = gates + (block * s.heads + head) * kGateFloats + lane;
        const float since = expf((float)x), high = (float)x;
        to[kBeta * kBlock] = b;
        to[kBetaSince * kBlock] = b * since;
        to[kSince * kBlock] = since;
        to[kUntil * kBlock] = expf((float)(whole - x));
        to[kSumHigh * kBlock] = high;
        to[kSumLow * kBlock] = (float)(x - (double)high);
    }
    __syncthreads();

    fx4 kk[kTiles], qk[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) kk[j] = qk[j] = fx4{0, 0, 0, 0};
    for (int d = 0; d < DK; d += 32) {
        const Operand<NI> a = kt.along(16 * wave + c, d, g), b = qt.along(16 * wave + c, d, g);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            if (j <= wave) {
                const Operand<NI> o = kt.along(16 * j + c, d, g);
                kk[j] = mma<NI, NI>(a, o, kk[j]);
                qk[j] = mma<NI, NI>(b, o, qk[j]);
            }
        }
    }
    __syncthreads();  // the tiles' memory is taken over by the three matrices

    constexpr int kRow = 65;
    float *lm = reinterpret_cast<float*>(smem), *xm = lm + kBlock * kRow, *pm = xm + kBlock * kRow;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * wave + 4 * g + r, col = 16 * j + c;
            float l = 0.0f, p = 0.0f;
            if (col <= row) {
                const float e = expf((float)(sum[row] - sum[col]));
                p = s.scale * e * qk[j][r];
                if (col < row) l = rate[row] * e * kk[j][r];
            }
            lm[row * kRow + col] = l;
            pm[row * kRow + col] = p;
            xm[row * kRow + col] = 0.0f;
        }
    }
    __syncthreads();

    // inverse of I + L: the diagonal's 16 x 16 tiles by substitution, a column to a lane (and its copies)
    {
        float x[16];
        const float* l = lm + 16 * wave * (kRow + 1);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = i == c ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; ++j) v -= l[i * kRow + j] * x[j];
            x[i] = v;
        }
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) xm[(16 * wave + i) * kRow + 16 * wave + c] = x[i];
        }
    }
    __syncthreads();
    // tile (i, j) of the inverse = -X(i, i) sum over k from j to i - 1 of L(i, k) X(k, j), one distance i - j at a time
#pragma unroll
    for (int d = 1; d < kTiles; ++d) {
        const int j = wave, i = wave + d;
        if (i < kTiles) {
            fx4 acc = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            for (int n = j; n < i; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(lm[(16 * i + c) * kRow + 16 * n + 4 * g + r],
                                                               xm[(16 * n + 4 * g + r) * kRow + 16 * j + c], acc, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                y = __builtin_amdgcn_mfma_f32_16x16x4f32(xm[(16 * i + c) * kRow + 16 * i + 4 * g + r], acc[r], y, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) xm[(16 * i + 4 * g + r) * kRow + 16 * j + c] = -y[r];
        }
        __syncthreads();
    }

    char* t_to = t_out + (block * s.heads + head) * kMatrixBytes<NS>;
    char* p_to = p_out + (block * s.heads + head) * kMatrixBytes<NS>;
    for (int i = tid; i < kPairs * 64; i += 256) {
        const int pair = i >> 6;
        const int m = upper ? (pair < 4 ? pair >> 1 : pair - 2) : (pair < 2 ? pair : (pair + 2) >> 1);
        const int h = upper ? (pair < 4 ? pair & 1 : 1) : (pair < 2 ? 0 : pair & 1);
        const int row = 16 * m + c;
        float t[8], p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int col = 32 * h + 4 * g + (e & 3) + (e & 4) * 4;
            const int from = upper ? col * kRow + row : row * kRow + col;
            t[e] = xm[from] - (row == col ? 1.0f : 0.0f);
            p[e] = pm[from];
        }
        if constexpr (NS == 0) {
            __builtin_memcpy(t_to + i * 32, t, 32);
            __builtin_memcpy(p_to + i * 32, p, 32);
        } else {
            const Operand<NS> to = operand_of<NS>(fx4{t[0], t[1], t[2], t[3]}, fx4{t[4], t[5], t[6], t[7]});
            const Operand<NS> po = operand_of<NS>(fx4{p[0], p[1], p[2], p[3]}, fx4{p[4], p[5], p[6], p[7]});
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                *reinterpret_cast<bx8*>(t_to + (n * kPairs * 64 + i) * 16) = to.p[n];
                *reinterpret_cast<bx8*>(p_to + (n * kPairs * 64 + i) * 16) = po.p[n];
            }
        }
    }
}

// Operand `pair` of a matrix that delta_prepare wrote.
template <int P>
__device__ __forceinline__ Operand<P> matrix_operand(Buffer m, int pair, int lane) {
    Operand<P> o;
    if constexpr (P == 0) {
        o.t[0] = fetch16(m, (pair * 64 + lane) * 32);
        o.t[1] = fetch16(m, (pair * 64 + lane) * 32 + 16);
    } else {
#pragma unroll
        for (int n = 0; n < P; ++n) o.p[n] = __builtin_bit_cast(bx8, fetch16(m, ((n * kPairs + pair) * 64 + lane) * 16));
    }
    return o;
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_PREPARE_H_
