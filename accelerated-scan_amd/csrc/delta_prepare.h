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

constexpr int kMatrixTiles = 2 * kPairs;                // of a triangular matrix in memory, fp32
constexpr int kMatrixBytes = kMatrixTiles * 64 * 4 * 4;

// Where products of depth 32 stand in a triangular matrix: row tile m, depths 32 s .. 32 s + 31.
__device__ __forceinline__ constexpr int pair_lower(int m, int s) { return m < 2 ? m : 2 * m - 2 + s; }
__device__ __forceinline__ constexpr int pair_upper(int m, int s) { return m < 2 ? 2 * m + s : m + 2; }

// Where in memory lane `lane` has its four values of tile n of a product.
__device__ __forceinline__ constexpr int matrix_place(int pair, int n, int lane) { return ((2 * pair + n) * 64 + lane) * 16; }

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
        n = (uint32_t)block / (uint32_t)((s.tokens + kBlock - 1) / kBlock);  // (both below 2^31)
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
    const int64_t left = first < 0 ? 0 : q.length - first;  // (first entries of a table that does not ascend do not either)
    return BlockAt{q.row + first, (int)(left < 0 ? 0 : (left > kBlock ? kBlock : left)), n};
}

// A log gate as the sums take it: e^-1000 is 0 like e^-inf, but differences of sums stay defined.
__device__ __forceinline__ double gate_sum_term(float g) { return g < -1000.0f ? -1000.0 : (double)g; }

template <class E>
__device__ __forceinline__ float load_gate(const DeltaShape& s, const void* p, int64_t i) {
    return s.wide_gates ? static_cast<const float*>(p)[i] : E::get(static_cast<const typename E::S*>(p)[i]);
}

constexpr int kMatrixRow = kBlock + 4;  // floats from row to row of a matrix in LDS: 16-byte rows, banks apart
template <int NI, int DK>
constexpr int kPrepareBytes = 2 * Tile<NI, DK>::kBytes > 2 * kBlock * kMatrixRow * 4 ? 2 * Tile<NI, DK>::kBytes
                                                                                    : 2 * kBlock * kMatrixRow * 4;

// c + a * b for two 16 x 16 tiles, fp32: a given by its rows, b as an accumulator holds it.
__device__ __forceinline__ fx4 tile_product(const fx4& a, const fx4& b, fx4 c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
}

// Sums over the lanes of a wave up to each, 64 bits wide: shifts within rows of 16 lanes, then rows onto later rows.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double x) {
    const uint64_t w = __builtin_bit_cast(uint64_t, x);
    const uint32_t a = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)w, CTRL, ROWS, 0xf, false);
    const uint32_t b = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(w >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)b << 32 | a);
}
__device__ __forceinline__ double wave_prefix(double x) {
    x += moved<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: 0 where there is no lane
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);  // row_bcast 15 to rows 1 and 3
    x += moved<0x143, 0xc>(x);  // row_bcast 31 to rows 2 and 3
    return x;
}
__device__ __forceinline__ double last_lane(double x) {
    const uint64_t w = __builtin_bit_cast(uint64_t, x);
    const uint32_t a = __builtin_amdgcn_readlane((int)(uint32_t)w, 63), b = __builtin_amdgcn_readlane((int)(uint32_t)(w >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)b << 32 | a);
}

// Where row `row`, features d .. d+7 of a block's queries stand in the copy for the forward chain: in the order in which its
// lanes take operands.
template <int DK>
__device__ __forceinline__ constexpr int query_place(int row, int d) {
    return (((row >> 4) * (DK / 32) + (d >> 5)) * 64 + ((d >> 3) & 3) * 16 + (row & 15)) * 8;
}

// grid (blocks, heads), 256 threads.  `upper`: the transposes of T and P, for the backward pass.
//
// P leaves from the accumulators: the tile K_j Q_i^T has token i in a lane's column and its rows j along the depth, as
// the operand wants it (Q_i K_j^T for the transpose).  The inverse of I + L is made by substitution inside the
// diagonal's 16 x 16 tiles, which is exact to rounding whatever the keys are (a series in L is not: its
// terms grow), and joined from there to 32 and to 64 with fp32 products.
//
// The block's keys and queries are copied to where they stand without gaps, missing rows and features as zeros: in the
// tensors the rows of a head are a power of two apart as a rule, so that one channel of the cache holds them all, and the
// chain's workgroups, which all want the same rows at the same time, waited for it (bf16 (1, 16384, 32 heads of 128 x 128):
// the chain 463 us without copies, 439 with; they cost this kernel 14).
//
// What bounds it: there it reads 130 MB and writes 350 MB in 104 to 112 us, 4.3 to 4.6 TB/s.
template <class E, int NI, int DK, bool upper>
__global__ __launch_bounds__(256, 4) void delta_prepare(DeltaShape s, const typename E::S* __restrict__ q,
                                                     const typename E::S* __restrict__ k,
                                                     const void* __restrict__ log_gates, const void* __restrict__ beta,
                                                     float* __restrict__ gates, char* __restrict__ t_out,
                                                     char* __restrict__ p_out, typename E::S* __restrict__ k_out,
                                                     typename E::S* __restrict__ q_out) {
    extern __shared__ __align__(16) char smem[];
    __shared__ float high[kBlock], low[kBlock], rate[kBlock];
    __shared__ int odd_at;
    const int64_t block = blockIdx.x;
    const int head = blockIdx.y, key_head = head / (s.heads / s.key_heads);
    const BlockAt at = block_at(s, block);
    if (at.length <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;

    const Tile<NI, DK> kt(smem), qt(smem + Tile<NI, DK>::kBytes);
    float b = 0.0f, x = 0.0f;
    if (tid == 0) odd_at = kBlock;
    {
        constexpr uint32_t kSize = sizeof(typename E::S);
        const int64_t row0 = uniform(at.row);
        const int length = __builtin_amdgcn_readfirstlane(at.length);
        const uint32_t step = s.key_heads * s.dk * kSize;
        const int64_t from = row0 * step + (int64_t)key_head * s.dk * kSize, bytes = (length - 1) * (int64_t)step + s.dk * kSize;
        const Buffer kb = buffer_of(reinterpret_cast<const char*>(k) + from, bytes);
        const Buffer qb = buffer_of(reinterpret_cast<const char*>(q) + from, bytes);
        if (wave == 0 && lane < length) {
            b = load_gate<E>(s, beta, (row0 + lane) * s.heads + head);
            x = load_gate<E>(s, log_gates, (row0 + lane) * s.heads + head);
        }
        Eight<E> k_raw[DK / 32], q_raw[DK / 32];
#pragma unroll
        for (int i = 0; i < DK / 32; ++i) {
            const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
            const uint32_t cell = d < s.dk ? row * step + d * kSize : kOutside;
            k_raw[i] = fetch8<E>(kb, cell);
            q_raw[i] = fetch8<E>(qb, cell);
        }
#pragma unroll
        for (int i = 0; i < DK / 32; ++i) {
            const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
            kt.template put8<E>(row, d, k_raw[i]);
            qt.template put8<E>(row, d, q_raw[i]);
        }
        if (head % (s.heads / s.key_heads) == 0) {
            const int64_t to = (block * s.key_heads + key_head) * kBlock * DK;
#pragma unroll
            for (int i = 0; i < DK / 32; ++i) {
                const int row = (tid + 256 * i) / (DK / 8), d = (tid + 256 * i) % (DK / 8) * 8;
                store8<E>(k_out + to + (tid + 256 * i) * 8, k_raw[i]);
                store8<E>(q_out + to + (upper ? (tid + 256 * i) * 8 : query_place<DK>(row, d)), q_raw[i]);
            }
        }
    }
    __syncthreads();
    if (wave == 0) {
        double sum = gate_sum_term(x);  // (0 behind the last token, like its beta)
        sum = wave_prefix(sum);
        const double whole = last_lane(sum);
        float* to = gates + (block * s.heads + head) * kGateFloats + lane;
        const float since = exp_of((float)sum), h = (float)sum, l = (float)(sum - (double)h);
        high[lane] = h;
        low[lane] = l;
        rate[lane] = b;
        to[kBeta * kBlock] = b;
        to[kBetaSince * kBlock] = b * since;
        to[kSince * kBlock] = since;
        to[kUntil * kBlock] = exp_of((float)(whole - sum));
        to[kSumHigh * kBlock] = h;
        to[kSumLow * kBlock] = l;
        if (is_odd(h) || is_odd(b)) atomicMin(&odd_at, lane);
    }

    // kk: K_j K_i^T with i the own tile and j up to it.  pq: K_j Q_i^T, or with `upper` Q_i K_j^T for j the own tile and
    // i from it on
    fx4 kk[kTiles], pq[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) kk[j] = pq[j] = fx4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < DK; d += 32) {
        const Operand<NI> mine = kt.along(16 * wave + c, d, g), theirs = upper ? mine : qt.along(16 * wave + c, d, g);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            if (j <= wave) {
                const Operand<NI> o = kt.along(16 * j + c, d, g);
                kk[j] = mma_all<NI, NI>(o, mine, kk[j]);
                if (!upper) pq[j] = mma_all<NI, NI>(o, theirs, pq[j]);
            }
            if (upper && j >= wave) pq[j] = mma_all<NI, NI>(qt.along(16 * j + c, d, g), theirs, pq[j]);
        }
    }
    const int here = 16 * wave + c;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
        if (j == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (4 * g + r == c && is_odd(kk[j][r])) atomicMin(&odd_at, here);
        }
    __syncthreads();  // the tiles' memory is taken over by L^T and the inverse
    // T and P have zeros from the first token on whose key (by its product with itself), beta or gate is not finite; the chain
    // finds that token by its R, which its beta makes NaN.
    const int odd = odd_at, here_up_to = here < odd ? here : -1;
    if (tid == odd && odd < kBlock) gates[(block * s.heads + head) * kGateFloats + kBeta * kBlock + tid] = __builtin_nanf("");
    const float high_here = high[here], low_here = low[here], rate_here = rate[here];

    float *lt = reinterpret_cast<float*>(smem), *xm = lt + kBlock * kMatrixRow;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
        const int row0 = 16 * j + 4 * g;
        const fx4 h = *reinterpret_cast<const fx4*>(high + row0), l = *reinterpret_cast<const fx4*>(low + row0);
        fx4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float far = (high_here - h[r]) + (low_here - l[r]);
            e[r] = exp_of(j <= wave ? far : -far);  // (a tile on the diagonal needs its lower half only, or its upper)
        }
        if (j <= wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                lt[(row0 + r) * kMatrixRow + here] = row0 + r < here_up_to ? rate_here * e[r] * kk[j][r] : 0.0f;
        }
        if (upper && j == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) e[r] = exp_of(-((high_here - h[r]) + (low_here - l[r])));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            pq[j][r] = (upper ? row0 + r >= here && row0 + r < odd : row0 + r <= here_up_to) ? s.scale * e[r] * pq[j][r] : 0.0f;
    }
    {
        char* to = p_out + (block * s.heads + head) * kMatrixBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool there = upper ? h >= (wave >> 1) : h <= (wave >> 1);
            if (there) {
                const int pair = upper ? pair_upper(wave, h) : pair_lower(wave, h);
#pragma unroll
                for (int n = 0; n < 2; ++n) *reinterpret_cast<fx4*>(to + matrix_place(pair, n, lane)) = pq[2 * h + n];
            }
        }
    }
    // (a wave's diagonal tile of L is its own work: no barrier before the substitution)
    {
        float x[16];
        const float* l = lt + 16 * wave * (kMatrixRow + 1);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == c ? 1.0f : 0.0f;
#pragma unroll
        for (int i = 0; i < 15; ++i) {
            // row i of the column is final: off the rows below with it
            float column[16];
#pragma unroll
            for (int n = (i + 1) / 4; n < 4; ++n) {
                const fx4 part = *reinterpret_cast<const fx4*>(l + i * kMatrixRow + 4 * n);
#pragma unroll
                for (int r = 0; r < 4; ++r) column[4 * n + r] = part[r];
            }
#pragma unroll
            for (int n = i + 1; n < 16; ++n) x[n] = fmaf(-column[n], x[i], x[n]);
        }
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) xm[(16 * wave + i) * kMatrixRow + here] = x[i];
        }
        if ((wave & 1) == 0) {  // the zero tile beside it that an operand spans
#pragma unroll
            for (int r = 0; r < 4; ++r) xm[(16 * wave + 4 * g + r) * kMatrixRow + here + 16] = 0.0f;
        }
    }
    __syncthreads();
    const auto l_rows = [&](int i, int n) {  // tile (i, n) of L by its rows
        fx4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = lt[(16 * n + 4 * g + r) * kMatrixRow + 16 * i + c];
        return o;
    };
    const auto x_rows = [&](int i, int n) { return *reinterpret_cast<const fx4*>(xm + (16 * i + c) * kMatrixRow + 16 * n + 4 * g); };
    const auto x_tile = [&](int i, int n) {
        fx4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = xm[(16 * i + 4 * g + r) * kMatrixRow + 16 * n + c];
        return o;
    };
    const auto put_tile = [&](int i, int n, const fx4& o, float sign) {
#pragma unroll
        for (int r = 0; r < 4; ++r) xm[(16 * i + 4 * g + r) * kMatrixRow + 16 * n + c] = sign * o[r];
    };
    const fx4 zero = {0, 0, 0, 0};
    if (wave < 2) {  // tiles (1, 0) and (3, 2)
        const int n = 2 * wave;
        put_tile(n + 1, n, tile_product(x_rows(n + 1, n + 1), tile_product(l_rows(n + 1, n), x_tile(n, n), zero), zero), -1.0f);
    }
    __syncthreads();
    {
        // the lower left quarter: -X(2..3, 2..3) M, M = L(2..3, 0..1) X(0..1, 0..1), a tile to a wave; M waits in the
        // upper right quarter, which nobody reads
        const int i = 2 + (wave >> 1), j = wave & 1;
        fx4 m = tile_product(l_rows(i, 1), x_tile(1, j), zero);
        if (j == 0) m = tile_product(l_rows(i, 0), x_tile(0, 0), m);
        put_tile(i - 2, j + 2, m, 1.0f);
        __syncthreads();
        fx4 y = tile_product(x_rows(i, 2), x_tile(0, j + 2), zero);
        if (i == 3) y = tile_product(x_rows(3, 3), x_tile(1, j + 2), y);
        put_tile(i, j, y, -1.0f);
    }
    __syncthreads();

    char* to = t_out + (block * s.heads + head) * kMatrixBytes;
    for (int i = tid; i < kPairs * 64; i += 256) {
        const int pair = i >> 6;
        const int m = upper ? (pair < 4 ? pair >> 1 : pair - 2) : (pair < 2 ? pair : (pair + 2) >> 1);
        const int h = upper ? (pair < 4 ? pair & 1 : 1) : (pair < 2 ? 0 : pair & 1);
        const int row = 16 * m + c, col = 32 * h + 4 * g;
        fx4 a, b;
        if (upper) {
            a = x_tile(2 * h, m);
            b = x_tile(2 * h + 1, m);
        } else {
            a = x_rows(m, 2 * h);
            b = x_rows(m, 2 * h + 1);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            a[r] -= row == col + r ? 1.0f : 0.0f;
            b[r] -= row == col + 16 + r ? 1.0f : 0.0f;
        }
        *reinterpret_cast<fx4*>(to + matrix_place(pair, 0, lane)) = a;
        *reinterpret_cast<fx4*>(to + matrix_place(pair, 1, lane)) = b;
    }
}

// The tiles of product `pair` of a matrix that delta_prepare wrote, or zeros where it is not `there`.
__device__ __forceinline__ void fetch_matrix(Buffer m, bool there, int pair, int lane, fx4 (&x)[2]) {
#pragma unroll
    for (int n = 0; n < 2; ++n) x[n] = fetch16(m, there ? matrix_place(pair, n, lane) : kOutside);
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_PREPARE_H_
