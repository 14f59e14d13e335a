// Forward pass of the gated delta rule: the chain over the blocks of a sequence (delta.h).
//
// The blocks of a sequence follow each other, so what counts is the time from a state to the next: a chain of
// three products (K S0, T R, K^T U) that are too small to fill a wave's matrix unit for long.  A workgroup
// therefore takes only 16 columns of one head's state and divides the rows: state wave w (0 to 3) keeps state rows
// dk/4 w .. in its accumulators and computes tokens 16w .. 16w+15 of every block.  State, R and U go round through LDS
// in the order in which the next product reads them, with one barrier each.  What the chain does not wait for
// is done by waves of their own beside these on the same SIMDs: four compute the outputs, four bring keys, values, T
// and gates to LDS blocks ahead.  (The loads are 60 KiB a block, which the 64 bytes per clock of a compute unit's
// cache turn into 960 clocks of issue: a wave that loads is late for its barrier if it has anything else to do.)
//
// What bounds it: bf16 (1, 16384, 32 heads of 128 x 128) takes 455 to 540 us, 256 blocks of 1.8 to 2.1 us, one chain to
// a compute unit.  LDS is at work 54 % of the time (240 KiB a block, 1900 clocks), vector instructions 46 % (most of them splitting
// values into parts), the matrix units 24 %, beside three round trips (write, barrier, read, product) of 300 to 400 clocks that
// nothing overlaps but the other waves' work.  More columns to a workgroup
// would read less per column and leave compute units without one.  The chain that also writes states and U moves 0.41 GB
// in 141 to 155 us (2, 4096, 16 heads).
// Registers, at 12 waves to a compute unit and a key size above 64: two of the bf16 chain are kept in memory, 14 of the
// fp16 one and one of the fp32 one, nearly all of them addresses that the loop does not touch.
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

// Whether a chain kernel asks for its blocks ahead (touch below).  It gains where a block's loads are many beside its work:
// chains that also write states (`keeps`) or run backward, training step bf16 (2, 4096, 16 heads of 128 x 128) 654 -> 599 us,
// (4, 2048, 32 heads) 1336 -> 1210, and half values, whose keys take twice the room in LDS, (1, 16384, 32 heads) 822 -> 750 us,
// (16, 512, 32 heads) 482 -> 469; it costs bf16 prompts 1 to 3 % (526 -> 530, 332 -> 343), and gives nothing where blocks are
// small (key size 64: chains of 71 and 89 us 71 and 92) and where fp32 products take longer than the loads (73 and 73).
template <int NI, int NS, int DK>
constexpr bool chain_touches(bool keeps) { return NS > 0 && DK == 128 && (NI > 1 || keeps); }

// A chain's workgroup may have as many lines of 128 bytes on their way as its compute unit's cache holds, 256.  At the
// latency of memory, a microsecond, that is 32 KiB per microsecond where a block wants 60 (and nobody else uses the
// bandwidth); at that of the die's second cache it is three times as much.  So every line is asked for blocks ahead by
// one of the workgroups that will read it: line `id` of up to five pieces of memory, one after the other.
struct Lines {
    const char* at[5];
    int count[5];  // of 128 bytes
    int row_lines;   // of the last piece: lines of a row, which are `step` bytes apart
    int64_t step;
};
__device__ __forceinline__ int touch(const Lines& l, int id) {
    const char* p = nullptr;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        const char* here = i < 4 ? l.at[i] + id * 128 : l.at[4] + (int64_t)(id / l.row_lines) * l.step + id % l.row_lines * 128;
        if (id >= 0 && id < l.count[i]) p = here;
        id -= l.count[i];
    }
    return p != nullptr ? *reinterpret_cast<const int*>(p) : 0;
}

template <int NI, int NS, int DK>
constexpr int kChainBytes = 2 * Tile<NI, DK>::kBytes + 2 * Tile<NI, 16>::kBytes + Exchange<NS, DK / 32>::kBytes +
                            3 * Exchange<NS, 2>::kBytes + 2 * Exchange<NS, kPairs>::kBytes + 2 * 4 * kBlock * 4 + 64;

constexpr int kPieces = kMatrixTiles / 4;  // tiles of T that a wave of four carries to LDS

// Zeros for what is not finite in an operand of tokens; the first such token, where its first four are row0 ..
template <int P>
__device__ __forceinline__ int zero_odd(Operand<P>& o, int row0) {
    int odd = kBlock;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
        bool is;
        if constexpr (P == 0) {
            is = is_odd(o.t[e >> 2][e & 3]);
            if (is) o.t[e >> 2][e & 3] = 0.0f;
        } else {
            is = is_odd((float)o.p[0][e]);
#pragma unroll
            for (int n = 0; n < P; ++n)
                if (is) o.p[n][e] = (__bf16)0.0f;
        }
        if (is) odd = row0 + (e >> 2) * 16 + (e & 3);
    }
    return odd;
}

// q and k: the copies that delta_prepare made.  grid chain_grid(), 768 threads.  KEEP: write the states in front
// of the blocks and the rows U.
// States, R, U, T and P are in NS parts.  T and P come from memory in fp32 and their parts are made by the waves with time for it:
// as parts they are half as large again (bf16, 16384 tokens, 32 heads, with delta_prepare: 537 us so, 547 from fp32; packed
// fp16 400 and 389, training 619 and 603).
template <class E, int NI, int NS, int DK, bool KEEP>
__global__ __launch_bounds__(768) void delta_chain(DeltaShape s, const typename E::S* __restrict__ q,
                                                   const typename E::S* __restrict__ k,
                                                   const typename E::S* __restrict__ v,
                                                   const float* __restrict__ gates, const char* __restrict__ t_in,
                                                   const char* __restrict__ p_in, const float* __restrict__ initial,
                                                   typename E::S* __restrict__ out, float* __restrict__ final,
                                                   float* __restrict__ states, float* __restrict__ updates, bool ahead) {
    using ES = typename E::S;
    constexpr int kDepths = DK / 32, kOwn = DK / 64, kCopies = DK / 32;  // operands of a row, state tiles of a wave, loads of a thread
    extern __shared__ __align__(16) char smem[];
    const ChainAt where = chain_at(s);
    if (!where.there) return;
    const int64_t n = where.sequence;
    const int head = where.head, key_head = head / (s.heads / s.key_heads);
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int role = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8);
    const bool keeper = role == 0;  // a state wave
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
    m += 3 * Exchange<NS, 2>::kBytes;
    char* const matrix_at = m;
    float* const gate_at = reinterpret_cast<float*>(m + 2 * Exchange<NS, kPairs>::kBytes);
    // Per column the first token of the block at hand from which its state is not finite.  A NaN in R meets the zeros of T
    // and would meet those of P and reach earlier tokens: U, which shows it, is computed again with a zero in its place,
    // and state and outputs get the NaN by this number.  (A test of R itself stands on every block's way.)
    int* const odd_at = reinterpret_cast<int*>(gate_at + 2 * 4 * kBlock);

    constexpr uint32_t kSize = sizeof(ES);
    const uint32_t v_step = s.heads * s.dv * kSize;
    const int64_t seq_row = uniform(at.row), seq_length = uniform(at.length), seq_block = uniform(at.block);
    const int token = 16 * wave + c;
    // Where the block at hand begins in a tensor or table; moved on by a constant from block to block.
    const auto rows_of = [&](const char* p, int64_t first, uint32_t step, uint32_t bytes) {
        const int64_t left = seq_length - first;
        return buffer_of(p, left <= 0 ? 0 : ((left < kBlock ? (int)left : kBlock) - 1) * (int)step + (int)bytes);
    };
    const auto start_of = [&](const void* p, uint32_t step, int64_t at_head) { return static_cast<const char*>(p) + seq_row * step + at_head; };
    const int64_t entry0 = seq_block * s.heads + head;
    const int64_t gate_move = (int64_t)s.heads * kGateFloats * 4, matrix_move = (int64_t)s.heads * kMatrixBytes;
    constexpr int kKeyBytes = kBlock * DK * kSize;  // of a block, in the copies
    const int64_t k_move = (int64_t)s.key_heads * kKeyBytes, v_move = (int64_t)v_step * kBlock;
    const char* gate_p = reinterpret_cast<const char*>(gates + entry0 * kGateFloats);
    const auto gates_here = [&]() { return buffer_of(gate_p, kGateFloats * 4); };
    const auto keys_at = [&](int64_t first) { return Tile<NI, DK>(smem + ((first / kBlock) & 1) * Tile<NI, DK>::kBytes); };
    const auto matrix_of = [&](int64_t first) {
        return Exchange<NS, kPairs>(matrix_at + ((first / kBlock) & 1) * Exchange<NS, kPairs>::kBytes);
    };
    const auto gate_of = [&](int64_t first) { return gate_at + ((first / kBlock) & 1) * 4 * kBlock; };
    const auto values_at = [&](int64_t first) { return Tile<NI, 16>(vt_at + ((first / kBlock) & 1) * Tile<NI, 16>::kBytes); };

    const int64_t v_head = (int64_t)head * s.dv * kSize, copy0 = (seq_block * s.key_heads + key_head) * kBlock * DK;

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
        Operand<NI> ko[kDepths];
        fx4 x, beta, beta_since;
        const auto gate_rows = [&](int64_t first, int row) { return *reinterpret_cast<const fx4*>(gate_of(first) + row * kBlock + 16 * wave + 4 * g); };
        const auto read_block = [&](int64_t first) {  // what of the block at `first` the first product takes beside the state
#pragma unroll
            for (int d = 0; d < kDepths; ++d) ko[d] = keys_at(first).along(token, 32 * d, g);
            x = values_at(first).tile(16 * wave, 0, lane);
            beta = gate_rows(first, kBeta);
            beta_since = gate_rows(first, kBetaSince);
        };
        if (tid < 16) odd_at[tid] = kBlock;
        __builtin_amdgcn_s_setprio(3);
        if (seq_length > 0) {
            lds_barrier();  // the first block's keys and values are there
            read_block(0);
        }
        for (int64_t first = 0; first < seq_length; first += kBlock) {
            const bool more = first + kBlock < seq_length;
            const Tile<NI, DK> kb = keys_at(first);
#pragma unroll
            for (int t = 0; t < kOwn; ++t) xs.put(kOwn * wave + t, lane, S[t]);
            lds_barrier();

            // K S0 (rows: tokens, columns: state columns)
            fx4 u = {0, 0, 0, 0}, u2 = {0, 0, 0, 0};  // (two sums: half as many products that wait for each other)
            Operand<NS> tm[2];
            fx4 until;
            float whole;
            {
                Operand<NS> so[kDepths];
#pragma unroll
                for (int d = 0; d < kDepths; ++d) so[d] = xs.get(d, lane);
                tm[0] = matrix_of(first).get(pair_lower(wave, 0), lane);
                tm[1] = matrix_of(first).get(pair_lower(wave, wave >> 1), lane);
                until = gate_rows(first, kUntil);
                whole = gate_of(first)[kSince * kBlock + kBlock - 1];
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
            const fx4 own = u;
            xr.put(wave, lane, u);
            lds_barrier();

            // U = R + T R; what the next products take of the keys is read on the way
            Operand<NI> k_low[kOwn], k_high[kOwn];
            {
                const Operand<NS> low = xr.get(0, lane), high = xr.get(1, lane);
#pragma unroll
                for (int t = 0; t < kOwn; ++t) {
                    k_low[t] = kb.down_features(0, kOwn * wave + t, lane);
                    k_high[t] = kb.down_features(32, kOwn * wave + t, lane);
                }
                __builtin_amdgcn_sched_barrier(0);
                // (one branch around all of it: where a branch stands between a matrix instruction and the first use of its
                // result, the compiler has left out the wait)
                if (wave >= 2) {
                    u2 = mma<NS, NS>(tm[1], high, fx4{0, 0, 0, 0});
                    u = mma<NS, NS>(tm[0], low, u);
#pragma unroll
                    for (int r = 0; r < 4; ++r) u[r] += u2[r];
                } else {
                    u = mma<NS, NS>(tm[0], low, u);
                }
            }
            {
                fx4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = until[r] * u[r];
                xd.put(wave, lane, y);
            }
            xu.put(wave, lane, u);
            if (__any(is_odd(u[0]) || is_odd(u[1]) || is_odd(u[2]) || is_odd(u[3]))) {
                // again without what is not finite
                Operand<NS> low = xr.get(0, lane), high = xr.get(1, lane);
                int odd = wave >= 2 ? zero_odd(high, 32 + 4 * g) : kBlock;
                odd = min(odd, zero_odd(low, 4 * g));
                odd = min(odd, __shfl_xor(odd, 16));
                odd = min(odd, __shfl_xor(odd, 32));
                u = mma<NS, NS>(matrix_of(first).get(pair_lower(wave, 0), lane), low, fx4{0, 0, 0, 0});
                u2 = mma<NS, NS>(matrix_of(first).get(pair_lower(wave, wave >> 1), lane), high, fx4{0, 0, 0, 0});
                fx4 y;
#pragma unroll
                for (int r = 3; r >= 0; --r) {
                    u[r] += own[r] + (wave >= 2 ? u2[r] : 0.0f);
                    if (is_odd(u[r])) odd = min(odd, 16 * wave + 4 * g + r);
                }
                atomicMin(odd_at + c, odd);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool gone = 16 * wave + 4 * g + r >= odd;
                    y[r] = gone ? __builtin_nanf("") : until[r] * u[r];
                    u[r] = gone ? 0.0f : u[r];
                }
                xd.put(wave, lane, y);
                xu.put(wave, lane, u);
            }
            lds_barrier();

            // S1 = e^c[63] S0 + K^T diag(e^(c[63]-c)) U
            {
                const Operand<NS> low = xd.get(0, lane), high = xd.get(1, lane);
                __builtin_amdgcn_sched_barrier(0);
                fx4 S2[kOwn];
#pragma unroll
                for (int t = 0; t < kOwn; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[t][r] *= whole;
                    S[t] = mma<NI, NS>(k_low[t], low, S[t]);
                    S2[t] = mma<NI, NS>(k_high[t], high, fx4{0, 0, 0, 0});
                }
                read_block(more ? first + kBlock : first);
#pragma unroll
                for (int t = 0; t < kOwn; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[t][r] += S2[t][r];
            }
        }
        if (((seq_length + kBlock - 1) / kBlock) & 1) {  // the other waves go on by two blocks
            lds_barrier();
            lds_barrier();
            lds_barrier();
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
    } else if (role == 1 && seq_length > 0) {
        // The outputs.  Loads come back in the order of their issue, so all of them run more than a block ahead: one that
        // did not would make its wait one for all before it.  Behind the last block loads repeat it or give zero and
        // stores are dropped, so that no condition stands around them.
        Eight<E> q_raw[2][kDepths];
        fx4 p_raw[2][2][2];
        float since[2];
        const char *q_p = reinterpret_cast<const char*>(q + copy0), *p_p = p_in + entry0 * kMatrixBytes;
        const char* out_p = start_of(out, v_step, v_head);
        // KEEP: state and updates leave from their parts in LDS, to 2^-24
        const uint32_t u_step = s.heads * s.dv * 4;
        [[maybe_unused]] char* state_p = reinterpret_cast<char*>(states + entry0 * s.dk * s.dv);
        [[maybe_unused]] char* update_p = reinterpret_cast<char*>(updates + (seq_row * s.heads + head) * s.dv);
        const int quad = col0 + 4 * g;
        const auto load_q = [&](int64_t first, int set) __attribute__((always_inline)) {
            const Buffer b = buffer_of(q_p, kKeyBytes);
#pragma unroll
            for (int d = 0; d < kDepths; ++d) q_raw[set][d] = fetch8<E>(b, ((wave * kDepths + d) * 64 + lane) * 8 * kSize);
            if (first + kBlock < seq_length) q_p += k_move;
        };
        const auto load_p = [&](int64_t first, int set) __attribute__((always_inline)) {
            const Buffer b = buffer_of(p_p, kMatrixBytes);
            fetch_matrix(b, true, pair_lower(wave, 0), lane, p_raw[set][0]);
            fetch_matrix(b, wave >= 2, pair_lower(wave, 1), lane, p_raw[set][1]);  // (one product to a row of tiles in waves 0, 1)
            since[set] = fetch4(gates_here(), kSince * 256 + token * 4);
            if (first + kBlock < seq_length) {
                p_p += matrix_move;
                gate_p += gate_move;
            }
        };
        load_q(0, 0);
        load_p(0, 0);
        load_q(kBlock, 1);
        lds_barrier();
        const auto block = [&](int64_t first, int own) __attribute__((always_inline)) {
            lds_barrier();
            // (Q S0)^T (rows: state columns, columns: tokens)
            fx4 o = {0, 0, 0, 0}, o2 = {0, 0, 0, 0};
            Operand<NS> p_low, p_high;
            {
                Operand<NS> so[kDepths];
#pragma unroll
                for (int d = 0; d < kDepths; ++d) so[d] = xs.get(d, lane);
                __builtin_amdgcn_sched_barrier(0);
                // P's parts while the reads are under way: later they are on the chain's way
                p_low = operand_of<NS>(p_raw[own][0][0], p_raw[own][0][1]);
                p_high = operand_of<NS>(p_raw[own][1][0], p_raw[own][1][1]);
#pragma unroll
                for (int d = 0; d < kDepths; d += 2) {
                    o = mma<NS, NI>(so[d], operand_from<NI, E>(q_raw[own][d]), o);
                    o2 = mma<NS, NI>(so[d + 1], operand_from<NI, E>(q_raw[own][d + 1]), o2);
                }
            }
            if constexpr (KEEP) {
                const Buffer to = buffer_of(state_p, first < seq_length ? (int64_t)s.dk * s.dv * 4 : 0);
#pragma unroll
                for (int t = kOwn * wave; t < kOwn * wave + kOwn; ++t)
                    put4<ElemF32>(to, quad < s.dv ? (feature_row(t, c >> 2, c & 3) * s.dv + quad) * 4 : kOutside, exchanged_row(xs, t, lane));
                state_p += (int64_t)s.heads * s.dk * s.dv * 4;
            }
            lds_barrier();
            load_p(first + kBlock, own ^ 1);
            load_q(first + 2 * kBlock, own);
            const float f = s.scale * since[own];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = f * (o[r] + o2[r]);
            lds_barrier();
            // out^T = scale (Q S0)^T diag(e^c) + U^T P^T
            int odd[4];
            __builtin_memcpy(odd, odd_at + 4 * g, 16);
            if (wave >= 2) {
                o2 = mma<NS, NS>(xu.get(1, lane), p_high, fx4{0, 0, 0, 0});
                o = mma<NS, NS>(xu.get(0, lane), p_low, o);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] += o2[r];
            } else {
                o = mma<NS, NS>(xu.get(0, lane), p_low, o);
            }
            if (__any(odd[0] < kBlock || odd[1] < kBlock || odd[2] < kBlock || odd[3] < kBlock)) {
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = token >= odd[r] ? __builtin_nanf("") : o[r];
            }
            put4<E>(rows_of(out_p, first, v_step, s.dv * kSize), quad < s.dv ? token * v_step + quad * kSize : kOutside, o);
            out_p += v_move;
            if constexpr (KEEP) {
                put4<ElemF32>(rows_of(update_p, first, u_step, s.dv * 4), quad < s.dv ? token * u_step + quad * 4 : kOutside,
                              exchanged_row(xu, wave, lane));
                update_p += (int64_t)u_step * kBlock;
            }
        };
        for (int64_t first = 0; first < seq_length; first += 2 * kBlock) {
            block(first, 0);
            block(first + kBlock, 1);
        }
    } else if (seq_length > 0) {
        // Keys, values, T and gates to LDS, three blocks ahead.
        Eight<E> k_raw[2][kCopies], v_raw[2];
        fx4 t_raw[2][kPieces];
        float gate_raw[2];
        const char *k_p = reinterpret_cast<const char*>(k + copy0), *v_p = start_of(v, v_step, v_head);
        const char* t_p = t_in + entry0 * kMatrixBytes;
        const auto load_block = [&](int64_t first, int set) __attribute__((always_inline)) {
            const Buffer kb = buffer_of(k_p, kKeyBytes), vb = rows_of(v_p, first, v_step, s.dv * kSize);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) k_raw[set][i] = fetch8<E>(kb, (tid + 256 * i) * 8 * kSize);
            const int d = col0 + (tid & 1) * 8;  // (the upper two waves repeat what the lower two do)
            v_raw[set] = fetch8<E>(vb, d < s.dv ? ((tid & 127) >> 1) * v_step + d * kSize : kOutside);
            const Buffer tb = buffer_of(t_p, kMatrixBytes);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) t_raw[set][i] = fetch16(tb, (tid + 256 * i) * 16);
            gate_raw[set] = fetch4(gates_here(), tid * 4);
            v_p += v_move;
            if (first + kBlock < seq_length) {
                k_p += k_move;
                t_p += matrix_move;
                gate_p += gate_move;
            }
        };
        typename Exchange<NS, kPairs>::Kept t_kept[kPieces];
        const auto make_parts = [&](int set) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) t_kept[i] = Exchange<NS, kPairs>::kept(t_raw[set][i]);
        };
        const auto stage_block = [&](int64_t first, int set) __attribute__((always_inline)) {
            const Tile<NI, DK> kb = keys_at(first);
#pragma unroll
            for (int i = 0; i < kCopies; ++i) kb.template put8<E>((tid + 256 * i) / (DK / 8), (tid + 256 * i) % (DK / 8) * 8, k_raw[set][i]);
            values_at(first).template put8<E>((tid & 127) >> 1, (tid & 1) * 8, v_raw[set]);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) matrix_of(first).put(4 * i + wave, lane, t_kept[i]);
            gate_of(first)[tid] = gate_raw[set];
        };
        const int groups = (s.dv + 15) / 16, row_bytes = s.dv * (int)kSize;
        int touched = 0;
        const auto touch_block = [&](int64_t first) __attribute__((always_inline)) {
            asm volatile("" ::"v"(touched));  // (what the last call asked for has to have come by now: it keeps it in the program)
            if (ahead && first < seq_length) {
                const int64_t n_block = first / kBlock, rows = seq_length - first < kBlock ? seq_length - first : kBlock;
                const char* at_k = reinterpret_cast<const char*>(k + copy0) + n_block * k_move;
                const char* at_q = reinterpret_cast<const char*>(q + copy0) + n_block * k_move;
                const Lines lines{{at_k, at_q, t_in + entry0 * kMatrixBytes + n_block * matrix_move,
                                   p_in + entry0 * kMatrixBytes + n_block * matrix_move, start_of(v, v_step, v_head) + n_block * v_move},
                                  {kKeyBytes / 128, kKeyBytes / 128, kMatrixBytes / 128, kMatrixBytes / 128,
                                   (int)rows * ((row_bytes + 127) / 128)},
                                  (row_bytes + 127) / 128, (int64_t)v_step};
                touched = touch(lines, tid * groups + col0 / 16);
            }
        };
        load_block(0, 0);
        load_block(kBlock, 1);
        make_parts(0);
        stage_block(0, 0);
        load_block(2 * kBlock, 0);
        touch_block(3 * kBlock);
        touch_block(4 * kBlock);
        lds_barrier();
        const auto block = [&](int64_t first, int other) __attribute__((always_inline)) {
            lds_barrier();
            make_parts(other);
            lds_barrier();
            stage_block(first + kBlock, other);  // the tiles' last readers are behind the first barrier
            lds_barrier();
            load_block(first + 3 * kBlock, other);
            touch_block(first + 5 * kBlock);
        };
        for (int64_t first = 0; first < seq_length; first += 2 * kBlock) {
            block(first, 1);
            block(first + kBlock, 0);
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
