// One token of the gated delta rule for many conversations, their states updated in place.
//
// The state is read and written once and everything else is small: with s = a S0,
//   u = beta (v - s^T k),   out = scale (s^T q + (q.k) u),   S1 = s + k u^T
// so both products with the old state are taken in the pass that loads it, and the new state is formed from
// the registers that hold it.  Memory bounds it: 256 conversations of 32 heads of 128 x 128 move 1.08 GB in 209 us,
// 5.2 TB/s, what a large copy reaches; one conversation takes 6.0 us, a launch and the latency of a load and a store.
#ifndef ASCAN_DELTA_STEP_H_
#define ASCAN_DELTA_STEP_H_

#include "delta.h"
#include "delta_tile.h"

namespace ascan {
namespace {

// A workgroup of 256 threads takes 4 Q columns of one head's state; a thread four columns of every
// (256 / Q)th row, at most N rows.  grid: batch x heads x column groups, column groups fastest.
template <class E, int Q, int N>
__global__ __launch_bounds__(256) void delta_step(DeltaStep p, int groups) {
    using S = typename E::S;
    constexpr int kRowStep = 256 / Q;
    __shared__ fx4 part_k[4][Q], part_q[4][Q];
    __shared__ float part_d[4];
    __shared__ int earlier, later;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = tid % Q, row0 = tid / Q;
    int64_t id = blockIdx.x;
    const int group = (int)(id % groups);
    id /= groups;
    const int head = (int)(id % p.heads), key_head = head / (p.heads / p.key_heads);
    int64_t b = id / p.heads;
    const int col = (group * Q + quad) * 4;
    const bool mine = col < p.dv;

    int64_t slot = b;
    if (p.slot != nullptr)
        slot = p.wide_slots ? static_cast<const int64_t*>(p.slot)[b] : (int64_t) static_cast<const int32_t*>(p.slot)[b];
    const bool there = slot >= 0 && slot < p.slots;
    float* state = p.states + ((there ? slot : 0) * p.heads + head) * p.dk * p.dv + col;
    fx4 s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = row0 + i * kRowStep;
        s[i] = fx4{0, 0, 0, 0};
        if (there && mine && row < p.dk) s[i] = N > 4 ? __builtin_nontemporal_load(reinterpret_cast<const fx4*>(state + (int64_t)row * p.dv)) : *reinterpret_cast<const fx4*>(state + (int64_t)row * p.dv);
    }
    for (;;) {
        int64_t next = -1;
        if (p.slot != nullptr) {
            // rows that name one slot are steps of one state, in their order: the first row's workgroup takes them all
            if (tid == 0) {
                earlier = 0;
                later = 0x7fffffff;
            }
            __syncthreads();
            for (int64_t i = tid; i < p.batch; i += 256) {
                const int64_t other = p.wide_slots ? static_cast<const int64_t*>(p.slot)[i] : (int64_t) static_cast<const int32_t*>(p.slot)[i];
                if (other == slot && i < b) earlier = 1;
                if (other == slot && i > b) atomicMin(&later, (int)i);
            }
            __syncthreads();
            if (there && b == id / p.heads && earlier) return;
            if (there && later != 0x7fffffff) next = later;
        }
        S* out = static_cast<S*>(p.out) + (b * p.heads + head) * p.dv + col;
        if (!there) {
            if (mine && row0 == 0) store4<E>(out, fx4{0, 0, 0, 0});
            return;
        }
        const S* q = static_cast<const S*>(p.q) + (b * p.key_heads + key_head) * p.dk;
        const S* k = static_cast<const S*>(p.k) + (b * p.key_heads + key_head) * p.dk;
        const int64_t gate_at = b * p.heads + head;
        const float log_gate = p.wide_gates ? static_cast<const float*>(p.log_gates)[gate_at] : E::get(static_cast<const S*>(p.log_gates)[gate_at]);
        const float beta = p.wide_gates ? static_cast<const float*>(p.beta)[gate_at] : E::get(static_cast<const S*>(p.beta)[gate_at]);
        const float a = expf(log_gate);
        fx4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
        float dot = 0.0f, kr[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = row0 + i * kRowStep;
            const bool in = row < p.dk;
            kr[i] = in ? E::get(k[in ? row : 0]) : 0.0f;
            const float qr = in ? E::get(q[in ? row : 0]) : 0.0f;
            dot += kr[i] * qr;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] *= a;
                sk[e] += kr[i] * s[i][e];
                sq[e] += qr * s[i][e];
            }
        }
#pragma unroll
        for (int d = Q; d < 64; d *= 2) {
            dot += __shfl_xor(dot, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sk[e] += __shfl_xor(sk[e], d);
                sq[e] += __shfl_xor(sq[e], d);
            }
        }
        if (lane < Q) {
            part_k[wave][lane] = sk;
            part_q[wave][lane] = sq;
        }
        if (lane == 0) part_d[wave] = dot;
        __syncthreads();
        sk = part_k[0][quad] + part_k[1][quad] + part_k[2][quad] + part_k[3][quad];
        sq = part_q[0][quad] + part_q[1][quad] + part_q[2][quad] + part_q[3][quad];
        dot = part_d[0] + part_d[1] + part_d[2] + part_d[3];
        fx4 u = {0, 0, 0, 0}, o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = mine ? E::get(static_cast<const S*>(p.v)[(b * p.heads + head) * p.dv + col + e]) : 0.0f;
            u[e] = beta * (v - sk[e]);
            o[e] = p.scale * (sq[e] + dot * u[e]);
        }
        if (mine && row0 == 0) store4<E>(out, o);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] += kr[i] * u[e];
        if (next < 0) break;
        b = next;
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = row0 + i * kRowStep;
        if (mine && row < p.dk) {
            if (N > 4) __builtin_nontemporal_store(s[i], reinterpret_cast<fx4*>(state + (int64_t)row * p.dv));
            else *reinterpret_cast<fx4*>(state + (int64_t)row * p.dv) = s[i];
        }
    }
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_STEP_H_
