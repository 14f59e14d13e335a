// Gated delta rule: what the C entry points (delta.hip) call and what the kernels share.
//
//   S[t] = a[t] S[t-1] + beta[t] k[t] (v[t] - (a[t] S[t-1])^T k[t])^T,   out[t] = scale S[t]^T q[t]
//
// A block of 64 tokens that starts from the state S0 is solved at once.  With c the running sum of the
// block's log gates and U the rows u[i] = beta[i] (v[i] - ...) that the tokens add to the state,
//
//   (I + L) U = R = diag(beta) V - diag(beta e^c) K S0,     L[i][j] = beta[i] e^(c[i]-c[j]) k[i].k[j],  j < i
//   out       = scale diag(e^c) Q S0 + P U,                 P[i][j] = scale e^(c[i]-c[j]) q[i].k[j],    j <= i
//   S1        = e^c[63] S0 + K^T diag(e^(c[63]-c)) U
//
// (I + L)^-1 = I + T and P depend on keys, queries and gates alone: a first kernel makes them for all
// blocks at once.  What is left is a chain over the blocks of a sequence, one per head and column of
// the state: columns are independent.
#ifndef ASCAN_DELTA_H_
#define ASCAN_DELTA_H_

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ascan {

struct DeltaShape {
    int64_t rows;      // tokens of all sequences together (with the ones outside every sequence)
    int64_t tokens;    // tokens of a sequence where offsets is null
    int64_t sequences;
    int64_t blocks;    // of all sequences: table entries (some unused where offsets is given)
    int heads, key_heads, dk, dv;
    const void* offsets;  // sequences + 1 row numbers, or null
    bool wide_offsets;    // int64, else int32
    bool wide_gates;      // log gates and beta are fp32, else of the tensors' type
    float scale;
};

// Blocks that the sequences of a call can have: those of packed sequences are numbered from
// offset / 64 + sequence, which leaves every one room for its last, partial block.
inline int64_t delta_blocks(int64_t rows, int64_t sequences, bool packed) {
    if (packed) return rows / 64 + sequences;
    return sequences == 0 ? 0 : (rows / sequences + 63) / 64 * sequences;
}

struct DeltaForward {
    DeltaShape shape;
    const void *q, *k, *v, *log_gates, *beta;
    const float* initial;  // or null
    void* out;
    float* final;          // or null
    float* states;         // or null: the state in front of every block, for the backward pass
    float* updates;        // or null: the rows U, for the backward pass
    char* workspace;
    hipStream_t stream;
};

struct DeltaBackward {
    DeltaShape shape;
    const void *q, *k, *v, *log_gates, *beta;
    const float *states, *updates;
    const void* d_out;       // or null
    const float* d_final;    // or null
    void *d_q, *d_k, *d_v, *d_log_gates, *d_beta;
    float* d_initial;        // or null
    char* workspace;
    hipStream_t stream;
};

struct DeltaStep {
    int64_t batch, slots;
    int heads, key_heads, dk, dv;
    const void *q, *k, *v, *log_gates, *beta;
    float* states;
    const void* slot;     // batch slot numbers, or null: row b uses state b
    bool wide_slots, wide_gates;
    float scale;
    void* out;
    hipStream_t stream;
};

// Each returns an ascan_status; the workspace sizes are in bytes.
int delta_forward_f32(const DeltaForward&);
int delta_forward_bf16(const DeltaForward&);
int delta_forward_f16(const DeltaForward&);
int delta_backward_f32(const DeltaBackward&);
int delta_backward_bf16(const DeltaBackward&);
int delta_backward_f16(const DeltaBackward&);
int delta_step_f32(const DeltaStep&);
int delta_step_bf16(const DeltaStep&);
int delta_step_f16(const DeltaStep&);
size_t delta_workspace_f32(const DeltaShape&, bool backward);
size_t delta_workspace_bf16(const DeltaShape&, bool backward);
size_t delta_workspace_f16(const DeltaShape&, bool backward);

}  // namespace ascan

#endif  // ASCAN_DELTA_H_
