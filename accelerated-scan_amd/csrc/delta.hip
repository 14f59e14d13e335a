// C entry points of the gated delta rule (include/ascan.h).
#include "ascan.h"
#include "delta.h"
#include "dispatch.h"

using namespace ascan;

namespace {

int element_bytes(int dtype) { return dtype == ASCAN_F32 ? 4 : (dtype == ASCAN_BF16 || dtype == ASCAN_F16 ? 2 : 0); }

constexpr int64_t kMaxHeads = 65535, kMaxRows = INT64_C(1) << 40, kMaxSequences = 65535;
constexpr int64_t kMaxKeyDim = 128, kMaxValueDim = 4096;
constexpr int64_t kMaxRowElements = INT64_C(1) << 22;  // of a token: 64 tokens stay below 2^31 bytes
constexpr int64_t kMaxThreads = INT64_C(4294967295);   // of an axis of a launch

bool heads_ok(int64_t heads, int64_t key_heads, int64_t dk, int64_t dv) {
    return heads > 0 && heads <= kMaxHeads && key_heads > 0 && heads % key_heads == 0 && dk > 0 && dk <= kMaxKeyDim &&
           dk % 8 == 0 && dv > 0 && dv <= kMaxValueDim && dv % 8 == 0 &&
           heads * dv <= kMaxRowElements && key_heads * dk <= kMaxRowElements;
}

bool rows_ok(int64_t rows, int64_t sequences, bool packed) {
    if (rows < 0 || sequences < 0 || rows > kMaxRows || sequences > kMaxSequences) return false;
    if (!packed && (sequences == 0 ? rows != 0 : rows % sequences != 0)) return false;
    return delta_blocks(rows, sequences, packed) <= kMaxThreads / 512;
}
// Workgroups of the chains: one to 16 columns of every sequence's every head, in whole rounds of eight.
bool chains_ok(int64_t sequences, int64_t heads, int64_t dv) {
    return ((sequences * heads + 7) / 8 * 8) * ((dv + 15) / 16) <= kMaxThreads / 768;
}

bool misaligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

struct Range {
    const void* p;
    int64_t bytes;
};
bool meet(const Range& a, const Range& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.p != nullptr && b.p != nullptr && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
template <size_t NI, size_t NO>
bool outputs_meet(const Range (&in)[NI], const Range (&out)[NO]) {
    for (size_t o = 0; o < NO; ++o) {
        for (size_t i = 0; i < NI; ++i)
            if (meet(out[o], in[i])) return true;
        for (size_t i = o + 1; i < NO; ++i)
            if (meet(out[o], out[i])) return true;
    }
    return false;
}

DeltaShape shape_of(const void* offsets, int64_t rows, int64_t sequences, int64_t heads, int64_t key_heads, int64_t dk,
                    int64_t dv, float scale, int flags) {
    DeltaShape s;
    s.rows = rows;
    s.sequences = sequences;
    s.tokens = offsets == nullptr && sequences > 0 ? rows / sequences : 0;
    s.blocks = delta_blocks(rows, sequences, offsets != nullptr);
    s.heads = (int)heads;
    s.key_heads = (int)key_heads;
    s.dk = (int)dk;
    s.dv = (int)dv;
    s.offsets = offsets;
    s.wide_offsets = (flags & ASCAN_DELTA_OFFSETS_I64) != 0;
    s.wide_gates = (flags & ASCAN_DELTA_GATES_F32) != 0;
    s.scale = scale;
    return s;
}

size_t workspace_of(const DeltaShape& s, int dtype, bool backward) {
    switch (dtype) {
        case ASCAN_F32: return delta_workspace_f32(s, backward);
        case ASCAN_BF16: return delta_workspace_bf16(s, backward);
        default: return delta_workspace_f16(s, backward);
    }
}

// What both passes check of a call; `s` is filled where it is fine.
int check_scan(const void* const* inputs, size_t count, int64_t rows, int64_t sequences, int64_t heads, int64_t key_heads,
               int64_t dk, int64_t dv, int dtype, int flags, const void* offsets, int gate_bytes) {
    if (element_bytes(dtype) == 0) return ASCAN_ERR_BAD_DTYPE;
    if (!heads_ok(heads, key_heads, dk, dv)) return ASCAN_ERR_BAD_HEADS;
    if (!rows_ok(rows, sequences, offsets != nullptr) || !chains_ok(sequences, heads, dv)) return ASCAN_ERR_BAD_SHAPE;
    if (misaligned(offsets, flags & ASCAN_DELTA_OFFSETS_I64 ? 8 : 4)) return ASCAN_ERR_MISALIGNED;
    if (rows > 0 && sequences > 0) {
        for (size_t i = 0; i < count; ++i) {
            if (inputs[i] == nullptr) return ASCAN_ERR_NULL_POINTER;
            // gates are read by themselves, everything else 16 bytes at a time
            if (misaligned(inputs[i], i < 2 ? gate_bytes : 16)) return ASCAN_ERR_MISALIGNED;
        }
    }
    return ASCAN_OK;
}

// Two bytes to a thread: every output is a whole number of them.
__global__ __launch_bounds__(256) void zero_kernel(uint16_t* p, int64_t n) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += gridDim.x * (int64_t)256) p[i] = 0;
}

// A call whose offsets hold no sequence: all rows are outside, outputs are zero.  (A kernel, so that a graph can have it.)
template <size_t NI, size_t NO>
int zero_outputs(const Range (&in)[NI], const Range (&out)[NO], size_t alignment, void* stream) {
    for (const Range& o : out) {
        if (o.p == nullptr) return ASCAN_ERR_NULL_POINTER;
        if (misaligned(o.p, alignment)) return ASCAN_ERR_MISALIGNED;
    }
    if (outputs_meet(in, out)) return ASCAN_ERR_OVERLAP;
    for (const Range& o : out) {
        const int64_t groups = (o.bytes / 2 + 255) / 256;
        hipLaunchKernelGGL(zero_kernel, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, static_cast<hipStream_t>(stream),
                           static_cast<uint16_t*>(const_cast<void*>(o.p)), o.bytes / 2);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            g_last_hip_error = (int)e;
            return ASCAN_ERR_LAUNCH;
        }
    }
    return ASCAN_OK;
}

}  // namespace

extern "C" {

int64_t ascan_delta_blocks(int64_t rows, int64_t sequences, int packed) {
    return rows_ok(rows, sequences, packed != 0) ? delta_blocks(rows, sequences, packed != 0) : -1;
}

size_t ascan_delta_workspace_bytes(int64_t rows, int64_t sequences, int64_t heads, int64_t key_heads, int64_t dk,
                                   int64_t dv, int dtype, int packed, int backward) {
    if (element_bytes(dtype) == 0 || !heads_ok(heads, key_heads, dk, dv) || !rows_ok(rows, sequences, packed != 0) ||
        !chains_ok(sequences, heads, dv))
        return 0;
    static const int32_t some = 0;  // only whether there are offsets counts here
    return workspace_of(shape_of(packed ? &some : nullptr, rows, sequences, heads, key_heads, dk, dv, 1.0f, 0), dtype, backward != 0);
}

int ascan_delta_forward(const void* q, const void* k, const void* v, const void* log_gates, const void* beta,
                        const float* initial, const void* offsets, void* out, float* final, float* states,
                        float* updates, int64_t rows, int64_t sequences, int64_t heads, int64_t key_heads, int64_t dk,
                        int64_t dv, float scale, int dtype, int flags, void* workspace, size_t workspace_bytes,
                        void* stream) {
    const int es = element_bytes(dtype), gs = flags & ASCAN_DELTA_GATES_F32 ? 4 : es;
    const void* needed[] = {log_gates, beta, q, k, v, out};
    const int status = check_scan(needed, 6, rows, sequences, heads, key_heads, dk, dv, dtype, flags, offsets, gs);
    if (status != ASCAN_OK) return status;
    if (sequences == 0 && rows > 0) {  // (packed: others have no rows then)
        const Range in[] = {{q, rows * key_heads * dk * es}, {k, rows * key_heads * dk * es}, {v, rows * heads * dv * es},
                            {log_gates, rows * heads * gs}, {beta, rows * heads * gs}};
        const Range to[] = {{out, rows * heads * dv * es}};
        return zero_outputs(in, to, es, stream);
    }
    if (sequences == 0 || (rows == 0 && final == nullptr)) return ASCAN_OK;
    for (const void* p : {static_cast<const void*>(initial), static_cast<const void*>(final),
                          static_cast<const void*>(states), static_cast<const void*>(updates)})
        if (misaligned(p, 16)) return ASCAN_ERR_MISALIGNED;
    const DeltaShape s = shape_of(offsets, rows, sequences, heads, key_heads, dk, dv, scale, flags);
    const int64_t need = (int64_t)workspace_of(s, dtype, false);
    if (need > 0 && workspace == nullptr) return ASCAN_ERR_NULL_POINTER;
    if ((int64_t)workspace_bytes < need) return ASCAN_ERR_WORKSPACE;
    if (misaligned(workspace, 16)) return ASCAN_ERR_MISALIGNED;
    const int64_t state = sequences * heads * dk * dv * 4;
    const Range in[] = {{q, rows * key_heads * dk * es}, {k, rows * key_heads * dk * es}, {v, rows * heads * dv * es},
                        {log_gates, rows * heads * gs}, {beta, rows * heads * gs}, {initial, state},
                        {offsets, (sequences + 1) * (s.wide_offsets ? 8 : 4)}};
    const Range to[] = {{out, rows * heads * dv * es}, {final, state}, {states, s.blocks * heads * dk * dv * 4},
                        {updates, rows * heads * dv * 4}, {workspace, need}};
    if (outputs_meet(in, to)) return ASCAN_ERR_OVERLAP;
    if (rows > 0 && (states == nullptr) != (updates == nullptr)) return ASCAN_ERR_NULL_POINTER;
    const DeltaForward f{s, q, k, v, log_gates, beta, initial, out, final, states, updates,
                         static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
    switch (dtype) {
        case ASCAN_F32: return delta_forward_f32(f);
        case ASCAN_BF16: return delta_forward_bf16(f);
        default: return delta_forward_f16(f);
    }
}

int ascan_delta_backward(const void* q, const void* k, const void* v, const void* log_gates, const void* beta,
                         const float* states, const float* updates, const void* offsets, const void* d_out,
                         const float* d_final, void* d_q, void* d_k, void* d_v, void* d_log_gates, void* d_beta,
                         float* d_initial, int64_t rows, int64_t sequences, int64_t heads, int64_t key_heads, int64_t dk,
                         int64_t dv, float scale, int dtype, int flags, void* workspace, size_t workspace_bytes,
                         void* stream) {
    const int es = element_bytes(dtype), gs = flags & ASCAN_DELTA_GATES_F32 ? 4 : es;
    const void* needed[] = {log_gates, beta, q, k, v, states, updates, d_q, d_k, d_v};
    const int status = check_scan(needed, 10, rows, sequences, heads, key_heads, dk, dv, dtype, flags, offsets, gs);
    if (status != ASCAN_OK) return status;
    if (sequences == 0 && rows > 0) {
        const Range in[] = {{q, rows * key_heads * dk * es}, {k, rows * key_heads * dk * es}, {v, rows * heads * dv * es},
                            {log_gates, rows * heads * gs}, {beta, rows * heads * gs}, {d_out, rows * heads * dv * es}};
        const Range to[] = {{d_q, rows * key_heads * dk * es}, {d_k, rows * key_heads * dk * es}, {d_v, rows * heads * dv * es},
                            {d_log_gates, rows * heads * gs}, {d_beta, rows * heads * gs}};
        return zero_outputs(in, to, es, stream);
    }
    if (sequences == 0 || (rows == 0 && d_initial == nullptr)) return ASCAN_OK;
    if (rows > 0 && (d_log_gates == nullptr || d_beta == nullptr)) return ASCAN_ERR_NULL_POINTER;
    if (misaligned(d_log_gates, gs) || misaligned(d_beta, gs)) return ASCAN_ERR_MISALIGNED;
    for (const void* p : {static_cast<const void*>(d_out), static_cast<const void*>(d_final), static_cast<const void*>(d_initial)})
        if (misaligned(p, 16)) return ASCAN_ERR_MISALIGNED;
    const DeltaShape s = shape_of(offsets, rows, sequences, heads, key_heads, dk, dv, scale, flags);
    const int64_t need = (int64_t)workspace_of(s, dtype, true);
    if (need > 0 && workspace == nullptr) return ASCAN_ERR_NULL_POINTER;
    if ((int64_t)workspace_bytes < need) return ASCAN_ERR_WORKSPACE;
    if (misaligned(workspace, 16)) return ASCAN_ERR_MISALIGNED;
    const int64_t state = sequences * heads * dk * dv * 4, qk = rows * key_heads * dk * es, vo = rows * heads * dv * es;
    const Range in[] = {{q, qk}, {k, qk}, {v, vo}, {log_gates, rows * heads * gs}, {beta, rows * heads * gs},
                        {states, s.blocks * heads * dk * dv * 4}, {updates, rows * heads * dv * 4}, {d_out, vo},
                        {d_final, state}, {offsets, (sequences + 1) * (s.wide_offsets ? 8 : 4)}};
    const Range to[] = {{d_q, qk}, {d_k, qk}, {d_v, vo}, {d_log_gates, rows * heads * gs}, {d_beta, rows * heads * gs},
                        {d_initial, state}, {workspace, need}};
    if (outputs_meet(in, to)) return ASCAN_ERR_OVERLAP;
    const DeltaBackward f{s, q, k, v, log_gates, beta, states, updates, d_out, d_final, d_q, d_k, d_v, d_log_gates,
                          d_beta, d_initial, static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
    switch (dtype) {
        case ASCAN_F32: return delta_backward_f32(f);
        case ASCAN_BF16: return delta_backward_bf16(f);
        default: return delta_backward_f16(f);
    }
}

int ascan_delta_step(const void* q, const void* k, const void* v, const void* log_gates, const void* beta, float* states,
                     const void* slots, void* out, int64_t batch, int64_t state_count, int64_t heads, int64_t key_heads,
                     int64_t dk, int64_t dv, float scale, int dtype, int flags, void* stream) {
    const int es = element_bytes(dtype), gs = flags & ASCAN_DELTA_GATES_F32 ? 4 : es;
    if (es == 0) return ASCAN_ERR_BAD_DTYPE;
    if (!heads_ok(heads, key_heads, dk, dv)) return ASCAN_ERR_BAD_HEADS;
    if (batch < 0 || state_count < 0 || state_count > INT64_MAX / 4 / (heads * dk * dv) ||
        batch > kMaxThreads / 256 / (heads * ((dv + 31) / 32)))
        return ASCAN_ERR_BAD_SHAPE;
    if (slots == nullptr && batch > state_count) return ASCAN_ERR_BAD_SHAPE;
    if (batch == 0) return ASCAN_OK;
    if (!q || !k || !v || !log_gates || !beta || !out || (!states && state_count > 0)) return ASCAN_ERR_NULL_POINTER;
    for (const void* p : {q, k, v, static_cast<const void*>(out), static_cast<const void*>(states)})
        if (misaligned(p, 16)) return ASCAN_ERR_MISALIGNED;
    if (misaligned(log_gates, gs) || misaligned(beta, gs) || misaligned(slots, flags & ASCAN_DELTA_OFFSETS_I64 ? 8 : 4))
        return ASCAN_ERR_MISALIGNED;
    const int64_t qk = batch * key_heads * dk * es, vo = batch * heads * dv * es;
    const Range in[] = {{q, qk}, {k, qk}, {v, vo}, {log_gates, batch * heads * gs}, {beta, batch * heads * gs},
                        {slots, batch * (flags & ASCAN_DELTA_OFFSETS_I64 ? 8 : 4)}};
    const Range to[] = {{out, vo}, {states, state_count * heads * dk * dv * 4}};
    if (outputs_meet(in, to)) return ASCAN_ERR_OVERLAP;
    const DeltaStep p{batch, state_count, (int)heads, (int)key_heads, (int)dk, (int)dv, q, k, v, log_gates, beta, states,
                      slots, (flags & ASCAN_DELTA_OFFSETS_I64) != 0, (flags & ASCAN_DELTA_GATES_F32) != 0, scale, out,
                      static_cast<hipStream_t>(stream)};
    switch (dtype) {
        case ASCAN_F32: return delta_step_f32(p);
        case ASCAN_BF16: return delta_step_bf16(p);
        default: return delta_step_f16(p);
    }
}

}  // extern "C"
