// C entry points of the gated norm (include/ascan.h).
#include "ascan.h"
#include "dispatch.h"
#include "norm_kernel.h"

namespace ascan {
namespace {

int norm_status(hipError_t e) {
    if (e == hipSuccess) return ASCAN_OK;
    g_last_hip_error = (int)e;
    return ASCAN_ERR_LAUNCH;
}

// Workgroups of the backward kernel: eight to a compute unit, so that one's loads cover another's sums, where its registers let
// as many in.  With the sum over their shares, for 512, 1024, 2048 and 4096 of them (us): bf16 rows of 128 (524288) 152, 140, 139, 141;
// of 1024 (65536) 309, 226, 215, 211; of 2048 (16384) 94, 80, 79, 83; fp32 of 1000 (5001) 29, 26, 27, 31.  Rows above 2048 elements, whose
// variant leaves room for one workgroup to a compute unit, would rather have fewer, since each costs a row of the shares: bf16 of
// 4096, 16384 rows 278, 284, 294, 313 and 2048 rows 42, 47, 58, 58 (39 with 256 workgroups); of 8192 (16384) 365, 374, 397, 437.
constexpr int64_t kNormParts = 2048;

template <int L>
int64_t norm_groups(int64_t rows) { return (rows + 256 / L - 1) / (256 / L); }

// Calls f(lanes, vector, kept) with the kernel variant for rows of `width` elements: as few lanes as hold the
// row at eight elements each, vectors of eight where every row starts on 16 bytes.
template <class F>
int choose_norm(int64_t width, bool aligned, F f) {
    using std::integral_constant;
    if (aligned && width % 8 == 0) {
        integral_constant<int, 8> v;
        if (width <= 128) return f(integral_constant<int, 16>{}, v, integral_constant<int, 1>{});
        if (width <= 512) return f(integral_constant<int, 64>{}, v, integral_constant<int, 1>{});
        if (width <= 2048) return f(integral_constant<int, 256>{}, v, integral_constant<int, 1>{});
        if (width <= 8192) return f(integral_constant<int, 256>{}, v, integral_constant<int, 4>{});
        return f(integral_constant<int, 256>{}, v, integral_constant<int, 0>{});
    }
    integral_constant<int, 1> v;
    if (width <= 128) return f(integral_constant<int, 16>{}, v, integral_constant<int, 8>{});
    if (width <= 512) return f(integral_constant<int, 64>{}, v, integral_constant<int, 8>{});
    if (width <= 4096) return f(integral_constant<int, 256>{}, v, integral_constant<int, 16>{});
    return f(integral_constant<int, 256>{}, v, integral_constant<int, 0>{});
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class E>
int norm_forward_any(const void* x, const void* gate, const void* weight, void* out, int64_t rows, int64_t width,
                     float eps, hipStream_t stream) {
    using S = typename E::S;
    const bool aligned = aligned16(x) && aligned16(gate) && aligned16(weight) && aligned16(out);
    return choose_norm(width, aligned, [&](auto lanes, auto vector, auto kept) {
        constexpr int L = decltype(lanes)::value;
        const int64_t groups = norm_groups<L>(rows);
        const unsigned grid = (unsigned)(groups < (1 << 20) ? groups : (1 << 20));
        hipLaunchKernelGGL((norm_forward<E, L, decltype(vector)::value, decltype(kept)::value>), dim3(grid), dim3(256), 0,
                           stream, static_cast<const S*>(x), static_cast<const S*>(gate), static_cast<const S*>(weight),
                           static_cast<S*>(out), rows, (int)width, eps);
        return norm_status(hipGetLastError());
    });
}

int64_t norm_parts(int64_t rows, int64_t width) {
    const int64_t groups = width <= 128 ? norm_groups<16>(rows) : (width <= 512 ? norm_groups<64>(rows) : rows);
    return groups < kNormParts ? groups : kNormParts;
}

template <class E>
int norm_backward_any(const void* x, const void* gate, const void* weight, const void* d_out, void* d_x, void* d_gate,
                      void* d_weight, int64_t rows, int64_t width, float eps, float* partial, hipStream_t stream) {
    using S = typename E::S;
    const bool aligned = aligned16(x) && aligned16(gate) && aligned16(weight) && aligned16(d_out) && aligned16(d_x) &&
                         aligned16(d_gate);
    const int64_t parts = norm_parts(rows, width);
    const int status = choose_norm(width, aligned, [&](auto lanes, auto vector, auto kept) {
        hipLaunchKernelGGL((norm_backward<E, decltype(lanes)::value, decltype(vector)::value, decltype(kept)::value>),
                           dim3((unsigned)parts), dim3(256), 0, stream, static_cast<const S*>(x),
                           static_cast<const S*>(gate), static_cast<const S*>(weight), static_cast<const S*>(d_out),
                           static_cast<S*>(d_x), static_cast<S*>(d_gate), partial, rows, (int)width, eps);
        return norm_status(hipGetLastError());
    });
    if (status != ASCAN_OK) return status;
    // (up to 2^20 workgroups, which walk over the columns: an axis of a launch holds 2^32 threads, 2^26 columns)
    const int64_t columns = (width + 15) / 16;
    hipLaunchKernelGGL((norm_fold<E>), dim3((unsigned)(columns < (1 << 20) ? columns : (1 << 20))), dim3(1024), 0, stream, partial,
                       static_cast<S*>(d_weight), (int)parts, (int)width);
    return norm_status(hipGetLastError());
}

}  // namespace
}  // namespace ascan

using namespace ascan;

namespace {
int norm_element_size(int dtype) { return dtype == ASCAN_F32 ? 4 : (dtype == ASCAN_BF16 || dtype == ASCAN_F16 ? 2 : 0); }

bool norm_shape_ok(int64_t rows, int64_t width) {
    if (rows < 0 || width < 0 || width > (1 << 30)) return false;
    return width == 0 || rows <= (INT64_MAX >> 5) / width;
}

// True when [a, a + n) of one output meets [b, b + m).
bool meet(const void* a, int64_t n, const void* b, int64_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a != nullptr && b != nullptr && x < y + (uintptr_t)m && y < x + (uintptr_t)n;
}
}  // namespace

extern "C" {

int ascan_gated_norm(const void* x, const void* gate, const void* weight, void* out, int64_t rows, int64_t width,
                     float eps, int dtype, void* stream) {
    const int es = norm_element_size(dtype);
    if (es == 0) return ASCAN_ERR_BAD_DTYPE;
    if (!norm_shape_ok(rows, width)) return ASCAN_ERR_BAD_SHAPE;
    if (rows == 0 || width == 0) return ASCAN_OK;
    if (!x || !gate || !weight || !out) return ASCAN_ERR_NULL_POINTER;
    for (const void* p : {x, gate, weight, static_cast<const void*>(out)})
        if (reinterpret_cast<uintptr_t>(p) % es) return ASCAN_ERR_MISALIGNED;
    const int64_t n = rows * width * es;
    if (meet(out, n, x, n) || meet(out, n, gate, n) || meet(out, n, weight, width * es)) return ASCAN_ERR_OVERLAP;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case ASCAN_F32: return norm_forward_any<ElemF32>(x, gate, weight, out, rows, width, eps, s);
        case ASCAN_BF16: return norm_forward_any<ElemBF16>(x, gate, weight, out, rows, width, eps, s);
        default: return norm_forward_any<ElemF16>(x, gate, weight, out, rows, width, eps, s);
    }
}

size_t ascan_gated_norm_workspace_bytes(int64_t rows, int64_t width) {
    if (!norm_shape_ok(rows, width) || rows == 0 || width == 0) return 0;
    return (size_t)norm_parts(rows, width) * (size_t)width * 4;
}

int ascan_gated_norm_backward(const void* x, const void* gate, const void* weight, const void* d_out, void* d_x,
                              void* d_gate, void* d_weight, int64_t rows, int64_t width, float eps, int dtype,
                              void* workspace, size_t workspace_bytes, void* stream) {
    const int es = norm_element_size(dtype);
    if (es == 0) return ASCAN_ERR_BAD_DTYPE;
    if (!norm_shape_ok(rows, width)) return ASCAN_ERR_BAD_SHAPE;
    if (rows == 0 || width == 0) return ASCAN_OK;
    if (!x || !gate || !weight || !d_out || !d_x || !d_gate || !d_weight || !workspace) return ASCAN_ERR_NULL_POINTER;
    for (const void* p : {x, gate, weight, d_out, static_cast<const void*>(d_x), static_cast<const void*>(d_gate),
                          static_cast<const void*>(d_weight)})
        if (reinterpret_cast<uintptr_t>(p) % es) return ASCAN_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(workspace) % 4) return ASCAN_ERR_MISALIGNED;
    if (workspace_bytes < ascan_gated_norm_workspace_bytes(rows, width)) return ASCAN_ERR_WORKSPACE;
    const int64_t n = rows * width * es, m = width * es;
    struct { const void* p; int64_t bytes; } in[] = {{x, n}, {gate, n}, {weight, m}, {d_out, n}},
        out[] = {{d_x, n}, {d_gate, n}, {d_weight, m}, {workspace, (int64_t)ascan_gated_norm_workspace_bytes(rows, width)}};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 4; ++i)
            if (meet(out[o].p, out[o].bytes, in[i].p, in[i].bytes)) return ASCAN_ERR_OVERLAP;
        for (int i = o + 1; i < 4; ++i)
            if (meet(out[o].p, out[o].bytes, out[i].p, out[i].bytes)) return ASCAN_ERR_OVERLAP;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* partial = static_cast<float*>(workspace);
    switch (dtype) {
        case ASCAN_F32: return norm_backward_any<ElemF32>(x, gate, weight, d_out, d_x, d_gate, d_weight, rows, width, eps, partial, s);
        case ASCAN_BF16: return norm_backward_any<ElemBF16>(x, gate, weight, d_out, d_x, d_gate, d_weight, rows, width, eps, partial, s);
        default: return norm_backward_any<ElemF16>(x, gate, weight, d_out, d_x, d_gate, d_weight, rows, width, eps, partial, s);
    }
}

}  // extern "C"
