// Gated norm of rows, the norm behind a delta rule layer:
//
//   y = w x / r silu(z),   r = sqrt(mean(x^2) + eps),   silu(z) = z s, s = 1 / (1 + e^-z)
//
// and its gradients, with h = x / r and e = dy w silu(z):
//
//   dx = (e - h mean(e h)) / r,   dz = dy w h s (1 + z (1 - s)),   dw = sum over rows of dy h silu(z)
//
// A pass over memory: a row's values stay in the registers of the lanes that share it while their sums go
// round.  Sums and all arithmetic are fp32.  Memory bounds it: bf16, 524288 rows of 128, forward 403 MB in 77.5 us
// (5.2 TB/s, what a large copy reaches), backward 671 MB in 126 us (5.3 TB/s) and 6 us for the sums over its workgroups.
#ifndef ASCAN_NORM_KERNEL_H_
#define ASCAN_NORM_KERNEL_H_

#include "delta_tile.h"

namespace ascan {
namespace {

// V neighbouring elements of a row.
template <class E, int V>
__device__ __forceinline__ void load_values(const typename E::S* p, bool there, float (&x)[V]) {
    if constexpr (V == 8) {
        const Eight<E> r = load8<E>(p, there);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = E::get(r.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = there ? E::get(p[i]) : 0.0f;
    }
}
template <class E, int V>
__device__ __forceinline__ void store_values(typename E::S* p, const float (&x)[V]) {
    if constexpr (V == 8) {
        typename E::S s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = E::put(x[i]);
        fx4 v[sizeof(s) / 16];
        __builtin_memcpy(v, s, sizeof(s));
#pragma unroll
        for (unsigned i = 0; i < sizeof(s) / 16; ++i) reinterpret_cast<fx4*>(p)[i] = v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = E::put(x[i]);
    }
}

// Sum over the L lanes of a row, to all of them (L = 256: over the workgroup; every thread takes part).
template <int L>
__device__ __forceinline__ float row_sum(float x, float* shared) {
#pragma unroll
    for (int d = 1; d < (L < 64 ? L : 64); d *= 2) x += __shfl_xor(x, d);
    if constexpr (L > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
        __syncthreads();
        x = shared[0] + shared[1] + shared[2] + shared[3];
    }
    return x;
}

__device__ __forceinline__ float sigmoid_of(float z) { return 1.0f / (1.0f + expf(-z)); }

// L lanes to a row, V elements to a vector, N vectors of a lane kept in registers (0: any width, the row is
// read a second time).  Workgroups walk over the rows.
template <class E, int L, int V, int N>
__global__ __launch_bounds__(256) void norm_forward(const typename E::S* __restrict__ x,
                                                    const typename E::S* __restrict__ gate,
                                                    const typename E::S* __restrict__ weight,
                                                    typename E::S* __restrict__ out, int64_t rows, int width, float eps) {
    __shared__ float shared[4];
    constexpr int kRows = 256 / L;
    const int lane = threadIdx.x % L;
    for (int64_t first = (int64_t)blockIdx.x * kRows; first < rows; first += (int64_t)gridDim.x * kRows) {
        const int64_t row = first + threadIdx.x / L;
        const bool there = row < rows;
        const int64_t at = (there ? row : 0) * width;
        float sum = 0.0f;
        float xv[N > 0 ? N : 1][V], zv[N > 0 ? N : 1][V];
        if constexpr (N > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int col = (i * L + lane) * V;
                load_values<E, V>(x + at + col, there && col < width, xv[i]);
                load_values<E, V>(gate + at + col, there && col < width, zv[i]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) sum += xv[i][e] * xv[i][e];
        } else {
            for (int col = lane * V; col < width; col += L * V) {
                load_values<E, V>(x + at + col, there, xv[0]);
#pragma unroll
                for (int e = 0; e < V; ++e) sum += xv[0][e] * xv[0][e];
            }
        }
        const float inverse = 1.0f / sqrtf(row_sum<L>(sum, shared) / (float)width + eps);
        const int turns = N > 0 ? N : (width + L * V - 1) / (L * V);
#pragma unroll
        for (int i = 0; i < (N > 0 ? N : turns); ++i) {
            const int col = (i * L + lane) * V;
            if (!there || col >= width) continue;
            float w[V], y[V];
            constexpr bool kKept = N > 0;
            const int slot = kKept ? i : 0;
            if constexpr (!kKept) {
                load_values<E, V>(x + at + col, true, xv[0]);
                load_values<E, V>(gate + at + col, true, zv[0]);
            }
            load_values<E, V>(weight + col, true, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float z = zv[slot][e];
                y[e] = xv[slot][e] * inverse * w[e] * (z * sigmoid_of(z));
            }
            store_values<E, V>(out + at + col, y);
        }
    }
}

// Gradients.  Each workgroup leaves its rows' share of dw as a row of `partial`.
template <class E, int L, int V, int N>
__global__ __launch_bounds__(256) void norm_backward(const typename E::S* __restrict__ x,
                                                     const typename E::S* __restrict__ gate,
                                                     const typename E::S* __restrict__ weight,
                                                     const typename E::S* __restrict__ d_out,
                                                     typename E::S* __restrict__ d_x, typename E::S* __restrict__ d_gate,
                                                     float* __restrict__ partial, int64_t rows, int width, float eps) {
    constexpr int kRows = 256 / L, kKeep = N > 0 ? N : 1;
    __shared__ float shared[4], shared2[4];
    __shared__ float fold[kRows > 1 ? 256 * kKeep * V : 1];
    const int lane = threadIdx.x % L;
    float dw[kKeep][V], w[kKeep][V];
    float* mine = partial + (int64_t)blockIdx.x * width;
    if constexpr (N > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int col = (i * L + lane) * V;
            load_values<E, V>(weight + col, col < width, w[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) dw[i][e] = 0.0f;
        }
    } else {
        for (int col = lane * V; col < width; col += L * V)
#pragma unroll
            for (int e = 0; e < V; ++e) mine[col + e] = 0.0f;
    }
    for (int64_t first = (int64_t)blockIdx.x * kRows; first < rows; first += (int64_t)gridDim.x * kRows) {
        const int64_t row = first + threadIdx.x / L;
        const bool there = row < rows;
        const int64_t at = (there ? row : 0) * width;
        float sum = 0.0f, cross = 0.0f;
        float xv[kKeep][V], zv[kKeep][V], dv[kKeep][V];
        const int turns = N > 0 ? N : (width + L * V - 1) / (L * V);
        if constexpr (N > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int col = (i * L + lane) * V;
                const bool in = there && col < width;
                load_values<E, V>(x + at + col, in, xv[i]);
                load_values<E, V>(gate + at + col, in, zv[i]);
                load_values<E, V>(d_out + at + col, in, dv[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < (N > 0 ? N : turns); ++i) {
            const int col = (i * L + lane) * V, slot = N > 0 ? i : 0;
            if constexpr (N == 0) {
                const bool in = there && col < width;
                load_values<E, V>(x + at + col, in, xv[0]);
                load_values<E, V>(gate + at + col, in, zv[0]);
                load_values<E, V>(d_out + at + col, in, dv[0]);
                load_values<E, V>(weight + col, in, w[0]);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xe = xv[slot][e], z = zv[slot][e];
                sum += xe * xe;
                cross += dv[slot][e] * w[slot][e] * (z * sigmoid_of(z)) * xe;
            }
        }
        sum = row_sum<L>(sum, shared);
        cross = row_sum<L>(cross, shared2);
        const float inverse = 1.0f / sqrtf(sum / (float)width + eps);
        const float mean = cross * inverse / (float)width;  // of e h
#pragma unroll
        for (int i = 0; i < (N > 0 ? N : turns); ++i) {
            const int col = (i * L + lane) * V, slot = N > 0 ? i : 0;
            if (!there || col >= width) continue;
            if constexpr (N == 0) {
                load_values<E, V>(x + at + col, true, xv[0]);
                load_values<E, V>(gate + at + col, true, zv[0]);
                load_values<E, V>(d_out + at + col, true, dv[0]);
                load_values<E, V>(weight + col, true, w[0]);
            }
            float gx[V], gz[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float z = zv[slot][e], s = sigmoid_of(z), d = dv[slot][e], h = xv[slot][e] * inverse;
                gx[e] = (d * w[slot][e] * (z * s) - h * mean) * inverse;
                gz[e] = d * w[slot][e] * h * (s * (1.0f + z * (1.0f - s)));
                const float g = d * h * (z * s);
                if constexpr (N > 0) dw[slot][e] += g;
                else mine[col + e] += g;
            }
            store_values<E, V>(d_x + at + col, gx);
            store_values<E, V>(d_gate + at + col, gz);
        }
    }
    if constexpr (N > 0 && kRows > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) fold[(threadIdx.x / L) * (L * N * V) + (i * L + lane) * V + e] = dw[i][e];
        __syncthreads();
        for (int col = threadIdx.x; col < width; col += 256) {
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < kRows; ++r) sum += fold[r * (L * N * V) + col];
            mine[col] = sum;
        }
    } else if constexpr (N > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int col = (i * L + lane) * V;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col < width) mine[col + e] = dw[i][e];
        }
    }
}

// dw from the workgroups' shares: 16 columns to a workgroup, 64 threads to a column, always in one order.  (With 64
// columns and 16 threads each, 1024 shares took 17 us, mostly one load after the other.)
template <class E>
__global__ __launch_bounds__(1024) void norm_fold(const float* __restrict__ partial, typename E::S* __restrict__ d_weight,
                                                  int parts, int width) {
    __shared__ float sums[64][17];
    const int lane = threadIdx.x & 15, strip = threadIdx.x >> 4;
    for (int first = blockIdx.x * 16; first < width; first += gridDim.x * 16) {
        const int col = first + lane;
        float sum = 0.0f;
        if (col < width) {
#pragma unroll 4
            for (int i = strip; i < parts; i += 64) sum += partial[(int64_t)i * width + col];
        }
        sums[strip][lane] = sum;
        __syncthreads();
        if (threadIdx.x < 256) {  // 16 threads to a column, four strips each, then across
            const int at = threadIdx.x & 15, c = threadIdx.x >> 4;
            float all = (sums[at][c] + sums[at + 16][c]) + (sums[at + 32][c] + sums[at + 48][c]);
            all = sum16(all);
            if (at == 0 && first + c < width) d_weight[first + c] = E::put(all);
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_NORM_KERNEL_H_
