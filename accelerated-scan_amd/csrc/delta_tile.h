// Building blocks of the gated delta rule kernels: blocks of 64 tokens in LDS, operands of the
// matrix instructions and their products.
//
// All products are chains of 16x16 tiles.  The accumulator of a tile holds, in lane l with
// g = l / 16, column l % 16 and rows 4g .. 4g+3; an operand of a product of depth 32 holds, in lane
// l, one row (left) or column (right) l % 16 and eight values of the depth axis.  The order of the
// depth axis is free as long as both operands use the same one, so the accumulators of two stacked
// tiles ARE an operand of the next product: lane group g holds rows 4g .. 4g+3 of either tile.  What stands for
// depths 32n .. 32n+31 there depends on what the tiles' rows are:
//   - tokens: the tiles are rows 32n .. +15 and 32n+16 .. +31, the other operand is read `down` a column of a
//     row-major tile with the transposing LDS read;
//   - features: the rows of the two tiles are dealt out in fours, row 4g+r of tile i being feature
//     32n + 8g + 4i + r (`feature_row`), so that the other operand is 16 neighbouring bytes `along` a row.
//
// Arithmetic (parameter P of an operand, its number of parts):
//   P = 0   fp32 values and fp32 matrix instructions, 256 operations per clock and compute unit;
//   P >= 1  a value is the sum of P bfloat16 parts (8 bits each: one part holds a bfloat16 value, two a
//           half value without loss, three an fp32 value to 2^-24), products are
//           summed over the pairs of parts that count, at 4096 operations per clock and pair.
// Tensors of 16 bits are taken in the parts that hold them, everything computed in three: states, their gradients and those
// of fp32 gates leave in 32 bits, and in two parts they were off by 0.7 to 6e-6 (with equal keys, whose U is a small difference
// of large terms, a state by 6e-5) where fp32 arithmetic gives 1 to 3e-7, and 16-bit outputs by a last bit ten times as often.
// Three parts throughout cost a bf16 prompt (1, 16384, 32 heads of 128 x 128) 430 -> 515 us, 16 packed fp16 sequences (12291
// tokens, 16 heads) 295 -> 365, a training step (bf16, 2 x 4096, 16 heads) 567 -> 594.
#ifndef ASCAN_DELTA_TILE_H_
#define ASCAN_DELTA_TILE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ascan {
namespace {

typedef float fx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bx4 __attribute__((ext_vector_type(4)));
typedef _Float16 hx4 __attribute__((ext_vector_type(4)));
typedef short sx4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 64;          // tokens of a block
constexpr int kTiles = kBlock / 16;
constexpr int kPairs = 6;           // products of depth 32 in a triangular 64 x 64 matrix of 16 x 16 tiles

template <int P>
struct Operand {
    bx8 p[P];
};
template <>
struct Operand<0> {
    fx4 t[2];
};

// Two values as parts, each the rounding (to nearest even) of what the earlier ones leave; the pair of part i as
// a word, from which both come back as fp32 with one operation.
template <int P>
__device__ __forceinline__ void pair_parts(float a, float b, uint32_t (&w)[P]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const f2 x = {a, b};
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, b2));
        if (i + 1 < P) {
            a -= __builtin_bit_cast(float, w[i] << 16);
            b -= __builtin_bit_cast(float, w[i] & 0xffff0000u);
        }
    }
}
// Elements e .. e+3 of an operand.
template <int P>
__device__ __forceinline__ void set_parts4(Operand<P>& o, int e, const fx4& x) {
    uint32_t low[P], high[P];
    pair_parts<P>(x[0], x[1], low);
    pair_parts<P>(x[2], x[3], high);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        uint32_t w[4];
        __builtin_memcpy(w, &o.p[i], 16);
        w[e / 2] = low[i];
        w[e / 2 + 1] = high[i];
        __builtin_memcpy(&o.p[i], w, 16);
    }
}

// Two stacked accumulator tiles as an operand.
template <int P>
__device__ __forceinline__ Operand<P> operand_of(const fx4& a, const fx4& b) {
    Operand<P> o;
    if constexpr (P == 0) {
        o.t[0] = a;
        o.t[1] = b;
    } else {
        set_parts4<P>(o, 0, a);
        set_parts4<P>(o, 4, b);
    }
    return o;
}

// c + a * b over 32 depths.  Pairs of parts below the last bit kept of the product are left out:
// part i of a has weight 2^-8i.
template <int PA, int PB>
__device__ __forceinline__ fx4 mma(const Operand<PA>& a, const Operand<PB>& b, fx4 c) {
    if constexpr (PA == 0) {
        static_assert(PB == 0, "operands of one kind");
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.t[t][r], b.t[t][r], c, 0, 0, 0);
    } else {
        constexpr int M = PA > PB ? PA : PB;
#pragma unroll
        for (int s = M - 1; s >= 0; --s)
#pragma unroll
            for (int i = 0; i < PA; ++i)
                if (s - i >= 0 && s - i < PB)
                    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[s - i], c, 0, 0, 0);
    }
    return c;
}

// The same over all pairs of parts: for two half values, whose second parts' product is as large as 2^-18.
template <int PA, int PB>
__device__ __forceinline__ fx4 mma_all(const Operand<PA>& a, const Operand<PB>& b, fx4 c) {
    if constexpr (PA == 0) {
        return mma<PA, PB>(a, b, c);
    } else {
#pragma unroll
        for (int s = PA + PB - 2; s >= 0; --s)
#pragma unroll
            for (int i = 0; i < PA; ++i)
                if (s - i >= 0 && s - i < PB)
                    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[s - i], c, 0, 0, 0);
        return c;
    }
}

// ---------------------------------------------------------------------------
// Elements in memory
// ---------------------------------------------------------------------------
struct ElemF32 {
    using S = float;
    static constexpr bool kWide = true;
    static __device__ __forceinline__ float get(S s) { return s; }
    static __device__ __forceinline__ S put(float x) { return x; }
};
struct ElemBF16 {
    using S = __bf16;
    static constexpr bool kWide = false;
    static __device__ __forceinline__ float get(S s) { return (float)s; }
    static __device__ __forceinline__ S put(float x) { return (__bf16)x; }
};
struct ElemF16 {
    using S = _Float16;
    static constexpr bool kWide = false;
    static __device__ __forceinline__ float get(S s) { return (float)s; }
    static __device__ __forceinline__ S put(float x) { return (_Float16)x; }
};

// Eight neighbouring elements, as they travel from memory to LDS (16 or 32 aligned bytes).
template <class E>
struct Eight {
    typename E::S v[8];
};
template <class E>
__device__ __forceinline__ Eight<E> load8(const typename E::S* p, bool there) {
    Eight<E> r;
    if (there) {
        if constexpr (E::kWide) {
            const fx4 a = *reinterpret_cast<const fx4*>(p), b = *reinterpret_cast<const fx4*>(p + 4);
            __builtin_memcpy(&r.v[0], &a, 16);
            __builtin_memcpy(&r.v[4], &b, 16);
        } else {
            const fx4 a = *reinterpret_cast<const fx4*>(p);
            __builtin_memcpy(&r.v[0], &a, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = E::put(0.0f);
    }
    return r;
}

// ---------------------------------------------------------------------------
// Memory through buffer descriptors, whose hardware bounds check stands in for conditions: a load beyond the end
// gives zero, a store there is dropped.  Without branches around them the compiler counts the requests in flight
// and waits for the one it needs only; with them it waits for all.
// ---------------------------------------------------------------------------
typedef __amdgpu_buffer_rsrc_t Buffer;
typedef uint32_t ux2 __attribute__((ext_vector_type(2)));
typedef uint32_t ux4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kOutside = 0x7ffffff0u;  // an offset beyond every buffer

// `p` and `bytes` (below 2^31) the same in all lanes.
__device__ __forceinline__ Buffer buffer_of(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes < 0 ? 0 : (int)bytes, 0x00027000);
}
__device__ __forceinline__ fx4 fetch16(Buffer b, uint32_t at) {
    return __builtin_bit_cast(fx4, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0));
}
__device__ __forceinline__ float fetch4(Buffer b, uint32_t at) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0));
}
// Eight neighbouring elements at byte `at`.
template <class E>
__device__ __forceinline__ Eight<E> fetch8(Buffer b, uint32_t at) {
    Eight<E> r;
    const fx4 x = fetch16(b, at);
    __builtin_memcpy(&r.v[0], &x, 16);
    if constexpr (E::kWide) {
        const fx4 y = fetch16(b, at + 16);
        __builtin_memcpy(&r.v[4], &y, 16);
    }
    return r;
}
// Four neighbouring values to byte `at`.
template <class E>
__device__ __forceinline__ void put4(Buffer b, uint32_t at, const fx4& x) {
    typename E::S s[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = E::put(x[r]);
    if constexpr (E::kWide) {
        ux4 v;
        __builtin_memcpy(&v, s, 16);
        __builtin_amdgcn_raw_buffer_store_b128(v, b, at, 0, 0);
    } else {
        ux2 v;
        __builtin_memcpy(&v, s, 8);
        __builtin_amdgcn_raw_buffer_store_b64(v, b, at, 0, 0);
    }
}
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

template <int P, class E>
__device__ __forceinline__ Operand<P> operand_from(const Eight<E>& x) {
    Operand<P> o;
    if constexpr (P == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o.t[0][i] = E::get(x.v[i]);
            o.t[1][i] = E::get(x.v[i + 4]);
        }
    } else if constexpr (P == 1) {
        static_assert(sizeof(typename E::S) == 2, "one part holds a bfloat16 value");
        __builtin_memcpy(&o.p[0], x.v, 16);
    } else {
        fx4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = E::get(x.v[i]);
            b[i] = E::get(x.v[i + 4]);
        }
        o = operand_of<P>(a, b);
    }
    return o;
}

template <class E>
__device__ __forceinline__ void store8(typename E::S* p, const Eight<E>& x) {
    fx4 v[sizeof(x.v) / 16];
    __builtin_memcpy(v, x.v, sizeof(x.v));
#pragma unroll
    for (unsigned i = 0; i < sizeof(x.v) / 16; ++i) reinterpret_cast<fx4*>(p)[i] = v[i];
}

// Four neighbouring values to memory.
template <class E>
__device__ __forceinline__ void store4(typename E::S* p, const fx4& x) {
    typename E::S s[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = E::put(x[r]);
    if constexpr (E::kWide) {
        fx4 v;
        __builtin_memcpy(&v, s, 16);
        *reinterpret_cast<fx4*>(p) = v;
    } else {
        uint64_t v;
        __builtin_memcpy(&v, s, 8);
        *reinterpret_cast<uint64_t*>(p) = v;
    }
}

// Feature that row 4g + r of state tile t stands for.
__device__ __forceinline__ constexpr int feature_row(int t, int g, int r) { return 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r; }

// ---------------------------------------------------------------------------
// 64 rows of W values in LDS, as fp32 (P = 0, rows padded by 16 bytes) or as P planes of bfloat16 parts.  The planes'
// rows have no padding; their 16-byte pieces change places instead, so that neither the 16 rows of an operand (a piece of
// each) nor the four rows of a transposing read (four pieces of each, every one 16 or 32 bytes on) meet in a bank.
// ---------------------------------------------------------------------------
template <int P, int W>
struct Tile {
    static constexpr int kStride = W;  // (rows of 16 values: four of them are the 128 bytes of a transposing read)
    static constexpr int kPlane = kBlock * kStride;
    static constexpr int kBytes = P * kPlane * 2;
    __bf16* base;

    // Where element (row, col) stands; columns col .. col+7 stay together for col a multiple of 8.
    static __device__ __forceinline__ int place(int row, int col) {
        if constexpr (W < 64) return row * kStride + col;
        const int turn = W >= 128 ? (row & 3) * 4 + ((row >> 2) & 3) : (row & 2) * 2 + ((row >> 2) & 3);
        return row * kStride + (col ^ (turn * 8));
    }

    __device__ __forceinline__ explicit Tile(void* p) : base(static_cast<__bf16*>(p)) {}

    template <class E>
    __device__ __forceinline__ void put8(int row, int col, const Eight<E>& x) const {
        __bf16* at = base + place(row, col);
        if constexpr (P == 1 && sizeof(typename E::S) == 2) {
            fx4 v;
            __builtin_memcpy(&v, x.v, 16);
            *reinterpret_cast<fx4*>(at) = v;
        } else {
            const Operand<P> o = operand_from<P, E>(x);
#pragma unroll
            for (int i = 0; i < P; ++i) *reinterpret_cast<bx8*>(at + i * kPlane) = o.p[i];
        }
    }
    // Depths k0 .. k0+31 of row `row` (lane % 16 chooses the row in the caller).
    __device__ __forceinline__ Operand<P> along(int row, int k0, int g) const {
        Operand<P> o;
#pragma unroll
        for (int i = 0; i < P; ++i) o.p[i] = *reinterpret_cast<const bx8*>(base + i * kPlane + place(row, k0 + 8 * g));
        return o;
    }
    // Depths row0 .. row0+31 (tokens) of the features of state tile t, in the order of feature_row().
    __device__ __forceinline__ Operand<P> down_features(int row0, int t, int lane) const {
        const int g = lane >> 4, i = lane & 15;
        Operand<P> o;
#pragma unroll
        for (int n = 0; n < P; ++n) {
            __bf16* at = base + n * kPlane + place(row0 + 4 * g + (i >> 2), feature_row(t, i & 3, 0));
            const sx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4*)at);
            const sx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4*)(at + 16 * kStride));
            o.p[n] = __builtin_shufflevector(__builtin_bit_cast(bx4, a), __builtin_bit_cast(bx4, b), 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return o;
    }
    // Rows row0+4g .. +3 of column col0 + lane % 16: the transposing LDS read, whose 16 lanes of a group
    // fetch four rows of 16 columns and receive a column each.
    __device__ __forceinline__ bx4 column4(int plane, int row0, int col0, int lane) const {
        const int g = lane >> 4, i = lane & 15;
        __bf16* at = base + plane * kPlane + place(row0 + 4 * g + (i >> 2), col0 + (i & 3) * 4);
        const sx4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4*)at);
        return __builtin_bit_cast(bx4, v);
    }
    // Depths row0 .. row0+31 of column col0 + lane % 16.
    __device__ __forceinline__ Operand<P> down(int row0, int col0, int lane) const {
        Operand<P> o;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const bx4 a = column4(i, row0, col0, lane), b = column4(i, row0 + 16, col0, lane);
            o.p[i] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return o;
    }
    // The 16 x 16 tile at (row0, col0) in the accumulator's layout.
    __device__ __forceinline__ fx4 tile(int row0, int col0, int lane) const {
        return summed([&](int i) { return __builtin_bit_cast(uint64_t, column4(i, row0, col0, lane)); });
    }
    // Columns col .. col+3 (col a multiple of 4) of row `row`.
    __device__ __forceinline__ fx4 quad(int row, int col) const {
        return summed([&](int i) { return *reinterpret_cast<const uint64_t*>(base + i * kPlane + place(row, col)); });
    }
    // Four values of which part i is four bfloat16 values in a word.
    template <class F>
    static __device__ __forceinline__ fx4 summed(F word) {
        fx4 x;
#pragma unroll
        for (int i = P - 1; i >= 0; --i) {
            const uint64_t w = word(i);
            const uint32_t a = (uint32_t)w, b = (uint32_t)(w >> 32);
            const fx4 part = {__builtin_bit_cast(float, a << 16), __builtin_bit_cast(float, a & 0xffff0000u),
                              __builtin_bit_cast(float, b << 16), __builtin_bit_cast(float, b & 0xffff0000u)};
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = i == P - 1 ? part[r] : x[r] + part[r];
        }
        return x;
    }
};

template <int W>
struct Tile<0, W> {
    static constexpr int kStride = W + 4;
    static constexpr int kBytes = kBlock * kStride * 4;
    float* base;

    __device__ __forceinline__ explicit Tile(void* p) : base(static_cast<float*>(p)) {}

    template <class E>
    __device__ __forceinline__ void put8(int row, int col, const Eight<E>& x) const {
        fx4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = E::get(x.v[i]);
            b[i] = E::get(x.v[i + 4]);
        }
        float* at = base + row * kStride + col;
        *reinterpret_cast<fx4*>(at) = a;
        *reinterpret_cast<fx4*>(at + 4) = b;
    }
    __device__ __forceinline__ fx4 quad(int row, int col) const { return *reinterpret_cast<const fx4*>(base + row * kStride + col); }
    __device__ __forceinline__ Operand<0> along(int row, int k0, int g) const {
        const float* at = base + row * kStride + k0 + 8 * g;
        Operand<0> o;
        o.t[0] = *reinterpret_cast<const fx4*>(at);
        o.t[1] = *reinterpret_cast<const fx4*>(at + 4);
        return o;
    }
    __device__ __forceinline__ Operand<0> down_features(int row0, int t, int lane) const {
        const float* at = base + (row0 + 4 * (lane >> 4)) * kStride + feature_row(t, (lane >> 2) & 3, lane & 3);
        Operand<0> o;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            o.t[0][r] = at[r * kStride];
            o.t[1][r] = at[(16 + r) * kStride];
        }
        return o;
    }
    __device__ __forceinline__ fx4 tile(int row0, int col0, int lane) const {
        const float* at = base + (row0 + 4 * (lane >> 4)) * kStride + col0 + (lane & 15);
        fx4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = at[r * kStride];
        return x;
    }
    __device__ __forceinline__ Operand<0> down(int row0, int col0, int lane) const {
        Operand<0> o;
        o.t[0] = tile(row0, col0, lane);
        o.t[1] = tile(row0 + 16, col0, lane);
        return o;
    }
};

// Accumulator tiles that the waves of a workgroup hand to each other as operands: N operands of two stacked tiles.
template <int P, int N>
struct Exchange {
    static constexpr int kBytes = (P == 0 ? 2 : P) * N * 64 * 16;
    char* base;

    __device__ __forceinline__ explicit Exchange(char* p) : base(p) {}

    // A lane's four values as they are kept here.
    struct Kept {
        ux2 w[P == 0 ? 2 : P];
    };
    static __device__ __forceinline__ Kept kept(const fx4& x) {
        Kept k;
        if constexpr (P == 0) {
            __builtin_memcpy(k.w, &x, 16);
        } else {
            uint32_t low[P], high[P];
            pair_parts<P>(x[0], x[1], low);
            pair_parts<P>(x[2], x[3], high);
#pragma unroll
            for (int i = 0; i < P; ++i) k.w[i] = ux2{low[i], high[i]};
        }
        return k;
    }
    __device__ __forceinline__ void put(int tile, int lane, const Kept& k) {
        if constexpr (P == 0) {
            fx4 x;
            __builtin_memcpy(&x, k.w, 16);
            *reinterpret_cast<fx4*>(base + (tile * 64 + lane) * 16) = x;
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) *reinterpret_cast<ux2*>(base + ((i * N + (tile >> 1)) * 64 + lane) * 16 + (tile & 1) * 8) = k.w[i];
        }
    }
    __device__ __forceinline__ void put(int tile, int lane, const fx4& x) { put(tile, lane, kept(x)); }
    __device__ __forceinline__ Operand<P> get(int n, int lane) const {
        Operand<P> o;
        if constexpr (P == 0) {
            o.t[0] = *reinterpret_cast<const fx4*>(base + (2 * n * 64 + lane) * 16);
            o.t[1] = *reinterpret_cast<const fx4*>(base + ((2 * n + 1) * 64 + lane) * 16);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) o.p[i] = *reinterpret_cast<const bx8*>(base + ((i * N + n) * 64 + lane) * 16);
        }
        return o;
    }
};

// Row lane % 16 of an exchanged tile, columns 4 (lane / 16) .. + 3: what goes to memory as 16 bytes of a row.  (From
// the accumulator itself a store would be four bytes to a lane: four times the instructions.)
template <int P, int N>
__device__ __forceinline__ fx4 exchanged_row(const Exchange<P, N>& x, int tile, int lane) {
    const int i = lane & 15, c0 = 4 * (lane >> 4);
    fx4 y;
    if constexpr (P == 0) {
        const char* at = x.base + (tile * 64 + (i >> 2) * 16 + c0) * 16 + (i & 3) * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = *reinterpret_cast<const float*>(at + r * 16);
    } else {
#pragma unroll
        for (int n = P - 1; n >= 0; --n) {
            char* at = x.base + ((n * N + (tile >> 1)) * 64 + (i & 3) * 16 + c0 + (i >> 2)) * 16 + (tile & 1) * 8;
            const bx4 part = __builtin_bit_cast(
                bx4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4*)at));
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = n == P - 1 ? (float)part[r] : y[r] + (float)part[r];
        }
    }
    return y;
}

// Workgroup barrier for data in LDS: loads from memory stay in flight across it, which __syncthreads() does not
// promise.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Sum over the 16 lanes that share lane / 16, to all of them: rotations within the row of lanes.
template <int N>
__device__ __forceinline__ float rotated(float x) {
    const int i = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum16(float x) {
    x += rotated<8>(x);
    x += rotated<4>(x);
    x += rotated<2>(x);
    x += rotated<1>(x);
    return x;
}

// NaN or infinite.
__device__ __forceinline__ bool is_odd(float x) { return __builtin_amdgcn_classf(x, 0x207); }

// e^x to 2^-22 of its value: 2^(x log2 e) from the hardware, with the product's rounding error put back.
__device__ __forceinline__ float exp_of(float x) {
    constexpr float kHigh = 1.44269502f, kLow = 1.92596299e-8f;  // log2 e
    x = x < -200.0f ? -200.0f : x;  // (0 from there on, and -inf has no product with a rounding error; NaN stays)
    const float t = x * kHigh;
    const float rest = fmaf(x, kHigh, -t) + x * kLow;
    const float p = __builtin_amdgcn_exp2f(t);
    return fmaf(p, rest * 0.693147182f, p);
}

}  // namespace
}  // namespace ascan

#endif  // ASCAN_DELTA_TILE_H_
