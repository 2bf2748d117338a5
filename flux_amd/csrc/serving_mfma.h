// Register layouts of the 16 x 16 matrix instructions that the serving attention kernels share, by element type.
//
// Scores are S^T = K Q^T: the left operand holds 16 keys (lane % 16), the right one 16 query rows (lane % 16), and a
// dot product may take its terms in any order as long as both operands use the same one; so each lane loads 16
// consecutive bytes of its row and group g = lane / 16 covers dims [step * f + per * g, + per) in fragment f.
// The result leaves lane (n, g) with the scores of keys 4 g .. 4 g + 3 for query row n, which is the right operand of
// O^T = V^T P over those keys.  V^T's left operand needs, in lane (m, g), one dim of the same keys: the lane loads
// consecutive dims of the four rows and each component (or byte permute of 16-bit components) is a block of 16 dims.
#pragma once

#include "flux_common.h"

namespace flux {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int wave_scan_int(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int below = __shfl_up(v, step, kWave);
        if (lane >= step) v += below;
    }
    return v;
}

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
    for (int step = 1; step < 64; step *= 2) v += __shfl_xor(v, step, kWave);
    return v;
}

// How rows are read: element by element, in 16-byte loads, or those where the head fills the padded dims.  Loads are not
// masked (masks put each one in a block of its own, behind a wait for the register's last value): dims behind the head's
// repeat its first ones, which meet zeros of the query (and are cleared themselves where an infinity in them must not
// show, by multiply_keys) or results that are not stored.
enum Rows : int { kNarrow = 0, kWideRows = 1, kFullRows = 2 };

template <class T>
struct Mfma;

template <>
struct Mfma<float> {
    using Fragment = f32x4;
    static constexpr int kKeyStep = 16;
    static constexpr int kPer = 4;
    static constexpr float kWeightShift = 0.0f;
    template <int kDim>
    using ValueChunk = f32x4;
    template <int kDim>
    static constexpr int key_fragments() { return kDim / 16; }
    template <int kDim>
    static constexpr int value_chunks() { return kDim / 64; }

    static __device__ __forceinline__ Fragment load_strided(const float* row, int64_t stride, int d, int dim) {
        Fragment f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = row[(d + j < dim ? d + j : 0) * stride];
        return f;
    }
    static __device__ __forceinline__ Fragment zero_behind(Fragment f, int d, int dim) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = d + j < dim ? f[j] : 0.0f;
        return f;
    }
    template <Rows kRows>
    static __device__ __forceinline__ Fragment load_row(const float* row, int d, int dim) {
        if constexpr (kRows == kNarrow) return load_strided(row, 1, d, dim);
        if constexpr (kRows == kWideRows) d = d < dim ? d : 0;
        return *reinterpret_cast<const f32x4*>(row + d);
    }
    template <int kDim, Rows kRows>
    static __device__ __forceinline__ f32x4 load_value(const float* row, int chunk, int m, int dim) {
        return load_row<kRows>(row, 64 * chunk + 4 * m, dim);
    }
    static __device__ __forceinline__ void multiply_key(const Fragment& key, const Fragment& query, f32x4& score) {
#pragma unroll
        for (int j = 0; j < 4; ++j) score = __builtin_amdgcn_mfma_f32_16x16x4f32(key[j], query[j], score, 0, 0, 0);
    }
    template <int kDim, int kSubs>
    static __device__ __forceinline__ void multiply_value(const f32x4 (&value)[kSubs][4][kDim / 64],
                                                          const float (&p)[kSubs][4], f32x4* out) {
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < kDim / 64; ++c)
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        out[4 * c + b] = __builtin_amdgcn_mfma_f32_16x16x4f32(value[s][i][c][b], p[s][i],
                                                                              out[4 * c + b], 0, 0, 0);
    }
    // Row m = 4 g + r of block i is dim 64 (i / 4) + 4 m + i % 4.
    template <int kDim, class F>
    static __device__ __forceinline__ void each_dim(int g, int dim, F&& f) {
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 64 * (i / 4) + 16 * g + 4 * r + i % 4;
                if (d < dim) f(i, r, d);
            }
    }
};

// What the two 16-bit types share.  The weights are split in two terms of 16 bits, so that their rounding (2^-16 of a weight
// in bfloat16; float16's is below) does not show beside that of the result; the matrix units wait for memory here.
template <class T, class Derived>
struct Mfma16 {
    using Fragment = u32x4;
    static constexpr int kKeyStep = 32;
    static constexpr int kPer = 8;
    template <int kDim>
    static constexpr int words() { return kDim == 64 ? 2 : 4; }  // of a value chunk
    template <int kDim>
    using ValueChunk = u32x4;
    template <int kDim>
    static constexpr int key_fragments() { return kDim / 32; }
    template <int kDim>
    static constexpr int value_chunks() { return kDim == 64 ? 1 : kDim / 128; }

    static __device__ __forceinline__ uint32_t bits(T v) { return __builtin_bit_cast(uint16_t, v); }

    static __device__ __forceinline__ Fragment load_strided(const T* row, int64_t stride, int d, int dim) {
        Fragment f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t low = bits(row[(d + 2 * j < dim ? d + 2 * j : 0) * stride]);
            const uint32_t high = bits(row[(d + 2 * j + 1 < dim ? d + 2 * j + 1 : 0) * stride]);
            f[j] = low | high << 16;
        }
        return f;
    }
    static __device__ __forceinline__ Fragment zero_behind(Fragment f, int d, int dim) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] &= (d + 2 * j < dim ? 0xffffu : 0u) | (d + 2 * j + 1 < dim ? 0xffff0000u : 0u);
        return f;
    }
    template <Rows kRows>
    static __device__ __forceinline__ Fragment load_row(const T* row, int d, int dim) {
        if constexpr (kRows == kNarrow) return load_strided(row, 1, d, dim);
        if constexpr (kRows == kWideRows) d = d < dim ? d : 0;
        return *reinterpret_cast<const u32x4*>(row + d);
    }
    template <int kDim, Rows kRows>
    static __device__ __forceinline__ u32x4 load_value(const T* row, int chunk, int m, int dim) {
        if constexpr (kDim == 64) {
            int d = 4 * m;
            if constexpr (kRows == kNarrow) return load_strided(row, 1, d, dim);
            if constexpr (kRows == kWideRows) d = d < dim ? d : 0;
            const u32x2 half = *reinterpret_cast<const u32x2*>(row + d);
            return u32x4{half[0], half[1], 0, 0};
        } else {
            return load_row<kRows>(row, 128 * chunk + 8 * m, dim);
        }
    }
    static __device__ __forceinline__ void multiply_key(const Fragment& key, const Fragment& query, f32x4& score) {
        score = Derived::multiply32(key, query, score);
    }
    // The 16-bit components `odd` of two dwords, side by side.
    static __device__ __forceinline__ uint32_t pair(uint32_t first, uint32_t second, bool odd) {
        return __builtin_amdgcn_perm(second, first, odd ? 0x07060302u : 0x05040100u);
    }
    template <int kDim, int kSubs>
    static __device__ __forceinline__ void multiply_value(const u32x4 (&value)[kSubs][4][value_chunks<kDim>()],
                                                          const float (&p)[kSubs][4], f32x4* out) {
        u32x4 high = {0, 0, 0, 0}, low = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const T h0 = static_cast<T>(p[s][2 * j]), h1 = static_cast<T>(p[s][2 * j + 1]);
                high[2 * s + j] = bits(h0) | bits(h1) << 16;
                const T l0 = static_cast<T>(p[s][2 * j] - static_cast<float>(h0));
                const T l1 = static_cast<T>(p[s][2 * j + 1] - static_cast<float>(h1));
                low[2 * s + j] = bits(l0) | bits(l1) << 16;
            }
#pragma unroll
        for (int c = 0; c < value_chunks<kDim>(); ++c)
#pragma unroll
            for (int b = 0; b < 2 * words<kDim>(); ++b) {
                u32x4 left = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < kSubs; ++s) {
                    left[2 * s] = pair(value[s][0][c][b / 2], value[s][1][c][b / 2], b & 1);
                    left[2 * s + 1] = pair(value[s][2][c][b / 2], value[s][3][c][b / 2], b & 1);
                }
                f32x4& o = out[2 * words<kDim>() * c + b];
                if constexpr (kSubs == 2) {
                    o = Derived::multiply32(left, high, o);
                    o = Derived::multiply32(left, low, o);
                } else {
                    o = Derived::multiply16(left, high, o);
                    o = Derived::multiply16(left, low, o);
                }
            }
    }
    // Row m = 4 g + r of block i: dim 4 m + i for heads up to 64, else 128 (i / 8) + 8 m + i % 8.
    template <int kDim, class F>
    static __device__ __forceinline__ void each_dim(int g, int dim, F&& f) {
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = kDim == 64 ? 16 * g + 4 * r + i : 128 * (i / 8) + 8 * (4 * g + r) + i % 8;
                if (d < dim) f(i, r, d);
            }
    }
};

template <>
struct Mfma<__bf16> : Mfma16<__bf16, Mfma<__bf16>> {
    static constexpr float kWeightShift = 0.0f;
    static __device__ __forceinline__ f32x4 multiply32(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 multiply16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, u32x2{a[0], a[1]}),
                                                         __builtin_bit_cast(s16x4, u32x2{b[0], b[1]}), c, 0, 0, 0);
    }
};

// float16's smallest step is 2^-24: weights are held 2^12 times as large (at most 4096), sums of weights with them.  Each term
// is off by at most 2^-11 of itself, so that a split weight loses 2^-22 of itself where its lower term is a normal number, and
// else half a smallest step, 2^-25 of 4096: 2^-37 of the largest weight.
template <>
struct Mfma<_Float16> : Mfma16<_Float16, Mfma<_Float16>> {
    static constexpr float kWeightShift = 12.0f;
    static __device__ __forceinline__ f32x4 multiply32(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x4 multiply16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, u32x2{a[0], a[1]}),
                                                     __builtin_bit_cast(f16x4, u32x2{b[0], b[1]}), c, 0, 0, 0);
    }
};

// The scores of 16 keys, whose rows were loaded by load_row; kClear clears the dims behind the head's.
template <class M, bool kClear, int kFragments>
__device__ __forceinline__ f32x4 multiply_keys(const typename M::Fragment (&key)[kFragments],
                                               const typename M::Fragment (&query)[kFragments], int group, int dim) {
    f32x4 score = {0, 0, 0, 0};
#pragma unroll
    for (int f = 0; f < kFragments; ++f)
        M::multiply_key(kClear ? M::zero_behind(key[f], M::kKeyStep * f + M::kPer * group, dim) : key[f], query[f], score);
    return score;
}

// The fragments of one query row, zero behind its dims, all zero unless `real` (the row's memory is valid either way:
// products with zeros draw less power).
template <class T, int kFragments, int kStep>
__device__ __forceinline__ void load_query(typename Mfma<T>::Fragment (&query)[kFragments], const T* row, int64_t stride,
                                           bool wide, int first, int dim, bool real) {
    using M = Mfma<T>;
    if (wide) {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) query[f] = M::template load_row<kWideRows>(row, kStep * f + first, dim);
    } else {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) query[f] = M::load_strided(row, stride, kStep * f + first, dim);
    }
    if (dim < kFragments * kStep || !__all(real)) {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) query[f] = M::zero_behind(query[f], kStep * f + first, real ? dim : 0);
    }
}

// ---- 32 x 32 tiles of the 16-bit kernels that stage keys and values ----

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The weights' place in the type (kShift: powers of two that they are held larger by) and how far a tile's largest score may
// exceed the running maximum's before the sums are rescaled (kLazy).
template <class T>
struct Wide;
template <>
struct Wide<__bf16> {
    static constexpr float kShift = 0.0f, kLazy = 8.0f;
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t round(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), Pair));
    }
    static __device__ __forceinline__ f32x16 multiply(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};
template <>
struct Wide<_Float16> {
    // Weights are held 2^11 times as large, at most 2^15 with kLazy.  Those from 2^-25 of the reference on are normal numbers;
    // smaller ones are off by at most half of float16's smallest step, 2^-36 of the reference, and the 2^24 keys that a
    // sequence can have together by 2^-12 of the largest value.
    static constexpr float kShift = 11.0f, kLazy = 4.0f;
    typedef _Float16 Pair __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t round(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), Pair));
    }
    static __device__ __forceinline__ f32x16 multiply(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
};

__device__ __forceinline__ float half_max(float v) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return fmaxf(__int_as_float(both[0]), __int_as_float(both[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(both[0]) + __int_as_float(both[1]);
}

}  // namespace flux
