// Causal attention with a sliding window and sink tokens over contiguous keys and values: prompts, chunks of prompts,
// and single tokens (which take the split kernel of paged_attention.hip).
//
// The query at position p of a sequence of n keys sees j <= p, j < n, with j > p - window or j < sinks (window 0: all);
// a row that sees nothing, nothing whose score is above -inf, or whose position is no key's, gives zeros.
//
// A workgroup takes kRows rows of one KV head, a row being a query position and one of the head's query heads, so that a
// group of heads shares each key and value row.  Its four waves split the keys, hold the running maximum and sum per
// row, and join at the end in registers.  Keys outside every row's range are never read.
#include "serving.h"
#include "serving_mfma.h"

namespace flux {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

struct RowRange {
    int position;  // -1: sees nothing
    int low;       // first key of the window
};

// A row whose result is not finite, computed again over the keys it sees alone: a matrix instruction multiplies a
// masked key's zero weight with its value too, and a NaN or infinity there must not reach the row.  One wave; `out`
// gets dim values.
template <class T>
__device__ void exact_row(const AttentionArgs& a, const T* query, const T* keys, const T* values, const RowRange& r,
                          T* out) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY, weight = 0.0f, sum[kServingMaxDim / kWave];
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c) sum[c] = 0.0f;
    const int sinks = a.sinks < r.low ? a.sinks : r.low;
    const int count = sinks + r.position + 1 - r.low;
    for (int base = 0; base < count; base += kWave) {
        const int index = base + lane;
        const int key = index < sinks ? index : r.low + index - sinks;
        float score = -INFINITY;
        if (index < count) {
            score = 0.0f;
            for (int d = 0; d < a.dim; ++d)
                score = fmaf(static_cast<float>(query[d * a.query_strides[3]]),
                             static_cast<float>(keys[key * a.key_strides[2] + d]), score);
            score *= a.scale;
        }
        const float now = fmaxf(top, wave_max(score));
        const float reference = now == -INFINITY ? 0.0f : now;
        const float shrink = top == -INFINITY ? 0.0f : fast_exp2((top - reference) * kLog2e);
        top = now;
        const float p = index < count ? fast_exp2((score - reference) * kLog2e) : 0.0f;
        weight = weight * shrink + wave_sum(p);
#pragma unroll
        for (int c = 0; c < kServingMaxDim / kWave; ++c) sum[c] *= shrink;
        const int here = count - base < kWave ? count - base : kWave;
        for (int j = 0; j < here; ++j) {
            const float pj = __shfl(p, j, kWave);
            const int of = base + j;
            const T* value = values + (of < sinks ? of : r.low + of - sinks) * a.value_strides[2];
#pragma unroll
            for (int c = 0; c < kServingMaxDim / kWave; ++c)
                if (kWave * c + lane < a.dim) sum[c] = fmaf(pj, static_cast<float>(value[kWave * c + lane]), sum[c]);
        }
        // What is NaN stays NaN: a row whose sums all are is done.
        bool lost = true;
#pragma unroll
        for (int c = 0; c < kServingMaxDim / kWave; ++c) lost = lost && (kWave * c + lane >= a.dim || sum[c] != sum[c]);
        if (__all(weight != weight || lost)) break;
    }
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c)
        if (kWave * c + lane < a.dim) out[kWave * c + lane] = static_cast<T>(weight == 0.0f ? 0.0f : sum[c] / weight);
}

// Blocks that an XCD (block index modulo 8) takes one after the other: consecutive tiles share most of their keys.  The
// runs are short and the XCDs change places with every eight of them, because a padded batch's sequences differ in length.
constexpr int kTileRun = 16;
__device__ __forceinline__ int tile_of_block() {
    const int eight = blockIdx.x / (8 * kTileRun);
    return (8 * eight + (blockIdx.x + eight) % 8) * kTileRun + blockIdx.x / 8 % kTileRun;
}
int64_t blocks_of_tiles(int64_t tiles) { return (tiles + 8 * kTileRun - 1) / (8 * kTileRun) * (8 * kTileRun); }

// One tile's place and the rows' common quantities.
struct TileRows {
    int row0, all_rows, kv_head;
    int64_t b, n, start;

    __device__ __forceinline__ TileRows(const AttentionArgs& a, int tile, int row_tiles, int rows) {
        row0 = tile % row_tiles * rows;
        kv_head = tile / row_tiles % a.kv_heads;
        b = tile / row_tiles / a.kv_heads;
        all_rows = a.queries * a.group;
        n = a.lengths ? a.lengths[b] : a.keys;
        n = n < 0 ? 0 : (n > a.keys ? a.keys : n);
        start = a.starts ? a.starts[b] : n - a.queries;
        start = start < -a.queries ? -a.queries : (start > a.keys ? a.keys : start);  // no row beyond these sees a key
    }
    // Query index and head of a row.
    __device__ __forceinline__ void place(const AttentionArgs& a, int r, int64_t& i, int64_t& head) const {
        i = divide(r, a.group_of);
        head = kv_head * a.group + r - i * a.group;
    }
    __device__ __forceinline__ RowRange range(const AttentionArgs& a, int r, int64_t i) const {
        const int64_t position = start + i;
        RowRange range;
        range.position = r < all_rows && position >= 0 && position < n ? static_cast<int>(position) : -1;
        range.low = a.window > 0 && range.position >= a.window ? range.position - a.window + 1 : 0;
        return range;
    }
    // Positions of the rows [from, from + count), cut to those that are a key's; first > last when there is none.
    __device__ __forceinline__ void positions(const AttentionArgs& a, int from, int count, int& first, int& last) const {
        const int to = from + count < all_rows ? from + count - 1 : all_rows - 1;
        const int64_t p = start + divide(from, a.group_of), q = start + divide(to, a.group_of);
        first = static_cast<int>(p < 0 ? 0 : p);
        last = static_cast<int>(q >= n ? n - 1 : q);
        if (from > to) last = first - 1;
    }
    // The row again over the keys it sees alone.
    template <class T>
    __device__ __forceinline__ void again(const AttentionArgs& a, int r, const T* keys, const T* values) const {
        int64_t i, head;
        place(a, r, i, head);
        exact_row<T>(a, static_cast<const T*>(a.query) + b * a.query_strides[0] + head * a.query_strides[1] + i * a.query_strides[2],
                     keys, values, range(a, r, i), static_cast<T*>(a.out) + ((b * a.query_heads + head) * a.queries + i) * a.dim);
    }
};

// The keys that any of a tile's rows sees, as tiles of kTile: the sinks', then the window's.
template <int kTile>
struct KeyTiles {
    int seen, sink_tiles, first_tile, count;
    __device__ __forceinline__ KeyTiles(const AttentionArgs& a, int first, int last) {
        const int low = a.window > 0 && first >= a.window ? first - a.window + 1 : 0;
        const int sinks = a.sinks < low ? a.sinks : low;
        const int of_sinks = (sinks + kTile - 1) / kTile;
        seen = last + 1;
        first_tile = low / kTile;
        sink_tiles = of_sinks < first_tile ? of_sinks : first_tile;
        count = first > last ? 0 : sink_tiles + (seen + kTile - 1) / kTile - first_tile;
    }
    __device__ __forceinline__ int base(int t) const { return (t < sink_tiles ? t : first_tile + t - sink_tiles) * kTile; }
};

template <int kDim, Rows kRowsRead>
__global__ void __launch_bounds__(kThreads, kDim <= 64 ? 4 : (kDim <= 128 ? 2 : 1)) window_attention_kernel(AttentionArgs a, int row_tiles, int tiles_total) {
    using M = Mfma<float>;
    constexpr int kCols = kDim == 256 ? 1 : 2;  // tiles of 16 rows
    constexpr int kRows = 16 * kCols;
    constexpr int kTile = 16;
    constexpr int kSubs = kTile / 16;
    constexpr int kFragments = M::template key_fragments<kDim>();
    constexpr int kChunks = M::template value_chunks<kDim>();
    constexpr int kBlocks = kDim / 16;
    constexpr int kWords = kBlocks * 4 + 2;
    __shared__ float merge[2][kCols * kWords][kWave];

    const int tile = tile_of_block();
    if (tile >= tiles_total) return;
    const TileRows rows(a, tile, row_tiles, kRows);
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int n16 = lane & 15;
    const int g = lane >> 4;
    const float* keys = static_cast<const float*>(a.key) + rows.b * a.key_strides[0] + rows.kv_head * a.key_strides[1];
    const float* values = static_cast<const float*>(a.value) + rows.b * a.value_strides[0] + rows.kv_head * a.value_strides[1];

    int first_p, last_p;
    rows.positions(a, rows.row0, kRows, first_p, last_p);
    const KeyTiles<kTile> tiles(a, first_p, last_p);
    RowRange mine[kCols];
    int sink_end[kCols];
    f32x4 query[kCols][kFragments];
    f32x4 out[kCols][kBlocks];
    float top[kCols], weight[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        const int r = rows.row0 + 16 * c + n16;
        const bool real = r < rows.all_rows;
        int64_t i, head;
        rows.place(a, real ? r : rows.row0, i, head);
        mine[c] = rows.range(a, r, i);
        sink_end[c] = a.sinks < mine[c].low ? a.sinks : mine[c].low;
        const float* q = static_cast<const float*>(a.query) + rows.b * a.query_strides[0] + head * a.query_strides[1] + i * a.query_strides[2];
        if (tiles.count > 0)  // a padded batch has many tiles of rows that are no key's
            load_query<float, kFragments, M::kKeyStep>(query[c], q, a.query_strides[3], a.query_wide, M::kPer * g, a.dim, real);
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) out[c][k] = f32x4{0, 0, 0, 0};
        top[c] = -INFINITY;
        weight[c] = 0.0f;
    }
    const int low_of_last = a.window > 0 && last_p >= a.window ? last_p - a.window + 1 : 0;

    struct Tile {
        f32x4 key[kSubs][kFragments];
        f32x4 value[kSubs][4][kChunks];
    };
    // Rows behind the last key repeat it: their weights are zero.
    auto load = [&](int t, Tile& into) {
        const int base = tiles.base(t), end = tiles.seen - 1;
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
            const int position = base + 16 * s + n16;
            const float* k = keys + (position < end ? position : end) * a.key_strides[2];
#pragma unroll
            for (int f = 0; f < kFragments; ++f)
                into.key[s][f] = M::template load_row<kRowsRead>(k, M::kKeyStep * f + M::kPer * g, a.dim);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int value_position = base + 16 * s + 4 * g + i;
                const float* v = values + (value_position < end ? value_position : end) * a.value_strides[2];
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
                    into.value[s][i][c] = M::template load_value<kDim, kRowsRead>(v, c, n16, a.dim);
            }
        }
    };
    auto work = [&](int t, const Tile& of) {
        const int base = tiles.base(t);
        // Every key of the tile is seen by every row that sees any (the others are zeroed at the end).
        const bool inside = base >= low_of_last && base + kTile - 1 <= first_p;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            f32x4 score[kSubs];
            float highest = -INFINITY;
#pragma unroll
            for (int s = 0; s < kSubs; ++s) {
                score[s] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int f = 0; f < kFragments; ++f) M::multiply_key(of.key[s][f], query[c][f], score[s]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = base + 16 * s + 4 * g + i;
                    // Without branches: low <= key <= position as one unsigned comparison, or a sink.
                    const bool visible = inside | (static_cast<uint32_t>(j - mine[c].low) <=
                                                   static_cast<uint32_t>(mine[c].position - mine[c].low)) | (j < sink_end[c]);
                    score[s][i] = visible ? score[s][i] * a.scale : -INFINITY;
                    highest = fmaxf(highest, score[s][i]);
                }
            }
            highest = fmaxf(highest, __shfl_xor(highest, 16, kWave));
            highest = fmaxf(highest, __shfl_xor(highest, 32, kWave));
            if (__any(highest > top[c])) {
                const float now = fmaxf(top[c], highest);
                const float shrink = top[c] == -INFINITY ? 0.0f : fast_exp2((top[c] - now) * kLog2e);
                top[c] = now;
                weight[c] *= shrink;
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) out[c][i] *= shrink;
            }
            const float reference = top[c] == -INFINITY ? 0.0f : top[c];
            float p[kSubs][4];
#pragma unroll
            for (int s = 0; s < kSubs; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[s][i] = fast_exp2((score[s][i] - reference) * kLog2e);
                    weight[c] += p[s][i];
                }
            M::template multiply_value<kDim, kSubs>(of.value, p, out[c]);
        }
    };

    // Many waves with one small tile each do better than few with two larger ones in flight (4096 tokens, 9 / 3 heads of 64,
    // window 1024: 16 keys and four waves per SIMD 110 us, three 115; 32 keys, one more in flight, two waves 132).  A wave's
    // tile numbers are the same in all its lanes.
    Tile held;
    for (int t = __builtin_amdgcn_readfirstlane(wave); t < tiles.count; t += kWaves) {
        load(t, held);
        work(t, held);
    }

#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        weight[c] += __shfl_xor(weight[c], 16, kWave);
        weight[c] += __shfl_xor(weight[c], 32, kWave);
    }
    // Join the four waves: 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
    for (int half = kWaves / 2; half >= 1; half /= 2) {
        if (half == 1) __syncthreads();
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                float(*to)[kWave] = merge[wave - half] + c * kWords;
#pragma unroll
                for (int i = 0; i < kBlocks * 4; ++i) to[i][lane] = out[c][i / 4][i % 4];
                to[kBlocks * 4][lane] = top[c];
                to[kBlocks * 4 + 1][lane] = weight[c];
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                const float(*other)[kWave] = merge[wave] + c * kWords;
                const float other_top = other[kBlocks * 4][lane];
                const float now = fmaxf(top[c], other_top);
                const float mine_scale = top[c] == -INFINITY ? 0.0f : fast_exp2((top[c] - now) * kLog2e);
                const float other_scale = other_top == -INFINITY ? 0.0f : fast_exp2((other_top - now) * kLog2e);
                top[c] = now;
                weight[c] = weight[c] * mine_scale + other[kBlocks * 4 + 1][lane] * other_scale;
#pragma unroll
                for (int i = 0; i < kBlocks * 4; ++i)
                    out[c][i / 4][i % 4] = out[c][i / 4][i % 4] * mine_scale + other[i][lane] * other_scale;
            }
        }
    }
    if (wave != 0) return;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        float worst = fabsf(weight[c]);
        M::template each_dim<kDim>(g, a.dim, [&](int i, int r, int) { worst += fabsf(out[c][i][r]); });  // keeps NaN, infinity
        const uint64_t odd = __ballot(mine[c].position >= 0 && !(worst < INFINITY));
        uint32_t again = static_cast<uint32_t>((odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xffff);
        const int r = rows.row0 + 16 * c + n16;
        if (r < rows.all_rows && !(again >> n16 & 1)) {
            int64_t i, head;
            rows.place(a, r, i, head);
            float* o = static_cast<float*>(a.out) + ((rows.b * a.query_heads + head) * a.queries + i) * a.dim;
            M::template each_dim<kDim>(g, a.dim, [&](int k, int j, int d) {
                o[d] = mine[c].position < 0 || weight[c] == 0.0f ? 0.0f : out[c][k][j] / weight[c];
            });
        }
        while (again) {
            const int which = __ffs(again) - 1;
            again &= again - 1;
            rows.template again<float>(a, rows.row0 + 16 * c + which, keys, values);
        }
    }
}

// ---------------------------------------------------------------------------
// 16-bit prompts.  Here matrix instructions, exponentials and LDS reads cost about the same, so that keys and values are
// staged once for the workgroup's four waves, 32 rows each.  4 x 4096 tokens (padded), 32 / 8 heads of 128, window 1024 in
// bfloat16: 239 to 250 us, 670 to 700 TFLOP/s.  A 32 x 32 tile costs a SIMD 512 cycles of matrix instructions and as many of vector
// instructions (half of them exponentials), and the two waves of a SIMD overlap them in part: 64 rows a wave (one wave
// per SIMD) took 640 us, a workgroup of eight waves 236, two tiles per maximum 244.
//
// A stage holds kKeys keys: K rows as they are, V transposed (the staging thread permutes the 16-bit halves of four
// keys), its keys in the order in which a lane's scores lie.  S^T = K Q^T on 32 x 32 tiles leaves lane (n, h) with the
// keys 8 (r / 4) + 4 h + r % 4 of row n, which rounded in pairs are the right operand of O^T = V^T P.  Rows are padded by
// 16 bytes so that eight lanes' 16-byte reads fall on different banks.
// The running maximum moves only when a tile exceeds it by 2^kLazy: a rescaling of the sums costs as much as the
// exponentials, and weights up to 2^kLazy are as exact.  Weights are rounded once to the values' type for the product: by
// at most half a step of that type relative to themselves, which moves a weighted mean of the values by at most half a step
// of the largest of them, as the result's own rounding does.  They are summed unrounded in float32.  (Two terms a weight, as
// in paged_attention.hip, would double the matrix instructions of the product, here where they bound the kernel.)
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
constexpr int64_t kStagedStride = 1 << 22;

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

// Rows of one stage.  With kWide 16 bytes at a byte offset through a buffer that ends with the last row (kStagedStride
// keeps offsets in 31 bits); else eight elements, of the last row where there is none.
template <class T, bool kWide>
struct StagedRows {
    const T* base;
    __amdgpu_buffer_rsrc_t buffer;
    __device__ __forceinline__ StagedRows(const T* from, int64_t bytes) : base(from) {
        if constexpr (kWide)
            buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(from), 0, static_cast<int>(bytes), 0x00020000);
    }
    __device__ __forceinline__ u32x4 load(int at, int row, int d, int rows, int64_t stride, int dim) const {
        if constexpr (kWide) return __builtin_amdgcn_raw_buffer_load_b128(buffer, at, 0, 0);
        return Mfma<T>::load_strided(base + (row < rows ? row : rows - 1) * stride, 1, d, dim);
    }
};

template <class T, int kDim, bool kWide>
__global__ void __launch_bounds__(kThreads, kDim <= 128 ? 2 : 1)
window_tile_kernel(AttentionArgs a, int row_tiles, int tiles_total) {
    using W = Wide<T>;
    constexpr int kKeys = kDim == 64 ? 128 : (kDim == 128 ? 64 : 32);
    constexpr int kSubs = kKeys / 32;
    constexpr int kSteps = kDim / 16;             // of a score
    constexpr int kBlocks = kDim / 32;            // of the result
    constexpr int kRows = kWaves * 32;
    constexpr int kKeyRow = kDim * 2 + 16;        // bytes
    constexpr int kValueRow = kKeys * 2 + 16;
    constexpr int kStage = kKeys * kKeyRow + kDim * kValueRow;
    constexpr int kKeyLoads = kKeys * kDim / 8 / kThreads;        // 16 bytes per thread
    static_assert(kKeys / 4 * (kDim / 8) == kThreads, "every thread stages four keys by eight dims of the values");
    extern __shared__ char stages[];

    const int tile = tile_of_block();
    if (tile >= tiles_total) return;
    const TileRows rows(a, tile, row_tiles, kRows);
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int n32 = lane & 31;
    const int half = lane >> 5;
    int block_first, block_last, wave_first, wave_last;
    rows.positions(a, rows.row0, kRows, block_first, block_last);
    const int wave_row = rows.row0 + wave * 32;
    rows.positions(a, wave_row, 32, wave_first, wave_last);
    wave_first = __builtin_amdgcn_readfirstlane(wave_first);
    wave_last = __builtin_amdgcn_readfirstlane(wave_last);

    const T* keys = static_cast<const T*>(a.key) + rows.b * a.key_strides[0] + rows.kv_head * a.key_strides[1];
    const T* values = static_cast<const T*>(a.value) + rows.b * a.value_strides[0] + rows.kv_head * a.value_strides[1];

    const int r = wave_row + n32;  // this lane's row
    const bool real = r < rows.all_rows;
    int64_t query_index, head;
    rows.place(a, real ? r : rows.row0, query_index, head);
    const RowRange mine = rows.range(a, r, query_index);
    const int sink_end = a.sinks < mine.low ? a.sinks : mine.low;
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // the scale's sign goes to the query
    // Its size goes into the exponent's argument, unless it is 0 (which makes a masked score's -inf NaN, and has to make an
    // infinite score NaN) or next to what float32 holds: then it multiplies the scores before they are masked.
    const float size = fabsf(a.scale);
    const bool ordinary = size >= 1e-30f && size <= 1e30f;
    const float factor = ordinary ? size * kLog2e : kLog2e;
    f32x16 out[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) out[i][j] = 0.0f;
    float top = -INFINITY, weight = 0.0f;

    if (block_first <= block_last) {  // a padded batch has many tiles of rows that are no key's
        u32x4 query[kSteps];
        load_query<T, kSteps, 16>(query, static_cast<const T*>(a.query) + rows.b * a.query_strides[0] + head * a.query_strides[1] +
                                             query_index * a.query_strides[2],
                                  a.query_strides[3], a.query_wide, 8 * half, a.dim, real);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) query[s] ^= sign;
        const KeyTiles<kKeys> tiles(a, block_first, block_last);
        const int seen = tiles.seen, count = tiles.count;
        auto low_of = [&](int p) { return a.window > 0 && p >= a.window ? p - a.window + 1 : 0; };

        // Rows behind the last key are zeros (a buffer's range check) or repeat it, and weigh nothing; dims behind the head's
        // repeat its first ones, which meet a zero in the query or are not stored.
        u32x4 held_key[kKeyLoads];
        u32x4 held_value[4];
        const int key_row = threadIdx.x / (kDim / 8), key_d = threadIdx.x % (kDim / 8) * 8;
        const int value_row = threadIdx.x % (kKeys / 4) * 4, value_d = threadIdx.x / (kKeys / 4) * 8;
        constexpr int kKeyRows = kThreads / (kDim / 8);  // rows that one load of all threads covers
        const int key_stride = static_cast<int>(a.key_strides[2]), value_stride = static_cast<int>(a.value_strides[2]);
        const int key_at = (key_row * key_stride + (key_d < a.dim ? key_d : 0)) * 2;
        const int value_at = (value_row * value_stride + (value_d < a.dim ? value_d : 0)) * 2;
        auto fetch_keys = [&](int t) {
            const int base = tiles.base(t), rows = seen - base < kKeys ? seen - base : kKeys;
            const T* from = keys + base * a.key_strides[2];
            const StagedRows<T, kWide> staged(from, ((rows - 1) * a.key_strides[2] + a.dim) * 2);
#pragma unroll
            for (int i = 0; i < kKeyLoads; ++i)
                held_key[i] = staged.load(key_at + kKeyRows * i * key_stride * 2, key_row + kKeyRows * i, key_d, rows, a.key_strides[2], a.dim);
        };
        auto fetch_values = [&](int t) {
            const int base = tiles.base(t), rows = seen - base < kKeys ? seen - base : kKeys;
            const T* from = values + base * a.value_strides[2];
            const StagedRows<T, kWide> staged(from, ((rows - 1) * a.value_strides[2] + a.dim) * 2);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                held_value[j] = staged.load(value_at + j * value_stride * 2, value_row + j, value_d, rows, a.value_strides[2], a.dim);
        };
        auto put_keys = [&](char* stage) {
#pragma unroll
            for (int i = 0; i < kKeyLoads; ++i) {
                const int unit = threadIdx.x + kThreads * i;
                *reinterpret_cast<u32x4*>(stage + unit / (kDim / 8) * kKeyRow + unit % (kDim / 8) * 16) = held_key[i];
            }
        };
        auto put_values = [&](char* stage) {
            char* turned = stage + kKeys * kKeyRow;
            // Quads 0, 1, 2, 3 of 16 keys lie as 0, 2, 1, 3: a lane's eight keys side by side.
            const int quad = value_row / 4, at = (quad & ~3) | (quad & 1) << 1 | (quad >> 1 & 1);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<u32x2*>(turned + (value_d + j) * kValueRow + at * 8) =
                    u32x2{Mfma<T>::pair(held_value[0][j / 2], held_value[1][j / 2], j & 1),
                          Mfma<T>::pair(held_value[2][j / 2], held_value[3][j / 2], j & 1)};
        };

        const int wave_low = low_of(wave_first), low_of_last = low_of(wave_last);
        fetch_keys(0);
        fetch_values(0);
        put_keys(stages);
        put_values(stages);
        for (int t = 0; t < count; ++t) {
            __syncthreads();
            const char* stage = stages + (t & 1) * kStage;
            const char* turned = stage + kKeys * kKeyRow;
            const int base = tiles.base(t);
            char* next = stages + ((t + 1) & 1) * kStage;
            if (t + 1 < count) fetch_keys(t + 1);
#pragma unroll
            for (int s = 0; s < kSubs; ++s) {
                if (s == kSubs / 2 && t + 1 < count) {  // K and V take the same registers on their way
                    put_keys(next);
                    fetch_values(t + 1);
                }
                const int first = base + 32 * s, last = first + 31;
                // Nothing of this wave's rows sees these keys.
                if (first > wave_last || (last < wave_low && first >= a.sinks)) continue;
                u32x4 key[kSteps];
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
                    key[k] = *reinterpret_cast<const u32x4*>(stage + (32 * s + n32) * kKeyRow + 32 * k + 16 * half);
                __builtin_amdgcn_sched_barrier(0);  // all reads first: one wait
                f32x16 score;
#pragma unroll
                for (int j = 0; j < 16; ++j) score[j] = 0.0f;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) score = W::multiply(key[k], query[k], score);
                if (!ordinary) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) score[j] *= size;
                }
                if (first < low_of_last || last > wave_first) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        // Without branches: low <= key <= position as one unsigned comparison, or a sink.
                        const int of = first + 8 * (j / 4) + 4 * half + j % 4;
                        const bool visible = (static_cast<uint32_t>(of - mine.low) <= static_cast<uint32_t>(mine.position - mine.low)) |
                                             (of < sink_end);
                        score[j] = visible ? score[j] : -INFINITY;
                    }
                }
                float highest = score[0];
#pragma unroll
                for (int j = 1; j < 16; ++j) highest = fmaxf(highest, score[j]);
                highest = half_max(highest) * factor;
                if (__any(highest > top + W::kLazy)) {
                    const float now = fmaxf(top, highest);
                    const float shrink = top == -INFINITY ? 0.0f : fast_exp2(top - now);
                    top = now;
                    weight *= shrink;
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) out[i][j] *= shrink;
                }
                u32x4 value[kBlocks][2];
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        value[i][k] = *reinterpret_cast<const u32x4*>(turned + (32 * i + n32) * kValueRow + (32 * s + 16 * k) * 2 + 16 * half);
                __builtin_amdgcn_sched_barrier(0);
                const float reference = W::kShift - (top == -INFINITY ? 0.0f : top);
                u32x4 p[2];
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float p0 = fast_exp2(fmaf(score[j], factor, reference));
                    const float p1 = fast_exp2(fmaf(score[j + 1], factor, reference));
                    weight += p0 + p1;
                    p[j / 8][j % 8 / 2] = W::round(p0, p1);
                }
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) out[i] = W::multiply(value[i][k], p[k], out[i]);
            }
            if (t + 1 < count) put_values(next);
        }
    }

    weight = half_sum(weight);
    float worst = fabsf(weight);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) worst += fabsf(out[i][j]);  // keeps NaN, infinity
    const uint64_t odd = __ballot(mine.position >= 0 && !(worst < INFINITY));
    uint32_t again = static_cast<uint32_t>(odd | odd >> 32);
    if (real && !(again >> n32 & 1)) {
        T* o = static_cast<T*>(a.out) + ((rows.b * a.query_heads + head) * a.queries + query_index) * a.dim;
        const float inverse = weight == 0.0f ? 0.0f : 1.0f / weight;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const int d = 32 * i + 2 * j + 4 * half;  // four dims side by side
                float four[4];
#pragma unroll
                for (int l = 0; l < 4; ++l) four[l] = mine.position < 0 ? 0.0f : out[i][j + l] * inverse;
                const u32x2 rounded = {W::round(four[0], four[1]), W::round(four[2], four[3])};
                if constexpr (kWide) {
                    if (d < a.dim) *reinterpret_cast<u32x2*>(o + d) = rounded;
                } else {
#pragma unroll
                    for (int l = 0; l < 4; ++l)
                        if (d + l < a.dim) o[d + l] = __builtin_bit_cast(T, static_cast<uint16_t>(rounded[l / 2] >> 16 * (l % 2)));
                }
            }
    }
    while (again) {
        const int which = __ffs(again) - 1;
        again &= again - 1;
        rows.template again<T>(a, wave_row + which, keys, values);
    }
}

template <class T, int kDim, bool kWide>
hipError_t launch_window_tiles(const AttentionArgs& a, hipStream_t stream) {
    constexpr int kKeys = kDim == 64 ? 128 : (kDim == 128 ? 64 : 32);
    constexpr int kRows = kWaves * 32;
    constexpr size_t kLds = 2 * (kKeys * (kDim * 2 + 16) + kDim * (kKeys * 2 + 16));
    const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
    const int row_tiles = static_cast<int>((rows + kRows - 1) / kRows);
    const int64_t tiles = static_cast<int64_t>(row_tiles) * a.kv_heads * a.batch;
    if (tiles >= (int64_t{1} << 24) - 256) return hipErrorInvalidValue;  // a grid has below 2^32 threads
    const hipError_t room = hipFuncSetAttribute(
        reinterpret_cast<const void*>(window_tile_kernel<T, kDim, kWide>),
        hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLds));
    if (room != hipSuccess) return room;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(window_tile_kernel<T, kDim, kWide>),
                       dim3(static_cast<uint32_t>(blocks_of_tiles(tiles))), dim3(kThreads), kLds, stream, a, row_tiles,
                       static_cast<int>(tiles));
    return hipGetLastError();
}

template <class T, int kDim>
hipError_t launch_window(const AttentionArgs& a, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (a.wide && reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && a.key_strides[2] <= kStagedStride &&
            a.value_strides[2] <= kStagedStride)
            return launch_window_tiles<T, kDim, true>(a, stream);
        return launch_window_tiles<T, kDim, false>(a, stream);
    } else {
        constexpr int kRows = kDim == 256 ? 16 : 32;
        const int64_t row_tiles = (static_cast<int64_t>(a.queries) * a.group + kRows - 1) / kRows;
        const int64_t tiles = row_tiles * a.kv_heads * a.batch;
        if (tiles >= (int64_t{1} << 24) - 256) return hipErrorInvalidValue;  // a grid has below 2^32 threads
        const dim3 grid(static_cast<uint32_t>(blocks_of_tiles(tiles)));
        const int in_row = static_cast<int>(row_tiles), all = static_cast<int>(tiles);
        if (a.wide && a.dim == kDim) hipLaunchKernelGGL(HIP_KERNEL_NAME(window_attention_kernel<kDim, kFullRows>), grid, dim3(kThreads), 0, stream, a, in_row, all);
        else if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(window_attention_kernel<kDim, kWideRows>), grid, dim3(kThreads), 0, stream, a, in_row, all);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(window_attention_kernel<kDim, kNarrow>), grid, dim3(kThreads), 0, stream, a, in_row, all);
        return hipGetLastError();
    }
}

template <class T>
hipError_t launch_window_dim(const AttentionArgs& a, hipStream_t stream) {
    if (a.dim <= 64) return launch_window<T, 64>(a, stream);
    if (a.dim <= 128) return launch_window<T, 128>(a, stream);
    return launch_window<T, 256>(a, stream);
}

}  // namespace

hipError_t launch_window_attention(const AttentionArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_window_dim<float>(args, stream);
        case Type::kFloat16: return launch_window_dim<_Float16>(args, stream);
        default: return launch_window_dim<__bf16>(args, stream);
    }
}

}  // namespace flux
