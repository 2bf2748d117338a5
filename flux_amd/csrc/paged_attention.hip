// Attention of one new token per sequence over a K/V cache in pages (or in one run per sequence), with an optional
// sliding window and sink tokens:
//
//   s_j = scale * <q, k_j>,  m = max s_j,  p_j = exp(s_j - m),  o = sum p_j v_j / sum p_j   over the visible keys j;
//   a sequence of n keys sees j < n with j >= n - window or j < sinks (window 0: all); nothing visible, or nothing whose
//   score is above -inf, gives zeros.
//
// Every key and value row is read once for all query heads of its KV head, and HBM bounds the whole.  A sequence is cut
// into parts of about the same number of tiles as every other part of the batch, one per workgroup, so that ragged
// lengths load the card evenly; the parts of a sequence that was cut leave (o, m, l) in the workspace and a second launch
// joins them: o = sum o_c exp(m_c - M) / sum l_c exp(m_c - M).  (48 sequences to 16384, 32 / 8 heads of 128 in bfloat16:
// 400 us, 4.5 TB/s; 24 to 8192, 9 / 3 heads of 64 in float32: 45 us, the join 4.4 of them.)
//
// A wave takes 16 or 32 keys at a time straight into registers, laid out as the matrix instruction wants them, while the
// tile before is worked on.  Scores come as S^T = K Q^T (rows: keys, columns: query heads), so the lane that holds
// scores of four keys holds what O^T = V^T P needs as its right operand; V's left operand is transposed inside the
// lane by byte permutes.
#include "serving.h"
#include "serving_mfma.h"

namespace flux {
namespace {

constexpr int kDecodeThreads = 256;
constexpr int kDecodeWaves = 4;
constexpr int kColumns = 16;          // query heads of one workgroup
constexpr int kLeastTiles = 4;        // tiles that are worth a workgroup: one per wave
// A call whose sequences have no more tiles than this, by the table's width or the window, leaves each to one workgroup and
// saves the join's launch: two tiles a wave, or eight where the sequences fill the card uncut.  (100 sequences to 1000 keys, 40 / 8 heads of 128 in bfloat16: 55
// against 59 us cut; one of 900 keys, 9 / 3 heads of 64 in float32: 20 us cut, 26 whole.)
constexpr int kWholeTiles = 8, kWholeTilesFull = 32;

// The visible keys of one sequence, as tiles: first the sinks', then the window's.
struct Span {
    int tiles;
    int sink_tiles;
    int first_tile;  // of the window
    int seen;        // keys up to the query's own
    int low;         // first key of the window
    int sinks;
};

// Keys up to the query's own, 0 for a sequence that sees nothing.
__device__ __forceinline__ int seen_of(const AttentionArgs& a, int64_t b) {
    const int64_t slot = a.slots ? a.slots[b] : b;
    if (slot < 0 || slot >= a.slot_count) return 0;
    int64_t n = a.lengths ? a.lengths[slot] : a.keys;
    n = n < 0 ? 0 : (n > a.keys ? a.keys : n);
    const int64_t position = a.starts ? a.starts[b] : n - 1;
    return position < 0 || position >= n ? 0 : static_cast<int>(position) + 1;
}

template <int kTile>
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int seen) {
    Span s;
    s.seen = seen;
    s.low = a.window > 0 && seen > a.window ? seen - a.window : 0;
    s.sinks = a.sinks < s.low ? a.sinks : s.low;
    s.first_tile = s.low / kTile;
    const int of_sinks = (s.sinks + kTile - 1) / kTile;
    s.sink_tiles = of_sinks < s.first_tile ? of_sinks : s.first_tile;
    s.tiles = s.sink_tiles + (seen + kTile - 1) / kTile - s.first_tile;
    return s;
}

// Tiles of a part and the parts of a sequence; one that sees nothing has one part, which writes its zeros.
__device__ __forceinline__ int part_tiles(int64_t total, int target, int least) {
    const int64_t even = (total + target - 1) / target;
    return even < least ? least : static_cast<int>(even);
}
__device__ __forceinline__ int parts_of(int tiles, int each) { return tiles > each ? (tiles + each - 1) / each : 1; }
__device__ __forceinline__ int part_begin(int tiles, int parts, int part) {
    return static_cast<int>(static_cast<int64_t>(tiles) * part / parts);
}

__device__ __forceinline__ int64_t partial_offset(const AttentionArgs& a, int64_t head_tile, int64_t block, int column) {
    const int columns = a.group < kColumns ? a.group : kColumns;
    return ((head_tile * (a.blocks + a.batch) + block) * columns + column) * (a.dim + 2);
}

// The parts' place of each sequence, behind the partials: its first workgroup and their number.  The sequence's first part
// leaves it for the launch that joins them (derived from the lengths again, a join takes 1.2 us longer).
__device__ __host__ __forceinline__ int64_t plan_offset(const AttentionArgs& a) {
    const int64_t columns = a.group < kColumns ? a.group : kColumns;
    const int64_t heads = static_cast<int64_t>(a.kv_heads) * ((a.group + kColumns - 1) / kColumns);
    return heads * (a.blocks + a.batch) * columns * (a.dim + 2);
}

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ int64_t block_sum(int v, int* sums) {
    const int sum = wave_sum_int(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    return static_cast<int64_t>(sums[0]) + sums[1] + sums[2] + sums[3];
}

constexpr int tile_of(int dim, int bytes) { return dim * bytes <= 256 ? 32 : 16; }

// A part of one query head in float32, for 16-bit results that are not finite: the two terms of a weight are of either sign or
// zero, and their products with an infinite value would add up to NaN.  One wave.  It derives all it needs from the
// arguments and `chosen` again: values kept for it would cost the kernel's loop registers.
template <class T, int kTile, bool kPaged>
__device__ void exact_part(const AttentionArgs& a, const int* chosen, int column) {
    const int lane = threadIdx.x & 63;
    const int column_tiles = (a.group + kColumns - 1) / kColumns;
    const int kv_head = blockIdx.y / column_tiles;
    const int64_t head = kv_head * static_cast<int64_t>(a.group) + blockIdx.y % column_tiles * kColumns + column;
    const int b = chosen[0], part = chosen[2], parts = chosen[3];
    const Span span = span_of<kTile>(a, chosen[1]);
    const int from = part_begin(span.tiles, parts, part), to = part_begin(span.tiles, parts, part + 1);
    const int32_t* row = kPaged ? a.table + (a.slots ? a.slots[b] : b) * a.table_stride : nullptr;
    const T* query = static_cast<const T*>(a.query) + b * a.query_strides[0] + head * a.query_strides[1];
    const T* keys = static_cast<const T*>(a.key) + kv_head * a.key_strides[1] + (kPaged ? 0 : b * a.key_strides[0]);
    const T* values = static_cast<const T*>(a.value) + kv_head * a.value_strides[1] + (kPaged ? 0 : b * a.value_strides[0]);

    float top = -INFINITY, weight = 0.0f, sum[kServingMaxDim / kWave];
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c) sum[c] = 0.0f;
    for (int base = from * kTile; base < to * kTile; base += kWave) {
        const int t = (base + lane) / kTile;
        const int position = (t < span.sink_tiles ? t : span.first_tile + t - span.sink_tiles) * kTile + (base + lane) % kTile;
        bool seen = t < to && position < span.seen && (position >= span.low || position < span.sinks);
        int64_t page = 0, in_page = position;
        if (kPaged && seen) {
            const uint32_t column_of = divide(position, a.page);
            page = row[column_of];
            in_page = position - column_of * a.page.divisor;
            seen = page >= 0 && page < a.pages;
        }
        float score = -INFINITY;
        if (seen) {
            const T* key = keys + (kPaged ? page * a.key_strides[0] : 0) + in_page * a.key_strides[2];
            score = 0.0f;
            for (int d = 0; d < a.dim; ++d)
                score = fmaf(static_cast<float>(query[d * a.query_strides[3]]), static_cast<float>(key[d]), score);
            score *= a.scale;
        }
        const float now = fmaxf(top, wave_max(score));
        const float reference = now == -INFINITY ? 0.0f : now;
        const float shrink = top == -INFINITY ? 0.0f : fast_exp2((top - reference) * kLog2e);
        top = now;
        const float p = seen ? fast_exp2((score - reference) * kLog2e + Mfma<T>::kWeightShift) : 0.0f;
        weight = weight * shrink + wave_sum(p);
#pragma unroll
        for (int c = 0; c < kServingMaxDim / kWave; ++c) sum[c] *= shrink;
        const int64_t mine = seen ? (kPaged ? page * a.value_strides[0] : 0) + in_page * a.value_strides[2] : -1;
        for (int j = 0; j < kWave; ++j) {
            const int64_t of = __shfl(mine, j, kWave);
            const float pj = __shfl(p, j, kWave);
            if (of < 0) continue;
#pragma unroll
            for (int c = 0; c < kServingMaxDim / kWave; ++c)
                if (kWave * c + lane < a.dim) sum[c] = fmaf(pj, static_cast<float>(values[of + kWave * c + lane]), sum[c]);
        }
        // What is NaN stays NaN: a head whose sums all are is done.
        bool lost = true;
#pragma unroll
        for (int c = 0; c < kServingMaxDim / kWave; ++c) lost = lost && (kWave * c + lane >= a.dim || sum[c] != sum[c]);
        if (__all(weight != weight || lost)) break;
    }
    T* out = static_cast<T*>(a.out) + (b * static_cast<int64_t>(a.query_heads) + head) * a.dim;
    float* partial = a.workspace + partial_offset(a, blockIdx.y, blockIdx.x, column);
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c) {
        const int d = kWave * c + lane;
        if (d >= a.dim) continue;
        if (parts == 1) out[d] = static_cast<T>(weight == 0.0f ? 0.0f : sum[c] / weight);
        else partial[d] = sum[c];
    }
    if (parts > 1 && lane == 0) {
        partial[a.dim] = top;
        partial[a.dim + 1] = weight;
    }
}

template <class T, int kDim, bool kPaged, Rows kRows>
__global__ void __launch_bounds__(kDecodeThreads, kDim * sizeof(T) <= 512 ? 2 : 1) decode_attention_kernel(AttentionArgs a) {
    using M = Mfma<T>;
    constexpr int kTile = tile_of(kDim, sizeof(T));
    constexpr int kSubs = kTile / 16;
    constexpr int kFragments = M::template key_fragments<kDim>();  // of 16 bytes per lane
    constexpr int kChunks = M::template value_chunks<kDim>();
    constexpr int kBlocks = kDim / 16;  // accumulators of 16 dims
    using Value = typename M::template ValueChunk<kDim>;

    __shared__ int sums[kDecodeWaves];
    __shared__ int chosen[4];  // sequence, keys it sees, part, parts
    __shared__ float merge[2][kBlocks * 4 + 2][kWave];

    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int n16 = lane & 15;
    const int g = lane >> 4;
    const int column_tiles = (a.group + kColumns - 1) / kColumns;
    const int kv_head = blockIdx.y / column_tiles;
    const int column0 = blockIdx.y % column_tiles * kColumns;
    const int columns = a.group - column0 < kColumns ? a.group - column0 : kColumns;

    // The part of this workgroup: the blockIdx.x-th of all sequences' parts.
    int64_t total = 0;
    int seen = 0;
    for (int base = 0; base < a.batch; base += kDecodeThreads) {
        const int b = base + static_cast<int>(threadIdx.x);
        seen = b < a.batch ? seen_of(a, b) : 0;
        total += block_sum(span_of<kTile>(a, seen).tiles, sums);
    }
    const int each = part_tiles(total, a.blocks, a.least);
    int64_t running = 0;
    for (int base = 0; base < a.batch; base += kDecodeThreads) {
        const int b = base + static_cast<int>(threadIdx.x);
        if (a.batch > kDecodeThreads) seen = b < a.batch ? seen_of(a, b) : 0;
        const int parts = b < a.batch ? parts_of(span_of<kTile>(a, seen).tiles, each) : 0;
        const int inclusive = wave_scan_int(parts);
        __syncthreads();
        if (lane == 63) sums[wave] = inclusive;
        __syncthreads();
        int64_t begin = running + inclusive - parts;
        for (int w = 0; w < wave; ++w) begin += sums[w];
        running += static_cast<int64_t>(sums[0]) + sums[1] + sums[2] + sums[3];
        if (blockIdx.x >= begin && blockIdx.x < begin + parts) {
            chosen[0] = b;
            chosen[1] = seen;
            chosen[2] = static_cast<int>(blockIdx.x - begin);
            chosen[3] = parts;
        }
        if (running > blockIdx.x) break;
    }
    if (running <= blockIdx.x) return;
    __syncthreads();
    const int b = chosen[0], part = chosen[2], parts = chosen[3];
    const Span span = span_of<kTile>(a, chosen[1]);
    if (blockIdx.y == 0 && part == 0 && threadIdx.x == 0) {
        int* plan = reinterpret_cast<int*>(a.workspace + plan_offset(a)) + 2 * b;
        plan[0] = blockIdx.x;
        plan[1] = parts;
    }
    const int from = part_begin(span.tiles, parts, part), to = part_begin(span.tiles, parts, part + 1);
    const int64_t slot = kPaged && a.slots ? a.slots[b] : b;
    const int32_t* row = kPaged ? a.table + (span.tiles > 0 ? slot : 0) * a.table_stride : nullptr;
    const T* keys = static_cast<const T*>(a.key) + kv_head * a.key_strides[1] + (kPaged ? 0 : b * a.key_strides[0]);
    const T* values = static_cast<const T*>(a.value) + kv_head * a.value_strides[1] + (kPaged ? 0 : b * a.value_strides[0]);

    // A tile's positions, and the page of this lane's key in it (-1: not attended).
    auto tile_key = [&](int t) { return (t < span.sink_tiles ? t : span.first_tile + t - span.sink_tiles) * kTile; };
    struct Pages {
        int page[kSubs];
    };
    auto look_up = [&](int t, Pages& p) {
        const int base = tile_key(t);
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
            const int position = base + 16 * s + n16;
            p.page[s] = t < to && position < span.seen && (position >= span.low || position < span.sinks) ? 0 : -1;
            if constexpr (kPaged) {
                if (p.page[s] == 0) p.page[s] = row[divide(position, a.page)];
            }
        }
    };
    struct Tile {
        typename M::Fragment key[kSubs][kFragments];
        Value value[kSubs][4][kChunks];
        int held[kSubs][4];  // page of each value row, -1: not attended
        bool partial;        // some key of the tile is not attended; its rows are the pool's first
    };
    auto load = [&](int t, const Pages& p, Tile& tile) {
        const int base = tile_key(t);
        bool whole = true;
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
            int page = p.page[s];
            if constexpr (kPaged) page = page < a.pages ? page : -1;
            whole = whole && page >= 0;
            const int position = base + 16 * s + n16;
            const uint32_t in_page = kPaged ? position - divide(position, a.page) * a.page.divisor : (page >= 0 ? position : 0);
            const T* k = keys + (kPaged && page > 0 ? page * a.key_strides[0] : 0) + in_page * a.key_strides[2];
#pragma unroll
            for (int f = 0; f < kFragments; ++f)
                tile.key[s][f] = M::template load_row<kRows>(k, M::kKeyStep * f + M::kPer * g, a.dim);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int of = __shfl(page, 4 * g + i, kWave);
                tile.held[s][i] = of;
                const uint32_t value_position = base + 16 * s + 4 * g + i;
                const uint32_t value_row = kPaged ? value_position - divide(value_position, a.page) * a.page.divisor : (of >= 0 ? value_position : 0);
                const T* v = values + (kPaged && of > 0 ? of * a.value_strides[0] : 0) + value_row * a.value_strides[2];
#pragma unroll
                for (int c = 0; c < kChunks; ++c) tile.value[s][i][c] = M::template load_value<kDim, kRows>(v, c, n16, a.dim);
            }
        }
        tile.partial = !__all(whole);
    };

    f32x4 out[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) out[i] = f32x4{0, 0, 0, 0};
    float top = -INFINITY, weight = 0.0f;
    typename M::Fragment query[kFragments];  // right operand of S^T: this lane's query head, zero behind the last one

    auto work = [&](Tile& tile) {
        if (tile.partial) {  // a weight of zero does not undo a NaN
#pragma unroll
            for (int s = 0; s < kSubs; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) tile.value[s][i][c] = tile.held[s][i] >= 0 ? tile.value[s][i][c] : Value{};
        }
        f32x4 score[kSubs];
        float highest = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
            score[s] = multiply_keys<M, false>(tile.key[s], query, g, a.dim);
            sum += (score[s][0] + score[s][1]) + (score[s][2] + score[s][3]);
        }
        // An infinity of a key repeated behind the head's dims met a zero there: again without it, which is rare (clearing
        // every tile costs 4% of 64 windows of 2052 keys, 8 heads of 80 in float16).
        if constexpr (kRows != kFullRows) {
            if (__any(!(fabsf(sum) < INFINITY))) {
#pragma unroll
                for (int s = 0; s < kSubs; ++s) score[s] = multiply_keys<M, true>(tile.key[s], query, g, a.dim);
            }
        }
#pragma unroll
        for (int s = 0; s < kSubs; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                score[s][i] = tile.held[s][i] >= 0 ? score[s][i] * a.scale : -INFINITY;
                highest = fmaxf(highest, score[s][i]);
            }
        }
        highest = fmaxf(highest, __shfl_xor(highest, 16, kWave));
        highest = fmaxf(highest, __shfl_xor(highest, 32, kWave));
        if (__any(highest > top)) {
            const float now = fmaxf(top, highest);
            const float shrink = top == -INFINITY ? 0.0f : fast_exp2((top - now) * kLog2e);
            top = now;
            weight *= shrink;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) out[i] *= shrink;
        }
        const float reference = top == -INFINITY ? 0.0f : top;
        float p[kSubs][4];
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[s][i] = fast_exp2((score[s][i] - reference) * kLog2e + M::kWeightShift);
                weight += p[s][i];
            }
        M::template multiply_value<kDim, kSubs>(tile.value, p, out);
    };

    // Two tiles in registers where two waves per SIMD still fit: the next one's rows arrive while one is worked on (48
    // sequences of 2 to 16k keys, 8 KV heads of 128 in bfloat16: 406 us; one tile: 417; two tiles and one wave: 511).
    constexpr bool kAhead = kDim * static_cast<int>(sizeof(T)) <= 256;
    Pages pages;
    Tile even;
    look_up(from + wave, pages);
    {
        const int64_t head = kv_head * static_cast<int64_t>(a.group) + column0 + (n16 < columns ? n16 : 0);
        const T* q = static_cast<const T*>(a.query) + b * a.query_strides[0] + head * a.query_strides[1];
        load_query<T, kFragments, M::kKeyStep>(query, q, a.query_strides[3], a.query_wide, M::kPer * g, a.dim, n16 < columns);
    }
    // A wave's tile numbers are the same in all its lanes, and said to be: the branches on them are scalar.
    const int first_tile = __builtin_amdgcn_readfirstlane(from + wave);
    if constexpr (kAhead) {
        Tile odd;
        if (first_tile < to) load(first_tile, pages, even);
        look_up(first_tile + kDecodeWaves, pages);
        for (int t = first_tile; t < to; t += 2 * kDecodeWaves) {
            const bool second = t + kDecodeWaves < to;
            if (second) load(t + kDecodeWaves, pages, odd);
            look_up(t + 2 * kDecodeWaves, pages);
            work(even);
            if (!second) break;
            if (t + 2 * kDecodeWaves < to) load(t + 2 * kDecodeWaves, pages, even);
            look_up(t + 3 * kDecodeWaves, pages);
            work(odd);
        }
    } else {
        for (int t = first_tile; t < to; t += kDecodeWaves) {
            load(t, pages, even);
            look_up(t + kDecodeWaves, pages);
            work(even);
        }
    }
    weight += __shfl_xor(weight, 16, kWave);
    weight += __shfl_xor(weight, 32, kWave);

    // Join the four waves in registers: 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
    for (int half = kDecodeWaves / 2; half >= 1; half /= 2) {
        if (half == 1) __syncthreads();
        if (wave >= half && wave < 2 * half) {
            float(*to_merge)[kWave] = merge[wave - half];
#pragma unroll
            for (int i = 0; i < kBlocks * 4; ++i) to_merge[i][lane] = out[i / 4][i % 4];
            to_merge[kBlocks * 4][lane] = top;
            to_merge[kBlocks * 4 + 1][lane] = weight;
        }
        __syncthreads();
        if (wave < half) {
            const float(*other)[kWave] = merge[wave];
            const float other_top = other[kBlocks * 4][lane];
            const float now = fmaxf(top, other_top);
            const float mine_scale = top == -INFINITY ? 0.0f : fast_exp2((top - now) * kLog2e);
            const float other_scale = other_top == -INFINITY ? 0.0f : fast_exp2((other_top - now) * kLog2e);
            top = now;
            weight = weight * mine_scale + other[kBlocks * 4 + 1][lane] * other_scale;
#pragma unroll
            for (int i = 0; i < kBlocks * 4; ++i)
                out[i / 4][i % 4] = out[i / 4][i % 4] * mine_scale + other[i][lane] * other_scale;
        }
    }
    if (wave != 0) return;
    uint32_t again = 0;  // heads whose sums are not finite
    if constexpr (sizeof(T) == 2) {
        f32x4 sum = out[0];  // keeps NaN and infinity; dims behind the head's repeat its first ones
#pragma unroll
        for (int i = 1; i < kBlocks; ++i) sum += out[i];
        const uint64_t odd = __ballot(n16 < columns && !(fabsf((sum[0] + sum[1]) + (sum[2] + sum[3]) + weight) < INFINITY));
        again = static_cast<uint32_t>((odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xffff);
    }
    if (n16 < columns && !(again >> n16 & 1)) {
        if (parts == 1) {
            const int64_t head = kv_head * static_cast<int64_t>(a.group) + column0 + n16;
            T* o = static_cast<T*>(a.out) + (b * static_cast<int64_t>(a.query_heads) + head) * a.dim;
            M::template each_dim<kDim>(g, a.dim, [&](int i, int r, int d) {
                o[d] = static_cast<T>(weight == 0.0f ? 0.0f : out[i][r] / weight);
            });
        } else {
            float* o = a.workspace + partial_offset(a, blockIdx.y, blockIdx.x, n16);
            M::template each_dim<kDim>(g, a.dim, [&](int i, int r, int d) { o[d] = out[i][r]; });
            if (g == 0) {
                o[a.dim] = top;
                o[a.dim + 1] = weight;
            }
        }
    }
    if constexpr (sizeof(T) == 2) {
        if (again) {
            // The arguments by their address, which the compiler does not see through: read here, not held since the start.
            uint64_t held = reinterpret_cast<uint64_t>((const void*)__builtin_amdgcn_kernarg_segment_ptr());
            asm volatile("" : "+s"(held));
            for (; again; again &= again - 1)
                exact_part<T, kTile, kPaged>(*reinterpret_cast<const AttentionArgs*>(held), chosen, __ffs(again) - 1);
        }
    }
}

// Joins the parts of a sequence that was cut.  Workgroup (sequence, column tile of a KV head, 256 of the
// tile's heads and dims): the parts' shares first.
constexpr int kJoinParts = 128;  // parts whose shares are kept

template <class T>
__global__ void __launch_bounds__(kDecodeThreads) decode_join_kernel(AttentionArgs a) {
    __shared__ float share[kJoinParts][kColumns];
    __shared__ float tops[kColumns], weights[kColumns];
    const int b = blockIdx.x;
    const int* plan = reinterpret_cast<const int*>(a.workspace + plan_offset(a)) + 2 * b;
    const int first = plan[0], parts = plan[1];
    if (parts == 1) return;
    const int column_tiles = (a.group + kColumns - 1) / kColumns;
    const int column0 = blockIdx.y % column_tiles * kColumns;
    const int columns = a.group - column0 < kColumns ? a.group - column0 : kColumns;
    const int64_t stride = partial_offset(a, 0, 1, 0);
    const float* o = a.workspace + partial_offset(a, blockIdx.y, first, 0);
    const int width = a.dim + 2;

    // Sixteen lanes go over the parts of one head: its maximum, the parts' shares (kept where there is room), their sum.
    {
        const int column = threadIdx.x / 16, lane = threadIdx.x % 16;
        const float* mine = o + column * width + a.dim;
        float top = -INFINITY, weight = 0.0f;
        if (column < columns) {
#pragma unroll 4
            for (int p = lane; p < parts; p += 16) {
                const float part_top = mine[p * stride], part_weight = mine[p * stride + 1];
                if (p < kJoinParts) share[p][column] = part_top;
                const float now = fmaxf(top, part_top);
                const float kept = top == -INFINITY ? 0.0f : fast_exp2((top - now) * kLog2e);
                const float added = part_top == -INFINITY ? 0.0f : fast_exp2((part_top - now) * kLog2e);
                weight = weight * kept + part_weight * added;
                top = now;
            }
        }
        const float all = row16_max(top);
        weight = row16_sum(weight * (top == -INFINITY ? 0.0f : fast_exp2((top - all) * kLog2e)));
        if (column < columns)
            for (int p = lane; p < parts && p < kJoinParts; p += 16)
                share[p][column] = share[p][column] == -INFINITY ? 0.0f : fast_exp2((share[p][column] - all) * kLog2e);
        if (lane == 0) {
            tops[column] = all;
            weights[column] = weight;
        }
    }
    const int64_t head = static_cast<int64_t>(blockIdx.y / column_tiles) * a.group + column0;
    T* out = static_cast<T*>(a.out) + (b * static_cast<int64_t>(a.query_heads) + head) * a.dim;
    const int items = columns * a.dim;
    __syncthreads();
    const int item = blockIdx.z * kDecodeThreads + threadIdx.x;
    if (item < items) {
        const int column = item / a.dim, d = item - column * a.dim;
        const float* from = o + column * width + d;
        float sum = 0.0f;
        const int kept = parts < kJoinParts ? parts : kJoinParts;
#pragma unroll 8
        for (int p = 0; p < kept; ++p) sum += from[p * stride] * share[p][column];
        for (int p = kept; p < parts; ++p) {
            const float part_top = from[p * stride + a.dim - d];
            sum += from[p * stride] * (part_top == -INFINITY ? 0.0f : fast_exp2((part_top - tops[column]) * kLog2e));
        }
        out[item] = static_cast<T>(weights[column] == 0.0f ? 0.0f : sum / weights[column]);
    }
}

constexpr int padded_dim(int dim) { return dim <= 64 ? 64 : (dim <= 128 ? 128 : 256); }

// Tiles that a sequence can have.
int64_t most_tiles(const AttentionArgs& a, int tile) {
    const int64_t all = (a.keys + tile - 1) / tile;
    if (a.window == 0) return all;
    const int64_t windowed = (a.sinks + tile - 1) / tile + (a.window + tile - 1) / tile + 1;
    return windowed < all ? windowed : all;
}

template <class T, int kDim>
hipError_t launch_decode(AttentionArgs a, hipStream_t stream) {
    const int column_tiles = (a.group + kColumns - 1) / kColumns;
    const int limit = static_cast<int64_t>(a.batch) * a.kv_heads * column_tiles >= 512 ? kWholeTilesFull : kWholeTiles;
    const bool whole = most_tiles(a, tile_of(kDim, sizeof(T))) <= limit;
    a.least = whole ? limit : kLeastTiles;
    const dim3 grid(a.blocks + a.batch, a.kv_heads * column_tiles);
    if (a.pages > 0) {
        if (a.wide && a.dim == kDim) hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, true, kFullRows>), grid, dim3(kDecodeThreads), 0, stream, a);
        else if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, true, kWideRows>), grid, dim3(kDecodeThreads), 0, stream, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, true, kNarrow>), grid, dim3(kDecodeThreads), 0, stream, a);
    } else {
        if (a.wide && a.dim == kDim) hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, false, kFullRows>), grid, dim3(kDecodeThreads), 0, stream, a);
        else if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, false, kWideRows>), grid, dim3(kDecodeThreads), 0, stream, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, false, kNarrow>), grid, dim3(kDecodeThreads), 0, stream, a);
    }
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess) return launched;
    if (whole) return hipSuccess;
    const int items = ((a.group < kColumns ? a.group : kColumns) * a.dim + kDecodeThreads - 1) / kDecodeThreads;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_join_kernel<T>), dim3(a.batch, a.kv_heads * column_tiles, items),
                       dim3(kDecodeThreads), 0, stream, a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_decode_dim(const AttentionArgs& a, hipStream_t stream) {
    switch (padded_dim(a.dim)) {
        case 64: return launch_decode<T, 64>(a, stream);
        case 128: return launch_decode<T, 128>(a, stream);
        default: return launch_decode<T, 256>(a, stream);
    }
}

}  // namespace

// Parts that the batch is cut into: two workgroups on each of 256 CUs, less one per sequence, whose last part may be short;
// none without kLeastTiles tiles of 16 keys.
int decode_attention_blocks(int batch, int64_t keys, int kv_heads, int group, int window, int sinks) {
    int64_t seen = keys;
    if (window > 0 && static_cast<int64_t>(window) + sinks + 32 < keys) seen = static_cast<int64_t>(window) + sinks + 32;
    const int64_t most = (batch * ((seen + 15) / 16 + 2) + kLeastTiles - 1) / kLeastTiles;
    const int64_t heads = static_cast<int64_t>(kv_heads) * ((group + kColumns - 1) / kColumns);
    int64_t blocks = (512 + heads - 1) / heads;
    blocks = blocks - batch > blocks / 2 ? blocks - batch : (blocks + 1) / 2;
    if (blocks > most) blocks = most;
    return static_cast<int>(blocks < 1 ? 1 : blocks);
}

size_t decode_attention_workspace_floats(const AttentionArgs& a) {
    return static_cast<size_t>(plan_offset(a) + 2 * static_cast<int64_t>(a.batch));
}

hipError_t launch_decode_attention(const AttentionArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_decode_dim<float>(args, stream);
        case Type::kFloat16: return launch_decode_dim<_Float16>(args, stream);
        default: return launch_decode_dim<__bf16>(args, stream);
    }
}

}  // namespace flux
