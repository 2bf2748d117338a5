// Attention of one new token per sequence over a K/V cache in pages (or in one run per sequence), with an optional
// sliding window and sink tokens:
//
//   s_j = scale * <q, k_j>,  m = max s_j,  p_j = exp(s_j - m),  o = sum p_j v_j / sum p_j   over the visible keys j;
//   a sequence of n keys sees j < n with j >= n - window or j < sinks (window 0: all); nothing visible gives zeros.
//
// Every key and value row is read once for all query heads of its KV head, and HBM bounds the whole.  The tiles of all
// sequences form one line that is cut into equal parts, one per workgroup, so that ragged lengths load the card
// evenly; a part that begins or ends inside a sequence leaves (o, m, l) in the workspace and a second launch joins
// them: o = sum o_c exp(m_c - M) / sum l_c exp(m_c - M).
//
// A wave takes 16 or 32 keys at a time straight into registers, laid out as the matrix instruction wants them.  Scores
// come as S^T = K Q^T (rows: keys, columns: query heads), so the lane that holds scores of four keys holds what
// O^T = V^T P needs as its right operand; V's left operand is transposed inside the lane by byte permutes.
#include "serving.h"
#include "serving_mfma.h"

namespace flux {
namespace {

constexpr int kDecodeThreads = 256;
constexpr int kDecodeWaves = 4;
constexpr int kColumns = 16;          // query heads of one workgroup
constexpr int kLeastTiles = 4;        // tiles that are worth a workgroup: one per wave

// The visible keys of one sequence, as tiles: first the sinks', then the window's.
struct Span {
    int tiles;
    int sink_tiles;
    int first_tile;  // of the window
    int seen;        // keys up to the query's own
    int low;         // first key of the window
    int sinks;
};

template <int kTile>
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int64_t b) {
    Span s{0, 0, 0, 0, 0, 0};
    const int64_t slot = a.slots ? a.slots[b] : b;
    if (slot < 0 || slot >= a.slot_count) return s;
    int64_t n = a.lengths ? a.lengths[slot] : a.keys;
    n = n < 0 ? 0 : (n > a.keys ? a.keys : n);
    const int64_t position = a.starts ? a.starts[b] : n - 1;
    if (position < 0 || position >= n) return s;
    s.seen = static_cast<int>(position) + 1;
    s.low = a.window > 0 && s.seen > a.window ? s.seen - a.window : 0;
    s.sinks = a.sinks < s.low ? a.sinks : s.low;
    s.first_tile = s.low / kTile;
    const int of_sinks = (s.sinks + kTile - 1) / kTile;
    s.sink_tiles = of_sinks < s.first_tile ? of_sinks : s.first_tile;
    s.tiles = s.sink_tiles + (s.seen + kTile - 1) / kTile - s.first_tile;
    return s;
}

// Parts in use and the tiles [lo, hi) of one of them, of `total` tiles.
__device__ __forceinline__ int parts_of(int64_t total, int blocks) {
    const int64_t most = (total + kLeastTiles - 1) / kLeastTiles;
    return static_cast<int>(most < blocks ? most : blocks);
}
__device__ __forceinline__ int64_t part_begin(int64_t total, int parts, int64_t part) { return total * part / parts; }
// The part that holds a tile: the largest one that begins at or before it.
__device__ __forceinline__ int part_of(int64_t total, int parts, int64_t tile) {
    int64_t part = (tile * parts) / total;
    while (part + 1 < parts && part_begin(total, parts, part + 1) <= tile) ++part;
    return static_cast<int>(part);
}

__device__ __forceinline__ int64_t partial_offset(const AttentionArgs& a, int64_t head_tile, int part, int which,
                                                  int column) {
    const int columns = a.group < kColumns ? a.group : kColumns;
    return (((head_tile * a.blocks + part) * 2 + which) * columns + column) * (a.dim + 2);
}

__device__ __forceinline__ int64_t block_sum(int v, int* sums) {
    const int inclusive = static_cast<int>(wave_sum_int(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = inclusive;
    __syncthreads();
    return static_cast<int64_t>(sums[0]) + sums[1] + sums[2] + sums[3];
}

template <class T, int kDim, bool kPaged, bool kWide>
__global__ void __launch_bounds__(kDecodeThreads) decode_attention_kernel(AttentionArgs a) {
    using M = Mfma<T>;
    constexpr int kTile = kDim * static_cast<int>(sizeof(T)) <= 256 ? 32 : 16;
    constexpr int kSubs = kTile / 16;
    constexpr int kFragments = M::template key_fragments<kDim>();  // of 16 bytes per lane
    constexpr int kChunks = M::template value_chunks<kDim>();
    constexpr int kBlocks = kDim / 16;  // accumulators of 16 dims
    using Value = typename M::template ValueChunk<kDim>;

    __shared__ int sums[kDecodeWaves];
    __shared__ int prefix[kDecodeThreads + 1];
    __shared__ int first_index;
    __shared__ float merge[2][kBlocks * 4 + 2][kWave];

    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int n16 = lane & 15;
    const int g = lane >> 4;
    const int column_tiles = (a.group + kColumns - 1) / kColumns;
    const int kv_head = blockIdx.y / column_tiles;
    const int column0 = blockIdx.y % column_tiles * kColumns;
    const int columns = a.group - column0 < kColumns ? a.group - column0 : kColumns;

    int64_t total = 0;
    for (int base = 0; base < a.batch; base += kDecodeThreads) {
        const int b = base + threadIdx.x;
        total += block_sum(b < a.batch ? span_of<kTile>(a, b).tiles : 0, sums);
    }
    if (total == 0) return;
    const int parts = parts_of(total, a.blocks);
    const int part = blockIdx.x;
    if (part >= parts) return;
    const int64_t lo = part_begin(total, parts, part), hi = part_begin(total, parts, part + 1);

    int64_t running = 0;
    for (int base = 0; base < a.batch && running < hi; base += kDecodeThreads) {
        // Where this round's sequences begin on the line.
        const int mine = base + static_cast<int>(threadIdx.x) < a.batch ? span_of<kTile>(a, base + threadIdx.x).tiles : 0;
        const int inclusive = wave_scan_int(mine);
        __syncthreads();
        if (lane == 63) sums[wave] = inclusive;
        if (threadIdx.x == 0) first_index = kDecodeThreads;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < wave; ++w) before += sums[w];
        const int begin = before + inclusive - mine;
        prefix[threadIdx.x] = begin;
        if (threadIdx.x == kDecodeThreads - 1) prefix[kDecodeThreads] = begin + mine;
        if (mine > 0 && running + begin + mine > lo && running + begin <= lo) first_index = threadIdx.x;
        if (mine > 0 && begin == 0 && running > lo) first_index = threadIdx.x;
        __syncthreads();
        const int round_total = prefix[kDecodeThreads];

        for (int j = first_index; j < kDecodeThreads && running + prefix[j] < hi; ++j) {
            const int tiles = prefix[j + 1] - prefix[j];
            if (tiles == 0) continue;
            const int b = base + j;
            const int64_t begins = running + prefix[j];
            const int from = static_cast<int>(lo > begins ? lo - begins : 0);
            const int to = static_cast<int>(hi - begins < tiles ? hi - begins : tiles);
            const Span span = span_of<kTile>(a, b);
            const int64_t slot = a.slots ? a.slots[b] : b;
            const int32_t* row = kPaged ? a.table + slot * a.table_stride : nullptr;
            const T* keys = static_cast<const T*>(a.key) + kv_head * a.key_strides[1] + (kPaged ? 0 : b * a.key_strides[0]);
            const T* values = static_cast<const T*>(a.value) + kv_head * a.value_strides[1] +
                              (kPaged ? 0 : b * a.value_strides[0]);

            // Right operand of S^T: this lane's query head, zero behind the last one.
            typename M::Fragment query[kFragments];
            {
                const int64_t head = kv_head * static_cast<int64_t>(a.group) + column0 + n16;
                const T* q = static_cast<const T*>(a.query) + b * a.query_strides[0] + head * a.query_strides[1];
#pragma unroll
                for (int f = 0; f < kFragments; ++f)
                    query[f] = M::load_query(q, a.query_strides[3], M::kKeyStep * f + M::kPer * g, a.dim, n16 < columns);
            }

            f32x4 out[kBlocks];
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) out[i] = f32x4{0, 0, 0, 0};
            float top = -INFINITY, weight = 0.0f;

            for (int t = from + wave; t < to; t += kDecodeWaves) {
                const int base_key = (t < span.sink_tiles ? t : span.first_tile + t - span.sink_tiles) * kTile;
                typename M::Fragment key[kSubs][kFragments];
                Value value[kSubs][4][kChunks];
                int held[kSubs][4];  // page of this lane's value rows, -1: not attended
#pragma unroll
                for (int s = 0; s < kSubs; ++s) {
                    const int position = base_key + 16 * s + n16;
                    int page = position < span.seen && (position >= span.low || position < span.sinks) ? 0 : -1;
                    uint32_t in_page = position;
                    if constexpr (kPaged) {
                        const uint32_t column = divide(position, a.page);
                        in_page = position - column * a.page.divisor;
                        if (page == 0) {
                            page = row[column];
                            if (page >= a.pages) page = -1;
                        }
                    }
                    const T* k = keys + (kPaged ? page * a.key_strides[0] : 0) + in_page * a.key_strides[2];
#pragma unroll
                    for (int f = 0; f < kFragments; ++f)
                        key[s][f] = M::template load_row<kWide>(k, M::kKeyStep * f + M::kPer * g, a.dim, page >= 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        held[s][i] = __shfl(page, 4 * g + i, kWave);
                        const uint32_t value_position = base_key + 16 * s + 4 * g + i;
                        uint32_t value_row = value_position;
                        if constexpr (kPaged) value_row -= divide(value_position, a.page) * a.page.divisor;
                        const T* v = values + (kPaged ? held[s][i] * a.value_strides[0] : 0) + value_row * a.value_strides[2];
#pragma unroll
                        for (int c = 0; c < kChunks; ++c)
                            value[s][i][c] = M::template load_value<kDim, kWide>(v, c, n16, a.dim, held[s][i] >= 0);
                    }
                }

                f32x4 score[kSubs];
                float highest = -INFINITY;
#pragma unroll
                for (int s = 0; s < kSubs; ++s) {
                    score[s] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int f = 0; f < kFragments; ++f) M::multiply_key(key[s][f], query[f], score[s]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        score[s][i] = held[s][i] >= 0 ? score[s][i] * a.scale : -INFINITY;
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
                M::template multiply_value<kDim, kSubs>(value, p, out);
            }
            weight += __shfl_xor(weight, 16, kWave);
            weight += __shfl_xor(weight, 32, kWave);

            // Join the four waves in registers: 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
            for (int half = kDecodeWaves / 2; half >= 1; half /= 2) {
                __syncthreads();
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

            if (wave == 0 && n16 < columns) {
                const bool whole = from == 0 && to == tiles;
                const int64_t head = kv_head * static_cast<int64_t>(a.group) + column0 + n16;
                if (whole) {
                    T* o = static_cast<T*>(a.out) + (b * static_cast<int64_t>(a.query_heads) + head) * a.dim;
                    M::template each_dim<kDim>(g, a.dim, [&](int i, int r, int d) {
                        o[d] = static_cast<T>(weight == 0.0f ? 0.0f : out[i][r] / weight);
                    });
                } else {
                    float* o = a.workspace + partial_offset(a, blockIdx.y, part, from == 0 ? 1 : 0, n16);
                    M::template each_dim<kDim>(g, a.dim, [&](int i, int r, int d) { o[d] = out[i][r]; });
                    if (g == 0) {
                        o[a.dim] = top;
                        o[a.dim + 1] = weight;
                    }
                }
            }
        }
        running += round_total;
    }
}

// Joins the parts of a sequence that was cut, or writes zeros for one that sees nothing.  Workgroup (sequence, head).
template <class T, int kTile>
__global__ void __launch_bounds__(kDecodeThreads) decode_join_kernel(AttentionArgs a) {
    __shared__ int sums[kDecodeWaves];
    const int64_t b = blockIdx.x / a.query_heads;
    const int head = blockIdx.x % a.query_heads;
    int64_t total = 0, begins = 0;
    for (int base = 0; base < a.batch; base += kDecodeThreads) {
        const int i = base + threadIdx.x;
        const int tiles = i < a.batch ? span_of<kTile>(a, i).tiles : 0;
        total += block_sum(tiles, sums);
        begins += block_sum(i < b ? tiles : 0, sums);
    }
    const int tiles = span_of<kTile>(a, b).tiles;
    T* out = static_cast<T*>(a.out) + (b * a.query_heads + head) * a.dim;
    const int d = threadIdx.x;
    if (tiles == 0) {
        if (d < a.dim) out[d] = static_cast<T>(0.0f);
        return;
    }
    const int parts = parts_of(total, a.blocks);
    const int first = part_of(total, parts, begins), last = part_of(total, parts, begins + tiles - 1);
    if (first == last) return;
    const int kv_head = head / a.group, in_group = head % a.group;
    const int64_t head_tile = static_cast<int64_t>(kv_head) * ((a.group + kColumns - 1) / kColumns) + in_group / kColumns;
    const int column = in_group % kColumns;
    float top = -INFINITY;
    for (int part = first; part <= last; ++part)
        top = fmaxf(top, a.workspace[partial_offset(a, head_tile, part, part == first ? 1 : 0, column) + a.dim]);
    float weight = 0.0f, sum = 0.0f;
    for (int part = first; part <= last; ++part) {
        const float* o = a.workspace + partial_offset(a, head_tile, part, part == first ? 1 : 0, column);
        const float share = o[a.dim] == -INFINITY ? 0.0f : fast_exp2((o[a.dim] - top) * kLog2e);
        weight += o[a.dim + 1] * share;
        if (d < a.dim) sum += o[d] * share;
    }
    if (d < a.dim) out[d] = static_cast<T>(weight == 0.0f ? 0.0f : sum / weight);
}

constexpr int tile_of(int dim, int bytes) { return dim * bytes <= 256 ? 32 : 16; }
constexpr int padded_dim(int dim) { return dim <= 64 ? 64 : (dim <= 128 ? 128 : 256); }

template <class T, int kDim>
hipError_t launch_decode(const AttentionArgs& a, hipStream_t stream) {
    const int column_tiles = (a.group + kColumns - 1) / kColumns;
    const dim3 grid(a.blocks, a.kv_heads * column_tiles);
    if (a.pages > 0) {
        if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, true, true>), grid, dim3(kDecodeThreads), 0, stream, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, true, false>), grid, dim3(kDecodeThreads), 0, stream, a);
    } else {
        if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, false, true>), grid, dim3(kDecodeThreads), 0, stream, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_attention_kernel<T, kDim, false, false>), grid, dim3(kDecodeThreads), 0, stream, a);
    }
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess) return launched;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(decode_join_kernel<T, tile_of(kDim, sizeof(T))>), dim3(a.batch * a.query_heads),
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

// Two workgroups per CU of the 256, and none without kLeastTiles tiles of 16 keys.
int decode_attention_blocks(int batch, int64_t keys, int kv_heads, int group, int window, int sinks) {
    int64_t seen = keys;
    if (window > 0 && static_cast<int64_t>(window) + sinks + 32 < keys) seen = static_cast<int64_t>(window) + sinks + 32;
    const int64_t most = (batch * ((seen + 15) / 16 + 2) + kLeastTiles - 1) / kLeastTiles;
    const int64_t heads = static_cast<int64_t>(kv_heads) * ((group + kColumns - 1) / kColumns);
    int64_t blocks = (512 + heads - 1) / heads;
    if (blocks > most) blocks = most;
    return static_cast<int>(blocks < 1 ? 1 : blocks);
}

size_t decode_attention_workspace_floats(const AttentionArgs& a) {
    const size_t columns = a.group < kColumns ? a.group : kColumns;
    const size_t heads = static_cast<size_t>(a.kv_heads) * ((a.group + kColumns - 1) / kColumns);
    return heads * a.blocks * 2 * columns * (a.dim + 2);
}

hipError_t launch_decode_attention(const AttentionArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_decode_dim<float>(args, stream);
        case Type::kFloat16: return launch_decode_dim<_Float16>(args, stream);
        default: return launch_decode_dim<__bf16>(args, stream);
    }
}

}  // namespace flux
