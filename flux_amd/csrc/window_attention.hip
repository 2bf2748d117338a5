// Causal attention with a sliding window and sink tokens over contiguous keys and values: prompts, chunks of prompts,
// and single tokens (which take the split kernel of paged_attention.hip).
//
// The query at position p of a sequence of n keys sees j <= p, j < n, with j > p - window or j < sinks (window 0: all);
// a row that sees nothing, or whose position is no key's, gives zeros.
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
    }
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c)
        if (kWave * c + lane < a.dim) out[kWave * c + lane] = static_cast<T>(sum[c] / weight);
}

template <class T, int kDim, bool kWide>
__global__ void __launch_bounds__(kThreads) window_attention_kernel(AttentionArgs a) {
    using M = Mfma<T>;
    constexpr int kCols = kDim == 256 ? 1 : 2;  // tiles of 16 rows
    constexpr int kRows = 16 * kCols;
    constexpr int kTile = kDim * static_cast<int>(sizeof(T)) <= 256 ? 32 : 16;
    constexpr int kSubs = kTile / 16;
    constexpr int kFragments = M::template key_fragments<kDim>();
    constexpr int kChunks = M::template value_chunks<kDim>();
    constexpr int kBlocks = kDim / 16;
    constexpr int kWords = kBlocks * 4 + 2;
    using Value = typename M::template ValueChunk<kDim>;
    __shared__ float merge[2][kCols * kWords][kWave];

    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int n16 = lane & 15;
    const int g = lane >> 4;
    const int kv_head = blockIdx.y;
    const int64_t b = blockIdx.z;
    int64_t n = a.lengths ? a.lengths[b] : a.keys;
    n = n < 0 ? 0 : (n > a.keys ? a.keys : n);
    int64_t start = a.starts ? a.starts[b] : n - a.queries;
    start = start < -a.queries ? -a.queries : (start > a.keys ? a.keys : start);  // no row beyond these sees a key
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
    const int64_t all_rows = static_cast<int64_t>(a.queries) * a.group;

    // This lane's rows, one per column tile.
    RowRange mine[kCols];
    const T* query_row[kCols];
    int64_t out_row[kCols];
    bool real[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        const int64_t r = row0 + 16 * c + n16;
        const int64_t i = r / a.group, head = kv_head * static_cast<int64_t>(a.group) + r % a.group;
        real[c] = r < all_rows;
        const int64_t position = start + i;
        mine[c].position = real[c] && position >= 0 && position < n ? static_cast<int>(position) : -1;
        mine[c].low = a.window > 0 && mine[c].position >= a.window ? mine[c].position - a.window + 1 : 0;
        query_row[c] = static_cast<const T*>(a.query) + b * a.query_strides[0] + head * a.query_strides[1] +
                       i * a.query_strides[2];
        out_row[c] = (b * a.query_heads + head) * a.queries + i;
    }
    // The tile's first and last position that is a key's; all of its rows lie between.
    const int64_t last_row = row0 + kRows < all_rows ? row0 + kRows - 1 : all_rows - 1;
    int64_t first_position = start + row0 / a.group, last_position = start + last_row / a.group;
    if (first_position < 0) first_position = 0;
    if (last_position >= n) last_position = n - 1;
    const bool any = first_position <= last_position;

    const T* keys = static_cast<const T*>(a.key) + b * a.key_strides[0] + kv_head * a.key_strides[1];
    const T* values = static_cast<const T*>(a.value) + b * a.value_strides[0] + kv_head * a.value_strides[1];

    typename M::Fragment query[kCols][kFragments];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int f = 0; f < kFragments; ++f)
            query[c][f] = M::load_query(query_row[c], a.query_strides[3], M::kKeyStep * f + M::kPer * g, a.dim, real[c]);

    f32x4 out[kCols][kBlocks];
    float top[kCols], weight[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        top[c] = -INFINITY;
        weight[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) out[c][i] = f32x4{0, 0, 0, 0};
    }

    if (any) {
        const int first_p = static_cast<int>(first_position), last_p = static_cast<int>(last_position);
        const int seen = last_p + 1;
        const int low = a.window > 0 && first_p >= a.window ? first_p - a.window + 1 : 0;
        const int low_of_last = a.window > 0 && last_p >= a.window ? last_p - a.window + 1 : 0;
        const int sinks = a.sinks < low ? a.sinks : low;
        const int first_tile = low / kTile;
        const int of_sinks = (sinks + kTile - 1) / kTile;
        const int sink_tiles = of_sinks < first_tile ? of_sinks : first_tile;
        const int tiles = sink_tiles + (seen + kTile - 1) / kTile - first_tile;

        for (int t = wave; t < tiles; t += kWaves) {
            const int base_key = (t < sink_tiles ? t : first_tile + t - sink_tiles) * kTile;
            typename M::Fragment key[kSubs][kFragments];
            Value value[kSubs][4][kChunks];
#pragma unroll
            for (int s = 0; s < kSubs; ++s) {
                const int position = base_key + 16 * s + n16;
                const T* k = keys + position * a.key_strides[2];
#pragma unroll
                for (int f = 0; f < kFragments; ++f)
                    key[s][f] = M::template load_row<kWide>(k, M::kKeyStep * f + M::kPer * g, a.dim, position < seen);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int value_position = base_key + 16 * s + 4 * g + i;
                    const T* v = values + value_position * a.value_strides[2];
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
                        value[s][i][c] = M::template load_value<kDim, kWide>(v, c, n16, a.dim, value_position < seen);
                }
            }
            // Every key of the tile is seen by every row that sees any (the others are zeroed at the end).
            const bool inside = base_key >= low_of_last && base_key + kTile - 1 <= first_p;
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                f32x4 score[kSubs];
                float highest = -INFINITY;
#pragma unroll
                for (int s = 0; s < kSubs; ++s) {
                    score[s] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int f = 0; f < kFragments; ++f) M::multiply_key(key[s][f], query[c][f], score[s]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = base_key + 16 * s + 4 * g + i;
                        const bool visible = inside || (j <= mine[c].position && (j >= mine[c].low || j < a.sinks));
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
                        p[s][i] = fast_exp2((score[s][i] - reference) * kLog2e + M::kWeightShift);
                        weight[c] += p[s][i];
                    }
                M::template multiply_value<kDim, kSubs>(value, p, out[c]);
            }
        }
    }

#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        weight[c] += __shfl_xor(weight[c], 16, kWave);
        weight[c] += __shfl_xor(weight[c], 32, kWave);
    }
    // Join the four waves: 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
    for (int half = kWaves / 2; half >= 1; half /= 2) {
        __syncthreads();
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
        uint32_t rows = static_cast<uint32_t>((odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xffff);
        if (real[c] && !(rows >> n16 & 1)) {
            T* o = static_cast<T*>(a.out) + out_row[c] * a.dim;
            M::template each_dim<kDim>(g, a.dim, [&](int i, int r, int d) {
                o[d] = static_cast<T>(mine[c].position < 0 ? 0.0f : out[c][i][r] / weight[c]);
            });
        }
        while (rows) {
            const int which = __ffs(rows) - 1;
            rows &= rows - 1;
            const int64_t r = row0 + 16 * c + which;
            const int64_t i = r / a.group, head = kv_head * static_cast<int64_t>(a.group) + r % a.group;
            RowRange range;
            range.position = static_cast<int>(start + i);
            range.low = a.window > 0 && range.position >= a.window ? range.position - a.window + 1 : 0;
            exact_row<T>(a, static_cast<const T*>(a.query) + b * a.query_strides[0] + head * a.query_strides[1] +
                                i * a.query_strides[2],
                         keys, values, range, static_cast<T*>(a.out) + ((b * a.query_heads + head) * a.queries + i) * a.dim);
        }
    }
}

template <class T, int kDim>
hipError_t launch_window(const AttentionArgs& a, hipStream_t stream) {
    constexpr int kRows = kDim == 256 ? 16 : 32;
    const int64_t rows = static_cast<int64_t>(a.queries) * a.group;
    const dim3 grid(static_cast<uint32_t>((rows + kRows - 1) / kRows), a.kv_heads, a.batch);
    if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(window_attention_kernel<T, kDim, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(window_attention_kernel<T, kDim, false>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
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
