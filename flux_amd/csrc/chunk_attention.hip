// Attention of a step's packed tokens over a K/V cache in pages: chunks of prompts next to single tokens.
//
//   o = sum exp(s_j - m) v_j / sum exp(s_j - m),  s_j = scale <q, k_j>,  m = max s_j   over the keys j that the token sees:
//   j <= p and j < n, with j > p - window or j < sinks (window 0: all), on a page of the pool; nothing seen gives zeros.
//
// A tile is kRows rows of one request and KV head, a row being a token and one of the head's query heads, so that a
// group of heads shares each key and value row.  Tiles whose keys are many for the step's work are cut into parts of whole
// stages (kStage keys): every workgroup derives from the lists which part of which tile is its own, so that neither the
// host nor a launch before has to know the lengths, and a second launch joins the parts: o = sum o_c 2^(m_c - M) / sum l_c 2^(m_c - M).
#include "serving.h"
#include "serving_mfma.h"

#include "prefill_limb.h"

#include <type_traits>

namespace flux {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
// Stages that are worth a workgroup.  16-bit, with 1, 2, 3, 4 and 6 of them: 512 tokens over 512 keys 51, 42, 39, 36 and 36
// us.  float32's stages of 64 keys are four times as long for 32 rows: 16 tokens over 900 keys 21 us with 1, 24 with 4.
template <class T>
constexpr int least_stages() { return sizeof(T) == 2 ? 4 : 1; }
constexpr int kWholeStages = 4;  // up to which no tile is cut, which saves the join's launch

template <class T>
constexpr int rows_of_tile(int dim) { return sizeof(T) == 2 ? 32 * kWaves : (dim <= 128 ? 32 : 16); }
template <class T>
constexpr int stage_keys(int dim) { return sizeof(T) == 2 && dim == 64 ? 128 : 64; }
constexpr int padded_dim(int dim) { return dim <= 64 ? 64 : (dim <= 128 ? 128 : 256); }

// What the launches of one call agree on.
struct ChunkPlan {
    int rows;          // of a tile
    int64_t tiles;     // at most, of one KV head
    int target;        // parts of one KV head that a step's work is cut into
    bool whole;        // no tile is cut
    int least;         // stages of a part, but for a tile's shorter ones
    int64_t units;     // parts and whole tiles, at most, of one KV head
    int64_t slots;     // parts of cut tiles, at most, of one KV head
    int64_t splits;    // cut tiles, at most
    int slot_rows;     // rows of a slot
    int width;         // floats of a row: the dims in fours, the maximum, the sum
};

// In the workspace: the cut tiles' number, their descriptions, the parts' rows.
constexpr int kDescription = 8;  // ints
__host__ __device__ __forceinline__ int64_t parts_offset(const ChunkPlan& p) { return kDescription * (p.splits + 1); }
__device__ __forceinline__ float* part_row(const ChunkArgs& a, const ChunkPlan& p, int kv_head, int64_t slot, int row) {
    return a.workspace + parts_offset(p) + ((kv_head * p.slots + slot) * p.slot_rows + row) * p.width;
}

struct Sequence {
    int begin, count;  // tokens
    int64_t slot;      // row of the table; -1: none, and no keys
    int n;             // keys
    int start;         // position of the first token
};

__device__ __forceinline__ Sequence sequence_of(const ChunkArgs& a, int b) {
    Sequence s;
    const int64_t from = a.offsets[b], to = a.offsets[b + 1];
    const int64_t begin = from < 0 ? 0 : (from < a.tokens ? from : a.tokens);
    const int64_t end = to < begin ? begin : (to < a.tokens ? to : a.tokens);
    s.begin = static_cast<int>(begin);
    s.count = static_cast<int>(end - begin);
    s.slot = a.slots ? a.slots[b] : b;
    if (s.slot < 0 || s.slot >= a.slot_count) s.slot = -1;
    int64_t n = s.slot >= 0 ? a.lengths[s.slot] : 0;
    n = n < 0 ? 0 : (n < a.keys ? n : a.keys);
    const int64_t length = static_cast<int64_t>(static_cast<uint64_t>(to) - static_cast<uint64_t>(from));
    int64_t start = a.positions ? a.positions[b] : n - (length < 0 ? 0 : (length < (1 << 30) ? length : (1 << 30)));
    start = start < -s.count ? -s.count : (start < a.keys ? start : a.keys);  // no token beyond these has a key's position
    s.n = static_cast<int>(n);
    s.start = static_cast<int>(start);
    return s;
}

// The keys that any token of the positions first .. last sees, as stages: first the sinks', then the window's.
template <int kStage>
struct KeyStages {
    int seen, sink_stages, first_stage, count;
    __device__ __forceinline__ KeyStages(const ChunkArgs& a, int first, int last) {
        first = __builtin_amdgcn_readfirstlane(first);  // the same in all lanes
        last = __builtin_amdgcn_readfirstlane(last);
        const int low = a.window > 0 && first >= a.window ? first - a.window + 1 : 0;
        const int sinks = a.sinks < low ? a.sinks : low;
        const int of_sinks = (sinks + kStage - 1) / kStage;
        seen = last + 1;
        first_stage = low / kStage;
        sink_stages = of_sinks < first_stage ? of_sinks : first_stage;
        count = first > last ? 0 : sink_stages + (seen + kStage - 1) / kStage - first_stage;
    }
    __device__ __forceinline__ int base(int t) const { return (t < sink_stages ? t : first_stage + t - sink_stages) * kStage; }
};

// Positions of the rows [from, from + rows) that are a key's; 0 and -1 when there is none.
__device__ __forceinline__ void positions_of(const ChunkArgs& a, const Sequence& s, int from, int rows, int& first, int& last) {
    const int all = s.count * a.group, to = from + rows < all ? from + rows - 1 : all - 1;
    const int p = s.start + static_cast<int>(divide(from, a.group_of)), q = s.start + static_cast<int>(divide(to < 0 ? 0 : to, a.group_of));
    first = p < 0 ? 0 : p;
    last = q >= s.n ? s.n - 1 : q;
    if (from > to || first > last) first = 0, last = -1;
}

// Stages of a request's longest tile, at most.
template <int kRows, int kStage>
__device__ __forceinline__ int most_stages(const ChunkArgs& a, const Sequence& s) {
    const int last = s.start + s.count - 1 < s.n ? s.start + s.count - 1 : s.n - 1;
    if (last < 0 || s.count == 0) return 0;
    const int all = last / kStage + 1;
    if (a.window == 0) return all;
    const int windowed = (a.sinks + kStage - 1) / kStage + (a.window + static_cast<int>(divide(kRows, a.group_of)) + 1) / kStage + 2;
    return windowed < all ? windowed : all;
}

// The part that a workgroup works on.
struct Part {
    int request, tile, part, parts;
    int slot;   // of the part, when the tile is cut
    bool real;  // some request has it

    // Its stages, of a tile's `count`.
    __device__ __forceinline__ int from(int count) const {
        return __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(count) * part / parts));
    }
    __device__ __forceinline__ int to(int count) const {
        return __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<int64_t>(count) * (part + 1) / parts));
    }
};

struct PlanShared {
    int sums[3][kWaves];
    int chosen[4];
    Sequence sequence;
    int first_row, behind;  // of the requests' tokens
};

__device__ __forceinline__ int64_t sum_of_block(int64_t v, int64_t* sums) {
#pragma unroll
    for (int step = 1; step < 64; step *= 2) v += __shfl_xor(static_cast<long long>(v), step, kWave);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    return sums[0] + sums[1] + sums[2] + sums[3];
}

// Rows before the first request and behind the last are zeros.
template <class T>
__device__ __forceinline__ void clear_other_rows(const ChunkArgs& a, int before, int behind) {
    const int64_t others = before + a.tokens - behind;
    const int width = a.query_heads * a.dim;
    T* out = static_cast<T*>(a.out);
    for (int64_t i = blockIdx.x; i < others; i += gridDim.x) {
        T* row = out + (i < before ? i : behind + i - before) * width;
        for (int d = threadIdx.x; d < width; d += kThreads) row[d] = static_cast<T>(0.0f);
    }
}

// Parts lie in kStrips strips, from which the workgroups take one each in turn: what runs at the same time is then of all
// requests, chunks that matrix instructions bound next to single tokens that memory does.  A step of both in bfloat16 (2
// chunks of some 1000 tokens, 48 single tokens, 15000 keys and fewer) took 765, 762, 788 and 729 us with 1, 4, 16 and 64, and at a later step 729, 668 and 730 with 16, 64 and 256.
constexpr int kStrips = 64;

template <class T, int kRows, int kStage>
__device__ Part part_of(const ChunkArgs& a, const ChunkPlan& plan, int place, bool describes, Sequence& sequence) {
    __shared__ PlanShared s;
    __shared__ int64_t work_sums[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sequence mine;
    int tiles = 0, stages = 0;
    auto look = [&](int b) {
        tiles = stages = 0;
        if (b >= a.requests) return;
        mine = sequence_of(a, b);
        tiles = static_cast<int>((static_cast<int64_t>(mine.count) * a.group + kRows - 1) / kRows);
        stages = most_stages<kRows, kStage>(a, mine);
        if (b == 0) s.first_row = mine.begin;
        if (b == a.requests - 1) s.behind = mine.begin + mine.count;
    };
    int each = 1 << 30;
    if (!plan.whole) {
        int64_t work = 0;
        for (int base = 0; base < a.requests; base += kThreads) {
            look(base + threadIdx.x);
            work += sum_of_block(static_cast<int64_t>(tiles) * stages, work_sums);
        }
        const int64_t even = (work + plan.target - 1) / plan.target;
        each = even < plan.least ? plan.least : (even < each ? static_cast<int>(even) : each);
    }
    const bool one_round = a.requests <= kThreads;
    int all_units = 0, all_splits = 0, unit = -1;
    for (int round = one_round ? 1 : 0; round < 2; ++round) {  // the first one of two counts all parts
        int units_before = 0, slots_before = 0, splits_before = 0;
        for (int base = 0; base < a.requests; base += kThreads) {
            const int b = base + static_cast<int>(threadIdx.x);
            if (plan.whole || !one_round) look(b);
            const int parts = stages > each ? (stages + each - 1) / each : 1;
            const int units = tiles * parts;
            const int slots = parts > 1 ? units : 0, splits = parts > 1 ? tiles : 0;
            int units_to = wave_scan_int(units), slots_to = wave_scan_int(slots), splits_to = wave_scan_int(splits);
            __syncthreads();
            if (lane == 63) s.sums[0][wave] = units_to, s.sums[1][wave] = slots_to, s.sums[2][wave] = splits_to;
            __syncthreads();
            int units_here = 0, slots_here = 0, splits_here = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) units_to += s.sums[0][w], slots_to += s.sums[1][w], splits_to += s.sums[2][w];
                units_here += s.sums[0][w], slots_here += s.sums[1][w], splits_here += s.sums[2][w];
            }
            units_to += units_before, slots_to += slots_before, splits_to += splits_before;
            units_before += units_here, slots_before += slots_here, splits_before += splits_here;
            // Only offsets that decrease come this far; a round adds 2^30 and some at most, and no part from there on is anybody's.
            constexpr int kMost = 1 << 29;
            units_before = units_before < kMost ? units_before : kMost;
            slots_before = slots_before < kMost ? slots_before : kMost;
            splits_before = splits_before < kMost ? splits_before : kMost;
            if (one_round) all_units = units_before, all_splits = splits_before;
            if (round == 0) continue;
            const int strip = (all_units + kStrips - 1) / kStrips;
            unit = place / kStrips < strip ? place % kStrips * strip + place / kStrips : all_units;
            if (unit < units_to && unit >= units_to - units) {
                const int local = unit - (units_to - units);
                // Offsets that decrease could name more rows than there are: what has no room is left out.
                const int split = splits_to - splits + local / parts, slot = slots_to - slots + local;
                const bool room = parts == 1 || (slot >= 0 && slot - local % parts + parts <= plan.slots && split >= 0 && split < plan.splits);
                s.chosen[0] = b;
                s.chosen[1] = local;
                s.chosen[2] = parts;
                s.chosen[3] = room ? slot : -1;
                s.sequence = mine;
                if (describes && parts > 1 && room && local % parts == 0) {
                    int* d = reinterpret_cast<int*>(a.workspace) + kDescription * (1 + split);
                    const int row0 = (tiles - 1 - local / parts) * kRows, rows = mine.count * a.group - row0;
                    d[0] = mine.begin;
                    d[1] = row0;
                    d[2] = rows < kRows ? rows : kRows;
                    d[3] = slot;
                    d[4] = parts;
                }
            }
        }
        all_units = units_before, all_splits = splits_before;
    }
    if (describes && place == 0 && threadIdx.x == 0 && !plan.whole)
        *reinterpret_cast<int*>(a.workspace) = all_splits < plan.splits ? all_splits : static_cast<int>(plan.splits);
    __syncthreads();
    clear_other_rows<T>(a, s.first_row, s.behind);
    Part part{0, 0, 0, 1, 0, unit >= 0 && unit < all_units};
    if (!part.real) return part;
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // in all lanes
    part.request = same(s.chosen[0]);
    part.parts = same(s.chosen[2]);
    const int local = same(s.chosen[1]);
    part.part = local % part.parts;
    part.slot = same(s.chosen[3]);
    sequence = s.sequence;
    sequence.begin = same(sequence.begin);
    sequence.count = same(sequence.count);
    sequence.n = same(sequence.n);
    sequence.start = same(sequence.start);
    sequence.slot = static_cast<int64_t>(same(static_cast<int>(sequence.slot >> 32))) << 32 | static_cast<uint32_t>(same(static_cast<int>(sequence.slot)));
    // The longest tiles first.
    part.tile = static_cast<int>((static_cast<int64_t>(sequence.count) * a.group + kRows - 1) / kRows) - 1 - local / part.parts;
    part.real = part.slot >= 0 && part.tile >= 0;
    return part;
}

// This lane's row of the tile.
struct Row {
    int position;  // -1: sees nothing
    int low;       // first key of the window
    int sink_end;
};
__device__ __forceinline__ Row row_of(const ChunkArgs& a, const Sequence& s, int r) {
    Row row;
    const int position = s.start + static_cast<int>(divide(r, a.group_of));
    row.position = r < s.count * a.group && position >= 0 && position < s.n ? position : -1;
    row.low = a.window > 0 && row.position >= a.window ? row.position - a.window + 1 : 0;
    row.sink_end = a.sinks < row.low ? a.sinks : row.low;
    return row;
}

// Weights are 2^(s log2(e) - top) by one fused product, top = m log2(e) rounded: what that moves is common to all weights that
// refer to one maximum.  Where sums are rescaled or joined it is not, and below kFar it is then 2^-16 of a weight at most (with
// kShift in the sum).  From kFar on the difference s - m is taken first.
constexpr float kFar = 256.0f;
// Of a weight relative to one of another maximum.
__device__ __forceinline__ float exponent_of(float maximum, float other) {
    const float scaled = other * kLog2e;
    return fabsf(scaled) < kFar ? maximum * kLog2e - scaled : (maximum - other) * kLog2e;
}

// What a score <q, k> is multiplied by: before the maximum is looked for, and in the argument of 2^x.  16-bit types' leave all of the
// scale's size to the argument, where it is neither 0 nor next to what float32 holds (chunk_tile_kernel says why).
template <class T>
struct ScoreScale {
    float before, argument;
    __device__ __forceinline__ ScoreScale(float scale) : before(scale), argument(kLog2e) {
        const float size = fabsf(scale);
        if (sizeof(T) == 2 && size >= 1e-30f && size <= 1e30f) before = scale < 0.0f ? -1.0f : 1.0f, argument = size * kLog2e;
    }
};

// What the join needs to know of a part's row: the maximum that its weights refer to, in powers of two, its sum of weights, and the
// maximum of the scores, as ScoreScale leaves them before the argument: the difference of two of them does not overflow.
__device__ __forceinline__ void put_statistics(float* to, float top, float weight, float natural) {
    to[0] = top;
    to[1] = weight;
    to[2] = natural;
}

// A row whose sums are not finite, computed again over the keys it sees alone: a matrix instruction multiplies a masked
// key's zero weight with its value too, and a NaN or infinity there must not reach the row.  One wave.
template <class T, int kStage>
__device__ void exact_row(const ChunkArgs& a, const ChunkPlan& plan, const Sequence& s, const Part& part, int kv_head, int row0, int r,
                          const KeyStages<kStage>& stages, int from, int to, float shift) {
    const int lane = threadIdx.x & 63;
    const Row row = row_of(a, s, r);
    const int i = static_cast<int>(divide(r, a.group_of)), head = kv_head * a.group + r - i * a.group;
    const int64_t token = s.begin + i;
    const T* query = static_cast<const T*>(a.query) + token * a.query_strides[0] + head * a.query_strides[1];
    const T* keys = static_cast<const T*>(a.key) + kv_head * a.key_strides[1];
    const T* values = static_cast<const T*>(a.value) + kv_head * a.value_strides[1];
    const int32_t* table = a.table + (s.slot < 0 ? 0 : s.slot) * a.table_stride;
    const ScoreScale<T> scale(a.scale);
    float top = -INFINITY, weight = 0.0f, sum[kServingMaxDim / kWave];
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c) sum[c] = 0.0f;
    for (int at = from * kStage; at < to * kStage; at += kWave) {
        const int t = (at + lane) / kStage, position = stages.base(t) + (at + lane) % kStage;
        bool seen = t < to && row.position >= 0 && position <= row.position && (position >= row.low || position < row.sink_end);
        int64_t page = 0, in_page = 0;
        if (seen) {
            const uint32_t column = divide(position, a.page);
            page = table[column];
            in_page = position - column * a.page.divisor;
            seen = page >= 0 && page < a.pages;
        }
        float score = -INFINITY;
        if (seen) {
            const T* key = keys + page * a.key_strides[0] + in_page * a.key_strides[2];
            score = 0.0f;
            for (int d = 0; d < a.dim; ++d)
                score = fmaf(static_cast<float>(query[d * a.query_strides[2]]), static_cast<float>(key[d]), score);
            score *= scale.before;
        }
        const float now = fmaxf(top, wave_max(score));
        const float reference = now == -INFINITY ? 0.0f : now, scaled = reference * scale.argument;
        const bool near = fabsf(scaled) < kFar;
        auto difference = [&](float x) { return near ? fmaf(x, scale.argument, -scaled) : (x - reference) * scale.argument; };
        const float shrink = top == -INFINITY ? 0.0f : fast_exp2(difference(top));
        top = now;
        const float p = seen ? fast_exp2(difference(score) + shift) : 0.0f;
        weight = weight * shrink + wave_sum(p);
#pragma unroll
        for (int c = 0; c < kServingMaxDim / kWave; ++c) sum[c] *= shrink;
        const int64_t place = seen ? page * a.value_strides[0] + in_page * a.value_strides[2] : -1;
        for (int j = 0; j < kWave; ++j) {
            const int64_t of = __shfl(static_cast<long long>(place), j, kWave);
            const float pj = __shfl(p, j, kWave);
            if (of < 0) continue;
#pragma unroll
            for (int c = 0; c < kServingMaxDim / kWave; ++c)
                if (kWave * c + lane < a.dim) sum[c] = fmaf(pj, static_cast<float>(values[of + kWave * c + lane]), sum[c]);
        }
        // What is NaN stays NaN: a row whose sums all are is done.
        bool lost = true;
#pragma unroll
        for (int c = 0; c < kServingMaxDim / kWave; ++c) lost = lost && (kWave * c + lane >= a.dim || sum[c] != sum[c]);
        if (__all(weight != weight || lost)) break;
    }
    T* out = static_cast<T*>(a.out) + (token * a.query_heads + head) * a.dim;
    float* partial = part.parts > 1 ? part_row(a, plan, kv_head, part.slot, r - row0) : nullptr;
#pragma unroll
    for (int c = 0; c < kServingMaxDim / kWave; ++c) {
        const int d = kWave * c + lane;
        if (d >= a.dim) continue;
        if (partial) partial[d] = sum[c];
        else out[d] = static_cast<T>(weight == 0.0f ? 0.0f : sum[c] / weight);
    }
    if (partial && lane == 0) put_statistics(partial + plan.width - 4, top * scale.argument, weight, top);
}

// ---------------------------------------------------------------------------
// float32 with the float32 matrix instruction: everything in registers; a workgroup's four waves split the keys of the rows
// [row0, row0 + kRows) of a tile that starts at tile_row0, and join at the end.  `merge` holds merge_words<kDim>() words.
template <int kDim>
constexpr int merge_words() { return 2 * (rows_of_tile<float>(kDim) / 16) * (kDim / 4 + 2) * kWave; }

template <int kDim, Rows kRowsRead>
__device__ __forceinline__ void register_rows(const ChunkArgs& a, const ChunkPlan& plan, const Sequence& s, const Part& part, int kv_head,
                                              int tile_row0, int row0, const KeyStages<stage_keys<float>(kDim)>& stages, int from, int to,
                                              float* merge_memory) {
    using M = Mfma<float>;
    constexpr int kRows = rows_of_tile<float>(kDim);
    constexpr int kCols = kRows / 16;
    constexpr int kStage = stage_keys<float>(kDim);
    constexpr int kTile = 16;
    constexpr int kFragments = M::template key_fragments<kDim>();
    constexpr int kChunks = M::template value_chunks<kDim>();
    constexpr int kBlocks = kDim / 16;
    constexpr int kWords = kBlocks * 4 + 2;
    static_assert(kStage == kTile * kWaves, "a stage is one tile for each wave");
    auto merge = reinterpret_cast<float(*)[kCols * kWords][kWave]>(merge_memory);
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int n16 = lane & 15;
    const int g = lane >> 4;
    const int all_rows = s.count * a.group;
    const float* keys = static_cast<const float*>(a.key) + kv_head * a.key_strides[1];
    const float* values = static_cast<const float*>(a.value) + kv_head * a.value_strides[1];
    const int32_t* table = a.table + (s.slot < 0 ? 0 : s.slot) * a.table_stride;

    int first_p, last_p;
    positions_of(a, s, row0, kRows, first_p, last_p);
    Row mine[kCols];
    f32x4 query[kCols][kFragments];
    f32x4 out[kCols][kBlocks];
    float top[kCols], weight[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        const int r = row0 + 16 * c + n16;
        const bool real = r < all_rows;
        const int i = static_cast<int>(divide(real ? r : row0, a.group_of)), head = kv_head * a.group + (real ? r : row0) - i * a.group;
        mine[c] = row_of(a, s, r);
        const float* q = static_cast<const float*>(a.query) + static_cast<int64_t>(s.begin + i) * a.query_strides[0] + head * a.query_strides[1];
        load_query<float, kFragments, M::kKeyStep>(query[c], q, a.query_strides[2], a.query_wide, M::kPer * g, a.dim, real);
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) out[c][k] = f32x4{0, 0, 0, 0};
        top[c] = -INFINITY;
        weight[c] = 0.0f;
    }
    const int low_of_last = a.window > 0 && last_p >= a.window ? last_p - a.window + 1 : 0;

    // This wave's tile of stage t.  Rows behind the last key repeat it; keys on no page are the pool's first row.
    auto position_of = [&](int t) {
        const int position = stages.base(t) + kTile * wave + n16;
        return position < stages.seen ? position : stages.seen - 1;
    };
    auto look_up = [&](int t) { return t < to ? table[divide(position_of(t), a.page)] : -1; };
    auto work = [&](int t, int page) {
        const int base = stages.base(t) + kTile * wave;
        if (base >= stages.seen) return;
        const bool held = page >= 0 && page < a.pages;
        const bool whole = __all(held);
        const int position = position_of(t);
        const int in_page = held ? position - static_cast<int>(divide(position, a.page) * a.page.divisor) : 0;
        const int64_t of_page = held ? page : 0;
        f32x4 key[kFragments], value[4][kChunks];
        const float* k = keys + of_page * a.key_strides[0] + in_page * a.key_strides[2];
#pragma unroll
        for (int f = 0; f < kFragments; ++f) key[f] = M::template load_row<kRowsRead>(k, M::kKeyStep * f + M::kPer * g, a.dim);
        const int64_t value_at = of_page * a.value_strides[0] + in_page * a.value_strides[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* v = values + __shfl(static_cast<long long>(value_at), 4 * g + i, kWave);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) value[i][c] = M::template load_value<kDim, kRowsRead>(v, c, n16, a.dim);
        }
        uint32_t missing = 0;
        if (!whole) {
            missing = static_cast<uint32_t>(__ballot(!held));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (missing >> (4 * g + i) & 1) {
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) value[i][c] = f32x4{0, 0, 0, 0};
                }
        }
        // Every key of the tile is seen by every row that sees any (the others are zeroed at the end).
        const bool inside = whole && base >= low_of_last && base + kTile - 1 <= first_p;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            f32x4 score = {0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < kFragments; ++f) M::multiply_key(key[f], query[c][f], score);
            float highest = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = base + 4 * g + i;
                // Without branches: low <= key <= position as one unsigned comparison, or a sink.
                const bool visible = inside | (((static_cast<uint32_t>(j - mine[c].low) <=
                                                 static_cast<uint32_t>(mine[c].position - mine[c].low)) | (j < mine[c].sink_end)) &
                                               !(missing >> (4 * g + i) & 1));
                score[i] = visible ? score[i] * a.scale : -INFINITY;
                highest = fmaxf(highest, score[i]);
            }
            highest = fmaxf(highest, __shfl_xor(highest, 16, kWave));
            highest = fmaxf(highest, __shfl_xor(highest, 32, kWave));
            if (__any(highest > top[c])) {
                const float now = fmaxf(top[c], highest);
                const float shrink = top[c] == -INFINITY ? 0.0f : fast_exp2(exponent_of(top[c], now));
                top[c] = now;
                weight[c] *= shrink;
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) out[c][i] *= shrink;
            }
            const float reference = top[c] == -INFINITY ? 0.0f : top[c];
            const float scaled = reference * kLog2e;
            const bool near = fabsf(scaled) < kFar;
            float p[1][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[0][i] = fast_exp2(near ? fmaf(score[i], kLog2e, -scaled) : (score[i] - reference) * kLog2e);
                weight[c] += p[0][i];
            }
            f32x4 turned[1][4][kChunks];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k2 = 0; k2 < kChunks; ++k2) turned[0][i][k2] = value[i][k2];
            M::template multiply_value<kDim, 1>(turned, p, out[c]);
        }
    };
    int page = look_up(from);
    for (int t = from; t < to; ++t) {
        const int next = look_up(t + 1);
        work(t, page);
        page = next;
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
                float(*into)[kWave] = merge[wave - half] + c * kWords;
#pragma unroll
                for (int i = 0; i < kBlocks * 4; ++i) into[i][lane] = out[c][i / 4][i % 4];
                into[kBlocks * 4][lane] = top[c];
                into[kBlocks * 4 + 1][lane] = weight[c];
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                const float(*other)[kWave] = merge[wave] + c * kWords;
                const float other_top = other[kBlocks * 4][lane];
                const float now = fmaxf(top[c], other_top);
                const float mine_scale = top[c] == -INFINITY ? 0.0f : fast_exp2(exponent_of(top[c], now));
                const float other_scale = other_top == -INFINITY ? 0.0f : fast_exp2(exponent_of(other_top, now));
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
        const int r = row0 + 16 * c + n16;
        if (r < all_rows && !(again >> n16 & 1)) {
            const int i = static_cast<int>(divide(r, a.group_of)), head = kv_head * a.group + r - i * a.group;
            if (part.parts == 1) {
                float* o = static_cast<float*>(a.out) + (static_cast<int64_t>(s.begin + i) * a.query_heads + head) * a.dim;
                M::template each_dim<kDim>(g, a.dim, [&](int k, int j, int d) {
                    o[d] = mine[c].position < 0 || weight[c] == 0.0f ? 0.0f : out[c][k][j] / weight[c];
                });
            } else {
                float* o = part_row(a, plan, kv_head, part.slot, r - tile_row0);
                M::template each_dim<kDim>(g, a.dim, [&](int k, int j, int d) { o[d] = mine[c].position < 0 ? 0.0f : out[c][k][j]; });
                const float highest = mine[c].position < 0 ? -INFINITY : top[c];
                if (g == 0) put_statistics(o + plan.width - 4, highest * kLog2e, mine[c].position < 0 ? 0.0f : weight[c], highest);
            }
        }
        while (again) {
            const int which = __ffs(again) - 1;
            again &= again - 1;
            exact_row<float, kStage>(a, plan, s, part, kv_head, tile_row0, row0 + 16 * c + which, stages, from, to, 0.0f);
        }
    }
}

// Other float32 work: bound by latency where it is little (16 tokens over 900 keys: 13 us, of which the plan, the table and the first
// keys are dependent reads), by the float32 matrix instruction where it is much.
template <int kDim, Rows kRowsRead>
__global__ void __launch_bounds__(kThreads, kDim <= 64 ? 3 : (kDim <= 128 ? 2 : 1)) chunk_register_kernel(ChunkArgs a, ChunkPlan plan) {
    constexpr int kRows = rows_of_tile<float>(kDim);
    constexpr int kStage = stage_keys<float>(kDim);
    __shared__ float merge[merge_words<kDim>()];
    const int kv_head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    Sequence s;
    const Part part = part_of<float, kRows, kStage>(a, plan, unit, kv_head == 0, s);
    if (!part.real) return;
    const int row0 = part.tile * kRows;
    int first_p, last_p;
    positions_of(a, s, row0, kRows, first_p, last_p);
    const KeyStages<kStage> stages(a, first_p, last_p);
    register_rows<kDim, kRowsRead>(a, plan, s, part, kv_head, row0, row0, stages, part.from(stages.count), part.to(stages.count), merge);
}

// ---------------------------------------------------------------------------
// 16-bit types: keys and values are staged in LDS, row by row as they are, for the workgroup's four waves of 32 rows each, and
// copied there past the registers while the stage before is worked on.  S^T = K Q^T on 32 x 32 tiles leaves lane (n, h) with the
// keys 8 (r / 4) + 4 h + r % 4 of row n, which rounded in pairs are the right operand of O^T = V^T P; V's left operand, one dim
// of four keys, comes by reads that transpose 4 x 16 blocks.  A row's 16-byte pieces lie permuted, so that these reads meet
// different banks: piece c of row r is at c ^ swizzle(r).  Where a stage's rows lie is looked up two stages ahead.  Weights are
// rounded once to the values' type for the product and summed unrounded (half a step of a mean's largest value, as the result's own
// rounding; two terms would double that product); the running maximum moves only when a tile exceeds it by 2^kLazy.
//
// Bound by matrix and vector instructions that overlap in part: 4096 tokens behind 28672 (32 / 8 heads of 128, bfloat16) take
// 2230 us, 930 TFLOP/s; the matrix units are busy for 40% of a SIMD's cycles, the vector ones for 46%, and no bank conflicts.  Keys
// and values through registers took 3780 us against 2500; a priority for one of a SIMD's two waves changes nothing, and a loop unrolled over
// the stages' parity spills.  Single tokens fill few of the 128 rows, and HBM bounds them: 32 of them over 4000 keys 95 us,
// 3.3 TB/s.
template <int kDim>
__device__ __forceinline__ int swizzle(int r) {
    if constexpr (kDim == 64) return (r >> 1 & 1) << 2 | (r >> 2 & 3);  // rows of half the banks
    else return (r & 3) << 2 | (r >> 2 & 3);
}

__device__ __forceinline__ uint32_t lds_address(const char* at) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(at)));
}
// Sixteen bytes of every lane to the LDS at `to` + 16 lane.  In assembly, because the compiler waits for a copy before the next
// read of any LDS; the kernel waits itself, before the barrier that hands a stage over.  The address register needs one state
// between its write and its use.
__device__ __forceinline__ void copy_to_lds(const void* from, uint32_t to) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(to) : "memory");
}

__device__ __forceinline__ u32x2 read_transposed(const char* at) {
    typedef __attribute__((address_space(3))) s16x4 Block;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Block*)(at)));
}

// out *= shrink where `moves`.  In assembly, with its branch inside: behind a branch of the compiler's the sums' registers are
// moved in the other arm, 64 moves a tile.  The compiler does not count what an assembly block needs, so it waits itself: a matrix
// instruction's result is there 11 states later (what the compiler leaves before its own reads of one), here 32; the next one may
// read a product after 2, here 8.
//
// Not for more than 128 dims, whose sums, scores and keys leave it no registers: with it the kernel keeps 280 to 290 bytes a lane in
// memory, without it 170 to 180.  One such build gave wrong float16 results: the compiler had saved registers (a row's number, token
// and head) where a branch had lanes off, so that rows were written to other places.  The sums were right.
// tests/test_assembly_cpu.py looks for such saves in every kernel.
template <int kBlocks>
__device__ __forceinline__ void scale_if(bool moves, float shrink, f32x16 (&out)[kBlocks]) {
    if constexpr (kBlocks > 4) {
        if (moves) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) out[b] *= shrink;
        }
        return;
    }
    const int some = __builtin_amdgcn_readfirstlane(moves);
#pragma unroll
    for (int b = 0; b + 1 < kBlocks; b += 2) {
        float o[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = out[b + j / 16][j % 16];
        asm volatile(
            "s_cmp_eq_u32 %32, 0\n\ts_cbranch_scc1 .Lkept%=\n\ts_nop 15\n\ts_nop 15\n\t"
            "v_mul_f32 %0, %33, %0\n\tv_mul_f32 %1, %33, %1\n\tv_mul_f32 %2, %33, %2\n\tv_mul_f32 %3, %33, %3\n\t"
            "v_mul_f32 %4, %33, %4\n\tv_mul_f32 %5, %33, %5\n\tv_mul_f32 %6, %33, %6\n\tv_mul_f32 %7, %33, %7\n\t"
            "v_mul_f32 %8, %33, %8\n\tv_mul_f32 %9, %33, %9\n\tv_mul_f32 %10, %33, %10\n\tv_mul_f32 %11, %33, %11\n\t"
            "v_mul_f32 %12, %33, %12\n\tv_mul_f32 %13, %33, %13\n\tv_mul_f32 %14, %33, %14\n\tv_mul_f32 %15, %33, %15\n\t"
            "v_mul_f32 %16, %33, %16\n\tv_mul_f32 %17, %33, %17\n\tv_mul_f32 %18, %33, %18\n\tv_mul_f32 %19, %33, %19\n\t"
            "v_mul_f32 %20, %33, %20\n\tv_mul_f32 %21, %33, %21\n\tv_mul_f32 %22, %33, %22\n\tv_mul_f32 %23, %33, %23\n\t"
            "v_mul_f32 %24, %33, %24\n\tv_mul_f32 %25, %33, %25\n\tv_mul_f32 %26, %33, %26\n\tv_mul_f32 %27, %33, %27\n\t"
            "v_mul_f32 %28, %33, %28\n\tv_mul_f32 %29, %33, %29\n\tv_mul_f32 %30, %33, %30\n\tv_mul_f32 %31, %33, %31\n\t"
            "s_nop 7\n.Lkept%=:"
            : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]), "+v"(o[4]), "+v"(o[5]), "+v"(o[6]), "+v"(o[7]),
              "+v"(o[8]), "+v"(o[9]), "+v"(o[10]), "+v"(o[11]), "+v"(o[12]), "+v"(o[13]), "+v"(o[14]), "+v"(o[15]),
              "+v"(o[16]), "+v"(o[17]), "+v"(o[18]), "+v"(o[19]), "+v"(o[20]), "+v"(o[21]), "+v"(o[22]), "+v"(o[23]),
              "+v"(o[24]), "+v"(o[25]), "+v"(o[26]), "+v"(o[27]), "+v"(o[28]), "+v"(o[29]), "+v"(o[30]), "+v"(o[31])
            : "s"(some), "v"(shrink)
            : "scc");
#pragma unroll
        for (int j = 0; j < 32; ++j) out[b + j / 16][j % 16] = o[j];
    }
    if constexpr (kBlocks % 2) {
        float o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = out[kBlocks - 1][j];
        asm volatile(
            "s_cmp_eq_u32 %16, 0\n\ts_cbranch_scc1 .Lkept%=\n\ts_nop 15\n\ts_nop 15\n\t"
            "v_mul_f32 %0, %17, %0\n\tv_mul_f32 %1, %17, %1\n\tv_mul_f32 %2, %17, %2\n\tv_mul_f32 %3, %17, %3\n\t"
            "v_mul_f32 %4, %17, %4\n\tv_mul_f32 %5, %17, %5\n\tv_mul_f32 %6, %17, %6\n\tv_mul_f32 %7, %17, %7\n\t"
            "v_mul_f32 %8, %17, %8\n\tv_mul_f32 %9, %17, %9\n\tv_mul_f32 %10, %17, %10\n\tv_mul_f32 %11, %17, %11\n\t"
            "v_mul_f32 %12, %17, %12\n\tv_mul_f32 %13, %17, %13\n\tv_mul_f32 %14, %17, %14\n\tv_mul_f32 %15, %17, %15\n\t"
            "s_nop 7\n.Lkept%=:"
            : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]), "+v"(o[4]), "+v"(o[5]), "+v"(o[6]), "+v"(o[7]),
              "+v"(o[8]), "+v"(o[9]), "+v"(o[10]), "+v"(o[11]), "+v"(o[12]), "+v"(o[13]), "+v"(o[14]), "+v"(o[15])
            : "s"(some), "v"(shrink)
            : "scc");
#pragma unroll
        for (int j = 0; j < 16; ++j) out[kBlocks - 1][j] = o[j];
    }
}

// kUsed: dims that are worked on, of the kDim that a row in LDS has.
template <class T, int kDim, int kUsed, bool kWide>
__global__ void __launch_bounds__(kThreads, kDim <= 128 ? 2 : 1) chunk_tile_kernel(ChunkArgs a, ChunkPlan plan) {
    using W = Wide<T>;
    constexpr int kStage = stage_keys<T>(kDim);
    constexpr int kSubs = kStage / 32;
    constexpr int kSteps = kUsed / 16;            // of a score
    constexpr int kBlocks = kUsed / 32;           // of the result
    constexpr int kRows = rows_of_tile<T>(kDim);
    constexpr int kRowBytes = kDim * 2;
    constexpr int kSide = kStage * kRowBytes;     // keys or values of a stage
    constexpr int kPieces = kDim / 8;             // of a row, 16 bytes each
    constexpr int kCopyRows = 64 / kPieces;       // of one copy of a wave
    constexpr int kCopies = kStage / kCopyRows / kWaves;  // of a wave, for each side
    extern __shared__ char stages_memory[];
    __shared__ int64_t places[2][2][kStage];   // bytes from the head's first, by stage parity
    __shared__ uint32_t missing[2][kSubs];     // keys of a stage that are on no page

    const int kv_head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    Sequence s;
    const Part part = part_of<T, kRows, kStage>(a, plan, unit, kv_head == 0, s);
    if (!part.real) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31;
    const int half = lane >> 5;
    const int row0 = part.tile * kRows, all_rows = s.count * a.group, wave_row = row0 + wave * 32;
    int block_first, block_last, wave_first, wave_last;
    positions_of(a, s, row0, kRows, block_first, block_last);
    positions_of(a, s, wave_row, 32, wave_first, wave_last);
    wave_first = __builtin_amdgcn_readfirstlane(wave_first);
    wave_last = __builtin_amdgcn_readfirstlane(wave_last);
    const KeyStages<kStage> stages(a, block_first, block_last);
    const int from = part.from(stages.count), to = part.to(stages.count);

    const char* keys = static_cast<const char*>(a.key) + 2 * kv_head * a.key_strides[1];
    const char* values = static_cast<const char*>(a.value) + 2 * kv_head * a.value_strides[1];
    const int32_t* table = a.table + (s.slot < 0 ? 0 : s.slot) * a.table_stride;

    const int r = wave_row + n32;  // this lane's row
    const bool real = r < all_rows;
    const int index = static_cast<int>(divide(real ? r : row0, a.group_of)), head = kv_head * a.group + (real ? r : row0) - index * a.group;
    const Row mine = row_of(a, s, r);
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

    if (from < to) {
        u32x4 query[kSteps];
        load_query<T, kSteps, 16>(query, static_cast<const T*>(a.query) + static_cast<int64_t>(s.begin + index) * a.query_strides[0] +
                                             head * a.query_strides[1],
                                  a.query_strides[2], a.query_wide, 8 * half, a.dim, real);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) query[k] ^= sign;
        auto low_of = [&](int p) { return a.window > 0 && p >= a.window ? p - a.window + 1 : 0; };

        // Threads below kStage look up one key each.  Rows behind the last key repeat it; keys on no page are the pool's first.
        auto position_of = [&](int t) {
            const int position = stages.base(t) + static_cast<int>(threadIdx.x);
            return position < stages.seen ? position : stages.seen - 1;
        };
        auto look_up = [&](int t) {
            return t < to && static_cast<int>(threadIdx.x) < kStage ? table[divide(position_of(t), a.page)] : 0;
        };
        auto put_places = [&](int t, int page) {
            if (t >= to || static_cast<int>(threadIdx.x) >= kStage) return;
            const int position = position_of(t);
            const bool held = page >= 0 && page < a.pages;
            const int64_t of_page = held ? page : 0;
            const int in_page = held ? position - static_cast<int>(divide(position, a.page) * a.page.divisor) : 0;
            places[t & 1][0][threadIdx.x] = 2 * (of_page * a.key_strides[0] + in_page * a.key_strides[2]);
            places[t & 1][1][threadIdx.x] = 2 * (of_page * a.value_strides[0] + in_page * a.value_strides[2]);
            const uint64_t gone = __ballot(!held);
            if (lane == 0) missing[t & 1][threadIdx.x / 32] = static_cast<uint32_t>(gone);
            if (lane == 32) missing[t & 1][threadIdx.x / 32] = static_cast<uint32_t>(gone >> 32);
        };
        // Copy j of a wave: rows kCopyRows (kWaves j + wave) and on, of which this lane brings one piece.  Dims behind the head's
        // repeat its first ones, which meet zeros of the query or results that are not stored.
        const uint32_t memory = lds_address(stages_memory);
        auto copy = [&](int t) {
            const int stage = (t & 1) * 2 * kSide;
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                const int row = kCopyRows * (kWaves * j + wave) + lane / kPieces;
                const int piece = (lane % kPieces) ^ swizzle<kDim>(row), d = 8 * piece < a.dim ? 8 * piece : 0;
                const int to_key = stage + kCopyRows * (kWaves * j + wave) * kRowBytes;
                const char* key = keys + places[t & 1][0][row];
                const char* value = values + places[t & 1][1][row];
                if constexpr (kWide) {
                    copy_to_lds(key + 2 * d, memory + to_key);
                    copy_to_lds(value + 2 * d, memory + to_key + kSide);
                } else {
                    *reinterpret_cast<u32x4*>(stages_memory + to_key + 16 * lane) = Mfma<T>::load_strided(reinterpret_cast<const T*>(key), 1, 8 * piece, a.dim);
                    *reinterpret_cast<u32x4*>(stages_memory + to_key + kSide + 16 * lane) =
                        Mfma<T>::load_strided(reinterpret_cast<const T*>(value), 1, 8 * piece, a.dim);
                }
            }
        };
        int key_at[kSteps], value_at[kBlocks][2];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) key_at[k] = n32 * kRowBytes + (((2 * k + half) ^ swizzle<kDim>(n32)) * 16);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * e + 4 * half + (lane & 15) / 4, piece = 4 * b + 2 * (lane >> 4 & 1) + (lane & 3) / 2;
                value_at[b][e] = kSide + row * kRowBytes + (piece ^ swizzle<kDim>(row)) * 16 + 8 * (lane & 1);
            }

        const int wave_low = low_of(wave_first), low_of_last = low_of(wave_last);
        // 32 keys, `first` on, of the stage at `at`.
        auto work = [&](const char* at, int first, uint32_t gone, auto masked) {
            u32x4 key[kSteps];
#pragma unroll
            for (int k = 0; k < kSteps; ++k) key[k] = *reinterpret_cast<const u32x4*>(at + key_at[k]);
            __builtin_amdgcn_sched_barrier(0);  // all reads first
            f32x16 score;
#pragma unroll
            for (int j = 0; j < 16; ++j) score[j] = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) score = W::multiply(key[k], query[k], score);
            if (!ordinary) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float product = score[j];
                    asm volatile("" : "+v"(product));  // a branch stays: else all scores pay for the product
                    score[j] = product * size;
                }
            }
            if constexpr (decltype(masked)::value) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    // Without branches: low <= key <= position as one unsigned comparison, or a sink.
                    const int in = 8 * (j / 4) + 4 * half + j % 4, of = first + in;
                    const bool visible = ((static_cast<uint32_t>(of - mine.low) <= static_cast<uint32_t>(mine.position - mine.low)) |
                                          (of < mine.sink_end)) & !(gone >> in & 1);
                    score[j] = visible ? score[j] : -INFINITY;
                }
            }
            float highest = fmaxf(score[0], score[1]);
#pragma unroll
            for (int j = 2; j < 16; j += 2) highest = fmaxf(fmaxf(highest, score[j]), score[j + 1]);
            highest = half_max(highest);
            // By 2^(old maximum - new one), where a row's moved: in few tiles behind the first.
            const bool moves = __any((highest - top) * factor > W::kLazy);  // NaN where both are -inf
            float shrink = 1.0f;
            if (moves) {
                const float now = fmaxf(top, highest);
                const float scaled = now * factor;
                shrink = top == -INFINITY ? 0.0f : fast_exp2(fabsf(scaled) < kFar ? top * factor - scaled : (top - now) * factor);
                top = now;
                weight *= shrink;
            }
            scale_if<kBlocks>(moves, shrink, out);
            u32x4 value[kBlocks][2];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x2 low = read_transposed(at + value_at[b][0] + 16 * k * kRowBytes);
                    const u32x2 high = read_transposed(at + value_at[b][1] + 16 * k * kRowBytes);
                    value[b][k] = u32x4{low[0], low[1], high[0], high[1]};
                }
            const float scaled = top == -INFINITY ? 0.0f : top * factor;
            const bool far = !(fabsf(scaled) < kFar);
            const float reference = W::kShift - (far ? 0.0f : scaled);
            if (__any(far)) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float difference = score[j];
                    asm volatile("" : "+v"(difference));
                    score[j] = far ? difference - top : difference;
                }
            }
            u32x4 p[2];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float p0 = fast_exp2(fmaf(score[j], factor, reference));
                const float p1 = fast_exp2(fmaf(score[j + 1], factor, reference));
                weight += p0 + p1;
                p[j / 8][j % 8 / 2] = W::round(p0, p1);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = W::multiply(value[b][k], p[k], out[b]);
        };

        put_places(from, look_up(from));
        put_places(from + 1, look_up(from + 1));
        __syncthreads();
        uint32_t gone_next[kSubs];
#pragma unroll
        for (int i = 0; i < kSubs; ++i) gone_next[i] = missing[from & 1][i];
        copy(from);
        for (int t = from; t < to; ++t) {
            __builtin_amdgcn_s_waitcnt(0);  // this wave's copies have landed
            __syncthreads();
            char* stage = stages_memory + (t & 1) * 2 * kSide;
            const int base = stages.base(t);
            uint32_t gone[kSubs], any_gone = 0;  // read a stage ahead: that of this one may be another's already
#pragma unroll
            for (int i = 0; i < kSubs; ++i) {
                gone[i] = gone_next[i];
                any_gone |= gone[i];
                gone_next[i] = missing[(t + 1) & 1][i];  // of no stage behind the last
            }
            const int page = look_up(t + 2);
            if (t + 1 < to) copy(t + 1);
            any_gone = __builtin_amdgcn_readfirstlane(any_gone);
            if (any_gone) {  // a weight of zero does not undo a NaN
#pragma unroll
                for (int i = 0; i < kSubs; ++i)
                    for (int piece = threadIdx.x; piece < 32 * kPieces; piece += kThreads)
                        if (gone[i] >> (piece / kPieces) & 1)
                            *reinterpret_cast<u32x4*>(stage + kSide + 32 * i * kRowBytes + 16 * piece) = u32x4{0, 0, 0, 0};
                __syncthreads();
            }
            const int last = base + kStage - 1;
            const bool seen = base <= wave_last && (last >= wave_low || base < a.sinks);
            if (seen && !any_gone && base >= low_of_last && last <= wave_first) {  // all of it, by all rows
#pragma unroll
                for (int i = 0; i < kSubs; ++i) work(stage + 32 * i * kRowBytes, base + 32 * i, 0, std::false_type{});
            } else if (seen) {
#pragma unroll 1
                for (int i = 0; i < kSubs; ++i) {
                    const int first = base + 32 * i;
                    if (first > wave_last || (first + 31 < wave_low && first >= a.sinks)) continue;
                    work(stage + 32 * i * kRowBytes, first, gone[i], std::true_type{});
                }
            }
            put_places(t + 2, page);
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
        if (part.parts == 1) {
            T* o = static_cast<T*>(a.out) + (static_cast<int64_t>(s.begin + index) * a.query_heads + head) * a.dim;
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
        } else {
            float* o = part_row(a, plan, kv_head, part.slot, r - row0);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const int d = 32 * i + 2 * j + 4 * half;
                    if (d < a.dim)
                        *reinterpret_cast<f32x4*>(o + d) = mine.position < 0 ? f32x4{0, 0, 0, 0} : f32x4{out[i][j], out[i][j + 1], out[i][j + 2], out[i][j + 3]};
                }
            const float highest = mine.position < 0 ? -INFINITY : top;
            if (half == 0)
                put_statistics(o + plan.width - 4, highest * factor, mine.position < 0 ? 0.0f : weight, highest);
        }
    }
    while (again) {
        const int which = __ffs(again) - 1;
        again &= again - 1;
        exact_row<T, kStage>(a, plan, s, part, kv_head, row0, wave_row + which, stages, from, to, W::kShift);
    }
}

// ---------------------------------------------------------------------------
// float32 chunks of heads up to 64: products of three bf16 limbs, six of the nine (prefill_limb.h states what they carry), whose rate
// is 16 / 6 times that of the float32 instruction, closer to 64 bits than that one's sums.  A workgroup's four waves take 32 rows each.
// The threads fetch a stage's rows while the stage before is worked on, and split them into limbs on the way to LDS, where
// each limb's rows lie as a 16-bit type's do above.  Scores are in powers of two: the query is multiplied by scale * log2(e).
// Where limbs do not do (an infinity, a NaN, magnitudes beyond kLimbMostScore or kLimbMostValue, scores of kLimbFar on, sums so small that
// bits are lacking) the tile is computed again by register_rows.
//
// Bound as the 16-bit kernel is: 4 chunks of prompts (up to 1024 tokens over 7168 keys, 9 / 3 heads of 64) take 216 us,
// 135 TFLOP/s of float32 products; the matrix units are busy for 37% of the cycles, the vector ones for 41%, most of them splitting
// rows and weights.  Eight waves 333 us against 287 at that step; sums of their own for the small products 287 against 247 (they spill).
constexpr float kLimbMostScore = 0x1p60f;  // of a scaled query and of a key: no sum of 64 products overflows
constexpr float kLimbMostValue = 0x1p19f;
constexpr float kLimbFar = 1024.0f;  // of a score, whose rounding then moves a weight by 2^-14 of itself at most
constexpr float kLimbLeastSum = 0x1p-82f;  // of a row, per 64 keys: bits below 2^-134 of each factor are under 2^-26 of it

__device__ __forceinline__ bool beyond(const f32x4& a, const f32x4& b, float most) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = __builtin_elementwise_maximum(m, __builtin_elementwise_maximum(fabsf(a[j]), fabsf(b[j])));  // keeps NaN
    return !(m <= most);
}

template <bool kWide>
__global__ void __launch_bounds__(kThreads, 2) chunk_limb_kernel(ChunkArgs a, ChunkPlan plan) {
    constexpr int kDim = 64, kStage = 64, kRows = 32 * kWaves;
    constexpr int kSteps = kDim / 16, kBlocks = kDim / 32, kSubs = kStage / 32, kPieces = kDim / 8;
    constexpr int kRowBytes = kDim * 2, kPlane = kStage * kRowBytes, kSide = kLimbs * kPlane;
    constexpr int kPerThread = kStage * kPieces / kThreads;  // pieces of eight dims, for each side
    constexpr float kLazy = 4.0f;
    __shared__ __attribute__((aligned(16))) char planes[2 * kSide];
    __shared__ int64_t places[2][2][kStage];  // elements from the head's first, by stage parity
    __shared__ uint32_t missing[2][kSubs];
    static_assert(sizeof(float) * merge_words<kDim>() <= sizeof(planes), "register_rows uses the planes");

    const int kv_head = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    Sequence s;
    const Part part = part_of<float, kRows, kStage>(a, plan, unit, kv_head == 0, s);
    if (!part.real) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31;
    const int half = lane >> 5;
    const int row0 = part.tile * kRows, all_rows = s.count * a.group, wave_row = row0 + wave * 32;
    int block_first, block_last, wave_first, wave_last;
    positions_of(a, s, row0, kRows, block_first, block_last);
    positions_of(a, s, wave_row, 32, wave_first, wave_last);
    wave_first = __builtin_amdgcn_readfirstlane(wave_first);
    wave_last = __builtin_amdgcn_readfirstlane(wave_last);
    const KeyStages<kStage> stages(a, block_first, block_last);
    const int from = part.from(stages.count), to = part.to(stages.count);

    const float* keys = static_cast<const float*>(a.key) + kv_head * a.key_strides[1];
    const float* values = static_cast<const float*>(a.value) + kv_head * a.value_strides[1];
    const int32_t* table = a.table + (s.slot < 0 ? 0 : s.slot) * a.table_stride;
    const int r = wave_row + n32;  // this lane's row
    const bool real = r < all_rows;
    const int index = static_cast<int>(divide(real ? r : row0, a.group_of)), head = kv_head * a.group + (real ? r : row0) - index * a.group;
    const Row mine = row_of(a, s, r);
    f32x16 out[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) out[i][j] = 0.0f;
    float top = -INFINITY, weight = 0.0f;
    bool unsure = false;

    if (from < to) {
        u32x4 query[kSteps][kLimbs];
        {
            const float* q = static_cast<const float*>(a.query) + static_cast<int64_t>(s.begin + index) * a.query_strides[0] + head * a.query_strides[1];
            const float factor = a.scale * kLog2e;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                f32x4 four[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int d = 16 * k + 8 * half + 4 * j;
                    if (a.query_wide) four[j] = *reinterpret_cast<const f32x4*>(q + (d < a.dim ? d : 0));
                    else four[j] = Mfma<float>::load_strided(q, a.query_strides[2], d, a.dim);
                    four[j] = Mfma<float>::zero_behind(four[j], d, real ? a.dim : 0) * factor;
                }
                unsure |= beyond(four[0], four[1], kLimbMostScore);
                const Limbs8 limbs = split8(four[0], four[1]);
#pragma unroll
                for (int l = 0; l < kLimbs; ++l) query[k][l] = limbs.limb[l];
            }
        }
        auto low_of = [&](int p) { return a.window > 0 && p >= a.window ? p - a.window + 1 : 0; };

        // Threads below kStage look up one key each.  Rows behind the last key repeat it; keys on no page are the pool's first.
        auto position_of = [&](int t) {
            const int position = stages.base(t) + static_cast<int>(threadIdx.x);
            return position < stages.seen ? position : stages.seen - 1;
        };
        auto look_up = [&](int t) {
            return t < to && static_cast<int>(threadIdx.x) < kStage ? table[divide(position_of(t), a.page)] : 0;
        };
        auto put_places = [&](int t, int page) {
            if (t >= to || static_cast<int>(threadIdx.x) >= kStage) return;
            const int position = position_of(t);
            const bool held = page >= 0 && page < a.pages;
            const int64_t of_page = held ? page : 0;
            const int in_page = held ? position - static_cast<int>(divide(position, a.page) * a.page.divisor) : 0;
            places[t & 1][0][threadIdx.x] = of_page * a.key_strides[0] + in_page * a.key_strides[2];
            places[t & 1][1][threadIdx.x] = of_page * a.value_strides[0] + in_page * a.value_strides[2];
            const uint64_t gone = __ballot(!held);
            if (lane == 0) missing[t & 1][0] = static_cast<uint32_t>(gone);
            if (lane == 32) missing[t & 1][1] = static_cast<uint32_t>(gone >> 32);
        };
        f32x4 held[2][kPerThread][2];  // of this thread's pieces: row threadIdx.x / kPieces + 32 i, piece threadIdx.x % kPieces
        const int piece = threadIdx.x % kPieces, piece_row = threadIdx.x / kPieces;
        auto fetch = [&](int t) {
#pragma unroll
            for (int side = 0; side < 2; ++side)
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    const float* row = (side ? values : keys) + places[t & 1][side][piece_row + 32 * i];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = 8 * piece + 4 * j;  // dims behind the head's: its first, which meet zeros or are not stored
                        if constexpr (kWide) held[side][i][j] = *reinterpret_cast<const f32x4*>(row + (d < a.dim ? d : 0));
                        else held[side][i][j] = Mfma<float>::load_strided(row, 1, d, a.dim);
                    }
                }
        };
        auto put = [&](const uint32_t (&gone)[kSubs]) {
#pragma unroll
            for (int side = 0; side < 2; ++side)
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    const int row = piece_row + 32 * i;
                    if (gone[i] >> piece_row & 1) held[side][i][0] = held[side][i][1] = f32x4{0, 0, 0, 0};
                    unsure |= beyond(held[side][i][0], held[side][i][1], side ? kLimbMostValue : kLimbMostScore);
                    const Limbs8 limbs = split8(held[side][i][0], held[side][i][1]);
                    char* at = planes + side * kSide + row * kRowBytes + (piece ^ swizzle<kDim>(row)) * 16;
#pragma unroll
                    for (int l = 0; l < kLimbs; ++l) *reinterpret_cast<u32x4*>(at + l * kPlane) = limbs.limb[l];
                }
        };
        int key_at[kSteps], value_at[kBlocks][2];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) key_at[k] = n32 * kRowBytes + (((2 * k + half) ^ swizzle<kDim>(n32)) * 16);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * e + 4 * half + (lane & 15) / 4, at = 4 * b + 2 * (lane >> 4 & 1) + (lane & 3) / 2;
                value_at[b][e] = kSide + row * kRowBytes + (at ^ swizzle<kDim>(row)) * 16 + 8 * (lane & 1);
            }

        const int wave_low = low_of(wave_first), low_of_last = low_of(wave_last);
        auto work = [&](const char* at, int first, uint32_t gone, auto masked) {
            f32x16 score;
#pragma unroll
            for (int j = 0; j < 16; ++j) score[j] = 0.0f;
            u32x4 lead[kSteps];
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {  // the small products first
                lead[k] = *reinterpret_cast<const u32x4*>(at + key_at[k]);
                const u32x4 middle = *reinterpret_cast<const u32x4*>(at + key_at[k] + kPlane);
                const u32x4 last = *reinterpret_cast<const u32x4*>(at + key_at[k] + 2 * kPlane);
                score = mfma_bf16(last, query[k][0], score);
                score = mfma_bf16(lead[k], query[k][2], score);
                score = mfma_bf16(middle, query[k][1], score);
                score = mfma_bf16(middle, query[k][0], score);
                score = mfma_bf16(lead[k], query[k][1], score);
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) score = mfma_bf16(lead[k], query[k][0], score);
            if constexpr (decltype(masked)::value) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    // Without branches: low <= key <= position as one unsigned comparison, or a sink.
                    const int in = 8 * (j / 4) + 4 * half + j % 4, of = first + in;
                    const bool visible = ((static_cast<uint32_t>(of - mine.low) <= static_cast<uint32_t>(mine.position - mine.low)) |
                                          (of < mine.sink_end)) & !(gone >> in & 1);
                    score[j] = visible ? score[j] : -INFINITY;
                }
            }
            float highest = fmaxf(score[0], score[1]);
#pragma unroll
            for (int j = 2; j < 16; j += 2) highest = fmaxf(fmaxf(highest, score[j]), score[j + 1]);
            highest = half_max(highest);
            const bool moves = __any(highest - top > kLazy);  // NaN where both are -inf
            float shrink = 1.0f;
            if (moves) {
                const float now = fmaxf(top, highest);
                shrink = top == -INFINITY ? 0.0f : fast_exp2(top - now);
                top = now;
                weight *= shrink;
            }
            scale_if<kBlocks>(moves, shrink, out);
            const float reference = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                f32x4 p[2];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j / 4][j % 4] = fast_exp2(score[8 * k + j] - reference);
                    weight += p[j / 4][j % 4];
                }
                const Limbs8 limbs = split8(p[0], p[1]);
                u32x4 value[kBlocks][kLimbs];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int l = 0; l < kLimbs; ++l) {
                        const u32x2 low = read_transposed(at + value_at[b][0] + l * kPlane + 16 * k * kRowBytes);
                        const u32x2 high = read_transposed(at + value_at[b][1] + l * kPlane + 16 * k * kRowBytes);
                        value[b][l] = u32x4{low[0], low[1], high[0], high[1]};
                    }
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = mfma_bf16(value[b][2], limbs.limb[0], out[b]);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = mfma_bf16(value[b][0], limbs.limb[2], out[b]);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = mfma_bf16(value[b][1], limbs.limb[1], out[b]);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = mfma_bf16(value[b][1], limbs.limb[0], out[b]);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = mfma_bf16(value[b][0], limbs.limb[1], out[b]);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) out[b] = mfma_bf16(value[b][0], limbs.limb[0], out[b]);
            }
        };

        put_places(from, look_up(from));
        put_places(from + 1, look_up(from + 1));
        __syncthreads();
        uint32_t gone[kSubs];
#pragma unroll
        for (int i = 0; i < kSubs; ++i) gone[i] = missing[from & 1][i];
        fetch(from);
        for (int t = from; t < to; ++t) {
            __syncthreads();  // the stage before has been read
            put(gone);
            const int page = look_up(t + 2);
            __syncthreads();
            uint32_t next[kSubs];
#pragma unroll
            for (int i = 0; i < kSubs; ++i) next[i] = missing[(t + 1) & 1][i];  // of no stage behind the last
            if (t + 1 < to) fetch(t + 1);
            const uint32_t any_gone = __builtin_amdgcn_readfirstlane(gone[0] | gone[1]);
            const int base = stages.base(t), last = base + kStage - 1;
            const bool seen = base <= wave_last && (last >= wave_low || base < a.sinks);
            if (seen && !any_gone && base >= low_of_last && last <= wave_first) {  // all of it, by all rows
#pragma unroll
                for (int i = 0; i < kSubs; ++i) work(planes + 32 * i * kRowBytes, base + 32 * i, 0, std::false_type{});
            } else if (seen) {
#pragma unroll 1
                for (int i = 0; i < kSubs; ++i) {
                    const int first = base + 32 * i;
                    if (first > wave_last || (first + 31 < wave_low && first >= a.sinks)) continue;
                    work(planes + 32 * i * kRowBytes, first, gone[i], std::true_type{});
                }
            }
#pragma unroll
            for (int i = 0; i < kSubs; ++i) gone[i] = next[i];
            put_places(t + 2, page);
        }
    }

    weight = half_sum(weight);
    unsigned least = ~0u;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            least = min(least, magnitude_key(out[b][j]));
        }
    unsure |= least < magnitude_key(kLimbLeastSum * static_cast<float>(to - from + 1));
    unsure |= mine.position >= 0 && top != -INFINITY && !(fabsf(top) < kLimbFar);
    if (__syncthreads_or(unsure)) {
        for (int row = row0; row < row0 + kRows && row < all_rows; row += rows_of_tile<float>(kDim)) {
            register_rows<kDim, kWide ? kWideRows : kNarrow>(a, plan, s, part, kv_head, row0, row, stages, from, to, reinterpret_cast<float*>(planes));
            __syncthreads();
        }
        return;
    }
    if (!real) return;
    const bool cut = part.parts > 1;
    float* o = cut ? part_row(a, plan, kv_head, part.slot, r - row0)
                   : static_cast<float*>(a.out) + (static_cast<int64_t>(s.begin + index) * a.query_heads + head) * a.dim;
    const float inverse = cut ? 1.0f : (weight == 0.0f || mine.position < 0 ? 0.0f : 1.0f / weight);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const int d = 32 * b + 2 * j + 4 * half;  // four dims side by side
            const f32x4 four = {out[b][j] * inverse, out[b][j + 1] * inverse, out[b][j + 2] * inverse, out[b][j + 3] * inverse};
            if (kWide || cut) {
                if (d < a.dim) *reinterpret_cast<f32x4*>(o + d) = four;
            } else {
#pragma unroll
                for (int l = 0; l < 4; ++l)
                    if (d + l < a.dim) o[d + l] = four[l];
            }
        }
    if (cut && half == 0) {
        const float highest = mine.position < 0 ? -INFINITY : top;
        put_statistics(o + plan.width - 4, highest, mine.position < 0 ? 0.0f : weight, highest / kLog2e);
    }
}

// Joins the parts of a tile that was cut.  Workgroup (cut tile, KV head, a share of the rows).  With few parts a thread takes four
// dims of a row.  With more a wave takes a row, its lanes the parts' shares first, then fours of dims, of which a narrow head's
// lanes divide the parts among them (63 parts of 64 rows, 8 heads of 128: 37 us a call against 81; 4387 rows of 2 to 4
// parts, 8 heads of 80: 12 us against 26 with a wave a row).
constexpr int kFewParts = 8;
constexpr int kJoinParts = 1024;  // whose shares are kept

// Nothing is left out where a share is 0: a part's sums may be NaN or infinite, and 0 times these is NaN as in a tile that is not cut.
__device__ __forceinline__ float share_of(const float* statistics, float top, float natural, float argument) {
    const bool near = fabsf(top) < kFar && fabsf(statistics[0]) < kFar;
    const float share = fast_exp2(near ? statistics[0] - top : (statistics[2] - natural) * argument);
    return statistics[2] == -INFINITY ? 0.0f : share;  // it saw nothing, or no score above -inf that is a number
}

template <class T>
__device__ __forceinline__ void store_joined(const ChunkArgs& a, int begin, int row, int kv_head, int four, float weight, const f32x4& sum) {
    const int i = static_cast<int>(divide(row, a.group_of)), head = kv_head * a.group + row - i * a.group;
    T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(begin + i) * a.query_heads + head) * a.dim + 4 * four;
#pragma unroll
    for (int l = 0; l < 4; ++l)
        if (4 * four + l < a.dim) out[l] = static_cast<T>(weight == 0.0f ? 0.0f : sum[l] / weight);
}

// kMost parts or fewer: a thread takes four dims of a row, all of its loads ahead of their use.
template <class T, int kMost>
__device__ __forceinline__ void join_few(const ChunkArgs& a, const ChunkPlan& plan, int begin, int row0, int slot, int parts, int from, int to) {
    const int kv_head = blockIdx.y, fours = (a.dim + 3) / 4;
    const int64_t stride = static_cast<int64_t>(plan.slot_rows) * plan.width;
    const ScoreScale<T> scale(a.scale);
    for (int item = threadIdx.x; item < (to - from) * fours; item += kThreads) {
        const int r = from + item / fours, four = item % fours;
        const float* o = part_row(a, plan, kv_head, slot, r);
        const float* of = o + plan.width - 4;
        float top = -INFINITY, natural = -INFINITY, weight = 0.0f;
        f32x4 statistics[kMost], sums[kMost], sum = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < kMost; ++p) {  // of the first part where there is none
            const int64_t at = p < parts ? p * stride : 0;
            statistics[p] = *reinterpret_cast<const f32x4*>(of + at);
            sums[p] = *reinterpret_cast<const f32x4*>(o + at + 4 * four);
        }
#pragma unroll
        for (int p = 0; p < kMost; ++p) top = fmaxf(top, statistics[p][0]), natural = fmaxf(natural, statistics[p][2]);
#pragma unroll
        for (int p = 0; p < kMost; ++p) {
            const float own[3] = {statistics[p][0], statistics[p][1], statistics[p][2]};
            const float share = share_of(own, top, natural, scale.argument);
            weight += p < parts ? own[1] * share : 0.0f;
#pragma unroll
            for (int l = 0; l < 4; ++l) sum[l] += p < parts ? sums[p][l] * share : 0.0f;
        }
        store_joined<T>(a, begin, row0 + r, kv_head, four, weight, sum);
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) chunk_join_kernel(ChunkArgs a, ChunkPlan plan, int fours_bits) {
    __shared__ float shares[kWaves][kJoinParts];
    const int* header = reinterpret_cast<const int*>(a.workspace);
    if (static_cast<int>(blockIdx.x) >= header[0]) return;
    const int* d = header + kDescription * (1 + blockIdx.x);
    const int begin = d[0], row0 = d[1], rows = d[2], slot = d[3], parts = d[4];
    // With offsets that decrease some tile's first part may be no workgroup's, and its description anything.
    if (begin < 0 || row0 < 0 || rows < 0 || rows > plan.slot_rows || parts < 2 || slot < 0 ||
        static_cast<int64_t>(slot) + parts > plan.slots || static_cast<int64_t>(row0) + rows > (a.tokens - begin) * a.group)
        return;
    const int kv_head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t stride = static_cast<int64_t>(plan.slot_rows) * plan.width;
    const int each = (rows + gridDim.z - 1) / gridDim.z, from = blockIdx.z * each, to = from + each < rows ? from + each : rows;
    if (parts <= 2) return join_few<T, 2>(a, plan, begin, row0, slot, parts, from, to);
    if (parts <= 4) return join_few<T, 4>(a, plan, begin, row0, slot, parts, from, to);
    if (parts <= kFewParts) return join_few<T, kFewParts>(a, plan, begin, row0, slot, parts, from, to);
    const ScoreScale<T> scale(a.scale);
    const int four = lane & ((1 << fours_bits) - 1), turn = lane >> fours_bits, turns = kWave >> fours_bits;
    for (int r = from + wave; r < to; r += kWaves) {
        const float* o = part_row(a, plan, kv_head, slot, r);
        const float* of = o + plan.width - 4;
        float top = -INFINITY, natural = -INFINITY;
#pragma unroll 2
        for (int p = lane; p < parts; p += kWave) top = fmaxf(top, of[p * stride]), natural = fmaxf(natural, of[p * stride + 2]);
        top = wave_max(top);
        natural = wave_max(natural);
        float weight = 0.0f;
        for (int p = lane; p < parts; p += kWave) {
            const float share = share_of(of + p * stride, top, natural, scale.argument);
            weight += of[p * stride + 1] * share;
            if (p < kJoinParts) shares[wave][p] = share;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes of the wave read them
        weight = wave_sum(weight);
        f32x4 sum = {0, 0, 0, 0};
        if (4 * four < a.dim) {
#pragma unroll 8
            for (int p = turn; p < parts; p += turns) {
                const f32x4 part_sum = *reinterpret_cast<const f32x4*>(o + p * stride + 4 * four);
                const float share = p < kJoinParts ? shares[wave][p] : share_of(of + p * stride, top, natural, scale.argument);
#pragma unroll
                for (int l = 0; l < 4; ++l) sum[l] += part_sum[l] * share;
            }
        }
        for (int step = 1 << fours_bits; step < kWave; step *= 2)
#pragma unroll
            for (int l = 0; l < 4; ++l) sum[l] += __shfl_xor(sum[l], step, kWave);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the next row's shares take their places
        if (turn == 0) store_joined<T>(a, begin, row0 + r, kv_head, four, weight, sum);
    }
}

constexpr int64_t kJoinBlocks = 1024;  // about, many of which find no cut tile (4096: 89 us for 88 of a call, 16384: 93)

// Parts that a step's work is cut into: 16-bit two rounds of two workgroups on each of 256 CUs, so that a CU whose parts end early
// takes others; more parts write and join more sums.  With 512, 768, 1024, 1280 and 1536 the step of chunks and single tokens took 796, 720,
// 668, 687 and 645 us, the 16 chunks in a window 121, 82, 88, 89 and 90.  float32, whose single tokens' workgroups are three a
// CU: 32 of them over 4000 keys 44 us with 768 and 52 with 1024, prompts 226 and 235.
template <class T>
constexpr int parts_of_step() { return sizeof(T) == 2 ? 1024 : 768; }

// Whether float32 takes the limb kernel: its tiles have 128 rows, which single tokens leave empty, and few of them leave CUs
// idle.  Limbs and float32 products: 4 x 512 tokens over 512 keys each 161 and 238 us, 2048 tokens over 8192 253 and 443;
// but 512 tokens over 512 keys in 4 heads 38 and 28, 64 over 2000 55 and 27, 32 single tokens over 4000 89 and 51.
constexpr int64_t kLimbRows = 64, kLimbAll = 2048;
bool by_limbs(const ChunkArgs& a) {
    const int64_t rows = a.tokens * a.group;
    return a.dim <= 64 && rows >= kLimbRows * a.requests && rows >= kLimbAll;
}

template <class T>
ChunkPlan plan_of(const ChunkArgs& a) {
    const int dim = padded_dim(a.dim);
    ChunkPlan p{};
    p.rows = sizeof(T) == 4 && by_limbs(a) ? 32 * kWaves : rows_of_tile<T>(dim);
    const int stage = stage_keys<T>(dim);
    const int64_t rows = a.tokens * a.group;
    p.tiles = rows / p.rows + a.requests;
    if (p.tiles > rows) p.tiles = rows;
    p.target = (parts_of_step<T>() + a.kv_heads - 1) / a.kv_heads;
    int64_t stages = (a.keys + stage - 1) / stage;
    if (a.window > 0) {
        const int64_t windowed = (static_cast<int64_t>(a.sinks) + stage - 1) / stage + (static_cast<int64_t>(a.window) + p.rows / a.group + 1) / stage + 2;
        if (windowed < stages) stages = windowed;
    }
    p.whole = stages <= kWholeStages;
    p.least = sizeof(T) == 4 && by_limbs(a) ? 4 : least_stages<T>();
    p.units = p.tiles;
    if (!p.whole) {
        // A tile of S > each stages has at most S / each + 1 < 2 S / each parts, and the sum of all S is at most target times
        // each; the least number of stages bounds them as well.
        const int64_t most = p.tiles * ((stages + p.least - 1) / p.least);
        p.slots = 2 * static_cast<int64_t>(p.target) < most ? 2 * static_cast<int64_t>(p.target) : most;
        p.splits = p.target < p.tiles ? p.target : p.tiles;
        p.units = p.tiles + p.target < most ? p.tiles + p.target : most;
    }
    p.slot_rows = rows < p.rows ? static_cast<int>(rows) : p.rows;
    p.width = (a.dim + 3) / 4 * 4 + 4;
    return p;
}

template <class T, int kDim, int kUsed>
hipError_t launch_tiles(const ChunkArgs& a, const ChunkPlan& plan, dim3 grid, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        constexpr int kStage = stage_keys<T>(kDim);
        constexpr size_t kLds = 4 * kStage * kDim * 2;
        auto launch = [&](auto* kernel) {
            const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                        static_cast<int>(kLds));
            if (room != hipSuccess) return room;
            hipLaunchKernelGGL(kernel, grid, dim3(kThreads), kLds, stream, a, plan);
            return hipGetLastError();
        };
        if (a.wide && reinterpret_cast<uintptr_t>(a.out) % 8 == 0) return launch(chunk_tile_kernel<T, kDim, kUsed, true>);
        return launch(chunk_tile_kernel<T, kDim, kUsed, false>);
    } else {
        if constexpr (kDim == 64) {
            if (by_limbs(a)) {
                if (a.wide && reinterpret_cast<uintptr_t>(a.out) % 16 == 0) hipLaunchKernelGGL(chunk_limb_kernel<true>, grid, dim3(kThreads), 0, stream, a, plan);
                else hipLaunchKernelGGL(chunk_limb_kernel<false>, grid, dim3(kThreads), 0, stream, a, plan);
                return hipGetLastError();
            }
        }
        if (a.wide && a.dim == kDim) hipLaunchKernelGGL(HIP_KERNEL_NAME(chunk_register_kernel<kDim, kFullRows>), grid, dim3(kThreads), 0, stream, a, plan);
        else if (a.wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(chunk_register_kernel<kDim, kWideRows>), grid, dim3(kThreads), 0, stream, a, plan);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(chunk_register_kernel<kDim, kNarrow>), grid, dim3(kThreads), 0, stream, a, plan);
        return hipGetLastError();
    }
}

// Every strip ends with a whole turn of kStrips.
int64_t workgroups_of(const ChunkArgs& a, const ChunkPlan& plan) { return (plan.units + kStrips - 1) * a.kv_heads; }

template <class T>
hipError_t launch_chunks(const ChunkArgs& a, hipStream_t stream) {
    const ChunkPlan plan = plan_of<T>(a);
    const dim3 grid(static_cast<uint32_t>(workgroups_of(a, plan)));
    hipError_t launched;
    // The 16-bit kernel leaves the last quarter of a row out: 97 us for 103 at 80 dims.
    constexpr int kNarrower = sizeof(T) == 2 ? 96 : 128;
    if (a.dim <= 64) launched = launch_tiles<T, 64, 64>(a, plan, grid, stream);
    else if (a.dim <= kNarrower) launched = launch_tiles<T, 128, kNarrower>(a, plan, grid, stream);
    else if (a.dim <= 128) launched = launch_tiles<T, 128, 128>(a, plan, grid, stream);
    else launched = launch_tiles<T, 256, 256>(a, plan, grid, stream);
    if (launched != hipSuccess || plan.whole) return launched;
    int fours_bits = 0;
    while (4 << fours_bits < a.dim) ++fours_bits;
    const int64_t tiles = plan.splits * a.kv_heads, most = (plan.slot_rows + kWaves - 1) / kWaves;
    int64_t folds = (kJoinBlocks + tiles - 1) / tiles;
    if (folds > most) folds = most;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(chunk_join_kernel<T>), dim3(static_cast<uint32_t>(plan.splits), a.kv_heads, static_cast<uint32_t>(folds)),
                       dim3(kThreads), 0, stream, a, plan, fours_bits);
    return hipGetLastError();
}

}  // namespace

size_t chunk_attention_workspace_floats(const ChunkArgs& a, Type type) {
    const ChunkPlan p = type == Type::kFloat32 ? plan_of<float>(a) : plan_of<__bf16>(a);
    return p.whole ? 0 : static_cast<size_t>(parts_offset(p) + a.kv_heads * p.slots * p.slot_rows * p.width);
}

int64_t chunk_attention_workgroups(const ChunkArgs& a, Type type) {
    return workgroups_of(a, type == Type::kFloat32 ? plan_of<float>(a) : plan_of<__bf16>(a));
}

hipError_t launch_chunk_attention(const ChunkArgs& args, Type type, hipStream_t stream) {
    switch (type) {
        case Type::kFloat32: return launch_chunks<float>(args, stream);
        case Type::kFloat16: return launch_chunks<_Float16>(args, stream);
        default: return launch_chunks<__bf16>(args, stream);
    }
}

}  // namespace flux
