// Pages of a K/V cache: reserving, writing, copying, forking, freeing and compacting them without the host.
//
// The books are a page table [slots, columns] (-1: no page), the slots' lengths and a count of holders per page (0:
// free).  A page that is needed is always the lowest free one, and requests are served in their order, so that
// results do not depend on scheduling.  Every operator is one launch of bookkeeping, or one and a copy over the whole
// card: the bookkeeping is a few KB and bound by latency, the copies by HBM.
#include "serving.h"

namespace flux {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

// Values that other threads of this workgroup wrote: past the L1.
__device__ __forceinline__ int32_t load_shared_word(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared_word(int32_t* p, int32_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void plan_barrier() {
    __threadfence();
    __syncthreads();
}

__device__ __forceinline__ int wave_inclusive_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int below = __shfl_up(v, step, kWave);
        if (lane >= step) v += below;
    }
    return v;
}

// Exclusive prefix over the workgroup's threads and the total.  `sums` holds kPlanWaves words.
__device__ __forceinline__ int block_exclusive_scan(int v, int* sums, int* total) {
    const int wave = threadIdx.x >> 6;
    const int inclusive = wave_inclusive_scan(v);
    __syncthreads();  // sums may still be read from the call before
    if ((threadIdx.x & 63) == 63) sums[wave] = inclusive;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const int s = sums[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return before + inclusive - v;
}

// The first `wanted` free pages, lowest first, into `list`; returns how many there are (at most `wanted`).
__device__ int find_free_pages(const int32_t* refcounts, int64_t pages, int wanted, int32_t* list, int* sums) {
    int found = 0;
    for (int64_t base = 0; base < pages && found < wanted; base += 4 * kPlanThreads) {
        const int64_t first = base + 4 * threadIdx.x;
        int free[4], count = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            free[j] = first + j < pages && refcounts[first + j] <= 0;
            count += free[j];
        }
        int total = 0;
        int rank = found + block_exclusive_scan(count, sums, &total);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!free[j]) continue;
            if (rank < wanted) store_shared_word(list + rank, static_cast<int32_t>(first + j));
            ++rank;
        }
        found += total;
    }
    plan_barrier();
    return found < wanted ? found : wanted;
}

// Marks the first request that names each slot: first[slot] == i afterwards exactly for that one.
__device__ void mark_first(const int64_t* list, int64_t requests, int64_t slots, int32_t* first) {
    for (int64_t i = threadIdx.x; i < requests; i += kPlanThreads) {
        const int64_t slot = list[i];
        if (slot >= 0 && slot < slots) store_shared_word(first + slot, 0x7fffffff);
    }
    plan_barrier();
    for (int64_t i = threadIdx.x; i < requests; i += kPlanThreads) {
        const int64_t slot = list[i];
        if (slot >= 0 && slot < slots) atomicMin(first + slot, static_cast<int32_t>(i));
    }
    plan_barrier();
}

// In place: need[i] -> sum of need[0..i]; returns the total.  A request without pages to get has need 0.
__device__ int prefix_in_place(int32_t* need, int64_t requests, int* sums) {
    int running = 0;
    for (int64_t base = 0; base < requests; base += kPlanThreads) {
        const int64_t i = base + threadIdx.x;
        const int mine = i < requests ? load_shared_word(need + i) : 0;
        int total = 0;
        const int before = block_exclusive_scan(mine, sums, &total);
        if (i < requests) store_shared_word(need + i, running + before + mine);
        running += total;
    }
    plan_barrier();
    return running;
}

// ---------------------------------------------------------------------------
// Reserve.  Sixteen lanes share a request: a decode step looks at one column each, a prompt at one per page.
constexpr int kReserveLanes = 16;

struct ReserveRange {
    int64_t slot, length, first, last;  // columns [first, last)
    int32_t status;
};

__device__ ReserveRange reserve_range(const PageBooks& b, const int64_t* slots, const int64_t* counts, int64_t i,
                                      const int32_t* first_request) {
    ReserveRange r{slots[i], 0, 0, 0, kPageDone};
    const int64_t count = counts ? counts[i] : 1;
    if (r.slot < 0 || r.slot >= b.slots || count < 0) {
        r.status = kPageOutOfRange;
    } else if (load_shared_word(first_request + r.slot) != static_cast<int32_t>(i)) {
        r.status = kPageRepeated;
    } else {
        r.length = b.lengths[r.slot];
        const int64_t capacity = b.columns * b.page;
        if (r.length < 0 || r.length > capacity) {
            r.status = kPageOutOfRange;
        } else if (count > capacity - r.length) {
            r.status = kPageNoRoom;
        } else if (count > 0) {
            r.first = r.length / b.page;
            r.last = (r.length + count - 1) / b.page + 1;
        }
    }
    return r;
}

__global__ void __launch_bounds__(kPlanThreads) page_reserve_kernel(PageBooks b, const int64_t* __restrict__ slots,
                                                                    const int64_t* __restrict__ counts,
                                                                    int64_t requests, int64_t* positions,
                                                                    int32_t* status, int32_t* workspace) {
    __shared__ int sums[kPlanWaves];
    int32_t* first_request = workspace;             // [slots]
    int32_t* need = first_request + b.slots;        // [requests]: pages of each request, then their prefix
    int32_t* list = need + requests;                // [pages]
    const int lane = threadIdx.x % kReserveLanes;
    const int group = threadIdx.x / kReserveLanes;
    constexpr int kGroups = kPlanThreads / kReserveLanes;
    mark_first(slots, requests, b.slots, first_request);

    for (int64_t base = 0; base < requests; base += kGroups) {
        const int64_t i = base + group;
        int count = 0;
        if (i < requests) {
            const ReserveRange r = reserve_range(b, slots, counts, i, first_request);
            const int32_t* row = b.table + r.slot * b.table_stride;
            for (int64_t c = r.first + lane; c < r.last; c += kReserveLanes) count += row[c] < 0;
        }
#pragma unroll
        for (int step = 1; step < kReserveLanes; step *= 2) count += __shfl_xor(count, step, kWave);
        if (i < requests && lane == 0) store_shared_word(need + i, count);
    }
    plan_barrier();
    const int total = prefix_in_place(need, requests, sums);
    const int64_t most = total < b.pages ? total : b.pages;
    const int found = total > 0 ? find_free_pages(b.refcounts, b.pages, static_cast<int>(most), list, sums) : 0;

    for (int64_t base = 0; base < requests; base += kGroups) {
        const int64_t i = base + group;
        if (i >= requests) continue;  // whole groups: the ballots below stay within one
        ReserveRange r = reserve_range(b, slots, counts, i, first_request);
        const int upto = load_shared_word(need + i);
        int rank = i > 0 ? load_shared_word(need + i - 1) : 0;
        if (r.status == kPageDone && upto > rank && upto > found) r.status = kPageNoRoom;
        if (r.status == kPageDone) {
            int32_t* row = b.table + r.slot * b.table_stride;
            for (int64_t c0 = r.first; c0 < r.last; c0 += kReserveLanes) {
                const int64_t c = c0 + lane;
                const bool empty = c < r.last && row[c] < 0;
                const uint64_t all = __ballot(empty);
                const int shift = (threadIdx.x & 63) / kReserveLanes * kReserveLanes;
                const uint32_t mine = static_cast<uint32_t>(all >> shift) & 0xffffu;
                if (empty) {
                    const int32_t page = load_shared_word(list + rank + __popc(mine & ((1u << lane) - 1u)));
                    row[c] = page;
                    b.refcounts[page] = 1;
                }
                rank += __popc(mine);
            }
        }
        if (lane == 0) {
            status[i] = r.status;
            positions[i] = r.status == kPageDone ? r.length : -1;
            if (r.status == kPageDone && r.last > r.first) b.lengths[r.slot] = r.length + (counts ? counts[i] : 1);
        }
    }
}

// ---------------------------------------------------------------------------
// Free.  One workgroup per request; counts saturate at zero, so the result does not depend on the order.
__global__ void __launch_bounds__(256) page_free_kernel(PageBooks b, const int64_t* __restrict__ slots,
                                                        int32_t* status) {
    const int64_t i = blockIdx.x;
    const int64_t slot = slots[i];
    if (slot < 0 || slot >= b.slots) {
        if (threadIdx.x == 0) status[i] = kPageOutOfRange;
        return;
    }
    int repeated = 0;
    for (int64_t j = threadIdx.x; j < i; j += 256) repeated |= slots[j] == slot;
    if (__syncthreads_or(repeated)) {
        if (threadIdx.x == 0) status[i] = kPageRepeated;
        return;
    }
    int32_t* row = b.table + slot * b.table_stride;
    for (int64_t c = threadIdx.x; c < b.columns; c += 256) {
        const int32_t page = row[c];
        if (page >= 0 && page < b.pages && atomicSub(b.refcounts + page, 1) <= 0) atomicAdd(b.refcounts + page, 1);
        row[c] = -1;
    }
    if (threadIdx.x == 0) {
        b.lengths[slot] = 0;
        status[i] = kPageDone;
    }
}

// ---------------------------------------------------------------------------
// Rows of one page of one layer's keys or values, `rows` of each head.  kUnit: 16 bytes where rows allow it.
template <class Unit>
__device__ __forceinline__ void copy_page_rows(char* base, const int64_t* strides, int64_t heads, int rows, int width,
                                               int element, int64_t layer, int64_t from, int64_t to) {
    const Unit* src = reinterpret_cast<const Unit*>(base + (layer * strides[0] + from * strides[1]) * element);
    Unit* dst = reinterpret_cast<Unit*>(base + (layer * strides[0] + to * strides[1]) * element);
    const int64_t head_stride = strides[2] * element / static_cast<int>(sizeof(Unit));
    const int64_t row_stride = strides[3] * element / static_cast<int>(sizeof(Unit));
    const int per_head = rows * width;
    const int items = static_cast<int>(heads) * per_head;
    constexpr int kAhead = 4;
    for (int base_item = threadIdx.x; base_item < items; base_item += kAhead * 256) {
        Unit held[kAhead];
        int64_t at[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int item = base_item + 256 * j;
            if (item < items) {
                const int head = item / per_head, rest = item % per_head;
                at[j] = head * head_stride + (rest / width) * row_stride + rest % width;
                held[j] = src[at[j]];
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (base_item + 256 * j < items) dst[at[j]] = held[j];
    }
}

template <class Unit>
__device__ __forceinline__ void copy_rows(const PagePool& p, int64_t layer, int side, int64_t from, int64_t to,
                                          int64_t rows) {
    copy_page_rows<Unit>(side ? p.value : p.key, side ? p.value_strides : p.key_strides, p.heads,
                         static_cast<int>(rows), static_cast<int>(p.dim * p.element / static_cast<int>(sizeof(Unit))),
                         p.element, layer, from, to);
}

// Copy.  Workgroup (request, 2 * layer + side).  Every workgroup of a request looks through the lists for the
// conflicts that would make its result depend on the order: a few loads against a page's rows.
template <class Unit>
__global__ void __launch_bounds__(256) page_copy_kernel(PagePool p, const int64_t* __restrict__ source,
                                                        const int64_t* __restrict__ target, int64_t requests,
                                                        int32_t* status) {
    const int64_t i = blockIdx.x;
    const int64_t from = source[i], to = target[i];
    int result = kPageDone;
    if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
        result = kPageOutOfRange;
    } else {
        int clash = 0;
        for (int64_t j = threadIdx.x; j < requests; j += 256)
            clash |= (j < i && target[j] == to) || (j != i && source[j] == to);
        if (__syncthreads_or(clash)) result = kPageRepeated;
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) status[i] = result;
    if (result != kPageDone || from == to) return;
    copy_rows<Unit>(p, blockIdx.y >> 1, blockIdx.y & 1, from, to, p.page);
}

// ---------------------------------------------------------------------------
// Fork.  The plan reads the books as they were; the second launch shares full pages and copies partial ones.
struct ForkPlan {
    int32_t* first_request;  // [slots]
    int32_t* need;           // [requests]
    int32_t* list;           // [pages]
    int32_t* length;         // [requests]: tokens of the parent, -1: refused
    int32_t* fresh;          // [requests]: new page of the partial rows
};

__device__ __host__ ForkPlan fork_plan(int32_t* workspace, int64_t requests, int64_t slots, int64_t pages) {
    ForkPlan f;
    f.first_request = workspace;
    f.need = f.first_request + slots;
    f.list = f.need + requests;
    f.length = f.list + pages;
    f.fresh = f.length + requests;
    return f;
}

__global__ void __launch_bounds__(kPlanThreads) page_fork_plan_kernel(PageBooks b,
                                                                      const int64_t* __restrict__ parents,
                                                                      const int64_t* __restrict__ children,
                                                                      int64_t requests, int32_t* status,
                                                                      int32_t* workspace) {
    __shared__ int sums[kPlanWaves];
    const ForkPlan f = fork_plan(workspace, requests, b.slots, b.pages);
    mark_first(children, requests, b.slots, f.first_request);
    constexpr int kGroups = kPlanThreads / kReserveLanes;
    const int lane = threadIdx.x % kReserveLanes;
    const int group = threadIdx.x / kReserveLanes;
    for (int64_t base = 0; base < requests; base += kGroups) {
        const int64_t i = base + group;
        int result = kPageDone, bad = 0;
        int64_t length = 0;
        if (i < requests) {
            const int64_t parent = parents[i], child = children[i];
            if (parent < 0 || parent >= b.slots || child < 0 || child >= b.slots) {
                result = kPageOutOfRange;
            } else if (load_shared_word(f.first_request + child) != static_cast<int32_t>(i)) {
                result = kPageRepeated;
            } else if (b.lengths[child] != 0) {
                result = kPageOccupied;
            } else {
                // A slot of length 0 may still hold pages that no token has filled.
                const int32_t* own = b.table + child * b.table_stride;
                for (int64_t c = lane; c < b.columns; c += kReserveLanes) bad |= own[c] >= 0 ? 2 : 0;
                length = b.lengths[parent];
                if (length < 0 || length > b.columns * b.page) {
                    result = kPageOutOfRange;
                } else {
                    const int64_t held = (length + b.page - 1) / b.page;
                    const int32_t* row = b.table + parent * b.table_stride;
                    for (int64_t c = lane; c < held; c += kReserveLanes) bad |= row[c] < 0 || row[c] >= b.pages;
                }
            }
        }
#pragma unroll
        for (int step = 1; step < kReserveLanes; step *= 2) bad |= __shfl_xor(bad, step, kWave);
        if (i < requests && lane == 0) {
            if (bad & 2) result = kPageOccupied;
            else if (bad & 1) result = kPageOutOfRange;
            store_shared_word(f.need + i, result == kPageDone && length % b.page != 0);
            store_shared_word(f.length + i, result == kPageDone ? static_cast<int32_t>(length) : -1 - result);
        }
    }
    plan_barrier();
    const int total = prefix_in_place(f.need, requests, sums);
    const int64_t most = total < b.pages ? total : b.pages;
    const int found = total > 0 ? find_free_pages(b.refcounts, b.pages, static_cast<int>(most), f.list, sums) : 0;
    for (int64_t i = threadIdx.x; i < requests; i += kPlanThreads) {
        const int32_t length = load_shared_word(f.length + i);
        const int upto = load_shared_word(f.need + i);
        const int before = i > 0 ? load_shared_word(f.need + i - 1) : 0;
        int32_t result = length < 0 ? -1 - length : kPageDone;
        int32_t fresh = -1;
        if (upto > before) {
            if (upto > found) {
                result = kPageNoRoom;
            } else {
                fresh = load_shared_word(f.list + before);
                b.refcounts[fresh] = 1;
            }
        }
        if (result != kPageDone) f.length[i] = -1;
        f.fresh[i] = fresh;
        status[i] = result;
    }
}

// Workgroup (request, part): part 0 writes the child's books, part 1 + 2 * layer + side copies partial rows.
template <class Unit>
__global__ void __launch_bounds__(256) page_fork_kernel(PagePool p, PageBooks b, const int64_t* __restrict__ parents,
                                                        const int64_t* __restrict__ children, int64_t requests,
                                                        int32_t* workspace) {
    const ForkPlan f = fork_plan(workspace, requests, b.slots, b.pages);
    const int64_t i = blockIdx.x;
    const int64_t length = f.length[i];
    if (length < 0) return;
    const int64_t full = length / b.page, rest = length % b.page;
    // A parent that is itself a child of this call was empty: none of its columns is read.
    const int32_t* from = b.table + parents[i] * b.table_stride;
    if (blockIdx.y == 0) {
        int32_t* to = b.table + children[i] * b.table_stride;
        for (int64_t c = threadIdx.x; c < full; c += 256) {
            const int32_t page = from[c];
            to[c] = page;
            atomicAdd(b.refcounts + page, 1);
        }
        if (threadIdx.x == 0) {
            if (rest) to[full] = f.fresh[i];
            b.lengths[children[i]] = length;
        }
    } else if (rest) {
        const int part = blockIdx.y - 1;
        copy_rows<Unit>(p, part >> 1, part & 1, from[full], f.fresh[i], rest);
    }
}

// ---------------------------------------------------------------------------
// Compact.  U pages are in use; the k-th used page at or above U moves to the k-th free page below it.
struct CompactPlan {
    int32_t* moves;   // [1]
    int32_t* source;  // [pages]
    int32_t* target;  // [pages]
};

__device__ __host__ CompactPlan compact_plan(int32_t* workspace, int64_t pages) {
    return CompactPlan{workspace, workspace + 4, workspace + 4 + pages};
}

__global__ void __launch_bounds__(kPlanThreads) page_compact_plan_kernel(int32_t* refcounts, int64_t pages,
                                                                         int32_t* page_map, int64_t* used,
                                                                         int32_t* workspace) {
    __shared__ int sums[kPlanWaves];
    const CompactPlan plan = compact_plan(workspace, pages);
    int count = 0;
    for (int64_t i = threadIdx.x; i < pages; i += kPlanThreads) count += refcounts[i] > 0;
    int held = 0;
    block_exclusive_scan(count, sums, &held);
    int holes = 0, movers = 0;
    for (int64_t base = 0; base < pages; base += 4 * kPlanThreads) {
        const int64_t first = base + 4 * threadIdx.x;
        int kind[4];  // 1: hole, 2: mover
        int mine_holes = 0, mine_movers = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kind[j] = 0;
            if (first + j >= pages) continue;
            const bool in_use = refcounts[first + j] > 0;
            kind[j] = in_use ? (first + j >= held ? 2 : 0) : (first + j < held ? 1 : 0);
            page_map[first + j] = in_use ? static_cast<int32_t>(first + j) : -1;
            mine_holes += kind[j] == 1;
            mine_movers += kind[j] == 2;
        }
        int total_holes = 0, total_movers = 0;
        int hole = holes + block_exclusive_scan(mine_holes, sums, &total_holes);
        int mover = movers + block_exclusive_scan(mine_movers, sums, &total_movers);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (kind[j] == 1) store_shared_word(plan.target + hole++, static_cast<int32_t>(first + j));
            if (kind[j] == 2) store_shared_word(plan.source + mover++, static_cast<int32_t>(first + j));
        }
        holes += total_holes;
        movers += total_movers;
    }
    plan_barrier();
    for (int k = threadIdx.x; k < movers; k += kPlanThreads) {  // holes == movers
        const int32_t from = load_shared_word(plan.source + k), to = load_shared_word(plan.target + k);
        page_map[from] = to;
        refcounts[to] = refcounts[from];
        refcounts[from] = 0;
    }
    if (threadIdx.x == 0) {
        *plan.moves = movers;
        *used = held;
    }
}

template <class Unit>
__global__ void __launch_bounds__(256) page_compact_kernel(PagePool p, PageBooks b,
                                                           const int32_t* __restrict__ page_map,
                                                           int32_t* workspace) {
    const CompactPlan plan = compact_plan(workspace, p.pages);
    const int64_t entries = b.slots * b.columns;
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < entries;
         e += static_cast<int64_t>(gridDim.x) * 256) {
        int32_t* entry = b.table + e / b.columns * b.table_stride + e % b.columns;
        const int32_t page = *entry;
        if (page >= 0) *entry = page < p.pages ? page_map[page] : -1;
    }
    const int64_t units = static_cast<int64_t>(*plan.moves) * p.layers * 2;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t k = unit / (2 * p.layers), part = unit % (2 * p.layers);
        copy_rows<Unit>(p, part >> 1, part & 1, plan.source[k], plan.target[k], p.page);
    }
}

// ---------------------------------------------------------------------------
// Write.  Workgroup (tokens, request): rows of new tokens, all heads, keys then values.
constexpr int kWriteTokens = 16;

template <class Unit>
__global__ void __launch_bounds__(256) page_write_kernel(PagePool p, PageWriteArgs a) {
    constexpr int kBytes = sizeof(Unit);
    const int64_t i = blockIdx.y;
    const int64_t slot = a.slot_list[i], start = a.positions[i];
    if (slot < 0 || slot >= a.slots || start < 0) return;
    int64_t count = a.counts ? a.counts[i] : a.tokens;
    if (count > a.tokens) count = a.tokens;
    const int64_t capacity = a.columns * p.page;
    if (start >= capacity) return;
    if (count > capacity - start) count = capacity - start;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kWriteTokens;
    const int tokens = static_cast<int>(count - t0 < kWriteTokens ? count - t0 : kWriteTokens);
    const int width = static_cast<int>(p.dim * p.element / kBytes);
    const int heads = static_cast<int>(p.heads);
    const int side_items = tokens * heads * width;
    const int32_t* row = a.table + slot * a.table_stride;
    for (int item = threadIdx.x; item < 2 * side_items; item += 256) {
        const int side = item >= side_items;
        const int at = side ? item - side_items : item;
        const int unit = at % width, head = at / width % heads;
        const int64_t t = t0 + at / width / heads;
        const int64_t position = start + t;
        const int32_t page = row[position / p.page];
        if (page < 0 || page >= p.pages) continue;
        const int64_t* from = side ? a.value_strides : a.key_strides;
        const int64_t* to = side ? p.value_strides : p.key_strides;
        const char* src = (side ? a.value : a.key) + (i * from[0] + head * from[1] + t * from[2]) * p.element;
        char* dst = (side ? p.value : p.key) +
                    (page * to[1] + head * to[2] + position % p.page * to[3]) * p.element;
        reinterpret_cast<Unit*>(dst)[unit] = reinterpret_cast<const Unit*>(src)[unit];
    }
}

bool rows_of(const PagePool& p, int64_t bytes) {
    if (p.dim * p.element % bytes) return false;
    if (reinterpret_cast<uintptr_t>(p.key) % bytes || reinterpret_cast<uintptr_t>(p.value) % bytes) return false;
    for (int i = 0; i < 4; ++i)
        if (p.key_strides[i] * p.element % bytes || p.value_strides[i] * p.element % bytes) return false;
    return true;
}

bool rows_of(const PageWriteArgs& a, int element, int64_t bytes) {
    if (reinterpret_cast<uintptr_t>(a.key) % bytes || reinterpret_cast<uintptr_t>(a.value) % bytes) return false;
    for (int i = 0; i < 3; ++i)
        if (a.key_strides[i] * element % bytes || a.value_strides[i] * element % bytes) return false;
    return true;
}

}  // namespace

size_t page_reserve_workspace(int64_t requests, int64_t slots, int64_t pages) { return requests + slots + pages; }
size_t page_fork_workspace(int64_t requests, int64_t slots, int64_t pages) { return 3 * requests + slots + pages; }
size_t page_compact_workspace(int64_t pages) { return 4 + 2 * pages; }

hipError_t launch_page_reserve(const PageBooks& books, const int64_t* slots, const int64_t* counts, int64_t requests,
                               int64_t* positions, int32_t* status, int32_t* workspace, hipStream_t stream) {
    hipLaunchKernelGGL(page_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, stream, books, slots, counts, requests,
                       positions, status, workspace);
    return hipGetLastError();
}

hipError_t launch_page_free(const PageBooks& books, const int64_t* slots, int64_t requests, int32_t* status,
                            hipStream_t stream) {
    hipLaunchKernelGGL(page_free_kernel, dim3(static_cast<uint32_t>(requests)), dim3(256), 0, stream, books, slots,
                       status);
    return hipGetLastError();
}

// The widest unit that every row's start and length is a multiple of: 16 bytes, else one element.
#define FLUX_BY_UNIT(wide, element, kernel, grid, ...)                                                              \
    if (wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(kernel<uint4>), grid, dim3(256), 0, stream, __VA_ARGS__);          \
    else if ((element) == 4) hipLaunchKernelGGL(HIP_KERNEL_NAME(kernel<uint32_t>), grid, dim3(256), 0, stream,      \
                                                __VA_ARGS__);                                                       \
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(kernel<uint16_t>), grid, dim3(256), 0, stream, __VA_ARGS__);            \
    return hipGetLastError()

hipError_t launch_page_copy(const PagePool& pool, const int64_t* source, const int64_t* target, int64_t requests,
                            int32_t* status, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(requests), static_cast<uint32_t>(2 * pool.layers));
    FLUX_BY_UNIT(rows_of(pool, 16), pool.element, page_copy_kernel, grid, pool, source, target, requests, status);
}

hipError_t launch_page_fork(const PagePool& pool, const PageBooks& books, const int64_t* parents,
                            const int64_t* children, int64_t requests, int32_t* status, int32_t* workspace,
                            hipStream_t stream) {
    hipLaunchKernelGGL(page_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, books, parents, children,
                       requests, status, workspace);
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess) return launched;
    const dim3 grid(static_cast<uint32_t>(requests), static_cast<uint32_t>(1 + 2 * pool.layers));
    FLUX_BY_UNIT(rows_of(pool, 16), pool.element, page_fork_kernel, grid, pool, books, parents, children, requests,
                 workspace);
}

hipError_t launch_page_compact(const PagePool& pool, const PageBooks& books, int32_t* page_map, int64_t* used,
                               int32_t* workspace, hipStream_t stream) {
    hipLaunchKernelGGL(page_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, books.refcounts, pool.pages,
                       page_map, used, workspace);
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess) return launched;
    const dim3 grid(2048);
    FLUX_BY_UNIT(rows_of(pool, 16), pool.element, page_compact_kernel, grid, pool, books, page_map, workspace);
}

hipError_t launch_page_write(const PagePool& pool, const PageWriteArgs& args, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>((args.tokens + kWriteTokens - 1) / kWriteTokens),
                    static_cast<uint32_t>(args.requests));
    FLUX_BY_UNIT(rows_of(pool, 16) && rows_of(args, pool.element, 16), pool.element, page_write_kernel, grid, pool,
                 args);
}

#undef FLUX_BY_UNIT

}  // namespace flux
