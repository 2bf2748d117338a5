// Pages of a K/V cache: reserving, writing, copying, forking, freeing and compacting them without the host.
//
// The books are a page table [slots, columns] (-1: no page), the slots' lengths and a count of holders per page (0:
// free).  A page that is needed is always the lowest free one, and requests are served in their order, so that
// results do not depend on scheduling.  Every operator is one launch of bookkeeping, or one and a copy over the whole
// card: the bookkeeping is a few KB and bound by the latency of dependent reads (16 prompts reserved in 8.7 us, 64 forks
// planned in 7.5), the copies by HBM (40 pages of 30 layers, 59 MB moved, in 11.8 us).
#include "serving.h"

#include <type_traits>

namespace flux {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

// Values that other threads of this workgroup wrote: past the L1, because some of them come from atomics.
__device__ __forceinline__ int32_t load_shared_word(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared_word(int32_t* p, int32_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
    __syncthreads();
    return found < wanted ? found : wanted;
}

// Marks the first request that names each slot: first[slot] == i afterwards exactly for that one.
__device__ void mark_first(const int64_t* list, int64_t requests, int64_t slots, int32_t* first) {
    for (int64_t i = threadIdx.x; i < requests; i += kPlanThreads) {
        const int64_t slot = list[i];
        if (slot >= 0 && slot < slots) store_shared_word(first + slot, 0x7fffffff);
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < requests; i += kPlanThreads) {
        const int64_t slot = list[i];
        if (slot >= 0 && slot < slots) atomicMin(first + slot, static_cast<int32_t>(i));
    }
    __syncthreads();
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
    __syncthreads();
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
    __syncthreads();
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
// `rows` rows of each head of one page of one layer, keys and values.  Unit: 16 bytes where every row allows it.  Units
// are numbered by row, head and place in the row, or by their address where a whole page lies in one run; every thread
// requests kAhead of them before it writes any.
constexpr int kAhead = 4;

// Past the caches in units of 16 bytes (40 pages of 30 layers, 29 MB: 22.0 us a call through the caches, 12.9 past
// them; 12 MB of new rows: 13.8 and 8.8; 1920 partial pages, 12 MB: 23.3 and 8.6).
template <class Unit>
__device__ __forceinline__ void store_unit(char* to, const Unit& held) {
    if constexpr (sizeof(Unit) == 16) store_past_caches(to, held);
    else *reinterpret_cast<Unit*>(to) = held;
}

template <class Unit>
struct PageRows {
    const PagePool& p;
    const char* from[2];  // key, value
    char* to[2];
    int units;
    bool run;

    __device__ __forceinline__ PageRows(const PagePool& pool, int64_t layer, int64_t source, int64_t target, int rows) : p(pool) {
        units = rows * static_cast<int>(p.row_units.divisor * p.of_heads.divisor);
        run = rows == p.page;
        char* base[2] = {p.key, p.value};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int64_t* strides = s ? p.value_strides : p.key_strides;
            from[s] = base[s] + (layer * strides[0] + source * strides[1]) * p.element;
            to[s] = base[s] + (layer * strides[0] + target * strides[1]) * p.element;
            run = run && strides[3] == p.dim && strides[2] == p.page * p.dim;
        }
    }
    __device__ __forceinline__ int64_t offset(int unit, int s) const {
        if (run) return static_cast<int64_t>(unit) * sizeof(Unit);
        const uint32_t line = divide(unit, p.row_units), row = divide(line, p.of_heads);
        const int64_t* strides = s ? p.value_strides : p.key_strides;
        return ((line - row * p.of_heads.divisor) * strides[2] + row * strides[3]) * p.element +
               (unit - line * p.row_units.divisor) * static_cast<int>(sizeof(Unit));
    }
    // Units first, first + 256, ... of one side.
    __device__ __forceinline__ void load(int s, int first, Unit (&held)[kAhead], int64_t (&at)[kAhead]) const {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            at[j] = offset(first + 256 * j, s);
            if (first + 256 * j < units) held[j] = *reinterpret_cast<const Unit*>(from[s] + at[j]);
        }
    }
    __device__ __forceinline__ void store(int s, int first, const Unit (&held)[kAhead], const int64_t (&at)[kAhead]) const {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (first + 256 * j < units) store_unit(to[s] + at[j], held[j]);
    }
    __device__ __forceinline__ void copy_side(int s, int first) const {
        for (; first < units; first += kAhead * 256) {
            Unit held[kAhead];
            int64_t at[kAhead];
            load(s, first, held, at);
            store(s, first, held, at);
        }
    }
    __device__ __forceinline__ void copy_from(int first) const {
        for (; first < units; first += kAhead * 256) {
            Unit key[kAhead], value[kAhead];
            int64_t key_at[kAhead], value_at[kAhead];
            load(0, first, key, key_at);
            load(1, first, value, value_at);
            store(0, first, key, key_at);
            store(1, first, value, value_at);
        }
    }
};

// Copy.  Workgroup (request, layer).  Every workgroup of a request looks through the lists for the conflicts that would make
// its result depend on the order, while the first rows are on their way.
template <class Unit>
__global__ void __launch_bounds__(256) page_copy_kernel(PagePool p, const int64_t* __restrict__ source,
                                                        const int64_t* __restrict__ target, int64_t requests,
                                                        int32_t* status) {
    const int64_t i = blockIdx.x;
    const int64_t from = source[i], to = target[i];
    if (from < 0 || from >= p.pages || to < 0 || to >= p.pages) {
        if (blockIdx.y == 0 && threadIdx.x == 0) status[i] = kPageOutOfRange;
        return;
    }
    const PageRows<Unit> rows(p, blockIdx.y, from, to, static_cast<int>(p.page));
    Unit key[kAhead], value[kAhead];
    int64_t key_at[kAhead], value_at[kAhead];
    rows.load(0, threadIdx.x, key, key_at);
    rows.load(1, threadIdx.x, value, value_at);
    int clash = 0;
    for (int64_t j = threadIdx.x; j < requests; j += 256)
        clash |= (j < i && target[j] == to) || (j != i && source[j] == to);
    clash = __syncthreads_or(clash);
    if (blockIdx.y == 0 && threadIdx.x == 0) status[i] = clash ? kPageRepeated : kPageDone;
    if (clash || from == to) return;
    rows.store(0, threadIdx.x, key, key_at);
    rows.store(1, threadIdx.x, value, value_at);
    rows.copy_from(threadIdx.x + kAhead * 256);
}

// ---------------------------------------------------------------------------
// Fork.  The plan reads the books as they were; the second launch shares full pages and copies partial ones.
struct ForkPlan {
    int32_t* first_request;  // [slots]
    int32_t* need;           // [requests]
    int32_t* list;           // [pages]
    int32_t* length;         // [requests]: tokens of the parent, -1: refused
    int32_t* fresh;          // [requests]: new page of the partial rows
    int32_t* last;           // [requests]: the parent's page that holds them
};

__device__ __host__ ForkPlan fork_plan(int32_t* workspace, int64_t requests, int64_t slots, int64_t pages) {
    ForkPlan f;
    f.first_request = workspace;
    f.need = f.first_request + slots;
    f.list = f.need + requests;
    f.length = f.list + pages;
    f.fresh = f.length + requests;
    f.last = f.fresh + requests;
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
    __syncthreads();
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
        if (fresh >= 0) f.last[i] = b.table[parents[i] * b.table_stride + length / b.page];
        status[i] = result;
    }
}

// Workgroup (request, part): part 0 writes the child's books, part 1 + layer copies partial rows.
template <class Unit>
__global__ void __launch_bounds__(256) page_fork_kernel(PagePool p, PageBooks b, const int64_t* __restrict__ parents,
                                                        const int64_t* __restrict__ children, int64_t requests,
                                                        int32_t* workspace) {
    const ForkPlan f = fork_plan(workspace, requests, b.slots, b.pages);
    const int64_t i = blockIdx.x;
    const int64_t length = f.length[i];
    const int32_t fresh = f.fresh[i], last = f.last[i];  // together: last holds nothing where fresh is -1
    if (length < 0) return;
    if (blockIdx.y == 0) {
        const int64_t full = length / b.page;
        // A parent that is itself a child of this call was empty: none of its columns is read.
        const int32_t* from = b.table + parents[i] * b.table_stride;
        int32_t* to = b.table + children[i] * b.table_stride;
        for (int64_t c = threadIdx.x; c < full; c += 256) {
            const int32_t page = from[c];
            to[c] = page;
            atomicAdd(b.refcounts + page, 1);
        }
        if (threadIdx.x == 0) {
            if (fresh >= 0) to[full] = fresh;
            b.lengths[children[i]] = length;
        }
    } else if (fresh >= 0) {
        PageRows<Unit>(p, blockIdx.y - 1, last, fresh, static_cast<int>(length % b.page)).copy_from(threadIdx.x);
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
    __syncthreads();
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
    const int64_t parts = 2 * p.layers, units = *plan.moves * parts;
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t k = unit / parts, part = unit % parts;
        PageRows<Unit>(p, part >> 1, plan.source[k], plan.target[k], static_cast<int>(p.page)).copy_side(part & 1, threadIdx.x);
    }
}

// ---------------------------------------------------------------------------
// Write.  Workgroup (tokens, request): rows of kWriteTokens new tokens, all heads, keys then values.  The tokens' places are
// looked up once; every thread requests kAhead units before it writes any.
constexpr int kWriteTokens = 16;

// Two forms of the arguments: a padded batch whose places are looked up, and packed tokens whose rows of the pool are given (row
// r is row r % page of page r / page).  16384 packed tokens of 8 heads of 128 in 16 bits take 24 us, 5.7 TB/s read and written (partly
// out of the memory-side cache); 16 tokens 3.9.  Both forms in one kernel, because a loop that two of them call takes 81 registers
// instead of 67, five waves instead of seven (16 prompts to 1000 tokens 9.7 us against 8.6).
template <class Unit, class Args>
__global__ void __launch_bounds__(256) page_write_kernel(PagePool p, Args a) {
    constexpr int kBytes = sizeof(Unit);
    constexpr bool kPacked = std::is_same_v<Args, PageRowsArgs>;
    constexpr int kHead = 1, kToken = kPacked ? 0 : 2;  // strides
    __shared__ int64_t place[2][kWriteTokens];  // bytes from the pool's start, -1: no page
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kWriteTokens;
    int64_t i = 0, count = a.tokens, page = -1, row = 0;
    if constexpr (!kPacked) {
        i = blockIdx.y;
        const int64_t slot = a.slot_list[i], start = a.positions[i];
        if (slot < 0 || slot >= a.slots || start < 0) return;
        if (a.counts) count = a.counts[i];
        if (count > a.tokens) count = a.tokens;
        const int64_t capacity = a.columns * p.page;
        if (start >= capacity) return;
        if (count > capacity - start) count = capacity - start;
        if (t0 >= count) return;
        if (static_cast<int>(threadIdx.x) < kWriteTokens && t0 + static_cast<int>(threadIdx.x) < count) {
            const uint32_t position = static_cast<uint32_t>(start + t0 + threadIdx.x), rows = static_cast<uint32_t>(p.page);
            page = a.table[slot * a.table_stride + position / rows];
            row = position % rows;
        }
    } else if (static_cast<int>(threadIdx.x) < kWriteTokens && t0 + static_cast<int>(threadIdx.x) < count) {
        const int64_t of = a.rows[t0 + threadIdx.x];
        page = of < 0 ? -1 : of / p.page;
        row = of - page * p.page;
    }
    const int tokens = static_cast<int>(count - t0 < kWriteTokens ? count - t0 : kWriteTokens);
    if (static_cast<int>(threadIdx.x) < tokens) {
        const bool held = page >= 0 && page < p.pages;
        place[0][threadIdx.x] = held ? (page * p.key_strides[1] + row * p.key_strides[3]) * p.element : -1;
        place[1][threadIdx.x] = held ? (page * p.value_strides[1] + row * p.value_strides[3]) * p.element : -1;
    }
    __syncthreads();
    const uint32_t width = p.row_units.divisor, heads = p.of_heads.divisor;
    const int side = static_cast<int>(tokens * heads * width);
    const char* sources[2] = {a.key + ((kPacked ? 0 : i * a.key_strides[0]) + t0 * a.key_strides[kToken]) * p.element,
                              a.value + ((kPacked ? 0 : i * a.value_strides[0]) + t0 * a.value_strides[kToken]) * p.element};
    constexpr int kEach = 2 * kAhead;
    for (int first = threadIdx.x; first < 2 * side; first += kEach * 256) {
        Unit held[kEach];
        char* to[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int unit = first + 256 * j, s = unit >= side;
            to[j] = nullptr;
            if (unit >= 2 * side) continue;
            const uint32_t at = unit - s * side, row = divide(at, p.row_units), u = at - row * width;
            const uint32_t t = divide(row, p.of_heads), head = row - t * heads;
            const int64_t where = place[s][t];
            if (where < 0) continue;
            to[j] = (s ? p.value : p.key) + where + head * (s ? p.value_strides : p.key_strides)[2] * p.element + u * kBytes;
            held[j] = *reinterpret_cast<const Unit*>((s ? sources[1] : sources[0]) +
                                                     (head * (s ? a.value_strides : a.key_strides)[kHead] +
                                                      t * (s ? a.value_strides : a.key_strides)[kToken]) * p.element + u * kBytes);
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (to[j]) store_unit(to[j], held[j]);
    }
}

// ---------------------------------------------------------------------------
// Layout.  The tokens of a step lie packed one request after the other, and each workgroup places kPlanThreads of them: it
// sums the requests' counts itself (all of them up to its own last token; they are a few KB in the L2), so that one launch
// does.  Sums stop at the number of tokens, which also keeps them in 32 bits.  Bound by latency: 4.8 us for 1024 requests, 2.9 for 4.
__device__ __forceinline__ int saturating_scan(int v, int most) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int below = __shfl_up(v, step, kWave);
        if (lane >= step) v = v + below < most ? v + below : most;
    }
    return v;
}

__global__ void __launch_bounds__(kPlanThreads) step_layout_kernel(StepLayoutArgs a) {
    __shared__ int sums[kPlanWaves];
    __shared__ int ends[kPlanThreads];
    const int wave = threadIdx.x >> 6, most = static_cast<int>(a.tokens);
    const int token = static_cast<int>(blockIdx.x) * kPlanThreads + static_cast<int>(threadIdx.x);
    const int last = static_cast<int>(blockIdx.x) * kPlanThreads + kPlanThreads - 1;
    int running = 0, request = -1, first = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[0] = 0;
    for (int base = 0; base < a.requests && (blockIdx.x == 0 || running <= last); base += kPlanThreads) {
        const int i = base + static_cast<int>(threadIdx.x);
        int64_t count = 0;
        if (i < a.requests) {
            count = a.counts ? a.counts[i] : 1;
            const int64_t slot = a.slots[i];
            if (a.positions[i] < 0 || slot < 0 || slot >= a.slot_count || count < 0) count = 0;
        }
        int end = saturating_scan(static_cast<int>(count < most ? count : most), most);
        if ((threadIdx.x & 63) == 63) sums[wave] = end;
        __syncthreads();
        int before = running;
        for (int w = 0; w < wave; ++w) before = before + sums[w] < most ? before + sums[w] : most;
        end = before + end < most ? before + end : most;
        ends[threadIdx.x] = end;
        if (blockIdx.x == 0 && i < a.requests) a.offsets[i + 1] = end;
        __syncthreads();
        const int reached = ends[kPlanThreads - 1];
        if (token >= running && token < reached) {  // the first request that ends behind the token
            int low = 0;
#pragma unroll
            for (int step = kPlanThreads / 2; step >= 1; step /= 2)
                if (ends[low + step - 1] <= token) low += step;
            request = base + low;
            first = low ? ends[low - 1] : running;
        }
        running = reached;
    }
    if (token >= most) return;
    int64_t position = -1, row = -1;
    if (request >= 0) {
        position = static_cast<int64_t>(static_cast<uint64_t>(a.positions[request]) + static_cast<uint64_t>(token - first));
        if (position >= 0 && position < a.columns * a.page) {
            const uint32_t column = static_cast<uint32_t>(position) / static_cast<uint32_t>(a.page);
            const int64_t page = a.table[a.slots[request] * a.table_stride + column];
            if (page >= 0) row = page * a.page + (position - column * a.page);
        }
    }
    a.token_requests[token] = request;
    a.token_positions[token] = position;
    a.token_rows[token] = row;
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

bool rows_of(const PageRowsArgs& a, int element, int64_t bytes) {
    if (reinterpret_cast<uintptr_t>(a.key) % bytes || reinterpret_cast<uintptr_t>(a.value) % bytes) return false;
    for (int i = 0; i < 2; ++i)
        if (a.key_strides[i] * element % bytes || a.value_strides[i] * element % bytes) return false;
    return true;
}

}  // namespace

size_t page_reserve_workspace(int64_t requests, int64_t slots, int64_t pages) { return requests + slots + pages; }
size_t page_fork_workspace(int64_t requests, int64_t slots, int64_t pages) { return 4 * requests + slots + pages; }
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
PagePool with_units(PagePool pool, bool wide) {
    pool.unit = wide ? 16 : pool.element;
    pool.row_units = make_divider(static_cast<uint32_t>(pool.dim * pool.element / pool.unit));
    pool.of_heads = make_divider(static_cast<uint32_t>(pool.heads));
    return pool;
}

#define FLUX_BY_UNIT(pool, kernel, grid, ...)                                                                       \
    if ((pool).unit == 16)                                                                                          \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(kernel<Quad>), grid, dim3(256), 0, stream, pool, __VA_ARGS__);          \
    else if ((pool).unit == 4)                                                                                      \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(kernel<uint32_t>), grid, dim3(256), 0, stream, pool, __VA_ARGS__);       \
    else                                                                                                            \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(kernel<uint16_t>), grid, dim3(256), 0, stream, pool, __VA_ARGS__);       \
    return hipGetLastError()

hipError_t launch_page_copy(const PagePool& plain, const int64_t* source, const int64_t* target, int64_t requests,
                            int32_t* status, hipStream_t stream) {
    const PagePool pool = with_units(plain, rows_of(plain, 16));
    const dim3 grid(static_cast<uint32_t>(requests), static_cast<uint32_t>(pool.layers));
    FLUX_BY_UNIT(pool, page_copy_kernel, grid, source, target, requests, status);
}

hipError_t launch_page_fork(const PagePool& plain, const PageBooks& books, const int64_t* parents,
                            const int64_t* children, int64_t requests, int32_t* status, int32_t* workspace,
                            hipStream_t stream) {
    hipLaunchKernelGGL(page_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, books, parents, children,
                       requests, status, workspace);
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess) return launched;
    const PagePool pool = with_units(plain, rows_of(plain, 16));
    const dim3 grid(static_cast<uint32_t>(requests), static_cast<uint32_t>(1 + pool.layers));
    FLUX_BY_UNIT(pool, page_fork_kernel, grid, books, parents, children, requests,
                 workspace);
}

hipError_t launch_page_compact(const PagePool& plain, const PageBooks& books, int32_t* page_map, int64_t* used,
                               int32_t* workspace, hipStream_t stream) {
    hipLaunchKernelGGL(page_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, books.refcounts, plain.pages,
                       page_map, used, workspace);
    const hipError_t launched = hipGetLastError();
    if (launched != hipSuccess) return launched;
    const PagePool pool = with_units(plain, rows_of(plain, 16));
    const dim3 grid(8192);
    FLUX_BY_UNIT(pool, page_compact_kernel, grid, books, page_map, workspace);
}

hipError_t launch_page_write(const PagePool& plain, const PageWriteArgs& args, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>((args.tokens + kWriteTokens - 1) / kWriteTokens),
                    static_cast<uint32_t>(args.requests));
    const PagePool pool = with_units(plain, rows_of(plain, 16) && rows_of(args, plain.element, 16));
    FLUX_BY_UNIT(pool, page_write_kernel, grid, args);
}

hipError_t launch_page_write_rows(const PagePool& plain, const PageRowsArgs& args, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>((args.tokens + kWriteTokens - 1) / kWriteTokens));
    const PagePool pool = with_units(plain, rows_of(plain, 16) && rows_of(args, plain.element, 16));
    FLUX_BY_UNIT(pool, page_write_kernel, grid, args);
}

#undef FLUX_BY_UNIT

hipError_t launch_step_layout(const StepLayoutArgs& args, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>((args.tokens + kPlanThreads - 1) / kPlanThreads));
    hipLaunchKernelGGL(step_layout_kernel, grid, dim3(kPlanThreads), 0, stream, args);
    return hipGetLastError();
}

}  // namespace flux
