// kv_pages.cu -- writing new tokens into the pages of a cache, and giving,
// sharing, taking back and moving pages.
//
// The tables (pages of each slot, tokens of each slot, references of each page)
// live on the device, so a serving loop changes them between two steps without
// reading anything back. One block (or one cluster of blocks) plans a change: it checks every slot, page
// and length that the change touches, and only when all are sound writes the
// tables; else it records a device status and changes nothing. Free pages are
// taken in ascending order, so results do not depend on scheduling. What is to
// be copied goes into a list in the workspace, and a second kernel copies it for
// all layers: whole 16-byte words of K and V, bound by HBM.
// Measured: compaction that moves 240 pages of 32 layers 180 us (1.0 GB; the plan
// takes 7 us of them, the copies run at 6 TB/s); free, fork and reserve of seven
// slots of up to 44 pages 19 us for the four launches, which are chains of dependent
// reads by one block; reordering the beams of 32 sequences of 4 (32 layers, 50 to 400
// tokens) 35 us, 19 of them the copies (117 MB, 6.2 TB/s) and 14 the plan, of one
// sequence 14 us; the cache write of 5296 tokens (32 heads) 67.8 us
// (437 MB, 6.4 TB/s), of 32 tokens (64 heads on 8) 3.4 us.
#include "paged.h"
#include "abi_errors.h"
#include "qmatvec.h"
#include "trace.h"

#include <algorithm>

namespace hesa_cuda {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxSlots = 65536;

// Reordering n slots is planned by one block up to this many table entries (n times max_pages),
// and by a cluster of kPlanBlocks beyond: 32 slots of 126 entries 19.7 us (cluster 21.0), 64 of
// them 24.6 (22.5), 128 of them 33 (25), 576 of 251 170 (50; a cluster of four 75). The barriers
// and the start of a cluster cost 3 us of the smallest call.
constexpr int kPlanBlocks = 8;
constexpr int64_t kMostEntries = 6000;

struct Tables {
    int32_t* table;      // [n_slots][max_pages]
    int32_t* seq_len;    // [n_slots]
    int32_t* refs;       // [n_pages]
    int32_t n_slots, max_pages, n_pages, page_size;
    int* status;
};

// Workspace of the page operations, in int32: [0] items of the copy list, then
// three words for each item (page from, page to, slots), then new_of[n_pages]
// and a scratch list.
struct PageWork {
    int32_t* n_items;
    int32_t* items;      // [max(n_pages, n_slots)][3]
    int32_t* map;        // [n_pages]
    int32_t* list;       // [max(n_pages, n_slots)]
    int32_t* start;      // [n_slots + 1]
};

__host__ __device__ inline int64_t most_items(int32_t n_pages, int32_t n_slots) { return n_pages > n_slots ? n_pages : n_slots; }

template <typename KV>
PageWork page_work(void* ws, const KV* kv) {
    const int64_t most = most_items(kv->n_pages, kv->n_slots);
    PageWork w;
    w.n_items = static_cast<int32_t*>(ws);
    w.items = w.n_items + 4;
    w.map = w.items + 3 * most;
    w.list = w.map + kv->n_pages;
    w.start = w.list + most;
    return w;
}

__device__ __forceinline__ int pages_for(int32_t len, int32_t page) { return (len + page - 1) / page; }

// Sum of x over the block before this thread (exclusive) and the block's total.
// Two block-wide barriers; s must hold 33 words.
__device__ __forceinline__ int block_scan(int x, int* s, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warp = blockDim.x >> 5;
    int v = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    if (lane == 31) s[warp] = v;
    __syncthreads();
    const int y = lane < n_warp ? s[lane] : 0;
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
    total = __reduce_add_sync(0xffffffffu, y);
    __syncthreads();
    return before + v - x;
}

// The lowest `want` free pages into list, ascending; false when there are fewer. A thread looks at several
// pages side by side: a pass over the block costs a read's latency, a scan and three barriers.
constexpr int kFreeAhead = 8;

__device__ bool lowest_free(const Tables& t, int want, int32_t* list, int* s) {
    int found = 0;
    for (int64_t b = 0; b < t.n_pages && found < want; b += kPlanThreads * kFreeAhead) {
        const int64_t first = b + threadIdx.x * kFreeAhead;
        uint32_t is_free = 0;
#pragma unroll
        for (int k = 0; k < kFreeAhead; ++k)
            if (first + k < t.n_pages && t.refs[first + k] == 0) is_free |= 1u << k;
        int total;
        int at = found + block_scan(__popc(is_free), s, total);
        for (; is_free && at < want; is_free &= is_free - 1) list[at++] = static_cast<int32_t>(first) + __ffs(is_free) - 1;
        found += total;
    }
    __syncthreads();
    return found >= want;
}

// Every listed slot in range and listed once: marks them in bits (a word for 32 slots).
__device__ bool mark_slots(const int32_t* slots, int n, int n_slots, uint32_t* bits) {
    bool bad = false;
    for (int i = threadIdx.x; i < (n_slots + 31) / 32; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = slots[i];
        if (s < 0 || s >= n_slots) {
            bad = true;
            continue;
        }
        bad |= (atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1u;
    }
    return !__syncthreads_or(bad);
}

// A slot's length and pages are sound (a warp's lanes share the pages).
__device__ bool slot_sound(const Tables& t, int slot, int lane) {
    const int len = t.seq_len[slot];
    if (len < 0 || len > static_cast<int64_t>(t.max_pages) * t.page_size) return false;
    bool ok = true;
    const int n = pages_for(len, t.page_size);
    for (int j = lane; j < n; j += 32) {
        const int p = t.table[static_cast<int64_t>(slot) * t.max_pages + j];
        ok &= p >= 0 && p < t.n_pages && t.refs[p] > 0;
    }
    return __all_sync(0xffffffffu, ok);
}

__device__ bool slots_sound(const Tables& t, const int32_t* slots, int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool bad = false;
    for (int i = warp; i < n; i += kPlanThreads / 32) bad |= !slot_sound(t, slots[i], lane);
    return !__syncthreads_or(bad);
}

// One reference more or less for every page of the slots; false where a length or a
// page is not sound (what is not has no reference changed, so that the opposite call
// undoes this one), or a page had no reference left to take. All threads of the
// block; a barrier at its end.
__device__ bool add_refs(const Tables& t, const int32_t* slots, int n, int by) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool bad = false;
    for (int i = warp; i < n; i += kPlanThreads / 32) {
        const int len = t.seq_len[slots[i]];
        if (len < 0 || len > static_cast<int64_t>(t.max_pages) * t.page_size) {
            bad = true;
            continue;
        }
        const int np = pages_for(len, t.page_size);
        const int32_t* row = t.table + static_cast<int64_t>(slots[i]) * t.max_pages;
        for (int j = lane; j < np; j += 32) {
            const int p = row[j];
            if (p < 0 || p >= t.n_pages) bad = true;
            else bad |= atomicAdd(&t.refs[p], by) + by < 0;
        }
    }
    return !__syncthreads_or(bad);
}

__device__ __forceinline__ void refuse(const Tables& t, int code) {
    if (threadIdx.x == 0) record_status(t.status, code);
}

__global__ void __launch_bounds__(kPlanThreads)
free_kernel(const Tables t, const int32_t* slots, int n) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ uint32_t bits[kMaxSlots / 32];
    if (!mark_slots(slots, n, t.n_slots, bits)) return refuse(t, kStatusBadPosition);
    // A page that the slots hold more often than it has references would end below
    // zero: the references are taken, and given back if one was not there.
    if (!add_refs(t, slots, n, -1)) {
        add_refs(t, slots, n, 1);
        return refuse(t, kStatusBadPosition);
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = warp; i < n; i += kPlanThreads / 32) {
        const int s = slots[i];
        const int np = pages_for(t.seq_len[s], t.page_size);
        for (int j = lane; j < np; j += 32) t.table[static_cast<int64_t>(s) * t.max_pages + j] = -1;
        __syncwarp();
        if (lane == 0) t.seq_len[s] = 0;
    }
}

__global__ void __launch_bounds__(kPlanThreads)
reserve_kernel(const Tables t, const int32_t* slots, const int32_t* add, int n, PageWork w) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ uint32_t bits[kMaxSlots / 32];
    __shared__ int s[33];
    if (!mark_slots(slots, n, t.n_slots, bits)) return refuse(t, kStatusBadPosition);
    bool bad = false;
    int total = 0;
    for (int b = 0; b < n; b += kPlanThreads) {
        const int i = b + threadIdx.x;
        int need = 0;
        if (i < n) {
            const int64_t len = t.seq_len[slots[i]], a = add[i];
            if (len < 0 || a < 0 || len + a > static_cast<int64_t>(t.max_pages) * t.page_size) bad = true;
            else need = pages_for(static_cast<int32_t>(len + a), t.page_size) - pages_for(static_cast<int32_t>(len), t.page_size);
        }
        // a sum above n_pages is refused below; capped here so that it cannot wrap
        need = min(need, t.n_pages + 1);
        int all;
        const int at = block_scan(need, s, all);
        if (i < n) w.start[i] = total + at;
        // 1024 needs of at most 2^20 + 1 pages each stay within 32 bits
        total = min(total + all, t.n_pages + 1);
    }
    if (__syncthreads_or(bad)) return refuse(t, kStatusBadPosition);
    if (total > t.n_pages || !lowest_free(t, total, w.list, s)) return refuse(t, kStatusNoPages);
    // page r of the list belongs to the last slot whose first page is at or before r
    for (int r = threadIdx.x; r < total; r += kPlanThreads) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (w.start[mid] <= r) lo = mid;
            else hi = mid - 1;
        }
        const int slot = slots[lo], p = w.list[r];
        t.table[static_cast<int64_t>(slot) * t.max_pages + pages_for(t.seq_len[slot], t.page_size) + r - w.start[lo]] = p;
        t.refs[p] = 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) t.seq_len[slots[i]] += add[i];
}

__global__ void __launch_bounds__(kPlanThreads)
fork_plan_kernel(const Tables t, const int32_t* src, const int32_t* dst, int n, PageWork w) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ uint32_t bits[kMaxSlots / 32];
    __shared__ int s[33];
    if (threadIdx.x == 0) *w.n_items = 0;
    bool bad = !mark_slots(dst, n, t.n_slots, bits);
    for (int i = threadIdx.x; i < n && !bad; i += kPlanThreads) {
        const int a = src[i];
        // a source outside the table, or one that is itself a target; a target in use
        bad = a < 0 || a >= t.n_slots || ((bits[a >> 5] >> (a & 31)) & 1u) || t.seq_len[dst[i]] != 0;
    }
    if (__syncthreads_or(bad) || !slots_sound(t, src, n)) return refuse(t, kStatusBadPosition);
    int total = 0;
    for (int b = 0; b < n; b += kPlanThreads) {
        const int i = b + threadIdx.x;
        int all;
        const int at = block_scan(i < n && t.seq_len[src[i]] % t.page_size != 0 ? 1 : 0, s, all);
        if (i < n) w.start[i] = total + at;
        total += all;
    }
    if (total > t.n_pages || !lowest_free(t, total, w.list, s)) return refuse(t, kStatusNoPages);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = warp; i < n; i += kPlanThreads / 32) {
        const int len = t.seq_len[src[i]], full = len / t.page_size, tail = len % t.page_size;
        const int32_t* from = t.table + static_cast<int64_t>(src[i]) * t.max_pages;
        int32_t* to = t.table + static_cast<int64_t>(dst[i]) * t.max_pages;
        for (int j = lane; j < full; j += 32) {
            const int p = from[j];
            to[j] = p;
            atomicAdd(&t.refs[p], 1);
        }
        if (lane == 0) {
            int32_t* item = w.items + 3 * static_cast<int64_t>(i);
            item[2] = 0;
            if (tail) {
                const int p = w.list[w.start[i]];
                to[full] = p;
                t.refs[p] = 1;
                item[0] = from[full];
                item[1] = p;
                item[2] = tail;
            }
            t.seq_len[dst[i]] = len;
        }
    }
    if (threadIdx.x == 0) *w.n_items = n;
}

// The blocks that plan together: one, or a cluster. `mine` of `all` warps.
template <int BLOCKS> struct Team {
    int rank, mine;
    static constexpr int all = kPlanThreads / 32 * BLOCKS;
    int* flags;   // a word for each vote, zeros, in every block
    __device__ explicit Team(int* votes) : rank(BLOCKS > 1 ? blockIdx.x : 0), mine(rank * (kPlanThreads / 32) + (threadIdx.x >> 5)), flags(votes) {}
    __device__ __forceinline__ void sync() const {
        if constexpr (BLOCKS > 1) cluster_sync();
        else __syncthreads();
    }
    // x of any thread; what they wrote before is seen after it
    __device__ __forceinline__ bool any(bool x, int vote) const {
        x = __syncthreads_or(x);
        if constexpr (BLOCKS > 1) {
            if (x && threadIdx.x < BLOCKS) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_block(flags + vote, threadIdx.x)), "r"(1) : "memory");
            cluster_sync();
            x = *static_cast<volatile int*>(flags + vote) != 0;
        }
        return x;
    }
};

// The pages of the listed slots, by what becomes of them. kDrop: those of slots that no
// slot takes over lose a reference each; kGiveBack undoes that (what is not sound has
// no reference changed); kKept: those of the other slots have references left. True
// where a length or a page is not sound, or there is no reference to take or left.
// A warp takes kSlotsAhead slots at a time, whose reads go side by side, its lanes
// their pages; with few slots 2^share warps have a slot.
enum Refs { kDrop, kGiveBack, kKept };
constexpr int kSlotsAhead = 4;

template <Refs MODE, typename T>
__device__ bool slot_refs(const Tables& t, const T& team, int share, const int32_t* slots, const int32_t* parents, int n, int width) {
    const int lane = threadIdx.x & 31, step = T::all >> share, cols = 32 << share, col = (team.mine * 32 + lane) & (cols - 1);
    bool bad = false;
    auto look = [&](int p, bool mine) {
        if (p < 0 || p >= t.n_pages) bad = true;
        else if (!mine) return;
        else if (MODE == kDrop) bad |= atomicAdd(&t.refs[p], -1) <= 0;
        else if (MODE == kGiveBack) atomicAdd(&t.refs[p], 1);
        else bad |= t.refs[p] <= 0;
    };
    for (int i0 = team.mine >> share; i0 < n; i0 += kSlotsAhead * step) {
        const int32_t* row[kSlotsAhead];
        uint32_t np[kSlotsAhead];
        int first[kSlotsAhead];
        bool mine[kSlotsAhead];
#pragma unroll
        for (int k = 0; k < kSlotsAhead; ++k) {
            const int i = i0 + k * step, b = i % width;
            const int slot = i < n ? slots[i] : 0, par = i < n && lane < width ? parents[i - b + lane] : -1;
            const int len = i < n ? t.seq_len[slot] : 0;
            const bool ok = len >= 0 && len <= static_cast<int64_t>(t.max_pages) * t.page_size;
            bad |= !ok;
            np[k] = ok ? pages_for(len, t.page_size) : 0;
            row[k] = t.table + static_cast<int64_t>(slot) * t.max_pages;
            mine[k] = __any_sync(0xffffffffu, par == b) == (MODE == kKept);
        }
#pragma unroll
        for (int k = 0; k < kSlotsAhead; ++k) first[k] = col < np[k] ? row[k][col] : 0;
#pragma unroll
        for (int k = 0; k < kSlotsAhead; ++k) {
            if (col < np[k]) look(first[k], mine[k]);
            for (uint32_t j = col + cols; j < np[k]; j += cols) look(row[k][j], mine[k]);
        }
    }
    return bad;
}

// Slot b of a group becomes what slot parents[b] of it was. References that go are taken first, so that the pages
// they free can be taken for the copies, then those that come are added. The table's entries of a group's columns are
// changed by one warp: a lane has one slot's in some columns, and a slot's new entries are the old ones of its parent's
// lane; a column is read before it is written, by the same warp. Bound by latency: a chain of dependent reads.
constexpr int kColumnSteps = 8;   // reads of a row that a lane has under way

template <int BLOCKS>
__global__ void __launch_bounds__(kPlanThreads)
reorder_plan_kernel(const Tables t, const int32_t* slots, const int32_t* parents, int n, int width, int slot_share, int group_share, PageWork w) {
    __shared__ uint32_t bits[kMaxSlots / 32];
    __shared__ int s[33], votes[4];
    const Team<BLOCKS> team(votes);
    if (BLOCKS > 1) {
        if (threadIdx.x < 4) votes[threadIdx.x] = 0;
        team.sync();   // every block is there, with its votes at 0
    }
    grid_dep_wait();
    grid_dep_launch();
    const bool lead = team.rank == 0;
    if (lead && threadIdx.x == 0) *w.n_items = 0;
    bool bad = !mark_slots(slots, n, t.n_slots, bits);   // each block all of them, and the parents
    for (int i = threadIdx.x; i < n && !bad; i += kPlanThreads) bad = parents[i] < 0 || parents[i] >= width;
    const bool listed = !__syncthreads_or(bad);
    if (team.any(!listed || slot_refs<kDrop>(t, team, slot_share, slots, parents, n, width), 0) ||
        team.any(slot_refs<kKept>(t, team, slot_share, slots, parents, n, width), 1)) {
        if (listed) slot_refs<kGiveBack>(t, team, slot_share, slots, parents, n, width);
        if (lead) refuse(t, kStatusBadPosition);
        return;
    }
    // a slot whose parent has a partly filled page and an earlier child gets a page of its own
    int total = 0;
    if (lead) {
        for (int b = 0; b < n; b += kPlanThreads) {
            const int i = b + threadIdx.x;
            bool copy = false;
            if (i < n) {
                const int g = i - i % width, par = parents[i];
                for (int x = g; x < i; ++x) copy |= parents[x] == par;
                copy = copy && t.seq_len[slots[g + par]] % t.page_size != 0;
            }
            int all;
            const int at = block_scan(copy ? 1 : 0, s, all);
            if (i < n) w.start[i] = copy ? total + at : -1;
            total += all;
        }
        bad = total > t.n_pages || !lowest_free(t, total, w.list, s);
    }
    if (team.any(bad, 2)) {
        slot_refs<kGiveBack>(t, team, slot_share, slots, parents, n, width);
        if (lead) refuse(t, kStatusNoPages);
        return;
    }
    const int lane = threadIdx.x & 31, cols = 32 / width;   // columns of the table a warp has in hand at a time
    const int part = team.mine & ((1 << group_share) - 1), step = kColumnSteps * cols;   // of the 2^group_share warps of a group
    const int beam = lane % width, col = lane / width;
    int new_slot = -1, new_len = 0;
    for (int g = (team.mine >> group_share) * width; g < n; g += (team.all >> group_share) * width) {
        const int par = parents[g + beam], slot = slots[g + beam];
        const int old_len = t.seq_len[slot], len = __shfl_sync(0xffffffffu, old_len, par);
        const uint32_t old_pages = pages_for(old_len, t.page_size), pages = pages_for(len, t.page_size), full = len / t.page_size;
        const int take = w.start[g + beam], fresh = take >= 0 ? w.list[take] : -1;
        bool later = false;   // the parent has an earlier child
        for (int x = 0; x < beam; ++x) later |= parents[g + x] == par;
        int32_t* row = t.table + static_cast<int64_t>(slot) * t.max_pages;
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(old_pages, pages));
        for (uint32_t j0 = part * step; j0 < most; j0 += step << group_share) {
            int old[kColumnSteps];
#pragma unroll
            for (int k = 0; k < kColumnSteps; ++k) {
                const uint32_t j = j0 + k * cols + col;
                old[k] = col < cols && j < old_pages ? row[j] : -1;
            }
#pragma unroll
            for (int k = 0; k < kColumnSteps; ++k) {
                const uint32_t j = j0 + k * cols + col;
                const int from = __shfl_sync(0xffffffffu, old[k], col < cols ? col * width + par : lane);
                if (col >= cols || j >= most) continue;
                if (j < pages) {
                    const bool copy = j == full && fresh >= 0;
                    const int now = copy ? fresh : from;
                    if (now != old[k]) row[j] = now;
                    if (copy) {
                        int32_t* item = w.items + 3 * static_cast<int64_t>(take);
                        item[0] = from;
                        item[1] = fresh;
                        item[2] = len % t.page_size;
                        t.refs[fresh] = 1;
                    }
                    if (later && j < full) atomicAdd(&t.refs[from], 1);   // for every child but the first
                } else if (j < old_pages) {
                    row[j] = -1;
                }
            }
        }
        __syncwarp();
        if (col == 0 && part == 0) {
            if (group_share == 0) t.seq_len[slot] = len;
            else new_slot = slot, new_len = len;   // once the group's other warps have read it
        }
    }
    if (group_share > 0) {   // each warp has had one group at most
        team.sync();
        if (new_slot >= 0) t.seq_len[new_slot] = new_len;
    }
    if (lead && threadIdx.x == 0) *w.n_items = total;
}

// live pages to the front: free pages below n_live take the pages in use from n_live on
__global__ void __launch_bounds__(kPlanThreads)
compact_plan_kernel(const Tables t, PageWork w, int32_t* n_live_out) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int s[33];
    if (threadIdx.x == 0) *w.n_items = 0;
    // a table entry outside the pool, or of a page that is free, would be lost: nothing is moved then
    bool bad = false;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = warp; i < t.n_slots; i += kPlanThreads / 32) bad |= !slot_sound(t, i, lane);
    int mine = 0;
    for (int i = threadIdx.x; i < t.n_pages; i += kPlanThreads) {
        mine += t.refs[i] > 0;
        bad |= t.refs[i] < 0;
        w.map[i] = i;
    }
    int live;
    block_scan(mine, s, live);
    if (__syncthreads_or(bad)) return refuse(t, kStatusBadPosition);
    int holes = 0, movers = 0;
    for (int b = 0; b < t.n_pages; b += kPlanThreads) {
        const int i = b + threadIdx.x;
        const bool in = i < t.n_pages, used = in && t.refs[i] > 0;
        const bool hole = in && !used && i < live, mover = used && i >= live;
        int all;
        // both counts in one scan: holes in the low half, movers in the high half (1024 of each at most)
        const int at = block_scan((hole ? 1 : 0) | (mover ? 1 << 16 : 0), s, all);
        if (hole) w.items[3 * static_cast<int64_t>(holes + (at & 0xffff)) + 1] = i;
        if (mover) w.items[3 * static_cast<int64_t>(movers + (at >> 16))] = i;
        holes += all & 0xffff;
        movers += all >> 16;
    }
    __syncthreads();
    // as many holes below n_live as pages in use from it on
    for (int i = threadIdx.x; i < holes; i += kPlanThreads) {
        int32_t* item = w.items + 3 * static_cast<int64_t>(i);
        item[2] = t.page_size;
        w.map[item[0]] = item[1];
        t.refs[item[1]] = t.refs[item[0]];
        t.refs[item[0]] = 0;
    }
    if (threadIdx.x == 0) {
        *w.n_items = holes;
        if (n_live_out) *n_live_out = live;
    }
}

// The listed pairs of pages: in the pool, no page written twice or also read.
__global__ void __launch_bounds__(kPlanThreads)
copy_plan_kernel(const Tables t, const int32_t* src, const int32_t* dst, int n, PageWork w) {
    grid_dep_wait();
    grid_dep_launch();
    if (threadIdx.x == 0) *w.n_items = 0;
    for (int i = threadIdx.x; i < t.n_pages; i += kPlanThreads) w.map[i] = 0;
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int a = src[i], b = dst[i];
        if (a < 0 || a >= t.n_pages || b < 0 || b >= t.n_pages) {
            bad = true;
            continue;
        }
        atomicOr(&w.map[a], 1);
        bad |= (atomicOr(&w.map[b], 2) & 2) != 0;
    }
    if (__syncthreads_or(bad)) return refuse(t, kStatusBadPosition);
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        bad |= (w.map[dst[i]] & 1) != 0;
        int32_t* item = w.items + 3 * static_cast<int64_t>(i);
        item[0] = src[i];
        item[1] = dst[i];
        item[2] = t.page_size;
    }
    if (__syncthreads_or(bad)) return refuse(t, kStatusBadPosition);
    if (threadIdx.x == 0) *w.n_items = n;
}

// The pools whose pages go together: K and V, or the codes and scales of both. In bytes; a place of a pool of scales
// may be no multiple of 16, a page's start is.
struct CopyPools {
    uint8_t* base[4];
    int64_t page[4], layer[4];
    int32_t place[4];
    int32_t n;
};

// The copy list, for every layer and pool: item, layer and pool one after another
// over a fixed grid (the list's length is known on the device only). A page's
// filled slots are one contiguous range. With map, the tables' entries are replaced
// by map[entry] in the same launch.
__global__ void __launch_bounds__(256)
copy_kernel(const __grid_constant__ CopyPools pools, int n_layer, const int32_t* n_items, const int32_t* items, const Tables t,
            const int32_t* map) {
    grid_dep_wait();
    grid_dep_launch();
    if (map) {
        const int64_t all = static_cast<int64_t>(t.n_slots) * t.max_pages;
        for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < all; e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
            const int slot = static_cast<int>(e / t.max_pages), j = static_cast<int>(e - static_cast<int64_t>(slot) * t.max_pages);
            // with nothing to move the tables stay as they are (a refused plan leaves map unwritten)
            if (*n_items > 0 && j < pages_for(t.seq_len[slot], t.page_size)) t.table[e] = map[t.table[e]];
        }
    }
    const int64_t n = static_cast<int64_t>(*n_items) * n_layer * pools.n;
    for (int64_t x = blockIdx.x; x < n; x += gridDim.x) {
        const int64_t it = x / (pools.n * n_layer);
        const int lk = static_cast<int>(x - it * pools.n * n_layer), layer = lk / pools.n, p = lk - layer * pools.n;
        const int64_t bytes = static_cast<int64_t>(items[3 * it + 2]) * pools.place[p];
        if (bytes == 0) continue;
        const int words = static_cast<int>(bytes / 16);
        const uint8_t* pool = pools.base[p] + layer * pools.layer[p];
        const uint4* from = reinterpret_cast<const uint4*>(pool + items[3 * it] * pools.page[p]);
        uint4* to = reinterpret_cast<uint4*>(const_cast<uint8_t*>(pool) + items[3 * it + 1] * pools.page[p]);
        for (int i = threadIdx.x; i < words; i += 4 * blockDim.x) {
            uint4 r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * static_cast<int>(blockDim.x) < words) r[u] = __ldcs(from + i + u * blockDim.x);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * static_cast<int>(blockDim.x) < words) __stcs(to + i + u * blockDim.x, r[u]);
        }
        if (threadIdx.x < (bytes & 15) / 4)
            reinterpret_cast<uint32_t*>(to + words)[threadIdx.x] = reinterpret_cast<const uint32_t*>(from + words)[threadIdx.x];
    }
}

// ---- new tokens into their pages ----

// A unit is 16 values of one head of one token: with rope, 8 of the first half
// of the head and the 8 that they are rotated with. A block takes one token's
// units (grid.y covers long rows); q, then k, then v. HBM-bound: each value is
// read once and written once.
__global__ void __launch_bounds__(256)
rope_kv_paged_kernel(PagedLayer c, BatchView b, float* q, int64_t ldq, const float* k, int64_t ldk,
                     const float* v, int64_t ldv, int n_head, const float* table, int table_rows,
                     int* status) {
    grid_dep_wait();
    grid_dep_launch();
    const int row = blockIdx.x;
    // the last sequence that starts at or before this row and is not empty there
    int lo = 0, hi = b.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.q_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    const SeqView s = seq_view(c, b, lo);
    const int t = row - s.q0;
    if (!s.ok) {
        if (threadIdx.x == 0) record_status(status, kStatusBadPosition);
        return;
    }
    if (t < 0 || t >= s.n_new) return;   // a row behind the last sequence
    const int pos = s.len - s.n_new + t;
    const int page = pos >= 0 ? c.table[static_cast<int64_t>(s.slot) * c.max_pages + c.page_div.div(pos)] : -1;
    if (pos < 0 || page < 0 || page >= c.n_pages || (table && pos >= table_rows)) {
        if (threadIdx.x == 0) record_status(status, kStatusBadPosition);
        return;
    }
    const int hd = c.head_dim, per = hd / 16, half = hd / 2;
    const int n_rot = n_head + c.n_kv;
    const int units = (n_rot + c.n_kv) * per;
    const int64_t at = static_cast<int64_t>(page) * c.page_stride + static_cast<int64_t>(pos - c.page_div.div(pos) * c.page_size) * c.n_kv * hd;
    __half* kc = const_cast<__half*>(c.k) + at;
    __half* vc = const_cast<__half*>(c.v) + at;
    const float* cs = table ? table + static_cast<int64_t>(pos) * hd : nullptr;
    for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < units; u += gridDim.y * blockDim.x) {
        const int h = u / per, d = (u - h * per) * 8;
        if (h < n_head && !table) continue;   // nothing to rotate: q stays as it is
        const float* src = h < n_head ? q + row * ldq + static_cast<int64_t>(h) * hd
                           : h < n_rot ? k + row * ldk + static_cast<int64_t>(h - n_head) * hd
                                       : v + row * ldv + static_cast<int64_t>(h - n_rot) * hd;
        float x[8], y[8];
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(src + d);
        *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(src + d + 4);
        *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(src + half + d);
        *reinterpret_cast<float4*>(y + 4) = *reinterpret_cast<const float4*>(src + half + d + 4);
        if (table && h < n_rot) {
            float co[8], si[8];
            *reinterpret_cast<float4*>(co) = *reinterpret_cast<const float4*>(cs + d);
            *reinterpret_cast<float4*>(co + 4) = *reinterpret_cast<const float4*>(cs + d + 4);
            *reinterpret_cast<float4*>(si) = *reinterpret_cast<const float4*>(cs + half + d);
            *reinterpret_cast<float4*>(si + 4) = *reinterpret_cast<const float4*>(cs + half + d + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) {   // each product and sum rounded by itself, as the library's other rope kernels
                const float a = x[i], e = y[i];
                x[i] = __fsub_rn(__fmul_rn(a, co[i]), __fmul_rn(e, si[i]));
                y[i] = __fadd_rn(__fmul_rn(a, si[i]), __fmul_rn(e, co[i]));
            }
        }
        if (h < n_head) {
            float* o = q + row * ldq + static_cast<int64_t>(h) * hd;
            *reinterpret_cast<float4*>(o + d) = *reinterpret_cast<float4*>(x);
            *reinterpret_cast<float4*>(o + d + 4) = *reinterpret_cast<float4*>(x + 4);
            *reinterpret_cast<float4*>(o + half + d) = *reinterpret_cast<float4*>(y);
            *reinterpret_cast<float4*>(o + half + d + 4) = *reinterpret_cast<float4*>(y + 4);
        } else {
            __half* o = (h < n_rot ? kc + (h - n_head) * hd : vc + (h - n_rot) * hd) + d;
            __half2 a[4], e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                e[i] = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
            }
            *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(a);
            *reinterpret_cast<uint4*>(o + half) = *reinterpret_cast<const uint4*>(e);
        }
    }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check(const hesa_cuda_paged_kv* kv) { return check_paged_kv(kv); }
int check(const hesa_cuda_paged_kv4* kv) { return check_paged_kv4(kv); }

template <typename KV>
size_t pages_workspace(const KV* kv) {
    if (check(kv) != HESA_CUDA_OK) return 0;
    if (kv->n_pages > (1 << 20)) return 0;
    const size_t most = static_cast<size_t>(most_items(kv->n_pages, kv->n_slots));
    return (4 + 4 * most + static_cast<size_t>(kv->n_pages) + static_cast<size_t>(kv->n_slots) + 1) * sizeof(int32_t);
}

// Checks that every page operation shares, and its tables.
template <typename KV>
int page_op(const KV* kv, int32_t n, void* ws, size_t ws_bytes, Tables* t) {
    const int rc = check(kv);
    if (rc != HESA_CUDA_OK) return rc;
    if (!kv->page_refs || !aligned(kv->page_refs, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "page operations need page_refs");
    if (n < 0) return record_error(HESA_CUDA_SHAPE_MISMATCH, "negative count");
    if (kv->n_pages > (1 << 20)) return record_error(HESA_CUDA_SHAPE_MISMATCH, "page operations take at most 2^20 pages");
    if (!ws || !aligned(ws, 16)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    if (ws_bytes < pages_workspace(kv)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    t->table = kv->table;
    t->seq_len = kv->seq_len;
    t->refs = kv->page_refs;
    t->n_slots = kv->n_slots;
    t->max_pages = kv->max_pages;
    t->n_pages = kv->n_pages;
    t->page_size = kv->page_size;
    return HESA_CUDA_OK;
}

CopyPools copy_pools(const hesa_cuda_paged_kv* kv) {
    CopyPools p{};
    p.n = 2;
    for (int i = 0; i < 2; ++i) {
        p.base[i] = static_cast<uint8_t*>(i ? kv->v : kv->k);
        p.page[i] = kv->page_stride * 2;
        p.layer[i] = kv->layer_stride * 2;
        p.place[i] = kv->n_kv_head * kv->head_dim * 2;
    }
    return p;
}
CopyPools copy_pools(const hesa_cuda_paged_kv4* kv) {
    CopyPools p{};
    p.n = 4;
    void* const base[4] = {kv->k, kv->v, kv->k_scale, kv->v_scale};
    for (int i = 0; i < 4; ++i) {
        const int group = i < 2 ? 16 : 2;   // bytes
        p.base[i] = static_cast<uint8_t*>(base[i]);
        p.page[i] = kv->page_stride * group;
        p.layer[i] = kv->layer_stride * group;
        p.place[i] = kv->n_kv_head * (kv->head_dim / kGroup) * group;
    }
    return p;
}

template <typename KV>
cudaError_t launch_copy(const KV* kv, const Tables& t, const PageWork& w, int64_t most, const int32_t* map, cudaStream_t s) {
    const CopyPools pools = copy_pools(kv);
    // eight blocks an SM keep enough loads in flight; fewer where fewer pages can move
    const int64_t blocks = std::min<int64_t>(148 * 8, std::max<int64_t>(1, most * kv->n_layer * pools.n));
    return launch_dep(copy_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, s, pools, kv->n_layer, w.n_items, w.items, t, map);
}

template <typename KV>
int kv_reserve(const KV* kv, const int32_t* slots, const int32_t* n_new, int32_t n, void* workspace,
                         size_t workspace_bytes, void* stream) {
    Tables t{};
    const int rc = page_op(kv, n, workspace, workspace_bytes, &t);
    if (rc != HESA_CUDA_OK) return rc;
    if (n > kv->n_slots) return record_error(HESA_CUDA_SHAPE_MISMATCH, "more slots than the cache has");
    if (n == 0) return HESA_CUDA_OK;
    if (!slots || !n_new) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (!aligned(slots, 4) || !aligned(n_new, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the lists must be 4-byte aligned");
    cudaError_t e = status_word(&t.status);
    if (e == cudaSuccess) {
        e = launch_dep(reserve_kernel, dim3(1), kPlanThreads, 0, static_cast<cudaStream_t>(stream), t, slots, n_new, n, page_work(workspace, kv));
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv_reserve kernel");
}

template <typename KV>
int kv_free(const KV* kv, const int32_t* slots, int32_t n, void* workspace, size_t workspace_bytes,
                      void* stream) {
    Tables t{};
    const int rc = page_op(kv, n, workspace, workspace_bytes, &t);
    if (rc != HESA_CUDA_OK) return rc;
    if (n > kv->n_slots) return record_error(HESA_CUDA_SHAPE_MISMATCH, "more slots than the cache has");
    if (n == 0) return HESA_CUDA_OK;
    if (!slots) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (!aligned(slots, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the lists must be 4-byte aligned");
    cudaError_t e = status_word(&t.status);
    if (e == cudaSuccess) {
        e = launch_dep(free_kernel, dim3(1), kPlanThreads, 0, static_cast<cudaStream_t>(stream), t, slots, n);
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv_free kernel");
}

template <typename KV>
int kv_fork(const KV* kv, const int32_t* src, const int32_t* dst, int32_t n, void* workspace,
                      size_t workspace_bytes, void* stream) {
    Tables t{};
    const int rc = page_op(kv, n, workspace, workspace_bytes, &t);
    if (rc != HESA_CUDA_OK) return rc;
    if (n > kv->n_slots) return record_error(HESA_CUDA_SHAPE_MISMATCH, "more slots than the cache has");
    if (n == 0) return HESA_CUDA_OK;
    if (!src || !dst) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (!aligned(src, 4) || !aligned(dst, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the lists must be 4-byte aligned");
    const PageWork w = page_work(workspace, kv);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = status_word(&t.status);
    if (e == cudaSuccess) {
        e = launch_dep(fork_plan_kernel, dim3(1), kPlanThreads, 0, s, t, src, dst, n, w);
    }
    if (e == cudaSuccess) e = launch_copy(kv, t, w, n, nullptr, s);
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv_fork kernels");
}

template <typename KV>
int kv_compact(const KV* kv, int32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
    Tables t{};
    const int rc = page_op(kv, 0, workspace, workspace_bytes, &t);
    if (rc != HESA_CUDA_OK) return rc;
    if (!aligned(n_live, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "n_live must be 4-byte aligned");
    const PageWork w = page_work(workspace, kv);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = status_word(&t.status);
    if (e == cudaSuccess) {
        e = launch_dep(compact_plan_kernel, dim3(1), kPlanThreads, 0, s, t, w, n_live);
    }
    if (e == cudaSuccess) e = launch_copy(kv, t, w, kv->n_pages / 2, w.map, s);
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv_compact kernels");
}

template <typename KV>
int kv_copy_pages(const KV* kv, const int32_t* src_pages, const int32_t* dst_pages, int32_t n,
                            void* workspace, size_t workspace_bytes, void* stream) {
    Tables t{};
    const int rc = page_op(kv, n, workspace, workspace_bytes, &t);
    if (rc != HESA_CUDA_OK) return rc;
    if (n > kv->n_pages) return record_error(HESA_CUDA_SHAPE_MISMATCH, "more pairs than pages");
    if (n == 0) return HESA_CUDA_OK;
    if (!src_pages || !dst_pages) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (!aligned(src_pages, 4) || !aligned(dst_pages, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the lists must be 4-byte aligned");
    const PageWork w = page_work(workspace, kv);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = status_word(&t.status);
    if (e == cudaSuccess) {
        e = launch_dep(copy_plan_kernel, dim3(1), kPlanThreads, 0, s, t, src_pages, dst_pages, n, w);
    }
    if (e == cudaSuccess) e = launch_copy(kv, t, w, n, nullptr, s);
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv_copy_pages kernels");
}

// Warps that share one of n things, none with less than a step of `columns` of the table: the logarithm of a power of two
int share_of(int warps, int n, int32_t max_pages, int columns) {
    int x = 0;
    while ((warps >> (x + 1)) >= n && max_pages > static_cast<int64_t>(columns) << x) ++x;
    return x;
}

template <typename KV>
int kv_reorder(const KV* kv, const int32_t* slots, const int32_t* parents, int32_t n, int32_t width, void* workspace, size_t workspace_bytes,
               void* stream) {
    Tables t{};
    const int rc = page_op(kv, n, workspace, workspace_bytes, &t);
    if (rc != HESA_CUDA_OK) return rc;
    if (n > kv->n_slots) return record_error(HESA_CUDA_SHAPE_MISMATCH, "more slots than the cache has");
    if (width < 1 || width > 32 || n % width != 0) return record_error(HESA_CUDA_SHAPE_MISMATCH, "width must be 1 .. 32 and divide n");
    if (n == 0) return HESA_CUDA_OK;
    if (!slots || !parents) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (!aligned(slots, 4) || !aligned(parents, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the lists must be 4-byte aligned");
    const PageWork w = page_work(workspace, kv);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = status_word(&t.status);
    if (e == cudaSuccess) {
        const bool wide = static_cast<int64_t>(n) * kv->max_pages > kMostEntries;
        const int blocks = wide ? kPlanBlocks : 1, warps = kPlanThreads / 32 * blocks;
        e = launch_clusters(wide ? reorder_plan_kernel<kPlanBlocks> : reorder_plan_kernel<1>, blocks, dim3(blocks), kPlanThreads, 0, s, t, slots, parents, n, width,
                            share_of(warps, n, kv->max_pages, 32),
                            share_of(warps, n / width, kv->max_pages, kColumnSteps * (32 / width)), w);
    }
    if (e == cudaSuccess) e = launch_copy(kv, t, w, n, nullptr, s);
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv_reorder kernels");
}

}  // namespace
}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_kv_pages_workspace_size(const hesa_cuda_paged_kv* kv) { return pages_workspace(kv); }

int hesa_cuda_kv_reserve(const hesa_cuda_paged_kv* kv, const int32_t* slots, const int32_t* n_new, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_reserve");
    return kv_reserve(kv, slots, n_new, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv_free(const hesa_cuda_paged_kv* kv, const int32_t* slots, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_free");
    return kv_free(kv, slots, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv_fork(const hesa_cuda_paged_kv* kv, const int32_t* src, const int32_t* dst, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_fork");
    return kv_fork(kv, src, dst, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv_compact(const hesa_cuda_paged_kv* kv, int32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_compact");
    return kv_compact(kv, n_live, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv_copy_pages(const hesa_cuda_paged_kv* kv, const int32_t* src_pages, const int32_t* dst_pages, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_copy_pages");
    return kv_copy_pages(kv, src_pages, dst_pages, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv_reorder(const hesa_cuda_paged_kv* kv, const int32_t* slots, const int32_t* parents, int32_t n, int32_t width, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_reorder");
    return kv_reorder(kv, slots, parents, n, width, workspace, workspace_bytes, stream);
}

size_t hesa_cuda_kv4_pages_workspace_size(const hesa_cuda_paged_kv4* kv) { return pages_workspace(kv); }

int hesa_cuda_kv4_reserve(const hesa_cuda_paged_kv4* kv, const int32_t* slots, const int32_t* n_new, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_reserve");
    return kv_reserve(kv, slots, n_new, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv4_free(const hesa_cuda_paged_kv4* kv, const int32_t* slots, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_free");
    return kv_free(kv, slots, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv4_fork(const hesa_cuda_paged_kv4* kv, const int32_t* src, const int32_t* dst, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_fork");
    return kv_fork(kv, src, dst, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv4_compact(const hesa_cuda_paged_kv4* kv, int32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_compact");
    return kv_compact(kv, n_live, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv4_copy_pages(const hesa_cuda_paged_kv4* kv, const int32_t* src_pages, const int32_t* dst_pages, int32_t n, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_copy_pages");
    return kv_copy_pages(kv, src_pages, dst_pages, n, workspace, workspace_bytes, stream);
}

int hesa_cuda_kv4_reorder(const hesa_cuda_paged_kv4* kv, const int32_t* slots, const int32_t* parents, int32_t n, int32_t width, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_reorder");
    return kv_reorder(kv, slots, parents, n, width, workspace, workspace_bytes, stream);
}

int hesa_cuda_rope_kv_paged(const hesa_cuda_paged_kv* kv, int32_t layer, const hesa_cuda_token_batch* batch, float* q, int64_t ldq,
                            const float* k, int64_t ldk, const float* v, int64_t ldv, int64_t n_head, const float* rope_table,
                            int32_t rope_rows, void* stream) {
    HESA_TRACE("hesa_cuda_rope_kv_paged");
    int rc = check_paged_kv(kv);
    if (rc == HESA_CUDA_OK) rc = check_batch(kv, layer, batch, n_head);
    if (rc != HESA_CUDA_OK) return rc;
    if (batch->n_tokens == 0) return HESA_CUDA_OK;   // no rows: their buffers may be null
    if (!k || !v || (rope_table && !q)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    const int64_t kv_width = static_cast<int64_t>(kv->n_kv_head) * kv->head_dim;
    if (ldk < kv_width || ldv < kv_width || (rope_table && (ldq < n_head * kv->head_dim || rope_rows <= 0)))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "leading dimension or rope table too small");
    if (ldq > (int64_t(1) << 40) || ldk > (int64_t(1) << 40) || ldv > (int64_t(1) << 40))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "leading dimension too large");
    if (!aligned(k, 16) || !aligned(v, 16) || (ldk & 3) || (ldv & 3) || (rope_table && (!aligned(q, 16) || !aligned(rope_table, 16) || (ldq & 3))))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "q, k, v and the rope table must be 16-byte aligned with leading dimensions multiples of 4");
    int* status = nullptr;
    cudaError_t e = status_word(&status);
    if (e == cudaSuccess) {
        const int64_t units = (n_head + 2 * kv->n_kv_head) * (kv->head_dim / 16);
        // one block a token where tokens are many; few tokens are spread over more blocks
        const int64_t y = batch->n_tokens >= 148 * 4 ? 1 : std::min<int64_t>((units + 255) / 256, 1024);
        e = launch_dep(rope_kv_paged_kernel, dim3(static_cast<unsigned>(batch->n_tokens), static_cast<unsigned>(y)), 256, 0,
                       static_cast<cudaStream_t>(stream), layer_of(kv, layer), view_of(batch), q, ldq, k, ldk, v, ldv,
                       static_cast<int>(n_head), rope_table, rope_rows, status);
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "rope_kv_paged kernel");
}

}  // extern "C"
