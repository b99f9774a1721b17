// kv_pages.cu -- writing new tokens into the pages of a cache, and giving,
// sharing, taking back and moving pages.
//
// The tables (pages of each slot, tokens of each slot, references of each page)
// live on the device, so a serving loop changes them between two steps without
// reading anything back. One block plans a change: it checks every slot, page
// and length that the change touches, and only when all are sound writes the
// tables; else it records a device status and changes nothing. Free pages are
// taken in ascending order, so results do not depend on scheduling. What is to
// be copied goes into a list in the workspace, and a second kernel copies it for
// all layers: whole 16-byte words of K and V, bound by HBM.
// Measured: compaction that moves 240 pages of 32 layers 180 us (1.0 GB; the plan
// takes 7 us of them, the copies run at 6 TB/s); free, fork and reserve of seven
// slots of up to 44 pages 19 us for the four launches, which are chains of dependent
// reads by one block; the cache write of 5296 tokens (32 heads) 67.8 us
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

PageWork page_work(void* ws, const hesa_cuda_paged_kv* kv) {
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
    int before = 0, all = 0;
    for (int w = 0; w < n_warp; ++w) {
        const int y = s[w];
        before += w < warp ? y : 0;
        all += y;
    }
    __syncthreads();
    total = all;
    return before + v - x;
}

// The lowest `want` free pages into list, ascending; false when there are fewer.
__device__ bool lowest_free(const Tables& t, int want, int32_t* list, int* s) {
    int found = 0;
    for (int b = 0; b < t.n_pages && found < want; b += kPlanThreads) {
        const int i = b + threadIdx.x;
        const bool is_free = i < t.n_pages && t.refs[i] == 0;
        int total;
        const int at = found + block_scan(is_free ? 1 : 0, s, total);
        if (is_free && at < want) list[at] = i;
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

// The copy list, for every layer and for K and V: item, layer and pool one
// after another over a fixed grid (the list's length is known on the device
// only). A page's filled slots are one contiguous range. With map, the tables'
// entries are replaced by map[entry] in the same launch.
__global__ void __launch_bounds__(256)
copy_kernel(uint4* k, uint4* v, int64_t page_words, int64_t layer_words, int n_layer,
            int slot_words, const int32_t* n_items, const int32_t* items, const Tables t,
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
    const int64_t n = static_cast<int64_t>(*n_items) * n_layer * 2;
    for (int64_t x = blockIdx.x; x < n; x += gridDim.x) {
        const int64_t it = x / (2 * n_layer);
        const int lk = static_cast<int>(x - it * 2 * n_layer);
        const int words = items[3 * it + 2] * slot_words;
        if (words == 0) continue;
        uint4* pool = (lk & 1) ? v : k;
        const uint4* from = pool + (lk >> 1) * layer_words + items[3 * it] * page_words;
        uint4* to = pool + (lk >> 1) * layer_words + items[3 * it + 1] * page_words;
        for (int i = threadIdx.x; i < words; i += 4 * blockDim.x) {
            uint4 r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * static_cast<int>(blockDim.x) < words) r[u] = __ldcs(from + i + u * blockDim.x);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * static_cast<int>(blockDim.x) < words) __stcs(to + i + u * blockDim.x, r[u]);
        }
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

// Checks that every page operation shares, and its tables.
int page_op(const hesa_cuda_paged_kv* kv, int32_t n, void* ws, size_t ws_bytes, Tables* t) {
    const int rc = check_paged_kv(kv);
    if (rc != HESA_CUDA_OK) return rc;
    if (!kv->page_refs || !aligned(kv->page_refs, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "page operations need page_refs");
    if (n < 0) return record_error(HESA_CUDA_SHAPE_MISMATCH, "negative count");
    if (kv->n_pages > (1 << 20)) return record_error(HESA_CUDA_SHAPE_MISMATCH, "page operations take at most 2^20 pages");
    if (!ws || !aligned(ws, 16)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    if (ws_bytes < hesa_cuda_kv_pages_workspace_size(kv)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    t->table = kv->table;
    t->seq_len = kv->seq_len;
    t->refs = kv->page_refs;
    t->n_slots = kv->n_slots;
    t->max_pages = kv->max_pages;
    t->n_pages = kv->n_pages;
    t->page_size = kv->page_size;
    return HESA_CUDA_OK;
}

cudaError_t launch_copy(const hesa_cuda_paged_kv* kv, const Tables& t, const PageWork& w, int64_t most, const int32_t* map, cudaStream_t s) {
    const int slot_words = kv->n_kv_head * kv->head_dim / 8;
    // eight blocks an SM keep enough loads in flight; fewer where fewer pages can move
    const int64_t blocks = std::min<int64_t>(148 * 8, std::max<int64_t>(1, most * kv->n_layer * 2));
    return launch_dep(copy_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, s, static_cast<uint4*>(kv->k), static_cast<uint4*>(kv->v),
                      kv->page_stride / 8, kv->layer_stride / 8, kv->n_layer, slot_words, w.n_items, w.items, t, map);
}

}  // namespace
}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_kv_pages_workspace_size(const hesa_cuda_paged_kv* kv) {
    if (check_paged_kv(kv) != HESA_CUDA_OK) return 0;
    if (kv->n_pages > (1 << 20)) return 0;
    const size_t most = static_cast<size_t>(most_items(kv->n_pages, kv->n_slots));
    return (4 + 4 * most + static_cast<size_t>(kv->n_pages) + static_cast<size_t>(kv->n_slots) + 1) * sizeof(int32_t);
}

int hesa_cuda_kv_reserve(const hesa_cuda_paged_kv* kv, const int32_t* slots, const int32_t* n_new, int32_t n, void* workspace,
                         size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_reserve");
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

int hesa_cuda_kv_free(const hesa_cuda_paged_kv* kv, const int32_t* slots, int32_t n, void* workspace, size_t workspace_bytes,
                      void* stream) {
    HESA_TRACE("hesa_cuda_kv_free");
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

int hesa_cuda_kv_fork(const hesa_cuda_paged_kv* kv, const int32_t* src, const int32_t* dst, int32_t n, void* workspace,
                      size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_fork");
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

int hesa_cuda_kv_compact(const hesa_cuda_paged_kv* kv, int32_t* n_live, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_compact");
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

int hesa_cuda_kv_copy_pages(const hesa_cuda_paged_kv* kv, const int32_t* src_pages, const int32_t* dst_pages, int32_t n,
                            void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_kv_copy_pages");
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
