// paged_rows.cuh -- what the kernels for tiles of 8 rows share (paged_attention.cu
// for the fp16 cache, paged_attention4.cu for the one in 4 bits): the work as a
// row of units that equal runs of CTAs take, and the adding up of what is cut.
#pragma once

#include "paged.h"

namespace hesa_cuda {

constexpr int kRowTile = 8;
constexpr int kRowsCtas = 148;       // one an SM
constexpr int kMostTiles = 1024;     // of a launch: the tiles' blocks are summed in shared memory
constexpr int kLeastUnits = 4;       // of a run

// A CTA's warps, and the workspace: the list of what is to be added up, then the
// parts' rows (m, l), then their acc[HD]; a part has [warps][rows] of them.
template <int HD, int WARPS> struct RowParts {
    static constexpr int warps = WARPS;
    static constexpr size_t cut_bytes = kMostTiles * 32;
    static constexpr size_t part_rows(int64_t parts) { return static_cast<size_t>(parts) * WARPS * kRowTile; }
    static constexpr size_t bytes(int64_t parts) { return cut_bytes + part_rows(parts) * (2 + HD) * 4; }
};

// Heads of a group (a CTA's warps have one each) and how many warps share a head.
struct HeadGroups {
    int groups, heads, subs, recip, cost, sub_bits;   // subs is a power of two, `warps` being one
    int least = kLeastUnits;                          // units of a run
    // `most` heads a group at most, a power of two up to `warps`; starting a (tile, group) takes as long as seg_cost blocks of every warp
    HeadGroups(int n_kv, int warps, int most, int seg_cost) {
        groups = (n_kv + most - 1) / most;
        heads = (n_kv + groups - 1) / groups;
        for (sub_bits = 0; (heads << (sub_bits + 1)) <= warps;) ++sub_bits;
        subs = 1 << sub_bits;
        recip = (256 + heads - 1) / heads;
        cost = seg_cost * subs;
    }
    __device__ __forceinline__ int sub_of(int warp) const { return warp * recip >> 8; }   // warp / heads for warp < 16, heads <= 16: the excess of warp * (recip - 256 / heads) / 256 is less than 1 / heads
};

// Parts of a launch: two a CTA (its run's first (tile, group) and its last), and,
// where several warps share a head, one for each (tile, group) that lies in one run.
__host__ __device__ inline int64_t part_count(int tiles, const HeadGroups& hg) {
    return 2 * kRowsCtas + (hg.subs > 1 ? static_cast<int64_t>(tiles) * hg.groups : 0);
}

// Whether every (tile, group) has an entry in the list of what is to be added up.
__host__ __device__ inline bool by_tile(int tiles, const HeadGroups& hg) {
    return hg.subs > 1 || static_cast<int64_t>(tiles) * hg.groups <= kRowsCtas;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 64-bit quotients of numbers that are small nearly always
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// The runs: CTA c of n_cta has units [start(c), start(c + 1)), `each` of them,
// the first `more` CTAs one more.
struct Runs {
    int64_t each, more;
    int n_cta;
    __device__ __forceinline__ Runs(int64_t units, int most, int least) {
        n_cta = static_cast<int>(max(int64_t(1), min(static_cast<int64_t>(most), units / least)));
        each = quotient(units, n_cta);
        more = units - each * n_cta;
    }
    __device__ __forceinline__ int64_t start(int c) const { return each * c + min(static_cast<int64_t>(c), more); }
    __device__ __forceinline__ int cta_of(int64_t u) const {   // the last c with start(c) <= u
        const int64_t head = more * (each + 1);
        return static_cast<int>(u < head ? quotient(u, each + 1) : more + quotient(u - head, each));
    }
};

// What a CTA's run has of one (tile, group): blocks [b0, b1).
struct Segment {
    int tile, grp, b0, b1;
    int64_t first;   // its first unit; the blocks' units start hg.cost later
    int64_t units;
};

// The next segment with blocks of the run [u, end); u moves behind it. `lo` is a
// tile that starts at or before u.
__device__ __forceinline__ bool next_segment(const int64_t* pre, const HeadGroups& hg, int64_t& u, int64_t end, int& lo, Segment& s) {
    while (u < end) {
        while (pre[lo + 1] * hg.groups <= u) ++lo;   // tiles without rows have no units
        s.tile = lo;
        s.units = pre[lo + 1] - pre[lo];
        s.grp = static_cast<int>(quotient(u - pre[lo] * hg.groups, s.units));
        s.first = pre[lo] * hg.groups + s.grp * s.units;
        const int64_t from = max(u, s.first + hg.cost), stop = min(end, s.first + s.units);
        u = stop;
        s.b0 = static_cast<int>(from - s.first - hg.cost);
        s.b1 = static_cast<int>(stop - s.first - hg.cost);
        if (s.b1 > s.b0) return true;
    }
    return false;
}

// The rows and keys of a tile; kb counts blocks of BLOCK keys.
struct TileView {
    SeqView sv;
    int n_rows, r0, base;   // base: position of the sequence's first new token
    int32_t p_lo, p_hi;
    Mask mask;
    KeyBlocks kb;
};

template <int BLOCK>
__device__ __forceinline__ TileView tile_view(const AttnArgs& A, int idx) {
    TileView v;
    int seq, tile;
    const bool some = locate_tile(A.b, A.group, kRowTile, A.per_seq, A.tile0 + idx, seq, tile);
    v.sv = seq_view(A.c, A.b, seq);
    v.n_rows = some ? v.sv.n_new * A.group : 0;
    v.r0 = tile * kRowTile;
    v.base = v.sv.len - v.sv.n_new;
    v.p_lo = v.base + A.group_div.div(v.r0);
    v.p_hi = v.base + A.group_div.div(max(min(v.r0 + kRowTile, v.n_rows), 1) - 1);
    v.mask = Mask{v.sv.len, A.window, 0};
    if (A.prefix && v.sv.ok) v.mask.prefix = max(0, min(A.prefix[seq], v.sv.len));
    v.kb = key_blocks(v.mask, v.p_lo, v.p_hi, BLOCK);
    return v;
}

// Units before each of the launch's tiles, for one group, into pre[0 .. tiles]:
// a unit for each block of keys and hg.cost for starting, none for a tile without
// rows. sums holds a word a warp. All threads of the block; returns the total.
template <int WARPS, int BLOCK>
__device__ __forceinline__ int64_t tile_units(const AttnArgs& A, const HeadGroups& hg, int tiles, int64_t* pre, int64_t* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t before = 0;
    for (int i0 = 0; i0 < tiles; i0 += WARPS * 32) {
        const int i = i0 + threadIdx.x;
        int64_t v = 0;
        if (i < tiles) {
            const TileView tv = tile_view<BLOCK>(A, i);
            if (!tv.sv.ok && blockIdx.x == 0) record_status(A.status, kStatusBadPosition);
            // a tile whose rows see nothing has one block too: its zeros are written there
            if (tv.sv.ok && tv.r0 < tv.n_rows) v = max(1, tv.kb.n) + hg.cost;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += y;
        }
        if (lane == 31) sums[warp] = v;
        __syncthreads();
        int64_t all = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) v += sums[w];
            all += sums[w];
        }
        if (i < tiles) pre[i + 1] = before + v;
        before += all;
        __syncthreads();
    }
    return before;
}

// The last tile that starts at or before unit u.
__device__ __forceinline__ int tile_at(const int64_t* pre, const HeadGroups& hg, int tiles, int64_t u) {
    int lo = 0, hi = tiles - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] * hg.groups <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// What combine_kernel adds up, and where it belongs: rows r0 .. r0 + rows - 1 of
// the sequence whose first row of q is q0. The parts are `first`, then the
// first part of each of the next n - 1 CTAs, each of hg.subs warps. n = 0, or one
// part of one warp: nothing. With by_tile every (tile, group) has an entry (groups
// of fewer heads are only made of few tiles, so kMostTiles entries are enough); else
// there is one for each CTA, for the cut before its run (if it is the first one of
// what it cuts).
struct __align__(16) Cut {
    int32_t grp, first, n, rows;
    int32_t r0, q0, pad[2];
};

// Adds up what is cut: block (entry, head of the group), or one for each row too
// where these are few (then there are many parts). The rows are shared out over
// the warps; where they are fewer than eight, several warps take every second,
// fourth or eighth part of a row. Two contexts of 131072 and 100001 tokens with a
// block for all eight rows: 180 us; with one for each: 163. A batch of 64 short
// sequences: 13.7 us and 17.6.
template <int HD, int WARPS>
__global__ void __launch_bounds__(256)
combine_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ HeadGroups hg) {
    using S = RowParts<HD, WARPS>;
    constexpr int V = HD / 32;     // values of a lane
    constexpr int AHEAD = 32 / V;  // parts of which a warp has the loads under way
    __shared__ float s_o[8][HD + 1];
    const int hl = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dep_wait();
    grid_dep_launch();
    const int4* c4 = reinterpret_cast<const int4*>(A.part) + 2 * blockIdx.x;
    const int4 ca = __ldcg(c4), cb = __ldcg(c4 + 1);
    const Cut cut{ca.x, ca.y, ca.z, ca.w, cb.x, cb.y};
    const int n = cut.n * hg.subs, kvh = cut.grp * hg.heads + hl;
    if (n < 2 || kvh >= A.c.n_kv) return;
    const int row0 = blockIdx.z, rows = min(gridDim.z > 1 ? 1 : kRowTile, cut.rows - row0);
    if (rows <= 0) return;
    const int slots = rows > 4 ? 8 : rows > 2 ? 4 : rows;   // a power of two
    const int row = warp & (slots - 1), share = warp / slots, shares = 8 / slots;   // row: of row0 ..
    const float* ml = A.part + S::cut_bytes / 4;
    const float* acc = ml + S::part_rows(part_count(A.n_split, hg)) * 2;
    auto at = [&](int i) {   // part i: sub-part i % subs of CTA part i / subs
        const int p = i >> hg.sub_bits, x = i & (hg.subs - 1);
        return (static_cast<int64_t>(p == 0 ? cut.first : 2 * ((cut.first >> 1) + p)) * S::warps + x * hg.heads + hl) * kRowTile + row0 + row;
    };
    float L = 0.f, O[V];
#pragma unroll
    for (int k = 0; k < V; ++k) O[k] = 0.f;
    if (row < rows) {
        float2 p[AHEAD];
        float v[AHEAD][V];
        auto load = [&](int i0) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int i = i0 + k * shares;
                if (i >= n) break;
                const int64_t a = at(i);
                p[k] = __ldcg(reinterpret_cast<const float2*>(ml + a * 2));
                const float* src = acc + a * HD + lane * V;
                if constexpr (V == 2) *reinterpret_cast<float2*>(v[k]) = __ldcg(reinterpret_cast<const float2*>(src));
                else
#pragma unroll
                    for (int c = 0; c < V; c += 4) *reinterpret_cast<float4*>(v[k] + c) = __ldcg(reinterpret_cast<const float4*>(src + c));
            }
        };
        load(share);   // on their way while the maximum is found
        float M = -INFINITY;
#pragma unroll 8
        for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(ml + at(i) * 2));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        for (int i0 = share;;) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (i0 + k * shares >= n) break;
                // a part that saw nothing adds zeros, or the NaN of a row that is not finite
                const float f = p[k].x == -INFINITY ? 1.f : ex2(p[k].x - M);
                L = fmaf(p[k].y, f, L);
#pragma unroll
                for (int c = 0; c < V; ++c) O[c] = fmaf(v[k][c], f, O[c]);
            }
            i0 += AHEAD * shares;
            if (i0 >= n) break;
            load(i0);
        }
        if (shares > 1) {
#pragma unroll
            for (int c = 0; c < V; ++c) s_o[warp][lane * V + c] = O[c];
            if (lane == 0) s_o[warp][HD] = L;
        }
    }
    if (shares > 1) __syncthreads();
    if (row >= rows || share > 0) return;
    for (int x = 1; x < shares; ++x) {
        L += s_o[warp + x * slots][HD];
#pragma unroll
        for (int c = 0; c < V; ++c) O[c] += s_o[warp + x * slots][lane * V + c];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int r = cut.r0 + row0 + row, t = A.group_div.div(r), h = kvh * A.group + r - t * A.group;
    float* o = A.out + static_cast<int64_t>(cut.q0 + t) * A.ldo + static_cast<int64_t>(h) * HD + lane * V;
#pragma unroll
    for (int c = 0; c < V; c += 2) *reinterpret_cast<float2*>(o + c) = make_float2(O[c] * inv, O[c + 1] * inv);
}

}  // namespace hesa_cuda
