// paged_attention4.cu -- attention of new tokens over a paged cache in 4 bits.
//
// The formulas, rows, tiles, masks and the equal runs of work are those of
// paged_attention.cu; a value is d (code - 8), an fp16 number exactly.
//
// rows4_kernel: tiles of 8 rows, for the next tokens of a decode step. A warp has a
// kv head of its own and takes blocks of 32 keys of it. Four more warps copy codes and
// scales of all heads of the block's tokens (they lie side by side) into a ring, with
// 16-byte asynchronous copies that put every key's row where the warps' reads meet no
// bank twice (k_at, v_at), and run ahead across sequences. (When every warp copied
// its own head's blocks, copies were a sixth of its instructions: two contexts of
// 131072 and 100001 tokens, 64 heads on 8, 110 us and 103.)
//   * codes become fp16 pairs in registers, in the places of the operands of
//     m16n8k16 products: the order of dims within a sum is free, so the thread
//     that needs keys of column n and dims of quarter c takes 16 consecutive bytes
//     of key n (head_dim 128: a whole group, one scale), and q is read in that
//     order, from shared memory (in registers it made the warps spill: 196 us and
//     112). For P V a pair has two keys: one byte permutation of two keys' words
//     brings them together, and the thread of column n takes head_dim / 8
//     consecutive dims. code_pairs and code_pairs_fma (paged.h) are the two ways from
//     codes to values; K takes one, V the other, which loads the pipes most evenly
//     (both alike: 102 us; so: 100).
//   * q and P are split into fp16 halves that are the two halves of the A operand
//     (16 rows), as in paged_attention.cu.
//   * with fewer heads than warps several warps have a head, take its blocks in turn
//     and add their sums up in shared memory at a segment's end, so that a sequence
//     that lies in one CTA's run is written at once.
// Bound by the warps' instructions and their waits for one another's pipes, not by
// HBM: a block of 32 keys of one head is 730 instructions of a warp (K 235, V 300,
// softmax 66), 40% of the time each of the tensor, fp16 and integer pipes; without
// the copies the kernel takes 90 us, without the products 65. More warps would fill
// the pipes, but their registers are all taken (32 of a thread's are sums).
// Measured (with combine_kernel): two contexts of 131072 and 100001 tokens, 64 heads on
// 8, 100 us (301 MB, 3.0 TB/s; the fp16 cache 167); 32 of 1 to 8192 tokens 29.7 us (34);
// one of 2048 tokens, 32 heads, 14.3 us (15.4): 5.4 us until the first products, 3 a
// block, 4 to join the parts.
//
// Chunks: the tokens of a few sequences at a time are laid out in fp16 in the
// workspace (values are fp16 numbers, nothing is rounded) as a cache of their own,
// and the kernel of paged_attention_tc.cu reads that. A chunk's keys are read once
// for each of its many tiles, so the pass before costs little: 2048 tokens at 16384, 64
// heads on 8, 1.76 ms (fp16 1.75); 512 at 2048, 32 heads, 48 us (41); 12 mixed chunks 40
// us (36).
#include "paged.h"
#include "paged_rows.cuh"
#include "paged_tc.h"
#include "abi_errors.h"
#include "qmatvec.h"
#include "trace.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace hesa_cuda {
namespace {

constexpr int kKeys4 = 32;           // of a block
constexpr int kCopyWarps4 = 4;
constexpr int kSegCost4 = 2;         // blocks of every warp that starting a (tile, group) takes the time of,
constexpr int kSegCostMost4 = 8;     // and blocks of a head: 100 sequences of 1 to 3000 tokens, 8 heads on 1, 21.2 us (32: 27.6, 16: 22.9), 12 on 2 21.8 (16: 24.1, 4: 25.5)
constexpr int kScratchPage = 128;    // tokens of a page of the fp16 copy
constexpr int64_t kScratchBytes = int64_t(1) << 30;

// Rows of a kv head and sequence above which the chunk kernel takes over, rather than
// tiles of 8 that each read the codes again (of the chunk, the codes are read once,
// and fp16 is written and read). Eight sequences of 4000 tokens, 64 heads on 8: 32 rows
// 36 us in tiles, 61 as a chunk; 64 rows 57 and 65; 96 rows 93 and 72. Two of 60000: 64
// rows 186 and 238, 96 rows 462 and 239. 16 heads of 256 on 4, eight of 4000: 64 rows 61
// and 85, 128 rows 104 and 91. 32 heads of 64 on 8: 64 rows 37 and 46, 96 rows 59 and 50.
constexpr int kMostRows4 = 64;

// 16 warps (8 with head_dim 256) and a warpgroup that copies. Registers a thread
// after setmaxnreg: 512 x 112 + 128 x 32 = 640 x 96, and 256 x 232 + 128 x 40 = 384 x 168,
// what the block is launched with.
template <int HD> struct Rows4Shape : RowParts<HD, (HD == 256 ? 8 : 16)> {
    using RowParts<HD, (HD == 256 ? 8 : 16)>::warps;
    static constexpr int threads = (warps + kCopyWarps4) * 32;
    static constexpr int regs = HD == 256 ? 232 : 112, copy_regs = HD == 256 ? 40 : 32;
    static constexpr int groups = HD / kGroup;             // of a head: 16-byte pieces of a key's codes
    static constexpr int row = HD / 2, srow = groups * 2;  // bytes of a key's codes and scales
    static constexpr int v = kKeys4 * row, ks = 2 * v, vs = ks + kKeys4 * srow;   // K's codes, V's, then the scales
    static constexpr int block = vs + kKeys4 * srow;       // bytes of a block of one head
    static constexpr int depth = HD == 64 ? 4 : 2;         // blocks of a warp in the ring
    static constexpr int q = HD / 16 * 512;                // a warp's q: a k-step's operand is 16 bytes a lane; also its sums
    static constexpr size_t smem = static_cast<size_t>(block * depth + q) * warps;
    static_assert(q == kRowTile * HD * 4, "a warp's sums fit where its q was");
};

// Where piece ch (16 bytes) of key j lies in a block. K: a thread (n, c) of a warp
// reads quarter c of key n; eight threads side by side cover 128 bytes that differ
// in their banks: two keys of 64 bytes; of 128-byte rows the lower half of an even
// key and the upper half of an odd one.
template <int HD> __device__ __forceinline__ int k_at(int j, int ch) {
    if constexpr (HD == 256) ch ^= (j & 1) << 2;
    return j * (HD / 2) + ch * 16;
}
// V: thread (n, c) reads dims of column n of keys 2 c and 2 c + 1. Keys 0, 2, 4, 6
// lie side by side, and pieces change places so that those of the four keys that
// are read together differ.
__device__ __forceinline__ int v_row(int j) { return (j & ~7) | ((j & 1) << 2) | ((j >> 1) & 3); }
template <int HD> __device__ __forceinline__ int v_at(int j, int ch) {
    const int r = v_row(j);
    if constexpr (HD == 128) ch ^= r & 2;
    if constexpr (HD == 256) ch ^= (r & 3) << 1;
    return r * (HD / 2) + ch * 16;
}
// 16 bytes from global to shared memory, both addresses with a constant in the instruction
template <int DST, int SRC> __device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
// BYTES (4, 8 or 16), of which n come from src and the others are zeros
template <int BYTES, int DST, int SRC> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.ca.shared.global [%0+%4], [%1+%5], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n), "n"(DST), "n"(SRC) : "memory");
}
// An arrival at `bar` once this thread's copies so far have landed
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// d = a b, in fp32 from zero
__device__ __forceinline__ void mma16816_0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// The ring: `depth` blocks for each of the CTA's hg.subs sets of warps (one warp a
// head), which take the blocks of a segment in turn. Block k of set x lies in place
// x * depth + k % depth, as S::block bytes for each head.
template <int HD> struct Ring4 {
    uint8_t* smem;
    uint64_t *full, *empty;   // [subs * depth]: every copying thread arrives at full, hg.heads warps at empty
    uint32_t stage;           // bytes of a place
    bool ok;                  // no wait has run out
    __device__ __forceinline__ int place(int x, uint32_t k) const { return x * Rows4Shape<HD>::depth + k % Rows4Shape<HD>::depth; }
    __device__ __forceinline__ uint32_t phase(uint32_t k) const { return (k / Rows4Shape<HD>::depth) & 1u; }
};

// Pieces Y, Y + 1, .. 3 of four, of K and V: piece l + 4 y of a key's row in the pools lies 64 y bytes on, in the ring
// with the head that it is of.
template <int HD, int Y = 0> __device__ __forceinline__ void copy_four(uint32_t k0, uint32_t k1, uint32_t v0, uint32_t v1, const uint4* kp, const uint4* vp, int n) {
    using S = Rows4Shape<HD>;
    if constexpr (Y < 4) {
        constexpr int head = (HD == 64 ? 2 * Y : HD == 128 ? Y : Y / 2) * S::block;
        if (Y < n) {
            copy_async16<head, 64 * Y>(HD == 256 && (Y & 1) ? k1 : k0, kp);
            copy_async16<head, 64 * Y>(HD == 256 && (Y & 1) ? v1 : v0, vp);
        }
        copy_four<HD, Y + 1>(k0, k1, v0, v1, kp, vp, n);
    }
}
// The scales of heads l + 4 Y, .. of a key, up to four.
template <int HD, int Y = 0> __device__ __forceinline__ void copy_scales(uint32_t to, const __half* kp, const __half* vp, int n, int heads) {
    using S = Rows4Shape<HD>;
    if constexpr (Y < 4) {
        if (4 * Y < heads) {
            copy_async<S::srow, 4 * Y * S::block + S::ks, 4 * Y * S::srow>(to, kp, n);
            copy_async<S::srow, 4 * Y * S::block + S::vs, 4 * Y * S::srow>(to, vp, n);
            copy_scales<HD, Y + 1>(to, kp, vp, n, heads);
        }
    }
}

// Copying warp pw: eight keys of every block of a segment, for all heads of the group;
// four lanes a key, so that a copy's addresses are a lane's own plus constants. Lane x
// has `used`, the blocks of set x so far. Where there is no key, or no page, the scales
// are zeros and the codes any.
template <int HD>
__device__ __forceinline__ void copy_segment4(const AttnArgs& A, const Pools4& pools, const HeadGroups& hg, Ring4<HD>& ring, const Segment& seg, int pw,
                                              uint32_t& used) {
    using S = Rows4Shape<HD>;
    const int lane = threadIdx.x & 31, h0 = seg.grp * hg.heads, heads = min(hg.heads, A.c.n_kv - h0);
    const TileView tv = tile_view<kKeys4>(A, seg.tile);
    const int i1 = min(tv.kb.n, seg.b1);
    const int32_t* table = A.c.table + static_cast<int64_t>(tv.sv.slot) * A.c.max_pages;
    const int key = pw * 8 + (lane >> 2), l = lane & 3;
    auto page_of = [&](int i) {
        const int32_t j = tv.kb.at(i) * kKeys4 + key;
        return j < tv.sv.len ? table[A.c.page_div.div(j)] : -1;
    };
    int32_t page = seg.b0 < i1 ? page_of(seg.b0) : -1;
    // this lane's pieces of a row, l, l + 4, ..: with head_dim 64 and an odd head left over, lanes 2 and 3 have one less
    const int pieces = (heads * S::groups + 3 - l) / 4;
    const int my_heads = heads - l;   // scales of heads l, l + 4, ..
    const uint32_t base = smem_addr(ring.smem) + (HD == 64 ? l / 2 * S::block : 0);
    const uint32_t k0 = base + k_at<HD>(key, l % S::groups), v0 = base + S::v + v_at<HD>(key, l % S::groups);
    const uint32_t k1 = HD == 256 ? base + k_at<HD>(key, l + 4) : 0, v1 = HD == 256 ? base + S::v + v_at<HD>(key, l + 4) : 0;
    const uint32_t s0 = smem_addr(ring.smem) + l * S::block + key * S::srow;
    constexpr int four = (HD == 64 ? 8 : HD == 128 ? 4 : 2) * S::block;   // four pieces on in the ring
    for (int i = seg.b0; i < i1; ++i) {
        const int x = (i - seg.b0) & (hg.subs - 1);
        const uint32_t k = __shfl_sync(0xffffffffu, used, x);
        const int at_place = ring.place(x, k);
        const int32_t j = tv.kb.at(i) * kKeys4 + key;
        const bool good = page >= 0 && page < A.c.n_pages;
        if (!good && j < tv.sv.len) record_status(A.status, kStatusBadPosition);
        int64_t at = static_cast<int64_t>(((j - A.c.page_div.div(j) * A.c.page_size) * A.c.n_kv + h0) * S::groups) + page * A.c.page_stride;
        if (!good) at = 0;
        if (i + 1 < i1) page = page_of(i + 1);   // on its way meanwhile
        if (k >= S::depth && ring.ok) ring.ok = mbar_warp_wait(&ring.empty[at_place], ring.phase(k) ^ 1u, A.status, kStatusWaitTimeout);
        if (!ring.ok) return;
        uint32_t to = at_place * ring.stage;
        copy_scales<HD>(s0 + to, pools.ks + at + l * S::groups, pools.vs + at + l * S::groups, good ? S::srow : 0, my_heads);
        const uint4 *kp = pools.k + at + l, *vp = pools.v + at + l;
        int y = good ? pieces : 0;   // no reads of any one place in its stead: 148 CTAs' would meet there (74 sequences of 2 tokens, 32 heads: 23 us)
        for (; y >= 4; y -= 4, to += four, kp += 16, vp += 16) copy_four<HD>(k0 + to, k1 + to, v0 + to, v1 + to, kp, vp, 4);
        if (y > 0) copy_four<HD>(k0 + to, k1 + to, v0 + to, v1 + to, kp, vp, y);
        copy_arrive(&ring.full[at_place]);
        if (lane == x) ++used;
    }
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ __half2 half2_of(uint32_t x) { return half2_bits(prmt(x, x, 0x1010u)); }

// Where 16-byte piece p of row n of q lies among a warp's eight rows: written by the row and read by the thread (n, c)
// of a quarter, both without bank conflicts.
template <int HD> __device__ __forceinline__ int stage_at(int n, int p) {
    return n * (HD / 4) + (p ^ (HD == 64 ? (n & 1) * 2 + (p >> 3) : (n & 1) * 4 + ((p >> 3) & 3)));
}

// This warp's head's attention over its blocks of a segment; the first of the
// head's warps adds up what they have. part < 0: these are all blocks that the rows
// see, and the result goes to out; else (m, l, acc) go to that part. `used`: blocks
// of the warp's set so far. ONE: no tile has more than one row.
template <int HD, bool ONE>
__device__ __forceinline__ void rows4_segment(const AttnArgs& A, const HeadGroups& hg, Ring4<HD>& ring, uint32_t& used, uint8_t* own, float2 (*s_ml)[kRowTile],
                                              const Segment& seg, const TileView& tv, int part) {
    using S = Rows4Shape<HD>;
    constexpr int KW = HD / 32;                  // words of codes of a key's quarter: two k-steps of Q K^T each
    constexpr int VW = HD / 64;                  // words of codes of a column's dims
    constexpr int NT = HD / 8;                   // column tiles of P V
    constexpr int KT = kKeys4 / 8;               // column tiles of Q K^T
    constexpr int PIECES = HD / 4, STEPS = kRowTile * PIECES / 32;   // 16-byte pieces of a row of q; what a lane has of the warp's eight rows
    float4* const stage = reinterpret_cast<float4*>(own);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, c = lane & 3;
    const int sub = hg.sub_of(warp), hl = warp - sub * hg.heads, kvh = seg.grp * hg.heads + hl;
    const SeqView& sv = tv.sv;
    const Mask& mask = tv.mask;
    const int i1 = min(tv.kb.n, seg.b1);
    if (kvh >= A.c.n_kv) {   // a head that the last group does not have: nothing but to keep the ring going
        for (int i = seg.b0 + sub; i < i1; i += hg.subs, ++used) {
            const int at = ring.place(sub, used);
            if (ring.ok) ring.ok = mbar_warp_wait(&ring.full[at], ring.phase(used), A.status, kStatusWaitTimeout);
            if (!ring.ok) return;
            if (lane == 0) mbar_arrive(&ring.empty[at]);
        }
        return;
    }

    // this thread's row and position
    const int r = tv.r0 + n;
    const bool row_ok = r < tv.n_rows;
    const int rc = min(r, tv.n_rows - 1), t = A.group_div.div(rc), h = kvh * A.group + rc - t * A.group;
    const int32_t pos = tv.base + t;
    const RowKeys keys = mask.row(pos);
    // a block [j0, j0 + kKeys4) is seen by every row where it lies in [all_lo, all_hi) or before the prefix's end
    const int32_t all_hi = min(mask.len, tv.p_lo + 1), all_lo = mask.window > 0 ? tv.p_hi - mask.window + 1 : 0;

    // ---- q as hi and lo halves of q * 2^-e, max |q| 2^-e in [2^14, 2^15), in the order of the codes' pairs ----
    const uint32_t qs = smem_addr(own) + lane * 16;
    float qscale;   // 2^e; NaN for a row that is not finite, unless it sees no key: its zeros have no q
    {
        const float* q = A.q + static_cast<int64_t>(sv.q0 + t) * A.ldq + static_cast<int64_t>(h) * HD;
        if constexpr (!ONE) {   // whole rows at a time: a thread's own dims are a line of their own in each load, 1 us for eight heads of eight rows
            float4 y[STEPS];
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const int row = (k * 32 + lane) / PIECES, piece = (k * 32 + lane) % PIECES;
                const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(q), 4 * row));
                y[k] = tv.r0 + row < tv.n_rows ? reinterpret_cast<const float4*>(from)[piece] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) stage[stage_at<HD>((k * 32 + lane) / PIECES, (k * 32 + lane) % PIECES)] = y[k];
            __syncwarp();
        }
        float v[KW][8];
        float mx = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            const int d = HD == 256 ? 32 * (c + (w & 4)) + 8 * (w & 3) : (HD / 4) * c + 8 * w;
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *reinterpret_cast<float4*>(v[w] + i) = !ONE     ? stage[stage_at<HD>(n, (d + i) / 4)]
                                                       : row_ok ? *reinterpret_cast<const float4*>(q + d + i)
                                                                : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmax_nan(mx, fabsf(v[w][i]));
        }
        mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (!ONE) __syncwarp();   // every lane has its dims
        const bool fin = mx < INFINITY;
        int e = 0;
        if (fin && mx > 0.f) e = ilogbf(mx) - 14;
        // two factors, so that 2^-e stays finite for the smallest subnormal q
        const float f1 = ldexpf(1.f, -(e / 2)), f2 = fin ? ldexpf(1.f, -(e - e / 2)) : 0.f;
        qscale = fin || (keys.hi <= keys.lo && keys.prefix <= 0) ? ldexpf(1.f, e) : NAN;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                uint32_t a[4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float x = fin ? v[w][i + k] * f1 * f2 : 0.f, y = fin ? v[w][i + k + 4] * f1 * f2 : 0.f;
                    split_half2(x, y, a[2 * k], a[2 * k + 1]);
                }
                sts128(qs + (2 * w + (i >> 1)) * 512, a);   // read by this lane alone
            }
    }
    const float sc = A.cap2 != 0.f ? qscale : qscale * A.scale2;
    const float slope2 = A.slopes ? A.slopes[h] * 1.44269504088896341f : 0.f;
    // Scores and their maximum are kept as the products come out, a score being `unit` of them; with a cap or a bias they
    // are scaled first, and the unit is 1.
    const bool plain = A.cap2 == 0.f && A.slopes == nullptr;
    const float unit = plain ? (sc == 0.f ? FLT_MIN : sc) : 1.f;   // a unit of 0 would make NaN of a hidden key's -inf

    float m = -INFINITY, l = -0.f;   // l stays -0 until there is a block, whose sums are never below +0
    float2 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = make_float2(0.f, 0.f);
    const int vg = n * HD / 256;   // the group of this thread's column's dims

    for (int i = seg.b0 + sub; i < i1; i += hg.subs, ++used) {
        const int at = ring.place(sub, used);
        if (ring.ok) ring.ok = mbar_warp_wait(&ring.full[at], ring.phase(used), A.status, kStatusWaitTimeout);
        if (!ring.ok) break;
        uint8_t* const block = ring.smem + at * ring.stage + hl * S::block;
        const uint32_t st = smem_addr(block);
        const int32_t j0 = tv.kb.at(i) * kKeys4;

        // ---- scores of keys 8 x + 2 c, + 1 ----
        float s[KT][4];
#pragma unroll
        for (int p = 0; p < (HD == 256 ? 2 : 1); ++p) {
            uint32_t w[KT][HD == 64 ? 2 : 4];
            __half2 d[KT];
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                const int key = 8 * x + n;
                if constexpr (HD == 64) {
                    const uint2 y = lds64(st + k_at<HD>(key, 0) + c * 8);
                    w[x][0] = y.x;
                    w[x][1] = y.y;
                } else {
                    const uint4 y = lds128(st + k_at<HD>(key, c + 4 * p));
                    w[x][0] = y.x;
                    w[x][1] = y.y;
                    w[x][2] = y.z;
                    w[x][3] = y.w;
                }
                d[x] = half2_of(lds16(st + S::ks + key * S::srow + (HD == 64 ? c >> 1 : c + 4 * p) * 2));
            }
#pragma unroll
            for (int y = 0; y < (HD == 64 ? 2 : 4); ++y) {
                const uint4 a0 = lds128(qs + 2 * (4 * p + y) * 512), a1 = lds128(qs + (2 * (4 * p + y) + 1) * 512);
                const uint32_t q0[4] = {a0.x, a0.y, a0.z, a0.w}, q1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
                for (int x = 0; x < KT; ++x) {
                    uint32_t b[4];
                    code_pairs(w[x][y], d[x], b);
                    if (p == 0 && y == 0) mma16816_0(s[x], q0, b[0], b[1]);
                    else mma16816(s[x], q0, b[0], b[1]);
                    mma16816(s[x], q1, b[2], b[3]);
                }
            }
        }
        float2 sx[KT];
#pragma unroll
        for (int x = 0; x < KT; ++x) sx[x] = fadd2(make_float2(s[x][0], s[x][1]), make_float2(s[x][2], s[x][3]));
        if (!plain) {
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                sx[x].x *= sc;
                sx[x].y *= sc;
                if (A.cap2 != 0.f) {
                    sx[x].x = capped(sx[x].x, A.cap2, A.cap_in);
                    sx[x].y = capped(sx[x].y, A.cap2, A.cap_in);
                }
            }
        }
        const int32_t jc = j0 + 2 * c;   // this thread's keys: jc + 8 x + k
        if (A.slopes) {
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                sx[x].x -= slope2 * fabsf(static_cast<float>(pos - (jc + 8 * x)));
                sx[x].y -= slope2 * fabsf(static_cast<float>(pos - (jc + 8 * x + 1)));
            }
        }
        if (!((j0 >= all_lo && j0 + kKeys4 <= all_hi) || j0 + kKeys4 <= mask.prefix)) {
#pragma unroll
            for (int x = 0; x < KT; ++x) {
                if (!keys.sees(jc + 8 * x)) sx[x].x = -INFINITY;
                if (!keys.sees(jc + 8 * x + 1)) sx[x].y = -INFINITY;
            }
            // A key that some row does not see has P = 0 there, which would make NaN of a
            // scale that is not finite. Such groups (there are none in a sound cache) are
            // added where they are seen and then cleared, so that they reach no other row.
            uint32_t odd = 0;
#pragma unroll
            for (int x = 0; x < S::srow / 4; ++x) odd |= nonfinite_mark(lds32(st + S::vs + lane * S::srow + 4 * x));
            if (__any_sync(0xffffffffu, (odd & kNonfinite) != 0)) {
                __half* vs = reinterpret_cast<__half*>(block + S::vs);
                for (int j = 0; j < kKeys4; ++j) {
                    if (!keys.sees(j0 + j)) continue;
#pragma unroll
                    for (int k = 0; k < 2; ++k)   // the columns 2 c + k of this thread's sums
                        if (!isfinite(__half2float(vs[j * S::groups + (2 * c + k) * HD / 256]))) {
#pragma unroll
                            for (int x = 0; x < NT; ++x) (k ? acc[x].y : acc[x].x) = NAN;
                        }
                }
                __syncwarp();
                for (int x = lane; x < kKeys4 * S::groups; x += 32)
                    if (!isfinite(__half2float(vs[x]))) vs[x] = __float2half_rn(0.f);
                __syncwarp();
            }
        }
        float mx = m;
#pragma unroll
        for (int x = 0; x < KT; ++x) mx = fmaxf(mx, fmaxf(sx[x].x, sx[x].y));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float ms = mx == -INFINITY ? 0.f : mx;   // nothing seen yet: P = 2^-inf = 0
        const float corr = m == -INFINITY ? 0.f : ex2((m - ms) * unit);
        m = mx;
        const float2 less = make_float2(-ms, -ms), by = make_float2(unit, unit), up = make_float2(kPShift, kPShift);
        uint32_t pa[KT / 2][4];
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int x = 0; x < KT; ++x) {
            const float2 e = ffma2(fadd2(sx[x], less), by, up), pr = make_float2(ex2(e.x), ex2(e.y));
            sum = fadd2(sum, pr);
            split_half2(pr.x, pr.y, pa[x >> 1][2 * (x & 1)], pa[x >> 1][2 * (x & 1) + 1]);
        }
        l = fmaf(l, corr, sum.x + sum.y);

        // ---- P V: keys 2 c, + 1, + 8, + 9 of each 16, dims of column n ----
        uint32_t vw[kKeys4 / 4][VW];   // [k-step, + 8, second of the pair]
        __half2 vd[KT], vm[KT];
#pragma unroll
        for (int x = 0; x < KT; ++x) {
            uint32_t d16[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int key = 8 * x + 2 * c + k;
                if constexpr (HD == 64) vw[2 * x + k][0] = lds32(st + S::v + v_at<HD>(key, n >> 2) + (n & 3) * 4);
                if constexpr (HD == 128) {
                    const uint2 y = lds64(st + S::v + v_at<HD>(key, n >> 1) + (n & 1) * 8);
                    vw[2 * x + k][0] = y.x;
                    vw[2 * x + k][1] = y.y;
                }
                if constexpr (HD == 256) {
                    const uint4 y = lds128(st + S::v + v_at<HD>(key, n));
                    vw[2 * x + k][0] = y.x;
                    vw[2 * x + k][1] = y.y;
                    vw[2 * x + k][2] = y.z;
                    vw[2 * x + k][3] = y.w;
                }
                d16[k] = lds16(st + S::vs + key * S::srow + vg * 2);
            }
            vd[x] = half2_bits(prmt(d16[0], d16[1], 0x5410u));
            vm[x] = __hmul2(vd[x], __float2half2_rn(-24.f));
        }
#pragma unroll
        for (int y = 0; y < 2 * VW; ++y) {   // four dims of the column
            float o[4][4];
#pragma unroll
            for (int x = 0; x < KT; x += 2) {
                uint32_t b0[4], b1[4];
                code_pairs_fma(prmt(vw[2 * x][y >> 1], vw[2 * x + 1][y >> 1], (y & 1) ? 0x7632u : 0x5410u), vd[x], vm[x], b0);
                code_pairs_fma(prmt(vw[2 * x + 2][y >> 1], vw[2 * x + 3][y >> 1], (y & 1) ? 0x7632u : 0x5410u), vd[x + 1], vm[x + 1], b1);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (x == 0) mma16816_0(o[k], pa[0], b0[k], b1[k]);
                    else mma16816(o[k], pa[x >> 1], b0[k], b1[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                acc[4 * y + k] = ffma2(acc[4 * y + k], make_float2(corr, corr), fadd2(make_float2(o[k][0], o[k][1]), make_float2(o[k][2], o[k][3])));
            }
        }
        __syncwarp();   // every lane has read the block
        if (lane == 0) mbar_arrive(&ring.empty[at]);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    m = m == -INFINITY ? m : m * unit;
    if (hg.subs > 1) {
        // the other warps' sums in the place of their q, 16 bytes a lane at a time
        float4* mine = reinterpret_cast<float4*>(own) + lane;
        if (sub > 0) {
#pragma unroll
            for (int x = 0; x < NT; x += 2) mine[x * 16] = make_float4(acc[x].x, acc[x].y, acc[x + 1].x, acc[x + 1].y);
            if (c == 0) s_ml[warp][n] = make_float2(m, l);
        }
        named_barrier(1 + hl, hg.subs * 32);
        if (sub == 0) {
            for (int y = 1; y < hg.subs; ++y) {
                const int w = y * hg.heads + hl;
                const float2 ml = s_ml[w][n];
                if (__float_as_uint(ml.y) == 0x80000000u) break;   // a warp without a block, and so are those behind it
                const float4* theirs = mine + (w - hl) * (S::q / 16);
                const float top = fmaxf(m, ml.x);
                // a part that saw nothing adds zeros, or the NaN of a row that is not finite
                const float f0 = m == -INFINITY ? 1.f : ex2(m - top), f1 = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);
                m = top;
                l = fmaf(l, f0, ml.y * f1);
                const float2 g0 = make_float2(f0, f0), g1 = make_float2(f1, f1);
#pragma unroll
                for (int x = 0; x < NT; x += 2) {
                    const float4 v = theirs[x * 16];
                    const float2 z = make_float2(0.f, 0.f);
                    acc[x] = ffma2(make_float2(v.x, v.y), g1, ffma2(acc[x], g0, z));
                    acc[x + 1] = ffma2(make_float2(v.z, v.w), g1, ffma2(acc[x + 1], g0, z));
                }
            }
        }
        named_barrier(1 + hl, hg.subs * 32);   // read: q may be written again
        if (sub > 0) return;
    }
    if (!row_ok) return;
    float* o;
    float inv = 1.f;
    if (part < 0) {
        o = A.out + static_cast<int64_t>(sv.q0 + t) * A.ldo + static_cast<int64_t>(h) * HD;
        inv = l == 0.f ? 0.f : 1.f / l;   // nothing seen: zeros
    } else {
        const int64_t at_row = (static_cast<int64_t>(part) * S::warps + hl) * kRowTile + n;
        float* ml = A.part + S::cut_bytes / 4;
        if (c == 0) *reinterpret_cast<float2*>(ml + at_row * 2) = make_float2(m, l);
        o = ml + S::part_rows(2 * kRowsCtas) * 2 + at_row * HD;
    }
#pragma unroll
    for (int x = 0; x < NT; x += 4) {
        *reinterpret_cast<float4*>(o + 2 * c * NT + x) = make_float4(acc[x].x * inv, acc[x + 1].x * inv, acc[x + 2].x * inv, acc[x + 3].x * inv);
        *reinterpret_cast<float4*>(o + (2 * c + 1) * NT + x) = make_float4(acc[x].y * inv, acc[x + 1].y * inv, acc[x + 2].y * inv, acc[x + 3].y * inv);
    }
}

// hg: heads and sets of warps. What is added up later has one part a head (its warps have added up theirs), as if one
// warp had it: `whole`.
template <int HD, bool ONE>
__global__ void __launch_bounds__(Rows4Shape<HD>::threads, 1)
rows4_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ Pools4 pools, const __grid_constant__ HeadGroups hg,
             const __grid_constant__ HeadGroups whole) {
    using S = Rows4Shape<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_pre[kMostTiles + 1];
    __shared__ int64_t s_sum[S::warps + kCopyWarps4];
    __shared__ __align__(8) uint64_t s_full[S::warps * S::depth], s_empty[S::warps * S::depth];
    __shared__ float2 s_ml[S::warps][kRowTile];
    const int warp = threadIdx.x >> 5, tiles = A.n_split, cta = blockIdx.x;
    if (threadIdx.x == 0) {
        for (int i = 0; i < hg.subs * S::depth; ++i) {
            mbar_init(&s_full[i], kCopyWarps4 * 32);
            mbar_init(&s_empty[i], hg.heads);
        }
        s_pre[0] = 0;
        fence_mbar_init();
    }
    grid_dep_wait();
    grid_dep_launch();   // combine_kernel may be set up meanwhile; it waits for this grid's end
    const int64_t units = tile_units<S::warps + kCopyWarps4, kKeys4>(A, hg, tiles, s_pre, s_sum) * hg.groups;
    const Runs runs(units, gridDim.x, hg.least);
    const bool listed_by_tile = by_tile(tiles, whole);
    Cut* cuts = reinterpret_cast<Cut*>(A.part);
    int64_t u = 0, end = 0;
    if (units > 0 && cta < runs.n_cta) {
        u = runs.start(cta);
        end = runs.start(cta + 1);
    }
    const int64_t begin = u;
    int lo = tile_at(s_pre, hg, tiles, u);
    Ring4<HD> ring{smem + S::q * S::warps, s_full, s_empty, static_cast<uint32_t>(hg.heads * S::block), true};
    Segment seg;
    if (warp >= S::warps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::copy_regs));
        uint32_t used = 0;
        while (ring.ok && next_segment(s_pre, hg, u, end, lo, seg)) copy_segment4<HD>(A, pools, hg, ring, seg, warp - S::warps, used);
        asm volatile("cp.async.wait_all;" ::: "memory");   // nothing may be in flight when the CTA ends
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::regs));
    if (listed_by_tile && cta == 0)   // those without rows
        for (int i = threadIdx.x; i < tiles * hg.groups; i += S::warps * 32)
            if (s_pre[i / hg.groups + 1] == s_pre[i / hg.groups]) cuts[i] = Cut{};
    const int sub = hg.sub_of(warp);
    uint32_t used = 0;
    Cut cut{};
    while (next_segment(s_pre, hg, u, end, lo, seg)) {
        const int c_first = runs.cta_of(seg.first + hg.cost), c_last = runs.cta_of(seg.first + seg.units - 1);
        const TileView tv = tile_view<kKeys4>(A, seg.tile);
        const Cut all{seg.grp, 2 * c_first + (runs.start(c_first) >= seg.first ? 0 : 1), c_last - c_first + 1, min(kRowTile, tv.n_rows - tv.r0), tv.r0, tv.sv.q0};
        if (cta == c_first + 1) cut = all;
        if (listed_by_tile && cta == c_first && threadIdx.x == 0) cuts[seg.tile * hg.groups + seg.grp] = all;
        if (sub < hg.subs) rows4_segment<HD, ONE>(A, hg, ring, used, smem + warp * S::q, s_ml, seg, tv, c_first == c_last ? -1 : 2 * cta + (begin >= seg.first ? 0 : 1));
    }
    if (!listed_by_tile && threadIdx.x == 0) cuts[cta] = cut;
}

// ---- chunks: a cache of fp16 pages, sequence i in slot i ----

struct Scratch {
    __half* k;
    __half* v;
    int32_t* table;     // [n_seq][pages]: page i * pages + x of slot i
    int32_t* seq_len;   // -1 for a sequence that is not sound
    int32_t pages;
};

// Blocks x of gridDim.x share out one sequence's tokens that its rows see, `tokens`
// (at most 64) at a time, and write the sequence's entries of the tables. A thread has
// a word of the row (or several, 256 apart; where rows are short, that word of every
// second, third .. token), and takes it of K and of V, kExpandSteps tokens or words
// under way.
constexpr int kExpandSteps = 4;
constexpr int kExpandTokens = 64;

__global__ void __launch_bounds__(256)
expand_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ Pools4 pools, const __grid_constant__ Scratch w, int tokens) {
    __shared__ int64_t s_from[kExpandTokens];   // first group of the token's K, -1: no page
    grid_dep_wait();
    grid_dep_launch();
    const int seq = blockIdx.y;
    const SeqView sv = seq_view(A.c, A.b, seq);
    for (int x = blockIdx.x * blockDim.x + threadIdx.x; x < w.pages; x += gridDim.x * blockDim.x)
        w.table[static_cast<int64_t>(seq) * w.pages + x] = seq * w.pages + x;
    if (blockIdx.x == 0 && threadIdx.x == 0) w.seq_len[seq] = sv.ok ? sv.len : -1;
    if (!sv.ok || sv.n_new == 0) return;
    const int32_t prefix = A.prefix ? max(0, min(A.prefix[seq], sv.len)) : 0;
    const int32_t first = A.window > 0 ? max(0, sv.len - sv.n_new + 1 - A.window) : 0;   // the first key in a window
    const int row_words = A.c.n_kv * A.c.head_dim / 8;
    const int abreast = max(1, 256 / row_words);                        // tokens that the block's threads take at a time
    const int tok = row_words < 256 ? threadIdx.x / row_words : 0, word = threadIdx.x - tok * row_words;
    const int32_t* table = A.c.table + static_cast<int64_t>(sv.slot) * A.c.max_pages;
    const int64_t base = static_cast<int64_t>(seq) * w.pages * kScratchPage;
    // whole pages, which hold the chunk kernel's blocks: what no row sees of a page that some row sees is zeros, since values
    // that are not finite, as scratch may hold, send a block the slow way (1092 new tokens, 12 heads on 2: 65 us instead of 30)
    const int32_t from_page = first & ~(kScratchPage - 1);
    const int64_t to_page = (static_cast<int64_t>(prefix) + kScratchPage - 1) & ~int64_t(kScratchPage - 1);
    const int64_t end = (static_cast<int64_t>(sv.len) + kScratchPage - 1) & ~int64_t(kScratchPage - 1);
    for (int64_t start = static_cast<int64_t>(blockIdx.x) * tokens; start < end; start += static_cast<int64_t>(gridDim.x) * tokens) {
        const int n = static_cast<int>(min(static_cast<int64_t>(tokens), end - start));
        if (start + n <= from_page && start >= to_page) continue;
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < n) {
            const int64_t at = start + threadIdx.x;
            int64_t from = -1;
            if (at < sv.len && (at >= first || at < prefix)) {   // what no row sees is not looked at
                const int32_t j = static_cast<int32_t>(at), pi = A.c.page_div.div(j), page = table[pi];
                if (page >= 0 && page < A.c.n_pages) from = page * A.c.page_stride + static_cast<int64_t>(j - pi * A.c.page_size) * (row_words / 4);
                else record_status(A.status, kStatusBadPosition);
            }
            s_from[threadIdx.x] = from;
        }
        __syncthreads();
        if (tok >= abreast) continue;
        int t = tok, at = word;   // the next token and word
        while (t < n) {
            uint32_t code[2][kExpandSteps];
            __half d[2][kExpandSteps];
            int64_t to[kExpandSteps];
#pragma unroll
            for (int x = 0; x < kExpandSteps; ++x) {
                to[x] = -1;
                if (t >= n) continue;
                const int64_t from = s_from[t];
                to[x] = (base + start + t) * row_words + at;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    code[p][x] = 0x88888888u;
                    d[p][x] = __float2half_rn(0.f);
                    if (from >= 0) {
                        code[p][x] = __ldcs(reinterpret_cast<const uint32_t*>((p ? pools.v : pools.k) + from) + at);
                        d[p][x] = ((p ? pools.vs : pools.ks) + from)[at / 4];
                    }
                }
                at += 256;
                if (at >= row_words) {
                    at = word;
                    t += abreast;
                }
            }
#pragma unroll
            for (int x = 0; x < kExpandSteps; ++x) {
                if (to[x] < 0) continue;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    uint32_t v[4];
                    code_pairs(code[p][x], __half2half2(d[p][x]), v);   // (0, 4) (1, 5) (2, 6) (3, 7)
                    reinterpret_cast<uint4*>(p ? w.v : w.k)[to[x]] = make_uint4(prmt(v[0], v[1], 0x5410u), prmt(v[2], v[3], 0x5410u),
                                                                               prmt(v[0], v[1], 0x7632u), prmt(v[2], v[3], 0x7632u));
                }
            }
        }
    }
}

struct Plan4 {
    bool chunk;
    int heads, per_seq, tiles;   // rows4_kernel
    int n_seq, pages;            // chunk: sequences at a time, pages of each
};

int warps4(int head_dim) { return head_dim == 256 ? Rows4Shape<256>::warps : Rows4Shape<128>::warps; }

// Whether groups of half as many heads, with `subs` warps a head, are better: for few
// segments, (tile, group)s, since each costs a start, and few blocks, since copies of
// fewer heads are narrower. 8 heads of 128 a group and 4: one sequence of 30000
// tokens, 64 heads on 8, 32 us and 27, two of 131072 and 100001 100 and 104, eight of
// up to 8192 22.5 and 19.1, 32 of them 33.5 and 33.2, 32 of 8192 99.8 and 106; 32 heads, ten of up to 1000 22.1
// and 23.1, 14 of 2 tokens 11.7 and 13.2 (16 heads: 14.2, 2: 18.1). Groups of 2: one of
// 2048, 64 heads on 8, 15.8 and 15.0, 32 heads 14.6 and 15.5.
bool halve_heads(int64_t segments, int64_t blocks, int subs) {
    const int64_t work = segments * blocks;
    if (subs > 4) return segments <= 16 && work <= 1000;
    return (segments <= 32 && work <= 8192) || (segments <= 64 && (work <= kRowsCtas));
}

// How a call is cut: from the host's bounds alone, so that a captured graph
// serves every later length within them.
Plan4 make_plan4(const hesa_cuda_paged_kv4* kv, const hesa_cuda_token_batch* b, int64_t n_head) {
    Plan4 p{};
    const int g = static_cast<int>(n_head / kv->n_kv_head);
    const int64_t rows_a_seq = static_cast<int64_t>(b->max_new) * g;
    p.chunk = rows_a_seq > kMostRows4;
    if (p.chunk) {
        p.pages = std::max(1, (b->max_len + kScratchPage - 1) / kScratchPage);
        const int64_t bytes = static_cast<int64_t>(p.pages) * kScratchPage * kv->n_kv_head * kv->head_dim * 4;
        p.n_seq = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(b->n_seq, kScratchBytes / bytes)));
        return p;
    }
    const int64_t most = (rows_a_seq + kRowTile - 1) / kRowTile;
    const int64_t bound = tile_bound(b->n_tokens, b->n_seq, g, kRowTile);
    p.per_seq = b->n_seq * most <= bound ? static_cast<int>(most) : 0;
    const int64_t tiles = p.per_seq ? b->n_seq * most : bound;
    p.tiles = static_cast<int>(tiles);
    const int64_t blocks = std::max<int64_t>(1, (b->max_len + kKeys4 - 1) / kKeys4);
    static_assert(4 * kRowsCtas <= kMostTiles, "a list for every (tile, group) where groups are made smaller");
    p.heads = warps4(kv->head_dim);
    while (p.heads > 2 && halve_heads(tiles * ((kv->n_kv_head + p.heads / 2 - 1) / (p.heads / 2)), blocks, warps4(kv->head_dim) / (p.heads / 2))) p.heads /= 2;
    return p;
}

size_t round16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// The chunk's scratch in the workspace: pools, table, lengths, then the chunk kernel's own.
struct ScratchSizes {
    size_t pool, table, len;
    size_t all() const { return 2 * pool + table + len; }
};
ScratchSizes scratch_sizes(const hesa_cuda_paged_kv4* kv, const Plan4& p) {
    const size_t pages = static_cast<size_t>(p.n_seq) * p.pages;
    return {pages * kScratchPage * kv->n_kv_head * kv->head_dim * 2, round16(pages * 4), round16(static_cast<size_t>(p.n_seq) * 4)};
}
hesa_cuda_paged_kv scratch_kv(const hesa_cuda_paged_kv4* kv, const Plan4& p, uint8_t* ws) {
    const ScratchSizes z = scratch_sizes(kv, p);
    hesa_cuda_paged_kv s{};
    s.k = ws;
    s.v = ws + z.pool;
    s.table = reinterpret_cast<int32_t*>(ws + 2 * z.pool);
    s.seq_len = reinterpret_cast<int32_t*>(ws + 2 * z.pool + z.table);
    s.page_stride = static_cast<int64_t>(kScratchPage) * kv->n_kv_head * kv->head_dim;
    s.n_layer = 1;
    s.n_pages = p.n_seq * p.pages;
    s.page_size = kScratchPage;
    s.n_kv_head = kv->n_kv_head;
    s.head_dim = kv->head_dim;
    s.n_slots = p.n_seq;
    s.max_pages = p.pages;
    return s;
}

// What the chunk kernel needs beside the scratch: the most that any of the passes over the batch takes. The last pass may
// have fewer sequences than the others, whose keys are then split over more CTAs, in parts that take room. 0: the copy would be no cache.
size_t inner_bytes(const hesa_cuda_paged_kv4* kv, const Plan4& p, const hesa_cuda_token_batch* batch, int64_t n_head) {
    const hesa_cuda_paged_kv s = scratch_kv(kv, p, reinterpret_cast<uint8_t*>(uintptr_t(16)));   // not looked into
    hesa_cuda_token_batch b = *batch;
    b.slots = nullptr;
    size_t most = 0;
    for (const int n : {p.n_seq, batch->n_seq % p.n_seq}) {
        if (n == 0) continue;
        b.n_seq = n;
        const size_t need = hesa_cuda_paged_attention_workspace_size(&s, &b, n_head);
        if (need == 0) return 0;
        most = std::max(most, need);
    }
    return most;
}

// As what is added up later sees them: a head's warps have added up theirs.
HeadGroups one_warp_a_head(HeadGroups hg) {
    hg.subs = 1;
    hg.sub_bits = 0;
    return hg;
}

size_t rows4_bytes(const hesa_cuda_paged_kv4* kv) {
    const int64_t parts = 2 * kRowsCtas;
    return kv->head_dim == 64 ? Rows4Shape<64>::bytes(parts) : kv->head_dim == 128 ? Rows4Shape<128>::bytes(parts) : Rows4Shape<256>::bytes(parts);
}

template <int HD, bool ONE>
cudaError_t launch_rows4(AttnArgs a, const Pools4& pools, const Plan4& p, cudaStream_t s) {
    static bool set[64] = {};   // per instance and device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    using S = Rows4Shape<HD>;
    if (!set[dev]) {
        e = cudaFuncSetAttribute(rows4_kernel<HD, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::smem));
        if (e != cudaSuccess) return e;
        set[dev] = true;
    }
    HeadGroups hg(a.c.n_kv, S::warps, p.heads, kSegCost4);
    hg.cost = std::min(hg.cost, kSegCostMost4);
    if (hg.subs < 4) hg.least = 2;   // a start and a block are few units: 40 sequences of 2 tokens, 32 heads 16.9 us, with 4 22.8
    const HeadGroups whole = one_warp_a_head(hg);
    for (a.tile0 = 0; a.tile0 < p.tiles && e == cudaSuccess; a.tile0 += kMostTiles) {
        a.n_split = std::min(kMostTiles, p.tiles - a.tile0);
        e = launch_dep(rows4_kernel<HD, ONE>, dim3(kRowsCtas), S::threads, S::smem, s, a, pools, hg, whole);
        const int cuts = by_tile(a.n_split, whole) ? a.n_split * hg.groups : kRowsCtas;
        const int rows = std::min(kRowTile, a.b.max_new * a.group);
        const unsigned z = static_cast<int64_t>(cuts) * hg.heads * rows <= 8 * kRowsCtas ? rows : 1;
        if (e == cudaSuccess)
            e = launch_dep(combine_kernel<HD, S::warps>, dim3(static_cast<unsigned>(cuts), static_cast<unsigned>(hg.heads), z), 256, 0, s, a, whole);
    }
    return e;
}

}  // namespace
}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_paged_attention_kv4_workspace_size(const hesa_cuda_paged_kv4* kv, const hesa_cuda_token_batch* batch, int64_t n_head) {
    if (check_paged_kv4(kv) != HESA_CUDA_OK || check_batch4(kv, 0, batch, n_head) != HESA_CUDA_OK) return 0;
    const Plan4 p = make_plan4(kv, batch, n_head);
    if (!p.chunk) return std::max<size_t>(rows4_bytes(kv), 16);
    const size_t inner = inner_bytes(kv, p, batch, n_head);
    return inner ? scratch_sizes(kv, p).all() + inner : 0;
}

int hesa_cuda_paged_attention_kv4(const hesa_cuda_paged_kv4* kv, int32_t layer, const hesa_cuda_token_batch* batch, const float* q,
                                  int64_t ldq, float* out, int64_t ldo, int64_t n_head, const hesa_cuda_attn_options* options,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_paged_attention_kv4");
    int rc = check_paged_kv4(kv);
    if (rc == HESA_CUDA_OK) rc = check_batch4(kv, layer, batch, n_head);
    if (rc != HESA_CUDA_OK) return rc;
    if (batch->n_tokens == 0) return HESA_CUDA_OK;   // no rows: their buffers may be null
    hesa_cuda_attn_options o{};
    if (options) o = *options;
    AttnArgs a{};
    rc = attention_args(kv->head_dim, kv->n_kv_head, batch, q, ldq, out, ldo, n_head, options, workspace, &a);
    if (rc != HESA_CUDA_OK) return rc;
    const size_t need = hesa_cuda_paged_attention_kv4_workspace_size(kv, batch, n_head);
    if (need == 0) return HESA_CUDA_SHAPE_MISMATCH;   // a chunk's copy that would be no cache; the message is there
    if (workspace_bytes < need) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    if (batch->max_new == 0) return HESA_CUDA_OK;

    const Plan4 p = make_plan4(kv, batch, n_head);
    const Pools4 pools = pools_of(kv, layer);
    a.c = layer_of4(kv);
    a.per_seq = p.per_seq;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = status_word(&a.status);
    if (e == cudaSuccess && p.chunk) {
        uint8_t* ws = static_cast<uint8_t*>(workspace);
        hesa_cuda_paged_kv c = scratch_kv(kv, p, ws);
        const size_t used = scratch_sizes(kv, p).all();
        hesa_cuda_token_batch b = *batch;
        b.slots = nullptr;
        for (int i = 0; i < batch->n_seq; i += p.n_seq) {
            b.n_seq = std::min(p.n_seq, batch->n_seq - i);
            b.q_start = batch->q_start + i;
            a.b.n_seq = b.n_seq;
            a.b.q_start = b.q_start;
            a.b.slots = batch->slots ? batch->slots + i : nullptr;
            PagedLayer& l = a.c;
            if (!batch->slots) {   // sequence i is in slot i
                l.table = kv->table + static_cast<int64_t>(i) * kv->max_pages;
                l.seq_len = kv->seq_len + i;
                l.n_slots = kv->n_slots - i;
            }
            o.prefix = options && options->prefix ? options->prefix + i : nullptr;
            a.prefix = o.prefix;
            // as many tokens a block as its threads have words under way for, but fewer, down to four, where there are not four
            // blocks for every SM: 49 tokens of eight sequences of up to 262, 64 heads on 8, 22.0 us (up to 16 tokens whatever
            // their number 24.6), one sequence of 45194, 8 heads on 1, 36.2 (39.1)
            const int row_words = kv->n_kv_head * kv->head_dim / 8, most = std::max(1, std::min(kExpandTokens, kExpandSteps * 256 / row_words));
            const int tokens = static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(4, static_cast<int64_t>(b.n_seq) * batch->max_len / (148 * 4))));
            const int share = std::max(1, std::min((batch->max_len + tokens - 1) / tokens, (148 * 16 + b.n_seq - 1) / b.n_seq));
            e = launch_dep(expand_kernel, dim3(static_cast<unsigned>(share), static_cast<unsigned>(b.n_seq)), 256, 0, s, a, pools,
                           Scratch{static_cast<__half*>(c.k), static_cast<__half*>(c.v), c.table, c.seq_len, p.pages}, tokens);
            if (e != cudaSuccess) break;
            rc = hesa_cuda_paged_attention(&c, 0, &b, q, ldq, out, ldo, n_head, &o, ws + used, workspace_bytes - used, stream);
            if (rc != HESA_CUDA_OK) return rc;
        }
    } else if (e == cudaSuccess) {
        const bool one = batch->max_new == 1 && a.group == 1;   // 74 sequences of 2 tokens, 32 heads: 14.2 us, with the code for eight rows 14.7
        switch (kv->head_dim) {
            case 64: e = one ? launch_rows4<64, true>(a, pools, p, s) : launch_rows4<64, false>(a, pools, p, s); break;
            case 128: e = one ? launch_rows4<128, true>(a, pools, p, s) : launch_rows4<128, false>(a, pools, p, s); break;
            default: e = one ? launch_rows4<256, true>(a, pools, p, s) : launch_rows4<256, false>(a, pools, p, s); break;
        }
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "paged attention kernel");
}

}  // extern "C"
