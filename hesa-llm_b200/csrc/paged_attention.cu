// paged_attention.cu -- attention of new tokens over a paged fp16 cache.
//
//   out[r] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),
//   s_j = log2(e) (cap(scale q . k_j) - slope |pos - j|) over the keys j that
//   row r sees, m their maximum.
//
// A row is one query head of one new token; the g = n_head / n_kv heads of a kv
// head and the tokens of a sequence form its rows t * g + h, so K and V are
// read once for all of them.
//
// rows_kernel: tiles of 8 rows, for the next tokens of a decode step (g * new
// <= 8 is one tile: every K and V byte is read once). Bound by HBM; the
// tensor-core work is two m16n8k16 products a key and 128 dims.
//   * fp32 accuracy from fp16 products: q and P are split into a high and a low
//     fp16 half (21 and 22 bits; K and V are fp16 already, products are exact and sums
//     are fp32). The 16 rows of the A operand are the 8 rows' high halves and
//     their low halves, so the split costs no product more: thread (row, 2
//     columns) holds the high part in c0, c1 and the low part in c2, c3 and adds
//     them. The same thread's scores become its A registers of P V.
//   * a warp has a kv head of its own, and the eight warps of a CTA work on the
//     same blocks of 16 keys: K and V of all heads of a token lie side by side,
//     and four producer warps copy them with one bulk copy a token and pool (2 KB
//     for eight heads of 128) into a ring of stages. (A head a CTA read 256-byte
//     rows 2 KB apart: 4.2 TB/s at two contexts of 131072 and 100001 tokens; 16
//     bytes a thread with cp.async: 5.4; a 256-byte bulk copy a row and head:
//     4.9, bound by the copies' number.) With fewer than eight kv heads the
//     warps share out the blocks of a stage. Rows are padded by 16 bytes so that
//     ldmatrix reads different banks; pages may have any size. The producer goes
//     on to the next run of blocks while the warps finish the last one.
//   * P V of a block starts at zero and is added with one fma that also
//     rescales (acc = acc * 2^(m_old - m_new) + c): the running sums round to
//     nearest in fp32 whatever the tensor core does.
//   * the work is a row of units, one for each block of keys of each (tile,
//     group of heads) and a few for starting one; a grid of one CTA an SM
//     takes equal runs of it, cut anywhere, so that sequences of all lengths
//     load every SM alike. The lengths are only known on the device: every CTA
//     adds up the tiles' blocks itself. What lies in several runs leaves (m, l,
//     acc) for each, which combine_kernel adds in the order of the runs.
// Measured (both kernels): two contexts of 131072 and 100001 tokens, 64 heads on 8,
// 167 us (6.4 TB/s); 32 of 1 to 8192 tokens 34.2 us (3.7 TB/s, the first copies and
// the joining cost 10 of them); one of 2048 tokens, 32 heads, 15.4 us (2.2 TB/s).
#include "paged.h"
#include "paged_rows.cuh"
#include "paged_tc.h"
#include "abi_errors.h"
#include "decode_ops.h"
#include "qmatvec.h"
#include "trace.h"

#include <algorithm>
#include <cmath>

namespace hesa_cuda {
namespace {

constexpr int kKeyBlock = 16;
constexpr int kCopyWarps = 4;        // a warp gets no more than one bulk copy under way in about 45 ns
// Rows of a sequence above which 128-row tiles are used, though they may be
// empty for the most part, rather than several tiles of 8 that each read K and V.
// Eight sequences of 4000 tokens, 64 heads of 128 on 8: 16 rows 31 us here, 38
// there; 32 rows 45 and 39; 64 rows 82 and 39. 16 heads of 256 on 4: 32 rows 52 and
// 74, 64 rows 89 and 75.
constexpr int most_rows(int head_dim) { return head_dim == 256 ? 48 : 16; }
constexpr int kSegCost = 5;          // stages that starting a (tile, group) takes the time of

// 8 warps (4 with head_dim 256) and kCopyWarps that copy
template <int HD> struct RowsShape : RowParts<HD, (HD == 256 ? 4 : 8)> {
    using RowParts<HD, (HD == 256 ? 4 : 8)>::warps;
    static constexpr int threads = (warps + kCopyWarps) * 32;
    static constexpr int stages = HD == 64 ? 5 : 3;
    // a stage: K then V of `subs` blocks, rows of `heads` heads padded by 16 bytes; heads * subs <= warps
    static constexpr size_t stage_bytes = 2 * kKeyBlock * (warps * HD * 2 + warps * 16);
    static constexpr size_t smem = stages * stage_bytes;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The ring between the producer and the consumer warps.
struct Ring {
    uint8_t* smem;
    uint64_t *full, *empty;
    uint32_t at;      // stages used so far (the same in every warp)
    uint32_t row;     // bytes of a row
    bool ok;          // no wait has run out
};

// Copying warp pw: a segment's blocks, `subs` a stage. Of the 16 rows of K and 16
// of V of a block (all heads of the group) it copies rows 8 pw .. 8 pw + 7, of
// four blocks at once.
template <int HD>
__device__ __forceinline__ void copy_segment(const AttnArgs& A, Ring& ring, const HeadGroups& hg, const Segment& seg, int pw) {
    using S = RowsShape<HD>;
    const int lane = threadIdx.x & 31;
    const TileView tv = tile_view<kKeyBlock>(A, seg.tile);
    const int i1 = min(tv.kb.n, seg.b1);
    const int32_t* table = A.c.table + static_cast<int64_t>(tv.sv.slot) * A.c.max_pages;
    const int row = pw * 8 + (lane & 7), v = row >> 4;
    const __half* pool = (v ? A.c.v : A.c.k) + seg.grp * hg.heads * HD;
    const int row_elems = A.c.n_kv * HD;
    const uint32_t bytes = static_cast<uint32_t>(min(hg.heads, A.c.n_kv - seg.grp * hg.heads)) * HD * 2;
    for (int i = seg.b0; i < i1; i += hg.subs) {
        const uint32_t slot = ring.at % S::stages;
        uint8_t* stage = ring.smem + slot * S::stage_bytes;
#pragma unroll 1
        for (int x0 = 0; x0 < hg.subs; x0 += 4) {
            const int x = x0 + (lane >> 3);
            const bool block = x < hg.subs && i + x < i1;
            const int32_t j = block ? tv.kb.at(i + x) * kKeyBlock + (row & 15) : tv.sv.len;
            const int32_t pi = A.c.page_div.div(j);
            const int32_t page = j < tv.sv.len ? table[pi] : -1;   // asked for before the wait
            const bool good = page >= 0 && page < A.c.n_pages;
            if (x0 == 0) {
                if (ring.at >= S::stages && ring.ok)
                    ring.ok = mbar_warp_wait(&ring.empty[slot], (ring.at / S::stages - 1) & 1u, A.status, kStatusWaitTimeout);
                if (!ring.ok) return;
            }
            uint8_t* dst = stage + ((v * hg.subs + x) * kKeyBlock + (row & 15)) * ring.row;
            const unsigned have = __ballot_sync(0xffffffffu, good), lost = __ballot_sync(0xffffffffu, !good && j < tv.sv.len);
            // zeros where there is no token's V (a K that no row sees may be anything) or no page
            unsigned zero = __ballot_sync(0xffffffffu, block && !good && v) | lost;
            if (zero) {
                for (; zero; zero &= zero - 1) {
                    uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), __ffs(zero) - 1));
                    for (uint32_t c = lane * 16; c < bytes; c += 512) *reinterpret_cast<uint4*>(to + c) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();   // in order before a later copy into the row
                if (lost && lane == 0) record_status(A.status, kStatusBadPosition);
            }
            __syncwarp();
            // the warp's one arrival at the stage comes with its last blocks' bytes
            if (lane == 0) {
                if (x0 + 4 < hg.subs) mbar_expect_tx(&ring.full[slot], __popc(have) * bytes);
                else mbar_arrive_expect_tx(&ring.full[slot], __popc(have) * bytes);
            }
            __syncwarp();
            if (good)
                bulk_g2s(dst, pool + static_cast<int64_t>(page) * A.c.page_stride + static_cast<int64_t>(j - pi * A.c.page_size) * row_elems, bytes,
                         &ring.full[slot]);
        }
        ++ring.at;
    }
}

// Consumer warp: its head's attention over a segment's blocks. part < 0: they
// are all that the rows see, and the result goes to out; else (m, l, acc) go to
// that part.
template <int HD>
__device__ __forceinline__ void rows_segment(const AttnArgs& A, Ring& ring, const HeadGroups& hg, const Segment& seg, const TileView& tv, int part) {
    using S = RowsShape<HD>;
    constexpr int KS = HD / 16;                  // k-steps of Q K^T
    constexpr int NT = HD / 8;                   // column tiles of P V
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = hg.sub_of(warp), hl = warp - sub * hg.heads, kvh = seg.grp * hg.heads + hl;
    const bool active = sub < hg.subs && kvh < A.c.n_kv;
    const SeqView& sv = tv.sv;
    const Mask& mask = tv.mask;

    // this thread's row and position
    const int r = tv.r0 + (lane >> 2);
    const bool row_ok = r < tv.n_rows && active;
    const int rc = min(r, tv.n_rows - 1), t = A.group_div.div(rc), h = min(kvh, A.c.n_kv - 1) * A.group + rc - t * A.group;
    const int32_t pos = tv.base + t;
    const RowKeys keys = mask.row(pos);
    const int i1 = min(tv.kb.n, seg.b1);

    // ---- q as hi and lo halves of q * 2^-e, max |q| 2^-e in [2^14, 2^15) ----
    uint32_t qa[KS][4];
    float qscale;   // 2^e; NaN for a row that is not finite
    {
        const float* q = A.q + static_cast<int64_t>(sv.q0 + t) * A.ldq + static_cast<int64_t>(h) * HD;
        float2 v[KS][2];
        float mx = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) v[k][i] = row_ok ? *reinterpret_cast<const float2*>(q + k * 16 + i * 8 + 2 * (lane & 3)) : make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) mx = fmax_nan(mx, fmax_nan(fabsf(v[k][i].x), fabsf(v[k][i].y)));
        mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const bool fin = mx < INFINITY;
        int e = 0;
        if (fin && mx > 0.f) e = ilogbf(mx) - 14;
        // two factors, so that 2^-e stays finite for the smallest subnormal q
        const float f1 = ldexpf(1.f, -(e / 2)), f2 = fin ? ldexpf(1.f, -(e - e / 2)) : 0.f;
        qscale = fin ? ldexpf(1.f, e) : NAN;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float x = fin ? v[k][i].x * f1 * f2 : 0.f, y = fin ? v[k][i].y * f1 * f2 : 0.f;
                split_away2(x, y, qa[k][2 * i], qa[k][2 * i + 1]);
            }
    }
    const float sc = A.cap2 != 0.f ? qscale : qscale * A.scale2;
    const float slope2 = A.slopes ? A.slopes[h] * 1.44269504088896341f : 0.f;

    float m = -INFINITY, l = 0.f;
    float acc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = 0.f;

    // ldmatrix row addresses: K matrices (keys 0-7 | 8-15) x (dims 0-7 | 8-15), V the same, transposed
    const uint32_t mine = static_cast<uint32_t>(sub * kKeyBlock) * ring.row + hl * HD * 2;   // this warp's block and head in a stage
    const uint32_t v_at = static_cast<uint32_t>(hg.subs * kKeyBlock) * ring.row;
    const uint32_t k_row = ((lane & 7) + ((lane >> 4) << 3)) * ring.row + ((lane >> 3) & 1) * 16;
    const uint32_t v_row = ((lane & 7) + (((lane >> 3) & 1) << 3)) * ring.row + (lane >> 4) * 16;

    for (int i0 = seg.b0; i0 < i1; i0 += hg.subs, ++ring.at) {
        const uint32_t slot = ring.at % S::stages;
        if (ring.ok) ring.ok = mbar_warp_wait(&ring.full[slot], (ring.at / S::stages) & 1u, A.status, kStatusWaitTimeout);
        if (!ring.ok) break;
        const int i = i0 + sub;
        if (active && i < i1) {
            uint8_t* kp = ring.smem + slot * S::stage_bytes + mine;
            uint8_t* vp = kp + v_at;
            const uint32_t sk = smem_addr(kp), sv_ = smem_addr(vp);
            const int32_t j0 = tv.kb.at(i) * kKeyBlock;

            // keys 0-7 and 8-15, each in two chains of products
            float s0[2][4] = {}, s1[2][4] = {};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t b[4];
                ldsm4(b, sk + k_row + k * 32);
                mma16816(s0[k & 1], qa[k], b[0], b[1]);
                mma16816(s1[k & 1], qa[k], b[2], b[3]);
            }
            float s[4] = {(s0[0][0] + s0[1][0]) + (s0[0][2] + s0[1][2]), (s0[0][1] + s0[1][1]) + (s0[0][3] + s0[1][3]),
                          (s1[0][0] + s1[1][0]) + (s1[0][2] + s1[1][2]), (s1[0][1] + s1[1][1]) + (s1[0][3] + s1[1][3])};
#pragma unroll
            for (int c = 0; c < 4; ++c) s[c] *= sc;
            if (A.cap2 != 0.f) {
#pragma unroll
                for (int c = 0; c < 4; ++c) s[c] = capped(s[c], A.cap2, A.cap_in);
            }
            const int32_t jc = j0 + 2 * (lane & 3);   // this thread's keys: jc, jc + 1, jc + 8, jc + 9
            if (A.slopes) {
#pragma unroll
                for (int c = 0; c < 4; ++c) s[c] -= slope2 * fabsf(static_cast<float>(pos - (jc + (c >> 1) * 8 + (c & 1))));
            }
            if (!mask.all(tv.p_lo, tv.p_hi, j0, j0 + kKeyBlock)) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (!keys.sees(jc + (c >> 1) * 8 + (c & 1))) s[c] = -INFINITY;
                // A key that some row does not see has P = 0 there, which would make
                // NaN of an infinite or NaN v. Such values (there are none in a sound
                // cache) are added where they are seen and then cleared, so that they
                // reach no other row. Keys past the sequence are zeros.
                uint32_t odd = 0;
                for (int c = lane; c < kKeyBlock * HD / 8; c += 32) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vp + (c / (HD / 8)) * ring.row + (c % (HD / 8)) * 16);
                    odd |= nonfinite_mark(w.x) | nonfinite_mark(w.y) | nonfinite_mark(w.z) | nonfinite_mark(w.w);
                }
                if (__any_sync(0xffffffffu, (odd & kNonfinite) != 0)) {
                    for (int j = 0; j < kKeyBlock; ++j) {
                        const bool seen = keys.sees(j0 + j);
                        const __half* vr = reinterpret_cast<const __half*>(vp + j * ring.row) + 2 * (lane & 3);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const float x = __half2float(vr[n * 8 + c]);
                                if (seen && !isfinite(x)) acc[n][c] += x;
                            }
                    }
                    __syncwarp();
                    for (int c = lane; c < kKeyBlock * HD; c += 32) {
                        __half& x = reinterpret_cast<__half*>(vp + (c / HD) * ring.row)[c % HD];
                        if (!isfinite(__half2float(x))) x = __float2half_rn(0.f);
                    }
                    fence_proxy_async_smem();   // before the stage is filled again
                    __syncwarp();
                }
            }
            float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mx = fmaxf(mx, m);
            const float ms = mx == -INFINITY ? 0.f : mx;   // nothing seen yet: P = 2^-inf = 0
            const float corr = m == -INFINITY ? 0.f : ex2(m - ms);
            m = mx;
            float p[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) p[c] = ex2(s[c] - ms + kPShift);
            l = fmaf(l, corr, (p[0] + p[1]) + (p[2] + p[3]));
            uint32_t pa[4];
            split_half2(p[0], p[1], pa[0], pa[1]);
            split_half2(p[2], p[3], pa[2], pa[3]);
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t b[4];
                ldsm4_t(b, sv_ + v_row + n * 16);
                float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(c0, pa, b[0], b[1]);
                mma16816(c1, pa, b[2], b[3]);
                acc[n][0] = fmaf(acc[n][0], corr, c0[0] + c0[2]);
                acc[n][1] = fmaf(acc[n][1], corr, c0[1] + c0[3]);
                acc[n + 1][0] = fmaf(acc[n + 1][0], corr, c1[0] + c1[2]);
                acc[n + 1][1] = fmaf(acc[n + 1][1], corr, c1[1] + c1[3]);
            }
        }
        __syncwarp();   // the warp is done with this stage
        if (lane == 0) mbar_arrive(&ring.empty[slot]);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (!row_ok) return;
    if (part < 0) {
        float* o = A.out + static_cast<int64_t>(sv.q0 + t) * A.ldo + static_cast<int64_t>(h) * HD + 2 * (lane & 3);
        const float inv = l == 0.f ? 0.f : 1.f / l;   // nothing seen: zeros
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(o + n * 8) = make_float2(acc[n][0] * inv, acc[n][1] * inv);
    } else {
        const int64_t at = (static_cast<int64_t>(part) * S::warps + warp) * kRowTile + (lane >> 2);
        float* ml = A.part + S::cut_bytes / 4;
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + at * 2) = make_float2(m, l);
        float* o = ml + S::part_rows(part_count(A.n_split, hg)) * 2 + at * HD + 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(o + n * 8) = make_float2(acc[n][0], acc[n][1]);
    }
}

template <int HD>
__global__ void __launch_bounds__(RowsShape<HD>::threads, 1)
rows_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ HeadGroups hg) {
    using S = RowsShape<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_pre[kMostTiles + 1];
    __shared__ int64_t s_sum[S::warps + kCopyWarps];
    __shared__ __align__(8) uint64_t s_full[S::stages], s_empty[S::stages];
    const int warp = threadIdx.x >> 5, tiles = A.n_split, cta = blockIdx.x;
    // the arguments come into the constant cache while the previous kernel ends
    if (A.c.n_pages <= 0 || A.b.n_seq <= 0 || A.ldq <= 0 || A.group <= 0 || A.part == nullptr || hg.heads <= 0) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::stages; ++i) {
            mbar_init(&s_full[i], kCopyWarps);
            mbar_init(&s_empty[i], S::warps);
        }
        s_pre[0] = 0;
        fence_mbar_init();
    }
    grid_dep_wait();
    grid_dep_launch();   // combine_kernel may be set up meanwhile; it waits for this grid's end
    const int64_t units = tile_units<S::warps + kCopyWarps, kKeyBlock>(A, hg, tiles, s_pre, s_sum) * hg.groups;
    const Runs runs(units, gridDim.x, kLeastUnits);   // a constant: 0.15 us less than from hg
    const bool listed_by_tile = by_tile(tiles, hg);
    Cut* cuts = reinterpret_cast<Cut*>(A.part);
    int64_t u = 0, end = 0;
    if (units > 0 && cta < runs.n_cta) {
        u = runs.start(cta);
        end = runs.start(cta + 1);
    }
    const int64_t begin = u;
    int lo = tile_at(s_pre, hg, tiles, u);
    Ring ring{smem, s_full, s_empty, 0u, static_cast<uint32_t>(hg.heads * HD * 2 + 16), true};
    Segment seg;
    if (warp >= S::warps) {
        while (next_segment(s_pre, hg, u, end, lo, seg)) copy_segment<HD>(A, ring, hg, seg, warp - S::warps);
        // nothing may be in flight when the CTA ends
        for (uint32_t i = ring.at > S::stages ? ring.at - S::stages : 0; i < ring.at; ++i)
            if (!mbar_wait_bounded(&s_full[i % S::stages], (i / S::stages) & 1u, A.status, kStatusDrainTimeout)) break;
        return;
    }
    if (listed_by_tile && cta == 0)   // those without rows
        for (int i = threadIdx.x; i < tiles * hg.groups; i += S::warps * 32)
            if (s_pre[i / hg.groups + 1] == s_pre[i / hg.groups]) cuts[i] = Cut{};
    Cut cut{};
    while (next_segment(s_pre, hg, u, end, lo, seg)) {
        const int c_first = runs.cta_of(seg.first + hg.cost), c_last = runs.cta_of(seg.first + seg.units - 1);
        const bool uncut = c_first == c_last;
        const int own_part = 2 * kRowsCtas + seg.tile * hg.groups + seg.grp;   // of what several warps share, uncut
        const TileView tv = tile_view<kKeyBlock>(A, seg.tile);
        const Cut all{seg.grp, uncut ? own_part : 2 * c_first + (runs.start(c_first) >= seg.first ? 0 : 1), c_last - c_first + 1,
                      min(kRowTile, tv.n_rows - tv.r0), tv.r0, tv.sv.q0};
        if (cta == c_first + 1) cut = all;
        if (listed_by_tile && cta == c_first && threadIdx.x == 0) cuts[seg.tile * hg.groups + seg.grp] = all;
        rows_segment<HD>(A, ring, hg, seg, tv, !uncut ? 2 * cta + (begin >= seg.first ? 0 : 1) : hg.subs > 1 ? own_part : -1);
    }
    if (!listed_by_tile && threadIdx.x == 0) cuts[cta] = cut;
}

struct Plan {
    bool tc;         // chunk_kernel of paged_attention_tc.cu
    int heads;       // rows_kernel: of a group at most
    int rows, per_seq, tiles, blocks_per_split, n_split;
};

// How a call is cut: from the host's bounds alone, so that a captured graph
// serves every later length within them.
Plan make_plan(const hesa_cuda_paged_kv* kv, const hesa_cuda_token_batch* b, int64_t n_head) {
    Plan p{};
    const int g = static_cast<int>(n_head / kv->n_kv_head);
    const int64_t rows_a_seq = static_cast<int64_t>(b->max_new) * g;
    p.tc = rows_a_seq > most_rows(kv->head_dim) && (kv->head_dim <= 128 || paged_attention_tiled(layer_of(kv, 0)));
    p.rows = p.tc ? kTcRows : kRowTile;
    const int64_t most = (rows_a_seq + p.rows - 1) / p.rows;
    const int64_t bound = tile_bound(b->n_tokens, b->n_seq, g, p.rows);
    p.per_seq = b->n_seq * most <= bound ? static_cast<int>(most) : 0;
    const int64_t tiles = p.per_seq ? b->n_seq * most : bound;
    p.tiles = static_cast<int>(tiles);
    if (!p.tc) {
        // All heads of a token at once read the longest rows, and an SM streams no
        // more than about 44 GB/s: where that would leave SMs without work, groups
        // of fewer heads. One context of 100 tokens, 64 heads on 8: 13.2 us with all
        // heads together, 10.3 with two; one of 2048 tokens, 32 heads: 14.3 with eight, 16.5 with two.
        // (A tile that sees no key is a block of work too. The loop ends with fewer
        // than 4 kRowsCtas (tile, group)s, and kMostTiles of them can be listed.)
        const int64_t blocks = std::max<int64_t>(1, (b->max_len + kKeyBlock - 1) / kKeyBlock);
        static_assert(4 * kRowsCtas <= kMostTiles, "a list for every (tile, group) where groups are made smaller");
        p.heads = kv->head_dim == 256 ? 4 : 8;
        while (p.heads > 2 && tiles * ((kv->n_kv_head + p.heads - 1) / p.heads) * blocks < 2 * kRowsCtas) p.heads /= 2;
        return p;
    }
    // one CTA an SM, no split under 256 keys
    const int keys = tc_keys(kv->head_dim);
    const int64_t blocks = std::max<int64_t>(1, (b->max_len + keys - 1) / keys);
    const int64_t pairs = tiles * kv->n_kv_head * (kv->head_dim / tc_dims(kv->head_dim));
    const int64_t want = std::max<int64_t>(1, 148 / pairs);   // 1 from 75 pairs on: nothing is split
    const int64_t per = std::max<int64_t>(256 / keys, (blocks + want - 1) / want);
    p.blocks_per_split = static_cast<int>(std::min(per, blocks));
    p.n_split = static_cast<int>((blocks + p.blocks_per_split - 1) / p.blocks_per_split);
    return p;
}

size_t part_bytes(const Plan& p, const hesa_cuda_paged_kv* kv) {
    if (!p.tc) {
        const HeadGroups hg(kv->n_kv_head, kv->head_dim == 256 ? RowsShape<256>::warps : RowsShape<128>::warps, p.heads, kSegCost);
        const int64_t parts = part_count(std::min(p.tiles, kMostTiles), hg);
        return kv->head_dim == 64 ? RowsShape<64>::bytes(parts) : kv->head_dim == 128 ? RowsShape<128>::bytes(parts) : RowsShape<256>::bytes(parts);
    }
    const int dims = tc_dims(kv->head_dim);
    const size_t rows = static_cast<size_t>(p.tiles) * kv->n_kv_head * (kv->head_dim / dims) * p.n_split * p.rows;
    return p.n_split > 1 ? rows * (dims + 2) * sizeof(float) : 0;
}

template <int HD>
cudaError_t launch_rows(AttnArgs a, const Plan& p, cudaStream_t s) {
    static bool set[64] = {};   // per instance and device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!set[dev]) {
        e = cudaFuncSetAttribute(rows_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(RowsShape<HD>::smem));
        if (e != cudaSuccess) return e;
        set[dev] = true;
    }
    using S = RowsShape<HD>;
    const HeadGroups hg(a.c.n_kv, S::warps, p.heads, kSegCost);
    for (a.tile0 = 0; a.tile0 < p.tiles && e == cudaSuccess; a.tile0 += kMostTiles) {
        a.n_split = std::min(kMostTiles, p.tiles - a.tile0);
        e = launch_dep(rows_kernel<HD>, dim3(kRowsCtas), S::threads, S::smem, s, a, hg);
        const int cuts = by_tile(a.n_split, hg) ? a.n_split * hg.groups : kRowsCtas;
        const int rows = std::min(kRowTile, a.b.max_new * a.group);
        const unsigned z = static_cast<int64_t>(cuts) * hg.heads * rows <= 8 * kRowsCtas ? rows : 1;
        if (e == cudaSuccess)
            e = launch_dep(combine_kernel<HD, S::warps>, dim3(static_cast<unsigned>(cuts), static_cast<unsigned>(hg.heads), z), 256, 0, s, a, hg);
    }
    return e;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

int check_paged_shape(const PagedShape& c) {
    if (c.n_layer <= 0 || c.n_pages <= 0 || c.page_size <= 0 || c.n_kv_head <= 0 || c.n_slots <= 0 || c.max_pages <= 0)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "non-positive dimension");
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "head_dim must be 64, 128 or 256");
    if (c.page_size > 65536 || c.n_kv_head > 1024 || c.n_slots > 65536 || c.n_layer > 4096 ||
        static_cast<int64_t>(c.max_pages) * c.page_size >= (int64_t(1) << 30))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "paged cache too large");
    const int64_t values = static_cast<int64_t>(c.page_size) * c.n_kv_head * c.head_dim, page = values / c.unit;
    if (values > (int64_t(1) << 30)) return record_error(HESA_CUDA_SHAPE_MISMATCH, "pages of more than 2^30 values");
    const int64_t most = int64_t(1) << 50;
    if (c.page_stride < page || c.page_stride > most || c.layer_stride < 0 || c.layer_stride > most || (c.page_stride & 7) || (c.layer_stride & 7))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "page_stride and layer_stride must be multiples of 8, page_stride at least a page");
    if (c.n_layer > 1 && c.layer_stride < (static_cast<int64_t>(c.n_pages) - 1) * c.page_stride + page &&
        (c.layer_stride < page || c.page_stride < (static_cast<int64_t>(c.n_layer) - 1) * c.layer_stride + page))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "the pages of two layers overlap");
    if (!aligned(c.table, 4) || !aligned(c.seq_len, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the tables must be 4-byte aligned");
    return HESA_CUDA_OK;
}

int check_paged_kv(const hesa_cuda_paged_kv* kv) {
    if (!kv || !kv->k || !kv->v || !kv->table || !kv->seq_len) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    const int rc = check_paged_shape({kv->table, kv->seq_len, kv->page_stride, kv->layer_stride, 1, kv->n_layer, kv->n_pages, kv->page_size, kv->n_kv_head,
                                      kv->head_dim, kv->n_slots, kv->max_pages});
    if (rc != HESA_CUDA_OK) return rc;
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the page pools must be 16-byte aligned");
    return HESA_CUDA_OK;
}

template <typename KV>
static int check_rows(const KV* kv, int32_t layer, const hesa_cuda_token_batch* b, int64_t n_head) {
    if (layer < 0 || layer >= kv->n_layer) return record_error(HESA_CUDA_INVALID_ARGUMENT, "no such layer");
    if (!b || !b->q_start) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (!aligned(b->q_start, 4) || !aligned(b->slots, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "q_start and slots must be 4-byte aligned");
    if (b->n_seq <= 0 || b->n_tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->max_new > b->n_tokens)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "bad batch");
    if (b->n_seq > 65536 || (!b->slots && b->n_seq > kv->n_slots)) return record_error(HESA_CUDA_SHAPE_MISMATCH, "more sequences than slots");
    if (b->max_len > static_cast<int64_t>(kv->max_pages) * kv->page_size)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "max_len is more than a slot's pages hold");
    if (n_head <= 0 || n_head % kv->n_kv_head != 0 || n_head > 16384) return record_error(HESA_CUDA_SHAPE_MISMATCH, "n_head must be a multiple of n_kv_head");
    if (static_cast<int64_t>(b->n_tokens) * n_head >= (int64_t(1) << 31) - (int64_t(1) << 20))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "too many rows");
    return HESA_CUDA_OK;
}
int check_batch(const hesa_cuda_paged_kv* kv, int32_t layer, const hesa_cuda_token_batch* b, int64_t n_head) { return check_rows(kv, layer, b, n_head); }
int check_batch4(const hesa_cuda_paged_kv4* kv, int32_t layer, const hesa_cuda_token_batch* b, int64_t n_head) { return check_rows(kv, layer, b, n_head); }

PagedLayer layer_of(const hesa_cuda_paged_kv* kv, int32_t layer) {
    PagedLayer c{};
    c.k = static_cast<const __half*>(kv->k) + layer * kv->layer_stride;
    c.v = static_cast<const __half*>(kv->v) + layer * kv->layer_stride;
    c.page_stride = kv->page_stride;
    c.n_pages = kv->n_pages;
    c.page_size = kv->page_size;
    c.n_kv = kv->n_kv_head;
    c.head_dim = kv->head_dim;
    c.table = kv->table;
    c.seq_len = kv->seq_len;
    c.n_slots = kv->n_slots;
    c.max_pages = kv->max_pages;
    c.page_div = FastDiv(kv->page_size);
    return c;
}

BatchView view_of(const hesa_cuda_token_batch* b) { return BatchView{b->slots, b->q_start, b->n_seq, b->n_tokens, b->max_new, b->max_len}; }

int attention_args(int32_t head_dim, int32_t n_kv_head, const hesa_cuda_token_batch* batch, const float* q, int64_t ldq, float* out, int64_t ldo,
                   int64_t n_head, const hesa_cuda_attn_options* options, void* workspace, AttnArgs* args) {
    AttnArgs& a = *args;
    if (!q || !out || !workspace) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    const int64_t width = n_head * head_dim;
    if (ldq < width || ldo < width || ldq > (int64_t(1) << 40) || ldo > (int64_t(1) << 40))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "leading dimension too small");
    if (!aligned(q, 16) || !aligned(out, 16) || (ldq & 3) || (ldo & 3))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "q / out must be 16-byte aligned with ldq, ldo multiples of 4");
    if (!aligned(workspace, 16)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    hesa_cuda_attn_options o{};
    if (options) o = *options;
    if (!(o.scale >= 0.f) || !std::isfinite(o.scale) || o.window < 0)
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "scale and window must be finite and not negative");
    if (o.softcap != 0.f && !(o.softcap >= 1e-6f && o.softcap <= 1e6f))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "softcap must be 0 or 1e-6 .. 1e6");
    if (!aligned(o.slopes, 4) || !aligned(o.prefix, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "slopes and prefix must be 4-byte aligned");
    if (batch->max_new == 0) return HESA_CUDA_OK;   // nothing will run
    a.b = view_of(batch);
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.n_head = static_cast<int32_t>(n_head);
    a.group = static_cast<int32_t>(n_head / n_kv_head);
    a.group_div = FastDiv(a.group);
    const double log2e = 1.4426950408889634;
    const double scale = o.scale > 0.f ? o.scale : 1.0 / std::sqrt(static_cast<double>(head_dim));
    a.scale2 = static_cast<float>(scale * log2e);
    a.cap2 = static_cast<float>(o.softcap * log2e);
    a.cap_in = o.softcap > 0.f ? static_cast<float>(scale / o.softcap) : 0.f;
    if (!std::isfinite(a.scale2) || !std::isfinite(a.cap_in))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "scale is too large for a float, by itself or by softcap");
    a.window = std::min(o.window, 1 << 30);   // wider than any context; a position less a window stays in 32 bits
    a.slopes = o.slopes;
    a.prefix = o.prefix;
    a.part = static_cast<float*>(workspace);
    return HESA_CUDA_OK;
}

}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_paged_attention_workspace_size(const hesa_cuda_paged_kv* kv, const hesa_cuda_token_batch* batch, int64_t n_head) {
    if (check_paged_kv(kv) != HESA_CUDA_OK || check_batch(kv, 0, batch, n_head) != HESA_CUDA_OK) return 0;
    const Plan p = make_plan(kv, batch, n_head);
    return std::max<size_t>(part_bytes(p, kv), 16);
}

int hesa_cuda_paged_attention(const hesa_cuda_paged_kv* kv, int32_t layer, const hesa_cuda_token_batch* batch, const float* q,
                              int64_t ldq, float* out, int64_t ldo, int64_t n_head, const hesa_cuda_attn_options* options,
                              void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_paged_attention");
    int rc = check_paged_kv(kv);
    if (rc == HESA_CUDA_OK) rc = check_batch(kv, layer, batch, n_head);
    if (rc != HESA_CUDA_OK) return rc;
    if (batch->n_tokens == 0) return HESA_CUDA_OK;   // no rows: their buffers may be null
    AttnArgs a{};
    rc = attention_args(kv->head_dim, kv->n_kv_head, batch, q, ldq, out, ldo, n_head, options, workspace, &a);
    if (rc != HESA_CUDA_OK) return rc;
    if (workspace_bytes < hesa_cuda_paged_attention_workspace_size(kv, batch, n_head))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    if (batch->max_new == 0) return HESA_CUDA_OK;

    const Plan p = make_plan(kv, batch, n_head);
    a.c = layer_of(kv, layer);
    a.per_seq = p.per_seq;
    a.blocks_per_split = p.blocks_per_split;
    a.n_split = p.n_split;
    cudaError_t e = status_word(&a.status);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (e == cudaSuccess && p.tc) {
        e = paged_attention_tc(a, p.tiles, s);
    } else if (e == cudaSuccess) {
        switch (kv->head_dim) {
            case 64: e = launch_rows<64>(a, p, s); break;
            case 128: e = launch_rows<128>(a, p, s); break;
            default: e = launch_rows<256>(a, p, s); break;
        }
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "paged attention kernel");
}

}  // extern "C"
