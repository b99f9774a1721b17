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
//     fp16 half (22 bits; K and V are fp16 already, products are exact and sums
//     are fp32). The 16 rows of the A operand are the 8 rows' high halves and
//     their low halves, so the split costs no product more: thread (row, 2
//     columns) holds the high part in c0, c1 and the low part in c2, c3 and adds
//     them. The same thread's scores become its A registers of P V.
//   * a warp has a kv head of its own, and the eight warps of a CTA take the
//     same blocks of 16 keys, so that the rows of all heads of a token, which
//     lie side by side, are read at about the same time. (With a head a CTA the
//     256-byte rows of a head were read 2 KB apart: 4.2 TB/s at two contexts of
//     131072 and 100001.) With fewer than eight kv heads the warps share out
//     the blocks. A warp has its own ring of cp.async stages and no block-wide
//     barrier in its loop; rows are padded by 16 bytes so that ldmatrix reads
//     different banks. Pages of any size: each lane looks up the page of one key
//     of the next block ahead of its copies.
//   * P V of a block starts at zero and is added with one fma that also
//     rescales (acc = acc * 2^(m_old - m_new) + c): the running sums round to
//     nearest in fp32 whatever the tensor core does.
//   * the work is a row of units, one for each block of keys of each (tile,
//     group of heads) and kSegCost for starting one; a grid of one CTA an SM
//     takes equal runs of it, cut anywhere, so that sequences of all lengths
//     load every SM alike. The lengths are only known on the device: every CTA
//     adds up the tiles' blocks itself. What lies in several runs leaves (m, l,
//     acc) for each, which combine_kernel adds in the order of the runs.
#include "paged.h"
#include "paged_tc.h"
#include "abi_errors.h"
#include "decode_ops.h"
#include "qmatvec.h"
#include "trace.h"

#include <algorithm>
#include <cmath>

namespace hesa_cuda {
namespace {

constexpr int kRowTile = 8;
constexpr int kKeyBlock = 16;
constexpr int kRowsCtas = 148;       // of a balanced launch: one an SM
constexpr int kMostTiles = 1024;     // of a balanced launch: the tiles' blocks are summed in shared memory
constexpr int kSegCost = 3;          // units for starting a (tile, group): about its time over that of a block
constexpr int kLeastUnits = 4;       // of a run

template <int HD> struct RowsShape {
    static constexpr int warps = HD == 256 ? 4 : 8;
    static constexpr int stages = HD == 64 ? 5 : 3;
    static constexpr int row_halves = HD + 8;                      // padded by 16 bytes
    static constexpr int stage_halves = 2 * kKeyBlock * row_halves;   // K, then V
    static constexpr size_t warp_bytes = static_cast<size_t>(stages) * stage_halves * 2;
    static constexpr size_t smem = warps * warp_bytes;
    // after its loop a warp's ring holds its (m, l, acc) of 8 rows
    static_assert(kRowTile * (HD + 2) * 4 <= warp_bytes, "merge region");
    // parts: two a CTA, each [warps][rows]: (m, l), then acc[HD]
    static constexpr size_t part_rows = 2 * static_cast<size_t>(kRowsCtas) * warps * kRowTile;
    static constexpr size_t cut_bytes = kRowsCtas * 16;
    static constexpr size_t part_bytes = cut_bytes + part_rows * (2 + HD) * 4;
};

// Heads of a group (a CTA's warps have one each) and how many warps share a head.
struct HeadGroups {
    int groups, heads, subs;
    __host__ __device__ HeadGroups(int n_kv, int warps) {
        groups = (n_kv + warps - 1) / warps;
        heads = (n_kv + groups - 1) / groups;
        subs = warps / heads;
    }
};

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool have) {
    const int n = have ? 16 : 0;   // 0: sixteen zero bytes, src is not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Blocks of a tile that has rows (one for a tile whose rows see nothing: its
// zeros are written there), else 0.
__device__ __forceinline__ int tile_blocks(const AttnArgs& A, int idx, bool report) {
    int seq, tile;
    locate_tile(A.b, A.group, kRowTile, A.per_seq, idx, seq, tile);
    const SeqView sv = seq_view(A.c, A.b, seq);
    if (!sv.ok) {
        if (report) record_status(A.status, kStatusBadPosition);
        return 0;
    }
    const int n_rows = sv.n_new * A.group, r0 = tile * kRowTile, base = sv.len - sv.n_new;
    if (r0 >= n_rows) return 0;
    Mask mask{sv.len, A.window, 0};
    if (A.prefix) mask.prefix = max(0, min(A.prefix[seq], sv.len));
    return max(1, key_blocks(mask, base + r0 / A.group, base + min(r0 + kRowTile - 1, n_rows - 1) / A.group, kKeyBlock).n);
}

// The runs: CTA c of n_cta has units [start(c), start(c + 1)).
struct Runs {
    int64_t units;
    int n_cta;
    __device__ __forceinline__ int64_t start(int c) const { return units * c / n_cta; }
    __device__ __forceinline__ int cta_of(int64_t u) const {   // the last c with start(c) <= u
        return static_cast<int>(((u + 1) * n_cta - 1) / units);
    }
};

// Blocks [b0, b1) of tile idx for the heads of group grp. part < 0: they are all
// of it, and the result goes to out; else (m, l, acc) go to that part.
template <int HD>
__device__ __forceinline__ void rows_segment(const AttnArgs& A, uint8_t* smem, const HeadGroups& hg, int idx, int grp, int b0, int b1, int part) {
    using S = RowsShape<HD>;
    constexpr int KS = HD / 16;                  // k-steps of Q K^T
    constexpr int NT = HD / 8;                   // column tiles of P V
    constexpr int RH = S::row_halves;
    constexpr int PIECES = HD / 8;               // 16-byte pieces of a row
    constexpr int COPIES = kKeyBlock * PIECES / 32;   // of K (and of V) for each lane and block

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = warp / hg.heads, kvh = grp * hg.heads + warp % hg.heads;
    const bool active = sub < hg.subs && kvh < A.c.n_kv;
    uint8_t* my_smem = smem + warp * S::warp_bytes;

    int seq, tile;
    locate_tile(A.b, A.group, kRowTile, A.per_seq, idx, seq, tile);
    const SeqView sv = seq_view(A.c, A.b, seq);   // sound: it has blocks
    const int n_rows = sv.n_new * A.group;
    const int r0 = tile * kRowTile;

    // this thread's row and position; the tile's positions
    const int r = r0 + (lane >> 2);
    const bool row_ok = r < n_rows;
    const int t = (row_ok ? r : n_rows - 1) / A.group, h = kvh * A.group + (row_ok ? r : n_rows - 1) - t * A.group;
    const int base = sv.len - sv.n_new;   // position of the sequence's first new token
    const int32_t pos = base + t;
    float m = -INFINITY, l = 0.f;
    float acc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = 0.f;

    if (active) {
        const int32_t p_lo = base + r0 / A.group;
        const int32_t p_hi = base + min(r0 + kRowTile - 1, n_rows - 1) / A.group;
        Mask mask{sv.len, A.window, 0};
        if (A.prefix) mask.prefix = max(0, min(A.prefix[seq], sv.len));
        const RowKeys keys = mask.row(pos);
        const KeyBlocks kb = key_blocks(mask, p_lo, p_hi, kKeyBlock);
        const int i0 = b0 + sub, i1 = min(kb.n, b1), step = hg.subs;

        // ---- copies of this warp's blocks i0, i0 + step, ... ----
        const int32_t* table = A.c.table + static_cast<int64_t>(sv.slot) * A.c.max_pages;
        const int row_elems = A.c.n_kv * HD;
        const uint32_t ring = smem_addr(my_smem);
        const int psz = A.c.page_size;
        // lane (key lane & 15 of block i): its page, -1 where it has none
        auto page_of = [&](int i) -> int32_t {
            if (i >= i1) return -1;
            const int32_t j = kb.at(i) * kKeyBlock + (lane & 15);
            return j < sv.len ? table[j / psz] : -1;
        };
        auto issue = [&](int i, int slot, int32_t page) {
            if (i < i1) {
                const int32_t j = kb.at(i) * kKeyBlock + (lane & 15);
                const bool in = j < sv.len;
                const bool good = in && page >= 0 && page < A.c.n_pages;
                if (in && !good) record_status(A.status, kStatusBadPosition);   // not read: zeros in its place
                const int64_t off = good ? static_cast<int64_t>(page) * A.c.page_stride +
                                               static_cast<int64_t>(j % psz) * row_elems + kvh * HD
                                         : -1;
                const uint32_t dst = ring + static_cast<uint32_t>(slot) * S::stage_halves * 2;
#pragma unroll
                for (int c = 0; c < COPIES; ++c) {
                    const int piece = c * 32 + lane, row = piece / PIECES, at = piece % PIECES;
                    const int64_t o = __shfl_sync(0xffffffffu, off, row);
                    const int64_t src = (o < 0 ? 0 : o) + at * 8;
                    const uint32_t d = dst + static_cast<uint32_t>(row * RH + at * 8) * 2;
                    cp_async16_zfill(d, A.c.k + src, o >= 0);
                    cp_async16_zfill(d + kKeyBlock * RH * 2, A.c.v + src, o >= 0);
                }
            }
            cp_commit();
        };
        int32_t next_page = page_of(i0);
#pragma unroll
        for (int s = 0; s < S::stages - 1; ++s) {
            const int i = i0 + s * step;
            const int32_t pg = next_page;
            next_page = page_of(i + step);
            issue(i, s, pg);
        }

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
                for (int i = 0; i < 2; ++i) {
                    v[k][i] = row_ok ? *reinterpret_cast<const float2*>(q + k * 16 + i * 8 + 2 * (lane & 3)) : make_float2(0.f, 0.f);
                    mx = fmax_nan(mx, fmax_nan(fabsf(v[k][i].x), fabsf(v[k][i].y)));
                }
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
                    split_half2(x, y, qa[k][2 * i], qa[k][2 * i + 1]);
                }
        }
        const float sc = A.cap2 != 0.f ? qscale : qscale * A.scale2;
        const float slope2 = A.slopes ? A.slopes[h] * 1.44269504088896341f : 0.f;

        // ldmatrix row addresses: K matrices (keys 0-7 | 8-15) x (dims 0-7 | 8-15), V the same, transposed
        const uint32_t k_row = static_cast<uint32_t>(((lane & 7) + ((lane >> 4) << 3)) * RH + ((lane >> 3) & 1) * 8) * 2;
        const uint32_t v_row = static_cast<uint32_t>(((lane & 7) + (((lane >> 3) & 1) << 3)) * RH + (lane >> 4) * 8) * 2;

        int slot = 0;
        for (int i = i0; i < i1; i += step) {
            {
                const int ahead = i + (S::stages - 1) * step;
                const int32_t pg = next_page;
                next_page = page_of(ahead + step);
                issue(ahead, slot == 0 ? S::stages - 1 : slot - 1, pg);   // the stage read in the last round
            }
            cp_wait<S::stages - 1>();
            __syncwarp();
            const uint32_t sk = ring + static_cast<uint32_t>(slot) * S::stage_halves * 2, sv_ = sk + kKeyBlock * RH * 2;
            __half* vb = reinterpret_cast<__half*>(my_smem + (sv_ - ring));
            const int32_t j0 = kb.at(i) * kKeyBlock;

            float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};   // keys 0-7, 8-15
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t b[4];
                ldsm4(b, sk + k_row + k * 32);
                mma16816(s0, qa[k], b[0], b[1]);
                mma16816(s1, qa[k], b[2], b[3]);
            }
            float s[4] = {s0[0] + s0[2], s0[1] + s0[3], s1[0] + s1[2], s1[1] + s1[3]};
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
            if (!mask.all(p_lo, p_hi, j0, j0 + kKeyBlock)) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (!keys.sees(jc + (c >> 1) * 8 + (c & 1))) s[c] = -INFINITY;
                // A key that some row does not see has P = 0 there, which would make
                // NaN of an infinite or NaN v. Such values (there are none in a sound
                // cache) are added where they are seen and then cleared, so that they
                // reach no other row. Keys past the sequence are zeros.
                bool odd = false;
                for (int c = lane; c < kKeyBlock * PIECES; c += 32) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vb + (c / PIECES) * RH + (c % PIECES) * 8);
                    odd |= nonfinite_h2(w.x) || nonfinite_h2(w.y) || nonfinite_h2(w.z) || nonfinite_h2(w.w);
                }
                if (__any_sync(0xffffffffu, odd)) {
                    for (int j = 0; j < kKeyBlock; ++j) {
                        const bool seen = keys.sees(j0 + j);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const float x = __half2float(vb[j * RH + n * 8 + 2 * (lane & 3) + c]);
                                if (seen && !isfinite(x)) acc[n][c] += x;
                            }
                    }
                    __syncwarp();
                    for (int c = lane; c < kKeyBlock * HD; c += 32) {
                        __half& x = vb[(c / HD) * RH + c % HD];
                        if (!isfinite(__half2float(x))) x = __float2half_rn(0.f);
                    }
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
            __syncwarp();   // the warp is done with this stage before it is refilled
            slot = slot + 1 == S::stages ? 0 : slot + 1;
        }
        cp_wait<0>();
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
    }

    if (hg.subs > 1) {
        // the warps that share a head, in order
        const int row = lane >> 2;
        float* mine = reinterpret_cast<float*>(my_smem) + row * (HD + 2);
        if (active && sub > 0) {
            if ((lane & 3) == 0) *reinterpret_cast<float2*>(mine) = make_float2(m, l);
#pragma unroll
            for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(mine + 2 + n * 8 + 2 * (lane & 3)) = make_float2(acc[n][0], acc[n][1]);
        }
        __syncthreads();
        if (active && sub == 0) {
            for (int s = 1; s < hg.subs; ++s) {
                const float* o = reinterpret_cast<const float*>(my_smem + static_cast<size_t>(s) * hg.heads * S::warp_bytes) + row * (HD + 2);
                const float2 ml = *reinterpret_cast<const float2*>(o);
                const float M = fmaxf(m, ml.x);
                // a side that saw nothing adds its l and acc too: zeros, or the NaN of a row that is not finite
                const float fa = m == -INFINITY ? 1.f : ex2(m - M), fb = ml.x == -INFINITY ? 1.f : ex2(ml.x - M);
                m = M;
                l = fmaf(ml.y, fb, l * fa);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 v = *reinterpret_cast<const float2*>(o + 2 + n * 8 + 2 * (lane & 3));
                    acc[n][0] = fmaf(v.x, fb, acc[n][0] * fa);
                    acc[n][1] = fmaf(v.y, fb, acc[n][1] * fa);
                }
            }
        }
        __syncthreads();   // shared memory is free again
    }
    if (!active || sub > 0 || !row_ok) return;
    if (part < 0) {
        float* o = A.out + static_cast<int64_t>(sv.q0 + t) * A.ldo + static_cast<int64_t>(h) * HD + 2 * (lane & 3);
        const float inv = l == 0.f ? 0.f : 1.f / l;   // nothing seen: zeros
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(o + n * 8) = make_float2(acc[n][0] * inv, acc[n][1] * inv);
    } else {
        const int64_t at = (static_cast<int64_t>(part) * S::warps + warp) * kRowTile + (lane >> 2);
        float* ml = A.part + S::cut_bytes / 4;
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + at * 2) = make_float2(m, l);
        float* o = ml + S::part_rows * 2 + at * HD + 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(o + n * 8) = make_float2(acc[n][0], acc[n][1]);
    }
}

// What combine_kernel adds up: the parts of (tile, grp) are `first`, then the
// first part of each of the next n - 1 CTAs. n < 2: nothing, it lies in one run.
// Few (tile, group)s have an entry each; else there is one for each CTA, for
// the cut before its run (if that is the first one of what it cuts).
struct __align__(16) Cut {
    int32_t tile, grp, first, n;
};

__host__ __device__ inline bool by_tile(int tiles, const HeadGroups& hg) { return static_cast<int64_t>(tiles) * hg.groups <= kRowsCtas; }

// A.n_split tiles in equal runs; 0: one CTA for each tile and group, where these are many.
template <int HD>
__global__ void __launch_bounds__(RowsShape<HD>::warps * 32, 1)
rows_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int W = RowsShape<HD>::warps;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_pre[kMostTiles + 1];
    __shared__ int64_t s_sum[W];
    const HeadGroups hg(A.c.n_kv, W);
    const int tiles = A.n_split;
    grid_dep_wait();
    if (tiles == 0) {
        const int nb = tile_blocks(A, static_cast<int>(blockIdx.x), threadIdx.x == 0);
        if (nb > 0) rows_segment<HD>(A, smem, hg, static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.y), 0, nb, -1);
        return;
    }
    grid_dep_launch();   // combine_kernel may be set up meanwhile; it waits for this grid's end
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t before = 0;
    if (threadIdx.x == 0) s_pre[0] = 0;
    for (int i0 = 0; i0 < tiles; i0 += W * 32) {
        const int i = i0 + threadIdx.x;
        const int nb = i < tiles ? tile_blocks(A, i, blockIdx.x == 0) : 0;
        int64_t v = nb > 0 ? nb + kSegCost : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += y;
        }
        if (lane == 31) s_sum[warp] = v;
        __syncthreads();
        int64_t all = 0;
        for (int w = 0; w < W; ++w) {
            if (w < warp) v += s_sum[w];
            all += s_sum[w];
        }
        if (i < tiles) s_pre[i + 1] = before + v;
        before += all;
        __syncthreads();
    }
    Runs runs{before * hg.groups, 1};
    runs.n_cta = static_cast<int>(max(int64_t(1), min(static_cast<int64_t>(gridDim.x), runs.units / kLeastUnits)));
    const int cta = blockIdx.x;
    const bool listed_by_tile = by_tile(tiles, hg);
    Cut* cuts = reinterpret_cast<Cut*>(A.part);
    if (listed_by_tile && cta == 0)   // those without rows
        for (int i = threadIdx.x; i < tiles * hg.groups; i += W * 32)
            if (s_pre[i / hg.groups + 1] == s_pre[i / hg.groups]) cuts[i] = Cut{0, 0, 0, 0};
    Cut cut{0, 0, 0, 0};
    if (runs.units > 0 && cta < runs.n_cta) {
        int64_t u = runs.start(cta);
        const int64_t begin = u, end = runs.start(cta + 1);
        int lo = 0, hi = tiles - 1;   // the last tile that starts at or before u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_pre[mid] * hg.groups <= u) lo = mid;
            else hi = mid - 1;
        }
        while (u < end) {
            while (s_pre[lo + 1] * hg.groups <= u) ++lo;   // tiles without rows have no units
            const int64_t n = s_pre[lo + 1] - s_pre[lo], off = u - s_pre[lo] * hg.groups;
            const int grp = static_cast<int>(off / n);
            const int64_t first = s_pre[lo] * hg.groups + grp * n;   // of kSegCost, then the blocks
            const int64_t stop = min(end, first + n);
            if (stop > first + kSegCost) {
                const int64_t b0 = max(u, first + kSegCost) - first - kSegCost, b1 = stop - first - kSegCost;
                const int c_first = runs.cta_of(first + kSegCost), c_last = runs.cta_of(first + n - 1);
                const int which = begin >= first ? 0 : 1;
                const Cut all{lo, grp, 2 * c_first + (runs.start(c_first) >= first ? 0 : 1), c_last - c_first + 1};
                if (cta == c_first + 1) cut = all;
                if (listed_by_tile && cta == c_first && threadIdx.x == 0) cuts[lo * hg.groups + grp] = all;
                rows_segment<HD>(A, smem, hg, lo, grp, static_cast<int>(b0), static_cast<int>(b1), c_first == c_last ? -1 : 2 * cta + which);
            }
            u = stop;
        }
    }
    if (!listed_by_tile && threadIdx.x == 0) cuts[cta] = cut;
}

// The parts of one row of what is cut: block (entry, head of the group, row).
template <int HD>
__global__ void __launch_bounds__(256)
combine_kernel(const __grid_constant__ AttnArgs A) {
    using S = RowsShape<HD>;
    __shared__ float s_w[kRowsCtas];
    __shared__ float s_red[2][8];
    __shared__ float4 s_o[256];
    grid_dep_wait();
    grid_dep_launch();
    const int4 c4 = __ldcg(reinterpret_cast<const int4*>(A.part) + blockIdx.x);
    const Cut cut{c4.x, c4.y, c4.z, c4.w};
    if (cut.n < 2) return;
    const HeadGroups hg(A.c.n_kv, S::warps);
    const int hl = blockIdx.y, row = blockIdx.z, kvh = cut.grp * hg.heads + hl;
    if (hl >= hg.heads || kvh >= A.c.n_kv) return;
    int seq, tile;
    locate_tile(A.b, A.group, kRowTile, A.per_seq, cut.tile, seq, tile);
    const SeqView sv = seq_view(A.c, A.b, seq);
    const int r = tile * kRowTile + row;
    if (r >= sv.n_new * A.group) return;
    const int t = r / A.group, h = kvh * A.group + r - t * A.group;
    const float* ml = A.part + S::cut_bytes / 4;
    const float* acc = ml + S::part_rows * 2;
    // parts `first`, then slot 0 of the CTAs after it
    auto at = [&](int i) { return (static_cast<int64_t>(i == 0 ? cut.first : 2 * ((cut.first >> 1) + i)) * S::warps + hl) * kRowTile + row; };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // every part's weight, and the sum (at most 148 parts: one a thread)
    float2 p = make_float2(-INFINITY, 0.f);
    if (static_cast<int>(threadIdx.x) < cut.n) p = __ldcg(reinterpret_cast<const float2*>(ml + at(threadIdx.x) * 2));
    float M = p.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) s_red[0][warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) M = fmaxf(M, s_red[0][w]);
    // a part that saw nothing adds zeros, or the NaN of a row that is not finite
    const float f = p.x == -INFINITY ? 1.f : ex2(p.x - M);
    if (static_cast<int>(threadIdx.x) < cut.n) s_w[threadIdx.x] = f;
    float L = p.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) s_red[1][warp] = L;
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) L += s_red[1][w];
    // thread (dims d .. d + 3, share of the parts)
    constexpr int Q = HD / 4, SHARES = 256 / Q;
    const int d = threadIdx.x % Q, share = threadIdx.x / Q;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = share; i < cut.n; i += SHARES) {
        const float4 a = __ldcg(reinterpret_cast<const float4*>(acc + at(i) * HD) + d);
        const float w = s_w[i];
        o.x = fmaf(a.x, w, o.x);
        o.y = fmaf(a.y, w, o.y);
        o.z = fmaf(a.z, w, o.z);
        o.w = fmaf(a.w, w, o.w);
    }
    s_o[threadIdx.x] = o;
    __syncthreads();
    if (share == 0) {
        for (int s = 1; s < SHARES; ++s) {
            const float4 a = s_o[s * Q + d];
            o.x += a.x;
            o.y += a.y;
            o.z += a.z;
            o.w += a.w;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        reinterpret_cast<float4*>(A.out + static_cast<int64_t>(sv.q0 + t) * A.ldo + static_cast<int64_t>(h) * HD)[d] =
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
}

struct Plan {
    bool tc;         // chunk_kernel of paged_attention_tc.cu
    bool balanced;   // rows_kernel in equal runs
    int rows, per_seq, tiles, blocks_per_split, n_split;
};

// How a call is cut: from the host's bounds alone, so that a captured graph
// serves every later length within them.
Plan make_plan(const hesa_cuda_paged_kv* kv, const hesa_cuda_token_batch* b, int64_t n_head) {
    Plan p{};
    const int g = static_cast<int>(n_head / kv->n_kv_head);
    const int64_t rows_a_seq = static_cast<int64_t>(b->max_new) * g;
    p.tc = kv->head_dim <= 128 && rows_a_seq > 4 * kRowTile;
    p.rows = p.tc ? kTcRows : kRowTile;
    const int64_t most = (rows_a_seq + p.rows - 1) / p.rows;
    const int64_t bound = tile_bound(b->n_tokens, b->n_seq, g, p.rows);
    p.per_seq = b->n_seq * most <= bound ? static_cast<int>(most) : 0;
    const int64_t tiles = p.per_seq ? b->n_seq * most : bound;
    p.tiles = static_cast<int>(tiles);
    const int64_t pairs = tiles * kv->n_kv_head;
    if (!p.tc) {
        p.balanced = tiles <= kMostTiles;
        return p;
    }
    // one CTA an SM, no split under 512 keys
    const int64_t blocks = std::max<int64_t>(1, (b->max_len + kTcKeys - 1) / kTcKeys);
    int64_t per = blocks;
    if (pairs <= kPagedPairs) {
        const int64_t want = std::max<int64_t>(1, 148 / pairs);
        per = std::max<int64_t>(4, (blocks + want - 1) / want);
    }
    p.blocks_per_split = static_cast<int>(std::min(per, blocks));
    p.n_split = static_cast<int>((blocks + p.blocks_per_split - 1) / p.blocks_per_split);
    return p;
}

size_t part_bytes(const Plan& p, const hesa_cuda_paged_kv* kv) {
    const size_t row = static_cast<size_t>(kv->head_dim + 2) * sizeof(float);
    if (!p.tc) return !p.balanced ? 0 : kv->head_dim == 64 ? RowsShape<64>::part_bytes : kv->head_dim == 128 ? RowsShape<128>::part_bytes : RowsShape<256>::part_bytes;
    return p.n_split > 1 ? static_cast<size_t>(p.tiles) * kv->n_kv_head * p.n_split * p.rows * row : 0;
}

template <int HD>
cudaError_t launch_rows(const AttnArgs& a, const Plan& p, cudaStream_t s) {
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
    const HeadGroups hg(a.c.n_kv, S::warps);
    const dim3 grid = p.balanced ? dim3(kRowsCtas) : dim3(static_cast<unsigned>(p.tiles), static_cast<unsigned>(hg.groups));
    e = launch_dep(rows_kernel<HD>, grid, S::warps * 32, S::smem, s, a);
    if (e != cudaSuccess || !p.balanced) return e;
    const int cuts = by_tile(a.n_split, hg) ? a.n_split * hg.groups : kRowsCtas;
    const int rows = std::min(kRowTile, a.b.max_new * a.group);
    return launch_dep(combine_kernel<HD>, dim3(static_cast<unsigned>(cuts), static_cast<unsigned>(hg.heads), static_cast<unsigned>(rows)), 256, 0, s, a);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace

int check_paged_kv(const hesa_cuda_paged_kv* kv) {
    if (!kv || !kv->k || !kv->v || !kv->table || !kv->seq_len) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (kv->n_layer <= 0 || kv->n_pages <= 0 || kv->page_size <= 0 || kv->n_kv_head <= 0 || kv->n_slots <= 0 || kv->max_pages <= 0)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "non-positive dimension");
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "head_dim must be 64, 128 or 256");
    if (kv->page_size > 65536 || kv->n_kv_head > 1024 || kv->n_slots > 65536 || kv->n_layer > 4096 ||
        static_cast<int64_t>(kv->max_pages) * kv->page_size >= (int64_t(1) << 30))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "paged cache too large");
    const int64_t page = static_cast<int64_t>(kv->page_size) * kv->n_kv_head * kv->head_dim;
    const int64_t most = int64_t(1) << 50;
    if (kv->page_stride < page || kv->page_stride > most || kv->layer_stride < 0 || kv->layer_stride > most || (kv->page_stride & 7) || (kv->layer_stride & 7))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "page_stride and layer_stride must be multiples of 8, page_stride at least a page");
    if (kv->n_layer > 1 && kv->layer_stride < (static_cast<int64_t>(kv->n_pages) - 1) * kv->page_stride + page &&
        (kv->layer_stride < page || kv->page_stride < (static_cast<int64_t>(kv->n_layer) - 1) * kv->layer_stride + page))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "the pages of two layers overlap");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the page pools must be 16-byte aligned");
    if (!aligned(kv->table, 4) || !aligned(kv->seq_len, 4)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "the tables must be 4-byte aligned");
    return HESA_CUDA_OK;
}

int check_batch(const hesa_cuda_paged_kv* kv, int32_t layer, const hesa_cuda_token_batch* b, int64_t n_head) {
    if (layer < 0 || layer >= kv->n_layer) return record_error(HESA_CUDA_INVALID_ARGUMENT, "no such layer");
    if (!b || !b->q_start) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
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
    return c;
}

BatchView view_of(const hesa_cuda_token_batch* b) { return BatchView{b->slots, b->q_start, b->n_seq, b->n_tokens, b->max_new, b->max_len}; }

}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_paged_attention_workspace_size(const hesa_cuda_paged_kv* kv, const hesa_cuda_token_batch* batch, int64_t n_head) {
    if (check_paged_kv(kv) != HESA_CUDA_OK || check_batch(kv, 0, batch, n_head) != HESA_CUDA_OK) return 0;
    const Plan p = make_plan(kv, batch, n_head);
    return kPagedCounterBytes + part_bytes(p, kv);
}

int hesa_cuda_paged_attention(const hesa_cuda_paged_kv* kv, int32_t layer, const hesa_cuda_token_batch* batch, const float* q,
                              int64_t ldq, float* out, int64_t ldo, int64_t n_head, const hesa_cuda_attn_options* options,
                              void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_paged_attention");
    int rc = check_paged_kv(kv);
    if (rc == HESA_CUDA_OK) rc = check_batch(kv, layer, batch, n_head);
    if (rc != HESA_CUDA_OK) return rc;
    if (!q || !out || !workspace) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    const int64_t width = n_head * kv->head_dim;
    if (ldq < width || ldo < width || ldq > (int64_t(1) << 40) || ldo > (int64_t(1) << 40))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "leading dimension too small");
    if (!aligned(q, 16) || !aligned(out, 16) || (ldq & 3) || (ldo & 3))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "q / out must be 16-byte aligned with ldq, ldo multiples of 4");
    if (!aligned(workspace, 16)) return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    if (workspace_bytes < hesa_cuda_paged_attention_workspace_size(kv, batch, n_head))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    hesa_cuda_attn_options o{};
    if (options) o = *options;
    if (!(o.scale >= 0.f) || !std::isfinite(o.scale) || !(o.softcap >= 0.f) || !std::isfinite(o.softcap) || o.window < 0)
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "scale, softcap and window must be finite and not negative");
    if (batch->n_tokens == 0 || batch->max_new == 0) return HESA_CUDA_OK;

    const Plan p = make_plan(kv, batch, n_head);
    AttnArgs a{};
    a.c = layer_of(kv, layer);
    a.b = view_of(batch);
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.n_head = static_cast<int32_t>(n_head);
    a.group = static_cast<int32_t>(n_head / kv->n_kv_head);
    const double log2e = 1.4426950408889634;
    const double scale = o.scale > 0.f ? o.scale : 1.0 / std::sqrt(static_cast<double>(kv->head_dim));
    a.scale2 = static_cast<float>(scale * log2e);
    a.cap2 = static_cast<float>(o.softcap * log2e);
    a.cap_in = o.softcap > 0.f ? static_cast<float>(scale / o.softcap) : 0.f;
    a.window = o.window;
    a.slopes = o.slopes;
    a.prefix = o.prefix;
    a.counters = static_cast<int32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kPagedCounterBytes);
    a.per_seq = p.per_seq;
    a.blocks_per_split = p.blocks_per_split;
    a.n_split = p.tc ? p.n_split : p.balanced ? p.tiles : 0;
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
