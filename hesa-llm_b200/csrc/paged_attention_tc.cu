// paged_attention_tc.cu -- paged attention of chunks on the 5th-generation
// tensor cores (tcgen05, TMEM): tiles of 128 rows (query heads of one kv head
// times new tokens) over blocks of 128 keys.
//
// The formulas and the split of q and P into two fp16 halves are those of
// paged_attention.cu. Here the halves are two products each: S = Q_lo K^T +
// Q_hi K^T and O = P_hi V + P_lo V, four 128 x 128 x head_dim products a block
// of keys, so the floor is twice that of fp16 attention's matrix work. It is
// bound by the tensor cores.
//
// TMEM (512 columns): Q_hi | Q_lo (head_dim columns), two S buffers of 128
// columns, O (head_dim columns). Q as a TMEM operand leaves all of shared memory
// to a ring of K and V blocks and halves the operand reads of Q K^T. A buffer's
// S is overwritten by its P where it lies: columns 16 c .. 16 c + 7 hold the high
// halves of keys 16 c .. 16 c + 15, the next 8 the low halves.
//
// Warps 0-3 and 4-7 (compute) take every second block each, a row a thread, with
// their own maximum, sum and output registers, which meet at the end: while one
// warpgroup waits for P V and adds the last O, the other makes its P. (With both
// on the same block, 64 keys a thread, the rows' maxima had to be exchanged and
// all eight warps wanted the same pipes at the same time: 3000 cycles a block,
// 1.75 ms for 2048 tokens at 16384, 64 heads on 8.) A block's maximum is found in
// a first pass over S in TMEM, P is made in a second. O is a fresh product for
// every block, added to fp32 registers with one fma that rescales: only 16
// products are summed by the tensor core, and long sums round to nearest.
// One thread of warp 8 issues P V, one of warp 9 Q K^T, so that neither's waits
// hold up the other's products. S of block j + 2 goes into the buffer
// that held P of block j once P V of block j has completed: no pair of products
// relies on an order that the instruction set does not promise. (Writing it in
// halves of 64 keys, each as soon as its half of P had been read, kept a product
// queued at all times, but a product of 64 columns takes 56 cycles where one of
// 128 takes 64.)
// Warps 10, 11 (producers): K and V blocks into the 128-byte swizzled layout with
// tiled copies (TMA) of boxes of gcd(page_size, 128) tokens by 64 dims; a page
// that is not there is a coordinate past the pool, which reads as zeros. Pages
// whose size is no multiple of 8 are copied with 16-byte cp.async (a K block
// takes each warp about 1800 cycles).
// With head_dim 256 q alone takes half of TMEM: blocks have 64 keys, and two CTAs
// share a tile, each with all of Q K^T and half of the dims of V. (Q K^T twice is
// half as much work again; one CTA for both halves would need 256 output registers
// a thread.)
// Measured, 64 heads on 8: 2048 tokens at 16384 1.72 ms with pages of 64 (600
// TFLOP/s, 1200 counting the halves' products; 88% of what the tensor cores keep
// up at the clock that the power limit leaves), 2.58 ms with pages of 7. 1024 tokens at
// 4096, 4 heads of 256: 71 us, where tiles of 8 rows take 194.
#include "paged.h"
#include "paged_tc.h"
#include "qmatvec.h"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <algorithm>
#include <numeric>

namespace hesa_cuda {
namespace {

constexpr int kM = kTcRows;                  // rows of a tile = TMEM lanes
constexpr int kComputeWarps = 8;
constexpr int kQkWarp = kComputeWarps + 1;   // issues Q K^T, the warp before it P V
constexpr int kProducerWarps = 2;
constexpr int kFirstProducer = kComputeWarps + 2;
constexpr int kThreads = 384;                // three warpgroups
// Registers a thread after setmaxnreg: 256 x 208 + 128 x 88 = 384 x 168, what
// the block is launched with.
constexpr int kComputeRegs = 208, kOtherRegs = 88;
constexpr int kInFlight = 3;                 // blocks that a producer has in flight with cp.async

template <int HD> struct TcShape {
    static constexpr int keys = tc_keys(HD), vd = tc_dims(HD);   // keys of a block, dims of V that a CTA works on
    static constexpr int parts = HD / vd;                        // CTAs of a (tile, kv head, split)
    static constexpr uint32_t slot = keys * HD * 2;          // one K block; a V block is no larger
    static constexpr int slots = HD == 64 ? 8 : 6;
    static constexpr uint32_t smem = slot * slots + 1024;    // + alignment of the swizzle
    static constexpr uint32_t q_hi = 0, q_lo = HD / 2, s0 = HD, o = HD + 2 * keys;
    static_assert(o + vd <= 512, "TMEM columns");
    static constexpr int64_t part = kM * (vd + 2);           // floats of a part: acc [kM][vd], then (m, l) [kM]
};

// ---- tcgen05 ----
// D (+)= A B, A from TMEM, B from shared memory, fp16 in, fp32 out.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1 : 0), "r"(0)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 / 32 consecutive columns of this warp's 32 lanes, one lane a thread
__device__ __forceinline__ void st16(uint32_t t, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void st8(uint32_t t, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void ld16(uint32_t t, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(t));
}
__device__ __forceinline__ void st32(uint32_t t, const float* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void ld32(uint32_t t, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
// wait for this thread's tcgen05.ld; the registers are redefined after it so
// that no use is scheduled before the wait
template <int N>
__device__ __forceinline__ void wait_ld(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

// Shared-memory descriptors of 128-byte swizzled blocks: 64 fp16 (128 bytes) a
// row, 8-row groups of 1024 bytes. K-major (K): the group stride is the second
// offset, the first is not used. MN-major (V: a row is a key, its 64 values run
// along N): the first offset is the stride to the next 64 of N, the second that
// to the next 8 keys.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t first, uint32_t second) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((first >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>((second >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// fp32 accumulator, fp16 operands, M = 128; bit 16: B is MN-major
constexpr uint32_t idesc_f16(int n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kM >> 4) << 24);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool have) {
    const int n = have ? 16 : 0;   // 0: sixteen zero bytes, src is not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// 4-D tiled copy of the box at (x, head, place in page, page)
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int head, int place, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(place), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// x = hi + lo to 22 bits for 0 <= x < 65504: hi is x cut to 11 bits, which costs no
// conversion back and so has lo follow from x by one mask and one subtraction
__device__ __forceinline__ void cut_half2(float2 x, uint32_t& hi, uint32_t& lo) {
    const float2 h = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xFFFFE000u), __uint_as_float(__float_as_uint(x.y) & 0xFFFFE000u));
    const float2 l = ffma2(h, make_float2(-1.f, -1.f), x);
    const __half2 a = __floats2half2_rn(h.x, h.y), b = __floats2half2_rn(l.x, l.y);
    hi = *reinterpret_cast<const uint32_t*>(&a);
    lo = *reinterpret_cast<const uint32_t*>(&b);
}

// cap2 tanh(x) for two |x| <= 0.6: tanh(x) = x + x u q(u), u = x^2, q of degree 4
// fitted to (tanh(x) / x - 1) / u at Chebyshev nodes of u in [0, 0.36]; with its
// coefficients in fp32 the relative error is below 1.5e-8.
__device__ __forceinline__ float2 capped2_small(float2 x, float cap2) {
    const float2 u = ffma2(x, x, make_float2(0.f, 0.f));
    float2 q = make_float2(-0.006276387721f, -0.006276387721f);
    q = ffma2(q, u, make_float2(0.021116213873f, 0.021116213873f));
    q = ffma2(q, u, make_float2(-0.053875137120f, -0.053875137120f));
    q = ffma2(q, u, make_float2(0.133329242468f, 0.133329242468f));
    q = ffma2(q, u, make_float2(-0.333333313465f, -0.333333313465f));
    const float2 y = ffma2(x, make_float2(cap2, cap2), make_float2(0.f, 0.f));
    return ffma2(y, ffma2(u, q, make_float2(0.f, 0.f)), y);
}

// The low n bits set, 0 <= n <= 32 or clamped to that.
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Places in the ring: K0, K1, V0, K2, V1, ... , the order in which they are used.
__device__ __forceinline__ int k_place(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_place(int j, int n) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; }

template <int HD, bool TMA>
__global__ void __launch_bounds__(kThreads, 1)
chunk_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int box) {
    using S = TcShape<HD>;
    constexpr int kN = S::keys, VD = S::vd, HH = VD / 2, HQ = HD / 2;   // HH, HQ: output dims and dims of q of a thread
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[S::slots], empty[S::slots], s_full[2], p_full[2][2], o_full[2], o_free, q_done, drained[2];
    __shared__ float2 s_ml[2][kM];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag, odd_block[2];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int kvh = blockIdx.y / S::parts, v0 = (blockIdx.y % S::parts) * VD, split = blockIdx.z;   // v0: its first dim of V
    grid_dep_wait();
    grid_dep_launch();
    int seq, tile;
    if (!locate_tile(A.b, A.group, kM, A.per_seq, static_cast<int>(blockIdx.x), seq, tile)) return;
    const SeqView sv = seq_view(A.c, A.b, seq);
    if (!sv.ok) {
        if (threadIdx.x == 0) record_status(A.status, kStatusBadPosition);
        return;
    }
    const int n_rows = sv.n_new * A.group;
    if (tile * kM >= n_rows) return;
    // later rows see more keys: the longest tiles of a sequence start first
    const int r0 = ((n_rows + kM - 1) / kM - 1 - tile) * kM;
    const int base = sv.len - sv.n_new;
    const int32_t p_lo = base + A.group_div.div(r0);
    const int32_t p_hi = base + A.group_div.div(min(r0 + kM - 1, n_rows - 1));
    Mask mask{sv.len, A.window, 0};
    if (A.prefix) mask.prefix = max(0, min(A.prefix[seq], sv.len));
    const KeyBlocks kb = key_blocks(mask, p_lo, p_hi, kN);
    const int n_parts = max(1, (kb.n + A.blocks_per_split - 1) / A.blocks_per_split);
    if (split >= n_parts) return;
    const int i0 = split * A.blocks_per_split;
    const int n = min(kb.n, i0 + A.blocks_per_split) - i0;   // blocks of this CTA; 0: the rows see nothing

    const uint32_t ring = (smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - smem_addr(smem_raw));
    volatile int* abort_v = &abort_flag;

    // q comes through the last slots of the ring, whole rows at a time (a thread that
    // read its own row from memory waited 7 us for rows 16 KB apart), 16-byte pieces
    // swizzled by the row so that a row a thread is read without bank conflicts
    constexpr int kQSlots = kM * HD * 4 / S::slot;
    static_assert(kM * HD * 4 == kQSlots * S::slot && kQSlots < S::slots, "q fills whole slots");
    uint8_t* q_smem = ring_ptr + (S::slots - kQSlots) * S::slot;
    if (warp < kComputeWarps) {
        constexpr int PIECES = HD / 4;
#pragma unroll
        for (int i = 0; i < kM * PIECES / (kComputeWarps * 32); ++i) {
            const int p = i * kComputeWarps * 32 + threadIdx.x, qr = p / PIECES, c = p % PIECES;
            const int rr = min(r0 + qr, n_rows - 1), qt = A.group_div.div(rr);
            const float* src = A.q + static_cast<int64_t>(sv.q0 + qt) * A.ldq + static_cast<int64_t>(kvh * A.group + rr - qt * A.group) * HD + c * 4;
            cp16(smem_addr(q_smem) + qr * HD * 4 + ((c ^ (qr & 7)) << 4), src, true);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::slots; ++i) {
            mbar_init(&full[i], kProducerWarps);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&drained[i], 1);
            for (int h = 0; h < 2; ++h) mbar_init(&p_full[i][h], kComputeWarps / 2);
        }
        mbar_init(&o_free, kComputeWarps / 2);
        mbar_init(&q_done, kComputeWarps);
        abort_flag = 0;
        odd_block[0] = odd_block[1] = -1;
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base;

    const int half = warp >> 2, wq = warp & 3;
    const int row = 32 * wq + lane;                       // of the tile, = TMEM lane
    const uint32_t tl = tmem + (static_cast<uint32_t>(32 * wq) << 16);
    const int r = min(r0 + row, n_rows - 1);
    const int t = A.group_div.div(r), h = kvh * A.group + r - t * A.group;
    const int32_t pos = base + t;

    if (warp >= kComputeWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (TMA && warp >= kFirstProducer) {
            // ---- producers: copy c of a block (64 dims of `box` keys) is lane c / 2's of warp c % 2 ----
            const int pw = warp - kFirstProducer, c = lane * kProducerWarps + pw, copies = (kN / box) * (HD / 64);
            const int g = c / (HD / 64), x = c % (HD / 64);   // which keys, which dims
            const uint32_t mine = static_cast<uint32_t>((copies - pw + kProducerWarps - 1) / kProducerWarps) * box * 128;   // bytes of the warp
            const int32_t* table = A.c.table + static_cast<int64_t>(sv.slot) * A.c.max_pages;
            const uint32_t to = ring + static_cast<uint32_t>(x * kN + g * box) * 128;
            bool dead = false;
            int issued = 0;   // places that this warp has filled, in their order
            // the page and the place in it of this lane's keys of block j; no page: one past the pool
            auto find = [&](int j, int& page, int& at) {
                page = A.c.n_pages;
                at = 0;
                if (j < n && c < copies) {
                    const int32_t key = kb.at(i0 + j) * kN + g * box;
                    const int32_t pi = A.c.page_div.div(key);
                    at = key - pi * A.c.page_size;
                    if (key < sv.len) {
                        const int32_t p = table[pi];
                        if (p >= 0 && p < A.c.n_pages) page = p;
                        else record_status(A.status, kStatusBadPosition);
                    }
                }
            };
            // dims [from, from + 64 * wide) of the block's keys
            auto put = [&](int place, const CUtensorMap* map, int page, int at, int from, int wide) {
                const int slot = place % S::slots;
                if (place >= S::slots && !dead)
                    dead = !mbar_warp_wait(&empty[slot], static_cast<uint32_t>(place / S::slots - 1) & 1u, A.status, kStatusWaitTimeout);
                else if (place >= S::slots - kQSlots && !dead)
                    dead = !mbar_warp_wait(&q_done, 0u, A.status, kStatusWaitTimeout);
                if (dead) return;
                if (lane == 0) mbar_arrive_expect_tx(&full[slot], mine * wide / (HD / 64));   // a warp's dims are every second 64 of a box, or all
                __syncwarp();
                issued = place + 1;
                if (c < copies && x < wide) tma_4d(to + static_cast<uint32_t>(slot) * S::slot, map, from + x * 64, kvh, at, page, &full[slot]);
            };
            if (n > 0) {
                int page, at, page1, at1;
                find(0, page, at);
                put(0, &kmap, page, at, 0, HD / 64);
                for (int j = 0; j < n; ++j) {
                    find(j + 1, page1, at1);
                    if (j + 1 < n) put(k_place(j + 1), &kmap, page1, at1, 0, HD / 64);
                    put(v_place(j, n), &vmap, page, at, v0, VD / 64);
                    page = page1;
                    at = at1;
                }
                // nothing may be in flight when the CTA ends, whoever gave up
                for (int p = max(0, issued - S::slots); p < issued; ++p)
                    if (!mbar_wait_bounded(&full[p % S::slots], static_cast<uint32_t>(p / S::slots) & 1u, A.status, kStatusDrainTimeout)) break;
            }
        } else if (!TMA && warp >= kFirstProducer) {
            // ---- producers: warp w of them copies keys 64 w .. 64 w + 63 of every block ----
            static_assert(TMA || (VD == HD && kN == 128), "the shapes that are copied without TMA");
            const int pw = warp - kFirstProducer;
            constexpr int PIECES = HD / 8;          // 16-byte pieces of a row
            constexpr int KEYS = kN / kProducerWarps, ROWS = 32 / PIECES;
            const int32_t* table = A.c.table + static_cast<int64_t>(sv.slot) * A.c.max_pages;
            const int64_t row_elems = static_cast<int64_t>(A.c.n_kv) * HD;
            const int at = lane % PIECES, psz = A.c.page_size;
            const uint32_t to = ring + static_cast<uint32_t>(at >> 3) * (kN * 128) + static_cast<uint32_t>(pw) * KEYS * 128;
            bool dead = false;
            // lane's keys lane, lane + 32 of block j: their pages, asked for one block ahead
            int32_t pg[2];
            auto ask = [&](int j) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int32_t key = j < n ? kb.at(i0 + j) * kN + pw * KEYS + u * 32 + lane : sv.len;
                    pg[u] = key < sv.len ? table[A.c.page_div.div(key)] : -1;
                }
            };
            // and where their rows lie; -1: nowhere, zeros are put there
            auto find = [&](int j, int64_t (&off)[2]) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int32_t key = kb.at(i0 + j) * kN + pw * KEYS + u * 32 + lane;
                    off[u] = -1;
                    if (key < sv.len) {
                        if (pg[u] >= 0 && pg[u] < A.c.n_pages) off[u] = pg[u] * A.c.page_stride + (key - A.c.page_div.div(key) * psz) * row_elems + kvh * HD;
                        else record_status(A.status, kStatusBadPosition);
                    }
                }
            };
            auto arrive = [&](int place) {   // this thread's copies into it have landed
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[place % S::slots]);
            };
            auto put = [&](int place, const __half* pool, const int64_t (&off)[2]) {
                const int slot = place % S::slots;
                if (place >= S::slots && !dead)
                    dead = !mbar_warp_wait(&empty[slot], static_cast<uint32_t>(place / S::slots - 1) & 1u, A.status, kStatusWaitTimeout);
                else if (place >= S::slots - kQSlots && !dead)
                    dead = !mbar_warp_wait(&q_done, 0u, A.status, kStatusWaitTimeout);
                if (!dead) {
                    const uint32_t dst = to + static_cast<uint32_t>(slot) * S::slot;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll 8
                        for (int i = 0; i < 32; i += ROWS) {
                            const int kr = i + lane / PIECES;   // of the 32 keys
                            const int64_t o = __shfl_sync(0xffffffffu, off[u], kr);
                            cp16(dst + (u * 32 + kr) * 128 + ((static_cast<uint32_t>(at & 7) ^ (kr & 7)) << 4), pool + (o < 0 ? 0 : o) + at * 8, o >= 0);
                        }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (place >= kInFlight) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kInFlight) : "memory");
                    arrive(place - kInFlight);
                }
            };
            if (n > 0) {
                int64_t cur[2], nxt[2];
                ask(0);
                find(0, cur);
                ask(1);
                put(0, A.c.k, cur);
                for (int j = 0; j < n; ++j) {
                    if (j + 1 < n) {
                        find(j + 1, nxt);
                        ask(j + 2);
                        put(k_place(j + 1), A.c.k, nxt);
                    }
                    put(v_place(j, n), A.c.v, cur);
                    cur[0] = nxt[0];
                    cur[1] = nxt[1];
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                for (int p = max(0, 2 * n - kInFlight); p < 2 * n; ++p) arrive(p);
            }
        } else if (lane == 0) {
            // ---- products ----
            auto place = [&](int p) { return ring + static_cast<uint32_t>(p % S::slots) * S::slot; };
            auto landed = [&](int p) { return mbar_wait_bounded(&full[p % S::slots], static_cast<uint32_t>(p / S::slots) & 1u, A.status, kStatusWaitTimeout); };
            bool ok = true;
            // the address field of a descriptor counts 16 bytes: k-steps are added to it
            if (warp == kQkWarp) {
                if (n > 0) ok = mbar_wait_bounded(&q_done, 0u, A.status, kStatusWaitTimeout);
                for (int j = 0; j < n && ok && !*abort_v; ++j) {
                    // S of block j goes where P of block j - 2 has been read. (One barrier for all blocks could be a
                    // phase ahead by now; each buffer's own is not: its next phase needs this S.)
                    ok = landed(k_place(j)) && (j < 2 || mbar_wait_bounded(&o_full[j & 1], static_cast<uint32_t>((j >> 1) - 1) & 1u, A.status, kStatusWaitTimeout));
                    if (!ok) break;
                    fence_after();
                    const uint32_t d = tmem + S::s0 + static_cast<uint32_t>((j & 1) * kN);
                    const uint64_t b = desc(place(k_place(j)), 16, 1024);
#pragma unroll 1
                    for (int part = 0; part < 2; ++part) {   // the small products first
                        const uint32_t a = tmem + (part == 0 ? S::q_lo : S::q_hi);
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)
                            mma_ts(d, a + 8 * k, b + ((k >> 2) * (kN * 128) + (k & 3) * 32) / 16, idesc_f16(kN, false), part > 0 || k > 0);
                    }
                    commit(&s_full[j & 1]);
                    commit(&empty[k_place(j) % S::slots]);
                }
            } else {
                for (int j = 0; j < n && ok && !*abort_v; ++j) {
                    const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u, each = static_cast<uint32_t>(j) & 1u;
                    const uint64_t b = desc(place(v_place(j, n)), kN * 128, 1024);
                    ok = landed(v_place(j, n)) && (j == 0 || mbar_wait_bounded(&o_free, each ^ 1u, A.status, kStatusWaitTimeout));
#pragma unroll 1
                    for (int hf = 0; hf < 2 && ok; ++hf) {   // each half of the keys when its P is there
                        ok = mbar_wait_bounded(&p_full[j & 1][hf], ph, A.status, kStatusWaitTimeout);
                        if (!ok) break;
                        fence_after();
                        const uint32_t p = tmem + S::s0 + static_cast<uint32_t>((j & 1) * kN + hf * (kN / 2));
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int k = 0; k < kN / 32; ++k)
                                mma_ts(tmem + S::o, p + 16 * k + (part == 0 ? 8 : 0), b + hf * (kN / 2) * 128 / 16 + k * 128,
                                       idesc_f16(VD, true), hf > 0 || part > 0 || k > 0);
                    }
                    if (!ok) break;
                    commit(&o_full[j & 1]);
                    commit(&empty[v_place(j, n) % S::slots]);
                }
            }
            if (!ok) *abort_v = 1;
            if (*abort_v) {   // its products may still read the ring and TMEM
                commit(&drained[warp - kComputeWarps]);
                mbar_wait_bounded(&drained[warp - kComputeWarps], 0u, A.status, kStatusDrainTimeout);
            }
        }
        __syncwarp();
    } else {
        // ---- compute ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
        // ---- q as hi and lo halves into TMEM ----
        float sc;
        {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            named_barrier(3, kComputeWarps * 32);
            auto q4 = [&](int i) { return *reinterpret_cast<const float4*>(q_smem + row * HD * 4 + ((i ^ (row & 7)) << 4)); };
            float mx = 0.f;
#pragma unroll 8
            for (int i = 0; i < HD / 4; ++i) {
                const float4 v = q4(i);
                mx = fmax_nan(mx, fmax_nan(fmax_nan(fabsf(v.x), fabsf(v.y)), fmax_nan(fabsf(v.z), fabsf(v.w))));
            }
            // q = 2^e (hi + lo) with the largest |hi| in [2^14, 2^15)
            const bool fin = mx < INFINITY;
            int e = 0;
            if (fin && mx > 0.f) e = max(ilogbf(mx) - 14, -120);
            const float f1 = ldexpf(1.f, -(e / 2)), f2 = fin ? ldexpf(1.f, -(e - e / 2)) : 0.f;
            sc = fin ? ldexpf(1.f, e) : NAN;
#pragma unroll
            for (int c = 0; c < HQ / 32; ++c) {   // 32 dims of this thread's half: 16 columns
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float4 v = q4(half * HQ / 4 + c * 8 + i);
                    if (!fin) v = make_float4(0.f, 0.f, 0.f, 0.f);
                    split_away2(v.x * f1 * f2, v.y * f1 * f2, hi[2 * i], lo[2 * i]);
                    split_away2(v.z * f1 * f2, v.w * f1 * f2, hi[2 * i + 1], lo[2 * i + 1]);
                }
                st16(tl + S::q_hi + half * HQ / 2 + c * 16, hi);
                st16(tl + S::q_lo + half * HQ / 2 + c * 16, lo);
            }
            wait_st();
            fence_before();
            fence_proxy_async_smem();   // the slots are filled by the async proxy next
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_done);
        }
        if (A.cap2 == 0.f) sc *= A.scale2;
        const float slope2 = A.slopes ? A.slopes[h] * 1.44269504088896341f : 0.f;
        const bool plain = A.cap2 == 0.f && !A.slopes;
        float m = -INFINITY, l = 0.f;
        float acc[VD];
#pragma unroll
        for (int i = 0; i < VD; ++i) acc[i] = 0.f;
        bool ok = true;   // a wait that ran out is waited for no more; the loop goes on to its end
        const RowKeys keys = mask.row(pos);

        for (int j = half; j < n; j += 2) {   // `half`: the warpgroup, and its S buffer
            const int32_t j0 = kb.at(i0 + j) * kN;
            const bool whole = mask.all(p_lo, p_hi, j0, j0 + kN);
            if (!whole) {
                // values of V that are not finite and hidden from some row: added where they are seen, then
                // cleared (paged_attention.cu). Keys past the sequence are zeros, or what their page holds. Looked for
                // while S is being made.
                const int place = v_place(j, n);
                uint8_t* vb = ring_ptr + static_cast<size_t>(place % S::slots) * S::slot;
                ok = ok && mbar_warp_wait(&full[place % S::slots], static_cast<uint32_t>(place / S::slots) & 1u, A.status, kStatusWaitTimeout);
                const uint32_t me = threadIdx.x & 127;
                uint32_t odd = 0;
#pragma unroll 8
                for (uint32_t c = me * 16; c < kN * VD * 2; c += 128 * 16) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vb + c);
                    odd |= nonfinite_mark(w.x) | nonfinite_mark(w.y) | nonfinite_mark(w.z) | nonfinite_mark(w.w);
                }
                // (no warp of the group is a block ahead: the O that it has added last needed every warp's P)
                if (odd & kNonfinite) odd_block[half] = j;
                named_barrier(1 + half, 128);
                if (*reinterpret_cast<volatile int*>(&odd_block[half]) == j) {
                    for (int kr = 0; kr < kN; ++kr) {
                        if (!keys.sees(j0 + kr)) continue;
#pragma unroll
                        for (int d = 0; d < VD; d += 8) {
                            const uint4 w = *reinterpret_cast<const uint4*>(vb + (d >> 6) * (kN * 128) + kr * 128 + ((((d >> 3) & 7) ^ (kr & 7)) << 4));
                            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float x = half_bits_to_float(ws[i >> 1] >> (16 * (i & 1)));
                                if (!isfinite(x)) acc[d + i] += x;
                            }
                        }
                    }
                    named_barrier(1 + half, 128);
                    for (uint32_t c = me * 2; c < kN * VD * 2; c += 128 * 2) {
                        unsigned short& x = *reinterpret_cast<unsigned short*>(vb + c);
                        if ((x & 0x7C00u) == 0x7C00u) x = 0;
                    }
                    fence_proxy_async_smem();
                    named_barrier(1 + half, 128);
                }
            }
            ok = ok && mbar_warp_wait(&s_full[half], static_cast<uint32_t>(j >> 1) & 1u, A.status, kStatusWaitTimeout);
            fence_after();
            const uint32_t sb = tl + S::s0 + half * kN;
            float k = sc;   // s * k is the score in base 2
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (plain && whole) {
                float s[2][32];
                ld32(sb, s[0]);
                wait_ld<32>(s[0]);
#pragma unroll
                for (int c = 0; c < kN / 32; ++c) {
                    if (c + 1 < kN / 32) ld32(sb + (c + 1) * 32, s[(c + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], s[c & 1][i], s[c & 1][i + 1]);
                    if (c + 1 < kN / 32) wait_ld<32>(s[(c + 1) & 1]);
                }
            } else {
                // the scores themselves go back into TMEM
#pragma unroll 1
                for (int c = 0; c < kN / 32; ++c) {
                    float s[32];
                    ld32(sb + c * 32, s);
                    wait_ld<32>(s);
                    const int32_t jc = j0 + c * 32;
                    const float dist = static_cast<float>(pos - jc);   // exact below 2^24, else to 24 bits
                    if (A.cap2 != 0.f) {
                        // 2^87 takes any S but 0 (at least 2^-48, below 2^40) past where tanh is 1, and none to infinity
                        const float x1 = sc * A.cap_in > 0x1p87f ? 0x1p87f : sc * A.cap_in;
                        float far = 0.f;
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 x = ffma2(make_float2(s[i], s[i + 1]), make_float2(x1, x1), make_float2(0.f, 0.f));
                            s[i] = x.x;
                            s[i + 1] = x.y;
                            far = fmax3(far, fabsf(x.x), fabsf(x.y));
                        }
                        // which form a score takes goes by its own size alone, so that no other key or row changes it
                        if (__any_sync(0xffffffffu, far > 0.6f)) {
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 y = capped2_small(make_float2(s[i], s[i + 1]), A.cap2);
                                const float t0 = A.cap2 * tanhf(s[i]), t1 = A.cap2 * tanhf(s[i + 1]);
                                s[i] = fabsf(s[i]) > 0.6f ? t0 : y.x;
                                s[i + 1] = fabsf(s[i + 1]) > 0.6f ? t1 : y.y;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 y = capped2_small(make_float2(s[i], s[i + 1]), A.cap2);
                                s[i] = y.x;
                                s[i + 1] = y.y;
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[i] *= sc;
                    }
                    if (A.slopes) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[i] = fmaf(-slope2, fabsf(dist - static_cast<float>(i)), s[i]);
                    }
                    if (!whole) {
                        const uint32_t seen = (low_bits(keys.hi - jc) & ~low_bits(keys.lo - jc)) | low_bits(keys.prefix - jc);
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[i] = seen >> i & 1u ? s[i] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], s[i], s[i + 1]);
                    st32(sb + c * 32, s);
                }
                wait_st();
                k = 1.f;
            }
            float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * k;
            // k is NaN for a row that is not finite: so are its maximum, its P and its result
            mn = mn > m ? mn : (mn == mn ? m : mn);
            const float ms = mn == -INFINITY ? 0.f : mn;
            const float al = m == -INFINITY ? 0.f : ex2(m - ms);
            m = mn;
            // P = 2^(14 + s k - ms), at most 2^14 and a rounding. From |ms| = 2^24 on that rounding would be past what a half
            // holds, or all there is: scores then count in units that put ms back below 2^24, a float's precision still.
            // (Subtracting ms from such rows' scores in a pass of their own took a vote a block: 512 tokens at 2048 0.5 us more.)
            float unit = 1.f;
            if (fabsf(ms) >= 0x1p24f) unit = __uint_as_float((277u - (__float_as_uint(ms) >> 23 & 255u)) << 23);   // 2^(23 - floor(log2 |ms|))
            k *= unit;
            const float off = fmaf(-ms, unit, kPShift);
            float2 sum = make_float2(0.f, 0.f);
            float s[2][16];   // the next 16 columns are on their way while these are made into P
            ld16(sb, s[0]);
            wait_ld<16>(s[0]);
#pragma unroll
            for (int c = 0; c < kN / 16; ++c) {
                if (c + 1 < kN / 16) ld16(sb + (c + 1) * 16, s[(c + 1) & 1]);
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 x = ffma2(make_float2(s[c & 1][2 * i], s[c & 1][2 * i + 1]), make_float2(k, k), make_float2(off, off));
                    const float2 p = make_float2(ex2(x.x), ex2(x.y));
                    sum = fadd2(sum, p);
                    cut_half2(p, hi[i], lo[i]);
                }
                if (c + 1 < kN / 16) wait_ld<16>(s[(c + 1) & 1]);   // before P goes over columns that are being read
                st8(sb + c * 16, hi);
                st8(sb + c * 16 + 8, lo);
                if (c % (kN / 32) == kN / 32 - 1) {   // half of the keys
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[half][c / (kN / 32)]);
                }
            }
            l = fmaf(l, al, sum.x + sum.y);
            // acc = acc * al + O of this block
            ok = ok && mbar_warp_wait(&o_full[half], static_cast<uint32_t>(j >> 1) & 1u, A.status, kStatusWaitTimeout);
            fence_after();
            float o[2][32];
            ld32(tl + S::o, o[0]);
            wait_ld<32>(o[0]);
#pragma unroll
            for (int c = 0; c < VD / 32; ++c) {
                if (c + 1 < VD / 32) ld32(tl + S::o + (c + 1) * 32, o[(c + 1) & 1]);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 x = ffma2(make_float2(acc[c * 32 + i], acc[c * 32 + i + 1]), make_float2(al, al), make_float2(o[c & 1][i], o[c & 1][i + 1]));
                    acc[c * 32 + i] = x.x;
                    acc[c * 32 + i + 1] = x.y;
                }
                if (c + 1 < VD / 32) wait_ld<32>(o[(c + 1) & 1]);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free);
        }
        if (!ok) *abort_v = 1;

        // ---- the two warpgroups' results: each finishes half of the dims ----
        named_barrier(3, kComputeWarps * 32);   // every block is through: the ring is read and written no more
        s_ml[half][row] = make_float2(m, l);
        float* xch = reinterpret_cast<float*>(ring_ptr) + static_cast<size_t>(half * kM + row) * (HH + 2);
#pragma unroll
        for (int i = 0; i < HH; i += 2)
            *reinterpret_cast<float2*>(xch + i) = half == 0 ? make_float2(acc[HH + i], acc[HH + i + 1]) : make_float2(acc[i], acc[i + 1]);
        named_barrier(3, kComputeWarps * 32);
        const float2 other = s_ml[half ^ 1][row];
        const float* theirs = reinterpret_cast<const float*>(ring_ptr) + static_cast<size_t>((half ^ 1) * kM + row) * (HH + 2);
        const float M = fmaxf(m, other.x);
        // a side that saw nothing adds zeros, or the NaN of a row that is not finite
        const float fa = m == -INFINITY ? 1.f : ex2(m - M), fb = other.x == -INFINITY ? 1.f : ex2(other.x - M);
        float res[HH];
#pragma unroll
        for (int i = 0; i < HH; i += 2) {
            const float2 v = *reinterpret_cast<const float2*>(theirs + i);
            res[i] = fmaf(v.x, fb, (half == 0 ? acc[i] : acc[HH + i]) * fa);
            res[i + 1] = fmaf(v.y, fb, (half == 0 ? acc[i + 1] : acc[HH + i + 1]) * fa);
        }
        m = M;
        l = fmaf(other.y, fb, l * fa);
        float* part = A.part + ((static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * A.n_split + split) * S::part;
        const float inv = n_parts > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;   // nothing seen: zeros
        // through shared memory, so that whole rows are written
        uint8_t* o_smem = ring_ptr + ((2 * kM * (HH + 2) * 4 + 1023) & ~1023);
#pragma unroll
        for (int i = 0; i < HH / 4; ++i)
            *reinterpret_cast<float4*>(o_smem + row * VD * 4 + (((half * (HH / 4) + i) ^ (row & 7)) << 4)) =
                make_float4(res[4 * i] * inv, res[4 * i + 1] * inv, res[4 * i + 2] * inv, res[4 * i + 3] * inv);
        named_barrier(3, kComputeWarps * 32);
        if (!*abort_v) {
            constexpr int PIECES = VD / 4;
#pragma unroll 4
            for (int i = 0; i < kM * PIECES / (kComputeWarps * 32); ++i) {
                const int p = i * kComputeWarps * 32 + threadIdx.x, orow = p / PIECES, c = p % PIECES, rr = r0 + orow;
                if (rr >= n_rows) break;   // rows rise with i
                const float4 v = *reinterpret_cast<const float4*>(o_smem + orow * VD * 4 + ((c ^ (orow & 7)) << 4));
                const int ot = A.group_div.div(rr);
                float* dst = n_parts > 1 ? part + orow * VD
                                         : A.out + static_cast<int64_t>(sv.q0 + ot) * A.ldo + static_cast<int64_t>(kvh * A.group + rr - ot * A.group) * HD + v0;
                *reinterpret_cast<float4*>(dst + c * 4) = v;
            }
        }
        if (n_parts > 1) {
            if (half == 0) *reinterpret_cast<float2*>(part + kM * VD + row * 2) = make_float2(m, l);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Adds the parts of a tile that was split over the keys, in their order: a warp a
// row, eight rows a block.
template <int HD>
__global__ void __launch_bounds__(256)
combine_kernel(const __grid_constant__ AttnArgs A) {
    using S = TcShape<HD>;
    constexpr int V = S::vd / 32, AHEAD = 8;   // values of a lane; parts whose loads are under way
    const int lane = threadIdx.x & 31, kvh = blockIdx.y / S::parts, v0 = (blockIdx.y % S::parts) * S::vd;
    int seq, tile;
    grid_dep_wait();
    grid_dep_launch();
    if (!locate_tile(A.b, A.group, kM, A.per_seq, static_cast<int>(blockIdx.x), seq, tile)) return;
    const SeqView sv = seq_view(A.c, A.b, seq);
    const int n_rows = sv.n_new * A.group;
    const int r0 = ((n_rows + kM - 1) / kM - 1 - tile) * kM, base = sv.len - sv.n_new;
    const int row = blockIdx.z * 8 + (threadIdx.x >> 5), r = r0 + row;
    if (!sv.ok || tile * kM >= n_rows || r >= n_rows) return;
    Mask mask{sv.len, A.window, 0};
    if (A.prefix) mask.prefix = max(0, min(A.prefix[seq], sv.len));
    const KeyBlocks kb = key_blocks(mask, base + A.group_div.div(r0), base + A.group_div.div(min(r0 + kM - 1, n_rows - 1)), S::keys);
    const int n = max(1, (kb.n + A.blocks_per_split - 1) / A.blocks_per_split);
    if (n == 1) return;
    const float* parts = A.part + (static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * A.n_split * S::part;
    const float* ml = parts + kM * S::vd + row * 2;
    const float* acc = parts + static_cast<int64_t>(row) * S::vd + lane * V;
    float M = -INFINITY;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(ml + i * S::part));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float L = 0.f, O[V];
#pragma unroll
    for (int c = 0; c < V; ++c) O[c] = 0.f;
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
        float2 p[AHEAD];
        float v[AHEAD][V];
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) {
            if (i0 + x >= n) break;
            p[x] = __ldcg(reinterpret_cast<const float2*>(ml + (i0 + x) * S::part));
            if constexpr (V == 2) *reinterpret_cast<float2*>(v[x]) = __ldcg(reinterpret_cast<const float2*>(acc + (i0 + x) * S::part));
            else *reinterpret_cast<float4*>(v[x]) = __ldcg(reinterpret_cast<const float4*>(acc + (i0 + x) * S::part));
        }
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) {
            if (i0 + x >= n) break;
            // a part that saw nothing adds zeros, or the NaN of a row that is not finite
            const float f = p[x].x == -INFINITY ? 1.f : ex2(p[x].x - M);
            L = fmaf(p[x].y, f, L);
#pragma unroll
            for (int c = 0; c < V; ++c) O[c] = fmaf(v[x][c], f, O[c]);
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int t = A.group_div.div(r);
    float* o = A.out + static_cast<int64_t>(sv.q0 + t) * A.ldo + static_cast<int64_t>(kvh * A.group + r - t * A.group) * HD + v0 + lane * V;
#pragma unroll
    for (int c = 0; c < V; c += 2) *reinterpret_cast<float2*>(o + c) = make_float2(O[c] * inv, O[c + 1] * inv);
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// One layer's pool as [page][place][head][dim]; the box: `box` places of one head, 64 dims (128 bytes, the swizzle's span).
bool encode_pool(CUtensorMap* map, const void* pool, const PagedLayer& c, int box) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.n_kv), static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.n_pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c.head_dim) * 2, static_cast<cuuint64_t>(c.n_kv) * c.head_dim * 2, static_cast<cuuint64_t>(c.page_stride) * 2};
    const cuuint32_t boxes[4] = {64, 1, static_cast<cuuint32_t>(box), 1}, one[4] = {1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pool), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool TMA>
cudaError_t launch(const AttnArgs& a, int tiles, int box, cudaStream_t s) {
    static bool set[64] = {};   // per instance and device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!set[dev]) {
        e = cudaFuncSetAttribute(chunk_kernel<HD, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(TcShape<HD>::smem));
        if (e != cudaSuccess) return e;
        set[dev] = true;
    }
    CUtensorMap k{}, v{};
    if (TMA && (!encode_pool(&k, a.c.k, a.c, box) || !encode_pool(&v, a.c.v, a.c, box))) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(a.c.n_kv * TcShape<HD>::parts), static_cast<unsigned>(a.n_split));
    e = launch_dep(chunk_kernel<HD, TMA>, grid, kThreads, TcShape<HD>::smem, s, a, k, v, box);
    if (e != cudaSuccess || a.n_split == 1) return e;
    const unsigned eights = static_cast<unsigned>((std::min(kM, a.b.max_new * a.group) + 7) / 8);
    return launch_dep(combine_kernel<HD>, dim3(grid.x, grid.y, eights), 256, 0, s, a);
}

}  // namespace

// A box of the tiled copies lies in one page and one block of keys, and its rows
// are whole groups of the swizzle; a tensor map's strides are below 2^40 bytes,
// each a multiple of the one before it.
bool paged_attention_tiled(const PagedLayer& c) {
    return std::gcd(c.page_size, tc_keys(c.head_dim)) >= 8 && c.page_stride < (int64_t(1) << 39) &&
           c.page_stride % (static_cast<int64_t>(c.n_kv) * c.head_dim) == 0;
}

cudaError_t paged_attention_tc(const AttnArgs& a, int tiles, cudaStream_t s) {
    const int box = std::gcd(a.c.page_size, tc_keys(a.c.head_dim));
    const bool tma = paged_attention_tiled(a.c);
    switch (a.c.head_dim) {
        case 64: return tma ? launch<64, true>(a, tiles, box, s) : launch<64, false>(a, tiles, box, s);
        case 128: return tma ? launch<128, true>(a, tiles, box, s) : launch<128, false>(a, tiles, box, s);
        default: return tma ? launch<256, true>(a, tiles, box, s) : cudaErrorInvalidValue;   // the caller asks first
    }
}

}  // namespace hesa_cuda
