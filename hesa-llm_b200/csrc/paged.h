// paged.h -- the paged KV cache as its kernels see it, and what they share:
// finding a block's rows in a ragged batch, the mask, and the checks of the
// lengths and tables that only the device knows.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/hesa_cuda.h"
#include "hesa_common.cuh"

namespace hesa_cuda {

// x / d for 0 <= x < 2^31 as the high word of x * mul, shifted: mul =
// ceil(2^(31 + b) / d), b = ceil(log2(d)); its excess of less than d over
// 2^(31 + b) adds less than 1 / d to the quotient.
struct FastDiv {
    uint32_t mul;
    int32_t shift;   // b - 1; -1: d = 1
    int32_t d;
    FastDiv() = default;
    __host__ explicit FastDiv(int32_t by) : mul(0), shift(-1), d(by) {
        int b = 0;
        while ((int64_t(1) << b) < by) ++b;
        if (b > 0) mul = static_cast<uint32_t>(((uint64_t(1) << (31 + b)) + by - 1) / by);
        shift = b - 1;
    }
    __device__ __forceinline__ int32_t div(int32_t x) const {
        return shift < 0 ? x : static_cast<int32_t>(__umulhi(static_cast<uint32_t>(x), mul) >> shift);
    }
};

// One layer of the cache. Element e of kv head h of the token in slot s of
// page p lies at p * page_stride + (s * n_kv + h) * head_dim + e.
struct PagedLayer {
    const __half* k;
    const __half* v;
    int64_t page_stride;
    int32_t n_pages, page_size, n_kv, head_dim;
    const int32_t* table;     // [n_slots][max_pages]
    const int32_t* seq_len;   // [n_slots]
    int32_t n_slots, max_pages;
    FastDiv page_div;         // by page_size
};

struct BatchView {
    const int32_t* slots;     // [n_seq] or null: sequence i is in slot i
    const int32_t* q_start;   // [n_seq + 1]
    int32_t n_seq, n_tokens, max_new, max_len;
};

// A sequence of the batch: rows [q0, q0 + n_new) of q, the last n_new of the
// slot's len tokens. ok is false where the device's numbers contradict the
// bounds that the host gave; such a sequence is skipped and status 3 recorded.
struct SeqView {
    int32_t q0, n_new, len, slot;
    bool ok;
};

__device__ __forceinline__ SeqView seq_view(const PagedLayer& c, const BatchView& b, int s) {
    SeqView r;
    const int32_t a = b.q_start[s], e = b.q_start[s + 1];
    r.slot = b.slots ? b.slots[s] : s;
    r.q0 = a;
    r.n_new = e - a;
    r.len = 0;
    r.ok = a >= 0 && e >= a && e <= b.n_tokens && e - a <= b.max_new && r.slot >= 0 && r.slot < c.n_slots;
    if (r.ok) {
        r.len = c.seq_len[r.slot];
        r.ok = r.len >= 0 && r.len <= b.max_len && r.len <= static_cast<int64_t>(c.max_pages) * c.page_size;
    }
    if (!r.ok) r.n_new = r.len = 0;
    return r;
}

// Rows of a batch in tiles of R rows, a row being one query head of a group of
// g that share a kv head: sequence s has the n_new * g rows t * g + h. Either
// every sequence has the same number of tiles (per_seq > 0: the bound of the
// longest one), or sequence s starts at tile floor(q_start[s] * g / R) + s:
// these starts rise by at least ceil(n_new * g / R) from one sequence to the
// next, since floor(a + b) - floor(a) + 1 >= ceil(b), so no sequence needs a
// prefix sum to find its tiles and at most one tile a sequence stays empty.
__host__ __device__ inline int64_t tile_bound(int64_t n_tokens, int64_t n_seq, int g, int r) {
    return n_tokens * g / r + n_seq;
}

// Tile idx of the launch: tile `tile` (>= 0, and possibly behind its rows) of
// sequence seq; false where it is no sequence's.
__host__ __device__ __forceinline__ bool locate_tile(const BatchView& b, int g, int r, int per_seq, int idx, int& seq, int& tile) {
    if (per_seq > 0) {
        seq = idx / per_seq;
        tile = idx - seq * per_seq;
        return true;
    }
    int lo = 0, hi = b.n_seq - 1;   // the last s with start(s) <= idx, or 0; in range whatever q_start holds
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        const int64_t at = static_cast<int64_t>(b.q_start[mid]) * g / r + mid;
        if (at <= idx) lo = mid;
        else hi = mid - 1;
    }
    seq = lo;
    const int64_t behind = idx - (static_cast<int64_t>(b.q_start[lo]) * g / r + lo);
    tile = behind < 0 ? 0 : behind < idx ? static_cast<int>(behind) : idx;   // more than idx: q_start[lo] < 0, which seq_view refuses
    return behind >= 0;
}

// Key j is seen from position p: j < len and ((j <= p and (no window, or
// j > p - window)) or j < prefix).
struct RowKeys {
    int32_t lo, hi, prefix;   // [lo, hi) and [0, prefix)
    __device__ __forceinline__ bool sees(int32_t j) const {
        return static_cast<uint32_t>(j - lo) < static_cast<uint32_t>(hi - lo) || j < prefix;
    }
};

struct Mask {
    int32_t len, window, prefix;   // prefix <= len
    __device__ __forceinline__ RowKeys row(int32_t p) const {
        const int32_t lo = window > 0 && p + 1 > window ? p + 1 - window : 0;
        const int32_t hi = p + 1 < len ? p + 1 : len;
        return RowKeys{lo, hi > lo ? hi : lo, prefix};
    }
    // every key of [j0, j1) is seen from every position of [p_lo, p_hi]
    __device__ __forceinline__ bool all(int32_t p_lo, int32_t p_hi, int32_t j0, int32_t j1) const {
        return j1 <= len && ((j1 - 1 <= p_lo && (window == 0 || j0 > p_hi - window)) || j1 <= prefix);
    }
};

// The keys that positions [p_lo, p_hi] see, as blocks of B keys: blocks
// [0, n_pre) of the prefix, then blocks from b_win on, n in all. Block i is
// block at(i) of the sequence.
struct KeyBlocks {
    int32_t n_pre, b_win, n;
    __device__ __forceinline__ int32_t at(int32_t i) const { return i < n_pre ? i : i - n_pre + b_win; }
};

__device__ __forceinline__ KeyBlocks key_blocks(const Mask& m, int32_t p_lo, int32_t p_hi, int block) {
    KeyBlocks r;
    int32_t hi = p_hi + 1;
    if (hi > m.len) hi = m.len;
    if (hi < 0) hi = 0;
    const int32_t lo = m.window > 0 && p_lo + 1 > m.window ? p_lo + 1 - m.window : 0;
    r.n_pre = (m.prefix + block - 1) / block;
    r.b_win = lo / block;
    if (r.b_win < r.n_pre) r.b_win = r.n_pre;
    const int32_t end = (hi + block - 1) / block;
    r.n = r.n_pre + (end > r.b_win ? end - r.b_win : 0);
    return r;
}

// What the attention kernels take.
struct AttnArgs {
    PagedLayer c;
    BatchView b;
    const float* q;
    int64_t ldq;
    float* out;
    int64_t ldo;
    int32_t n_head, group;         // group = n_head / n_kv
    FastDiv group_div;             // by group
    float scale2;                  // scale * log2(e): scores are kept in base 2
    float cap2, cap_in;            // softcap * log2(e) and scale / softcap; 0: not capped
    int32_t window;
    const float* slopes;           // [n_head] or null
    const int32_t* prefix;         // [n_seq] or null
    int* status;
    float* part;                   // m, l, acc of rows that are added up later
    int32_t per_seq;               // tiles of every sequence, 0: by q_start
    int32_t blocks_per_split;      // chunk_kernel: keys of a split
    int32_t n_split;               // chunk_kernel: splits; rows_kernel: tiles of this launch
    int32_t tile0;                 // rows_kernel: the first of them
};

// The largest P is 2^kPShift before its split into fp16 halves: the low half of
// a P down to 2^-28 of the row's largest is then still a normal or nearly
// normal fp16 number, and the factor cancels in P V / sum P.
constexpr float kPShift = 14.0f;

// Two fp16 values: a bit of kNonfinite is set for each whose exponent is all ones
// (one more in the exponent carries into the sign's place).
constexpr uint32_t kNonfinite = 0x80008000u;
__device__ __forceinline__ uint32_t nonfinite_mark(uint32_t w) { return (w & 0x7FFF7FFFu) + 0x04000400u; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The score in base 2 of a dot product (already in q's own scale).
__device__ __forceinline__ float capped(float dot, float cap2, float cap_in) { return cap2 * tanhf(dot * cap_in); }

// x = hi + lo to 22 bits, |x| < 65504
__device__ __forceinline__ void split_half2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// x = hi + lo to 21 bits, |x| < 2^15, for q: hi is x taken away from zero to 11
// bits, so that lo is zero or has the other sign. The score of an infinite k is then
// inf - inf or 0 inf: NaN in every row that sees it, as for a k that is NaN,
// whatever its sign and a cap on scores. (With hi to nearest, one bit more, it was
// -inf, which is a weight of 0, or NaN, as q's low bits had it; looking for -inf in
// the blocks' scores took 2 to 4% of a chunk's time.)
__device__ __forceinline__ void split_away2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const float h0 = __uint_as_float((__float_as_uint(x0) + 0x1FFFu) & 0xFFFFE000u), h1 = __uint_as_float((__float_as_uint(x1) + 0x1FFFu) & 0xFFFFE000u);
    const __half2 h = __floats2half2_rn(h0, h1);   // exact from 2^-14 on; below, lo is rounded to zero
    const __half2 l = __floats2half2_rn(x0 - h0, x1 - h1);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Launch with programmatic stream serialization: the grid may be set up while
// the previous kernel on the stream finishes. Every block of such a kernel calls
// grid_dep_wait, also one with nothing to do (the grid must not end before the one
// it follows), before it writes anything, and reads what earlier kernels wrote with
// plain loads (no read-only cache: the grid may be older than the data).
// cluster: blocks of a cluster, 1 for none.
template <typename... P, typename... T>
cudaError_t launch_clusters(void (*kernel)(P...), int cluster, dim3 grid, int threads, size_t smem, cudaStream_t s, T... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <typename... P, typename... T>
cudaError_t launch_dep(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, T... args) {
    return launch_clusters(kernel, 1, grid, threads, smem, s, args...);
}

// The host's checks of a cache and a batch (paged_attention.cu): 0, or an error
// code with its message recorded.
int check_paged_kv(const hesa_cuda_paged_kv* kv);
int check_batch(const hesa_cuda_paged_kv* kv, int32_t layer, const hesa_cuda_token_batch* b, int64_t n_head);
// The checks of strides, tables and counts that caches of both kinds share; strides count units of `unit` values.
struct PagedShape {
    const int32_t *table, *seq_len;
    int64_t page_stride, layer_stride;
    int32_t unit, n_layer, n_pages, page_size, n_kv_head, head_dim, n_slots, max_pages;
};
int check_paged_shape(const PagedShape& c);

// ---- the cache in 4 bits (paged_attention4.cu, kv4_cache.cu) ----
constexpr int kGroup = 32;          // values of a group: 16 bytes of codes, one scale
constexpr float kMostScale = 2720.f;   // 24 of it is an fp16 number

// One layer: group (s * n_kv + h) * (head_dim / 32) + g of page p lies p * page_stride groups behind the pools' starts.
struct Pools4 {
    const uint4* k;
    const uint4* v;
    const __half* ks;
    const __half* vs;
};
int check_paged_kv4(const hesa_cuda_paged_kv4* kv);
int check_batch4(const hesa_cuda_paged_kv4* kv, int32_t layer, const hesa_cuda_token_batch* b, int64_t n_head);
// The tables and the shape, strides in groups; k and v are null.
PagedLayer layer_of4(const hesa_cuda_paged_kv4* kv);
Pools4 pools_of(const hesa_cuda_paged_kv4* kv, int32_t layer);

// Eight codes of a word as four pairs of values, (e, e + 4) for e = 0 .. 3.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}
__device__ __forceinline__ uint32_t bits_of(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 half2_bits(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
// A code put into the low bits of the fp16 number 1024, or four bits higher into 64,
// is that number plus the code; the sum with -1032 (-72) and the product by a scale
// of 8 bits are exact. One shift for the four pairs.
__device__ __forceinline__ void code_pairs(uint32_t w, __half2 d, uint32_t (&p)[4]) {
    const __half2 low = half2_bits(0xE408E408u), high = half2_bits(0xD480D480u);
    const uint32_t x = w >> 8;
    p[0] = bits_of(__hmul2(__hadd2(half2_bits(and_or(w, 0x000F000Fu, 0x64006400u)), low), d));
    p[1] = bits_of(__hmul2(__hadd2(half2_bits(and_or(w, 0x00F000F0u, 0x54005400u)), high), d));
    p[2] = bits_of(__hmul2(__hadd2(half2_bits(and_or(x, 0x000F000Fu, 0x64006400u)), low), d));
    p[3] = bits_of(__hmul2(__hadd2(half2_bits(and_or(x, 0x00F000F0u, 0x54005400u)), high), d));
}
// Put behind the leading bit of an fp16 number it makes 16 + code, and (16 + code) d
// - 24 d is one fma, exact because 24 d is an fp16 number too (d has 8 bits). A shift
// for each pair, but half the fp16 instructions. m = -24 d.
__device__ __forceinline__ void code_pairs_fma(uint32_t w, __half2 d, __half2 m, uint32_t (&p)[4]) {
    p[0] = bits_of(__hfma2(half2_bits(and_or(w << 6, 0x03C003C0u, 0x4C004C00u)), d, m));
    p[1] = bits_of(__hfma2(half2_bits(and_or(w << 2, 0x03C003C0u, 0x4C004C00u)), d, m));
    p[2] = bits_of(__hfma2(half2_bits(and_or(w >> 2, 0x03C003C0u, 0x4C004C00u)), d, m));
    p[3] = bits_of(__hfma2(half2_bits(and_or(w >> 6, 0x03C003C0u, 0x4C004C00u)), d, m));
}

PagedLayer layer_of(const hesa_cuda_paged_kv* kv, int32_t layer);
BatchView view_of(const hesa_cuda_token_batch* b);
// The checks of attention's other arguments, and those that do not depend on the cache's kind in *args: b, q, out, the
// options and part.
int attention_args(int32_t head_dim, int32_t n_kv_head, const hesa_cuda_token_batch* batch, const float* q, int64_t ldq, float* out, int64_t ldo,
                   int64_t n_head, const hesa_cuda_attn_options* options, void* workspace, AttnArgs* args);

}  // namespace hesa_cuda
