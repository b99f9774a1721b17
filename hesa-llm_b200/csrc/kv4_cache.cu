// kv4_cache.cu -- writing new tokens into the pages of a cache in 4 bits, and
// reading them back.
//
//   m = the value of largest magnitude of 32 dims, d = round(m / -8) to 8
//   significant bits, code = floor(x / d + 8.5) in 0 .. 15, value = d (code - 8)
//
// The 8 bits of a scale (a step of the code is off by at most 1 / 512 of itself,
// and the codes are made for the scale as it is stored) and the 4 of a code make
// 11: every value is an fp16 number exactly, so attention can take values as fp16
// without another rounding. Scales below 2^-17 are multiples of 2^-24, fp16's
// last step, for the same reason.
//
// Both kernels are bound by HBM: each value is read once and written once. 5296 tokens
// of 32 heads: written with rope in 65 us (371 MB, 5.7 TB/s), read in 38 us (198 MB, 5.3
// TB/s); 32 tokens, 64 heads on 8: about 3 us each, their launches.
#include "paged.h"
#include "abi_errors.h"
#include "qmatvec.h"
#include "trace.h"

#include <algorithm>

namespace hesa_cuda {
namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The place of a row's token: group number of its first head's first group, or -1
// (with a status recorded where the tables are not sound), and its position.
struct Place {
    int64_t group;
    int32_t pos;
    bool row;      // the row is a sequence's
};

__device__ __forceinline__ Place find_place(const PagedLayer& c, const BatchView& b, int row, int* status) {
    // the last sequence that starts at or before this row and is not empty there
    int lo = 0, hi = b.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.q_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    const SeqView s = seq_view(c, b, lo);
    Place p{-1, 0, false};
    if (!s.ok) {
        record_status(status, kStatusBadPosition);
        return p;
    }
    const int t = row - s.q0;
    if (t < 0 || t >= s.n_new) return p;   // a row behind the last sequence
    p.row = true;
    p.pos = s.len - s.n_new + t;
    const int pi = p.pos >= 0 ? c.page_div.div(p.pos) : 0;
    const int page = p.pos >= 0 ? c.table[static_cast<int64_t>(s.slot) * c.max_pages + pi] : -1;
    if (page < 0 || page >= c.n_pages) {
        record_status(status, kStatusBadPosition);
        return p;
    }
    p.group = static_cast<int64_t>(page) * c.page_stride + static_cast<int64_t>(p.pos - pi * c.page_size) * c.n_kv * (c.head_dim / kGroup);
    return p;
}

// Eight values of a group whose other 24 the quad's other threads have (in order):
// the group's scale, and this thread's word of codes.
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], unsigned quad, float& scale) {
    // the largest and the smallest value: the one of larger magnitude makes the scale; NaN stays
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        hi = fmax_nan(hi, x[i]);
        lo = fmin_nan(lo, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        hi = fmax_nan(hi, __shfl_xor_sync(quad, hi, o));
        lo = fmin_nan(lo, __shfl_xor_sync(quad, lo, o));
    }
    float m = hi > -lo ? hi : lo;
    if (hi == -lo) {   // as large on either side: the first of them
        const int lane = threadIdx.x & 31;
        unsigned first = 8;
#pragma unroll
        for (int i = 7; i >= 0; --i) first = fabsf(x[i]) == hi ? i : first;
        const unsigned have = __ballot_sync(quad, first < 8) & quad;
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine = static_cast<int>(first) == i ? x[i] : mine;
        m = __shfl_sync(quad, mine, have ? __ffs(have) - 1 : lane);
    }
    const float s = m * -0.125f;
    const uint32_t u = __float_as_uint(s);
    float d = __uint_as_float((u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u);   // 8 bits, ties to even
    if (fabsf(s) < 0x1p-17f) d = rintf(s * 0x1p24f) * 0x1p-24f;
    if (!(hi - lo < INFINITY) || !(fabsf(d) <= kMostScale)) d = NAN;   // hi - lo: not finite where a value is not, or the scale is too large
    scale = d;
    if (!(fabsf(d) > 0.f)) return 0x88888888u;
    const float id = __frcp_rn(d);
    // a number of 0 .. 15.9 rounded down behind 2^23 has its whole part in the low bits
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = fminf(fmaxf(__fadd_rn(__fmul_rn(x[i], id), 8.5f), 0.f), 15.f);
        w += __float_as_uint(__fadd_rd(c, 0x1p23f)) << (4 * i);
    }
    return w - (0x4B000000u * 0x11111111u);
}

// A unit is 16 values of one head of one token: 8 of the first half of the head
// and the 8 that they are rotated with; four threads side by side have two whole
// groups. A block takes one token's units (grid.y covers long rows); q, then k,
// then v. 5296 tokens of 32 heads: 65 us (371 MB, 5.7 TB/s); with four and four values a
// thread, sixteen-byte accesses side by side but more shuffles a value, 71.
__global__ void __launch_bounds__(256)
rope_kv4_kernel(const PagedLayer c, const Pools4 pools, const BatchView b, float* q, int64_t ldq, const float* k, int64_t ldk,
                const float* v, int64_t ldv, int n_head, const float* table, int table_rows, int* status) {
    grid_dep_wait();
    grid_dep_launch();
    const int row = blockIdx.x;
    __shared__ Place s_at;
    if (threadIdx.x == 0) s_at = find_place(c, b, row, status);
    __syncthreads();
    const Place at = s_at;
    if (at.group < 0) return;
    if (table && at.pos >= table_rows) {
        if (threadIdx.x == 0) record_status(status, kStatusBadPosition);
        return;
    }
    const int hd = c.head_dim, per = hd / 16, per_bits = __ffs(per) - 1, half = hd / 2, groups = hd / kGroup;   // head_dim is a power of two
    const int n_rot = n_head + c.n_kv;
    const int units = (n_rot + c.n_kv) * per;   // a multiple of 4, as `per` is: a quad works or none of its threads does
    const float* cs = table ? table + static_cast<int64_t>(at.pos) * hd : nullptr;
    const unsigned quad = 0xFu << (threadIdx.x & 28);
    for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < units; u += gridDim.y * blockDim.x) {
        const int h = u >> per_bits, d = (u - (h << per_bits)) * 8;
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
            const bool is_k = h < n_rot;
            const int64_t g = at.group + static_cast<int64_t>(is_k ? h - n_head : h - n_rot) * groups;
            uint32_t* codes = reinterpret_cast<uint32_t*>(const_cast<uint4*>(is_k ? pools.k : pools.v) + g);
            __half* scales = const_cast<__half*>(is_k ? pools.ks : pools.vs) + g;
            float sx, sy;
            const uint32_t wx = quantize8(x, quad, sx), wy = quantize8(y, quad, sy);
            codes[d / 8] = wx;
            codes[(half + d) / 8] = wy;
            if ((threadIdx.x & 3) == 0) {
                scales[d / kGroup] = __float2half_rn(sx);   // exact
                scales[(half + d) / kGroup] = __float2half_rn(sy);
            }
        }
    }
}

// A block takes `rows` tokens' K and V, kReadChunk quads of dims at a time, and reads
// the codes of the next chunk before it writes the values of one: writing, which is
// nearly all of the traffic, does not wait for reads. (5296 tokens of 32 heads: 45 us
// without that, 26 without reading.) A thread's quad is half a word of codes, so that
// a warp writes 512 bytes in a row; with a word a thread, two stores 32 bytes apart, 55.
constexpr int kReadQuads = 8;                      // of a thread and chunk
constexpr int kReadChunk = kReadQuads * 256;
constexpr int kMostRows = 8;

__global__ void __launch_bounds__(256)
kv4_read_kernel(const PagedLayer c, const Pools4 pools, const BatchView b, float* k, int64_t ldk, float* v, int64_t ldv, int rows, int* status) {
    __shared__ Place s_at[kMostRows];
    grid_dep_wait();
    grid_dep_launch();
    const int row0 = blockIdx.x * rows;
    rows = min(rows, b.n_tokens - row0);
    if (static_cast<int>(threadIdx.x) < rows) s_at[threadIdx.x] = find_place(c, b, row0 + threadIdx.x, status);
    __syncthreads();
    const int quads = c.n_kv * c.head_dim / 4, chunks = (quads + kReadChunk - 1) / kReadChunk;   // of K, and as many of V
    uint32_t code[kReadQuads];
    __half d[kReadQuads];
    // chunk ch: of K where it is even, of V where it is odd; the grid's y shares them out
    auto load = [&](int r, int ch) {
        const int64_t group = s_at[r].group;
        const uint32_t* from = reinterpret_cast<const uint32_t*>((ch & 1 ? pools.v : pools.k) + group);
        const __half* scales = (ch & 1 ? pools.vs : pools.ks) + group;
        const bool some = group >= 0 && (ch & 1 ? v : k) != nullptr;
#pragma unroll
        for (int x = 0; x < kReadQuads; ++x) {
            const int u = (ch >> 1) * kReadChunk + x * 256 + threadIdx.x;
            code[x] = 0x88888888u;
            d[x] = __float2half_rn(0.f);
            if (some && u < quads) {
                code[x] = __ldcs(from + u / 2);
                d[x] = scales[u / 8];
            }
        }
    };
    int r = 0, ch = blockIdx.y;
    if (rows > 0 && ch < 2 * chunks) load(r, ch);
    while (r < rows && ch < 2 * chunks) {
        uint32_t now[kReadQuads];
        __half scale[kReadQuads];
#pragma unroll
        for (int x = 0; x < kReadQuads; ++x) {
            now[x] = code[x];
            scale[x] = d[x];
        }
        const int64_t row = row0 + r;
        const int at = ch;
        float* o = ch & 1 ? v : k;
        const bool some = s_at[r].row && o;
        ch += gridDim.y;
        if (ch >= 2 * chunks) {
            ch = blockIdx.y;
            ++r;
        }
        if (r < rows) load(r, ch);
        if (!some) continue;
        o += row * (at & 1 ? ldv : ldk);
#pragma unroll
        for (int x = 0; x < kReadQuads; ++x) {
            const int u = (at >> 1) * kReadChunk + x * 256 + threadIdx.x;
            if (u >= quads) break;
            // the quad's two bytes apart: codes 0 and 2 in the low nibbles, 1 and 3 in the next ones
            const uint32_t bytes = prmt(now[x], 0u, threadIdx.x & 1 ? 0x4342u : 0x4140u);
            const __half2 sc = __half2half2(scale[x]);
            const float2 even = __half22float2(__hmul2(__hadd2(half2_bits(and_or(bytes, 0x000F000Fu, 0x64006400u)), half2_bits(0xE408E408u)), sc));
            const float2 odd = __half22float2(__hmul2(__hadd2(half2_bits(and_or(bytes, 0x00F000F0u, 0x54005400u)), half2_bits(0xD480D480u)), sc));
            __stcs(reinterpret_cast<float4*>(o) + u, make_float4(even.x, odd.x, even.y, odd.y));   // exact, see code_pairs
        }
    }
}

}  // namespace

int check_paged_kv4(const hesa_cuda_paged_kv4* kv) {
    if (!kv || !kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !kv->table || !kv->seq_len)
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    const int rc = check_paged_shape({kv->table, kv->seq_len, kv->page_stride, kv->layer_stride, kGroup, kv->n_layer, kv->n_pages, kv->page_size, kv->n_kv_head,
                                      kv->head_dim, kv->n_slots, kv->max_pages});
    if (rc != HESA_CUDA_OK) return rc;
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->k_scale, 16) || !aligned(kv->v_scale, 16))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "the page pools must be 16-byte aligned");
    return HESA_CUDA_OK;
}

PagedLayer layer_of4(const hesa_cuda_paged_kv4* kv) {
    PagedLayer c{};
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

Pools4 pools_of(const hesa_cuda_paged_kv4* kv, int32_t layer) {
    const int64_t at = layer * kv->layer_stride;
    return Pools4{static_cast<const uint4*>(kv->k) + at, static_cast<const uint4*>(kv->v) + at, static_cast<const __half*>(kv->k_scale) + at,
                  static_cast<const __half*>(kv->v_scale) + at};
}

}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

int hesa_cuda_rope_kv4_paged(const hesa_cuda_paged_kv4* kv, int32_t layer, const hesa_cuda_token_batch* batch, float* q, int64_t ldq,
                             const float* k, int64_t ldk, const float* v, int64_t ldv, int64_t n_head, const float* rope_table,
                             int32_t rope_rows, void* stream) {
    HESA_TRACE("hesa_cuda_rope_kv4_paged");
    int rc = check_paged_kv4(kv);
    if (rc == HESA_CUDA_OK) rc = check_batch4(kv, layer, batch, n_head);
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
        e = launch_dep(rope_kv4_kernel, dim3(static_cast<unsigned>(batch->n_tokens), static_cast<unsigned>(y)), 256, 0, static_cast<cudaStream_t>(stream),
                       layer_of4(kv), pools_of(kv, layer), view_of(batch), q, ldq, k, ldk, v, ldv, static_cast<int>(n_head), rope_table, rope_rows, status);
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "rope_kv4_paged kernel");
}

int hesa_cuda_kv4_read(const hesa_cuda_paged_kv4* kv, int32_t layer, const hesa_cuda_token_batch* batch, float* k, int64_t ldk, float* v,
                       int64_t ldv, void* stream) {
    HESA_TRACE("hesa_cuda_kv4_read");
    int rc = check_paged_kv4(kv);
    if (rc == HESA_CUDA_OK) rc = check_batch4(kv, layer, batch, kv->n_kv_head);
    if (rc != HESA_CUDA_OK) return rc;
    if (batch->n_tokens == 0 || (!k && !v)) return HESA_CUDA_OK;
    const int64_t width = static_cast<int64_t>(kv->n_kv_head) * kv->head_dim;
    if ((k && (ldk < width || ldk > (int64_t(1) << 40))) || (v && (ldv < width || ldv > (int64_t(1) << 40))))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "leading dimension too small or too large");
    if (!aligned(k, 16) || !aligned(v, 16) || (k && (ldk & 3)) || (v && (ldv & 3)))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "k and v must be 16-byte aligned with leading dimensions multiples of 4");
    int* status = nullptr;
    cudaError_t e = status_word(&status);
    if (e == cudaSuccess) {
        // rows for one block after another only where there are blocks for every SM several times over
        const int64_t chunks = 2 * ((width / 4 + kReadChunk - 1) / kReadChunk);
        const int rows = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostRows, batch->n_tokens / (148 * 6))));
        const int64_t y = rows > 1 ? 1 : std::min<int64_t>(chunks, 1024);
        e = launch_dep(kv4_read_kernel, dim3(static_cast<unsigned>((batch->n_tokens + rows - 1) / rows), static_cast<unsigned>(y)), 256, 0, static_cast<cudaStream_t>(stream),
                       layer_of4(kv), pools_of(kv, layer), view_of(batch), k, ldk, v, ldv, rows, status);
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "kv4_read kernel");
}

}  // extern "C"
