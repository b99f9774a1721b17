// token_logprobs.cu -- log probabilities of given tokens, the entropy of each
// row and its most probable tokens, from fp32 logits in one pass.
//
//   z = sum_i e^(x_i - m), w = sum_i e^(x_i - m) (x_i - m), m = max_i x_i
//   logprob = (x_token - m) - log z,  entropy = log z - w / z
//
// Each thread keeps (m, z, w) of what it has read and rescales when its maximum
// grows: (z, w) -> 2^d-scaled (z e^d, e^d (w + z d)), d = m_old - m_new. The k
// largest are kept by warps, one (value, id) a lane in descending order: a value
// that exceeds the k-th goes in by one ballot and one shift. A first threshold
// comes from the lanes' maxima of the first quads, so that a warp starts with
// about k insertions instead of one for each value, and a block's warps share
// the largest k-th value any of them holds (the row's k-th is no smaller).
// HBM-bound: every logit is read once, as aligned 16-byte quads whatever the
// row's alignment (the first and the last quad of a row are read by the word).
// Few rows are split over blocks; the last block of a row to arrive adds the
// parts in split order.
#include "../../include/hesa_cuda.h"
#include "abi_errors.h"
#include "paged.h"
#include "qmatvec.h"
#include "trace.h"

#include <cuda/atomic>

#include <algorithm>

namespace hesa_cuda {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kLpRowsSplit = 1024;   // rows up to here may be split: one counter each, whatever the shape
constexpr size_t kLpCounterBytes = kLpRowsSplit * sizeof(int32_t);
constexpr int kUnroll = 4;           // quads a thread has in flight

constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float lp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Sums {
    float m, z, w;
};

// b's sums added to a's. Empty sides (m = -inf) add nothing but a NaN z.
__device__ __forceinline__ Sums merge(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    const float ms = m == -INFINITY ? 0.f : m;
    const float da = a.m == -INFINITY ? 0.f : a.m - ms, db = b.m == -INFINITY ? 0.f : b.m - ms;
    const float fa = lp_ex2(da * kLog2e), fb = lp_ex2(db * kLog2e);
    // an e^d that is zero has nothing to add, even where z d is not finite
    const float wa = fa > 0.f ? fa * fmaf(a.z, da, a.w) : 0.f, wb = fb > 0.f ? fb * fmaf(b.z, db, b.w) : 0.f;
    return Sums{m, fmaf(a.z, fa, b.z * fb), wa + wb};
}

// Order of logits: a larger number first, equal ones by the lower id; NaN with -inf.
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (!(x >= -INFINITY)) x = -INFINITY;
    if (x == 0.f) x = 0.f;   // -0 and 0 are equal
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t make_key(float x, int32_t id) {
    return static_cast<uint64_t>(order_bits(x)) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int32_t key_id(uint64_t k) { return static_cast<int32_t>(~static_cast<uint32_t>(k)); }

// c into the warp's descending list (lane i holds the i-th largest; 0: none)
__device__ __forceinline__ void insert(uint64_t& mine, uint64_t c, int lane) {
    const unsigned above = __ballot_sync(0xffffffffu, mine > c);
    const int at = __popc(above);
    const uint64_t up = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane > at) mine = up;
    else if (lane == at) mine = c;
}

struct LpOut {
    float* logprob;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
};

// A block's (or a row's) result from its warps' (or blocks') lists: warp 0 merges
// n lists of k keys, each descending.
__device__ __forceinline__ uint64_t merge_lists(const uint64_t* lists, int n, int stride, int k, int lane) {
    uint64_t mine = lane < k ? __ldcg(reinterpret_cast<const unsigned long long*>(lists) + lane) : 0;
    for (int l = 1; l < n; ++l) {
        const uint64_t theirs = lane < k ? __ldcg(reinterpret_cast<const unsigned long long*>(lists) + static_cast<int64_t>(l) * stride + lane) : 0;
        for (int i = 0; i < k; ++i) {
            const uint64_t c = __shfl_sync(0xffffffffu, theirs, i);
            const uint64_t last = __shfl_sync(0xffffffffu, mine, k - 1);
            if (c <= last) break;   // their later ones are smaller still
            insert(mine, c, lane);
        }
    }
    return mine;
}

__device__ __forceinline__ void finish_row(const LpOut& o, const float* row, int64_t r, int vocab, const int32_t* tokens,
                                           const Sums& s, uint64_t mine, int top_k, int lane, int* status) {
    const float lz = logf(s.z);
    const bool none = s.z == 0.f;   // every logit is -inf
    if (lane == 0) {
        if (o.logprob) {
            const int t = tokens[r];
            float lp = 0.f;
            if (t >= 0 && t < vocab) {
                lp = none ? -INFINITY : (row[t] - s.m) - lz;
            } else if (t != -1) {
                record_status(status, kStatusBadPosition);
                lp = NAN;
            }
            o.logprob[r] = lp;
        }
        if (o.entropy) o.entropy[r] = none ? 0.f : lz - s.w / s.z;
    }
    if (lane < top_k) {
        const int64_t at = r * top_k + lane;
        if (o.top_ids) o.top_ids[at] = key_id(mine);
        if (o.top_logprobs) o.top_logprobs[at] = none ? -INFINITY : (key_value(mine) - s.m) - lz;
    }
}

struct LpPart {
    float m, z, w, pad;
};

__global__ void __launch_bounds__(kLpThreads)
token_logprobs_kernel(const float* logits, int64_t ld, int n_rows, int vocab, const int32_t* tokens,
                      int top_k, int n_split, LpOut o, int32_t* counters, LpPart* parts,
                      uint64_t* part_keys, int* status) {
    __shared__ Sums s_sums[kLpWarps];
    __shared__ uint64_t s_keys[kLpWarps][kMaxTop];
    __shared__ int s_last;
    __shared__ unsigned s_thr;   // order bits of the largest k-th value that a warp holds
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dep_wait();
    grid_dep_launch();
    const int64_t r = blockIdx.x;
    const int split = blockIdx.y;
    const float* row = logits + r * ld;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    // quad q holds elements 4 q - mis .. + 3
    const int n_quads = (vocab + mis + 3) / 4;
    const int q0 = static_cast<int>(static_cast<int64_t>(n_quads) * split / n_split);
    const int q1 = static_cast<int>(static_cast<int64_t>(n_quads) * (split + 1) / n_split);
    if (threadIdx.x == 0) s_thr = 0;
    __syncthreads();

    Sums s{-INFINITY, 0.f, 0.f};
    uint64_t mine = 0;                    // lane i: the warp's i-th largest
    float thr = -INFINITY;                // the k-th of the warp, or a bound from elsewhere
    bool full = top_k == 0, first = true;
    volatile unsigned* vthr = &s_thr;

    for (int qb = q0 + warp * 32 * kUnroll; qb < q1; qb += kLpWarps * 32 * kUnroll) {
        float x[kUnroll][4];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int q = qb + u * 32 + lane, e = 4 * q - mis;
            if (q < q1 && e >= 0 && e + 3 < vocab) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(row + e));
                x[u][0] = f.x; x[u][1] = f.y; x[u][2] = f.z; x[u][3] = f.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[u][i] = q < q1 && e + i >= 0 && e + i < vocab ? row[e + i] : -INFINITY;
            }
        }
        float qm[kUnroll], mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            qm[u] = fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3]));
            mx = fmaxf(mx, qm[u]);
        }
        if (mx > s.m) {
            const float d = s.m == -INFINITY ? 0.f : s.m - mx, f = lp_ex2(d * kLog2e);
            s.w = f > 0.f ? f * fmaf(s.z, d, s.w) : 0.f;
            s.z *= f;
            s.m = mx;
        }
        const float ms = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float t = x[u][i] - ms, e = lp_ex2(t * kLog2e);
                s.z += e;
                s.w += e > 0.f ? e * t : 0.f;   // -inf, ruled out: adds nothing
            }
        if (top_k > 0) {
            if (first) {
                // at least k values are no smaller than the k-th of the lanes' maxima
                first = false;
                int above = 0;
                for (int l = 0; l < 32; ++l) {
                    const float y = __shfl_sync(0xffffffffu, mx, l);
                    above += y > mx || (y == mx && l < lane);
                }
                const unsigned kth = __ballot_sync(0xffffffffu, above == top_k - 1);
                thr = __shfl_sync(0xffffffffu, mx, __ffs(kth) - 1);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                // equal values pass until the list is full: ids rise along a row, so a later equal one ranks lower
                const bool pass = full ? qm[u] > thr : !(qm[u] < thr);
                if (!__any_sync(0xffffffffu, pass)) continue;
                const int e = 4 * (qb + u * 32 + lane) - mis;
                const bool in_split = qb + u * 32 + lane < q1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = in_split && e + i >= 0 && e + i < vocab;
                    unsigned cand = __ballot_sync(0xffffffffu, in && (full ? x[u][i] > thr : !(x[u][i] < thr)));
                    while (cand) {
                        const int l = __ffs(cand) - 1;
                        cand &= cand - 1;
                        const uint64_t c = __shfl_sync(0xffffffffu, make_key(x[u][i], e + i), l);
                        if (c > __shfl_sync(0xffffffffu, mine, top_k - 1)) insert(mine, c, lane);
                    }
                }
                const uint64_t kth = __shfl_sync(0xffffffffu, mine, top_k - 1);
                if (kth != 0) {
                    // values equal to the k-th of this warp come later here, so they lose; those equal to
                    // another warp's k-th may win by a lower id: only a value below that one is left out
                    full = true;
                    thr = fmaxf(thr, key_value(kth));
                    if (lane == 0) atomicMax(&s_thr, static_cast<unsigned>(kth >> 32));
                }
            }
            const unsigned o2 = *vthr;
            if (o2 != 0) {
                const float other = key_value(static_cast<uint64_t>(o2) << 32);
                // strictly below the block's k-th: cannot be among its k largest
                const float below = nextafterf(other, -INFINITY);
                if (full && below > thr) thr = below;
            }
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const Sums y{__shfl_xor_sync(0xffffffffu, s.m, off), __shfl_xor_sync(0xffffffffu, s.z, off), __shfl_xor_sync(0xffffffffu, s.w, off)};
        s = (lane & off) ? merge(y, s) : merge(s, y);   // the same order of operands on both sides
    }
    if (lane == 0) s_sums[warp] = s;
    if (lane < kMaxTop) s_keys[warp][lane] = mine;
    __syncthreads();
    if (warp != 0) return;

    s = s_sums[0];
    for (int w2 = 1; w2 < kLpWarps; ++w2) s = merge(s, s_sums[w2]);
    if (top_k > 0) {
        mine = lane < top_k ? s_keys[0][lane] : 0;
        for (int w2 = 1; w2 < kLpWarps; ++w2)
            for (int i = 0; i < top_k; ++i) {
                const uint64_t c = s_keys[w2][i];
                if (c <= __shfl_sync(0xffffffffu, mine, top_k - 1)) break;
                insert(mine, c, lane);
            }
    }
    if (n_split == 1) {
        finish_row(o, row, r, vocab, tokens, s, mine, top_k, lane, status);
        return;
    }
    const int64_t at = r * n_split + split;
    if (lane == 0) parts[at] = LpPart{s.m, s.z, s.w, 0.f};
    if (lane < top_k) part_keys[at * top_k + lane] = mine;
    __syncwarp();
    if (lane == 0) {
        cuda::atomic_ref<int32_t, cuda::thread_scope_device> c(counters[r]);
        s_last = c.fetch_add(1, cuda::memory_order_acq_rel) == n_split - 1;
    }
    __syncwarp();
    if (!s_last) return;
    cuda::atomic_thread_fence(cuda::memory_order_acquire, cuda::thread_scope_device);
    s = Sums{-INFINITY, 0.f, 0.f};
    for (int i = 0; i < n_split; ++i) {
        const float4 p = __ldcg(reinterpret_cast<const float4*>(parts + r * n_split + i));
        s = merge(s, Sums{p.x, p.y, p.z});
    }
    if (top_k > 0) mine = merge_lists(part_keys + r * n_split * top_k, n_split, top_k, top_k, lane);
    finish_row(o, row, r, vocab, tokens, s, mine, top_k, lane, status);
    if (lane == 0) {
        cuda::atomic_ref<int32_t, cuda::thread_scope_device> c(counters[r]);
        c.store(0, cuda::memory_order_relaxed);
    }
}

// Splits of a row: about two blocks an SM, at least 1024 quads (4 for each thread) a block.
int lp_splits(int64_t n_rows, int64_t vocab) {
    if (n_rows > kLpRowsSplit) return 1;
    const int64_t want = std::max<int64_t>(1, 148 * 2 / n_rows), most = std::max<int64_t>(1, vocab / 4 / (kLpThreads * kUnroll));
    return static_cast<int>(std::min(std::min(want, most), int64_t(64)));
}

}  // namespace
}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_token_logprobs_workspace_size(int64_t n_rows, int64_t vocab, int32_t top_k) {
    if (n_rows <= 0 || vocab <= 0 || n_rows >= (int64_t(1) << 31) || vocab >= (int64_t(1) << 30) || top_k < 0 || top_k > kMaxTop) return 0;
    const int s = lp_splits(n_rows, vocab);
    if (s == 1) return kLpCounterBytes;
    return kLpCounterBytes + static_cast<size_t>(n_rows) * s * (sizeof(LpPart) + static_cast<size_t>(top_k) * 8);
}

int hesa_cuda_token_logprobs(const float* logits, int64_t ld, int64_t n_rows, int64_t vocab, const int32_t* tokens, int32_t top_k,
                             float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs, void* workspace,
                             size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_token_logprobs");
    if (n_rows < 0 || vocab <= 0 || n_rows >= (int64_t(1) << 31) || vocab >= (int64_t(1) << 30) || ld < vocab || ld > (int64_t(1) << 40))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "bad shape");
    if (top_k < 0 || top_k > kMaxTop || top_k > vocab)
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "top_k must be 0 .. 32 and at most vocab");
    if (n_rows == 0) return HESA_CUDA_OK;
    if (!logits || !workspace || (logprob && !tokens) || (top_k > 0 && !top_ids && !top_logprobs))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if ((reinterpret_cast<uintptr_t>(logits) & 3) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "logits must be 4-byte and the workspace 16-byte aligned");
    if (workspace_bytes < hesa_cuda_token_logprobs_workspace_size(n_rows, vocab, top_k))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    int* status = nullptr;
    cudaError_t e = status_word(&status);
    if (e == cudaSuccess) {
        const int s = lp_splits(n_rows, vocab);
        uint8_t* ws = static_cast<uint8_t*>(workspace);
        LpPart* parts = reinterpret_cast<LpPart*>(ws + kLpCounterBytes);
        uint64_t* keys = reinterpret_cast<uint64_t*>(ws + kLpCounterBytes + static_cast<size_t>(n_rows) * s * sizeof(LpPart));
        e = launch_dep(token_logprobs_kernel, dim3(static_cast<unsigned>(n_rows), static_cast<unsigned>(s)), kLpThreads, 0,
                       static_cast<cudaStream_t>(stream), logits, ld, static_cast<int>(n_rows), static_cast<int>(vocab), tokens, top_k, s,
                       LpOut{logprob, entropy, top_ids, top_logprobs}, reinterpret_cast<int32_t*>(ws), parts, keys, status);
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "token_logprobs kernel");
}

}  // extern "C"
