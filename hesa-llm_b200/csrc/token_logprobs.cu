// token_logprobs.cu -- log probabilities of given tokens, the entropy of each
// row and its most probable tokens, from fp32 logits in one pass.
//
//   z = sum_i e^(x_i - m), w = sum_i e^(x_i - m) (x_i - m), m = max_i x_i
//   logprob = (x_token - m) - log z,  entropy = log z - w / z
//
// Each thread keeps (m, z, w) of what it has read and rescales when its maximum
// grows: z e^d, e^d (w + z d), d = m_old - m_new.
//
// The k largest cost the stream next to nothing (keeping lists in the warps took
// 146 us where the stream alone takes 85): a thread only notes where it met its
// maximum. The k-th of the 256 threads' maxima bounds the row's k-th from below,
// and what is no smaller lies with the k threads whose maxima are: their values
// alone (k / 256 of the row) are read again, those above the bound gathered, and
// each goes to the place of its rank. Values are compared with their ids, so all
// of this holds for rows of equal values.
// HBM-bound: every logit is read once, as aligned 16-byte quads whatever the
// row's alignment (the first and the last quad of a row are read by the word), a
// step ahead of its use. Few rows are split over blocks; the last block of a row
// to arrive joins the parts.
// 1024 rows of 131071, five alternatives: 99 us (537 MB, 5.4 TB/s), 32: 149 us, none: 85 us; one row of 32000:
// 9.2 us.
#include "../../include/hesa_cuda.h"
#include "abi_errors.h"
#include "paged.h"
#include "qmatvec.h"
#include "top_rows.cuh"
#include "trace.h"

#include <cuda/atomic>

#include <algorithm>

namespace hesa_cuda {
namespace {

constexpr int kMaxSplits = 64;       // of a row
constexpr int kLpRowsSplit = 1024;   // rows up to here may be split: one counter each, whatever the shape
constexpr size_t kLpCounterBytes = kLpRowsSplit * sizeof(int32_t);
struct LpOut {
    float* logprob;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
};

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

template <bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4)
token_logprobs_kernel(const float* logits, int64_t ld, int n_rows, int vocab, const int32_t* tokens, int top_k, int n_split, LpOut o,
                      int32_t* counters, LpPart* parts, uint64_t* part_keys, int* status) {
    __shared__ TopShared<TOP> sh;
    __shared__ int s_last;
    uint64_t *const s_cand = sh.cand, *const s_top = sh.top;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x;
    const int split = blockIdx.y;
    const float* row = logits + r * ld;
    Sums s = row_part<TOP>(row, vocab, split, n_split, top_k, sh);
    if (n_split == 1) {
        if (warp == 0) finish_row(o, row, r, vocab, tokens, s, TOP && lane < top_k ? s_top[lane] : 0, top_k, lane, status);
        return;
    }
    const int64_t at = r * n_split + split;
    if (threadIdx.x == 0) parts[at] = LpPart{s.m, s.z, s.w, 0.f};
    if (TOP && static_cast<int>(threadIdx.x) < top_k) part_keys[at * top_k + threadIdx.x] = s_top[threadIdx.x];
    __syncthreads();
    if (threadIdx.x == 0) {
        cuda::atomic_ref<int32_t, cuda::thread_scope_device> c(counters[r]);
        s_last = c.fetch_add(1, cuda::memory_order_acq_rel) == n_split - 1;
    }
    __syncthreads();
    if (!s_last) return;
    cuda::atomic_thread_fence(cuda::memory_order_acquire, cuda::thread_scope_device);
    if (TOP) {
        // each warp joins every eighth list; a list's keys descend, so the first that is too small ends it
        const unsigned long long* lists = reinterpret_cast<const unsigned long long*>(part_keys + r * n_split * top_k);
        uint64_t mine = 0, next = lane < top_k && warp < n_split ? __ldcg(lists + warp * top_k + lane) : 0;
        for (int l = warp; l < n_split; l += kLpWarps) {
            const uint64_t theirs = next;
            next = lane < top_k && l + kLpWarps < n_split ? __ldcg(lists + (l + kLpWarps) * top_k + lane) : 0;
            if (l == warp) {
                mine = theirs;
                continue;
            }
            for (int i = 0; i < top_k; ++i) {
                const uint64_t c = __shfl_sync(0xffffffffu, theirs, i);
                if (c <= __shfl_sync(0xffffffffu, mine, top_k - 1)) break;
                insert(mine, c, lane);
            }
        }
        if (lane < top_k) s_cand[warp * top_k + lane] = mine;
        __syncthreads();
        select<kLpWarps>(s_cand, kLpWarps * top_k, top_k, s_top);
    }
    if (warp == 0) {
        // the parts' sums: at most 64, two a lane, joined in a fixed tree
        Sums t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t[i] = Sums{-INFINITY, 0.f, 0.f};
            if (2 * lane + i < n_split) {
                const float4 p = __ldcg(reinterpret_cast<const float4*>(parts + r * n_split + 2 * lane + i));
                t[i] = Sums{p.x, p.y, p.z};
            }
        }
        s = merge(t[0], t[1]);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const Sums y{__shfl_xor_sync(0xffffffffu, s.m, off), __shfl_xor_sync(0xffffffffu, s.z, off), __shfl_xor_sync(0xffffffffu, s.w, off)};
            s = (lane & off) ? merge(y, s) : merge(s, y);
        }
        finish_row(o, row, r, vocab, tokens, s, TOP && lane < top_k ? s_top[lane] : 0, top_k, lane, status);
        if (lane == 0) {
            cuda::atomic_ref<int32_t, cuda::thread_scope_device> c(counters[r]);
            c.store(0, cuda::memory_order_relaxed);
        }
    }
}

// Splits of a row: about three blocks an SM, at least a quad for each thread a block.
int lp_splits(int64_t n_rows, int64_t vocab) {
    if (n_rows > kLpRowsSplit) return 1;
    const int64_t want = std::max<int64_t>(1, 148 * 3 / n_rows), most = std::max<int64_t>(1, vocab / (4 * kLpThreads));
    return static_cast<int>(std::min(std::min(want, most), static_cast<int64_t>(kMaxSplits)));
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
    if ((reinterpret_cast<uintptr_t>(tokens) | reinterpret_cast<uintptr_t>(logprob) | reinterpret_cast<uintptr_t>(entropy) |
         reinterpret_cast<uintptr_t>(top_ids) | reinterpret_cast<uintptr_t>(top_logprobs)) & 3)
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "tokens and outputs must be 4-byte aligned");
    if (workspace_bytes < hesa_cuda_token_logprobs_workspace_size(n_rows, vocab, top_k))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    int* status = nullptr;
    cudaError_t e = status_word(&status);
    if (e == cudaSuccess) {
        const int s = lp_splits(n_rows, vocab);
        uint8_t* ws = static_cast<uint8_t*>(workspace);
        LpPart* parts = reinterpret_cast<LpPart*>(ws + kLpCounterBytes);
        uint64_t* keys = reinterpret_cast<uint64_t*>(ws + kLpCounterBytes + static_cast<size_t>(n_rows) * s * sizeof(LpPart));
        e = launch_dep(top_k > 0 ? token_logprobs_kernel<true> : token_logprobs_kernel<false>, dim3(static_cast<unsigned>(n_rows), static_cast<unsigned>(s)), kLpThreads, 0,
                       static_cast<cudaStream_t>(stream), logits, ld, static_cast<int>(n_rows), static_cast<int>(vocab), tokens, top_k, s,
                       LpOut{logprob, entropy, top_ids, top_logprobs}, reinterpret_cast<int32_t*>(ws), parts, keys, status);
    }
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "token_logprobs kernel");
}

}  // extern "C"
