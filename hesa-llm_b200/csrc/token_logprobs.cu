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
// 1024 rows of 131071, five alternatives: 101 us (537 MB, 5.3 TB/s), 32: 150 us, none: 85 us; one row of 32000:
// 9.9 us.
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
constexpr int kMaxSplits = 64;       // of a row
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

constexpr int kCand = 2 * 1024 + kMaxTop;   // keys that are gathered before the k largest of them are kept

// The k largest of the n keys in cand (distinct; fewer than k are followed by
// zeros), descending, into out. All threads of the block.
__device__ __forceinline__ void select(const uint64_t* cand, int n, int k, uint64_t* out) {
    if (static_cast<int>(threadIdx.x) < k) out[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kLpThreads) {
        const uint64_t c = cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += cand[j] > c;
        if (rank < k && c != 0) out[rank] = c;
    }
    __syncthreads();
}

__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_key(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
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

template <bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4)
token_logprobs_kernel(const float* logits, int64_t ld, int n_rows, int vocab, const int32_t* tokens, int top_k, int n_split, LpOut o,
                      int32_t* counters, LpPart* parts, uint64_t* part_keys, int* status) {
    __shared__ Sums s_sums[kLpWarps];
    __shared__ uint64_t s_cand[TOP ? kCand : 1], s_top[kMaxTop], s_key[kLpWarps];
    __shared__ int s_from[TOP ? kLpThreads : 1];   // the threads in s_cand, then those whose values are read again
    __shared__ int s_last, s_n;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x;
    const int split = blockIdx.y;
    const float* row = logits + r * ld;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    // quad q holds elements 4 q - mis .. + 3
    const int n_quads = (vocab + mis + 3) / 4;
    const int q0 = static_cast<int>(static_cast<int64_t>(n_quads) * split / n_split);
    const int q1 = static_cast<int>(static_cast<int64_t>(n_quads) * (split + 1) / n_split);

    auto quad = [&](int q) {
        const int e = 4 * q - mis;
        if (q < q1 && e >= 0 && e + 3 < vocab) return __ldcs(reinterpret_cast<const float4*>(row + e));
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = q < q1 && e + i >= 0 && e + i < vocab ? row[e + i] : -INFINITY;
        return make_float4(x[0], x[1], x[2], x[3]);
    };
    // a quad's keys; 0 for what is not of the row
    auto keys = [&](int q, const float4& x, uint64_t (&k)[4]) {
        const int e = 4 * q - mis;
        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = q < q1 && e + i >= 0 && e + i < vocab ? make_key(v[i], e + i) : 0;
    };
    // the thread's quads: qb + u * 32 for u < kUnroll, then kStep further on
    constexpr int kStep = kLpWarps * 32 * kUnroll;
    Sums s{-INFINITY, 0.f, 0.f};
    float4 nx[kUnroll];
    int qb = q0 + warp * 32 * kUnroll + lane, best = qb;   // best: the quad of the first maximum
    if (qb < q1) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) nx[u] = quad(qb + u * 32);
    }
    for (; qb < q1; qb += kStep) {
        float4 x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) x[u] = nx[u];
        if (qb + kStep < q1) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) nx[u] = quad(qb + kStep + u * 32);
        }
        float qm[kUnroll], mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            qm[u] = fmaxf(fmaxf(x[u].x, x[u].y), fmaxf(x[u].z, x[u].w));
            mx = fmaxf(mx, qm[u]);
        }
        if (mx > s.m) {
            const float d = s.m == -INFINITY ? 0.f : s.m - mx, f = lp_ex2(d * kLog2e);
            s.w = f > 0.f ? f * fmaf(s.z, d, s.w) : 0.f;
            s.z *= f;
            s.m = mx;
#pragma unroll
            for (int u = kUnroll - 1; u >= 0; --u) best = qm[u] == mx ? qb + u * 32 : best;
        }
        const float ms = s.m == -INFINITY ? 0.f : s.m;
        float2 z = make_float2(0.f, 0.f), w = make_float2(0.f, 0.f);
        // e^-200 is 0 in fp32: what is further down (-inf, ruled out) adds nothing; NaN stays
        auto add = [&](float a, float b) {
            float2 t = fadd2(make_float2(a, b), make_float2(-ms, -ms));
            t.x = fmax_nan(t.x, -200.f);
            t.y = fmax_nan(t.y, -200.f);
            const float2 e = make_float2(lp_ex2(t.x * kLog2e), lp_ex2(t.y * kLog2e));
            z = fadd2(z, e);
            w = ffma2(e, t, w);
        };
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            add(x[u].x, x[u].y);
            add(x[u].z, x[u].w);
        }
        s.z += z.x + z.y;
        s.w += w.x + w.y;
    }
    if (TOP) {
        // the thread's largest key
        uint64_t mine;
        {
            uint64_t k[4];
            keys(best, quad(best), k);
            mine = max_key(max_key(k[0], k[1]), max_key(k[2], k[3]));
        }
        // each warp's ceil(k / 8)-th bounds the k-th of the block's from below; the threads above the least of them are ranked
        uint64_t rest = mine, nth = 0;
        for (int i = 0; i < (top_k + kLpWarps - 1) / kLpWarps; ++i) {
            nth = warp_max_key(rest);
            if (rest == nth) rest = 0;
        }
        if (lane == 0) s_key[warp] = nth;
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        uint64_t least = s_key[0];
#pragma unroll
        for (int w2 = 1; w2 < kLpWarps; ++w2) least = least < s_key[w2] ? least : s_key[w2];
        if (mine != 0 && mine >= least) {
            const int at = atomicAdd(&s_n, 1);
            s_cand[at] = mine;
            s_from[at] = threadIdx.x;
        }
        __syncthreads();
        const int n_max = s_n;
        int rank = kMaxTop, from = 0;
        if (static_cast<int>(threadIdx.x) < n_max) {
            const uint64_t c = s_cand[threadIdx.x];
            from = s_from[threadIdx.x];
            rank = 0;
            for (int j = 0; j < n_max; ++j) rank += s_cand[j] > c;
            if (rank < top_k) s_top[rank] = c;
        }
        __syncthreads();
        if (rank < top_k) s_from[rank] = from;
        const int n_from = min(n_max, top_k);
        uint64_t bound = n_max >= top_k ? s_top[top_k - 1] : 0;
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        // their values again: a warp takes one thread's quads, a quad a lane at a time
        for (int f0 = 0; f0 < n_from; f0 += kLpWarps) {
            const int f = f0 + warp < n_from ? s_from[f0 + warp] : -1;
            const int base = q0 + (f >> 5) * 32 * kUnroll + (f & 31);
            const int n_mine = (q1 - q0 + kStep - 1) / kStep * kUnroll;   // quads of a thread at most
            for (int i0 = 0; i0 < n_mine; i0 += 32) {
                if (f >= 0 && i0 + lane < n_mine) {
                    const int q = base + ((i0 + lane) / kUnroll) * kStep + ((i0 + lane) % kUnroll) * 32;
                    uint64_t k[4];
                    keys(q, quad(q), k);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (k[i] != 0 && k[i] >= bound) s_cand[atomicAdd(&s_n, 1)] = k[i];
                }
                __syncthreads();
                // 1024 more may come: keep the k largest, the k-th is the new bound
                const int n = s_n;
                __syncthreads();
                if (n > kCand - 4 * kLpThreads) {
                    select(s_cand, n, top_k, s_top);
                    if (static_cast<int>(threadIdx.x) < top_k) s_cand[threadIdx.x] = s_top[threadIdx.x];
                    bound = s_top[top_k - 1];
                    if (threadIdx.x == 0) s_n = top_k;
                    __syncthreads();
                }
            }
        }
        select(s_cand, s_n, top_k, s_top);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const Sums y{__shfl_xor_sync(0xffffffffu, s.m, off), __shfl_xor_sync(0xffffffffu, s.z, off), __shfl_xor_sync(0xffffffffu, s.w, off)};
        s = (lane & off) ? merge(y, s) : merge(s, y);   // the same order of operands on both sides
    }
    if (lane == 0) s_sums[warp] = s;
    __syncthreads();
    s = s_sums[0];
    for (int w2 = 1; w2 < kLpWarps; ++w2) s = merge(s, s_sums[w2]);
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
        select(s_cand, kLpWarps * top_k, top_k, s_top);
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
