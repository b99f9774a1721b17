// beam_select.cu -- the next beams of a beam search, over beams and vocabulary.
//
//   score(b, t) = scores[b] + (x_bt - m_b) - log z_b,  z_b = sum_t e^(x_bt - m_b)
//
// The best `width` of a sequence are among the best `width` of each of its beams,
// and within a beam the order is that of the logits. So the first kernel takes a
// pass over every beam's logits (a block a beam, or a part of one where beams are
// few) for its sums and its `width` largest logits; the second, a block a sequence,
// joins the parts of each beam and gives every candidate that is left its rank.
// Between beams it is the sums that decide, and they may be very close: they are
// made in 64 bits from z's fp32 terms.
// HBM-bound: every logit is read once (those of ended and ruled-out beams not at
// all); a few beams are bound by the latency of the two launches.
#include "../../include/hesa_cuda.h"
#include "abi_errors.h"
#include "paged.h"
#include "qmatvec.h"
#include "top_rows.cuh"
#include "trace.h"

#include <algorithm>

namespace hesa_cuda {
namespace {

constexpr int kMaxWidth = kMaxTop;
constexpr int kMostParts = 64;   // of a row

struct RowPart {
    float m, z;
};

// Whether a beam's logits count: it has not ended and its score is a number above -inf.
__device__ __forceinline__ bool counts(const float* scores, const int32_t* ended, int64_t r) {
    return !(ended && ended[r] != 0) && scores[r] > -INFINITY && scores[r] < INFINITY;
}

__global__ void __launch_bounds__(kLpThreads, 4)
beam_rows_kernel(const float* logits, int64_t ld, int vocab, const float* scores, const int32_t* ended, int top, int n_split, RowPart* parts,
                 uint64_t* keys) {
    __shared__ TopShared<true> sh;
    grid_dep_wait();
    grid_dep_launch();
    const int64_t r = blockIdx.x;
    if (!counts(scores, ended, r)) return;
    const Sums s = row_part<true>(logits + r * ld, vocab, blockIdx.y, n_split, top, sh);
    const int64_t at = r * n_split + blockIdx.y;
    if (threadIdx.x == 0) parts[at] = RowPart{s.m, s.z};
    if (static_cast<int>(threadIdx.x) < top) keys[at * top + threadIdx.x] = sh.top[threadIdx.x];
}

// Numbers in 64 bits as whole ones of the same order.
__device__ __forceinline__ uint64_t order_of(double x) {
    if (x == 0.0) x = 0.0;   // -0 and 0 are equal
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
    return u >> 63 ? ~u : u | (uint64_t(1) << 63);
}

__global__ void __launch_bounds__(kLpThreads)
beam_join_kernel(const float* scores, const int32_t* ended, int width, int vocab, int top, int n_split, const RowPart* parts, const uint64_t* keys,
                 float* next_scores, int32_t* parents, int32_t* tokens) {
    // candidate b * kMaxWidth + i: the i-th of beam b
    __shared__ uint64_t s_key[kMaxWidth * kMaxWidth];
    __shared__ double s_score[kMaxWidth * kMaxWidth];
    __shared__ int s_token[kMaxWidth * kMaxWidth];
    __shared__ int s_n[kMaxWidth];
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * width;
    for (int b = warp; b < width; b += kLpWarps) {
        const int64_t r = r0 + b;
        const float score = scores[r];
        const bool end = ended && ended[r] != 0, nan = !(score < INFINITY), dead = !end && !counts(scores, ended, r);
        double mine = nan ? NAN : score;
        uint64_t order = order_of(nan ? -INFINITY : score);
        int token = end ? -1 : lane;   // the lowest tokens of a beam whose candidates are all alike
        if (!end && !dead) {
            const RowPart* p = parts + r * n_split;
            float m = -INFINITY;
            for (int i = lane; i < n_split; i += 32) m = fmaxf(m, __ldcg(&p[i].m));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float ms = m == -INFINITY ? 0.f : m;
            double z = 0.0;
            for (int i = lane; i < n_split; i += 32) {
                const float pm = __ldcg(&p[i].m), pz = __ldcg(&p[i].z);
                z += pm == -INFINITY ? pz : pz * exp(static_cast<double>(pm) - ms);   // a part of nothing but NaN has m -inf and z NaN
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
            // the parts' lists joined: a lane has the heads of two of them (and what comes behind these on its way), the
            // largest of all heads is the next one
            const unsigned long long* lists = reinterpret_cast<const unsigned long long*>(keys + r * n_split * top);
            auto key_of = [&](int l, int i) -> uint64_t { return l < n_split && i < top ? __ldcg(lists + static_cast<int64_t>(l) * top + i) : 0; };
            uint64_t head0 = key_of(lane, 0), head1 = key_of(lane + 32, 0), next0 = key_of(lane, 1), next1 = key_of(lane + 32, 1), best = 0;
            int at0 = 1, at1 = 1;
            for (int i = 0; i < top; ++i) {
                const uint64_t c = warp_max_key(max_key(head0, head1));
                if (lane == i) best = c;
                if (head0 == c) {
                    head0 = next0;
                    next0 = key_of(lane, ++at0);
                } else if (head1 == c) {
                    head1 = next1;
                    next1 = key_of(lane + 32, ++at1);
                }
            }
            if (isfinite(z)) {
                // z = 0: every logit is ruled out
                const float x = key_value(best);
                mine = x == -INFINITY ? -INFINITY : score + (static_cast<double>(x) - m) - log(z);
                token = key_id(best);
                order = order_of(mine);
            } else {
                mine = NAN;   // NaN or +inf among the logits
                order = order_of(-INFINITY);
            }
        }
        const int n = end ? 1 : top;
        if (lane == 0) s_n[b] = n;
        if (lane < n) {
            s_key[b * kMaxWidth + lane] = order;
            s_score[b * kMaxWidth + lane] = mine;
            s_token[b * kMaxWidth + lane] = token;
        }
    }
    __syncthreads();
    // the rank of each: how many are larger, or equal with a lower number
    for (int c = threadIdx.x; c < width * kMaxWidth; c += kLpThreads) {
        const int b = c / kMaxWidth, i = c % kMaxWidth;
        if (i >= s_n[b]) continue;
        const uint64_t key = s_key[c];
        int rank = 0;
        for (int y = 0; y < width && rank < width; ++y)
            for (int x = 0; x < s_n[y]; ++x) {   // a beam's candidates descend
                const uint64_t k = s_key[y * kMaxWidth + x];
                if (k < key || (k == key && y * kMaxWidth + x >= c)) break;
                ++rank;
            }
        if (rank < width) {
            const int64_t o = r0 + rank;
            next_scores[o] = static_cast<float>(s_score[c]);
            parents[o] = b;
            tokens[o] = s_token[c];
        }
    }
}

// Parts of a row: blocks enough that the SMs end together though some beams have ended, at least a quad for each thread a block.
int parts_of(int64_t n_rows, int64_t vocab) {
    const int64_t want = (148 * 8 + n_rows - 1) / n_rows, most = std::max<int64_t>(1, vocab / (4 * kLpThreads));
    return static_cast<int>(std::min(std::min(want, most), static_cast<int64_t>(kMostParts)));
}

bool shape_ok(int64_t n_seq, int32_t width, int64_t vocab) {
    return n_seq >= 0 && width >= 1 && width <= kMaxWidth && vocab > 0 && vocab < (int64_t(1) << 30) && n_seq < (int64_t(1) << 31) / kMaxWidth;
}

}  // namespace
}  // namespace hesa_cuda

using namespace hesa_cuda;

extern "C" {

size_t hesa_cuda_beam_select_workspace_size(int64_t n_seq, int32_t width, int64_t vocab) {
    if (!shape_ok(n_seq, width, vocab) || n_seq == 0) return 0;
    const int64_t top = std::min<int64_t>(width, vocab), rows = n_seq * width;
    return static_cast<size_t>(rows) * parts_of(rows, vocab) * (sizeof(RowPart) + top * sizeof(uint64_t));
}

int hesa_cuda_beam_select(const float* logits, int64_t ld, int64_t n_seq, int32_t width, int64_t vocab, const float* scores, const int32_t* ended,
                          float* next_scores, int32_t* parents, int32_t* tokens, void* workspace, size_t workspace_bytes, void* stream) {
    HESA_TRACE("hesa_cuda_beam_select");
    if (!shape_ok(n_seq, width, vocab) || ld < vocab || ld > (int64_t(1) << 40))
        return record_error(HESA_CUDA_SHAPE_MISMATCH, "bad shape: width must be 1 .. 32, ld at least vocab");
    if (n_seq == 0) return HESA_CUDA_OK;
    if (!logits || !scores || !next_scores || !parents || !tokens || !workspace) return record_error(HESA_CUDA_INVALID_ARGUMENT, "null pointer");
    if (((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(ended) |
          reinterpret_cast<uintptr_t>(next_scores) | reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(tokens)) & 3) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "buffers must be 4-byte and the workspace 16-byte aligned");
    if (workspace_bytes < hesa_cuda_beam_select_workspace_size(n_seq, width, vocab))
        return record_error(HESA_CUDA_INVALID_ARGUMENT, "workspace too small");
    const int64_t rows = n_seq * width;
    const int top = static_cast<int>(std::min<int64_t>(width, vocab)), n_split = parts_of(rows, vocab);
    RowPart* parts = static_cast<RowPart*>(workspace);
    uint64_t* keys = reinterpret_cast<uint64_t*>(parts + rows * n_split);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_dep(beam_rows_kernel, dim3(static_cast<unsigned>(rows), static_cast<unsigned>(n_split)), kLpThreads, 0, s, logits, ld,
                               static_cast<int>(vocab), scores, ended, top, n_split, parts, keys);
    if (e == cudaSuccess)
        e = launch_dep(beam_join_kernel, dim3(static_cast<unsigned>(n_seq)), kLpThreads, 0, s, scores, ended, width, static_cast<int>(vocab), top, n_split, parts,
                       keys, next_scores, parents, tokens);
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "beam_select kernels");
}

}  // extern "C"
