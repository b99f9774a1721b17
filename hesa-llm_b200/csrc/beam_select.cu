// beam_select.cu -- the next beams of a beam search, over beams and vocabulary.
//
//   score(b, t) = scores[b] + (x_bt - m_b) - log z_b,  z_b = sum_t e^(x_bt - m_b)
//
// The best `width` of a sequence are among the best `width` of each of its beams,
// and within a beam the order is that of the logits. So the first kernel takes a
// pass over every beam's logits (a block a beam, or a part of one where beams are
// few) for its sums and its `width` largest logits; the second, a block a sequence,
// joins the parts of each beam and gives every candidate that is left its rank.
// Where a cluster of eight blocks is enough for a sequence, one kernel does both.
// Between beams it is the sums that decide, and they may be very close: they are
// made in 64 bits from z's fp32 terms.
// HBM-bound: every logit is read once (those of ended and ruled-out beams not at
// all); a few beams are bound by the chain of waits at a row's end, many short rows by
// what is done there. 64 sequences of 8 beams, 131071 tokens, 355 of the beams alive:
// 49 us (186 MB, 3.8 TB/s; without finding the largest 43, and the same with 1 to 5
// parts a beam); 128 of 16 beams, 3000 tokens 30 us (the first kernel 58% of issue slots, 13% of DRAM);
// one of 4 beams, 32000 tokens 9.8 us.
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

// Blocks of two warps, against eight. What a row's largest are found in again takes them top / 2 steps instead of
// top / 8, so that wide searches need more rows to gain: 62 sequences of 16 beams, 3000 tokens 22.1 us and 29.5, 31 of 32,
// 1500 tokens 48 and 42, 100 of 32 71 and 72, 333 of 3, 3000 tokens 13.7 and 24.7. Rows of up to kSmallOnce logits are read
// once at any address: 16 of 20, 1000 tokens 21.9 and 23.3, 200 of 16 25.2 and 49.2.
constexpr int kSmallWarps = 2;
constexpr int kSmallOnce = kSmallWarps * 32 * kUnroll * 4 - 3;

struct RowPart {
    float m, z;
};

// Whether a beam's logits count: it has not ended and its score is a number above -inf.
__device__ __forceinline__ bool counts(const float* scores, const int32_t* ended, int64_t r) {
    return !(ended && ended[r] != 0) && scores[r] > -INFINITY && scores[r] < INFINITY;
}

template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 4 * kLpWarps / WARPS)
beam_rows_kernel(const float* logits, int64_t ld, int vocab, const float* scores, const int32_t* ended, int top, int n_split, RowPart* parts,
                 uint64_t* keys) {
    __shared__ TopShared<true, WARPS> sh;
    grid_dep_wait();
    grid_dep_launch();
    const int64_t r = blockIdx.x;
    if (!counts(scores, ended, r)) return;
    const Sums s = row_part<true, WARPS>(logits + r * ld, vocab, blockIdx.y, n_split, top, sh);
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

struct BeamOut {
    float* scores;
    int32_t* parents;
    int32_t* tokens;
};

// Candidates of a sequence: b * kMaxWidth + i is the i-th of beam b.
struct JoinShared {
    uint64_t key[kMaxWidth * kMaxWidth];
    double score[kMaxWidth * kMaxWidth];
    int token[kMaxWidth * kMaxWidth];
    int n[kMaxWidth];
};

// The next beams of the sequence whose first beam is row r0, from the n_split (at most
// kMostParts) parts of each of its beams: part(b, l) and key_of(b, l, i), the i-th key
// of part l of beam b. All threads of a block.
template <int WARPS, typename PartOf, typename KeyOf>
__device__ __forceinline__ void join_beams(const float* scores, const int32_t* ended, int64_t r0, int width, int top, int n_split, const PartOf& part,
                                           const KeyOf& key_of, JoinShared& sh, const BeamOut& out) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = warp; b < width; b += WARPS) {
        const int64_t r = r0 + b;
        const float score = scores[r];
        const bool end = ended && ended[r] != 0, nan = !(score < INFINITY), dead = !end && !counts(scores, ended, r);
        double mine = nan ? NAN : score;
        uint64_t order = order_of(nan ? -INFINITY : score);
        int token = end ? -1 : lane;   // the lowest tokens of a beam whose candidates are all alike
        if (!end && !dead) {
            float m = -INFINITY;
            for (int i = lane; i < n_split; i += 32) m = fmaxf(m, part(b, i).m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float ms = m == -INFINITY ? 0.f : m;
            double z = 0.0;
            for (int i = lane; i < n_split; i += 32) {
                const RowPart p = part(b, i);
                z += p.m == -INFINITY ? p.z : p.z * exp(static_cast<double>(p.m) - ms);   // a part of nothing but NaN has m -inf and z NaN
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
            // the parts' lists joined: a lane has the heads of two of them (and what comes behind these on its way), the
            // largest of all heads is the next one
            auto at = [&](int l, int i) -> uint64_t { return l < n_split && i < top ? key_of(b, l, i) : 0; };
            uint64_t best = 0;
            if (n_split == 1) {
                best = at(0, lane);
            } else {
                uint64_t head0 = at(lane, 0), head1 = at(lane + 32, 0), next0 = at(lane, 1), next1 = at(lane + 32, 1);
                int at0 = 1, at1 = 1;
                for (int i = 0; i < top; ++i) {
                    const uint64_t c = warp_max_key(max_key(head0, head1));
                    if (lane == i) best = c;
                    if (head0 == c) {
                        head0 = next0;
                        next0 = at(lane, ++at0);
                    } else if (head1 == c) {
                        head1 = next1;
                        next1 = at(lane + 32, ++at1);
                    }
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
        if (lane == 0) sh.n[b] = n;
        if (lane < n) {
            sh.key[b * kMaxWidth + lane] = order;
            sh.score[b * kMaxWidth + lane] = mine;
            sh.token[b * kMaxWidth + lane] = token;
        }
    }
    __syncthreads();
    // the rank of each: how many are larger, or equal with a lower number
    for (int c = threadIdx.x; c < width * kMaxWidth; c += WARPS * 32) {
        const int b = c / kMaxWidth, i = c % kMaxWidth;
        if (i >= sh.n[b]) continue;
        const uint64_t key = sh.key[c];
        int rank = 0;
        for (int y = 0; y < width && rank < width; ++y)
            for (int x = 0; x < sh.n[y]; ++x) {   // a beam's candidates descend
                const uint64_t k = sh.key[y * kMaxWidth + x];
                if (k < key || (k == key && y * kMaxWidth + x >= c)) break;
                ++rank;
            }
        if (rank < width) {
            const int64_t o = r0 + rank;
            out.scores[o] = static_cast<float>(sh.score[c]);
            out.parents[o] = b;
            out.tokens[o] = sh.token[c];
        }
    }
}

constexpr int kJoinWarps = 16;

__global__ void __launch_bounds__(kJoinWarps * 32)
beam_join_kernel(const float* scores, const int32_t* ended, int width, int top, int n_split, const RowPart* parts, const uint64_t* keys, BeamOut out) {
    __shared__ JoinShared sh;
    grid_dep_wait();
    grid_dep_launch();
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * width;
    const unsigned long long* lists = reinterpret_cast<const unsigned long long*>(keys);
    join_beams<kJoinWarps>(
        scores, ended, r0, width, top, n_split,
        [&](int b, int l) {
            const float2 p = __ldcg(reinterpret_cast<const float2*>(parts + (r0 + b) * n_split + l));
            return RowPart{p.x, p.y};
        },
        [&](int b, int l, int i) -> uint64_t { return __ldcg(lists + ((r0 + b) * n_split + l) * top + i); }, sh, out);
}

// Both in one launch, a cluster of eight blocks a sequence: each takes a beam or a
// part of one, and the first joins what the others have in their shared memory. For
// few sequences, rows that a few blocks are quick with, and no more beams than blocks:
// 64 sequences of 8 beams, 24000 tokens 20 us (two kernels 25), 16 of them 12.7 (15.5);
// one sequence of 4 beams, 32000 tokens 10.7 (9.6), but 3 us less of the host's time;
// 128 sequences of 2 beams, 24000 tokens 24 (14), one of 16 beams 25 (16).
constexpr int kCluster = 8;
constexpr int64_t kClusterElems = 24576;                               // logits of a part
constexpr int64_t kClusterSeqs = 148 * 4 / kCluster;                   // that are on the SMs at a time

__device__ __forceinline__ uint64_t lds_cluster(uint32_t a) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

__global__ void __launch_bounds__(kLpThreads, 4)
beam_cluster_kernel(const float* logits, int64_t ld, int vocab, const float* scores, const int32_t* ended, int width, int top, int n_split, BeamOut out) {
    __shared__ union {   // the join follows the last row
        TopShared<true> rows;
        JoinShared join;
    } sh;
    __shared__ __align__(8) RowPart s_part;
    __shared__ uint64_t s_keys[kMaxTop];
    grid_dep_wait();
    grid_dep_launch();
    const int rank = blockIdx.x % kCluster;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x / kCluster) * width;
    // part `rank` of them all
    const int64_t r = r0 + rank / n_split;
    if (rank < width * n_split && counts(scores, ended, r)) {
        const Sums s = row_part<true>(logits + r * ld, vocab, rank % n_split, n_split, top, sh.rows);
        if (threadIdx.x == 0) s_part = RowPart{s.m, s.z};
        if (static_cast<int>(threadIdx.x) < top) s_keys[threadIdx.x] = sh.rows.top[threadIdx.x];
    }
    __syncthreads();   // sh is the join's from here
    cluster_sync();
    if (rank == 0) {
        join_beams<kLpWarps>(
            scores, ended, r0, width, top, n_split,
            [&](int b, int l) {
                const uint64_t p = lds_cluster(in_block(&s_part, b * n_split + l));
                return RowPart{__uint_as_float(static_cast<uint32_t>(p)), __uint_as_float(static_cast<uint32_t>(p >> 32))};
            },
            [&](int b, int l, int i) -> uint64_t { return lds_cluster(in_block(&s_keys[i], b * n_split + l)); },
            sh.join, out);
    }
    cluster_sync();   // the others' shared memory has been read
}

// Parts of a row: what fits on the SMs at a time (four blocks each), none below
// kPartElems logits; where there are rows for more than that, about two rounds of
// blocks, so that SMs end together though some beams have ended.
constexpr int kPartElems = 4096;
int parts_of(int64_t n_rows, int64_t vocab) {
    const int64_t one = 148 * 4, want = n_rows <= one / 2 ? one / n_rows : (2 * one + n_rows - 1) / n_rows, most = std::max<int64_t>(1, vocab / kPartElems);
    return static_cast<int>(std::min(std::min(want, most), static_cast<int64_t>(kMostParts)));
}

// Parts of a row of a cluster's; 0: the two kernels.
int cluster_parts(int64_t n_seq, int32_t width, int64_t vocab) {
    const int parts = std::max(1, kCluster / width);
    return width <= kCluster && n_seq <= kClusterSeqs && vocab <= parts * kClusterElems ? parts : 0;
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
    const int top = static_cast<int>(std::min<int64_t>(width, vocab)), n_split = parts_of(rows, vocab), in_cluster = cluster_parts(n_seq, width, vocab);
    const BeamOut out{next_scores, parents, tokens};
    if (in_cluster > 0) {
        const cudaError_t e = launch_clusters(beam_cluster_kernel, kCluster, dim3(static_cast<unsigned>(n_seq * kCluster)), kLpThreads, 0, static_cast<cudaStream_t>(stream),
                                              logits, ld, static_cast<int>(vocab), scores, ended, width, top, in_cluster, out);
        return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "beam_select kernel");
    }
    RowPart* parts = static_cast<RowPart*>(workspace);
    uint64_t* keys = reinterpret_cast<uint64_t*>(parts + rows * n_split);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    // many short rows: small blocks, so that more of them, and of the waits at a row's end, go side by side
    const bool small = vocab <= kPartElems && rows > 148 * 2 && (vocab <= kSmallOnce || n_seq > 2 * width);
    cudaError_t e = launch_dep(small ? beam_rows_kernel<kSmallWarps> : beam_rows_kernel<kLpWarps>, dim3(static_cast<unsigned>(rows), static_cast<unsigned>(n_split)),
                               (small ? kSmallWarps : kLpWarps) * 32, 0, s, logits, ld, static_cast<int>(vocab), scores, ended, top, n_split, parts, keys);
    if (e == cudaSuccess)
        e = launch_dep(beam_join_kernel, dim3(static_cast<unsigned>(n_seq)), kJoinWarps * 32, 0, s, scores, ended, width, top, n_split, parts, keys, out);
    return e == cudaSuccess ? HESA_CUDA_OK : record_cuda_error(e, "beam_select kernels");
}

}  // extern "C"
