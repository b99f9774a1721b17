// top_rows.cuh -- one pass over (a part of) a row of logits: its softmax sums, its
// entropy's sum and its largest values with their ids (token_logprobs.cu says how
// and why), for a block of WARPS warps.
#pragma once

#include <cstdint>

#include "hesa_common.cuh"

namespace hesa_cuda {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kUnroll = 4;           // quads a thread has in flight
constexpr int kAgain = 4;            // and when a few are read again

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

// Keys that are gathered before the k largest of them are kept: twice what may come in one step.
constexpr int cand_of(int warps) { return 2 * 4 * 32 * warps + kMaxTop; }

// The k largest of the n keys in cand (distinct; fewer than k are followed by
// zeros), descending, into out. All threads of the block.
template <int WARPS>
__device__ __forceinline__ void select(const uint64_t* cand, int n, int k, uint64_t* out) {
    if (static_cast<int>(threadIdx.x) < k) out[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += WARPS * 32) {
        const uint64_t c = cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += cand[j] > c;
        if (rank < k && c != 0) out[rank] = c;
    }
    __syncthreads();
}

__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t v) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(v >> 32) == hi ? static_cast<uint32_t>(v) : 0u);
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Shared memory of a block.
template <bool TOP, int WARPS = kLpWarps> struct TopShared {
    Sums sums[WARPS];
    uint64_t cand[TOP ? cand_of(WARPS) : 1], top[kMaxTop], key[WARPS];
    int from[TOP ? WARPS * 32 : 1];   // the threads in cand, then those whose values are read again
    int n;
};

// Part `split` of n_split of a row: its sums, in every thread, and with TOP its
// top_k largest keys, descending, in sh.top (zeros behind them).
template <bool TOP, int WARPS = kLpWarps>
__device__ __forceinline__ Sums row_part(const float* row, int vocab, int split, int n_split, int top_k, TopShared<TOP, WARPS>& sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
    constexpr int kStep = WARPS * 32 * kUnroll;
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
        // the thread's largest key; a thread that has read its quads at once still has them. No more than a thread a warp
        // are quicker read again, a quad a lane: 505 rows of 4029, 5 alternatives 8.3 us and 9.3, 19 of them 14.0 and 10.5
        const bool once = q1 - q0 <= kStep && top_k > WARPS;
        const int mine0 = q0 + warp * 32 * kUnroll + lane;
        uint64_t mine;
        {
            float4 v;
            if (once) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
                    if (u == 0 || best == mine0 + u * 32) v = nx[u];
            } else {
                v = quad(best);
            }
            uint64_t k[4];
            keys(best, v, k);
            mine = max_key(max_key(k[0], k[1]), max_key(k[2], k[3]));
        }
        // each warp's ceil(k / 8)-th bounds the k-th of the block's from below; the threads above the least of them are ranked
        uint64_t rest = mine, nth = 0;
        for (int i = 0; i < (top_k + WARPS - 1) / WARPS; ++i) {
            nth = warp_max_key(rest);
            if (rest == nth) rest = 0;
        }
        if (lane == 0) sh.key[warp] = nth;
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        uint64_t least = sh.key[0];
#pragma unroll
        for (int w2 = 1; w2 < WARPS; ++w2) least = least < sh.key[w2] ? least : sh.key[w2];
        if (mine != 0 && mine >= least) {
            const int at = atomicAdd(&sh.n, 1);
            sh.cand[at] = mine;
            sh.from[at] = threadIdx.x;
        }
        __syncthreads();
        const int n_max = sh.n;
        int rank = kMaxTop, from = 0;
        if (static_cast<int>(threadIdx.x) < n_max) {
            const uint64_t c = sh.cand[threadIdx.x];
            from = sh.from[threadIdx.x];
            rank = 0;
            for (int j = 0; j < n_max; ++j) rank += sh.cand[j] > c;
            if (rank < top_k) sh.top[rank] = c;
        }
        __syncthreads();
        if (rank < top_k) sh.from[rank] = from;
        const int n_from = min(n_max, top_k);
        uint64_t bound = n_max >= top_k ? sh.top[top_k - 1] : 0;
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        static_assert(cand_of(WARPS) >= kMaxTop * 4 * kUnroll, "what is read once fits");
        if (once) {   // at most kMaxTop threads, 16 values each
            if (mine != 0 && mine >= bound) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    uint64_t k[4];
                    keys(mine0 + u * 32, nx[u], k);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (k[i] != 0 && k[i] >= bound) sh.cand[atomicAdd(&sh.n, 1)] = k[i];
                }
            }
            __syncthreads();
        }
        // their values again: a warp takes one thread's quads, a quad a lane at a time
        for (int f0 = once ? n_from : 0; f0 < n_from; f0 += WARPS) {
            const int f = f0 + warp < n_from ? sh.from[f0 + warp] : -1;
            const int base = q0 + (f >> 5) * 32 * kUnroll + (f & 31);
            const int n_mine = (q1 - q0 + kStep - 1) / kStep * kUnroll;   // quads of a thread at most
            for (int i1 = 0; i1 < n_mine; i1 += 32 * kAgain) {
                // their reads side by side
                float4 v[kAgain];
                int q[kAgain];
#pragma unroll
                for (int a = 0; a < kAgain; ++a) {
                    if (i1 + a * 32 >= n_mine) break;   // (100 rows of 32000, 32 alternatives: 19.9 us, with reads of nothing 24.1)
                    const int i = i1 + a * 32 + lane;
                    q[a] = f >= 0 && i < n_mine ? base + (i / kUnroll) * kStep + (i % kUnroll) * 32 : q1;
                    if (q[a] < q1) v[a] = quad(q[a]);
                }
#pragma unroll
                for (int a = 0; a < kAgain; ++a) {
                    if (i1 + a * 32 >= n_mine) break;
                    if (q[a] < q1) {
                        uint64_t k[4];
                        keys(q[a], v[a], k);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (k[i] != 0 && k[i] >= bound) sh.cand[atomicAdd(&sh.n, 1)] = k[i];
                    }
                    __syncthreads();
                    // as many more may come: keep the k largest, the k-th is the new bound
                    const int n = sh.n;
                    __syncthreads();
                    if (n > cand_of(WARPS) - 4 * 32 * WARPS) {
                        select<WARPS>(sh.cand, n, top_k, sh.top);
                        if (static_cast<int>(threadIdx.x) < top_k) sh.cand[threadIdx.x] = sh.top[threadIdx.x];
                        bound = sh.top[top_k - 1];
                        if (threadIdx.x == 0) sh.n = top_k;
                        __syncthreads();
                    }
                }
            }
        }
        select<WARPS>(sh.cand, sh.n, top_k, sh.top);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const Sums y{__shfl_xor_sync(0xffffffffu, s.m, off), __shfl_xor_sync(0xffffffffu, s.z, off), __shfl_xor_sync(0xffffffffu, s.w, off)};
        s = (lane & off) ? merge(y, s) : merge(s, y);   // the same order of operands on both sides
    }
    if (lane == 0) sh.sums[warp] = s;
    __syncthreads();
    s = sh.sums[0];
    for (int w2 = 1; w2 < WARPS; ++w2) s = merge(s, sh.sums[w2]);
    return s;
}

}  // namespace hesa_cuda
