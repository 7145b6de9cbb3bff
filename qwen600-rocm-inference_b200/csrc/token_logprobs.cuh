// token_logprobs.cuh — log probabilities of given tokens, entropies and the
// likeliest tokens of rows of logits (qwen_token_logprobs).  No reference
// counterpart (the reference's sampler ends at a token, sampler.h:120-175).
//
// Mathematics.  With m the row's largest logit, y = (x - m) log2(e) / temperature,
// S = sum 2^y and U = sum 2^y y: log p(x) = ln 2 (y - log2 S) and the entropy is
// ln 2 (log2 S - U / S), both without cancellation.  One pass: every thread has a
// running (m, S, U) of its own elements; when m rises by d, U <- (U + S d') f and S <- S f
// with d' = -d log2(e) / temperature, f = 2^d'.  The threads' and the blocks' are joined the same way.
//
// The likeliest n.  The largest element of each thread falls out of the pass.  The n
// largest elements of a block lie with threads whose largest is among the n largest of
// those, so with T the n-th largest of the threads' largest, found bit by bit,
// only the threads at or above T have their elements read a second time
// (from the L2: n of 512 threads, by whole warps), and what is >= T is ranked by counting.
// Equal logits rank by their index, as one 64-bit number (value, then falling index), so no order of
// arrival shows.  Where kCand or more elements are >= T (many equal logits), those above T and the
// first ones equal to it are taken; should even those above be too many, one by one.
//
// Measured at 151,936 tokens: 2048 rows of bf16 with the likeliest 124 us (5.0 TB/s, floor 95), of fp32 without 197 us (6.3 TB/s);
// 128 rows of fp32 with the 5 likeliest 20 us (floor 11.9); one row with 20 10.7 us, 5.5 without.  Bound by memory
// traffic with many rows (bf16: close behind it the instructions, five an element), by latencies with few, which get
// a cluster of up to eight blocks each; the likeliest cost 5 us of barriers and second reads.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qwen_b200.h"
#include "ptx.cuh"
#include "tree_attention.cuh"

namespace qb {
namespace lp {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxTop = 64, kMaxCluster = 8, kCand = 1024;
constexpr int kAhead = 4;     // 16-byte pieces that a thread loads at once

struct Params {
    const uint8_t* logits;
    long long ld;
    int vocab, n_top;
    float c;                  // log2(e) / temperature
    const int* tokens;
    float *logprob, *entropy, *top_logprobs;
    int* top_ids;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Whole numbers in the order of the floats (0: below every one); -0 as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

template <int T>
struct Elem {
    static constexpr int kSize = T == QWEN_FP32 ? 4 : 2, kVec = 16 / kSize;
    static __device__ __forceinline__ float one(const uint8_t* p) {
        if constexpr (T == QWEN_FP32) return *reinterpret_cast<const float*>(p);
        else if constexpr (T == QWEN_BF16) return bf2f(*reinterpret_cast<const uint16_t*>(p));
        else return __half2float(*reinterpret_cast<const __half*>(p));
    }
    static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[kVec]) {
        const uint32_t r[4] = {w.x, w.y, w.z, w.w};
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (T == QWEN_FP32) {
                x[i] = __uint_as_float(r[i]);
            } else if constexpr (T == QWEN_BF16) {
                x[2 * i] = bf_lo(r[i]);
                x[2 * i + 1] = bf_hi(r[i]);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    }
};

__device__ __forceinline__ void fma2(float& a, float& b, float x, float y, float s, float t) {   // (a, b) + (x, y) * (s, t)
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\tfma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(a), "+f"(b) : "f"(x), "f"(y), "f"(s), "f"(t));
}
// A running (m, S, U).  S and U take in sums over kAhead pieces, so that the many small terms behind a large one are not lost one by one.
struct Sums {
    float m, s, u;
    __device__ __forceinline__ void rise(float to, float c) {
        const float d = fmaxf((m - to) * c, -200.0f), f = ex2(d);   // (m = -inf: nothing so far, f = 0)
        u = (u + s * d) * f;
        s *= f;
        m = to;
    }
    // elements x follow, the largest of them vm
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N], float vm, float c) {
        if (vm > m) rise(vm, c);
        if (m == -INFINITY) {                  // nothing above -inf so far; a NaN among them, which no maximum shows
            #pragma unroll
            for (int i = 0; i < N; i++) if (x[i] != x[i]) s = x[i];
            return;
        }
        float s0 = 0.f, s1 = 0.f, u0 = 0.f, u1 = 0.f;
        #pragma unroll
        for (int i = 0; i + 1 < N; i += 2) {
            float a = x[i], b = x[i + 1];
            ta::add2(a, b, -m, -m);
            ta::mul2(a, b, c, c);
            const float p = ex2(a), q = ex2(b);
            ta::add2(s0, s1, p, q);
            fma2(u0, u1, p, q, a, b);
        }
        if (N % 2) {
            const float a = (x[N - 1] - m) * c, p = ex2(a);
            s0 += p;
            u0 = fmaf(p, a, u0);
        }
        u0 += u1;
        if (u0 != u0) {                        // an element of -inf: 2^y is 0, and 0 is what it adds (a NaN stays one)
            u0 = 0.f;
            #pragma unroll
            for (int i = 0; i < N; i++) {
                const float a = max_nan((x[i] - m) * c, -200.0f);
                u0 = fmaf(ex2(a), a, u0);
            }
        }
        s += s0 + s1;
        u += u0;
    }
};

static_assert(kMaxCluster * kMaxTop <= kCand, "the blocks' likeliest are joined in one list");
// grid n_rows * cluster, kThreads threads, clusters of `cluster` blocks: rows one after the other.
template <int T>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(const Params P) {
    namespace cg = cooperative_groups;
    using E = Elem<T>;
    constexpr int kVec = E::kVec;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = (int)(blockIdx.x / blocks);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ unsigned long long cand[kCand];
    __shared__ unsigned long long best[kMaxTop];      // this block's likeliest, (ordered value, ~index); 0: none
    __shared__ float part[kWarps][3];
    __shared__ float sums[3];                         // this block's (m, S, U)
    __shared__ int chosen[kThreads], n_chosen, n_cand;
    __shared__ unsigned long long round_best[kWarps];

    // pieces of 16 bytes, this block's from v0 to v1; the loose elements before and behind them go to the first block
    const uint8_t* base = P.logits + (size_t)row * P.ld * E::kSize;
    const int head = min(P.vocab, (int)((16 - ((uintptr_t)base & 15)) & 15) / E::kSize), pieces = (P.vocab - head) / kVec;
    const int v0 = (int)((long long)pieces * rank / blocks), v1 = (int)((long long)pieces * (rank + 1) / blocks);
    const int loose = rank == 0 ? P.vocab - pieces * kVec : 0;
    auto loose_at = [&](int i) { return i < head ? i : pieces * kVec + i; };
    const uint4* vecs = reinterpret_cast<const uint4*>(base + (size_t)head * E::kSize);

    Sums a{-INFINITY, 0.f, 0.f};
    auto fetch = [&](int v, uint4 (&w)[kAhead]) {
        #pragma unroll
        for (int i = 0; i < kAhead; i++) if (v + i * kThreads < v1) w[i] = __ldg(vecs + v + i * kThreads);
    };
    uint4 next[kAhead];
    int v = v0 + tid;
    fetch(v, next);
    for (; v < v1; v += kAhead * kThreads) {
        uint4 w[kAhead];
        #pragma unroll
        for (int i = 0; i < kAhead; i++) w[i] = next[i];
        fetch(v + kAhead * kThreads, next);
        if (v + (kAhead - 1) * kThreads < v1) {
            float x[kAhead * kVec], vm = -INFINITY;
            #pragma unroll
            for (int i = 0; i < kAhead; i++) {
                float y[kVec];
                E::unpack(w[i], y);
                #pragma unroll
                for (int e = 0; e < kVec; e++) { x[i * kVec + e] = y[e]; vm = fmaxf(vm, y[e]); }
            }
            a.add(x, vm, P.c);
        } else {
            #pragma unroll
            for (int i = 0; i < kAhead; i++) {
                if (v + i * kThreads >= v1) break;
                float x[kVec];
                E::unpack(w[i], x);
                float vm = x[0];
                #pragma unroll
                for (int e = 1; e < kVec; e++) vm = fmaxf(vm, x[e]);
                a.add(x, vm, P.c);
            }
        }
    }
    if (tid < loose) {
        const float x[1] = {E::one(base + (size_t)loose_at(tid) * E::kSize)};
        a.add(x, x[0], P.c);
    }
    const float mine = a.m;                          // this thread's largest
    const bool some = v0 + tid < v1 || tid < loose;  // it has elements
    {
        const float wm = warp_max(a.m);
        if (lane == 0) part[warp][0] = wm;
        __syncthreads();
        float bm = part[0][0];
        #pragma unroll
        for (int i = 1; i < kWarps; i++) bm = fmaxf(bm, part[i][0]);
        if (a.m != -INFINITY) a.rise(bm, P.c);
        const float s = warp_sum(a.s), u = warp_sum(a.u);
        if (lane == 0) { part[warp][1] = s; part[warp][2] = u; }
        if (tid == 0) { n_chosen = 0; n_cand = 0; }
        if (tid < kMaxTop) best[tid] = 0;
        __syncthreads();
        if (warp == 0) {
            const float s2 = warp_sum(lane < kWarps ? part[lane][1] : 0.f), u2 = warp_sum(lane < kWarps ? part[lane][2] : 0.f);
            if (lane == 0) { sums[0] = bm; sums[1] = s2; sums[2] = u2; }
        }
        __syncthreads();
    }
    if (P.n_top > 0 && sums[1] == sums[1]) {         // (a row with a NaN or +inf has no likeliest)
        const uint32_t key = some ? ordered(mine) : 0u;
        uint32_t least = 0;                          // T: at least n_top threads (or all) have a largest >= T
        if (P.n_top == 1) {
            least = ordered(sums[0]);
        } else {
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                const int n = __syncthreads_count(key >= (least | bit));
                if (n >= P.n_top) least |= bit;
                if (n == P.n_top) break;
            }
        }
        if (key && key >= least) chosen[atomicAdd(&n_chosen, 1)] = tid;
        __syncthreads();
        auto add = [&](uint32_t k, int i) {
            if (*(volatile int*)&n_cand >= kCand) return;    // (full: the count says so)
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCand) cand[at] = (unsigned long long)k << 32 | (uint32_t)~i;
        };
        auto collect = [&](uint32_t from) {                  // the chosen threads' elements from there on
            for (int q = warp; q < n_chosen; q += kWarps) {
                const int t = chosen[q];
                for (int w = v0 + t + lane * kThreads; w < v1; w += 32 * kThreads) {
                    float x[kVec];
                    E::unpack(__ldg(vecs + w), x);
                    #pragma unroll
                    for (int e = 0; e < kVec; e++)
                        if (ordered(x[e]) >= from) add(ordered(x[e]), head + w * kVec + e);
                }
                if (lane == 0 && t < loose) {
                    const float x = E::one(base + (size_t)loose_at(t) * E::kSize);
                    if (ordered(x) >= from) add(ordered(x), loose_at(t));
                }
            }
            __syncthreads();
        };
        collect(least);
        bool listed = n_cand < kCand;
        if (!listed) {
            // Many equal logits, as where all but a few are -inf: those above T, and of those equal to it the first ones.
            __syncthreads();
            if (tid == 0) n_cand = 0;
            __syncthreads();
            collect(least + 1);
            listed = n_cand <= kCand - 32 * kVec - kMaxTop - 16;
            __syncthreads();
            if (listed && warp == 0) {
                if (lane < loose) {
                    const float x = E::one(base + (size_t)loose_at(lane) * E::kSize);
                    if (ordered(x) == least) add(least, loose_at(lane));
                }
                int equal = 0;
                for (int w0 = v0; w0 < v1 && equal < P.n_top; w0 += 32) {
                    int hits = 0;
                    if (w0 + lane < v1) {
                        float x[kVec];
                        E::unpack(__ldg(vecs + w0 + lane), x);
                        #pragma unroll
                        for (int e = 0; e < kVec; e++)
                            if (ordered(x[e]) == least) { add(least, head + (w0 + lane) * kVec + e); hits++; }
                    }
                    equal += __reduce_add_sync(~0u, hits);
                }
            }
            __syncthreads();
        }
        const int n = n_cand;
        if (listed) {
            for (int i = tid; i < n; i += kThreads) {
                const unsigned long long x = cand[i];
                int before = 0;
                for (int j = 0; j < n; j++) before += cand[j] > x;
                if (before < P.n_top) best[before] = x;
            }
            __syncthreads();
        } else {
            unsigned long long below = ~0ull;        // the last one taken
            for (int r = 0; r < P.n_top && below; r++) {
                unsigned long long top = 0;
                auto look = [&](float x, int i) {
                    const unsigned long long k = (unsigned long long)ordered(x) << 32 | (uint32_t)~i;
                    if (k < below && k > top) top = k;
                };
                for (int w = v0 + tid; w < v1; w += kThreads) {
                    float x[kVec];
                    E::unpack(__ldg(vecs + w), x);
                    #pragma unroll
                    for (int e = 0; e < kVec; e++) look(x[e], head + w * kVec + e);
                }
                if (tid < loose) look(E::one(base + (size_t)loose_at(tid) * E::kSize), loose_at(tid));
                #pragma unroll
                for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
                if (lane == 0) round_best[warp] = top;
                __syncthreads();
                top = round_best[0];
                for (int i = 1; i < kWarps; i++) top = max(top, round_best[i]);
                if (tid == 0) best[r] = top;
                below = top;
                __syncthreads();
            }
        }
    }
    cluster.sync();
    if (rank == 0) {
        __shared__ double joined[3];                 // m, S, U of the row
        if (warp == 0) {                             // lane b has block b's (m, S, U)
            Sums x{-INFINITY, 0.f, 0.f};
            if (lane < blocks) {
                const float* r = cluster.map_shared_rank(sums, lane);
                x = {r[0], r[1], r[2]};
            }
            const float m = warp_max(x.m);
            if (x.m != -INFINITY) x.rise(m, P.c);
            const float s = warp_sum(x.s), u = warp_sum(x.u);
            if (lane == 0) {
                const bool fine = s > 0 && m < INFINITY;  // (false for NaN)
                joined[0] = fine ? (double)m : NAN;
                joined[1] = fine ? log2((double)s) : NAN;
                joined[2] = fine ? (double)u / s : NAN;
            }
        }
        const int n = blocks * P.n_top;
        if (blocks > 1)
            for (int i = tid; i < n; i += kThreads) cand[i] = cluster.map_shared_rank(best, i / P.n_top)[i % P.n_top];
        __syncthreads();
        const double ln2 = 0.6931471805599453, m = joined[0], log_s = joined[1];
        const bool fine = m == m;
        auto logp = [&](float x) { return (float)(ln2 * (((double)x - m) * (double)P.c - log_s)); };
        if (tid == 0) {
            if (P.logprob) {
                const int t = P.tokens[row];
                P.logprob[row] = (unsigned)t < (unsigned)P.vocab ? logp(E::one(base + (size_t)t * E::kSize)) : NAN;
            }
            if (P.entropy) P.entropy[row] = (float)(ln2 * (log_s - joined[2]));
        }
        auto write = [&](int r, unsigned long long k) {
            const size_t at = (size_t)row * P.n_top + r;
            P.top_ids[at] = fine && k ? (int)~(uint32_t)k : -1;
            P.top_logprobs[at] = !fine ? NAN : k ? logp(unordered((uint32_t)(k >> 32))) : -INFINITY;
        };
        if (blocks > 1) {
            // ranked by counting; places that no block filled hold 0 and rank behind all
            for (int i = tid; i < n; i += kThreads) {
                const unsigned long long x = cand[i];
                int before = 0;
                for (int j = 0; j < n; j++) before += cand[j] > x || (cand[j] == x && j < i);
                if (before < P.n_top) write(before, x);
            }
        } else if (tid < P.n_top) {
            write(tid, best[tid]);
        }
    }
    cluster.sync();                                  // the other blocks' shared memory is read until here
}

}  // namespace lp
}  // namespace qb
