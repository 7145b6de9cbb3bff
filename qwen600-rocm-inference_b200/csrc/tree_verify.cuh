// tree_verify.cuh — which drafted tokens the target's probabilities keep, and
// the token after them (qwen_tree_verify).  No reference counterpart (the
// reference samples one token per forward, sampler.h:120-175).
//
// Mathematics.  At the reached node p = softmax(logits / T) is the target's
// distribution and q the drafter's.  A child with token x is kept with
// probability min(1, rest(x) / (left q(x))); after a refusal rest becomes
// max(rest - left q, 0) and left its sum.  Since max(max(p - S q, 0) - s q, 0) =
// max(p - (S + s) q, 0), the whole state is the one number S: rest = max(p - S q, 0),
// S grown by left at every refusal.  (Chosen drafts: q is 1 at the child's token,
// so rest is p without the refused tokens.)  Only the rows that the walk
// reaches are read.
//
// One cluster of CTAs per sequence, every warp a contiguous part of the
// vocabulary (whole runs of 128 tokens).  A level of the walk is a chain of
// latencies - the row's arrival, the largest logit and the sum, one exchange over
// the cluster - so a warp keeps its part of the row in shared memory where that
// fits, the first child's row is copied meanwhile (into a second buffer, or
// piece by piece over the row that is being read), and every warp's statistics go
// straight to every CTA through distributed shared memory: one cluster barrier a
// pass.
//
// Statistics that decide a comparison (largest logit, sum) are fp32 until a token with
// drafted probabilities, or most of the row's weight, is refused; then what is left is
// summed in fp64.  Sums that the drawn token's position depends on are fp64: the
// running sum crosses a border for each of up to 10^5 tokens, so 24 bits would misplace
// about one draw in a hundred.  Their powers of two are a polynomial of degree 8 in
// fp64, which interpolates 2^f at the nine Chebyshev nodes cos((2 k + 1) pi / 18) / 2
// of [-1/2, 1/2] (relative error 2^-39, 13 fp64 operations a token; a table of 256
// roots with three operations took as long, on bank conflicts).
//
// Measured on a vocabulary of 151,936 in fp32: a chain of 8 nodes of one
// sequence 21 us (greedy 7.6), 32 sequences with drafted probabilities 59 us (the
// rows that are reached and the last drafted rows are 13 us of memory traffic; the
// longest of the 32 walks is eight levels of 4.5 us: 2.6 us for a row's 38,000 tokens
// an SM, 1.3 us for the exchange).  Batches whose rows do not fit shared memory: 75
// sequences of 4 nodes 109 us of 18, 150 181 us of 37, a row's parts being read from
// the memory by one or two CTAs.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qwen_b200.h"
#include "ptx.cuh"

namespace qb {
namespace tv {

constexpr int kThreads = 512, kWarps = kThreads / 32, kRun = 128;
constexpr int kMaxNodes = 64, kMaxCluster = 16, kMaxParts = kMaxCluster * kWarps;

struct Params {
    const void* logits;
    const float* draft;
    const int *tokens, *parents;
    const float* uniforms;
    int *path, *n_path, *next;
    long long ld, ld_draft;
    int n_nodes, vocab, vec;   // vec: rows of logits and draft start on 16 bytes
    int buffers, part_bytes;   // row buffers in shared memory (0: parts do not fit), bytes of a warp's part (whole steps)
    int withheld;              // -1, or for failure tests a node: the last warp waits for 16 bytes of its row that never come
    unsigned long long wait_ns;   // longest wait for a copy from this GPU's own memory
    float temperature;
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster(const void* local, uint32_t rank, uint64_t v) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(local)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

// What the warps of a cluster tell one another: a word or two each, two buffers
// in turn (a buffer is written again only after the next exchange's barrier).
struct Shared {
    uint64_t box[2][kMaxParts];
    double run_sum[kWarps];          // the owner's second look: its runs' sums, last weighted tokens, the token
    int run_last[kWarps], found;
    uint64_t arrived[2][kWarps];     // a row buffer's bulk copies, per warp
    float lx[kMaxNodes], qx[kMaxNodes], u[kMaxNodes];
    int par[kMaxNodes], tok[kMaxNodes], gone[kMaxNodes];   // gone: refused tokens at this node (chosen drafts)
};

__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// a warp's largest value (no NaN), by the order of its bits as a whole number
__device__ __forceinline__ float max_lanes(float x) {
    const int b = __float_as_int(x);
    const int r = __reduce_max_sync(~0u, b < 0 ? b ^ 0x7fffffff : b);
    return __int_as_float(r < 0 ? r ^ 0x7fffffff : r);
}
__device__ __forceinline__ float sum_lanes(float x) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}
template <int T>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    if constexpr (T == QWEN_FP32) return __ldg((const float*)p + i);
    else if constexpr (T == QWEN_BF16) return bf2f(__ldg((const uint16_t*)p + i));
    else return __half2float(__ldg((const __half*)p + i));
}
// four values from 8 or 16 bytes
template <int T>
__device__ __forceinline__ void unpack4(const uint4& w, float (&x)[4]) {
    if constexpr (T == QWEN_FP32) {
        x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
    } else if constexpr (T == QWEN_BF16) {
        x[0] = bf_lo(w.x); x[1] = bf_hi(w.x); x[2] = bf_lo(w.y); x[3] = bf_hi(w.y);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), g = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        x[0] = f.x; x[1] = f.y; x[2] = g.x; x[3] = g.y;
    }
}
// four consecutive values of a row in global memory; past `end` they are `pad`
template <int T>
__device__ __forceinline__ void load4(const void* row, int i, int end, bool vec, float pad, float (&x)[4]) {
    if (vec && i + 4 <= end) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if constexpr (T == QWEN_FP32) {
            w = __ldg(reinterpret_cast<const uint4*>((const float*)row + i));
        } else {
            const uint2 a = __ldg(reinterpret_cast<const uint2*>((const uint16_t*)row + i));
            w.x = a.x; w.y = a.y;
        }
        unpack4<T>(w, x);
    } else {
        #pragma unroll
        for (int j = 0; j < 4; j++) x[j] = i + j < end ? load1<T>(row, i + j) : pad;
    }
}

// grid n_seqs * cluster CTAs, kThreads threads, buffers * kWarps * part_bytes of
// dynamic shared memory.  HELD: parts are held in row buffers (P.buffers > 0).
template <int T, bool HELD>
__global__ void __launch_bounds__(kThreads) verify_kernel(const Params P) {
    constexpr int K = HELD ? 2 : 4;   // runs of a step: 4 K tokens a lane
    constexpr int kEs = T == QWEN_FP32 ? 4 : 2;
    __shared__ Shared sh;
    extern __shared__ __align__(16) uint8_t parts_mem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank(), size = (int)cluster_size(), seq = blockIdx.x / size;
    const int N = P.n_nodes, V = P.vocab;
    const bool greedy = P.temperature == 0.0f, vec = P.vec != 0;
    // this warp's part of the vocabulary
    const int runs = (V + kRun - 1) / kRun, parts = size * kWarps, mine = rank * kWarps + warp;
    const int r0 = (int)((long long)runs * mine / parts), r1 = (int)((long long)runs * (mine + 1) / parts);
    const int lo = r0 * kRun, hi = min(r1 * kRun, V);

    auto row_of = [&](int node) { return (const uint8_t*)P.logits + ((size_t)seq * N + node) * (size_t)P.ld * kEs; };
    if (lane == 0) {
        mbar_init(&sh.arrived[0][warp], 1);
        mbar_init(&sh.arrived[1][warp], 1);
        fence_barrier_init();
    }
    __syncwarp();
    // Tokens from .. to-1 (from: a whole run) of this warp's part of a node's row into buffer b: by bulk copies, which take no
    // issue slots from the arithmetic, where rows start on 16 bytes.  first: the first piece of the part.
    // (Evicted first from the L2: the rows are dead afterwards.  With them at the highest or the ordinary priority the verification
    // takes as long, 59.5 us against 58.5 with 32 x 8, and a kernel that reads 50 MB behind it 19.6 us against 14.9.)
    uint32_t phase = 0;      // bit b: the parity that buffer b's next part completes
    uint32_t coming = 0;     // bit b: a part is on its way
    bool late = false;       // a wait ran out (the same for the warp): nothing is copied from then on
    auto fetch = [&](int node, int b, int from, int to, bool first) {
        if (late) return;
        uint8_t* dst = parts_mem + (size_t)(b * kWarps + warp) * P.part_bytes;
        const uint8_t* row = row_of(node);
        int k = from;        // tokens from here on are copied one by one
        if (vec) {
            const uint32_t n = (uint32_t)((to - from) * kEs) & ~15u, all = (uint32_t)((hi - lo) * kEs) & ~15u;
            if (lane == 0) {
                if (first && all) mbar_arrive_expect_tx(&sh.arrived[b][warp], all + (node == P.withheld && mine == parts - 1 ? 16u : 0u));
                if (n) bulk_g2s(dst + (size_t)(from - lo) * kEs, row + (size_t)from * kEs, n, &sh.arrived[b][warp], policy_evict_first());
            }
            if (all) coming |= 1u << b;
            k = from + (int)(n / kEs);
        }
        for (k += lane; k < to; k += 32) {
            if constexpr (kEs == 4) reinterpret_cast<float*>(dst)[k - lo] = __ldg((const float*)row + k);
            else reinterpret_cast<uint16_t*>(dst)[k - lo] = __ldg((const uint16_t*)row + k);
        }
    };
    // Waits for buffer b's part; a wait that runs out marks the warp, whose word to the others then is NaN or +inf (next = -1).
    // The part stays on its way: the kernel's end waits for it once more, and no other copy goes into its buffer.
    auto landed = [&](int b) {
        if (coming >> b & 1) {
            if (__all_sync(~0u, mbar_wait(&sh.arrived[b][warp], phase >> b & 1, P.wait_ns))) {
                phase ^= 1u << b;
                coming &= ~(1u << b);
            } else {
                late = true;
            }
        }
        __syncwarp();
    };
    if constexpr (HELD) {
        fetch(0, 0, lo, hi, true);
        // behind the part's end: -inf up to a whole step
        for (int b = 0; b < P.buffers; b++) {
            uint8_t* dst = parts_mem + (size_t)(b * kWarps + warp) * P.part_bytes;
            for (int k = hi - lo + lane; k < P.part_bytes / kEs; k += 32) {
                if constexpr (T == QWEN_FP32) reinterpret_cast<float*>(dst)[k] = -INFINITY;
                else reinterpret_cast<uint16_t*>(dst)[k] = T == QWEN_BF16 ? 0xff80 : 0xfc00;
            }
        }
    }

    if (tid < N) {
        sh.par[tid] = P.parents[(size_t)seq * N + tid];
        sh.tok[tid] = N > 1 ? P.tokens[(size_t)seq * N + tid] : 0;
        sh.u[tid] = greedy ? 0.f : P.uniforms[(size_t)seq * N + tid];
    }
    if (tid == 0) sh.found = INT_MAX;
    int* path = P.path + (size_t)seq * N;
    if (rank == 0 && tid < N) path[tid] = -1;
    __syncthreads();         // (path's -1 come before its entries)
    if (sh.par[0] != -1) {   // the same for the whole cluster
        if (rank == 0 && tid == 0) { P.n_path[seq] = 0; P.next[seq] = -1; }
        if constexpr (HELD) landed(0);
        return;
    }
    // every node's logit (and drafted probability) in its parent's row
    if (tid < N && !greedy) {
        const int up = sh.par[tid], x = sh.tok[tid];
        const bool in = up >= 0 && up < tid && x >= 0 && x < V;
        sh.lx[tid] = in ? load1<T>(row_of(up), x) : -INFINITY;
        sh.qx[tid] = in && P.draft ? __ldg(P.draft + ((size_t)seq * N + up) * (size_t)P.ld_draft + x) : 1.0f;
    }
    cluster_sync();          // every CTA runs before another writes to its box

    const float c32 = greedy ? 0.f : 1.4426950408889634f / P.temperature;
    const double c64 = greedy ? 1.0 : 1.4426950408889634074 / (double)P.temperature;
    const unsigned dmin = (unsigned)__double2hiint(-1000.0 / c64);   // high word of the lowest x - M that counts
    int turn = 0, held = 0;  // held: the buffer with the reached node's row
    int other = -1;          // two buffers: the node whose row is on its way into the second
    int inside = 0;          // one buffer: the node whose row it holds or receives

    int at = 0, count = 1;
    if (rank == 0 && tid == 0) path[0] = 0;
    for (;;) {
        const uint8_t* row = row_of(at);
        const float* qrow = P.draft && !greedy ? P.draft + ((size_t)seq * N + at) * (size_t)P.ld_draft : nullptr;
        // the children, and the first of them
        uint64_t children = __ballot_sync(~0u, lane > at && lane < N && sh.par[lane] == at) |
                            (uint64_t)__ballot_sync(~0u, lane + 32 > at && lane + 32 < N && sh.par[lane + 32] == at) << 32;
        const int child = __ffsll((long long)children) - 1;
        const bool next_row = child >= 0;
        if constexpr (HELD) {
            landed(held);
            if (next_row && P.buffers == 2) {
                landed(held ^ 1);
                fetch(child, held ^ 1, lo, hi, true);
                other = child;
            }
        } else if (next_row && vec && hi > lo) {   // as far as the L2
            const int n = (hi - lo) * kEs & ~15;
            if (lane == 0 && n) bulk_prefetch_l2(row_of(child) + (size_t)lo * kEs, n);
        }
        const uint8_t* part = parts_mem + (size_t)(held * kWarps + warp) * P.part_bytes;
        // one step's logits: runs i0 / kRun .., tokens i0 + kRun k + 4 lane + j at x[4 k + j]; -inf past the end
        auto step = [&](int i0, auto& x) {
            #pragma unroll
            for (int k = 0; k < (int)sizeof(x) / 16; k++) {
                float y[4];
                if constexpr (HELD) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    const uint8_t* p = part + (size_t)(i0 - lo + kRun * k + 4 * lane) * kEs;
                    if constexpr (kEs == 4) {
                        w = *reinterpret_cast<const uint4*>(p);
                    } else {
                        const uint2 a = *reinterpret_cast<const uint2*>(p);
                        w.x = a.x; w.y = a.y;
                    }
                    unpack4<T>(w, y);
                } else {
                    load4<T>(row, i0 + kRun * k + 4 * lane, hi, vec, -INFINITY, y);
                }
                #pragma unroll
                for (int j = 0; j < 4; j++) x[4 * k + j] = y[j];
            }
        };
        // ---- largest logit (its first place) and, unless greedy, the fp32 sum ----
        float m = -INFINITY, z = 0.f;
        int mi = INT_MAX, bad = 0;
        for (int i0 = lo; i0 < hi; i0 += K * kRun) {
            float x[4 * K];
            step(i0, x);
            if (greedy) {
                #pragma unroll
                for (int j = 0; j < 4 * K; j++) {
                    if (x[j] > m) { m = x[j]; mi = i0 + kRun * (j >> 2) + 4 * lane + (j & 3); }
                    bad |= x[j] != x[j];
                }
            } else {             // (a NaN makes z NaN; before any logit above -inf z stays 0)
                float t[4 * K];
                #pragma unroll
                for (int j = 0; j < 4 * K; j++) t[j] = x[j];
                #pragma unroll
                for (int o = 2 * K; o > 0; o >>= 1)
                    #pragma unroll
                    for (int j = 0; j < o; j++) t[j] = fmaxf(t[j], t[j + o]);
                const float top = fmaxf(m, t[0]), from = top > -INFINITY ? top : 0.f;
                #pragma unroll
                for (int j = 0; j < 4 * K; j++) t[j] = exp2_ftz((x[j] - from) * c32);
                #pragma unroll
                for (int o = 2 * K; o > 0; o >>= 1)
                    #pragma unroll
                    for (int j = 0; j < o; j++) t[j] += t[j + o];
                z = fmaf(z, exp2_ftz((m - from) * c32), t[0]);
                m = top;
            }
            // one buffer: the next row over what has been read, in pieces of four steps (smaller ones cost more to issue)
            if (HELD && next_row && P.buffers == 1 && (((i0 - lo) / (K * kRun) & 3) == 3 || i0 + K * kRun >= hi)) {
                const int piece = i0 - ((i0 - lo) / (K * kRun) & 3) * (K * kRun);
                __syncwarp();
                fetch(child, 0, piece, min(i0 + K * kRun, hi), piece == lo);
            }
        }
        if (HELD && next_row && P.buffers == 1) inside = child;
        if (!greedy) bad = z != z;
        // the warp's, then the cluster's: the largest first, then the sums on its scale.  A warp that met a NaN says +inf.
        float M = max_lanes(__any_sync(~0u, bad || late) ? INFINITY : m);
        {
            uint64_t* box = sh.box[turn & 1];
            turn++;
            uint32_t low;
            if (greedy) low = __reduce_min_sync(~0u, m == M ? mi : INT_MAX);
            else low = __float_as_uint(sum_lanes(m > -INFINITY && M < INFINITY ? z * exp2_ftz((m - M) * c32) : 0.f));
            if (lane < size) st_cluster(box + mine, lane, (uint64_t)__float_as_uint(M) << 32 | low);
            cluster_sync();
            uint64_t w[kMaxParts / 32];
            m = -INFINITY;
            #pragma unroll
            for (int k = 0; k < kMaxParts / 32; k++) {
                w[k] = lane + 32 * k < parts ? box[lane + 32 * k] : 0xff80000000000000ull;   // -inf
                m = fmaxf(m, __uint_as_float((uint32_t)(w[k] >> 32)));
            }
            M = max_lanes(m);
            z = 0.f;
            mi = INT_MAX;
            #pragma unroll
            for (int k = 0; k < kMaxParts / 32; k++) {
                const float mk = __uint_as_float((uint32_t)(w[k] >> 32));
                if (greedy) { if (mk == M) mi = min(mi, (int)(uint32_t)w[k]); }
                else if (mk > -INFINITY) z += __uint_as_float((uint32_t)w[k]) * exp2_ftz((mk - M) * c32);
            }
            if (greedy) mi = __reduce_min_sync(~0u, mi);
            else z = sum_lanes(z);
        }
        const bool none = !(M > -INFINITY) || M == INFINITY;

        // ---- children in index order ----
        int kept = -1, n_gone = 0;
        // left, S and rest are the row's sum times those of the walk's definition; low: where what is left must be summed anew
        double left = z, low = 0.0625 * left, S = 0.0;
        bool summed = false;     // left is the last sum pass's
        const double M64 = M;
        // weights 2^(c (x - M)) = 2^n 2^f, |f| <= 1/2, of K tokens; in[j]: the weight counts (not below 2^-1000).  The steps go
        // over all K in turn, so that each fp64 operation finds the others' in the pipe
        auto powers = [&](const auto& x, auto& e, auto& in) {
            constexpr int K = sizeof(x) / sizeof(float);
            double d[K], f[K];
            int n[K];
            #pragma unroll
            for (int j = 0; j < K; j++) d[j] = (double)x[j] - M64;
            #pragma unroll
            for (int j = 0; j < K; j++) f[j] = fma(d[j], c64, 6755399441055744.0);   // + 1.5 * 2^52: the nearest whole number in the low word
            #pragma unroll
            for (int j = 0; j < K; j++) { n[j] = __double2loint(f[j]); f[j] -= 6755399441055744.0; }
            #pragma unroll
            for (int j = 0; j < K; j++) f[j] = fma(d[j], c64, -f[j]);
            constexpr double kC[8] = {1.5310079402249296e-05, 1.5403455852453838e-04, 1.3333450568000645e-03, 9.618129159402558e-03,
                                      5.550410941205933e-02, 2.402265069581299e-01, 6.931471805459335e-01, 1.0};
            #pragma unroll
            for (int j = 0; j < K; j++) e[j] = fma(f[j], 1.3255224878668817e-06, kC[0]);
            #pragma unroll
            for (int i = 1; i < 8; i++)
                #pragma unroll
                for (int j = 0; j < K; j++) e[j] = fma(f[j], e[j], kC[i]);
            #pragma unroll
            for (int j = 0; j < K; j++) {
                e[j] = __hiloint2double(__double2hiint(e[j]) + (n[j] << 20), __double2loint(e[j]));
                in[j] = (unsigned)__double2hiint(d[j]) < dmin;   // d > -1000 / c by its high word (d is 0 or negative)
            }
        };
        auto power = [&](float x) {
            const float a[1] = {x};
            double e[1];
            bool in[1];
            powers(a, e, in);
            return in[0] ? e[0] : 0.0;
        };
        // what is left of the tokens' weights, where in[j] (S > 0: with draft)
        auto weights = [&](const auto& x, const auto& q, auto& e, auto& in) {
            powers(x, e, in);
            if (S > 0.0) {
                #pragma unroll
                for (int j = 0; j < (int)(sizeof(x) / sizeof(float)); j++) {
                    e[j] = fma(-S, (double)q[j], e[j]);
                    in[j] = in[j] && __double2hiint(e[j]) >= 0;
                }
            }
        };
        auto is_gone = [&](int i) {
            for (int g = 0; g < n_gone; g++) if (sh.gone[g] == i) return true;
            return false;
        };
        // of the last sum pass: the parts' sums of rest, lane * per .. of them this lane's; their sum and the running sum
        const uint64_t* sums = nullptr;
        const int per = (parts + 31) / 32;
        double lane_sum = 0.0, lane_run = 0.0;
        auto sum_pass = [&]() {
            if (HELD && P.buffers == 1 && inside != at) {
                landed(0);
                fetch(at, 0, lo, hi, true);
                landed(0);
                inside = at;
            }
            double sum[8] = {};
            bool any = false;
            for (int g = 0; g < n_gone; g++) any |= sh.gone[g] >= lo && sh.gone[g] < hi;
            auto add = [&](int i0, auto& x) {   // the step of sizeof(x) / 16 runs
                constexpr int kN = sizeof(x) / 4;
                float q[kN];
                double e[kN];
                bool in[kN];
                step(i0, x);
                if (S > 0.0) {
                    #pragma unroll
                    for (int k = 0; k < kN / 4; k++) {
                        float y[4];
                        load4<QWEN_FP32>(qrow, i0 + kRun * k + 4 * lane, hi, vec, 0.f, y);
                        #pragma unroll
                        for (int j = 0; j < 4; j++) q[4 * k + j] = y[j];
                    }
                }
                weights(x, q, e, in);
                if (any) {
                    #pragma unroll
                    for (int j = 0; j < kN; j++) if (is_gone(i0 + kRun * (j >> 2) + 4 * lane + (j & 3))) in[j] = false;
                }
                #pragma unroll
                for (int j = 0; j < kN; j++) if (in[j]) sum[j] += e[j];
            };
            int i0 = lo;
            for (; i0 + kRun < hi; i0 += 2 * kRun) { float x[8]; add(i0, x); }
            if (i0 < hi) { float x[4]; add(i0, x); }
            double s = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
            uint64_t* box = sh.box[turn & 1];
            turn++;
            if (lane < size) st_cluster(box + mine, lane, (uint64_t)__double_as_longlong(late ? NAN : s));
            cluster_sync();
            double t[kMaxParts / 32];
            #pragma unroll
            for (int k = 0; k < kMaxParts / 32; k++)
                t[k] = k < per && lane * per + k < parts ? __longlong_as_double((long long)box[lane * per + k]) : 0.0;
            #pragma unroll
            for (int o = kMaxParts / 64; o > 0; o >>= 1)
                #pragma unroll
                for (int k = 0; k < o; k++) t[k] += t[k + o];
            lane_sum = lane_run = t[0];
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(~0u, lane_run, o);
                if (lane >= o) lane_run += y;
            }
            sums = box;
            return __shfl_sync(~0u, lane_run, 31);
        };
        for (; children && kept < 0 && !none; children &= children - 1) {
            const int i = __ffsll((long long)children) - 1, x = sh.tok[i];
            if (x < 0 || x >= V) continue;
            if (greedy) {
                if (x == mi) kept = i;
                continue;
            }
            const double e = power(sh.lx[i]), q = sh.qx[i];
            const double rest = qrow ? fmax(fma(-S, q, e), 0.0) : is_gone(x) ? 0.0 : e;
            if ((double)sh.u[i] * left * q < rest) {
                kept = i;
            } else if (qrow) {
                if (!summed) left = sum_pass();   // to 64 bits from here on
                S += left;
                left = sum_pass();
                summed = true;
            } else if (!is_gone(x)) {
                left -= rest;
                __syncthreads();
                if (tid == 0) sh.gone[n_gone] = x;
                __syncthreads();
                n_gone++;
                summed = false;
                // Little is left, and the next child is compared with it: not with a difference of an fp32 sum, which is off by about
                // 2^-21 (2^-17 of a sixteenth of it), but with a sum in fp64.  (That is off by 2^-39: differences of it last longer.)
                if ((children & (children - 1)) && left < low) {
                    left = sum_pass();
                    low = 0x1p-16 * left;
                    summed = true;
                }
            }
        }
        if (kept >= 0) {
            at = kept;
            if (rank == 0 && tid == 0) path[count] = kept;
            count++;
            if (HELD && P.buffers == 2 && kept == other) {
                held ^= 1;
            } else if (HELD && (P.buffers == 2 || kept != inside)) {
                landed(held);
                fetch(kept, held, lo, hi, true);
                inside = kept;
            }
            other = -1;
            continue;
        }
        // ---- no child is kept: the token after the path ----
        if (greedy || none) {
            if (rank == 0 && tid == 0) P.next[seq] = none ? -1 : mi;
            break;
        }
        double total = summed ? left : sum_pass();
        if (!(total > 0.0)) {   // nothing is left: p itself
            S = 0.0;
            n_gone = 0;
            total = sum_pass();
        }
        if (!(total > 0.0)) {   // (a wait that ran out)
            if (rank == 0 && tid == 0) P.next[seq] = -1;
            break;
        }
        // the part in which the running sum crosses the target, or else the last one with any weight
        const double target = (double)sh.u[0] * total;
        const uint32_t some = __ballot_sync(~0u, lane_sum > 0.0), cross = __ballot_sync(~0u, lane_sum > 0.0 && lane_run > target);
        const bool over = cross == 0;              // nothing crosses: the last token with any weight
        const int at_lane = over ? 31 - __clz(some) : __ffs(cross) - 1;
        int owner = -1;
        double run = lane_run - lane_sum;          // the sum before the owner's part
        if (lane == at_lane) {
            double before = run;
            for (int k = 0; k < per && lane * per + k < parts; k++) {
                const double w = __longlong_as_double((long long)sums[lane * per + k]);
                if (w > 0.0) {
                    owner = lane * per + k;
                    run = before;
                    if (!over && before + w > target) break;
                }
                before += w;
            }
        }
        owner = __shfl_sync(~0u, owner, at_lane);
        run = __shfl_sync(~0u, run, at_lane);
        if (owner / kWarps == rank) {
            // the CTA's warps share the owner's part: run k of each round of kWarps runs
            const int o0 = (int)((long long)runs * owner / parts) * kRun, o1 = min((int)((long long)runs * (owner + 1) / parts) * kRun, V);
            const uint8_t* opart = parts_mem + (size_t)(held * kWarps + owner % kWarps) * P.part_bytes;
            int best = -1;             // the last token with any weight
            bool done = false;
            for (int b = o0; b < o1 && !done; b += kWarps * kRun) {
                const int i = b + warp * kRun + 4 * lane;
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, q[4] = {0.f, 0.f, 0.f, 0.f};
                if constexpr (HELD) {
                    #pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (i + j < o1) {
                            if constexpr (T == QWEN_FP32) x[j] = reinterpret_cast<const float*>(opart)[i + j - o0];
                            else if constexpr (T == QWEN_BF16) x[j] = bf2f(reinterpret_cast<const uint16_t*>(opart)[i + j - o0]);
                            else x[j] = __half2float(reinterpret_cast<const __half*>(opart)[i + j - o0]);
                        }
                } else {
                    load4<T>(row, i, o1, vec, -INFINITY, x);
                }
                if (S > 0.0) load4<QWEN_FP32>(qrow, i, o1, vec, 0.f, q);
                double e[4], s = 0.0;
                bool in[4];
                int mine_last = -1;
                weights(x, q, e, in);
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (!in[j] || i + j >= o1 || is_gone(i + j)) e[j] = 0.0;
                    if (e[j] > 0.0) mine_last = i + j;
                    s += e[j];
                }
                double inc = s;
                #pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(~0u, inc, o);
                    if (lane >= o) inc += y;
                }
                const int warp_last = __reduce_max_sync(~0u, mine_last);
                if (lane == 31) { sh.run_sum[warp] = inc; sh.run_last[warp] = warp_last; }
                __syncthreads();
                // the sums before this warp's run and behind the round (the same additions in every warp)
                double upto = lane < kWarps ? sh.run_sum[lane] : 0.0;
                best = max(best, __reduce_max_sync(~0u, lane < kWarps ? sh.run_last[lane] : -1));
                #pragma unroll
                for (int o = 1; o < kWarps; o <<= 1) {
                    const double y = __shfl_up_sync(~0u, upto, o);
                    if (lane >= o) upto += y;
                }
                const double behind = __shfl_sync(~0u, upto, (warp + 31) & 31), round = __shfl_sync(~0u, upto, kWarps - 1);
                const double before = run + (warp ? behind : 0.0);
                if (!over) {
                    const uint32_t cross = __ballot_sync(~0u, s > 0.0 && before + inc > target);
                    if (cross && lane == __ffs(cross) - 1) {
                        double a = before + (inc - s);
                        int f = -1;
                        #pragma unroll
                        for (int j = 0; j < 4; j++) {
                            a += e[j];
                            if (f < 0 && e[j] > 0.0 && a > target) f = i + j;
                        }
                        atomicMin(&sh.found, f >= 0 ? f : mine_last);   // (the rounding of inc - s)
                    }
                }
                run += round;
                __syncthreads();
                done = sh.found != INT_MAX;   // (the next round's first barrier comes before another write)
            }
            if (tid == 0) P.next[seq] = sh.found != INT_MAX ? sh.found : best;
        }
        break;
    }
    if (rank == 0 && tid == 0) P.n_path[seq] = count;
    if constexpr (HELD) {
        landed(0);
        landed(1);
    }
    // (a CTA's last writes to another's box came before a cluster barrier that both have passed)
}

}  // namespace tv
}  // namespace qb
