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
// One cluster of CTAs per sequence, every CTA a contiguous slice of the
// vocabulary, every warp a contiguous part of that.  Statistics that decide a
// comparison (largest logit, sum) are fp32 while nothing is refused; sums that
// the drawn token's position depends on (the running sum crosses a border for
// each of up to 10^5 tokens, so 24 bits would misplace about one draw in a
// hundred) are fp64.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qwen_b200.h"
#include "ptx.cuh"

namespace qb {
namespace tv {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxNodes = 64, kMaxCluster = 8;

struct Params {
    const void* logits;
    const float* draft;
    const int *tokens, *parents;
    const float* uniforms;
    int *path, *n_path, *next;
    long long ld, ld_draft;
    int n_nodes, vocab, vec;   // vec: rows of logits and draft start on 16 bytes
    float temperature;
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster(const void* local, uint32_t rank, uint64_t v) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(local)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

// What the CTAs of a cluster tell one another: two words each, two buffers in
// turn (a buffer is written again only after the next exchange's barrier).
struct Shared {
    uint64_t box[2][kMaxCluster][2];
    double wsum[kWarps];             // sums of rest over the warps' parts, of the last sum pass
    float wm[kWarps], wz[kWarps];
    int wi[kWarps], wf[kWarps];
    float lx[kMaxNodes], qx[kMaxNodes], u[kMaxNodes];
    int par[kMaxNodes], tok[kMaxNodes], gone[kMaxNodes];   // gone: refused tokens at this node (chosen drafts)
};

template <int T>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    if constexpr (T == QWEN_FP32) return __ldg((const float*)p + i);
    else if constexpr (T == QWEN_BF16) return bf2f(__ldg((const uint16_t*)p + i));
    else return __half2float(__ldg((const __half*)p + i));
}
// four consecutive values; past `end` they are `pad`
template <int T>
__device__ __forceinline__ void load4(const void* row, int i, int end, bool vec, float pad, float (&x)[4]) {
    if (vec && i + 4 <= end) {
        if constexpr (T == QWEN_FP32) {
            const float4 a = __ldg(reinterpret_cast<const float4*>((const float*)row + i));
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        } else {
            const uint2 a = __ldg(reinterpret_cast<const uint2*>((const uint16_t*)row + i));
            if constexpr (T == QWEN_BF16) {
                x[0] = bf_lo(a.x); x[1] = bf_hi(a.x); x[2] = bf_lo(a.y); x[3] = bf_hi(a.y);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a.x)), g = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
                x[0] = f.x; x[1] = f.y; x[2] = g.x; x[3] = g.y;
            }
        }
    } else {
        #pragma unroll
        for (int j = 0; j < 4; j++) x[j] = i + j < end ? load1<T>(row, i + j) : pad;
    }
}

// grid n_seqs * cluster CTAs, kThreads threads.
template <int T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const Params P) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank(), size = (int)cluster_size(), seq = blockIdx.x / size;
    const int N = P.n_nodes, V = P.vocab;
    const bool greedy = P.temperature == 0.0f, vec = P.vec != 0;
    // this warp's part of the vocabulary: whole runs of 128
    const int runs = (V + 127) / 128, parts = size * kWarps, mine = rank * kWarps + warp;
    const int lo = (int)((long long)runs * mine / parts) * 128, hi = min((int)((long long)runs * (mine + 1) / parts) * 128, V);

    if (tid < N) {
        sh.par[tid] = P.parents[(size_t)seq * N + tid];
        sh.tok[tid] = N > 1 ? P.tokens[(size_t)seq * N + tid] : 0;
        sh.u[tid] = greedy ? 0.f : P.uniforms[(size_t)seq * N + tid];
    }
    __syncthreads();
    int* path = P.path + (size_t)seq * N;
    if (rank == 0 && tid < N) path[tid] = -1;
    if (sh.par[0] != -1) {   // the same for the whole cluster
        if (rank == 0 && tid == 0) { P.n_path[seq] = 0; P.next[seq] = -1; }
        return;
    }
    __syncthreads();         // path's -1 before its entries (rank 0, thread 0 writes them)
    cluster_sync();          // every CTA runs before another writes to its box

    const float c32 = greedy ? 0.f : 1.4426950408889634f / P.temperature;
    const double it64 = greedy ? 0.0 : 1.0 / (double)P.temperature;
    int turn = 0;
    // every CTA's two words to every CTA; sh.box[result] then holds them by rank
    auto exchange = [&](uint64_t a, uint64_t b) {
        const int buf = turn & 1;
        turn++;
        if (tid < size) {
            st_cluster(&sh.box[buf][rank][0], tid, a);
            st_cluster(&sh.box[buf][rank][1], tid, b);
        }
        __syncwarp();
        cluster_sync();
        return buf;
    };

    int at = 0, count = 1;
    if (rank == 0 && tid == 0) path[0] = 0;
    for (;;) {
        const void* row = (const uint8_t*)P.logits + ((size_t)seq * N + at) * (size_t)P.ld * (T == QWEN_FP32 ? 4 : 2);
        const float* qrow = P.draft && !greedy ? P.draft + ((size_t)seq * N + at) * (size_t)P.ld_draft : nullptr;
        if (tid < N && tid > at && sh.par[tid] == at) {
            const int x = sh.tok[tid];
            const bool in = x >= 0 && x < V;
            sh.lx[tid] = in ? load1<T>(row, x) : -INFINITY;
            sh.qx[tid] = in && qrow ? __ldg(qrow + x) : 1.0f;
        }
        // ---- largest logit (its first place) and, unless greedy, the fp32 sum ----
        float m = -INFINITY, z = 0.f;
        int mi = INT_MAX, bad = 0;
        for (int i0 = lo; i0 < hi; i0 += 512) {
            float x[4][4];
            #pragma unroll
            for (int k = 0; k < 4; k++) load4<T>(row, i0 + 128 * k + 4 * lane, hi, vec, -INFINITY, x[k]);
            float m4 = m;
            #pragma unroll
            for (int k = 0; k < 4; k++)
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (x[k][j] > m4) { m4 = x[k][j]; mi = i0 + 128 * k + 4 * lane + j; }
                    bad |= x[k][j] != x[k][j];
                }
            if (!greedy && m4 > -INFINITY) {
                z *= exp2f((m - m4) * c32);
                #pragma unroll
                for (int k = 0; k < 4; k++)
                    #pragma unroll
                    for (int j = 0; j < 4; j++) z += exp2f((x[k][j] - m4) * c32);
            }
            m = m4;
        }
        auto join = [&](float m2, float z2, int i2) {
            const float mm = fmaxf(m, m2);
            if (mm > -INFINITY) z = (m > -INFINITY ? z * exp2f((m - mm) * c32) : 0.f) + (m2 > -INFINITY ? z2 * exp2f((m2 - mm) * c32) : 0.f);
            mi = m2 > m ? i2 : m2 == m ? min(mi, i2) : mi;
            m = mm;
        };
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(~0u, m, o), z2 = __shfl_xor_sync(~0u, z, o);
            const int i2 = __shfl_xor_sync(~0u, mi, o);
            join(m2, z2, i2);
        }
        bad = __any_sync(~0u, bad);
        if (lane == 0) { sh.wm[warp] = m; sh.wz[warp] = z; sh.wi[warp] = mi; sh.wf[warp] = bad; }
        __syncthreads();
        m = -INFINITY; z = 0.f; mi = INT_MAX; bad = 0;
        for (int w = 0; w < kWarps; w++) { join(sh.wm[w], sh.wz[w], sh.wi[w]); bad |= sh.wf[w]; }
        int buf = exchange((uint64_t)__float_as_uint(m) << 32 | __float_as_uint(z), (uint64_t)(uint32_t)mi << 32 | (uint32_t)bad);
        m = -INFINITY; z = 0.f; mi = INT_MAX; bad = 0;
        for (int r = 0; r < size; r++) {
            const uint64_t a = sh.box[buf][r][0], b = sh.box[buf][r][1];
            join(__uint_as_float((uint32_t)(a >> 32)), __uint_as_float((uint32_t)a), (int)(b >> 32));
            bad |= (int)(b & 1);
        }
        const float M = m;
        const bool none = bad || !(M > -INFINITY) || M == INFINITY;

        // ---- children in index order ----
        int kept = -1, n_gone = 0;
        double Z = z, left = 1.0, S = 0.0, total = 0.0;
        bool summed = false;
        // rest's sum over the vocabulary (fp64), unnormalised while S is 0; the warps' sums stay in sh.wsum
        auto weight = [&](float x, float q) {
            const double e = exp(((double)x - (double)M) * it64);
            return S > 0.0 ? fmax(e / Z - S * (double)q, 0.0) : e;
        };
        auto is_gone = [&](int i) {
            for (int g = 0; g < n_gone; g++) if (sh.gone[g] == i) return true;
            return false;
        };
        auto sum_pass = [&]() {
            double s = 0.0;
            bool any = false;
            for (int g = 0; g < n_gone; g++) any |= sh.gone[g] >= lo && sh.gone[g] < hi;
            for (int i0 = lo; i0 < hi; i0 += 256) {
                float x[2][4], q[2][4];
                #pragma unroll
                for (int k = 0; k < 2; k++) {
                    load4<T>(row, i0 + 128 * k + 4 * lane, hi, vec, -INFINITY, x[k]);
                    if (S > 0.0) load4<QWEN_FP32>(qrow, i0 + 128 * k + 4 * lane, hi, vec, 0.f, q[k]);
                }
                #pragma unroll
                for (int k = 0; k < 2; k++)
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int i = i0 + 128 * k + 4 * lane + j;
                        if (i < hi && !(any && is_gone(i))) s += weight(x[k][j], S > 0.0 ? q[k][j] : 0.f);
                    }
            }
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
            __syncthreads();   // readers of an earlier pass's wsum
            if (lane == 0) sh.wsum[warp] = s;
            __syncthreads();
            double cta = 0.0;
            for (int w = 0; w < kWarps; w++) cta += sh.wsum[w];
            buf = exchange((uint64_t)__double_as_longlong(cta), 0);
            double t = 0.0;
            for (int r = 0; r < size; r++) t += __longlong_as_double((long long)sh.box[buf][r][0]);
            return t;
        };
        for (int i = at + 1; i < N && kept < 0 && !none; i++) {
            if (sh.par[i] != at) continue;
            const int x = sh.tok[i];
            if (x < 0 || x >= V) continue;
            if (greedy) {
                if (x == mi) kept = i;
                continue;
            }
            const double p = exp(((double)sh.lx[i] - (double)M) * it64) / Z;
            const double q = sh.qx[i], rest = qrow ? fmax(p - S * q, 0.0) : is_gone(x) ? 0.0 : p;
            if ((double)sh.u[i] * left * q < rest) {
                kept = i;
            } else if (qrow) {
                if (!summed) Z = sum_pass();   // p to 64 bits from here on
                S += left;
                left = sum_pass();
                total = left;
                summed = true;
            } else if (!is_gone(x)) {
                left -= rest;
                __syncthreads();
                if (tid == 0) sh.gone[n_gone] = x;
                __syncthreads();
                n_gone++;
            }
        }
        if (kept >= 0) {
            at = kept;
            if (rank == 0 && tid == 0) path[count] = kept;
            count++;
            __syncthreads();   // lx, qx are rewritten
            continue;
        }
        // ---- no child is kept: the token after the path ----
        if (greedy || none) {
            if (rank == 0 && tid == 0) P.next[seq] = none ? -1 : mi;
            break;
        }
        if (!summed) total = sum_pass();
        if (!(total > 0.0)) {   // nothing is left: p itself
            S = 0.0;
            n_gone = 0;
            total = sum_pass();
        }
        // the part that the running sum crosses the target in, or else the last with any weight
        double target = (double)sh.u[0] * total;
        int owner = -1, last = 0;
        double before = 0.0, mine_before = 0.0;
        for (int r = 0; r < size; r++) {
            const double s = __longlong_as_double((long long)sh.box[buf][r][0]);
            if (s > 0.0) last = r;
            if (owner < 0 && before + s > target) { owner = r; mine_before = before; }
            before += s;
        }
        const bool over = owner < 0;
        if (over) owner = last;
        if (rank == owner) {
            int w = -1;
            last = 0;
            double run = over ? -INFINITY : mine_before;   // over: nothing crosses, the last weight is taken
            for (int k = 0; k < kWarps; k++) {
                if (sh.wsum[k] > 0.0) last = k;
                if (w < 0 && run + sh.wsum[k] > target) w = k;
                else if (w < 0) run += sh.wsum[k];
            }
            if (w < 0) { w = last; run = -INFINITY; }
            if (warp == w) {
                int found = -1, last_i = -1;
                for (int i0 = lo; i0 < hi && found < 0; i0 += 128) {
                    float x[4], q[4] = {0.f, 0.f, 0.f, 0.f};
                    double e[4];
                    load4<T>(row, i0 + 4 * lane, hi, vec, -INFINITY, x);
                    if (S > 0.0) load4<QWEN_FP32>(qrow, i0 + 4 * lane, hi, vec, 0.f, q);
                    double s = 0.0;
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int i = i0 + 4 * lane + j;
                        e[j] = i < hi && !is_gone(i) ? weight(x[j], q[j]) : 0.0;
                        if (e[j] > 0.0) last_i = i;
                        s += e[j];
                    }
                    double inc = s;
                    #pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double y = __shfl_up_sync(~0u, inc, o);
                        if (lane >= o) inc += y;
                    }
                    const uint32_t cross = __ballot_sync(~0u, run + inc > target);
                    if (cross) {
                        const int l = __ffs(cross) - 1;
                        int f = -1;
                        if (lane == l) {
                            double a = run + (inc - s);
                            #pragma unroll
                            for (int j = 0; j < 4; j++) {
                                a += e[j];
                                if (f < 0 && e[j] > 0.0 && a > target) f = i0 + 4 * lane + j;
                            }
                            if (f < 0) f = last_i;   // the rounding of inc - s
                        }
                        found = __shfl_sync(~0u, f, l);
                        if (found < 0) break;
                    }
                    run += __shfl_sync(~0u, inc, 31);
                }
                #pragma unroll
                for (int o = 16; o > 0; o >>= 1) last_i = max(last_i, __shfl_xor_sync(~0u, last_i, o));
                if (lane == 0) P.next[seq] = found >= 0 ? found : last_i;
            }
        }
        break;
    }
    if (rank == 0 && tid == 0) P.n_path[seq] = count;
    cluster_sync();   // no CTA leaves while another may still write to its box
}

}  // namespace tv
}  // namespace qb
