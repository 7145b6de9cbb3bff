// kv_pages.cuh — a K/V cache in pages as the kernels take it, and the pass that
// fills it: norms of query and key heads, rotation, rows to their pages
// (qwen_qk_rope).  No reference counterpart (the reference norms, rotates and
// stores one token of a contiguous bf16 cache in three kernels,
// qwen_model.cuh:253-347).
//
// Mathematics.  A head x of D values becomes y = x / sqrt(mean x^2 + eps) * gain,
// and the pairs (y_j, y_(j + D/2)) turn by a_j = position * base^(-2 j / D).  A turn
// is 2^64 units: F_j = base^(-2 j / D) / (2 pi) in units is made once on the host in
// extended precision, position * F_j wraps by itself, and what is left is the angle
// modulo a turn to 2^-64 turns times the position.  So no position is too far, and
// the cosine's argument is one conversion away.
//
// Bound by memory traffic and the instructions around it where there are many rows (8192 tokens, 16 + 8 + 8 heads of
// 128 in bf16, K to rows and pages: 34 us, 4.5 TB/s, floor 23), by the chain of loads (position,
// table, rows) where there are few (128 tokens 3.7 us).  Into 8-bit pages 64 us (e4m3) and 55 us (int8; floor
// 21).  A block takes up to 8 tokens: their sines and
// cosines go through shared memory once for all heads, then D / 16 threads take a head
// at a time, 8 values of either half each, so pairs meet in one thread, the mean needs
// 3 or 2 shuffles and every access is a 16-byte piece of a row.  A thread keeps its head for the block's tokens and
// loads a row ahead; with a division and a search for its place at every row it took 40 us.
#pragma once
#include "kv_rows.cuh"

namespace qb {
namespace pg {

struct Pages {
    uint8_t *k, *v;
    float *ks, *vs;
    const int* table;
    long long page_stride, head_stride;   // elements
    int n_pages, n_seqs, max_pages, shift;  // page_size = 1 << shift
    // the page that position p (>= 0) of sequence s lies in, -1: it is not there
    __device__ __forceinline__ int page_of(int s, int p) const {
        const int at = p >> shift;
        if ((unsigned)s >= (unsigned)n_seqs || at >= max_pages) return -1;
        const int page = __ldg(table + (size_t)s * max_pages + at);
        return (unsigned)page < (unsigned)n_pages ? page : -1;
    }
};

constexpr int kRopeThreads = 256, kRopeTokens = 8;   // tokens of a block at most

struct RopeParams {
    const uint8_t *q, *k, *v;
    long long ldq, ldk, ldv, ldqo, ldko;
    const uint8_t *q_gain, *k_gain;
    const int *positions, *seqs;
    uint8_t *q_out, *k_out;
    Pages pages;
    int n_rows, n_heads, n_kv_heads, gain_type, out_type, store, tokens;   // store: the pages' type, -1: no pages
    float eps;
    unsigned long long turn[64];   // F_j
};

__device__ __forceinline__ float one_value(const uint8_t* p, int type, int i) {
    if (type == QWEN_FP32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t w = reinterpret_cast<const uint16_t*>(p)[i];
    return type == QWEN_BF16 ? bf2f(w) : __half2float(__ushort_as_half(w));
}
// 8 consecutive values, rounded to the type
__device__ __forceinline__ void store8(uint8_t* p, int type, const float* x) {
    if (type == QWEN_FP32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) w[i] = type == QWEN_BF16 ? cvt_bf16x2(x[2 * i], x[2 * i + 1]) : kv::half2_bits(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// One head's row to its page: this thread's 8 values of either half, the row's threads together.
template <int D, bool Q8>
__device__ __forceinline__ void to_page(const RopeParams& P, bool value, int page, int row, int h, int part, const float (&x)[16]) {
    const size_t at = (size_t)page * P.pages.page_stride + (size_t)h * P.pages.head_stride + (size_t)row * D;
    uint8_t* base = value ? P.pages.v : P.pages.k;
    if constexpr (!Q8) {
        if (page < 0) return;
        store8(base + (at + part * 8) * 2, P.store, x);
        store8(base + (at + D / 2 + part * 8) * 2, P.store, x + 8);
        return;
    }
    uint32_t m = 0;   // magnitudes as bit patterns: NaN above infinity above every number
    #pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    #pragma unroll
    for (int o = 1; o < D / 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (page < 0) return;
    const bool finite = m < 0x7f800000u, e4 = P.store == QWEN_E4M3;
    const float a = fmaxf(__uint_as_float(m), kv::kMinAmax);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (finite) w = e4 ? kv::encode16<QWEN_FP32, QWEN_E4M3>(x, a) : kv::encode16<QWEN_FP32, QWEN_INT8>(x, a);
    *reinterpret_cast<uint2*>(base + at + part * 8) = make_uint2(w.x, w.y);
    *reinterpret_cast<uint2*>(base + at + D / 2 + part * 8) = make_uint2(w.z, w.w);
    if (part == 0) (value ? P.pages.vs : P.pages.ks)[at / D] = finite ? a / (e4 ? 448.0f : 127.0f) : __uint_as_float(0x7fffffffu);
}

// grid ceil(n_rows / tokens), kRopeThreads threads.
template <int SRC, int D, bool Q8>   // Q8: 8-bit pages
__global__ void __launch_bounds__(kRopeThreads, Q8 || SRC == QWEN_FP32 ? 3 : 4) qk_rope_kernel(const __grid_constant__ RopeParams P) {
    constexpr int kLanes = D / 16, kGroups = kRopeThreads / kLanes, kEs = SRC == QWEN_FP32 ? 4 : 2, kN = SRC == QWEN_FP32 ? 2 : 1;
    __shared__ __align__(16) float cosine[kRopeTokens][D / 2], sine[kRopeTokens][D / 2], gains[2][D];
    __shared__ int page_at[kRopeTokens], row_at[kRopeTokens];   // row_at: -1 where the token is left out
    const int tid = threadIdx.x, first = blockIdx.x * P.tokens, tokens = min(P.tokens, P.n_rows - first);
    const bool paged = P.store >= 0;
    for (int i = tid; i < tokens * (D / 2); i += kRopeThreads) {
        const int t = i / (D / 2), j = i % (D / 2), p = P.positions[first + t];
        const long long turns = (long long)((unsigned long long)(unsigned)max(p, 0) * P.turn[j]);
        float s, c;
        sincospif((float)turns * 0x1p-63f, &s, &c);   // half turns, -1 .. 1
        cosine[t][j] = c;
        sine[t][j] = s;
        if (j == 0) {
            row_at[t] = p < 0 ? -1 : paged ? p & ((1 << P.pages.shift) - 1) : 0;
            page_at[t] = paged && p >= 0 ? P.pages.page_of(P.seqs[first + t], p) : -1;
        }
    }
    if (P.q_gain) for (int i = tid; i < 2 * D; i += kRopeThreads) gains[i / D][i % D] = one_value(i < D ? P.q_gain : P.k_gain, P.gain_type, i % D);
    __syncthreads();
    const int part = tid % kLanes, per = P.n_heads + (paged ? 2 : 1) * P.n_kv_heads;
    // A thread keeps its head for all of its tokens; where a token's rows are fewer than the threads' groups, several tokens go side by side.
    // (A warp's threads stay together: they shuffle.)
    const int beside = max(kGroups / per, 1), own = tid / kLanes / per;
    for (int r0 = 0; r0 < per; r0 += kGroups) {
        const int r = beside > 1 ? tid / kLanes - own * per : r0 + tid / kLanes, t0 = beside > 1 ? own : 0;
        const int kind = r < P.n_heads ? 0 : r < P.n_heads + P.n_kv_heads ? 1 : 2;   // q, k, v
        const int h = kind == 0 ? r : kind == 1 ? r - P.n_heads : r - P.n_heads - P.n_kv_heads;
        const long long ld = kind == 0 ? P.ldq : kind == 1 ? P.ldk : P.ldv, ldo = kind == 0 ? P.ldqo : P.ldko;
        const uint8_t* src = (kind == 0 ? P.q : kind == 1 ? P.k : P.v) + ((size_t)first * ld + (size_t)h * D + part * 8) * kEs;
        const int es = P.out_type == QWEN_FP32 ? 4 : 2;
        uint8_t* out = kind == 0 ? P.q_out : kind == 1 ? P.k_out : nullptr;
        if (out) out += ((size_t)first * ldo + (size_t)h * D + part * 8) * es;
        const bool mine = r < per && t0 < beside;
        uint4 next[2 * kN];
        auto fetch = [&](int t) {
            #pragma unroll
            for (int n = 0; n < 2 * kN; n++) next[n] = make_uint4(0, 0, 0, 0);
            if (mine && t < tokens && row_at[t] >= 0) {
                const uint8_t* p = src + (size_t)t * ld * kEs;
                #pragma unroll
                for (int n = 0; n < kN; n++) {
                    next[n] = __ldg(reinterpret_cast<const uint4*>(p) + n);
                    next[kN + n] = __ldg(reinterpret_cast<const uint4*>(p + D / 2 * kEs) + n);
                }
            }
        };
        fetch(t0);
        for (int ta = 0; ta < tokens; ta += beside) {
            const int t = min(ta + t0, tokens - 1);
            float x[16];
            kv::unpack16<SRC>(next, x);
            fetch(ta + t0 + beside);
            const bool in = mine && ta + t0 < tokens && row_at[t] >= 0;
            if (P.q_gain) {
                float sum = 0.f;
                #pragma unroll
                for (int e = 0; e < 16; e++) sum = fmaf(x[e], x[e], sum);
                #pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float inv = kind < 2 ? 1.0f / sqrtf(fmaf(sum, 1.0f / D, P.eps)) : 1.0f;
                #pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 g = *reinterpret_cast<const float4*>(&gains[kind & 1][(e & 8 ? D / 2 - 8 : 0) + part * 8 + e]);
                    if (kind < 2) { x[e] *= inv * g.x; x[e + 1] *= inv * g.y; x[e + 2] *= inv * g.z; x[e + 3] *= inv * g.w; }
                }
            }
            if (kind < 2) {
                #pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 c4 = *reinterpret_cast<const float4*>(&cosine[t][part * 8 + e]), s4 = *reinterpret_cast<const float4*>(&sine[t][part * 8 + e]);
                    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float a = x[e + j], b = x[8 + e + j];
                        x[e + j] = fmaf(a, c[j], -(b * s[j]));
                        x[8 + e + j] = fmaf(b, c[j], a * s[j]);
                    }
                }
                if (in && out) {
                    uint8_t* p = out + (size_t)t * ldo * es;
                    store8(p, P.out_type, x);
                    store8(p + D / 2 * es, P.out_type, x + 8);
                }
            }
            const int page = in && kind > 0 ? page_at[t] : -1;
            if (__any_sync(0xffffffffu, page >= 0)) to_page<D, Q8>(P, kind == 2, page, max(row_at[t], 0), h, part, x);
        }
    }
}

}  // namespace pg
}  // namespace qb
