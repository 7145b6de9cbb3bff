// kv_rows.cuh — rows of a K/V cache: written (and quantised), read back, and
// moved (qwen_kv_append, qwen_kv_read, qwen_kv_keep).  No reference
// counterpart (the reference's cache is bf16 and written by its RoPE kernel,
// qwen_model.cuh:321-347).
//
// All three are bound by memory traffic where there is enough of it, a row being read
// once and written once (prompts of 16 x 2048 tokens to int8 and back: 70 us, 53 us at
// the copy rate; without short counts an append of all rows 41 us and a read 36 us of
// 31, in 16 bits 42 us each of 41), and by their chains of loads where there is not
// (128 tokens in and out 3.7 us, the kept rows of one sequence in 28 layers 2.8 us). A
// thread owns 16 elements of a row (one 16-byte store of 8-bit codes), 4 or 8
// neighbouring threads the row, so the row's largest magnitude needs 2 or 3 shuffles
// and every access is a full 32-byte sector.
//
// Quantising.  The code of x in a row of largest magnitude a is the nearest
// representable value to the real number x * top / a (top = 448 or 127), ties
// to even.  x and a are scaled by one power of two first (exact), so nothing
// below can overflow; then with 16-bit inputs n = x * top is exact in fp32 (at
// most 11 + 7 bits), and y = n / a is corrected once by its residual n - y a,
// which a fused multiply-add forms exactly.  A quotient that is a tie is
// representable, so the correction lands on it; one that is not a tie is
// further from it (2^-19 relative: the difference of two whole numbers below
// 2^18) than the rounding.  fp32 inputs have no such margin: where the values
// next to y, y (1 +- 2^-20), get different codes, the quotient is formed in 64
// bits and rounded once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qwen_b200.h"
#include "ptx.cuh"

namespace qb {
namespace kv {

constexpr int kThreads = 256;
constexpr float kMinAmax = 8.673617379884035e-19f;   // 2^-60: the smallest magnitude a scale is made for

// The view, as the kernels take it.
struct Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    long long seq_stride, head_stride;   // elements
    int capacity;
};

// 16 consecutive elements as fp32: from 2 (16 bits) or 4 pieces of 16 bytes, from memory
template <int T, int N>
__device__ __forceinline__ void unpack16(const uint4 (&raw)[N], float (&x)[16]) {
    static_assert(N == (T == QWEN_FP32 ? 4 : 2), "16 elements");
    #pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (T == QWEN_FP32) {
                x[4 * i + j] = __uint_as_float(w[j]);
            } else if constexpr (T == QWEN_BF16) {
                x[8 * i + 2 * j] = bf_lo(w[j]);
                x[8 * i + 2 * j + 1] = bf_hi(w[j]);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                x[8 * i + 2 * j] = f.x;
                x[8 * i + 2 * j + 1] = f.y;
            }
        }
    }
}
template <int T>
__device__ __forceinline__ void load16(const uint8_t* p, float (&x)[16]) {
    constexpr int kN = T == QWEN_FP32 ? 4 : 2;
    uint4 raw[kN];
    #pragma unroll
    for (int i = 0; i < kN; i++) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    unpack16<T>(raw, x);
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int T>
__device__ __forceinline__ void store16(uint8_t* p, const float (&x)[16]) {
    if constexpr (T == QWEN_FP32) {
        #pragma unroll
        for (int i = 0; i < 4; i++) reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
        uint32_t w[8];
        #pragma unroll
        for (int i = 0; i < 8; i++) w[i] = T == QWEN_BF16 ? cvt_bf16x2(x[2 * i], x[2 * i + 1]) : half2_bits(x[2 * i], x[2 * i + 1]);
        reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
// two values to two e4m3 codes (nearest, ties to even, magnitudes above 448 to 448)
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}
// four e4m3 codes to fp32 (exact: every code is an fp16 value)
__device__ __forceinline__ void e4m3x4_f32(uint32_t w, float* x) {
    #pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (16 * i))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

template <int STORE>
__host__ __device__ constexpr float top_of() { return STORE == QWEN_E4M3 ? 448.0f : 127.0f; }

// The code nearest to x * top / a for one element, from 64-bit arithmetic.  The
// fp64 quotient of a 24-bit and a 24-bit number times top is never rounded onto a
// tie that it is not; for e4m3 it is first cut to fp32 with the last bit set if
// anything was cut, so that the conversion rounds once.
template <int STORE>
__device__ __noinline__ uint32_t code_exact(float x, float a) {
    const double q = (double)x * (double)top_of<STORE>() / (double)a;
    if constexpr (STORE == QWEN_INT8) {
        return (uint32_t)__double2int_rn(q) & 0xffu;
    } else {
        float f = __double2float_rz(q);
        if ((double)f != q) f = __uint_as_float(__float_as_uint(f) | 1u);
        return e4m3x2(f, 0.f) & 0xffu;
    }
}

// Codes of 16 elements of a row with largest magnitude a (finite, >= kMinAmax).
template <int SRC, int STORE>
__device__ __forceinline__ uint4 encode16(const float (&x)[16], float a) {
    // s2 = 2^k with a * s2 in [256, 512)
    const uint32_t e = __float_as_uint(a) >> 23;   // 67 .. 254
    const float s2 = __uint_as_float((262u - e) << 23);
    const float den = a * s2, c = top_of<STORE>() * s2, inv = 1.0f / den;
    uint32_t w[4];
    #pragma unroll
    for (int g = 0; g < 4; g++) {
        float y[4];
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const float n = x[4 * g + j] * c;
            const float y0 = n * inv;
            y[j] = fmaf(fmaf(-y0, den, n), inv, y0);
        }
        if constexpr (STORE == QWEN_E4M3) {
            w[g] = e4m3x2(y[0], y[1]) | (e4m3x2(y[2], y[3]) << 16);
            if constexpr (SRC == QWEN_FP32) {
                constexpr float kUp = 1.0f + 0x1p-20f, kDown = 1.0f - 0x1p-20f;
                const uint32_t up = e4m3x2(y[0] * kUp, y[1] * kUp) | (e4m3x2(y[2] * kUp, y[3] * kUp) << 16);
                const uint32_t dn = e4m3x2(y[0] * kDown, y[1] * kDown) | (e4m3x2(y[2] * kDown, y[3] * kDown) << 16);
                if (up != dn) {
                    w[g] = 0;
                    #pragma unroll
                    for (int j = 0; j < 4; j++) w[g] |= code_exact<STORE>(x[4 * g + j], a) << (8 * j);
                }
            }
        } else {
            // |y| <= 127: adding 1.5 * 2^23 rounds to the nearest whole number (ties to even) in the low bits
            uint32_t b[4];
            bool near = false;
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const float r = y[j] + 12582912.0f;
                b[j] = __float_as_uint(r);
                if constexpr (SRC == QWEN_FP32) near |= fabsf(y[j] - (r - 12582912.0f)) > 0.5f - 0x1p-13f;
            }
            w[g] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            if (SRC == QWEN_FP32 && near) {
                w[g] = 0;
                #pragma unroll
                for (int j = 0; j < 4; j++) w[g] |= code_exact<STORE>(x[4 * g + j], a) << (8 * j);
            }
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A thread's place: rows of one sequence in the order (head, token), 16 elements
// of a row a thread.  grid (row blocks, n_seqs, 2: K and V).
template <int D>
struct Place {
    static constexpr int kLanes = D / 16;                  // threads a row
    static constexpr int kRows = kThreads / kLanes;        // rows that a block's threads cover at once
};

// SRC rows -> STORE cache.  A quantised element takes 16 instructions (16 x 2048
// tokens, bf16 to int8: 71 % of the issue slots, the memory at 54 % of the copy rate),
// so the number of those around the arithmetic counts.  U = 1: any number of tokens,
// threads over the rows in the order (head, token), a division a row; grid (ceil(rows /
// kRows), n_seqs, 2).  U = 2: a block takes 2 kRows tokens of one head, two a thread;
// grid (heads * ceil(tokens / (2 kRows)), n_seqs, 2).
template <int SRC, int STORE, int D, int U>
__global__ void __launch_bounds__(kThreads) append_kernel(Cache c, const uint8_t* __restrict__ k, const uint8_t* __restrict__ v, long long ld,
                                                          int n_heads, int n_tokens, const int* __restrict__ start,
                                                          const int* __restrict__ counts) {
    using P = Place<D>;
    const int seq = blockIdx.y, first = start[seq];
    const int live = counts ? min(counts[seq], n_tokens) : n_tokens;
    if (first < 0 || live <= 0) return;
    const unsigned part = threadIdx.x % P::kLanes;
    constexpr int kSrc = SRC == QWEN_FP32 ? 4 : 2;
    unsigned h, t;
    if constexpr (U == 1) {
        const unsigned row = blockIdx.x * P::kRows + threadIdx.x / P::kLanes;
        h = row / (unsigned)n_tokens;
        t = row - h * (unsigned)n_tokens;
    } else {
        const unsigned blocks = ((unsigned)n_tokens + U * P::kRows - 1) / (U * P::kRows);
        h = blockIdx.x / blocks;
        t = (blockIdx.x - h * blocks) * (U * P::kRows) + threadIdx.x / P::kLanes;
    }
    const uint8_t* src = (blockIdx.z ? v : k) + (((size_t)seq * n_tokens + t) * (size_t)ld + (size_t)h * D + part * 16) * kSrc;
    const size_t at0 = (size_t)seq * c.seq_stride + (size_t)h * c.head_stride + ((size_t)first + t) * D;
    uint8_t* base = blockIdx.z ? c.v : c.k;
    uint4 raw[U][kSrc];
    bool mine[U];
    #pragma unroll
    for (int u = 0; u < U; u++) {
        const unsigned tu = t + u * P::kRows;
        mine[u] = h < (unsigned)n_heads && tu < (unsigned)live && (long long)first + tu < c.capacity;
        if (mine[u]) {
            #pragma unroll
            for (int i = 0; i < kSrc; i++) raw[u][i] = __ldg(reinterpret_cast<const uint4*>(src + (size_t)u * P::kRows * (size_t)ld * kSrc) + i);
        }
    }
    #pragma unroll
    for (int u = 0; u < U; u++) {
        const size_t at = at0 + (size_t)u * P::kRows * D;
        float x[16];
        if (mine[u]) unpack16<SRC>(raw[u], x);
        if constexpr (STORE == QWEN_E4M3 || STORE == QWEN_INT8) {
            // magnitudes as bit patterns: NaN above infinity above every number
            uint32_t m = 0;
            if (mine[u]) {
                if constexpr (SRC == QWEN_FP32) {
                    #pragma unroll
                    for (int i = 0; i < 16; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
                } else {
                    #pragma unroll
                    for (int i = 0; i < kSrc; i++)
                        m = __vmaxu2(__vmaxu2(__vmaxu2(m, raw[u][i].x & 0x7fff7fffu), __vmaxu2(raw[u][i].y & 0x7fff7fffu, raw[u][i].z & 0x7fff7fffu)),
                                     raw[u][i].w & 0x7fff7fffu);
                    m = max(m & 0xffffu, m >> 16);
                }
            }
            #pragma unroll
            for (int o = 1; o < P::kLanes; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (!mine[u]) continue;
            float a;
            bool finite;
            if constexpr (SRC == QWEN_FP32) { a = __uint_as_float(m); finite = m < 0x7f800000u; }
            else if constexpr (SRC == QWEN_BF16) { a = __uint_as_float(m << 16); finite = m < 0x7f80u; }
            else { a = __half2float(__ushort_as_half((uint16_t)m)); finite = m < 0x7c00u; }
            a = fmaxf(a, kMinAmax);
            uint4 w = make_uint4(0, 0, 0, 0);
            if (finite) w = encode16<SRC, STORE>(x, a);
            *reinterpret_cast<uint4*>(base + at + part * 16) = w;
            if (part == 0) (blockIdx.z ? c.vs : c.ks)[at / D] = finite ? a / top_of<STORE>() : __uint_as_float(0x7fffffffu);
        } else {
            if (mine[u]) store16<STORE>(base + (at + part * 16) * 2, x);
        }
    }
}

// grid (ceil(rows / kRows), n_seqs, 2); STORE cache -> DST rows.
template <int DST, int STORE, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache c, uint8_t* __restrict__ k, uint8_t* __restrict__ v, long long ld, int n_heads,
                                                        int n_tokens, const int* __restrict__ start, const int* __restrict__ counts) {
    using P = Place<D>;
    const int seq = blockIdx.y, first = start[seq];
    const int live = counts ? min(counts[seq], n_tokens) : n_tokens;
    if (first < 0 || live <= 0) return;
    const unsigned row = blockIdx.x * P::kRows + threadIdx.x / P::kLanes, part = threadIdx.x % P::kLanes;
    const unsigned h = row / (unsigned)n_tokens, t = row - h * (unsigned)n_tokens;
    if (!(h < (unsigned)n_heads && t < (unsigned)live && (long long)first + t < c.capacity)) return;
    const size_t at = (size_t)seq * c.seq_stride + (size_t)h * c.head_stride + ((size_t)first + t) * D;
    const uint8_t* base = blockIdx.z ? c.v : c.k;
    float x[16];
    if constexpr (STORE == QWEN_E4M3 || STORE == QWEN_INT8) {
        const uint4 a = *reinterpret_cast<const uint4*>(base + at + part * 16);
        const float scale = (blockIdx.z ? c.vs : c.ks)[at / D];
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        #pragma unroll
        for (int g = 0; g < 4; g++) {
            if constexpr (STORE == QWEN_E4M3) {
                e4m3x4_f32(w[g], x + 4 * g);
            } else {
                #pragma unroll
                for (int j = 0; j < 4; j++) x[4 * g + j] = (float)(int)(int8_t)(w[g] >> (8 * j));
            }
        }
        #pragma unroll
        for (int i = 0; i < 16; i++) x[i] *= scale;
    } else {
        load16<STORE>(base + (at + part * 16) * 2, x);
    }
    constexpr int kDst = DST == QWEN_FP32 ? 4 : 2;
    store16<DST>((blockIdx.z ? v : k) + (((size_t)seq * n_tokens + t) * (size_t)ld + (size_t)h * D + part * 16) * kDst, x);
}

// Moves the rows of a kept branch.  A block takes kKeepHeads heads of a sequence:
// finding the rows that move is a chain of loads that all of them share.  Of as many
// heads as its threads hold in registers (kKeepPer pieces of 16 bytes each) all
// source rows of K and V are read before any is written, so paths may be in any
// order.  grid (ceil(n_heads / kKeepHeads), n_seqs).
constexpr int kKeepThreads = 256, kKeepHeads = 8, kKeepPer = 8;
constexpr int kMaxNodes = 64;
template <int ROW_BYTES, bool SCALED>
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(Cache c, const int* __restrict__ start, const int* __restrict__ path,
                                                            const int* __restrict__ n_path, int n_heads, int n_nodes, int elem_bytes) {
    constexpr int kChunks = ROW_BYTES / 16;
    static_assert(kMaxNodes * kChunks * 2 <= kKeepThreads * kKeepPer && kKeepPer <= 2 * kChunks, "a head's rows (and scales) fit the block's registers");
    __shared__ int from[kMaxNodes], to[kMaxNodes], moves;
    const int seq = blockIdx.y, tid = threadIdx.x, first = start[seq];
    const int n = min(n_path[seq], n_nodes);
    if (first < 0 || n <= 0) return;
    if (tid < 32) {   // the rows that move, in a list (a row that stays where it is does not)
        int have = 0;
        #pragma unroll
        for (int k = 0; k < kMaxNodes; k += 32) {
            const int r = k + tid, p = r < n ? path[(size_t)seq * n_nodes + r] : -1;
            const bool fine = p >= 0 && p < n_nodes && p != r && (long long)first + p < c.capacity && (long long)first + r < c.capacity;
            const uint32_t some = __ballot_sync(~0u, fine);
            if (fine) {
                const int i = have + __popc(some & ((1u << tid) - 1));
                from[i] = p;
                to[i] = r;
            }
            have += __popc(some);
        }
        if (tid == 0) moves = have;
    }
    __syncthreads();
    const int m = moves;
    if (m == 0) return;
    const int h1 = min(n_heads, (int)(blockIdx.x + 1) * kKeepHeads), per_head = 2 * kChunks * m;   // pieces of a head
    const int batch = kKeepThreads * kKeepPer / per_head;                                          // heads at a time
    const size_t seq0 = (size_t)seq * c.seq_stride;
    for (int h0 = blockIdx.x * kKeepHeads; h0 < h1; h0 += batch) {
        const int heads = min(batch, h1 - h0), pieces = heads * per_head;
        uint4 w[kKeepPer];
        uint8_t* dst[kKeepPer];
        #pragma unroll
        for (int i = 0; i < kKeepPer; i++) {
            const int x = tid + i * kKeepThreads;
            dst[i] = nullptr;
            if (x < pieces) {
                const int ch = x % kChunks, y = x / kChunks, kv = y & 1, z = y >> 1, h = z / m, r = z - h * m;
                uint8_t* row0 = (kv ? c.v : c.k) + (seq0 + (size_t)(h0 + h) * c.head_stride) * elem_bytes + (size_t)first * ROW_BYTES + ch * 16;
                w[i] = *reinterpret_cast<const uint4*>(row0 + (size_t)from[r] * ROW_BYTES);
                dst[i] = row0 + (size_t)to[r] * ROW_BYTES;
            }
        }
        float s[2];
        float* sdst[2] = {nullptr, nullptr};
        if constexpr (SCALED) {
            // (a batch has at most kKeepThreads kKeepPer / kChunks <= 2 kKeepThreads rows)
            #pragma unroll
            for (int i = 0; i < 2; i++) {
                const int x = tid + i * kKeepThreads;
                if (x < heads * m * 2) {
                    const int kv = x & 1, z = x >> 1, h = z / m, r = z - h * m;
                    float* row0 = (kv ? c.vs : c.ks) + (seq0 + (size_t)(h0 + h) * c.head_stride) / (ROW_BYTES / elem_bytes) + first;
                    s[i] = row0[from[r]];
                    sdst[i] = row0 + to[r];
                }
            }
        }
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < kKeepPer; i++)
            if (dst[i]) *reinterpret_cast<uint4*>(dst[i]) = w[i];
        if constexpr (SCALED) {
            #pragma unroll
            for (int i = 0; i < 2; i++) if (sdst[i]) *sdst[i] = s[i];
        }
    }
}

}  // namespace kv
}  // namespace qb
