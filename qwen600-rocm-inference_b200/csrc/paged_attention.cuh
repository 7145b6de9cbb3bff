// paged_attention.cuh — attention of one new token a sequence over a K/V cache in
// pages (qwen_paged_attention).  No reference counterpart (the reference's attention serves
// one contiguous bf16 cache, qwen_model.cuh:551-614).
//
// The mathematics, the division of the work into shares of a line of key tiles
// and the joining of partial results are tree_attention.cuh's, with a single node a
// sequence; here a position's rows are found through the page table.
//
// A K/V head's query heads (8 or 16 a block of rows) are the columns of the products:
// S^T = K Q^T (keys x heads) and O^T = V^T P^T (dims x heads), so few heads waste
// at most 8 columns where rows would waste 16: half the matrix instructions, half the
// exponentials, half the registers of O.  P^T reaches the second product by one 8 x 8
// transposition in registers (movmatrix) each.  A warp owns KW keys of a tile, its own ring
// of cp.async stages, its own sums l and O, and a base for each head that exponents
// are taken from: it rises only when the maximum has risen by 2^8 (base-2 exponents), so the tiles
// in between need one vote instead of a maximum over the warp.  The page numbers of
// a tile are loaded a tile before its rows.  Weights are rounded to 16 bits for the product
// with V (off by half a step, 2^-8 or 2^-11 relative); l sums them unrounded.
//
// Few sequences: a cluster of eight CTAs an item, each a run of tiles, joined through distributed shared
// memory, one launch.
//
// Measured: 128 ragged sequences up to 8191 over 1.08 GB of e4m3 pages 179 to 187 us (5.8 to 6.0 TB/s, floor 165), bound by memory traffic;
// 32 over 35 MB of int8 pages, seven heads of 64 each, 16.5 to 16.9 us (floor 5.4), by the plan, the first
// loads and the joining; one sequence at 1024 6.3 us (floor 0.6), by its latencies (in a table of more than 2,048 positions, which takes
// two launches, 8.6 us).
#pragma once
#include <cooperative_groups.h>

#include "kv_pages.cuh"
#include "tree_attention.cuh"

namespace qb {
namespace pa {

using ta::cp_async16;
using ta::cp_async4;
using ta::cp_async_commit;
using ta::cp_async_wait;
using ta::exp2_approx;
using ta::fma2;
using ta::kLeast;
using ta::mul2;
using ta::swz;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kItemCost = 2;   // what an item costs beside its tiles, in tiles
constexpr int kCluster = 8;    // CTAs that share an item
constexpr float kRise = 8.0f;  // a base follows when the maximum has risen by 2^8

struct Params {
    ta::Params t;    // cache.capacity: positions that a table names; q, out, lens, work, shares
    pg::Pages pages;
    int cluster;     // a cluster of kCluster CTAs has an item
};

// Keys of a tile, by the bytes of a cache row: 16 or 32 for each warp.
__host__ __device__ constexpr int tile_keys(int row_bytes) { return kWarps * (row_bytes == 256 ? 16 : 32); }
template <int STORE, int D, int NT>
struct Layout {
    static constexpr int kEs = STORE == QWEN_E4M3 || STORE == QWEN_INT8 ? 1 : 2;
    static constexpr bool k8 = kEs == 1;
    static constexpr int kRow = D * kEs;                       // bytes of a cache row
    static constexpr int KT = tile_keys(kRow);                 // keys of a tile
    static constexpr int KW = KT / kWarps;                     // keys of a warp's part of it
    static constexpr int kRows = 8 * NT;                       // query heads of an item
    static constexpr int kCtas = 2;                            // on an SM
    static constexpr int kPart = KW * kRow;                    // bytes of K (or V) of a warp's stage
    static constexpr int kScale = k8 ? 2 * KW * 4 : 0;         // its scales
    static constexpr int kStage = 2 * kPart + kScale + 16;     // and which of its keys are there
    static constexpr int kStages = (108 * 1024 / kWarps) / kStage < 6 ? (108 * 1024 / kWarps) / kStage : 6;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kPitch = D + 4;                       // floats of a row of O at the joining
    static constexpr int kJoin = kWarps * kRows * (kPitch + 2) * 4;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
    static_assert(kJoin + kRows * (D + 2) * 4 <= kSmem, "a cluster's parts lie behind the warps'");
    static constexpr int kSlot = kRows * (D + 2);              // floats of a workspace slot: O, then (m, l) pairs
    static_assert(kStage % 16 == 0, "rows of 16-byte pieces");
    static_assert(kStages >= 2 && kCtas * (kSmem + 1024) <= 228 * 1024, "kCtas CTAs an SM");
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// grid: a CTA for each share and block of rows beside it, kThreads threads, Layout::kSmem bytes.
template <int QT, int STORE, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) paged_kernel(const __grid_constant__ Params PP) {
    using L = Layout<STORE, D, NT>;
    constexpr bool BF = QT == QWEN_BF16 && !L::k8;       // type of the products
    // A base lies this far below the maximum that it was taken from: fp16 weights use the range up to 2^15, so that what is lost under
    // fp16's smallest steps is 2^-32 of the largest (of 8-bit caches: times the unit over the value's scale) and less.
    constexpr float kLift = BF ? 0.0f : 7.0f;
    constexpr int KW = L::KW, KB = KW / 16, KS = D / 16, kStages = L::kStages;
    constexpr int DT = D / 16;                           // tiles of 16 dims
    extern __shared__ __align__(128) uint8_t smem[];
    const ta::Params& P = PP.t;
    const pg::Pages& pages = PP.pages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    uint8_t* ring = smem + warp * kStages * L::kStage;
    pdl_wait();
    pdl_launch_dependents();   // after the wait: what the joining kernel reads early (lens) is then complete

    ta::Items<L::KT, kItemCost, L::kRows> it;
    const int rank = PP.cluster ? (int)blockIdx.x % kCluster : 0;
    if (!PP.cluster) {
        if (!it.start(P)) return;
    } else {
        const int unit = (int)blockIdx.x / kCluster, per = P.n_kv_heads * P.row_blocks;
        it.seq = unit / per;
        it.h = (unit - it.seq * per) / P.row_blocks;
        it.r_base = (unit - it.seq * per) % P.row_blocks * L::kRows;
        it.len = max(P.lens[it.seq], -1);
        it.end = ta::seq_end(P, it.len);
        it.n = ta::seq_tiles<L::KT>(P, it.len);
        it.t0 = (int)((long long)it.n * rank / kCluster);
        it.t1 = (int)((long long)it.n * (rank + 1) / kCluster);
        it.at = it.before = 0;                 // (the one item)
        it.to = it.step = 1;
    }
    const int in_page = (1 << pages.shift) - 1;
    do {
        const int seq = it.seq, end = it.end, h = it.h, r_base = it.r_base, t0 = it.t0, t1 = it.t1;
        // Page of key `lane` (or lane % KW) of this warp's part of tile t, -1: not there, or past the end
        auto look_up = [&](int t) {
            const int pos = t * L::KT + warp * KW + (lane & (KW - 1));
            return t < t1 && pos < end ? pages.page_of(seq, pos) : -1;
        };
        auto load = [&](int t, int s, int page) {   // this warp's part of tile t into stage s; keys that are not there as zeros
            uint8_t* stage = ring + s * L::kStage;
            const uint32_t st = smem_addr(stage);
            const int k0 = t * L::KT + warp * KW;
            constexpr int kChunks = L::kRow / 16, kPer = KW * kChunks / 32, kStep = 32 / kChunks;
            const uint32_t off0 = swz<L::kRow>(lane / kChunks, lane % kChunks);
            const size_t in_row = (size_t)h * pages.head_stride * L::kEs + lane % kChunks * 16;
            #pragma unroll
            for (int i = 0; i < kPer; i++) {
                const int r = lane / kChunks + kStep * i, pg = __shfl_sync(~0u, page, r);
                const uint32_t off = (off0 ^ (L::kRow >= 128 ? ((kStep * i) & 7) << 4 : 0)) + 512 * i;
                const size_t at = pg < 0 ? 0 : (size_t)pg * pages.page_stride * L::kEs + in_row + (size_t)((k0 + r) & in_page) * L::kRow;
                cp_async16(st + off, pages.k + at, pg >= 0);
                cp_async16(st + L::kPart + off, pages.v + at, pg >= 0);
            }
            const uint32_t there = __ballot_sync(~0u, page >= 0);
            if (lane == 0) *reinterpret_cast<uint32_t*>(stage + 2 * L::kPart + L::kScale) = there;
            if constexpr (L::k8) {
                static_assert(KW == 32, "one scale a lane");
                const size_t at = page < 0 ? 0 : ((size_t)page * pages.page_stride + (size_t)h * pages.head_stride) / D + ((k0 + lane) & in_page);
                cp_async4(st + 2 * L::kPart + 4 * lane, pages.ks + at, page >= 0);
                cp_async4(st + 2 * L::kPart + 4 * KW + 4 * lane, pages.vs + at, page >= 0);
            }
        };
        int page = look_up(t0);
        #pragma unroll
        for (int s = 0; s < kStages - 1; s++) {
            const int next = look_up(t0 + s + 1);
            if (t0 + s < t1) load(t0 + s, s, page);
            cp_async_commit();
            page = next;
        }
        // queries: the B fragments of head g of each 8 (dims 16 ks + 2j, + 8; 8-bit caches: the dims in the order in which the K codes
        // come out of ldmatrix, 4j, 4j+1 and 4j+2, 4j+3)
        uint32_t qb[NT][KS][2];
        float c[NT][2];               // score factors of heads 2j, 2j + 1
        {
            const uint32_t flip = P.scale_log2 < 0.f ? 0x80008000u : 0u;   // a negative scale: its sign goes to the queries
            const float a = fabsf(P.scale_log2);
            #pragma unroll
            for (int n = 0; n < NT; n++) {
                const int row = r_base + 8 * n + g;
                const bool live = row < P.group;
                const uint8_t* q = P.q + ((size_t)seq * P.ldq + (size_t)(h * P.group + row) * D) * 2;
                #pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint2 w = make_uint2(0, 0);
                    if (live) {
                        if constexpr (L::k8) w = __ldg(reinterpret_cast<const uint2*>(q + (16 * k + 4 * j) * 2));
                        else w = make_uint2(__ldg(reinterpret_cast<const uint32_t*>(q + (16 * k + 2 * j) * 2)),
                                            __ldg(reinterpret_cast<const uint32_t*>(q + (16 * k + 8 + 2 * j) * 2)));
                    }
                    qb[n][k][0] = w.x ^ flip;
                    qb[n][k][1] = w.y ^ flip;
                }
                float f = a;
                if constexpr (L::k8 && QT == QWEN_BF16) {
                    // into fp16's range: 2^e <= the row's largest magnitude < 2^(e+1); infinities and NaN go through as they are
                    uint32_t m = 0;
                    #pragma unroll
                    for (int k = 0; k < KS; k++) m = __vmaxu2(m, __vmaxu2(qb[n][k][0] & 0x7fff7fffu, qb[n][k][1] & 0x7fff7fffu));
                    m = max(m & 0xffffu, m >> 16);
                    m = max(m, __shfl_xor_sync(~0u, m, 1));
                    m = max(m, __shfl_xor_sync(~0u, m, 2));
                    const int e = min(max((int)(m >> 7), 1), 253);
                    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                    #pragma unroll
                    for (int k = 0; k < KS; k++)
                        #pragma unroll
                        for (int b = 0; b < 2; b++) qb[n][k][b] = kv::half2_bits(bf_lo(qb[n][k][b]) * down, bf_hi(qb[n][k][b]) * down);
                    f = a * __uint_as_float((uint32_t)e << 23);
                }
                f = fmaxf(f, kLeast);                                       // (above 0: -inf * 0 would be NaN)
                c[n][0] = __shfl_sync(~0u, f, 8 * j);                       // head 2j is lanes 8j .. 8j + 3
                c[n][1] = __shfl_sync(~0u, f, 8 * j + 4);
            }
        }
        float o[DT][NT][4], base[NT][2], l[NT][2];
        #pragma unroll
        for (int n = 0; n < NT; n++) {
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int e = 0; e < 4; e++) o[d][n][e] = 0.f;
            base[n][0] = base[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
        uint32_t ve = 1;   // 8-bit caches: O is in units of 2^(ve - 127)

        for (int t = t0; t < t1; t++) {
            {
                const int ahead = t + kStages - 1, next = look_up(ahead + 1);
                if (ahead < t1) load(ahead, (ahead - t0) % kStages, page);
                cp_async_commit();
                page = next;
            }
            cp_async_wait<kStages - 1>();
            __syncwarp();
            uint8_t* st = ring + (t - t0) % kStages * L::kStage;
            const uint32_t there = *reinterpret_cast<const uint32_t*>(st + 2 * L::kPart + L::kScale);
            if (there) {
                // ---- scores: keys 16 kb + g, + 8 of heads 2j, 2j + 1 ----
                float s[KB][NT][4];
                #pragma unroll
                for (int kb = 0; kb < KB; kb++)
                    #pragma unroll
                    for (int n = 0; n < NT; n++)
                        #pragma unroll
                        for (int e = 0; e < 4; e++) s[kb][n][e] = 0.f;
                #pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    if constexpr (!L::k8) {
                        #pragma unroll
                        for (int kb = 0; kb < KB; kb++) {
                            uint32_t a[4];
                            ldsm_x4(smem_addr(st + swz<L::kRow>(16 * kb + (lane & 15), 2 * ks + (lane >> 4))), a[0], a[1], a[2], a[3]);
                            #pragma unroll
                            for (int n = 0; n < NT; n++) ta::mma16816<BF>(s[kb][n], a, qb[n][ks][0], qb[n][ks][1]);
                        }
                    } else {                                // four key groups of one 16-byte piece
                        uint32_t b[4];
                        ldsm_x4(smem_addr(st + swz<L::kRow>(lane, ks)), b[0], b[1], b[2], b[3]);
                        #pragma unroll
                        for (int kb = 0; kb < KB; kb++) {
                            uint32_t a[4];
                            ta::codes_f16x2<STORE, false>(b[2 * kb], a[0], a[2]);
                            ta::codes_f16x2<STORE, false>(b[2 * kb + 1], a[1], a[3]);
                            #pragma unroll
                            for (int n = 0; n < NT; n++) ta::mma16816<BF>(s[kb][n], a, qb[n][ks][0], qb[n][ks][1]);
                        }
                    }
                }
                float vs[KB][2];
                if constexpr (L::k8) {
                    const float* sc = reinterpret_cast<const float*>(st + 2 * L::kPart);
                    #pragma unroll
                    for (int kb = 0; kb < KB; kb++)
                        #pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float k = sc[16 * kb + 8 * e + g];
                            vs[kb][e] = sc[KW + 16 * kb + 8 * e + g];
                            #pragma unroll
                            for (int n = 0; n < NT; n++) mul2(s[kb][n][2 * e], s[kb][n][2 * e + 1], k, k);
                        }
                }
                if (there != ~0u) {                         // (16 keys: the upper half says the same)
                    #pragma unroll
                    for (int kb = 0; kb < KB; kb++)
                        #pragma unroll
                        for (int e = 0; e < 2; e++)
                            if (!(there >> (16 * kb + 8 * e + g) & 1))
                                #pragma unroll
                                for (int n = 0; n < NT; n++) s[kb][n][2 * e] = s[kb][n][2 * e + 1] = -INFINITY;
                }
                // ---- softmax ----
                float mx[NT][2];
                bool rise = false;
                #pragma unroll
                for (int n = 0; n < NT; n++)
                    #pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float m = -INFINITY;
                        #pragma unroll
                        for (int kb = 0; kb < KB; kb++) m = fmaxf(m, fmaxf(s[kb][n][e], s[kb][n][2 + e]));
                        mx[n][e] = m;
                        rise |= fmaf(m, c[n][e], -kLift) > base[n][e] + kRise;
                    }
                uint32_t up = 0;                            // the rise of ve
                if constexpr (L::k8) {
                    const uint32_t e = __reduce_max_sync(~0u, there >> lane & 1 ? ta::scale_exponent(reinterpret_cast<const float*>(st + 2 * L::kPart)[KW + lane]) : 0u);
                    if (e > ve) { up = e - ve; ve = e; }
                    const float vinv = __uint_as_float((254u - ve) << 23);
                    #pragma unroll
                    for (int kb = 0; kb < KB; kb++) mul2(vs[kb][0], vs[kb][1], vinv, vinv);
                }
                if (__any_sync(~0u, rise) || up) {
                    const float w = !L::k8 ? 1.0f : up < 127u ? __uint_as_float((127u - up) << 23) : 0.f;
                    #pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float f[2];
                        #pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float m = mx[n][e];
                            #pragma unroll
                            for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
                            const float to = fmaxf(base[n][e], m == -INFINITY ? m : fmaf(m, c[n][e], -kLift));
                            f[e] = to == -INFINITY ? 1.0f : exp2_approx(base[n][e] - to);
                            base[n][e] = to;
                            l[n][e] *= f[e];
                            f[e] *= w;
                        }
                        #pragma unroll
                        for (int d = 0; d < DT; d++) {
                            mul2(o[d][n][0], o[d][n][1], f[0], f[1]);
                            mul2(o[d][n][2], o[d][n][3], f[0], f[1]);
                        }
                    }
                }
                uint32_t p[KB][NT][2];                      // P^T: keys 16 kb + 2j, + 1 (+ 8) of head g
                #pragma unroll
                for (int n = 0; n < NT; n++) {
                    float from[2];
                    #pragma unroll
                    for (int e = 0; e < 2; e++) from[e] = base[n][e] == -INFINITY ? 0.f : base[n][e];
                    #pragma unroll
                    for (int kb = 0; kb < KB; kb++)
                        #pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x = exp2_approx(fmaf(s[kb][n][2 * e], c[n][0], -from[0]));
                            float y = exp2_approx(fmaf(s[kb][n][2 * e + 1], c[n][1], -from[1]));
                            l[n][0] += x;
                            l[n][1] += y;
                            if constexpr (L::k8) mul2(x, y, vs[kb][e], vs[kb][e]);
                            p[kb][n][e] = transpose8x8(ta::pack2<BF>(x, y));
                        }
                }
                // ---- O^T += V^T P^T ----
                const uint8_t* sv = st + L::kPart;
                #pragma unroll
                for (int kb = 0; kb < KB; kb++) {
                    if constexpr (!L::k8) {
                        #pragma unroll
                        for (int d = 0; d < DT; d++) {
                            uint32_t a[4];
                            ta::ldsm_x4_t(smem_addr(sv + swz<L::kRow>(16 * kb + (lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1))), a[0], a[1], a[2], a[3]);
                            #pragma unroll
                            for (int n = 0; n < NT; n++) ta::mma16816<BF>(o[d][n], a, p[kb][n][0], p[kb][n][1]);
                        }
                    } else {
                        #pragma unroll
                        for (int d = 0; d < DT; d += 2) {   // two 16-byte pieces of the 16 keys' rows
                            uint32_t b[4];
                            ta::ldsm_x4_t(smem_addr(sv + swz<L::kRow>(16 * kb + (lane & 15), d + (lane >> 4))), b[0], b[1], b[2], b[3]);
                            #pragma unroll
                            for (int q = 0; q < 2; q++) {
                                uint32_t a[4];              // even and odd dims of the piece, keys 0-7 and 8-15
                                ta::codes_f16x2<STORE, true>(b[2 * q], a[0], a[1]);
                                ta::codes_f16x2<STORE, true>(b[2 * q + 1], a[2], a[3]);
                                #pragma unroll
                                for (int n = 0; n < NT; n++) ta::mma16816<BF>(o[d + q][n], a, p[kb][n][0], p[kb][n][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();   // the stage is free
        }
        cp_async_wait<0>();
        __syncthreads();    // the rings are free: the warps' results go over them
        float* join = reinterpret_cast<float*>(smem);               // [warp][head][kPitch], then [warp][head][2]
        float* join_ml = join + kWarps * L::kRows * L::kPitch;
        constexpr float kDown = BF ? 1.0f : 0x1p-7f;                // as if from the maximum itself: O and l 2^-kLift
        const float unit_v = L::k8 ? __uint_as_float(ve << 23) * kDown : kDown;
        #pragma unroll
        for (int n = 0; n < NT; n++)
            #pragma unroll
            for (int e = 0; e < 2; e++) {
                float sum = l[n][e];
                #pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(~0u, sum, x);
                const int row = warp * L::kRows + 8 * n + 2 * j + e;
                if (g == 0) {
                    join_ml[row * 2] = base[n][e] + kLift;
                    join_ml[row * 2 + 1] = sum * kDown;
                }
                #pragma unroll
                for (int d = 0; d < DT; d++) {
                    // 8-bit: rows g and g + 8 of a product are the dims 2g and 2g + 1 of the piece
                    join[row * L::kPitch + 16 * d + (L::k8 ? 2 * g : g)] = o[d][n][e] * unit_v;
                    join[row * L::kPitch + 16 * d + (L::k8 ? 2 * g + 1 : g + 8)] = o[d][n][2 + e] * unit_v;
                }
            }
        __syncthreads();
        auto joined = [&](int r, int d, float& mm, float& ll) {           // dims d .. d + 3 of head r, from the warps
            mm = -INFINITY;
            ll = 0.f;
            #pragma unroll
            for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, join_ml[(w * L::kRows + r) * 2]);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            #pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float mw = join_ml[(w * L::kRows + r) * 2], lw = join_ml[(w * L::kRows + r) * 2 + 1];
                const float fw = mm == -INFINITY ? 1.0f : exp2_approx(mw - mm);
                const float4 b = *reinterpret_cast<const float4*>(join + (w * L::kRows + r) * L::kPitch + d);
                ll += lw * fw;
                a.x += b.x * fw; a.y += b.y * fw; a.z += b.z * fw; a.w += b.w * fw;
            }
            return a;
        };
        auto write = [&](int row, int d, const float4& a, float ll) {
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
            uint8_t* dst = P.out + ((size_t)seq * P.ldo + (size_t)(h * P.group + row) * D + d) * 2;
            *reinterpret_cast<uint2*>(dst) = make_uint2(ta::pack2<QT == QWEN_BF16>(a.x * inv, a.y * inv), ta::pack2<QT == QWEN_BF16>(a.z * inv, a.w * inv));
        };
        if (PP.cluster) {
            // this CTA's part, then every CTA joins its share of the outputs from all parts in their order
            float* own = reinterpret_cast<float*>(smem + L::kJoin);       // [head][D], then (m, l) pairs
            for (int i = tid; i < L::kRows * (D / 4); i += kThreads) {
                const int r = i / (D / 4), d = i % (D / 4) * 4;
                float mm, ll;
                const float4 a = joined(r, d, mm, ll);
                *reinterpret_cast<float4*>(own + r * D + d) = a;
                if (d == 0) *reinterpret_cast<float2*>(own + L::kRows * D + 2 * r) = make_float2(mm, ll);
            }
            namespace cg = cooperative_groups;
            cg::cluster_group group = cg::this_cluster();
            group.sync();
            for (int i = rank * kThreads + tid; i < min(L::kRows, P.group - r_base) * (D / 4); i += kCluster * kThreads) {
                const int r = i / (D / 4), d = i % (D / 4) * 4;
                float2 ml[kCluster];
                float4 b[kCluster];
                float mm = -INFINITY, ll = 0.f;
                #pragma unroll
                for (int k = 0; k < kCluster; k++) {
                    const float* from = group.map_shared_rank(own, k);
                    ml[k] = *reinterpret_cast<const float2*>(from + L::kRows * D + 2 * r);
                    b[k] = *reinterpret_cast<const float4*>(from + r * D + d);
                    mm = fmaxf(mm, ml[k].x);
                }
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                #pragma unroll
                for (int k = 0; k < kCluster; k++) {
                    const float f = mm == -INFINITY ? 1.0f : exp2_approx(ml[k].x - mm);
                    ll += ml[k].y * f;
                    a.x += b[k].x * f; a.y += b[k].y * f; a.z += b[k].z * f; a.w += b[k].w * f;
                }
                write(r_base + r, d, a, ll);
            }
            group.sync();                      // the others read this CTA's part until here
            return;
        }
        const bool whole = t0 == 0 && t1 == it.n;
        float* slot = P.work + (size_t)(2 * blockIdx.x + (it.first ? 0 : 1)) * L::kSlot;
        for (int i = tid; i < L::kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = i % (D / 4) * 4, row = r_base + r;
            if (row >= P.group) break;
            float mm, ll;
            const float4 a = joined(r, d, mm, ll);
            if (whole) {
                write(row, d, a, ll);
            } else {
                *reinterpret_cast<float4*>(slot + r * D + d) = a;
                if (d == 0) *reinterpret_cast<float2*>(slot + L::kRows * D + 2 * r) = make_float2(mm, ll);
            }
        }
        __syncthreads();
    } while (it.next(P));
}

}  // namespace pa
}  // namespace qb
