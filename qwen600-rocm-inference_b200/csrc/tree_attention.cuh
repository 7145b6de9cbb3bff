// tree_attention.cuh — attention of a tree of drafted tokens over a K/V cache
// (qwen_tree_attention).  No reference counterpart (the reference's attention
// serves one token over a bf16 cache, qwen_model.cuh:551-614).
//
// Mathematics.  Node i of sequence s attends to positions [0, len) and to len + j
// for its ancestors-or-self j, a 64-bit mask.  One pass over the keys with the
// running maximum m and sum l of the softmax (base 2, scale * log2 e folded into
// the scores); O += P V with P = 2^(score - m), scaled down when m rises.
//
// The rows of a work item are the n_nodes * group (query head, node) pairs that
// share a K/V head, or a block of them, so each K/V byte is read once for all of
// them.  The items (sequence, K/V head) are laid end to end on a line of key tiles, each
// with a few positions more for its fixed cost, and the line is cut into equal
// shares, one a CTA: ragged lengths balance by themselves, and a single long
// sequence spreads over all SMs.  Where a K/V head's rows take several blocks, as many
// CTAs as blocks walk the same share side by side, so that the tiles come from
// the memory once and for the others from the L2.  An item that crosses a border
// between shares leaves partial (m, l, O) in the workspace, two slots a CTA, and
// combine_kernel joins them in the order of the keys, so results do not depend on
// timing.  The shares are computed on the device from lens.  Where the cache's
// capacity is a few tiles, a CTA takes a whole item and nothing is joined.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qwen_b200.h"
#include "kv_rows.cuh"
#include "ptx.cuh"

namespace qb {
namespace ta {

constexpr int kMaxNodes = 64;

struct Params {
    kv::Cache cache;
    const uint8_t* q;
    uint8_t* out;
    const int *lens, *parents;
    float* work;
    long long ldq, ldo;
    int n_seqs, n_kv_heads, group, n_nodes;
    int whole;                // a CTA for each item: CTA (sequence * n_kv_heads + head) * row_blocks + block
    int groups, by_item;      // shares of the line; combine_kernel's blocks are for the items (else: for the shares)
    int withheld;             // -1, or for failure tests: this part of the ring that K and V come through is never announced
    unsigned long long wait_ns;   // longest wait of the tensor-memory kernel
    int row_blocks, beside;   // blocks of rows that a K/V head has; CTAs side by side on a share (row_blocks, or 1 where that is more than the grid)
    float scale_log2;   // scale * log2(e)
    float per_group;    // 1 / group
    // The node of a row (row < 64 * group, group <= 2^14): (row + 1/2) / group lies at least 2^-15 from a whole number below 64,
    // and the product's two roundings move it by less than 2^-17.
    __device__ __forceinline__ int node_of(int row) const { return (int)(((float)row + 0.5f) * per_group); }
};

// ---- the line of key tiles -----------------------------------------------------
// Positions that sequence s has, its nodes' among them (0: nothing is present).
__device__ __forceinline__ int seq_end(const Params& P, int len) {
    return len < 0 || len >= P.cache.capacity ? 0 : min(len + min(P.n_nodes, P.cache.capacity - len), P.cache.capacity);
}
template <int KT>
__device__ __forceinline__ int seq_tiles(const Params& P, int len) { return max(1, (seq_end(P, len) + KT - 1) / KT); }

// The line cut into G shares (as many as positions at most, so that none is
// empty): share i begins at position i * n / G (rounded down).  Positions are below
// 2^31 (the host sees to it).
struct Shares {
    int n, whole, rest, G;
    __device__ __forceinline__ Shares() {}
    __device__ __forceinline__ Shares(int length, int g) : n(length), G(min(g, length)) {
        whole = (int)((unsigned)n / (unsigned)G);
        rest = n - whole * G;
    }
    __device__ __forceinline__ int begin(int i) const { return i >= G ? n : whole * i + (int)((unsigned)(rest * i) / (unsigned)G); }   // rest * i < G^2
    // the share that position x lies in: the last one that begins at x or before
    __device__ __forceinline__ int of(int x) const {
        int i = min((int)(((float)x + 0.5f) * (float)G / (float)n), G - 1);   // a guess
        while (i + 1 < G && begin(i + 1) <= x) i++;
        while (begin(i) > x) i--;
        return i;
    }
};

// The line of all items, units a sequence, by all lanes of a warp: every length
// is loaded once, up to kHeld sequences' with one wait.
template <int KT, int COST>
struct Line {
    static constexpr int kHeld = 128;
    int len[kHeld / 32];     // sequences lane, lane + 32, ... (all of them where there are no more)
    int units;
    Shares shares;
    __device__ __forceinline__ int positions(const Params& P, int s, int l) const {
        return s < P.n_seqs ? (seq_tiles<KT>(P, l) + COST) * units : 0;
    }
    __device__ __forceinline__ Line(const Params& P, int items, int groups) : units(items) {
        const int lane = threadIdx.x & 31;
        #pragma unroll
        for (int k = 0; k < kHeld / 32; k++) len[k] = lane + 32 * k < P.n_seqs ? P.lens[lane + 32 * k] : -1;
        int n = 0;
        #pragma unroll
        for (int k = 0; k < kHeld / 32; k++) n += positions(P, lane + 32 * k, len[k]);
        for (int s = kHeld + lane; s < P.n_seqs; s += 32) n += positions(P, s, P.lens[s]);
        shares = Shares(__reduce_add_sync(~0u, n), groups);
    }
    // The positions before sequence s.
    __device__ __forceinline__ int before(const Params& P, int s) const {
        const int lane = threadIdx.x & 31;
        int n = 0;
        #pragma unroll
        for (int k = 0; k < kHeld / 32; k++) n += lane + 32 * k < s ? positions(P, lane + 32 * k, len[k]) : 0;
        for (int i = kHeld + lane; i < s; i += 32) n += positions(P, i, P.lens[i]);
        return __reduce_add_sync(~0u, n);
    }
    // The sequence that position x (below shares.n) belongs to, the positions before it, its length.
    __device__ __forceinline__ int find(const Params& P, int x, int& before, int& length) const {
        const int lane = threadIdx.x & 31;
        before = 0;
        int s = P.n_seqs - 1;
        length = -1;
        bool found = false;
        auto look = [&](int s0, int l) {
            const int n = positions(P, s0 + lane, l);
            int inc = n;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(~0u, inc, o);
                if (lane >= o) inc += y;
            }
            const uint32_t hit = __ballot_sync(~0u, n > 0 && before + inc > x);
            if (hit) {
                const int f = __ffs(hit) - 1;
                before += __shfl_sync(~0u, inc - n, f);
                length = __shfl_sync(~0u, l, f);
                s = s0 + f;
                found = true;
            } else {
                before += __shfl_sync(~0u, inc, 31);
            }
        };
        #pragma unroll
        for (int k = 0; k < kHeld / 32; k++) if (!found && 32 * k < P.n_seqs) look(32 * k, len[k]);
        for (int s0 = kHeld; s0 < P.n_seqs && !found; s0 += 32) look(s0, s0 + lane < P.n_seqs ? P.lens[s0 + lane] : -1);
        return s;
    }
};

// This CTA's share of the line, item after item.
template <int KT, int COST, int ROWS>
struct Items {
    int at, to, before;      // positions of the line
    int seq, len, end, n, unit_blocks, units, beside, step;   // len: -1 for every negative length (differences to it are taken)
    int h, r_base, t0, t1;   // the item's K/V head, first row, tiles t0 .. t1-1 of n
    bool first;              // the share's first item: it holds the share's beginning

    __device__ __forceinline__ void item(const Params& P) {
        end = seq_end(P, len);
        n = seq_tiles<KT>(P, len);
        const int per = n + COST, unit = (int)((unsigned)(at - before) / (unsigned)per), v0 = at - before - unit * per;
        const int v1 = min(per, v0 + (to - at));
        step = v1 - v0;
        t0 = max(0, v0 - COST);
        t1 = v1 - COST;
        h = unit_blocks == 1 ? unit : unit / unit_blocks;
        r_base = (unit - h * unit_blocks + (int)blockIdx.x % beside) * ROWS;
    }
    __device__ __forceinline__ bool advance(const Params& P) {
        at += step;
        first = false;
        if (at >= to) return false;
        if (at - before == (n + COST) * units) {
            before = at;
            len = max(P.lens[++seq], -1);
        }
        item(P);
        return true;
    }
    // the next item that has tiles in the share
    __device__ __forceinline__ bool next(const Params& P) {
        do {
            if (!advance(P)) return false;
        } while (t1 <= t0);
        return true;
    }
    // all lanes of a warp; false: nothing to do
    __device__ __forceinline__ bool start(const Params& P) {
        if (P.whole) {
            const int item_i = blockIdx.x / P.row_blocks;
            beside = P.row_blocks;
            seq = item_i / P.n_kv_heads;
            h = item_i - seq * P.n_kv_heads;
            r_base = (blockIdx.x - item_i * P.row_blocks) * ROWS;
            len = max(P.lens[seq], -1);
            end = seq_end(P, len);
            n = t1 = seq_tiles<KT>(P, len);
            at = before = t0 = 0;
            to = step = 1;
            units = unit_blocks = 1;
            first = true;
            return true;
        }
        beside = P.beside;
        unit_blocks = beside == 1 ? P.row_blocks : 1;
        units = P.n_kv_heads * unit_blocks;
        const Line<KT, COST> line(P, units, gridDim.x / beside);
        at = line.shares.begin(blockIdx.x / beside);
        to = line.shares.begin(blockIdx.x / beside + 1);
        if (at >= to) return false;
        seq = line.find(P, at, before, len);
        len = max(len, -1);
        first = true;
        item(P);
        return t1 > t0 || next(P);
    }
};

// ---- the tree --------------------------------------------------------------------
// What each node sees (itself and its ancestors; 0: absent), nodes lane and lane +
// 32 of a warp, from their parents (load_parents): up to six rounds of doubling the
// step, by shuffles.
__device__ __forceinline__ void load_parents(const Params& P, int seq, int (&up)[2]) {
    const int lane = threadIdx.x & 31;
    #pragma unroll
    for (int k = 0; k < 2; k++) up[k] = lane + 32 * k < P.n_nodes ? P.parents[(size_t)seq * P.n_nodes + lane + 32 * k] : -2;
}
__device__ __forceinline__ void tree_masks(const Params& P, int len, int (&up)[2], uint64_t (&see)[2]) {
    const int lane = threadIdx.x & 31, N = P.n_nodes;
    #pragma unroll
    for (int k = 0; k < 2; k++) {
        const int i = lane + 32 * k;
        if (up[k] < -1 || up[k] >= i || len < 0 || (long long)len + i >= P.cache.capacity) up[k] = -2;
        see[k] = 1ull << i;
    }
    for (int step = 1; step < N; step <<= 1) {
        uint64_t a[2];
        int u[2];
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            if (k == 1 && N <= 32) break;
            const int p = max(up[k], 0);   // (every lane takes part in the shuffles)
            uint64_t x = __shfl_sync(~0u, see[0], p & 31);
            int y = __shfl_sync(~0u, up[0], p & 31);
            if (N > 32) {
                const uint64_t x1 = __shfl_sync(~0u, see[1], p & 31);
                const int y1 = __shfl_sync(~0u, up[1], p & 31);
                if (p >= 32) { x = x1; y = y1; }
            }
            a[k] = up[k] >= 0 ? see[k] | x : see[k];
            u[k] = up[k] >= 0 ? y : up[k];
        }
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            if (k == 1 && N <= 32) break;
            see[k] = a[k];
            up[k] = u[k];
        }
    }
    #pragma unroll
    for (int k = 0; k < 2; k++) if (up[k] != -1) see[k] = 0;
}

// Of the 64 positions len - before .. that begin `before` positions in front of the tree's first: bit x is set where a node that
// sees the nodes `see` sees position x (all of the context, and those nodes).  see 0: an absent node, whose row is dropped.
__device__ __forceinline__ uint64_t visible(uint64_t see, int before) {
    if (before >= 64) return ~0ull;
    if (before >= 0) return ((1ull << before) - 1) | (see << before);
    return before > -64 ? see >> -before : 0ull;
}

// ---- fragments ---------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
// Four 8-bit codes to two fp16 pairs (exact): bytes (0, 1) and (2, 3) of w, or, ODD_EVEN, (0, 2) and (1, 3).
template <int STORE, bool ODD_EVEN>
__device__ __forceinline__ void codes_f16x2(uint32_t w, uint32_t& p, uint32_t& q) {
    if constexpr (STORE == QWEN_INT8) {
        // 0x6400 | u is 1024 + u; u = code + 128
        const uint32_t u = w ^ 0x80808080u;
        const __half2 k = __half2half2(__ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(u, 0x64646464u, ODD_EVEN ? 0x4240u : 0x4140u), b = __byte_perm(u, 0x64646464u, ODD_EVEN ? 0x4341u : 0x4342u);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), k), y = __hsub2(*reinterpret_cast<const __half2*>(&b), k);
        p = *reinterpret_cast<const uint32_t*>(&x);
        q = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        const uint32_t u = ODD_EVEN ? __byte_perm(w, 0, 0x3120) : w;
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "mov.b32 {lo, hi}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(p), "=r"(q) : "r"(u));
    }
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Pairs of fp32 values, one instruction for both (each rounded as alone).
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
// (a, b) * m + s
__device__ __forceinline__ void fma2(float& a, float& b, float m, float s) {
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %2};\n\tmov.b64 r, {%3, %3};\n\tfma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(a), "+f"(b) : "f"(m), "f"(s));
}
// The exponent field of a power of two above a value scale (0: NaN or infinity, which the products carry by themselves).
__device__ __forceinline__ uint32_t scale_exponent(float vs) {
    const uint32_t e = __float_as_uint(vs) >> 23 & 0xffu;
    return e == 255u ? 0u : min(e + 1, 253u);
}
// Scales of the tree may lie up to 2^14 above the context's in the same units: weight times scale is then below 2^14, within fp16.
// Beyond that rows have units of their own: the largest exponent of the tree's keys that the row sees (own: lane x's is key x's; bit
// x of v: the row sees it), or was, where none of those is 2^14 above it; a byte for each of this lane's rows.  Out of line: seldom,
// and inline it costs the loop around it 1 to 3 %.
constexpr uint32_t kTreeRise = 14;
template <int ROWS>
__device__ __noinline__ uint32_t tree_exponents(uint32_t own, uint32_t was, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3, int from, int to) {
    const uint32_t v[4] = {v0, v1, v2, v3};
    uint32_t most = 0;
    for (int x = from; x < to; x++) {
        const uint32_t e = __shfl_sync(~0u, own, x);
        uint32_t seen = 0;
        #pragma unroll
        for (int r = 0; r < ROWS; r++) seen |= (v[r] >> x & 1 ? e : 0u) << (8 * r);
        most = __vmaxu4(most, seen);
    }
    const uint32_t above = __vcmpgtu4(most, __vaddus4(was, kTreeRise * 0x01010101u));
    return (most & above) | (was & ~above);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) { return BF ? cvt_bf16x2(lo, hi) : kv::half2_bits(lo, hi); }

// ---- few rows: warp-level tensor cores ------------------------------------------------
// Bound by the cache's bytes where it is long (128 sequences of 8 nodes over 1.1 GB of
// e4m3 cache: 202 us, 5.5 TB/s; what the instructions around the conversions need is
// close behind), by the chain of plan, first loads and joining where it is short (one
// token at 1024: 9.4 us), and with 32 rows of 64 dims by the fixed latencies of its own
// instructions, three warps a scheduler filling 53 % of the issue slots (32 sequences
// of 7 nodes over 37 MB of int8 cache: 23.7 us, 3,000 cycles a tile).  Four warps; each
// owns KW keys of a tile, its own ring of kStages cp.async stages and its own (m, l, O)
// over all rows, so the loop has no block barrier; the four are joined at the end of an
// item.  16-bit caches multiply in the cache's type.  8-bit codes become fp16 (exact
// for both types): queries are scaled by a power of two per row into fp16's range (bf16
// queries; the factor returns with the score), a key's scale multiplies its scores, a
// value row's scale its weights, divided by a power of two that is at least the
// largest scale so far of the keys that the row sees (within 2^14 for the tree's), so
// the weights stay within fp16 and unseen scales have no part in them.  P is rounded
// to 16 bits (off by half a step: 2^-8 or 2^-11 relative) as the product
// with V takes it; l sums it unrounded.
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kItemCost = 2;   // what an item costs beside its tiles, in tiles: set-up, queries, joining the warps

// CTAs on an SM: where O takes 64 registers a thread three (168 in all, two stages), with 32 rows of 128 dims two (255 and three).
__host__ __device__ constexpr int attention_ctas(int rows, int dim) { return rows * dim <= 16 * 128 ? 3 : 2; }
// Keys of a tile, by the bytes of a cache row: 16 or 32 for each warp.
__host__ __device__ constexpr int tile_keys(int row_bytes) { return kWarps * (row_bytes == 256 ? 16 : 32); }
template <int STORE, int D, int MT>
struct Layout {
    static constexpr int kEs = STORE == QWEN_E4M3 || STORE == QWEN_INT8 ? 1 : 2;
    static constexpr bool k8 = kEs == 1;
    static constexpr int kRow = D * kEs;                       // bytes of a cache row
    static constexpr int KT = tile_keys(kRow);                 // keys of a tile
    static constexpr int KW = KT / kWarps;                     // keys of a warp's part of it
    static constexpr int kRows = 16 * MT;                      // query rows of an item
    static constexpr int kCtas = attention_ctas(kRows, D);        // on an SM
    static constexpr int kStages = kCtas == 3 ? 2 : 3;
    static constexpr int kPart = KW * kRow;                    // bytes of K (or V) of a warp's stage
    static constexpr int kScale = k8 ? 2 * KW * 4 : 0;         // its scales
    static constexpr int kStage = 2 * kPart + kScale;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kJoin = kWarps * kRows * (D + 2) * 4; // the warps' (O, m, l) at the end of an item (over the ring)
    static constexpr int kQ = kRing > kJoin ? kRing : kJoin;   // query rows, 16 bits
    static constexpr int kAnc = kQ + kRows * D * 2;            // tree masks
    static constexpr int kQf = kAnc + kMaxNodes * 8;           // the rows' powers of two
    static constexpr int kSmem = kQf + kRows * 4;
    static constexpr int kSlot = kRows * (D + 2);              // floats of a workspace slot: O, then (m, l) pairs
    static_assert(kRing % 16 == 0 && kJoin % 16 == 0 && kStage % 16 == 0, "rows of 16-byte pieces");
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "kCtas CTAs an SM");
};
// Byte of 16-byte piece c of row r, so that 8 rows of one piece (or 8 pieces) meet no bank twice.
template <int ROW>
__device__ __forceinline__ int swz(int r, int c) {
    if constexpr (ROW >= 128) return r * ROW + ((c ^ (r & 7)) << 4);
    else return r * ROW + ((c ^ ((r >> 1) & 3)) << 4);
}

// grid: a CTA for each share and block of rows beside it, kThreads threads, Layout::kSmem bytes.
template <int QT, int STORE, int D, int MT>
__global__ void __launch_bounds__(kThreads, attention_ctas(16 * MT, D)) attention_kernel(const Params P) {
    using L = Layout<STORE, D, MT>;
    constexpr bool BF = QT == QWEN_BF16 && !L::k8;       // type of the products
    constexpr int KW = L::KW, NT = KW / 8, DT = D / 8, KS = D / 16, kStages = L::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    uint8_t* ring = smem + warp * kStages * L::kStage;
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + L::kAnc);
    float* qf = reinterpret_cast<float*>(smem + L::kQf);
    pdl_wait();
    pdl_launch_dependents();   // after the wait: what the joining kernel reads early (lens) is then complete

    Items<L::KT, kItemCost, L::kRows> it;
    if (!it.start(P)) return;
    const int M = P.n_nodes * P.group;
    do {
        const int seq = it.seq, len = it.len, end = it.end, h = it.h, r_base = it.r_base, t0 = it.t0, t1 = it.t1;
        const size_t head = (size_t)seq * P.cache.seq_stride + (size_t)h * P.cache.head_stride;
        const uint8_t *kb = P.cache.k + head * L::kEs, *vb = P.cache.v + head * L::kEs;
        const float *ksb = L::k8 ? P.cache.ks + head / D : nullptr, *vsb = L::k8 ? P.cache.vs + head / D : nullptr;

        auto load = [&](int t, int s) {   // this warp's part of tile t into stage s; positions >= end as zeros
            const uint32_t st = smem_addr(ring + s * L::kStage);
            const int k0 = t * L::KT + warp * KW;
            // the part is KW * kRow bytes in a row: lane's piece i lies 512 i bytes on, in row r0 + kStep i; with r0 < kStep the
            // swizzle's row bits of the two add up without a carry
            constexpr int kChunks = L::kRow / 16, kPer = KW * kChunks / 32, kStep = 32 / kChunks;
            const uint32_t off0 = swz<L::kRow>(lane / kChunks, lane % kChunks);
            const uint8_t *ksrc = kb + (size_t)k0 * L::kRow + lane * 16, *vsrc = vb + (size_t)k0 * L::kRow + lane * 16;
            if (k0 + KW <= end) {
                #pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const uint32_t off = (off0 ^ (L::kRow >= 128 ? ((kStep * i) & 7) << 4 : 0)) + 512 * i;
                    cp_async16(st + off, ksrc + 512 * i);
                    cp_async16(st + L::kPart + off, vsrc + 512 * i);
                }
            } else {
                #pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const uint32_t off = (off0 ^ (L::kRow >= 128 ? ((kStep * i) & 7) << 4 : 0)) + 512 * i;
                    const bool live = k0 + lane / kChunks + kStep * i < end;
                    cp_async16(st + off, live ? ksrc + 512 * i : kb, live);
                    cp_async16(st + L::kPart + off, live ? vsrc + 512 * i : vb, live);
                }
            }
            if constexpr (L::k8) {
                static_assert(KW == 32, "one scale a lane");
                const bool live = k0 + lane < end;
                const size_t off = live ? k0 + lane : 0;
                cp_async4(st + 2 * L::kPart + 4 * lane, ksb + off, live);
                cp_async4(st + 2 * L::kPart + 4 * KW + 4 * lane, vsb + off, live);
            }
        };
        #pragma unroll
        for (int s = 0; s < kStages - 1; s++) {
            if (t0 + s < t1) load(t0 + s, s);
            cp_async_commit();
        }
        // queries to shared memory, 16 bits; for 8-bit caches fp16 with the dims of each 16 in
        // the order in which the K codes come out of ldmatrix: 4j, 4j+1 at 2j, 4j+2, 4j+3 at 8 + 2j
        constexpr int kLanes = D / 8, kQStep = kThreads / kLanes, kQPer = L::kRows / kQStep;   // 8 elements a thread
        const int part = tid % kLanes, rq = tid / kLanes;
        int up[2];
        uint64_t nodes[2];        // what nodes lane and lane + 32 see
        load_parents(P, seq, up);
        uint4 qv[kQPer];
        #pragma unroll
        for (int i = 0; i < kQPer; i++) {
            const int row = r_base + rq + i * kQStep, node = P.node_of(row);
            qv[i] = make_uint4(0, 0, 0, 0);
            if (row < M)
                qv[i] = *reinterpret_cast<const uint4*>(P.q + (((size_t)seq * P.n_nodes + node) * (size_t)P.ldq +
                                                               (size_t)(h * P.group + row - node * P.group) * D + part * 8) * 2);
        }
        tree_masks(P, len, up, nodes);
        uint64_t see[2 * MT];     // what this lane's rows see of the tree
        #pragma unroll
        for (int i = 0; i < 2 * MT; i++) {
            const int row = r_base + 16 * (i >> 1) + g + 8 * (i & 1), node = min(P.node_of(row), kMaxNodes - 1);
            const uint64_t a = __shfl_sync(~0u, nodes[0], node & 31), b = __shfl_sync(~0u, nodes[1], node & 31);
            see[i] = row < M ? (node < 32 ? a : b) : 0;
        }
        if (warp == 0) {
            anc[lane] = nodes[0];
            anc[lane + 32] = nodes[1];
        }
        const uint32_t flip = P.scale_log2 < 0.f ? 0x80008000u : 0u;   // a negative scale: its sign goes to the queries
        #pragma unroll
        for (int i = 0; i < kQPer; i++) {
            const int r = rq + i * kQStep;
            uint32_t x[4] = {qv[i].x ^ flip, qv[i].y ^ flip, qv[i].z ^ flip, qv[i].w ^ flip};
            if constexpr (!L::k8) {
                *reinterpret_cast<uint4*>(smem + L::kQ + swz<D * 2>(r, part)) = make_uint4(x[0], x[1], x[2], x[3]);
            } else {
                if constexpr (QT == QWEN_BF16) {
                    uint32_t m = 0;
                    #pragma unroll
                    for (int e = 0; e < 4; e++) m = max(m, max(x[e] & 0x7fffu, (x[e] >> 16) & 0x7fffu));
                    #pragma unroll
                    for (int o = 1; o < kLanes; o <<= 1) m = max(m, __shfl_xor_sync(~0u, m, o));
                    // 2^e <= the row's largest magnitude < 2^(e+1); infinities and NaN go through as they are
                    const int e = min(max((int)(m >> 7), 1), 253);
                    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                    #pragma unroll
                    for (int e2 = 0; e2 < 4; e2++) x[e2] = kv::half2_bits(bf_lo(x[e2]) * down, bf_hi(x[e2]) * down);
                    if (part == 0) qf[r] = __uint_as_float((uint32_t)e << 23);
                } else if (part == 0) {
                    qf[r] = 1.0f;
                }
                // this thread's 8 dims are the first or second half of a 16: pairs p = 0..3 (dims 2p, 2p+1) of it
                const int half = part & 1, chunk = part & ~1;
                #pragma unroll
                for (int p = 0; p < 4; p++) {
                    const int d = 8 * half + 2 * p, jj = d >> 2, k = (d & 2) ? 8 + 2 * jj : 2 * jj;
                    *reinterpret_cast<uint32_t*>(smem + L::kQ + swz<D * 2>(r, chunk + (k >> 3)) + (k & 7) * 2) = x[p];
                }
            }
        }
        __syncthreads();
        float c[2 * MT];          // these rows' score factors (kept above 0: -inf * 0 would be NaN)
        #pragma unroll
        for (int i = 0; i < 2 * MT; i++) {
            const float a = fabsf(P.scale_log2);
            c[i] = fmaxf(L::k8 ? a * qf[16 * (i >> 1) + g + 8 * (i & 1)] : a, 1e-37f);
        }
        uint32_t qa[MT == 1 ? KS : 1][4];   // one block of rows: its fragments stay in registers
        auto q_frag = [&](int mt, int ks, uint32_t (&a)[4]) {
            const int r = 16 * mt + (lane & 15), p = 2 * ks + (lane >> 4);
            ldsm_x4(smem_addr(smem + L::kQ + swz<D * 2>(r, p)), a[0], a[1], a[2], a[3]);
        };
        if constexpr (MT == 1) {
            #pragma unroll
            for (int ks = 0; ks < KS; ks++) q_frag(0, ks, qa[ks]);
        }

        float o[MT][DT][4], m[2 * MT], l[2 * MT];
        #pragma unroll
        for (int mt = 0; mt < MT; mt++)
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int e = 0; e < 4; e++) o[mt][d][e] = 0.f;
        #pragma unroll
        for (int i = 0; i < 2 * MT; i++) { m[i] = -INFINITY; l[i] = 0.f; }
        uint32_t ve = 1;   // 8-bit caches: O is in units of 2^(ve - 127); above 255 a byte for each of this lane's rows

        for (int t = t0; t < t1; t++) {
            {
                const int ahead = t + kStages - 1;
                if (ahead < t1) load(ahead, (ahead - t0) % kStages);
                cp_async_commit();
            }
            cp_async_wait<kStages - 1>();
            __syncwarp();
            uint8_t* st = ring + (t - t0) % kStages * L::kStage;
            const int k0 = t * L::KT + warp * KW;
            if (k0 < end) {
                // ---- scores ----
                float s[MT][NT][4];
                #pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    #pragma unroll
                    for (int i = 0; i < NT; i++)
                        #pragma unroll
                        for (int e = 0; e < 4; e++) s[mt][i][e] = 0.f;
                #pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t a[MT][4];
                    #pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if constexpr (MT == 1) { a[0][0] = qa[ks][0]; a[0][1] = qa[ks][1]; a[0][2] = qa[ks][2]; a[0][3] = qa[ks][3]; }
                        else q_frag(mt, ks, a[mt]);
                    }
                    if constexpr (!L::k8) {
                        #pragma unroll
                        for (int i = 0; i < NT; i += 2) {   // keys 8i .. 8i+15, dims 16 ks .. +15
                            uint32_t b[4];
                            ldsm_x4(smem_addr(st + swz<L::kRow>(8 * i + (lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1))), b[0], b[1], b[2], b[3]);
                            #pragma unroll
                            for (int mt = 0; mt < MT; mt++) {
                                mma16816<BF>(s[mt][i], a[mt], b[0], b[1]);
                                mma16816<BF>(s[mt][i + 1], a[mt], b[2], b[3]);
                            }
                        }
                    } else {                                // four key groups of one 16-byte piece
                        uint32_t b[4];
                        ldsm_x4(smem_addr(st + swz<L::kRow>(lane, ks)), b[0], b[1], b[2], b[3]);
                        #pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t b0, b1;
                            codes_f16x2<STORE, false>(b[i], b0, b1);
                            #pragma unroll
                            for (int mt = 0; mt < MT; mt++) mma16816<BF>(s[mt][i], a[mt], b0, b1);
                        }
                    }
                }
                const bool tail = k0 + KW > len;   // the same for the warp: some keys are the tree's, or past the end
                float vs[NT][2];
                if constexpr (L::k8) {
                    const float* sc = reinterpret_cast<const float*>(st + 2 * L::kPart);
                    #pragma unroll
                    for (int i = 0; i < NT; i++) {
                        const float2 ks2 = *reinterpret_cast<const float2*>(sc + 8 * i + 2 * j);
                        const float2 vs2 = *reinterpret_cast<const float2*>(sc + KW + 8 * i + 2 * j);
                        vs[i][0] = vs2.x;
                        vs[i][1] = vs2.y;
                        #pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            mul2(s[mt][i][0], s[mt][i][1], ks2.x, ks2.y);
                            mul2(s[mt][i][2], s[mt][i][3], ks2.x, ks2.y);
                        }
                    }
                }
                uint32_t vis[2 * MT];   // bit x: the row sees position k0 + x (KW <= 32)
                if (tail) {
                    #pragma unroll
                    for (int r = 0; r < 2 * MT; r++) vis[r] = (uint32_t)visible(see[r], len - k0);
                }
                auto sees = [&](int row, int x) { return (vis[row] >> x & 1) != 0; };
                if (tail) {
                    #pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        #pragma unroll
                        for (int i = 0; i < NT; i++)
                            #pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (!sees(2 * mt + (e >> 1), 8 * i + 2 * j + (e & 1))) s[mt][i][e] = -INFINITY;
                }
                // ---- softmax ----
                uint32_t up = 0;        // 8-bit: the rise of ve, or of its bytes
                bool apart = false;     // rows have units of their own (the same for the warp)
                if constexpr (L::k8) {
                    const uint32_t own = scale_exponent(reinterpret_cast<const float*>(st + 2 * L::kPart)[KW + lane]);
                    const bool all_see = k0 + lane < len + (P.n_nodes == 1);   // (a single node's row sees itself, or is dropped)
                    const uint32_t e = __reduce_max_sync(~0u, all_see ? own : 0u);
                    apart = ve > 255u || (tail && __any_sync(~0u, !all_see && own > max(e, ve) + kTreeRise));
                    if (!apart) {
                        if (e > ve) { up = e - ve; ve = e; }
                        const float vinv = __uint_as_float((254u - ve) << 23);
                        #pragma unroll
                        for (int i = 0; i < NT; i++) mul2(vs[i][0], vs[i][1], vinv, vinv);
                    } else {
                        const uint32_t was = ve > 255u ? ve : ve * 0x01010101u;
                        ve = tree_exponents<2 * MT>(own, __vmaxu4(was, e * 0x01010101u), vis[0], vis[1], vis[2 * MT - 2], vis[2 * MT - 1], max(len - k0, 0),
                                                    min(KW, end - k0));
                        up = ve - was;   // (no byte falls)
                    }
                }
                float f[2 * MT];
                bool moved = up != 0;
                #pragma unroll
                for (int r = 0; r < 2 * MT; r++) {
                    float mx = -INFINITY;
                    #pragma unroll
                    for (int i = 0; i < NT; i++) mx = fmaxf(mx, fmaxf(s[r >> 1][i][2 * (r & 1)], s[r >> 1][i][2 * (r & 1) + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
                    const float mn = fmaxf(m[r], mx == -INFINITY ? mx : mx * c[r]);
                    const float base = mn == -INFINITY ? 0.f : mn;
                    f[r] = exp2_approx(m[r] - base);
                    moved |= mn > m[r];
                    m[r] = mn;
                    float sum0 = 0.f, sum1 = 0.f;
                    #pragma unroll
                    for (int i = 0; i < NT; i++) {
                        float &x = s[r >> 1][i][2 * (r & 1)], &y = s[r >> 1][i][2 * (r & 1) + 1];
                        fma2(x, y, c[r], -base);
                        x = exp2_approx(x);
                        y = exp2_approx(y);
                        add2(sum0, sum1, x, y);
                        if constexpr (L::k8) mul2(x, y, vs[i][0], vs[i][1]);
                    }
                    l[r] = l[r] * f[r] + (sum0 + sum1);
                }
                if (L::k8 && tail) {   // (a scale that a row does not see may be anything)
                    #pragma unroll
                    for (int r = 0; r < 2 * MT; r++)
                        #pragma unroll
                        for (int i = 0; i < NT; i++)
                            #pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (!sees(r, 8 * i + 2 * j + e)) s[r >> 1][i][2 * (r & 1) + e] = 0.f;
                    if (apart) {
                        #pragma unroll
                        for (int r = 0; r < 2 * MT; r++) {
                            const float vinv = __uint_as_float((254u - (ve >> (8 * r) & 0xffu)) << 23);
                            #pragma unroll
                            for (int i = 0; i < NT; i++) mul2(s[r >> 1][i][2 * (r & 1)], s[r >> 1][i][2 * (r & 1) + 1], vinv, vinv);
                        }
                    }
                }
                if (__any_sync(~0u, moved)) {
                    if constexpr (L::k8) {
                        if (!apart) {
                            const float w = up < 127u ? __uint_as_float((127u - up) << 23) : 0.f;
                            #pragma unroll
                            for (int r = 0; r < 2 * MT; r++) f[r] *= w;
                        } else {
                            #pragma unroll
                            for (int r = 0; r < 2 * MT; r++) {
                                const uint32_t u = up >> (8 * r) & 0xffu;
                                f[r] *= u < 127u ? __uint_as_float((127u - u) << 23) : 0.f;
                            }
                        }
                    }
                    #pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        #pragma unroll
                        for (int d = 0; d < DT; d++)
                            #pragma unroll
                            for (int e = 0; e < 4; e += 2) mul2(o[mt][d][e], o[mt][d][e + 1], f[2 * mt + (e >> 1)], f[2 * mt + (e >> 1)]);
                }
                uint8_t* sv = st + L::kPart;
                // the dim of column e (0, 1) of this lane in column tile d
                auto dim_of = [&](int d, int e) { return L::k8 ? (d >> 1) * 16 + 4 * j + 2 * e + (d & 1) : 8 * d + 2 * j + e; };
                if (STORE != QWEN_INT8 && tail) {
                    // An infinity or NaN in a V row of the tree may only reach the nodes that see the row, but 0 * NaN
                    // in the product is NaN: such values are added here, to those, and zeroed before the product.
                    const int from = max(len - k0, 0);
                    bool odd = false;
                    for (int i = lane; i < (KW - from) * (L::kRow / 4); i += 32) {
                        const int r = from + i / (L::kRow / 4), b = i % (L::kRow / 4);
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(sv + swz<L::kRow>(r, b >> 2) + 4 * (b & 3));
                        if constexpr (L::k8) {
                            #pragma unroll
                            for (int e = 0; e < 4; e++) odd |= ((w >> (8 * e)) & 0x7fu) == 0x7fu;
                        } else {
                            constexpr uint32_t kExp = QT == QWEN_BF16 ? 0x7f80u : 0x7c00u;
                            odd |= (w & kExp) == kExp || ((w >> 16) & kExp) == kExp;
                        }
                    }
                    if (__any_sync(~0u, odd)) {
                        constexpr uint32_t kExp = L::k8 ? 0x7fu : QT == QWEN_BF16 ? 0x7f80u : 0x7c00u;
                        for (int r = from; r < KW; r++)
                            #pragma unroll
                            for (int d = 0; d < DT; d++)
                                #pragma unroll
                                for (int e = 0; e < 2; e++) {
                                    const int byte = dim_of(d, e) * L::kEs;
                                    const uint8_t* p = sv + swz<L::kRow>(r, byte >> 4) + (byte & 15);
                                    const uint32_t w = L::k8 ? *p : *reinterpret_cast<const uint16_t*>(p);
                                    if ((w & kExp) != kExp) continue;
                                    const float x = L::k8 ? NAN : QT == QWEN_BF16 ? bf2f((uint16_t)w) : __half2float(__ushort_as_half((uint16_t)w));
                                    #pragma unroll
                                    for (int q = 0; q < 2 * MT; q++)
                                        if (sees(q, r)) o[q >> 1][d][2 * (q & 1) + e] += x;
                                }
                        __syncwarp();
                        for (int i = lane; i < (KW - from) * (L::kRow / L::kEs); i += 32) {
                            const int r = from + i / D, byte = i % D * L::kEs;
                            uint8_t* p = sv + swz<L::kRow>(r, byte >> 4) + (byte & 15);
                            if constexpr (L::k8) { if ((*p & kExp) == kExp) *p = 0; }
                            else { uint16_t* w = reinterpret_cast<uint16_t*>(p); if ((*w & kExp) == kExp) *w = 0; }
                        }
                        __syncwarp();
                    }
                }
                // ---- O += P V ----
                #pragma unroll
                for (int kk = 0; kk < KW / 16; kk++) {
                    uint32_t a[MT][4];
                    #pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        a[mt][0] = pack2<BF>(s[mt][2 * kk][0], s[mt][2 * kk][1]);
                        a[mt][1] = pack2<BF>(s[mt][2 * kk][2], s[mt][2 * kk][3]);
                        a[mt][2] = pack2<BF>(s[mt][2 * kk + 1][0], s[mt][2 * kk + 1][1]);
                        a[mt][3] = pack2<BF>(s[mt][2 * kk + 1][2], s[mt][2 * kk + 1][3]);
                    }
                    #pragma unroll
                    for (int p = 0; p < L::kRow / 16; p += 2) {   // two 16-byte pieces of the 16 keys' rows
                        uint32_t b[4];
                        ldsm_x4_t(smem_addr(sv + swz<L::kRow>(16 * kk + (lane & 15), p + (lane >> 4))), b[0], b[1], b[2], b[3]);
                        if constexpr (!L::k8) {
                            #pragma unroll
                            for (int mt = 0; mt < MT; mt++) {
                                mma16816<BF>(o[mt][p], a[mt], b[0], b[1]);
                                mma16816<BF>(o[mt][p + 1], a[mt], b[2], b[3]);
                            }
                        } else {
                            #pragma unroll
                            for (int q = 0; q < 2; q++) {
                                uint32_t e0, e1, d0, d1;   // even and odd dims of the piece, keys 0-7 and 8-15
                                codes_f16x2<STORE, true>(b[2 * q], e0, d0);
                                codes_f16x2<STORE, true>(b[2 * q + 1], e1, d1);
                                #pragma unroll
                                for (int mt = 0; mt < MT; mt++) {
                                    mma16816<BF>(o[mt][2 * (p + q)], a[mt], e0, e1);
                                    mma16816<BF>(o[mt][2 * (p + q) + 1], a[mt], d0, d1);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();   // the stage is free
        }
        cp_async_wait<0>();
        __syncthreads();    // the rings are free: the warps' results go over them
        float* join = reinterpret_cast<float*>(smem);               // [warp][row][D], then [warp][row][2]
        float* join_ml = join + kWarps * L::kRows * D;
        #pragma unroll
        for (int r = 0; r < 2 * MT; r++) {
            const float unit_v = L::k8 ? __uint_as_float((ve > 255u ? ve >> (8 * r) & 0xffu : ve) << 23) : 1.0f;
            float sum = l[r];
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            const int row = 16 * (r >> 1) + g + 8 * (r & 1);
            if (j == 0) {
                join_ml[(warp * L::kRows + row) * 2] = m[r];
                join_ml[(warp * L::kRows + row) * 2 + 1] = sum;
            }
            #pragma unroll
            for (int d = 0; d < DT; d++)
                #pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int dim = L::k8 ? (d >> 1) * 16 + 4 * j + 2 * e + (d & 1) : 8 * d + 2 * j + e;
                    join[(warp * L::kRows + row) * D + dim] = o[r >> 1][d][2 * (r & 1) + e] * unit_v;
                }
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == it.n;
        float* slot = P.work + (size_t)(2 * blockIdx.x + (it.first ? 0 : 1)) * L::kSlot;
        for (int i = tid; i < L::kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = i % (D / 4) * 4, row = r_base + r;
            if (row >= M) break;
            const bool present = anc[P.node_of(row)] != 0;
            float mm = -INFINITY, ll = 0.f;
            #pragma unroll
            for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, join_ml[(w * L::kRows + r) * 2]);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            #pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float mw = join_ml[(w * L::kRows + r) * 2], lw = join_ml[(w * L::kRows + r) * 2 + 1];
                const float fw = mm == -INFINITY ? 1.0f : exp2_approx(mw - mm);
                const float4 b = *reinterpret_cast<const float4*>(join + (w * L::kRows + r) * D + d);
                ll += lw * fw;
                a.x += b.x * fw; a.y += b.y * fw; a.z += b.z * fw; a.w += b.w * fw;
            }
            if (!present) { mm = -INFINITY; ll = 0.f; a = make_float4(0.f, 0.f, 0.f, 0.f); }
            if (whole) {
                const float inv = ll == 0.f ? 0.f : 1.0f / ll;
                const int node = P.node_of(row), hq = h * P.group + row - node * P.group;
                uint8_t* dst = P.out + (((size_t)seq * P.n_nodes + node) * (size_t)P.ldo + (size_t)hq * D + d) * 2;
                *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<QT == QWEN_BF16>(a.x * inv, a.y * inv), pack2<QT == QWEN_BF16>(a.z * inv, a.w * inv));
            } else {
                *reinterpret_cast<float4*>(slot + r * D + d) = a;
                if (d == 0) *reinterpret_cast<float2*>(slot + L::kRows * D + 2 * r) = make_float2(mm, ll);
            }
        }
        __syncthreads();
    } while (it.next(P));
}

// Bound by latency: the plan, two rounds of loads from the L2.
// Joins the partial results of the items that cross a border between shares:
// blocks (x, y) take item x, or where there are more items than shares the one that
// begins in share x and goes on in the next.
// ACROSS: a slot holds O as [dim / 4][row] (the tensor-memory kernel: a thread a
// row) and a thread here joins 8 dims of a row, lanes along the rows; otherwise O
// is [row][dim] and a thread joins 4 dims, lanes along the dims.
constexpr int kJoinThreads = 128;
template <int D, int ROWS, bool ACROSS>
__host__ __device__ constexpr int join_blocks() { return ROWS * (ACROSS ? D / 8 : D / 4) / kJoinThreads; }
template <int QT, int KT, int COST, int D, int ROWS, bool ACROSS>
__global__ void __launch_bounds__(kJoinThreads, 6) combine_kernel(const Params P) {
    constexpr int kSlot = ROWS * (D + 2), kVec = ACROSS ? 2 : 1, kAhead = ACROSS ? 5 : 8;   // float4s a thread; partial results loaded at once
    const int beside = P.beside, unit_blocks = beside == 1 ? P.row_blocks : 1, units = P.n_kv_heads * unit_blocks;
    const int i = blockIdx.x / beside, lane = blockIdx.x - i * beside;
    int s = 0, e = 0, seq, unit = 0;            // the item: its positions
    const Line<KT, COST> line(P, units, P.groups);
    const Shares& shares = line.shares;
    if (P.by_item) {
        seq = i / units;
        unit = i - seq * units;
        const int per = seq_tiles<KT>(P, P.lens[seq]) + COST;
        s = line.before(P, seq) + unit * per;
        e = s + per;
    } else {
        const int from = shares.begin(i), edge = shares.begin(i + 1);
        seq = 0;
        if (edge > from && edge < shares.n) {
            int before, len;
            seq = line.find(P, edge, before, len);
            const int per = seq_tiles<KT>(P, len) + COST;
            unit = (int)((unsigned)(edge - before) / (unsigned)per);
            s = before + unit * per;
            e = s + per;
            if (s >= edge || s < from) e = s;   // it begins at the border, or before this share
        }
    }
    pdl_wait();   // on every path: this kernel may not end before the one that it joins
    if (s >= e) return;
    const int begun = shares.of(s + COST), last = shares.of(e - 1);   // the shares with its tiles
    if (begun == last) return;                  // one has them all and has written the rows
    const bool second = shares.begin(begun) < s;   // a share that begins before the item holds it in its second slot
    const int t = blockIdx.y * kJoinThreads + threadIdx.x;
    const int h = unit / unit_blocks, r = ACROSS ? t % ROWS : t / (D / 4), d = ACROSS ? t / ROWS * 8 : t % (D / 4) * 4;
    const int row = (unit - h * unit_blocks + lane) * ROWS + r;
    if (row >= P.n_nodes * P.group) return;
    float mm = -INFINITY, ll = 0.f;
    float4 a[kVec];
    #pragma unroll
    for (int v = 0; v < kVec; v++) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = begun; k0 <= last; k0 += kAhead) {
        float2 ml[kAhead];
        float4 b[kAhead][kVec];
        #pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int k = k0 + j;
            ml[j] = make_float2(-INFINITY, 0.f);
            #pragma unroll
            for (int v = 0; v < kVec; v++) b[j][v] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k > last) continue;
            const float* slot = P.work + (2 * ((size_t)k * beside + lane) + (k == begun && second ? 1 : 0)) * kSlot;
            ml[j] = *reinterpret_cast<const float2*>(slot + ROWS * D + 2 * r);
            #pragma unroll
            for (int v = 0; v < kVec; v++) b[j][v] = *reinterpret_cast<const float4*>(ACROSS ? slot + ((d / 4 + v) * ROWS + r) * 4 : slot + r * D + d);
        }
        float mn = mm;
        #pragma unroll
        for (int j = 0; j < kAhead; j++) mn = fmaxf(mn, ml[j].x);
        const float f0 = mn == -INFINITY ? 1.0f : exp2_approx(mm - mn);
        ll *= f0;
        #pragma unroll
        for (int v = 0; v < kVec; v++) { a[v].x *= f0; a[v].y *= f0; a[v].z *= f0; a[v].w *= f0; }
        #pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const float f1 = mn == -INFINITY ? 1.0f : exp2_approx(ml[j].x - mn);
            ll += ml[j].y * f1;
            #pragma unroll
            for (int v = 0; v < kVec; v++) {
                a[v].x += b[j][v].x * f1; a[v].y += b[j][v].y * f1; a[v].z += b[j][v].z * f1; a[v].w += b[j][v].w * f1;
            }
        }
        mm = mn;
    }
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;
    const int node = P.node_of(row), hq = h * P.group + row - node * P.group;
    uint8_t* dst = P.out + (((size_t)seq * P.n_nodes + node) * (size_t)P.ldo + (size_t)hq * D + d) * 2;
    #pragma unroll
    for (int v = 0; v < kVec; v++)
        *reinterpret_cast<uint2*>(dst + 8 * v) = make_uint2(pack2<QT == QWEN_BF16>(a[v].x * inv, a[v].y * inv), pack2<QT == QWEN_BF16>(a[v].z * inv, a[v].w * inv));
}

}  // namespace ta
}  // namespace qb
