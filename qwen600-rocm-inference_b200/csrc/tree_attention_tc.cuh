// tree_attention_tc.cuh — tree attention of many query rows a K/V head on the
// sm_100a tensor cores (tcgen05.mma with accumulators in tensor memory); the
// mathematics and the division of the work are tree_attention.cuh's.  No
// reference counterpart.
//
// With 33 and more rows (nodes times query heads a K/V head) the warp-level products no
// longer fit under the cache's bytes, and blocks of 32 rows would read them several
// times (bf16, 40 rows, 16 sequences at 2048: 40 us here, 57 us there; 24 rows: 40 us
// here, 37 us there).  Here an item has 128 rows, tiles have 128 keys, and 256 softmax
// threads serve them, two a row (64 keys each; they agree on the row's maximum through
// shared memory).  A tile's two products take 512 cycles each (4,096 multiply-adds a
// cycle), its 16,384 exponentials 1,024 (16 a cycle), its bytes (bf16, 128 dims) 2,800
// of an SM's share of the memory bandwidth.  S and P have two buffers each, so that the
// next tile's S is formed during a tile's exponentials. (Two blocks of rows over shared
// tiles leave tensor memory for one S each: a chain of products and exponentials
// without overlap, 2,800 cycles a block and tile.)
//
// Measured, bf16: one sequence of 64 nodes at 8128 19.4 us with the joining (5.2 us of
// memory traffic; 3,000 cycles each for the plan and the first products), 8 ragged
// sequences of 64 nodes and 8 query heads a K/V head 119 to 153 us by the lengths that
// are drawn (42 us of products at the rate of a large matrix product, for lengths of
// the mean): bound by the chain of a tile, 2,100 cycles from its
// scores over the maximum and the exponentials to P (the pipes of both are a third busy).
// 8-bit caches: 16 x 20 nodes at 2048 59 us against bf16's 40, bound by the four producer
// warps (2,200 cycles a part of a tile: copies in, codes read, fp16 written, beside the
// scales' and the products' reads of shared memory).
//
// Warps: 0-7 softmax (warp w reads the tensor-memory lanes 32 (w % 4) .., its
// rows; w / 4 picks the keys' half), 8-11 producers, 12 issues the products.  S = Q
// K^T, P (16 bits) and O are in tensor memory; Q, K and V in shared memory, rows
// of 64 dims in the 128-byte swizzle: K is a K-major operand, V an MN-major one
// (its rows are keys, so the product P V needs no transposed copy).  K and V
// parts of tiles go through one ring in the order in which they are used.  16-bit
// rows arrive by cp.async; 8-bit rows arrive in a thread-private staging ring, become
// fp16 (exact) and are stored swizzled by the thread that loaded them.  Every
// wait is bounded; where one runs out, the item's rows become NaN.
#pragma once
#include "gemm_tc.cuh"
#include "tree_attention.cuh"

namespace qb {
namespace ta {

constexpr int kTcKT = 128, kTcRows = 128, kTcProducers = 128, kTcSoftmax = 256, kTcThreads = 416;
constexpr int kScaleRing = 8;

template <int STORE, int D>
struct TcLayout {
    static constexpr bool k8 = STORE == QWEN_E4M3 || STORE == QWEN_INT8;
    static constexpr int kRow = D * (k8 ? 1 : 2);          // bytes of a cache row
    static constexpr int kHalf = kTcKT * D * 2;            // K or V of a tile, or the query rows: 16 bits
    static constexpr int kRing = D == 64 ? (k8 ? 6 : 8) : k8 ? 4 : 5;   // K / V parts in flight
    static constexpr int kRawHalf = k8 ? kTcKT * D : 0;
    static constexpr int kRawRing = k8 ? (D == 64 ? 4 : 3) : 0;
    static constexpr int kQ = 0;
    static constexpr int kKV = kQ + kHalf;
    static constexpr int kRaw = kKV + kRing * kHalf;
    static constexpr int kScales = kRaw + kRawRing * kRawHalf;                        // [ring][ks 128, vs 128]
    static constexpr int kXm = kScales + (k8 ? kScaleRing * 2 * kTcKT * 4 : 0);       // [tile parity][half][row] maxima, then sums
    static constexpr int kAnc = kXm + 2 * 2 * kTcRows * 4;
    static constexpr int kQf = kAnc + kMaxNodes * 8;                                  // the rows' powers of two
    static constexpr int kVe = kQf + kTcRows * 4;                                       // [ring][producer warp] largest exponent of vs
    static constexpr int kBar = kVe + kScaleRing * 4 * 4;
    static constexpr int kBars = 2 * kRing + kScaleRing + 8;
    static constexpr int kMisc = kBar + kBars * 8;                                    // tensor-memory address, fault, odd[8]
    static constexpr int kSmem = kMisc + 48 + 1024;
    static constexpr int kSlot = kTcRows * (D + 2);
    static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
    static_assert(2 * kSmem > 228 * 1024, "one CTA an SM: the kernel allocates all of tensor memory");
};

// Instruction descriptor, kind::f16: D fp32 (bits 4-5), A and B bf16 (1) or fp16 (0) at bits 7 and 10, B MN-major at
// bit 16, N >> 3 at bit 17, M >> 4 at bit 24.
template <bool BF>
__host__ __device__ constexpr uint32_t tc_idesc(int N, bool mn_major_b) {
    return (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | (mn_major_b ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
}
// MN-major operand in the 128-byte swizzle: rows (keys) of 64 dims, 8 rows 1024 bytes, the next 64 dims `block` bytes on.
__device__ __forceinline__ uint64_t mn_major_sw128_desc(uint32_t saddr, uint32_t block) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1u << 46) |
           ((uint64_t)2u << 61);
}
// D (tensor memory) += A (tensor memory, 128 rows x 16) . B
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
          "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const float (&v)[32]) {
    uint32_t a[16], b[16];
    #pragma unroll
    for (int i = 0; i < 16; i++) { a[i] = __float_as_uint(v[i]); b[i] = __float_as_uint(v[16 + i]); }
    tc_st16(taddr, a);
    tc_st16(taddr + 16, b);
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Bounded wait without a suspend-time hint: these waits are short, and a thread that sleeps wakes late.
__device__ __forceinline__ bool mbar_spin(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
    uint64_t since = 0;
    for (uint32_t n = 0;; n++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((n & 255u) == 255u) {
            const uint64_t now = global_ns();
            if (!since) since = now;
            else if (now - since > limit_ns) return false;
        }
    }
}

// An item's K and V parts in the order in which the products take them: K 0, K 1, V 0, K 2, V 1, ..., K n-1, V n-2, V n-1.  (In
// the order K 0, V 0, K 1, ... a K part would wait for the slot of a V part that is taken a tile later.)
__device__ __forceinline__ uint32_t k_part(int t) { return t == 0 ? 0u : 2u * t - 1u; }
__device__ __forceinline__ uint32_t v_part(int t, int n) { return (uint32_t)min(2 * t + 2, 2 * n - 1); }
__device__ __forceinline__ int part_tile(int x, int n, int& kv) {   // part x's tile; kv: 0 K, 1 V
    kv = x > 0 && (!(x & 1) || x == 2 * n - 1);
    return x == 2 * n - 1 ? n - 1 : kv ? x / 2 - 1 : (x + 1) / 2;
}

constexpr int kTcItemCost = 3;   // what an item costs beside its tiles, in tiles: queries, first products, rows out

// grid: a CTA (one an SM) for each share and block of rows beside it, kTcThreads threads, TcLayout::kSmem bytes.
template <int QT, int STORE, int D>
__global__ void __launch_bounds__(kTcThreads, 1) attention_tc_kernel(const Params P) {
    using L = TcLayout<STORE, D>;
    using namespace qb::tc;
    constexpr bool BF = QT == QWEN_BF16 && !L::k8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBar);   // [kRing] a K or V part is in place (128 producers)
    uint64_t* empty = full + L::kRing;                              // [kRing] its products are done
    uint64_t* scaled = empty + L::kRing;                            // [kScaleRing] a tile's scales are in place (128 producers)
    // [2]: the S / P buffer of a tile's parity
    uint64_t* sfull = scaled + kScaleRing;                          // S formed
    uint64_t* pfull = sfull + 2;                                    // P written, O rescaled (8 warps)
    uint64_t* pvdone = sfull + 4;                                   // P V added
    uint64_t* qfull = sfull + 6;                                    // the item's queries (8 warps)
    uint64_t* drained = sfull + 7;                                  // all products are done, at the end
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
    volatile int* fault = reinterpret_cast<int*>(smem + L::kMisc + 4);
    volatile int* odd = fault + 1;                                  // [8] an item's V rows of the tree hold an infinity or NaN
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + L::kAnc);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_wait();
    pdl_launch_dependents();         // after the wait: what the joining kernel reads early (lens) is then complete
    Items<kTcKT, kTcItemCost, kTcRows> it;       // every role walks it alike
    const bool busy = it.start(P);               // the same for the whole CTA
    if (tid == 0) {
        for (int i = 0; i < L::kRing; i++) { mbar_init(&full[i], kTcProducers + (i == P.withheld)); mbar_init(&empty[i], 1); }
        for (int i = 0; i < kScaleRing; i++) mbar_init(&scaled[i], kTcProducers);
        for (int i = 0; i < 2; i++) { mbar_init(&sfull[i], 1); mbar_init(&pfull[i], 8); mbar_init(&pvdone[i], 1); }
        mbar_init(qfull, 8);
        mbar_init(drained, 1);
        fence_barrier_init();
        *fault = 0;
        for (int i = 0; i < 8; i++) odd[i] = 0;
    }
    constexpr int kProducer = 8, kIssuer = 12;
    if (warp == kIssuer) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    constexpr uint32_t kTmO = 256, kTmP = 384;   // columns: S buffers 0 and 128, O 256, P buffers 384 and 448
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok && !mbar_spin(bar, parity, P.wait_ns)) { ok = false; *fault = 1; }
        return ok;
    };
    if (busy && warp >= kProducer && warp < kIssuer) {
        // ---------------- producers ----------------
        const int pt = tid - 32 * kProducer;
        uint32_t part = 0;           // K / V parts so far: slot part % kRing
        uint32_t unsaid = 0;         // 16-bit rows: parts whose copies are committed but not yet announced
        uint32_t item = 0, tile = 0; // tile: of the CTA so far
        auto say = [&](uint32_t p) { fence_async_smem(); mbar_arrive(&full[p % L::kRing]); };
        auto free_slot = [&](uint32_t p) {   // the slot of part p: all products with the part before it in it are done
            if (p < (uint32_t)L::kRing) return true;
            return wait(&empty[p % L::kRing], (p / L::kRing - 1) & 1u);
        };
        do {
            const size_t head = (size_t)it.seq * P.cache.seq_stride + (size_t)it.h * P.cache.head_stride;
            const uint8_t* base[2] = {P.cache.k + head * (L::k8 ? 1 : 2), P.cache.v + head * (L::k8 ? 1 : 2)};
            if constexpr (!L::k8) {
                constexpr int kChunks = D / 8, kPer = kTcKT * kChunks / kTcProducers, kStep = kTcProducers / kChunks;
                const int c = pt % kChunks, r0 = pt / kChunks;
                const int n = it.t1 - it.t0;
                #pragma unroll 1
                for (int x = 0; x < 2 * n && ok; x++, part++) {
                    int kv;
                    const int k0 = (it.t0 + part_tile(x, n, kv)) * kTcKT;
                    if (part >= (uint32_t)L::kRing && unsaid && !mbar_try_wait(&empty[part % L::kRing], (part / L::kRing - 1) & 1u)) {
                        cp_async_wait<0>();   // the ring is full: announce all that is coming before the wait for a slot
                        for (; unsaid; unsaid--) say(part - unsaid);
                    }
                    if (!free_slot(part)) break;
                    uint8_t* dst = smem + L::kKV + part % L::kRing * L::kHalf + (c >> 3) * (kTcKT * 128);
                    static_assert(kStep % 8 == 0, "the rows of a thread share their swizzle");
                    const uint32_t to = smem_addr(dst + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4));
                    const uint8_t* src = base[kv] + (size_t)(k0 + r0) * L::kRow + c * 16;
                    if (k0 + kTcKT <= it.end) {
                        #pragma unroll
                        for (int i = 0; i < kPer; i++) cp_async16(to + i * kStep * 128, src + i * kStep * L::kRow);
                    } else {
                        #pragma unroll 1
                        for (int i = 0; i < kPer; i++) {
                            const bool live = k0 + r0 + i * kStep < it.end;
                            cp_async16(to + i * kStep * 128, live ? src + i * kStep * L::kRow : base[kv], live);
                        }
                    }
                    cp_async_commit();
                    unsaid++;
                    if (kv == 1 && k0 + kTcKT > it.len) {
                        // rows of the tree: infinities and NaN would reach nodes that do not see them (0 * NaN): they go to the
                        // softmax threads by another way (odd), and are zero in the product.  Every thread looks at its own copies.
                        if (unsaid > 1) {
                            cp_async_wait<1>();
                            for (; unsaid > 1; unsaid--) say(part + 1 - unsaid);
                        }
                        cp_async_wait<0>();
                        constexpr uint32_t kExp = QT == QWEN_BF16 ? 0x7f807f80u : 0x7c007c00u;
                        bool any = false;
                        #pragma unroll 4
                        for (int i = 0; i < kPer; i++) {
                            const int r = r0 + i * kStep;
                            uint4* p = reinterpret_cast<uint4*>(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                            const uint4 w = *p;
                            // all ones where a 16-bit half is not finite
                            uint4 m = make_uint4(__vcmpeq2(w.x & kExp, kExp), __vcmpeq2(w.y & kExp, kExp), __vcmpeq2(w.z & kExp, kExp),
                                                 __vcmpeq2(w.w & kExp, kExp));
                            if ((m.x | m.y | m.z | m.w) && k0 + r >= it.len) {
                                *p = make_uint4(w.x & ~m.x, w.y & ~m.y, w.z & ~m.z, w.w & ~m.w);
                                any = true;
                            }
                        }
                        if (any) odd[item & 7] = 1;
                        say(part);
                        unsaid = 0;
                    }
                    if (unsaid > 2) {
                        cp_async_wait<2>();
                        say(part + 1 - unsaid);
                        unsaid--;
                    }
                }
            } else {
                // raw part x of this item sits in staging slot x % kRawRing, copied by the thread that converts it
                constexpr int kChunks = D / 16, kPer = kTcKT * kChunks / kTcProducers, kStep = kTcProducers / kChunks;
                const int c = pt % kChunks, r0 = pt / kChunks, n = it.t1 - it.t0, parts = 2 * n;
                auto copy = [&](int x) {
                    if (x < parts) {
                        int kv;
                        const int t = part_tile(x, n, kv), k0 = (it.t0 + t) * kTcKT;
                        const uint32_t dst = smem_addr(smem + L::kRaw + x % L::kRawRing * L::kRawHalf + pt * 16);
                        const uint8_t* src = base[kv] + (size_t)k0 * L::kRow + pt * 16;   // (a head's rows lie one behind the other)
                        if (k0 + kTcKT <= it.end) {
                            #pragma unroll
                            for (int i = 0; i < kPer; i++) cp_async16(dst + i * kTcProducers * 16, src + i * kTcProducers * 16);
                        } else {
                            #pragma unroll 1
                            for (int i = 0; i < kPer; i++) {
                                const bool live = k0 + r0 + i * kStep < it.end;
                                cp_async16(dst + i * kTcProducers * 16, live ? src + i * kTcProducers * 16 : base[kv], live);
                            }
                        }
                        if (!kv) {        // the tile's scales come with K
                            const bool live = k0 + pt < it.end;
                            float* sc = reinterpret_cast<float*>(smem + L::kScales) + (tile + t) % kScaleRing * 2 * kTcKT + pt;
                            cp_async4(smem_addr(sc), P.cache.ks + head / D + (live ? k0 + pt : 0), live);
                            cp_async4(smem_addr(sc + kTcKT), P.cache.vs + head / D + (live ? k0 + pt : 0), live);
                        }
                    }
                    cp_async_commit();
                };
                #pragma unroll
                for (int x = 0; x < L::kRawRing - 1; x++) copy(x);
                for (int x = 0; x < parts && ok; x++, part++) {
                    copy(x + L::kRawRing - 1);
                    cp_async_wait<L::kRawRing - 1>();
                    if (!free_slot(part)) break;
                    int kv;
                    const int t = part_tile(x, n, kv), k0 = (it.t0 + t) * kTcKT;
                    const bool tail = STORE == QWEN_E4M3 && kv && k0 + kTcKT > it.len;
                    const uint8_t* src = smem + L::kRaw + x % L::kRawRing * L::kRawHalf + pt * 16;
                    uint8_t* dst = smem + L::kKV + part % L::kRing * L::kHalf + (c >> 2) * (kTcKT * 128);
                    #pragma unroll 4
                    for (int i = 0; i < kPer; i++) {
                        const int r = r0 + i * kStep;
                        const uint4 w = *reinterpret_cast<const uint4*>(src + i * kTcProducers * 16);
                        uint32_t q[4] = {w.x, w.y, w.z, w.w};
                        if (tail && k0 + r >= it.len) {
                            bool hit = false;
                            #pragma unroll
                            for (int e = 0; e < 16; e++)
                                if (((q[e >> 2] >> (8 * (e & 3))) & 0x7fu) == 0x7fu) { q[e >> 2] &= ~(0xffu << (8 * (e & 3))); hit = true; }
                            if (hit) odd[item & 7] = 1;
                        }
                        uint32_t o[8];
                        #pragma unroll
                        for (int e = 0; e < 4; e++) codes_f16x2<STORE, false>(q[e], o[2 * e], o[2 * e + 1]);
                        const int ch = (2 * c) & 7;
                        *reinterpret_cast<uint4*>(dst + r * 128 + ((ch ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4*>(dst + r * 128 + (((ch + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                    }
                    say(part);
                    if (!kv) {        // the largest exponent of the context's value scales, a warp's 32 keys
                        const uint32_t ring = (tile + t) % kScaleRing;
                        const float vs = reinterpret_cast<const float*>(smem + L::kScales)[ring * 2 * kTcKT + kTcKT + pt];
                        const uint32_t e = __reduce_max_sync(~0u, k0 + pt < it.len ? scale_exponent(vs) : 0u);
                        if (lane == 0) reinterpret_cast<volatile uint32_t*>(smem + L::kVe)[ring * 4 + (warp - kProducer)] = e;
                        __syncwarp();
                        mbar_arrive(&scaled[ring]);
                    }
                }
                cp_async_wait<0>();
                tile += it.t1 - it.t0;
            }
            item++;
        } while (ok && it.next(P));
        cp_async_wait<0>();
        if (ok) for (; unsaid; unsaid--) say(part - unsaid);
    } else if (busy && warp == kIssuer) {
        // ---------------- products (lane 0), the items' tree masks (all) ----------------
        constexpr uint32_t id_s = tc_idesc<BF>(kTcKT, false), id_o = tc_idesc<BF>(D, true);
        uint32_t part = 0, item = 0;
        uint32_t steps[2] = {0, 0};   // tiles of a buffer so far
        bool going = true;
        do {
            int up[2];
            uint64_t nodes[2];
            load_parents(P, it.seq, up);
            tree_masks(P, it.len, up, nodes);
            // every softmax thread has taken what it needs of the item before's masks (it announced that item's queries after)
            anc[lane] = nodes[0];
            anc[lane + 32] = nodes[1];
            named_bar(1, kTcSoftmax + 32);
            if (lane == 0 && going) {
                const int nt = it.t1 - it.t0;
                going = wait(qfull, item & 1u);
                tc_fence_after();
                // S 0, S 1, P V 0, S 2, P V 1, ...: buffer b = tile & 1 of S is free once P of the tile two before is written
                for (int v = 0; v < nt + 2 && going; v++) {
                    const int b = v & 1;
                    if (v >= 2) {
                        const uint32_t p = part + v_part(v - 2, nt);
                        going = wait(&pfull[b], (steps[b] - 1) & 1u) && wait(&full[p % L::kRing], p / L::kRing & 1u);
                        if (!going) break;
                        tc_fence_after();
                        const uint32_t vb = smem_addr(smem + L::kKV + p % L::kRing * L::kHalf);
                        #pragma unroll
                        for (int k = 0; k < kTcKT / 16; k++)
                            tc_mma_ts(tmem + kTmO, tmem + kTmP + 64 * b + 8 * k, mn_major_sw128_desc(vb + k * 2048, kTcKT * 128), id_o,
                                      (v > 2 || k) ? 1u : 0u);
                        mma_commit(&empty[p % L::kRing]);
                        mma_commit(&pvdone[b]);
                    }
                    if (v < nt) {
                        const uint32_t p = part + k_part(v);
                        going = wait(&full[p % L::kRing], p / L::kRing & 1u);
                        if (!going) break;
                        tc_fence_after();
                        const uint32_t kb = smem_addr(smem + L::kKV + p % L::kRing * L::kHalf), qb = smem_addr(smem + L::kQ);
                        #pragma unroll
                        for (int k = 0; k < D / 16; k++)
                            mma_bf16(tmem + 128 * b, kmajor_sw128_desc(qb + (k >> 2) * (kTcRows * 128) + (k & 3) * 32),
                                     kmajor_sw128_desc(kb + (k >> 2) * (kTcKT * 128) + (k & 3) * 32), id_s, k ? 1u : 0u);
                        mma_commit(&empty[p % L::kRing]);
                        mma_commit(&sfull[b]);
                        steps[b]++;
                    }
                }
                part += 2 * nt;
            }
            __syncwarp();
            item++;
        } while (it.next(P));
        if (lane == 0) {
            mma_commit(drained);
            if (!mbar_wait(drained, 0, P.wait_ns)) *fault = 1;
        }
        __syncwarp();
    } else if (busy && warp < kProducer) {
        // ---------------- softmax ----------------
        const int half = warp >> 2, rl = 32 * (warp & 3) + lane;           // half of the keys, row of the item
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, to = tmem + lanes + kTmO;
        float* xm = reinterpret_cast<float*>(smem + L::kXm);               // [tile parity][half][row]
        const int M = P.n_nodes * P.group;
        const bool flip = P.scale_log2 < 0.f;                              // a negative scale: its sign goes to the queries
        uint32_t item = 0, steps = 0, tile = 0;
        uint32_t uses[2] = {0, 0};                                         // tiles of a buffer so far
        do {
            const int nt = it.t1 - it.t0;
            // (the item before's products are done: its queries' place is free)
            const int row = it.r_base + rl;
            const int node = P.node_of(row);
            const bool live = row < M;
            float* qf = reinterpret_cast<float*>(smem + L::kQf);
            {   // the item's queries: D / 8 neighbouring threads a row
                constexpr int kLanes = D / 8, kStep = kTcSoftmax / kLanes, kPer = kTcRows / kStep;
                const int part = tid % kLanes, r0 = tid / kLanes;
                const uint32_t sign = flip ? 0x80008000u : 0u;
                const uint8_t* qbase = P.q + ((size_t)it.seq * P.n_nodes * (size_t)P.ldq + (size_t)it.h * P.group * D + part * 8) * 2;
                uint8_t* dst = smem + L::kQ + (part >> 3) * (kTcRows * 128);
                auto src = [&](int r, bool& in) {
                    const int qrow = it.r_base + r, qnode = P.node_of(qrow);
                    in = qrow < M;
                    return in ? qbase + ((size_t)qnode * (size_t)P.ldq + (size_t)(qrow - qnode * P.group) * D) * 2 : P.q;
                };
                if constexpr (!L::k8) {
                    #pragma unroll 2
                    for (int i = 0; i < kPer; i++) {
                        const int r = r0 + i * kStep;
                        bool in;
                        const uint8_t* from = src(r, in);
                        cp_async16(smem_addr(dst + r * 128 + (((part & 7) ^ (r & 7)) << 4)), from, in);
                    }
                    cp_async_commit();
                    cp_async_wait<0>();
                    if (flip) {
                        for (int i = 0; i < kPer; i++) {
                            const int r = r0 + i * kStep;
                            uint4* p = reinterpret_cast<uint4*>(dst + r * 128 + (((part & 7) ^ (r & 7)) << 4));
                            const uint4 w = *p;
                            *p = make_uint4(w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign);
                        }
                    }
                } else {
                    uint4 w[kPer];
                    #pragma unroll
                    for (int i = 0; i < kPer; i++) {
                        bool in;
                        const uint8_t* from = src(r0 + i * kStep, in);
                        w[i] = in ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0, 0, 0, 0);
                    }
                    #pragma unroll
                    for (int i = 0; i < kPer; i++) {
                        const int r = r0 + i * kStep;
                        uint32_t x[4] = {w[i].x ^ sign, w[i].y ^ sign, w[i].z ^ sign, w[i].w ^ sign};
                        if constexpr (QT == QWEN_BF16) {                   // into fp16's range, a power of two a row
                            const uint32_t y = __vmaxu2(__vmaxu2(x[0] & 0x7fff7fffu, x[1] & 0x7fff7fffu), __vmaxu2(x[2] & 0x7fff7fffu, x[3] & 0x7fff7fffu));
                            uint32_t m = max(y & 0xffffu, y >> 16);
                            #pragma unroll
                            for (int o = 1; o < kLanes; o <<= 1) m = max(m, __shfl_xor_sync(~0u, m, o));
                            const int e = min(max((int)(m >> 7), 1), 253);
                            const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                            #pragma unroll
                            for (int j = 0; j < 4; j++) x[j] = kv::half2_bits(bf_lo(x[j]) * down, bf_hi(x[j]) * down);
                            if (part == 0) qf[r] = __uint_as_float((uint32_t)e << 23);
                        }
                        *reinterpret_cast<uint4*>(dst + r * 128 + (((part & 7) ^ (r & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
            }
            fence_async_smem();
            tc_fence_before();
            named_bar(1, kTcSoftmax + 32);                                 // the masks are there; every thread is behind the item before
            if (tid == 0) odd[(item - 1) & 7] = 0;
            const float c = fmaxf(fabsf(P.scale_log2) * (L::k8 && QT == QWEN_BF16 ? qf[rl] : 1.0f), kLeast);   // (above 0: -inf * 0 would be NaN)
            const uint64_t see = live ? anc[node] : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(qfull);
            float top = -INFINITY, base = -INFINITY, l = 0.f;              // the row's running maximum; what exponents are taken from; this half's sum
            int ve_run = 37;                                               // 8 bits: largest exponent of a seen value scale so far, 2^-90 at least
            for (int i = 0; i < nt; i++, steps++) {
                const int k0 = (it.t0 + i) * kTcKT + 64 * half;
                const int b = i & 1;
                const float *ks = nullptr, *vs = nullptr;
                if constexpr (L::k8) {
                    const uint32_t ring = (tile + i) % kScaleRing;
                    wait(&scaled[ring], (tile + i) / kScaleRing & 1u);
                    ks = reinterpret_cast<const float*>(smem + L::kScales) + ring * 2 * kTcKT + 64 * half;
                    vs = ks + kTcKT;
                    const volatile uint32_t* v4 = reinterpret_cast<const volatile uint32_t*>(smem + L::kVe) + ring * 4;
                    ve_run = max(ve_run, (int)max(max(v4[0], v4[1]), max(v4[2], v4[3])));
                    const int t0 = k0 - 64 * half, first = it.len - t0;    // the tile's first key; its key that is node 0 (or beyond its ends)
                    if (first < kTcKT) {   // and of the tree's keys in the tile those that this row sees: the others' scales may be any
                        uint64_t own = see;
                        if (first < 0) own &= ~0ull << -first;
                        else if (first > kTcKT - 64) own &= (1ull << (kTcKT - first)) - 1;
                        const float* tree = vs - 64 * half + first;
                        for (; own; own &= own - 1) ve_run = max(ve_run, (int)scale_exponent(tree[__ffsll((long long)own) - 1]));
                        __syncwarp();
                    }
                }
                const uint32_t use = uses[b];
                wait(&sfull[b], use & 1u);
                tc_fence_after();
                const bool tail = k0 + 64 > it.len;
                // bit x: the row sees column x of this half
                const uint64_t vis = tail ? visible(see, it.len - k0) : ~0ull;
                // scores of columns c0 .. c0 + 31 of this half (of the first 32 read twice: for the maximum, and for the exponentials)
                auto scores = [&](int c0, float (&v)[32]) {
                    tmem_ld32(tmem + lanes + 128 * b + 64 * half + c0, v);
                    if constexpr (L::k8) {
                        #pragma unroll
                        for (int x = 0; x < 32; x += 4) {
                            const float4 a = *reinterpret_cast<const float4*>(ks + c0 + x);
                            mul2(v[x], v[x + 1], a.x, a.y);
                            mul2(v[x + 2], v[x + 3], a.z, a.w);
                        }
                    }
                    if (tail) {
                        const uint32_t m = (uint32_t)(vis >> c0);
                        #pragma unroll
                        for (int x = 0; x < 32; x++) if (!(m >> x & 1)) v[x] = -INFINITY;
                    }
                };
                float mx = -INFINITY, v[32];                               // v stays: columns 32 .. 63
                #pragma unroll 1
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    float my = -INFINITY;
                    scores(c0, v);
                    #pragma unroll
                    for (int x = 0; x < 32; x += 4) { mx = max3(mx, v[x], v[x + 1]); my = max3(my, v[x + 2], v[x + 3]); }
                    mx = fmaxf(mx, my);
                }
                xm[((steps & 1) * 2 + half) * 128 + rl] = mx;
                named_bar(2, kTcSoftmax);
                mx = fmaxf(mx, xm[((steps & 1) * 2 + (half ^ 1)) * 128 + rl]);
                // an all-masked tile stays -inf
                top = fmaxf(top, mx == -INFINITY ? mx : mx * c);
                const float want = L::k8 ? top + (float)(ve_run - 127) : top;
                float f = 1.0f;
                const bool move = want > base + 8.0f;                      // (from -inf: the first tile that has a key)
                if (move) {
                    f = exp2_approx(base - want);
                    l *= f;
                    base = want;
                }
                if (i > 0 && __any_sync(~0u, move)) {
                    wait(&pvdone[b ^ 1], (uses[b ^ 1] - 1) & 1u);          // O of the tile before
                    tc_fence_after();
                    #pragma unroll 1
                    for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
                        float o[32];
                        tmem_ld32(to + c0, o);
                        #pragma unroll
                        for (int x = 0; x < 32; x += 2) mul2(o[x], o[x + 1], f, f);
                        tc_st32(to + c0, o);
                    }
                }
                const float from = base == -INFINITY ? 0.f : base;
                if (i > 1) wait(&pvdone[b], (use - 1) & 1u);               // the P buffer's last product
                tc_fence_after();
                float sum0 = 0.f, sum1 = 0.f;
                #pragma unroll 1
                for (int c0 = 32; c0 >= 0; c0 -= 32) {
                    if (c0 == 0) scores(0, v);
                    uint32_t w[16];
                    const uint32_t m = (uint32_t)(vis >> c0);
                    #pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        float4 y;
                        if constexpr (L::k8) y = *reinterpret_cast<const float4*>(vs + c0 + x);
                        fma2(v[x], v[x + 1], c, -from);
                        fma2(v[x + 2], v[x + 3], c, -from);
                        float a[4];
                        #pragma unroll
                        for (int j = 0; j < 4; j++) a[j] = exp2_approx(v[x + j]);
                        add2(sum0, sum1, a[0], a[1]);
                        add2(sum0, sum1, a[2], a[3]);
                        if constexpr (L::k8) {
                            mul2(a[0], a[1], y.x, y.y);
                            mul2(a[2], a[3], y.z, y.w);
                        }
                        w[x / 2] = pack2<BF>(a[0], a[1]);
                        w[x / 2 + 1] = pack2<BF>(a[2], a[3]);
                    }
                    if (L::k8 && tail) {   // (a scale that the row does not see may be NaN)
                        #pragma unroll
                        for (int x = 0; x < 32; x += 2)
                            w[x / 2] &= (m >> x & 1 ? 0xffffu : 0u) | (m >> (x + 1) & 1 ? 0xffff0000u : 0u);
                    }
                    tc_st16(tmem + lanes + kTmP + 64 * b + 32 * half + c0 / 2, w);
                }
                l += sum0 + sum1;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[b]);
                uses[b]++;
            }
            tile += nt;
            {   // the next item's queries on their way while the last products run
                auto nx = it;
                if (nx.next(P)) {
                    const int nrow = nx.r_base + rl, nnode = P.node_of(nrow);
                    if (nrow < M)
                        asm volatile("prefetch.global.L1 [%0];" ::"l"(P.q + (((size_t)nx.seq * P.n_nodes + nnode) * (size_t)P.ldq +
                                                                             (size_t)(nx.h * P.group + nrow - nnode * P.group) * D + half * (D / 2)) * 2));
                }
            }
            // ---- the item's rows: this thread's half of the dims ----
            {
                const int b = (nt - 1) & 1;
                wait(&pvdone[b], (uses[b] - 1) & 1u);
            }
            tc_fence_after();
            xm[((steps & 1) * 2 + half) * 128 + rl] = l;
            named_bar(2, kTcSoftmax);
            l += xm[((steps & 1) * 2 + (half ^ 1)) * 128 + rl];
            steps++;                                                       // (the next tile's maxima go to the other half of xm)
            const bool odd_rows = odd[item & 7] != 0;                      // (every part of the item has been announced)
            const bool whole = it.t0 == 0 && it.t1 == it.n, present = see != 0, failed = *fault != 0;
            const float inv = !present || l == 0.f ? 0.f : 1.0f / l;
            float* slot = P.work + (size_t)(2 * blockIdx.x + (it.first ? 0 : 1)) * L::kSlot;
            #pragma unroll 1
            for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
                float o[32];
                tmem_ld32(to + c0, o);
                if (odd_rows) {                   // infinities and NaN of the tree's V rows, for the rows that see them
                    const size_t head = (size_t)it.seq * P.cache.seq_stride + (size_t)it.h * P.cache.head_stride;
                    for (int j = 0; j < P.n_nodes; j++) {
                        const long long pos = (long long)it.len + j;
                        if (!((see >> j) & 1) || pos < (long long)it.t0 * kTcKT || pos >= (long long)it.t1 * kTcKT) continue;
                        #pragma unroll
                        for (int x = 0; x < 32; x++) {
                            const size_t at = head + (size_t)pos * D + c0 + x;
                            if constexpr (STORE == QWEN_E4M3) { if ((P.cache.v[at] & 0x7f) == 0x7f) o[x] += NAN; }
                            else if constexpr (!L::k8) {
                                const uint16_t w = reinterpret_cast<const uint16_t*>(P.cache.v)[at];
                                constexpr uint32_t kExp = QT == QWEN_BF16 ? 0x7f80u : 0x7c00u;
                                if ((w & kExp) == kExp) o[x] += QT == QWEN_BF16 ? bf2f(w) : __half2float(__ushort_as_half(w));
                            }
                        }
                    }
                }
                #pragma unroll
                for (int x = 0; x < 32; x++) o[x] = failed ? NAN : present ? o[x] : 0.f;
                if (whole) {
                    // 16-bit rows into the queries' place, swizzled, and from there whole rows to memory
                    uint32_t w[16];
                    #pragma unroll
                    for (int x = 0; x < 16; x++) w[x] = pack2<QT == QWEN_BF16>(o[2 * x] * inv, o[2 * x + 1] * inv);
                    #pragma unroll
                    for (int x = 0; x < 4; x++)
                        *reinterpret_cast<uint4*>(smem + L::kQ + swz<D * 2>(rl, c0 / 8 + x)) = make_uint4(w[4 * x], w[4 * x + 1], w[4 * x + 2], w[4 * x + 3]);
                } else if (live) {
                    #pragma unroll
                    for (int x = 0; x < 32; x += 4)
                        *reinterpret_cast<float4*>(slot + (((c0 + x) / 4) * kTcRows + rl) * 4) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                    if (c0 == 0) *reinterpret_cast<float2*>(slot + kTcRows * D + 2 * rl) = present ? make_float2(base, l) : make_float2(-INFINITY, 0.f);
                }
            }
            if (whole) {                          // the same for all
                named_bar(2, kTcSoftmax);
                constexpr int kChunks = D / 8, kStep = kTcSoftmax / kChunks, kPer = kTcRows / kStep;
                const int ch = tid % kChunks, r0 = tid / kChunks;
                uint4 w[kPer];
                #pragma unroll
                for (int i = 0; i < kPer; i++) w[i] = *reinterpret_cast<const uint4*>(smem + L::kQ + swz<D * 2>(r0 + i * kStep, ch));
                uint8_t* out = P.out + ((size_t)it.seq * P.n_nodes * (size_t)P.ldo + (size_t)it.h * P.group * D + ch * 8) * 2;
                #pragma unroll
                for (int i = 0; i < kPer; i++) {
                    const int orow = it.r_base + r0 + i * kStep, onode = P.node_of(orow);
                    if (orow < M) *reinterpret_cast<uint4*>(out + ((size_t)onode * (size_t)P.ldo + (size_t)(orow - onode * P.group) * D) * 2) = w[i];
                }
                named_bar(2, kTcSoftmax);         // the queries' place is free again
            }
            tc_fence_before();
            item++;
        } while (it.next(P));
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

}  // namespace ta
}  // namespace qb
