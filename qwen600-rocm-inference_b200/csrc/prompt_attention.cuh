// prompt_attention.cuh — causal attention of packed prompts on the sm_100a tensor
// cores (qwen_prompt_attention).  No reference counterpart: the reference runs
// its decode attention once per prompt token (main.cu:141-145 over
// qwen_model.cuh:551-614).
//
// Mathematics.  Query i of a sequence with n queries and m keys sees keys 0 .. m - n +
// i.  One pass over tiles of 128 keys with the running maximum and sum of the softmax
// (base 2, scale * log2 e folded into the exponent): S = Q K^T, P = 2^(S c - base), O += P
// V.  A row's base follows its maximum only when that has risen by 2^8, so O is seldom scaled; O
// / l at the end.
//
// A row of a tile is a (token, query head) pair of one K/V head, head fastest: T = 128 /
// group tokens of all the K/V head's query heads, so K and V serve the whole group.
// An item is two such row tiles, A and B, one behind the other, and their common key
// tiles.  Tensor memory: one S (128 columns), which A and B use in turn, P of A and of B
// (16 bits, 64 columns each), O of A and of B.  S is in registers soon after it is formed, so the
// next tile's is formed while the softmax is at work, and no chain runs from a tile's P over its product
// to the next S.
//
// Measured (bf16, 16 query heads over 8 K/V heads of 128): one prompt of 8192 220 to 232 us, 1,185 to 1,250
// TFLOP/s, where a large matrix product has 1,637 for a moment and 1,370 for long (floor 168 us; without a pause for seconds 257 to
// 263 us); 2048 37 us; four of 4096 245 us.  Heads of 64: one of 8192 205 to 248 us, bound by the softmax in the same way.
// Many short prompts: 100 of 50 33 us, 500 272, 2000 4,350 (floor 188): an item is found by a search over all sequences, which the
// other warps wait for.  Few queries over a long context: 5 over 40,000 425 us (floor 25), as keys are not divided.
// Bound by the softmax warps: a tile of 256 x 128 takes 3,350 cycles, of which the tensor cores need 2,050 at
// their rate and 2,500 as they run (both operands of S come from shared memory), the exponentials 2,050; the warps
// issue in 54 % of the slots, each waiting for its own chain: scores (300 cycles), maximum and its exchange
// (800), exponentials (1,400), waits that find their barriers ready (100 to 200 each).  Steps on the way: one thread a row, P
// over S, products issued by a lane alone 374 us; descriptors in uniform registers and registers shared out anew 273; one S for both tiles
// with two threads a row 255; a warp each for the two products 232; all exponentials by the special-function unit 224 (a polynomial for a
// part of them cost more instructions than it spared).  Tried, not kept: turns of A and B at the exponentials (235 us).
//
// Warps: 0-7 softmax and output of A (two threads a row, 64 keys of a tile and half of the dims each; they agree on
// the row's maximum through shared memory), 8-15 of B, 16 finds the items and loads (TMA), 17 issues
// S, 18 issues P V, 19 looks for infinities and NaN among the V
// rows of tiles that are not seen as a whole: 0 * NaN would reach rows that do not see them,
// so such values are zeroed in shared memory and added at the end to the rows that see them.
// Items, heaviest first, are dealt out to the CTAs forwards and backwards in turn; they are found on the device from
// starts and k_starts.  Every wait on a barrier is bounded; where one runs out, the rows of all of the CTA's items become NaN
// at its end.
#pragma once
#include "tree_attention_tc.cuh"

namespace qb {
namespace pr {

using ta::exp2_approx;
using ta::kLeast;
using ta::max3;
using ta::mul2;
using ta::pack2;

constexpr int kKT = 128;                  // keys of a tile
constexpr int kSoftmax = 16;              // warps: two threads a row, 64 keys of a tile each
constexpr int kThreads = 640, kLoader = 16, kScores = 17, kValues = 18, kLooker = 19;
constexpr int kItems = 4;                 // items between the loader and the slowest warp

struct Params {
    uint8_t* out;
    const uint8_t* v;
    const int *starts, *k_starts;
    long long ldv, ldo;
    int n_seqs, n_rows, n_keys, n_kv_heads, group, tokens;   // tokens: of a row tile
    int out32;                            // rows of out start on 32 bytes
    long long items;                      // no more than these are dealt out: as many as starts in order can have
    int withheld;
    unsigned long long wait_ns;
    float scale_log2;
};

struct Item {
    int stop;
    int h;             // K/V head
    int q0, nq;        // its first query row, its queries (2 * tokens at most)
    int k0;            // the sequence's first key row
    int off;           // the first query sees keys 0 .. off (none where off < 0)
    int odd;           // V rows of its tail hold infinities or NaN
    int n[2];          // key tiles of A and B
    int pad[3];
};

template <int D>
struct Layout {
    static constexpr int kPart = kKT * D * 2;                 // K or V of a tile, or the rows of a row tile
    // K / V parts in flight.  K and V have a ring each: K's slots are the even ones, V's the odd ones.  So every warp that waits for a part of
    // a ring waits for all of them in turn, and a slot is filled anew only when they have: a wait by parity can neither take an
    // older phase for its own nor be overtaken by two.
    static constexpr int kRing = D == 64 ? 8 : 4, kSlots = kRing / 2;
    static constexpr int kQ = 0;
    static constexpr int kKV = 2 * kPart;
    static constexpr int kBar = kKV + kRing * kPart;
    static constexpr int kBars = 2 * kRing + kSlots + 2 * kItems + 15;
    static constexpr int kItem = kBar + (kBars * 8 + 15) / 16 * 16;
    static constexpr int kXm = kItem + kItems * (int)sizeof(Item);       // [row tile][parity][half][row] maxima, then sums
    static constexpr int kMisc = kXm + 2 * 2 * 2 * 128 * 4;
    static constexpr int kSmem = kMisc + 16 + 1024;
    static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
    static_assert(2 * kSmem > 228 * 1024, "one CTA an SM: the kernel allocates all of tensor memory");
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}
// 32 consecutive fp32 columns of this warp's 32 tensor-memory lanes (one row per lane); the values are there after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "{\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
    #pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// 8 columns of this warp's lanes times f; complete after tc_wait_st.
__device__ __forceinline__ void scale8(uint32_t taddr, float f) {
    float o[8];
    asm volatile(
        "{\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t}"
        : "=f"(o[0]), "=f"(o[1]), "=f"(o[2]), "=f"(o[3]), "=f"(o[4]), "=f"(o[5]), "=f"(o[6]), "=f"(o[7]) : "r"(taddr) : "memory");
    #pragma unroll
    for (int x = 0; x < 8; x += 2) mul2(o[x], o[x + 1], f, f);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "f"(o[0]), "f"(o[1]), "f"(o[2]), "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]), "f"(o[7]) : "memory");
}
// Two fp32 values in a 64-bit register: one instruction for both, and no moves between separate registers.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void halves(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// The sequences, by all lanes of a warp: where each one's rows and keys lie, and its items.
// Sequence s has tiles of 2 * tokens queries; tile t's level is t + 1 + the whole tiles that its context
// would make: tiles of a level have about as many keys.  Items go by falling level,
// within a level by sequence, then by head.
struct Finder {
    static constexpr int kHeld = 4;       // sequences a lane holds (lane, lane + 32, ..)
    int per;                              // queries of an item
    int first[kHeld], count[kHeld];       // levels first + 1 .. first + count
    int top;                              // the highest level
    __device__ __forceinline__ void bounds(const Params& P, int s, int& q0, int& nq, int& k0, int& nk) const {
        q0 = min(max(__ldg(P.starts + s), 0), P.n_rows);
        nq = max(min(max(__ldg(P.starts + s + 1), 0), P.n_rows) - q0, 0);
        if (P.k_starts) {
            k0 = min(max(__ldg(P.k_starts + s), 0), P.n_keys);
            nk = max(min(max(__ldg(P.k_starts + s + 1), 0), P.n_keys) - k0, 0);
        } else {
            k0 = min(q0, P.n_keys);
            nk = min(nq, P.n_keys - k0);
        }
    }
    __device__ __forceinline__ void levels(const Params& P, int s, int& f, int& c) const {
        f = c = 0;
        if (s >= P.n_seqs) return;
        int q0, nq, k0, nk;
        bounds(P, s, q0, nq, k0, nk);
        f = max(nk - nq, 0) / per;
        c = (nq + per - 1) / per;
    }
    // the tiles above level L.  A lane's count ends at 2^26 - 1: what memory holds has fewer tiles, starts that overlap may name more than
    // 32 bits count, and a rank below 0 would be looked for in front of the starts.
    __device__ __forceinline__ int above(const Params& P, int L) const {
        constexpr int kMost = (1 << 26) - 1;
        int n = 0;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) n = min(n + min(max(first[i] + count[i] - L, 0), count[i]), kMost);
        for (int s = 32 * kHeld + (threadIdx.x & 31); s < P.n_seqs; s += 32) {
            int f, c;
            levels(P, s, f, c);
            n = min(n + min(max(f + c - L, 0), c), kMost);
        }
        return __reduce_add_sync(~0u, n);
    }
    __device__ __forceinline__ Finder(const Params& P) : per(2 * P.tokens) {
        const int lane = threadIdx.x & 31;
        int t = 0;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            levels(P, lane + 32 * i, first[i], count[i]);
            t = max(t, count[i] ? first[i] + count[i] : 0);
        }
        for (int s = 32 * kHeld + lane; s < P.n_seqs; s += 32) {
            int f, c;
            levels(P, s, f, c);
            t = max(t, c ? f + c : 0);
        }
        top = __reduce_max_sync(~0u, t);
    }
    // tile number r of the order: its sequence and its place in it; false: there are not so many
    __device__ __forceinline__ bool find(const Params& P, int r, int& seq, int& tile) const {
        const int lane = threadIdx.x & 31;
        int lo = 0, hi = top;             // above(hi) <= r < above(lo)
        if (r >= above(P, 0)) return false;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (above(P, mid) <= r) hi = mid;
            else lo = mid;
        }
        int left = r - above(P, hi);      // among the tiles of level hi
        auto look = [&](int s0, int f, int c) {
            const uint32_t in = __ballot_sync(~0u, f < hi && hi <= f + c);
            const int n = __popc(in);
            if (left >= n) { left -= n; return false; }
            seq = s0 + (int)__fns(in, 0, left + 1);
            tile = hi - 1 - __shfl_sync(~0u, f, seq - s0);
            return true;
        };
        #pragma unroll
        for (int i = 0; i < kHeld; i++) if (look(32 * i, first[i], count[i])) return true;
        for (int s0 = 32 * kHeld; s0 < P.n_seqs; s0 += 32) {
            int f, c;
            levels(P, s0 + lane, f, c);
            if (look(s0, f, c)) return true;
        }
        return false;
    }
};

// grid: CTAs (one an SM at most), kThreads threads, Layout::kSmem bytes.
// map_q: q as [row][head][D], boxes of 64 dims x group heads x tokens; map_k, map_v: [key row][n_kv_heads * D], boxes of 64 x 128.
template <int T, int D>
__global__ void __launch_bounds__(kThreads, 1)
prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
              const __grid_constant__ Params P) {
    using namespace qb::tc;
    using L = Layout<D>;
    constexpr bool BF = T == QWEN_BF16;
    // fp16 weights are at most 2^15: the largest one has at least 2^7, so what is lost under fp16's smallest steps is 2^-32 of it and less
    // (with 2^0, 8,000 keys of 2^-25 each were nothing).  bf16 has fp32's range.
    constexpr float kLift = BF ? 0.0f : 7.0f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBar);   // [kRing] a K or V part has arrived
    uint64_t* empty = full + L::kRing;                              // [kRing] its products are done
    uint64_t* clean = empty + L::kRing;                             // [kSlots] a V part has been looked at
    uint64_t* given = clean + L::kSlots;                            // [kItems] an item is there
    uint64_t* taken = given + kItems;                               // [kItems] all warps are done with it
    // [2]: A, B
    uint64_t* qfull = taken + kItems;                               // the item's rows have arrived
    uint64_t* qempty = qfull + 2;                                   // their last S is formed
    uint64_t* sfull = qfull + 4;                                    // S formed
    uint64_t* odone = qfull + 6;                                    // P V added
    uint64_t* pfull = qfull + 8;                                    // [2][2] a half of P written (4 warps); for the first one O scaled too (all 8)
    uint64_t* sread = qfull + 12;                                   // S is in registers (8 warps)
    uint64_t* drained = qfull + 13;                                 // [2] all products of a warp are done, at the end
    Item* items = reinterpret_cast<Item*>(smem + L::kItem);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
    volatile int* fault = reinterpret_cast<int*>(smem + L::kMisc + 4);
    volatile uint32_t* beat = reinterpret_cast<uint32_t*>(smem + L::kMisc + 8);   // K and V parts asked for so far
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < L::kRing; i++) { mbar_init(&full[i], 1 + (i == P.withheld)); mbar_init(&empty[i], 1); }
        for (int i = 0; i < L::kSlots; i++) mbar_init(&clean[i], 1);
        for (int i = 0; i < kItems; i++) { mbar_init(&given[i], 1); mbar_init(&taken[i], kSoftmax + 3); }   // softmax, products, looker
        for (int w = 0; w < 2; w++) {
            mbar_init(&qfull[w], 1);
            mbar_init(&qempty[w], 1);
            mbar_init(&sfull[w], 1);
            mbar_init(&pfull[2 * w], 8);
            mbar_init(&pfull[2 * w + 1], 4);
            mbar_init(&odone[w], 1);
        }
        mbar_init(sread, 8);
        for (int i = 0; i < 2; i++) mbar_init(&drained[i], 1);
        fence_barrier_init();
        *fault = 0;
        *beat = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    if (warp == kScores) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Bounded; once a wait has run out anywhere in the CTA, none of the others is waited for (but an item's is).
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return;
        uint64_t since = 0;
        while (!*fault) {
            #pragma unroll 1
            for (int n = 0; n < 64; n++) if (mbar_try_wait(bar, parity)) return;
            const uint64_t now = global_ns();
            if (!since) since = now;
            else if (now - since > P.wait_ns) *fault = 1;
        }
    };
    // The same for warps that nobody waits for at once: asleep in between, so as to take no issue slots from the others.
    auto wait_asleep = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return;
        uint64_t since = 0;
        while (!*fault && !mbar_try_wait_sleep(bar, parity, 2000u)) {
            const uint64_t now = global_ns();
            if (!since) since = now;
            else if (now - since > P.wait_ns) *fault = 1;
        }
    };
    auto failed = [&]() { return __any_sync(~0u, *fault); };   // the same for a warp, whose lanes go on together
    auto finish = [&]() {                     // a warp's last step: all of the CTA's work is done behind it
        tc_fence_before();
        __syncthreads();
    };
    uint32_t seen = 0;                        // items so far
    Item it;
    // All lanes of a warp; false: no more.  A warp whose row tile has no keys may wait here for as long as the block's item takes: the
    // wait has run out where no part was asked for all the while.
    auto next_item = [&]() {
        const int slot = seen % kItems;
        for (uint32_t before = 0;;) {
            if (__all_sync(~0u, ta::mbar_spin(&given[slot], seen / kItems & 1u, 8 * P.wait_ns))) return !items[slot].stop;
            const uint32_t now = __shfl_sync(~0u, *beat, 0);
            if (now == before) break;
            before = now;
        }
        *fault = 1;
        return false;
    };
    auto item_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&taken[seen % kItems]);
        seen++;
    };

    // The block's 640 x 96 registers, shared out anew: 104 for a softmax thread, 64 for the others (512 x 104 + 128 x 64 = 640 x 96).
    auto fewer = [] { asm volatile("setmaxnreg.dec.sync.aligned.u32 64;"); };
    if (warp == kLoader) {
        // ---------------- items and loads ----------------
        fewer();
        const Finder finder(P);
        const int G = gridDim.x;
        auto deal = [&](int k) {               // item k of this CTA into `it`; false: there are not so many
            const long long at = (long long)k * G + (k & 1 ? G - 1 - (int)blockIdx.x : (int)blockIdx.x);   // forwards and backwards
            int seq = 0, tile = 0, q0, nq, k0, nk;
            it = {};
            if (at >= P.items || !finder.find(P, (int)(at / P.n_kv_heads), seq, tile)) return false;
            finder.bounds(P, seq, q0, nq, k0, nk);
            it.h = (int)(at % P.n_kv_heads);
            it.q0 = q0 + tile * finder.per;
            it.nq = min(nq - tile * finder.per, finder.per);
            it.k0 = k0;
            it.off = nk - nq + tile * finder.per;
            for (int w = 0; w < 2; w++) {
                const int count = min(it.nq - w * P.tokens, P.tokens), last = it.off + w * P.tokens + count - 1;
                it.n[w] = count <= 0 || last < 0 ? 0 : last / kKT + 1;
            }
            return true;
        };
        uint32_t parts[2] = {0, 0}, used[2] = {0, 0};   // K and V parts so far; items so far that have the row tile
        bool more = true;
        for (int k = 0; more; k++) {
            more = deal(k);
            it.stop = !more;
            const int slot = k % kItems;
            if (k >= kItems && !__all_sync(~0u, ta::mbar_spin(&taken[slot], (k / kItems - 1) & 1u, 8 * P.wait_ns))) { *fault = 1; break; }
            if (lane == 0) {
                items[slot] = it;
                mbar_arrive(&given[slot]);
                const int n = max(it.n[0], it.n[1]);
                auto rows = [&](int w) {
                    if (!it.n[w]) return;
                    if (used[w]) wait_asleep(&qempty[w], (used[w] - 1) & 1u);
                    if (*fault) return;
                    used[w]++;
                    mbar_arrive_expect_tx(&qfull[w], P.tokens * P.group * D * 2);
                    #pragma unroll
                    for (int x = 0; x < D / 64; x++)
                        tma_load_3d(smem + L::kQ + w * L::kPart + x * (128 * 128), &map_q, 64 * x, it.h * P.group, it.q0 + w * P.tokens, &qfull[w]);
                };
                auto keys = [&](int value, int i) {      // tile i of K or V
                    const CUtensorMap* map = value ? &map_v : &map_k;
                    const uint32_t part = parts[value], s = 2 * (part % L::kSlots) + value;
                    if (part >= (uint32_t)L::kSlots) wait_asleep(&empty[s], (part / L::kSlots - 1) & 1u);
                    if (*fault) return;
                    mbar_arrive_expect_tx(&full[s], L::kPart);
                    #pragma unroll
                    for (int x = 0; x < D / 64; x++)
                        tma_load_2d(smem + L::kKV + s * L::kPart + x * (kKT * 128), map, it.h * D + 64 * x, it.k0 + i * kKT, &full[s]);
                    *beat = ++parts[value] + parts[value ^ 1];
                };
                rows(0);
                for (int i = 0; i < n && !*fault; i++) {   // in the order in which the products take them
                    keys(0, i);
                    if (i == 0) rows(1);
                    else keys(1, i - 1);
                }
                if (n) keys(1, n - 1);
            }
            __syncwarp();
        }
        finish();
        if (*fault) {                          // (nobody sets it any more)
            if (lane == 0) {                   // nothing may still be on its way when the CTA ends
                for (int v = 0; v < 2; v++)
                    for (uint32_t p = parts[v] > (uint32_t)L::kSlots ? parts[v] - L::kSlots : 0; p < parts[v]; p++)
                        mbar_wait(&full[2 * (p % L::kSlots) + v], p / L::kSlots & 1u, 10000000ull);
                for (int w = 0; w < 2; w++) if (used[w]) mbar_wait(&qfull[w], (used[w] - 1) & 1u, 10000000ull);
            }
            __syncwarp();
            const int pieces = P.group * D / 8;   // no row that this CTA had may pass for a result
            for (int k = 0; deal(k); k++)
                for (int r = 0; r < it.nq; r++) {
                    uint4* row = reinterpret_cast<uint4*>(P.out + ((size_t)(it.q0 + r) * P.ldo + (size_t)it.h * P.group * D) * 2);
                    for (int x = lane; x < pieces; x += 32) row[x] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
                }
        }
    } else if (warp == kScores || warp == kValues) {
        // ---------------- products ----------------
        // A warp for S and one for P V, so that the waits of one pass under the products of the other.  The whole warp walks, one lane
        // issues: what a product takes is then the same for the warp and stays in uniform registers (with a lane alone, a product cost 110
        // cycles of address arithmetic, twice what it computes).
        fewer();
        constexpr uint32_t id_s = ta::tc_idesc<BF>(kKT, false), id_o = ta::tc_idesc<BF>(D, true);
        const bool leader = elect_one();
        const uint64_t qd = kmajor_sw128_desc(smem_addr(smem + L::kQ)), kd = kmajor_sw128_desc(smem_addr(smem + L::kKV)),
                       vd = ta::mn_major_sw128_desc(smem_addr(smem + L::kKV), kKT * 128);
        uint32_t parts = 0;                    // K (or V) parts of the items so far
        uint32_t used[2] = {0, 0}, steps[2] = {0, 0}, formed = 0;   // items, key tiles of a row tile so far; S so far
        while (next_item()) {
            const int n[2] = {__shfl_sync(~0u, items[seen % kItems].n[0], 0), __shfl_sync(~0u, items[seen % kItems].n[1], 0)}, most = max(n[0], n[1]);
            if (warp == kScores) {
                for (int i = 0; i < most && !failed(); i++) {
                    const uint32_t part = parts + i, slot = 2 * (part % L::kSlots);
                    const uint64_t b = kd + (uint64_t)(slot * (uint32_t)(L::kPart >> 4));
                    wait(&full[slot], part / L::kSlots & 1u);
                    #pragma unroll
                    for (int w = 0; w < 2; w++) {
                        if (i >= n[w]) continue;
                        if (i == 0) wait(&qfull[w], used[w]++ & 1u);
                        if (formed) wait(sread, (formed - 1) & 1u);
                        formed++;
                        tc_fence_after();
                        const uint64_t a = qd + (uint64_t)(w * (L::kPart >> 4));
                        if (leader) {
                            #pragma unroll
                            for (int k = 0; k < D / 16; k++)
                                mma_bf16(tmem, a + (((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4), b + (((k >> 2) * (kKT * 128) + (k & 3) * 32) >> 4), id_s, k ? 1u : 0u);
                            mma_commit(&sfull[w]);
                            if (i + 1 == n[w]) mma_commit(&qempty[w]);
                        }
                        __syncwarp();
                    }
                    if (leader) mma_commit(&empty[slot]);
                    __syncwarp();
                }
            } else {
                for (int i = 0; i < most && !failed(); i++) {
                    const uint32_t part = parts + i, place = part % L::kSlots, slot = 2 * place + 1;
                    const uint64_t b = vd + (uint64_t)(slot * (uint32_t)(L::kPart >> 4));
                    wait(&clean[place], part / L::kSlots & 1u);
                    #pragma unroll
                    for (int w = 0; w < 2; w++) {
                        if (i >= n[w]) continue;
                        #pragma unroll
                        for (int half = 0; half < 2; half++) {
                            wait(&pfull[2 * w + half], steps[w] & 1u);
                            tc_fence_after();
                            if (leader) {
                                #pragma unroll
                                for (int k = 4 * half; k < 4 * half + 4; k++)
                                    ta::tc_mma_ts(tmem + 256 + 128 * w, tmem + 128 + 64 * w + 8 * k, b + (k * 2048 >> 4), id_o, (i | k) ? 1u : 0u);
                                if (half) mma_commit(&odone[w]);
                            }
                            __syncwarp();
                        }
                        steps[w]++;
                    }
                    if (leader) mma_commit(&empty[slot]);
                    __syncwarp();
                }
            }
            parts += most;
            item_done();
        }
        if (leader) {
            mma_commit(&drained[warp - kScores]);
            if (!mbar_wait(&drained[warp - kScores], 0, P.wait_ns)) *fault = 1;
        }
        __syncwarp();
        finish();
        if (warp == kScores) tmem_dealloc(tmem, 512);
    } else if (warp == kLooker) {
        // ---------------- infinities and NaN among V rows that not all rows see ----------------
        fewer();
        uint32_t part = 0;                     // V parts so far
        while (next_item()) {
            it = items[seen % kItems];
            const int n = max(it.n[0], it.n[1]);
            for (int i = 0; i < n && !failed(); i++, part++) {
                const uint32_t place = part % L::kSlots, slot = 2 * place + 1;
                wait_asleep(&full[slot], part / L::kSlots & 1u);
                if (i * kKT + kKT - 1 > it.off) {
                    constexpr uint32_t kExp = BF ? 0x7f807f80u : 0x7c007c00u;
                    uint4* rows = reinterpret_cast<uint4*>(smem + L::kKV + slot * L::kPart);
                    bool any = false;
                    #pragma unroll 8
                    for (int x = lane; x < L::kPart / 16; x += 32) {
                        const uint4 w = rows[x];
                        // all ones where a 16-bit half is not finite
                        const uint4 m = make_uint4(__vcmpeq2(w.x & kExp, kExp), __vcmpeq2(w.y & kExp, kExp), __vcmpeq2(w.z & kExp, kExp),
                                                   __vcmpeq2(w.w & kExp, kExp));
                        if (m.x | m.y | m.z | m.w) {
                            rows[x] = make_uint4(w.x & ~m.x, w.y & ~m.y, w.z & ~m.z, w.w & ~m.w);
                            any = true;
                        }
                    }
                    if (any) {
                        *(volatile int*)&items[seen % kItems].odd = 1;
                        ta::fence_async_smem();
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&clean[place]);
            }
            item_done();
        }
        finish();
    } else {
        // ---------------- softmax and output ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int w = warp >> 3, half = warp >> 2 & 1, rl = 32 * (warp & 3) + lane;   // row tile, half of the keys, row
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = tmem + lanes + 64 * half, tp = tmem + lanes + 128 + 64 * w + 32 * half, to = tmem + lanes + 256 + 128 * w + half * (D / 2);
        const int token = w * P.tokens + rl / P.group, head = rl % P.group;
        const bool placed = rl < P.tokens * P.group;
        const float c = fmaxf(fabsf(P.scale_log2), kLeast);                // (above 0: -inf * 0 would be NaN)
        const bool flip = P.scale_log2 < 0.f;
        float* mine = reinterpret_cast<float*>(smem + L::kXm) + w * 512 + half * 128 + rl;   // + 256 for odd steps
        const float* other = reinterpret_cast<const float*>(smem + L::kXm) + w * 512 + (half ^ 1) * 128 + rl;
        uint32_t steps = 0, swaps = 0;                                     // key tiles, exchanges so far
        while (next_item()) {
            const Item* item = &items[seen % kItems];                      // (read where it is needed: registers are scarce)
            const int n = item->n[w], sees = placed && token < item->nq ? item->off + token : 1 << 30;   // the last key that the row sees (rows that are none: any)
            float base = -INFINITY, l = 0.f;
            for (int i = 0; i < n; i++, steps++, swaps++) {
                const int last = sees - i * kKT - 64 * half;               // columns 0 .. last are seen
                const bool part = __any_sync(~0u, last < 63);
                wait(&sfull[w], steps & 1u);
                tc_fence_after();
                float v[64];
                tmem_ld32_async(ts, v);
                tmem_ld32_async(ts + 32, v + 32);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(sread);
                const bool taken_p = i == 0 || mbar_try_wait(&odone[w], (steps - 1) & 1u);   // P of the tile before has been taken
                if (flip) {
                    #pragma unroll
                    for (int x = 0; x < 64; x++) v[x] = -v[x];
                }
                if (part) {
                    #pragma unroll
                    for (int x = 0; x < 64; x++) if (x > last) v[x] = -INFINITY;
                }
                float mx[4] = {v[0], v[1], v[2], v[3]};
                #pragma unroll
                for (int x = 4; x < 60; x += 8)
                    #pragma unroll
                    for (int y = 0; y < 4; y++) mx[y] = max3(mx[y], v[x + y], v[x + y + 4]);
                #pragma unroll
                for (int y = 0; y < 4; y++) mx[y] = fmaxf(mx[y], v[60 + y]);
                float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                mine[swaps % 2 * 256] = top;
                named_bar(2 + w, 256);
                top = fmaxf(top, other[swaps % 2 * 256]);
                const float want = top == -INFINITY ? top : fmaf(top, c, -kLift);   // an all-masked tile stays -inf
                const bool move = want > base + 8.0f;                      // (from -inf: the first tile that has a key)
                float f = 1.0f;
                if (move) {
                    f = exp2_approx(base - want);
                    l *= f;
                    base = want;
                }
                if (i > 0 && __any_sync(~0u, move)) {
                    if (!taken_p) wait(&odone[w], (steps - 1) & 1u);       // O of the tile before
                    tc_fence_after();
                    #pragma unroll 1
                    for (int c0 = 0; c0 < D / 2; c0 += 8) scale8(to + c0, f);
                    ta::tc_wait_st();
                }
                if (half) {                                                // the first half's product adds to all columns of O, these warps' too
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pfull[2 * w]);
                }
                const float from = base == -INFINITY ? 0.f : base;
                uint64_t sum = pair(0.f, 0.f);
                const uint64_t c2 = pair(c, c), from2 = pair(-from, -from);
                uint32_t p[16];
                #pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    #pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        float a, b;
                        halves(pair_fma(pair(v[c0 + x], v[c0 + x + 1]), c2, from2), a, b);
                        a = exp2_approx(a);
                        b = exp2_approx(b);
                        sum = pair_add(sum, pair(a, b));
                        p[x / 2] = pack2<BF>(a, b);
                    }
                    if (c0 == 0) {
                        if (!taken_p) wait(&odone[w], (steps - 1) & 1u);
                        tc_fence_after();
                    }
                    ta::tc_st16(tp + c0 / 2, p);
                }
                ta::tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[2 * w + half]);
                float sum0, sum1;
                halves(sum, sum0, sum1);
                l += sum0 + sum1;
            }
            // ---- the row: this thread's half of the dims ----
            if (n) {
                mine[swaps % 2 * 256] = l;
                named_bar(2 + w, 256);
                l += other[swaps % 2 * 256];
                swaps++;
                wait(&odone[w], (steps - 1) & 1u);
                tc_fence_after();
            }
            it = *item;
            const bool live = placed && token < it.nq;
            const bool odd = live && *(const volatile int*)&item->odd != 0;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            uint8_t* dst = P.out + ((size_t)(it.q0 + token) * P.ldo + (size_t)(it.h * P.group + head) * D + half * (D / 2)) * 2;
            #pragma unroll 1
            for (int c0 = 0; c0 < D / 2; c0 += 16) {
                float o[16];
                if (n) tmem_ld16(to + c0, o);
                if (odd) {
                    for (int key = (max(it.off, -1) + 1) / kKT * kKT; key <= sees; key++) {
                        const uint16_t* row = reinterpret_cast<const uint16_t*>(P.v) + (size_t)(it.k0 + key) * P.ldv + (size_t)it.h * D + half * (D / 2) + c0;
                        constexpr uint32_t kExp = BF ? 0x7f80u : 0x7c00u;
                        #pragma unroll
                        for (int x = 0; x < 16; x++) {
                            const uint16_t b = row[x];
                            if ((b & kExp) == kExp) o[x] += BF ? bf2f(b) : __half2float(__ushort_as_half(b));
                        }
                    }
                }
                uint32_t b[8];
                #pragma unroll
                for (int x = 0; x < 8; x++) {
                    const float y = sees < 0 ? 0.f : o[2 * x] * inv, z = sees < 0 ? 0.f : o[2 * x + 1] * inv;
                    b[x] = pack2<BF>(y, z);
                }
                if (live) {
                    if (P.out32) {
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c0 * 2), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3]),
                                     "r"(b[4]), "r"(b[5]), "r"(b[6]), "r"(b[7]) : "memory");
                    } else {
                        *reinterpret_cast<uint4*>(dst + c0 * 2) = make_uint4(b[0], b[1], b[2], b[3]);
                        *reinterpret_cast<uint4*>(dst + c0 * 2 + 16) = make_uint4(b[4], b[5], b[6], b[7]);
                    }
                }
            }
            tc_fence_before();
            item_done();
        }
        finish();
    }
}

}  // namespace pr
}  // namespace qb
