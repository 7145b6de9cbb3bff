// prompt_attention.cuh — causal attention of packed prompts on the sm_100a tensor
// cores (qwen_prompt_attention).  No reference counterpart: the reference runs
// its decode attention once per prompt token (main.cu:141-145 over
// qwen_model.cuh:551-614).
//
// Mathematics.  Query i of a sequence with n queries and m keys sees keys 0 .. m - n +
// i.  One pass over tiles of 128 keys with the running maximum and sum of the softmax
// (base 2, scale * log2 e folded into the exponent): S = Q K^T, P = 2^(S c - base), O += P
// V.  A row's base follows its maximum only when that lies 2^8 above it, so O is seldom scaled; O
// / l at the end.
//
// A row of a tile is a (token, query head) pair of one K/V head, head fastest: T = 128 /
// group tokens of all the K/V head's query heads, so K and V serve the whole group.
// An item is two such row tiles, A and B, one behind the other, and their common key
// tiles: while the softmax of one is at work, the tensor cores form the other's products.
// Tensor memory: S of A and B (128 columns each, P written over them in 16 bits), O of A
// and B.  The tensor cores take the products in the order in which they are issued: S_A(i+1)
// follows P_A(i) V(i), which reads what it overwrites.
//
// Warps: 0-3 softmax and output of A (a thread a row), 4-7 of B, 8 loads (TMA), 9
// issues the products, 10 finds the items, 11 looks for infinities and NaN among the V
// rows of tiles that are not seen as a whole: 0 * NaN would reach rows that do not see them,
// so such values are zeroed in shared memory and added at the end to the rows that see them.
// Items, heaviest first, are dealt out to the CTAs forwards and backwards in turn; they are found on the device from
// starts and k_starts.  Every wait is bounded; where one runs out, the CTA's rows become NaN.
#pragma once
#include "tree_attention_tc.cuh"

namespace qb {
namespace pr {

using ta::add2;
using ta::exp2_approx;
using ta::fma2;
using ta::max3;
using ta::mul2;
using ta::pack2;

constexpr int kKT = 128;                  // keys of a tile
constexpr int kThreads = 384, kLoader = 8, kIssuer = 9, kFinder = 10, kLooker = 11;
constexpr int kItems = 4;                 // items between the finder and the slowest warp
constexpr int kClean = 4;                 // V parts that the looker may be ahead

struct Params {
    uint8_t* out;
    const uint8_t* v;
    const int *starts, *k_starts;
    long long ldv, ldo;
    int n_seqs, n_rows, n_keys, n_kv_heads, group, tokens;   // tokens: of a row tile
    int out32;                            // rows of out start on 32 bytes
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
    static constexpr int kRing = D == 64 ? 8 : 5;             // K / V parts in flight: K 0, V 0, K 1, V 1, ...
    static constexpr int kQ = 0;
    static constexpr int kKV = 2 * kPart;
    static constexpr int kBar = kKV + kRing * kPart;
    static constexpr int kBars = 2 * kRing + kClean + 2 * kItems + 11;
    static constexpr int kItem = kBar + (kBars * 8 + 15) / 16 * 16;
    static constexpr int kMisc = kItem + kItems * (int)sizeof(Item);
    static constexpr int kSmem = kMisc + 16 + 1024;
    static_assert(kRing / 2 + kRing % 2 <= kClean, "V parts in flight");
    static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
    static_assert(2 * kSmem > 228 * 1024, "one CTA an SM: the kernel allocates all of tensor memory");
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}
// 128 consecutive fp32 columns of this warp's 32 tensor-memory lanes (one row per lane).
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&v)[128]) {
    uint32_t r[128];
    asm volatile(
        "{\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63, "
        "%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, "
        "%80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, "
        "%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, "
        "%112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%128];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
          "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
          "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
          "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
          "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
          "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
          "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
          "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
          "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
        : "r"(taddr)
        : "memory");
    #pragma unroll
    for (int i = 0; i < 128; i++) v[i] = __uint_as_float(r[i]);
}

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
    // the tiles above level L
    __device__ __forceinline__ int above(const Params& P, int L) const {
        int n = 0;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) n += min(max(first[i] + count[i] - L, 0), count[i]);
        for (int s = 32 * kHeld + (threadIdx.x & 31); s < P.n_seqs; s += 32) {
            int f, c;
            levels(P, s, f, c);
            n += min(max(f + c - L, 0), c);
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
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBar);   // [kRing] a K or V part has arrived
    uint64_t* empty = full + L::kRing;                              // [kRing] its products are done
    uint64_t* clean = empty + L::kRing;                             // [kClean] a V part has been looked at
    uint64_t* given = clean + kClean;                               // [kItems] an item is there
    uint64_t* taken = given + kItems;                               // [kItems] all warps are done with it
    // [2]: A, B
    uint64_t* qfull = taken + kItems;                               // the item's rows have arrived
    uint64_t* qempty = qfull + 2;                                   // their last S is formed
    uint64_t* sfull = qfull + 4;                                    // S formed
    uint64_t* pfull = qfull + 6;                                    // P written, O scaled (4 warps)
    uint64_t* odone = qfull + 8;                                    // P V added
    uint64_t* drained = qfull + 10;                                 // all products are done, at the end
    Item* items = reinterpret_cast<Item*>(smem + L::kItem);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
    volatile int* fault = reinterpret_cast<int*>(smem + L::kMisc + 4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < L::kRing; i++) { mbar_init(&full[i], 1 + (i == P.withheld)); mbar_init(&empty[i], 1); }
        for (int i = 0; i < kClean; i++) mbar_init(&clean[i], 1);
        for (int i = 0; i < kItems; i++) { mbar_init(&given[i], 1); mbar_init(&taken[i], 11); }   // 8 softmax warps, loads, products, looker
        for (int w = 0; w < 2; w++) {
            mbar_init(&qfull[w], 1);
            mbar_init(&qempty[w], 1);
            mbar_init(&sfull[w], 1);
            mbar_init(&pfull[w], 4);
            mbar_init(&odone[w], 1);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
        *fault = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    if (warp == kIssuer) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Bounded; once a wait has run out anywhere in the CTA, none of the others is waited for (but an item's is).
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(bar, parity)) return;
        uint64_t since = 0;
        for (uint32_t n = 0; !*fault && !mbar_try_wait(bar, parity); n++) {
            if ((n & 255u) == 255u) {
                const uint64_t now = global_ns();
                if (!since) since = now;
                else if (now - since > P.wait_ns) *fault = 1;
            }
        }
    };
    uint32_t seen = 0;                        // items so far
    Item it;
    auto next_item = [&]() {                  // all lanes of a warp; false: no more
        const int slot = seen % kItems;
        if (!ta::mbar_spin(&given[slot], seen / kItems & 1u, 8 * P.wait_ns)) { *fault = 1; return false; }
        it = items[slot];
        return !it.stop;
    };
    auto item_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&taken[seen % kItems]);
        seen++;
    };

    if (warp == kFinder) {
        // ---------------- items ----------------
        const Finder finder(P);
        const int G = gridDim.x;
        bool more = true;
        for (int k = 0; more; k++) {
            const long long at = (long long)k * G + (k & 1 ? G - 1 - (int)blockIdx.x : (int)blockIdx.x);   // forwards and backwards
            int seq = 0, tile = 0;
            more = at / P.n_kv_heads < 0x7fffffff && finder.find(P, (int)(at / P.n_kv_heads), seq, tile);
            Item x = {};
            x.stop = !more;
            if (more) {
                int q0, nq, k0, nk;
                finder.bounds(P, seq, q0, nq, k0, nk);
                x.h = (int)(at % P.n_kv_heads);
                x.q0 = q0 + tile * finder.per;
                x.nq = min(nq - tile * finder.per, finder.per);
                x.k0 = k0;
                x.off = nk - nq + tile * finder.per;
                for (int w = 0; w < 2; w++) {
                    const int count = min(x.nq - w * P.tokens, P.tokens), last = x.off + w * P.tokens + count - 1;
                    x.n[w] = count <= 0 || last < 0 ? 0 : last / kKT + 1;
                }
            }
            const int slot = k % kItems;
            if (k >= kItems && !ta::mbar_spin(&taken[slot], (k / kItems - 1) & 1u, 8 * P.wait_ns)) { *fault = 1; break; }
            if (lane == 0) {
                items[slot] = x;
                mbar_arrive(&given[slot]);
            }
            __syncwarp();
        }
    } else if (warp == kLoader) {
        // ---------------- loads ----------------
        uint32_t part = 0, used[2] = {0, 0};   // K / V parts so far; items so far that have the row tile
        while (next_item()) {
            if (lane == 0) {
                const int n = max(it.n[0], it.n[1]);
                auto rows = [&](int w) {
                    if (!it.n[w]) return;
                    if (used[w]) wait(&qempty[w], (used[w] - 1) & 1u);
                    if (*fault) return;
                    used[w]++;
                    mbar_arrive_expect_tx(&qfull[w], P.tokens * P.group * D * 2);
                    #pragma unroll
                    for (int x = 0; x < D / 64; x++)
                        tma_load_3d(smem + L::kQ + w * L::kPart + x * (128 * 128), &map_q, 64 * x, it.h * P.group, it.q0 + w * P.tokens, &qfull[w]);
                };
                auto keys = [&](const CUtensorMap* map, int i) {
                    const uint32_t s = part % L::kRing;
                    if (part >= (uint32_t)L::kRing) wait(&empty[s], (part / L::kRing - 1) & 1u);
                    if (*fault) return;
                    mbar_arrive_expect_tx(&full[s], L::kPart);
                    #pragma unroll
                    for (int x = 0; x < D / 64; x++)
                        tma_load_2d(smem + L::kKV + s * L::kPart + x * (kKT * 128), map, it.h * D + 64 * x, it.k0 + i * kKT, &full[s]);
                    part++;
                };
                rows(0);
                for (int i = 0; i < n && !*fault; i++) {
                    keys(&map_k, i);
                    if (i == 0) rows(1);
                    keys(&map_v, i);
                }
            }
            item_done();
        }
        if (*fault && lane == 0) {             // nothing may still be on its way when the CTA ends
            for (uint32_t p = part > (uint32_t)L::kRing ? part - L::kRing : 0; p < part; p++) mbar_wait(&full[p % L::kRing], p / L::kRing & 1u, 10000000ull);
            for (int w = 0; w < 2; w++) if (used[w]) mbar_wait(&qfull[w], (used[w] - 1) & 1u, 10000000ull);
        }
        __syncwarp();
    } else if (warp == kIssuer) {
        // ---------------- products ----------------
        constexpr uint32_t id_s = ta::tc_idesc<BF>(kKT, false), id_o = ta::tc_idesc<BF>(D, true);
        uint32_t part = 0, used[2] = {0, 0}, steps[2] = {0, 0};   // steps: key tiles of a row tile so far
        while (next_item()) {
            if (lane == 0) {
                const int n = max(it.n[0], it.n[1]);
                auto form_s = [&](int w, int i) {
                    if (i >= it.n[w]) return;
                    if (i == 0) { wait(&qfull[w], used[w] & 1u); used[w]++; tc_fence_after(); }
                    const uint32_t kb = smem_addr(smem + L::kKV + (part + 2 * i) % L::kRing * L::kPart), qb = smem_addr(smem + L::kQ + w * L::kPart);
                    #pragma unroll
                    for (int k = 0; k < D / 16; k++)
                        mma_bf16(tmem + 128 * w, kmajor_sw128_desc(qb + (k >> 2) * (128 * 128) + (k & 3) * 32),
                                 kmajor_sw128_desc(kb + (k >> 2) * (kKT * 128) + (k & 3) * 32), id_s, k ? 1u : 0u);
                    mma_commit(&sfull[w]);
                    if (i + 1 == it.n[w]) mma_commit(&qempty[w]);
                };
                auto add_pv = [&](int w, int i) {
                    if (i >= it.n[w]) return;
                    wait(&pfull[w], steps[w] & 1u);
                    steps[w]++;
                    tc_fence_after();
                    const uint32_t vb = smem_addr(smem + L::kKV + (part + 2 * i + 1) % L::kRing * L::kPart);
                    #pragma unroll
                    for (int k = 0; k < kKT / 16; k++)
                        ta::tc_mma_ts(tmem + 256 + 128 * w, tmem + 128 * w + 8 * k, ta::mn_major_sw128_desc(vb + k * 2048, kKT * 128), id_o, (i | k) ? 1u : 0u);
                    mma_commit(&odone[w]);
                };
                auto arrived = [&](uint64_t* bar, uint32_t parity) { wait(bar, parity); tc_fence_after(); };
                if (n) {
                    arrived(&full[part % L::kRing], part / L::kRing & 1u);
                    form_s(0, 0);
                    form_s(1, 0);
                    mma_commit(&empty[part % L::kRing]);
                }
                for (int i = 0; i < n && !*fault; i++) {
                    const uint32_t pv = part + 2 * i + 1, pk = part + 2 * i + 2;
                    arrived(&clean[(pv >> 1) % kClean], (pv >> 1) / kClean & 1u);
                    add_pv(0, i);
                    if (i + 1 < n) arrived(&full[pk % L::kRing], pk / L::kRing & 1u);
                    form_s(0, i + 1);
                    add_pv(1, i);
                    mma_commit(&empty[pv % L::kRing]);
                    form_s(1, i + 1);
                    if (i + 1 < n) mma_commit(&empty[pk % L::kRing]);
                }
                part += 2 * n;
            }
            item_done();
        }
        if (lane == 0) {
            mma_commit(drained);
            if (!mbar_wait(drained, 0, P.wait_ns)) *fault = 1;
        }
        __syncwarp();
    } else if (warp == kLooker) {
        // ---------------- infinities and NaN among V rows that not all rows see ----------------
        uint32_t part = 0;
        while (next_item()) {
            const int n = max(it.n[0], it.n[1]);
            for (int i = 0; i < n && !*fault; i++) {
                const uint32_t pv = part + 2 * i + 1;
                // (K parts too: a slot of an odd ring holds K and V in turn, and a wait that skips a phase may take the one before for it)
                wait(&full[(pv - 1) % L::kRing], (pv - 1) / L::kRing & 1u);
                wait(&full[pv % L::kRing], pv / L::kRing & 1u);
                if (i * kKT + kKT - 1 > it.off) {
                    constexpr uint32_t kExp = BF ? 0x7f807f80u : 0x7c007c00u;
                    uint4* rows = reinterpret_cast<uint4*>(smem + L::kKV + pv % L::kRing * L::kPart);
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
                if (lane == 0) mbar_arrive(&clean[(pv >> 1) % kClean]);
            }
            part += 2 * n;
            item_done();
        }
    } else {
        // ---------------- softmax and output ----------------
        const int w = warp >> 2, rl = 32 * (warp & 3) + lane;              // row tile, row of it
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = tmem + lanes + 128 * w, to = tmem + lanes + 256 + 128 * w;
        const int token = w * P.tokens + rl / P.group, head = rl % P.group;
        const bool placed = rl < P.tokens * P.group;
        const float c = fmaxf(fabsf(P.scale_log2), 1e-37f);                // (above 0: -inf * 0 would be NaN)
        const float sign = P.scale_log2 < 0.f ? -1.0f : 1.0f;
        uint32_t steps = 0;                                                // key tiles so far
        while (next_item()) {
            const bool live = placed && token < it.nq;
            const int n = it.n[w], sees = live ? it.off + token : 1 << 30;   // the last key that the row sees (rows that are none: any)
            float base = -INFINITY, l = 0.f;
            for (int i = 0; i < n; i++, steps++) {
                wait(&sfull[w], steps & 1u);
                tc_fence_after();
                float v[128];
                tmem_ld128(ts, v);
                if (sign < 0.f) {
                    #pragma unroll
                    for (int x = 0; x < 128; x++) v[x] = -v[x];
                }
                const int last = sees - i * kKT;                           // columns 0 .. last are seen
                if (__any_sync(~0u, last < kKT - 1)) {
                    #pragma unroll
                    for (int x = 0; x < 128; x++) if (x > last) v[x] = -INFINITY;
                }
                float mx[4] = {v[0], v[1], v[2], v[3]};
                #pragma unroll
                for (int x = 4; x < 124; x += 8)
                    #pragma unroll
                    for (int y = 0; y < 4; y++) mx[y] = max3(mx[y], v[x + y], v[x + y + 4]);
                const float top = fmaxf(max3(max3(mx[0], v[124], v[125]), mx[1], mx[2]), max3(mx[3], v[126], v[127]));
                const float want = top == -INFINITY ? top : top * c;       // an all-masked tile stays -inf
                const bool move = want > base + 8.0f;                      // (from -inf: the first tile that has a key)
                float f = 1.0f;
                if (move) {
                    f = exp2_approx(base - want);
                    l *= f;
                    base = want;
                }
                if (i > 0 && __any_sync(~0u, move)) {
                    wait(&odone[w], (steps - 1) & 1u);                     // O of the tile before
                    tc_fence_after();
                    #pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        float o[16];
                        tmem_ld16(to + c0, o);
                        #pragma unroll
                        for (int x = 0; x < 16; x += 2) mul2(o[x], o[x + 1], f, f);
                        uint32_t b[16];
                        #pragma unroll
                        for (int x = 0; x < 16; x++) b[x] = __float_as_uint(o[x]);
                        ta::tc_st16(to + c0, b);
                    }
                }
                const float from = base == -INFINITY ? 0.f : base;
                float sum0 = 0.f, sum1 = 0.f;
                #pragma unroll
                for (int c0 = 0; c0 < 128; c0 += 32) {
                    uint32_t p[16];
                    #pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        float &a = v[c0 + x], &b = v[c0 + x + 1];
                        fma2(a, b, c, -from);
                        a = exp2_approx(a);
                        b = exp2_approx(b);
                        add2(sum0, sum1, a, b);
                        p[x / 2] = pack2<BF>(a, b);
                    }
                    ta::tc_st16(ts + c0 / 2, p);
                }
                l += sum0 + sum1;
                ta::tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[w]);
            }
            // ---- the row ----
            if (n) {
                wait(&odone[w], (steps - 1) & 1u);
                tc_fence_after();
            }
            const bool failed = *fault != 0;
            const bool odd = live && *(volatile int*)&items[seen % kItems].odd != 0;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            uint8_t* dst = P.out + ((size_t)(it.q0 + token) * P.ldo + (size_t)(it.h * P.group + head) * D) * 2;
            #pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                float o[32];
                if (n) tmem_ld32(to + c0, o);
                if (odd) {
                    for (int key = (max(it.off, -1) + 1) / kKT * kKT; key <= sees; key++) {
                        const uint16_t* row = reinterpret_cast<const uint16_t*>(P.v) + (size_t)(it.k0 + key) * P.ldv + (size_t)it.h * D + c0;
                        constexpr uint32_t kExp = BF ? 0x7f80u : 0x7c00u;
                        #pragma unroll
                        for (int x = 0; x < 32; x++) {
                            const uint16_t b = row[x];
                            if ((b & kExp) == kExp) o[x] += BF ? bf2f(b) : __half2float(__ushort_as_half(b));
                        }
                    }
                }
                uint32_t b[16];
                #pragma unroll
                for (int x = 0; x < 16; x++) {
                    const float y = failed ? NAN : sees < 0 ? 0.f : o[2 * x] * inv, z = failed ? NAN : sees < 0 ? 0.f : o[2 * x + 1] * inv;
                    b[x] = pack2<BF>(y, z);
                }
                if (live) {
                    if (P.out32) {
                        #pragma unroll
                        for (int x = 0; x < 16; x += 8)
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c0 * 2 + x * 4), "r"(b[x]), "r"(b[x + 1]), "r"(b[x + 2]),
                                         "r"(b[x + 3]), "r"(b[x + 4]), "r"(b[x + 5]), "r"(b[x + 6]), "r"(b[x + 7]) : "memory");
                    } else {
                        #pragma unroll
                        for (int x = 0; x < 16; x += 4) *reinterpret_cast<uint4*>(dst + c0 * 2 + x * 4) = make_uint4(b[x], b[x + 1], b[x + 2], b[x + 3]);
                    }
                }
            }
            tc_fence_before();
            item_done();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

}  // namespace pr
}  // namespace qb
