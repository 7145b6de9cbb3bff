// draft_ops.cu — the C ABI of the drafted-token operators (qwen_kv_append,
// qwen_kv_read, qwen_kv_keep, qwen_tree_attention, qwen_tree_verify): argument
// checks, variant choice and launches.  No reference counterpart (the
// reference decodes one token per step, main.cu:141-145).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <string>

#include "../../include/qwen_b200.h"
#include "kv_rows.cuh"
#include "tree_attention.cuh"
#include "tree_attention_tc.cuh"
#include "tree_verify.cuh"

int qwen_internal_fail(int code, const std::string& msg);

namespace {

int fail(int code, const std::string& msg) { return qwen_internal_fail(code, msg); }
#define CU(call)                                                                                        \
    do {                                                                                                \
        cudaError_t e_ = (call);                                                                        \
        if (e_ != cudaSuccess) return fail(QWEN_E_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
    } while (0)
#define TRY(call)                          \
    do {                                   \
        int rc_ = (call);                  \
        if (rc_ != QWEN_OK) return rc_;    \
    } while (0)

// ---- waits (qwen_debug_draft_wait) ---------------------------------------------
constexpr unsigned long long kWaitNs = 1000000000ull;   // for copies and products on this GPU: they take microseconds
std::atomic<unsigned long long> g_wait_ns{kWaitNs};
std::atomic<int> g_withheld{-1};

// ---- argument checks -----------------------------------------------------------
struct Ptr {
    const void* p;
    const char* name;
    size_t align;
    bool used;   // false: may be anything
};
// NULL and alignment first (no GPU needed), then: device memory of the current device, *dev.
int check_ptrs(std::initializer_list<Ptr> ptrs, int* dev) {
    for (const Ptr& a : ptrs) {
        if (!a.used) continue;
        if (!a.p) return fail(QWEN_E_ARG, std::string(a.name) + " is NULL");
        if ((uintptr_t)a.p % a.align) return fail(QWEN_E_ARG, std::string(a.name) + " must be " + std::to_string(a.align) + "-byte aligned");
    }
    CU(cudaGetDevice(dev));
    for (const Ptr& a : ptrs) {
        if (!a.used) continue;
        cudaPointerAttributes at;
        const cudaError_t e = cudaPointerGetAttributes(&at, a.p);
        if (e != cudaSuccess) cudaGetLastError();   // not left behind for the caller's next query
        if (e != cudaSuccess || (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged))
            return fail(QWEN_E_ARG, std::string(a.name) + " is not device memory");
        if (at.type == cudaMemoryTypeDevice && at.device != *dev)
            return fail(QWEN_E_ARG, std::string(a.name) + " lies on another device than the current one");
    }
    return QWEN_OK;
}
bool is16(int t) { return t == QWEN_BF16 || t == QWEN_FP16; }
bool is8(int t) { return t == QWEN_E4M3 || t == QWEN_INT8; }

int check_view(const qwen_kv_cache_t* c) {
    if (!c) return fail(QWEN_E_ARG, "NULL cache view");
    if (!is16(c->dtype) && !is8(c->dtype)) return fail(QWEN_E_ARG, "cache dtype must be QWEN_BF16, QWEN_FP16, QWEN_E4M3 or QWEN_INT8");
    if (c->head_dim != 64 && c->head_dim != 128) return fail(QWEN_E_UNSUPPORTED, "head_dim must be 64 or 128");
    if (c->n_seqs < 1 || c->n_seqs > 65535) return fail(QWEN_E_ARG, "n_seqs out of [1, 65535]");
    if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return fail(QWEN_E_ARG, "n_kv_heads out of [1, 65535]");
    if (c->capacity < 1 || c->capacity > 1 << 30) return fail(QWEN_E_ARG, "capacity out of [1, 2^30]");
    const long long row = (long long)c->capacity * c->head_dim;
    if (c->head_stride % c->head_dim || c->seq_stride % c->head_dim || (c->n_kv_heads > 1 && c->head_stride < row) ||
        (c->n_seqs > 1 && c->seq_stride < row) || c->head_stride < 0 || c->seq_stride < 0)
        return fail(QWEN_E_ARG, "strides must be multiples of head_dim and at least capacity * head_dim");
    if (is16(c->dtype) && (c->k_scale || c->v_scale)) return fail(QWEN_E_ARG, "a 16-bit cache has no scales");
    return QWEN_OK;
}
// The view's pointers, as check_ptrs takes them.
#define QB_VIEW_PTRS(c)                                                                                              \
    Ptr{(c)->k, "cache k", 16, true}, Ptr{(c)->v, "cache v", 16, true}, Ptr{(c)->k_scale, "cache k_scale", 4, is8((c)->dtype)}, \
        Ptr{(c)->v_scale, "cache v_scale", 4, is8((c)->dtype)}
qb::kv::Cache device_view(const qwen_kv_cache_t* c) {
    return qb::kv::Cache{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, c->seq_stride, c->head_stride, c->capacity};
}
int sm_count(int dev, int* n) {
    static std::atomic<int> known[64];
    if (dev < 0 || dev >= 64) return fail(QWEN_E_ARG, "device index beyond 63");
    int v = known[dev].load();
    if (!v) {
        CU(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
        known[dev].store(v);
    }
    *n = v;
    return QWEN_OK;
}
// Sets a kernel's shared-memory limit once per device (not a stream operation: allowed during capture).
template <typename K>
int smem_limit(K kernel, std::atomic<uint64_t>& done, int dev, int bytes) {
    if (!((done.load() >> dev) & 1)) {
        CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(1ull << dev);
    }
    return QWEN_OK;
}

// ---- cache rows -------------------------------------------------------------------
template <template <int, int, int> class F, typename... A>
int by_types(int rows, int store, int dim, A... a) {
#define QB_STORES(R, D)                                                      \
    switch (store) {                                                         \
        case QWEN_BF16: return F<R, QWEN_BF16, D>::go(a...);                 \
        case QWEN_FP16: return F<R, QWEN_FP16, D>::go(a...);                 \
        case QWEN_E4M3: return F<R, QWEN_E4M3, D>::go(a...);                 \
        default: return F<R, QWEN_INT8, D>::go(a...);                        \
    }
#define QB_ROWS(D)                                                           \
    switch (rows) {                                                          \
        case QWEN_BF16: QB_STORES(QWEN_BF16, D)                              \
        case QWEN_FP16: QB_STORES(QWEN_FP16, D)                              \
        default: QB_STORES(QWEN_FP32, D)                                     \
    }
    if (dim == 64) { QB_ROWS(64) }
    QB_ROWS(128)
#undef QB_ROWS
#undef QB_STORES
}

template <int R, int S, int D>
struct Append {
    static int go(const qwen_kv_cache_t* c, const void* k, const void* v, long long ld, int n_tokens, const int* start, const int* counts,
                  cudaStream_t st) {
        // blocks of one head's tokens where a head has as many tokens as a block takes (measured at 16 x 2048 tokens, bf16 to int8:
        // 38 us against 44 with rows in one order; 3 x 517 tokens: 6.0 us against 5.2)
        const unsigned rows = (unsigned)c->n_kv_heads * (unsigned)n_tokens, per = qb::kv::Place<D>::kRows;
        const bool two = n_tokens >= 2 * (int)per && (double)rows * c->n_seqs >= 4096.0 * per;   // (and every SM gets several blocks)
        const dim3 grid(two ? (unsigned)c->n_kv_heads * ((n_tokens + 2 * per - 1) / (2 * per)) : (rows + per - 1) / per, c->n_seqs, 2);
        const auto kernel = two ? qb::kv::append_kernel<R, S, D, 2> : qb::kv::append_kernel<R, S, D, 1>;
        kernel<<<grid, qb::kv::kThreads, 0, st>>>(device_view(c), (const uint8_t*)k, (const uint8_t*)v, ld, c->n_kv_heads, n_tokens, start, counts);
        CU(cudaGetLastError());
        return QWEN_OK;
    }
};
template <int R, int S, int D>
struct Read {
    static int go(const qwen_kv_cache_t* c, void* k, void* v, long long ld, int n_tokens, const int* start, const int* counts, cudaStream_t st) {
        const unsigned rows = (unsigned)c->n_kv_heads * (unsigned)n_tokens, per = qb::kv::Place<D>::kRows;
        qb::kv::read_kernel<R, S, D><<<dim3((rows + per - 1) / per, c->n_seqs, 2), qb::kv::kThreads, 0, st>>>(
            device_view(c), (uint8_t*)k, (uint8_t*)v, ld, c->n_kv_heads, n_tokens, start, counts);
        CU(cudaGetLastError());
        return QWEN_OK;
    }
};

int check_rows(const qwen_kv_cache_t* c, const void* k, const void* v, int dtype, long long ld, int n_tokens, const int* start,
               const int* counts) {
    int dev = 0;
    TRY(check_view(c));
    if (!is16(dtype) && dtype != QWEN_FP32) return fail(QWEN_E_ARG, "rows must be QWEN_BF16, QWEN_FP16 or QWEN_FP32");
    if (n_tokens < 1 || n_tokens > c->capacity) return fail(QWEN_E_ARG, "n_tokens out of [1, capacity]");
    if ((long long)n_tokens * c->n_kv_heads >= 1ll << 31) return fail(QWEN_E_UNSUPPORTED, "n_tokens * n_kv_heads must be below 2^31");
    if (ld % 8 || ld < (long long)c->n_kv_heads * c->head_dim) return fail(QWEN_E_ARG, "ld must be a multiple of 8 and hold every head");
    return check_ptrs({QB_VIEW_PTRS(c), {k, "k", 16, true}, {v, "v", 16, true}, {start, "start", 4, true}, {counts, "counts", 4, counts != nullptr}},
                      &dev);
}

// ---- tree attention ----------------------------------------------------------------
// The kernel's variant, by the query rows of a K/V head (nodes times query heads):
// up to 16 and up to 32 the warp-level kernel, in one block of rows; above, where it
// would read the cache once for every 32 rows, the tensor-memory kernel in blocks
// of 128.  Both sides measured, 8 K/V heads of 128, warp-level / tensor memory: 24 rows, 16
// sequences at 2048 37.5 / 39.7 us (e4m3 34.0 / 57.9), one at 8128 21.4 / 18.1 (e4m3 17.1 /
// 22.1); 40 rows 57 / 40 us (e4m3 53.4 / 58.5), one at 8128 24.9 / 18.3 (e4m3 19.7 / 22.4).
// So the rule by rows alone costs up to 15 % in two places: one long sequence of 17 to
// 32 rows in 16 bits, and 33 to 64 rows over 8-bit caches.
int attention_rows(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : 128; }

struct Plan {
    int rows, row_blocks, beside, shares;   // shares: CTAs, beside for each share of the line
    int tiles, blocks;                      // of a cache's capacity: the kernel's tiles; blocks of 64 keys (tensor-memory kernel: 128)
    long long items;                        // sequences, K/V heads and blocks of rows
    float spare;
    bool whole, may_be_whole;               // a CTA for each item, no joining
    size_t bytes;
};
int check_tree(const qwen_kv_cache_t* c, int n_nodes, int n_heads) {
    if (n_nodes < 1 || n_nodes > qb::ta::kMaxNodes) return fail(QWEN_E_ARG, "n_nodes out of [1, 64]");
    if (n_heads < 1 || n_heads % c->n_kv_heads) return fail(QWEN_E_ARG, "n_heads must be a positive multiple of n_kv_heads");
    if (n_heads / c->n_kv_heads > 1 << 14) return fail(QWEN_E_UNSUPPORTED, "more than 2^14 query heads for each K/V head");
    return QWEN_OK;
}
// What the plan has without the device.  Caches of a few blocks of 64 keys have a CTA for each item: sharing the blocks out would
// spare a CTA all but items * blocks / CTAs of them, about 0.5 us each (1.3 us for 128 in the tensor-memory kernel), and joining
// costs 3.5 to 4.5 us.  Measured, a CTA for each item against shares, one query token and 8 K/V heads of 128, bf16: 1 sequence of
// 500 8.4 / 6.9 us, 8 of 500 8.5 / 10.7, 8 of 1000 14.5 / 12.5, 32 of 1000 24.6 / 29.7; e4m3: 1 of 500 8.4 / 7.7, 8 of 500 8.5 /
// 9.9, 8 of 1000 13.4 / 12.6, 32 of 1000 18.7 / 23.2.  Heads of 64, int8: 1 of 500 6.2 / 6.4, 8 of 1000 9.5 / 9.7; bf16: 1 of 500
// 5.7 / 6.4, 8 of 1000 8.2 / 9.6 (there the blocks cost less, and the rule shares out too soon).  64 nodes, bf16: 1 sequence of
// 440 12.7 / 12.0, 4 of 440 12.8 / 14.8, 4 of 900 18.2 / 16.3; e4m3: 1 of 240 21.0 / 17.3 (which the rule gives to one CTA), 4 of
// 440 22.6 / 23.1, 4 of 900 31.5 / 25.7.  Longer caches are shared out in any case, so that ragged lengths balance.
void attention_shape(const qwen_kv_cache_t* c, int n_nodes, int n_heads, Plan* p) {
    const int m = n_nodes * (n_heads / c->n_kv_heads);
    p->rows = attention_rows(m);
    p->row_blocks = (m + p->rows - 1) / p->rows;
    const bool tc = p->rows > 32;
    const int keys = tc ? qb::ta::kTcKT : qb::ta::tile_keys(is8(c->dtype) ? c->head_dim : 2 * c->head_dim);
    p->tiles = (c->capacity + keys - 1) / keys;
    p->blocks = (c->capacity + (tc ? 127 : 63)) / (tc ? 128 : 64);
    p->items = (long long)c->n_seqs * c->n_kv_heads * p->row_blocks;
    p->spare = tc ? 3.4f : 7.0f;      // so many blocks are worth the joining
    p->whole = p->blocks <= p->spare && p->items < 1 << 30;
    p->may_be_whole = p->blocks <= (tc ? 8 : 16) && p->items < 1 << 30;
}
int attention_plan(const qwen_kv_cache_t* c, int n_nodes, int n_heads, int dev, Plan* p) {
    attention_shape(c, n_nodes, n_heads, p);
    int nsm = 0, ctas = 0;
    if (!p->whole) {
        TRY(sm_count(dev, &nsm));
        ctas = p->rows <= 32 ? qb::ta::attention_ctas(p->rows, c->head_dim) * nsm : nsm;
        p->whole = p->may_be_whole && (double)p->blocks * std::max(0ll, ctas - p->items) <= (double)p->spare * ctas;
    }
    if (p->whole) {
        p->beside = p->row_blocks;
        p->shares = (int)p->items;
        p->bytes = 0;
        return QWEN_OK;
    }
    // as many CTAs as the SMs hold (the tensor-memory kernel: one each), shared out over the blocks of rows that walk side by side
    p->beside = p->row_blocks <= ctas ? p->row_blocks : 1;
    // no more shares than the line can have positions
    const double most = (double)c->n_seqs * c->n_kv_heads * (p->row_blocks / p->beside) *
                        (p->tiles + qb::ta::kTcItemCost);
    p->shares = (int)std::min((double)(ctas / p->beside), most) * p->beside;
    if (most >= 2147483648.0) return fail(QWEN_E_UNSUPPORTED, "too many sequences, heads and positions for one call");
    p->bytes = (size_t)2 * p->shares * p->rows * (c->head_dim + 2) * sizeof(float);
    return QWEN_OK;
}

// The kernel that joins the shares' partial results, launched so that it may start its set-up early.
template <int QT, int KT, int COST, int D, int ROWS, bool ACROSS>
int join_launch(const qb::ta::Params& P, const Plan& plan, int dev, cudaStream_t st) {
    int nsm = 0;
    TRY(sm_count(dev, &nsm));
    if (plan.whole || plan.shares == plan.beside) return QWEN_OK;
    cudaLaunchConfig_t cfg = {};
    const int wide = P.by_item ? P.n_seqs * P.n_kv_heads * P.row_blocks : plan.shares;
    cfg.gridDim = dim3(wide, qb::ta::join_blocks<D, ROWS, ACROSS>());
    if (P.by_item) {
        // Shared memory, so that no SM holds more blocks than an even spread over the SMs gives: the first SMs to finish their
        // share would take six and read those items' partial results alone (one sequence of 64 nodes at 8128: 24.3 us, against 19.9).
        const int each = std::max(1, ((int)cfg.gridDim.y * wide + nsm - 1) / nsm);
        cfg.dynamicSmemBytes = each <= 4 ? (220 * 1024 / each - 1024) / 1024 * 1024 : 0;
        static std::atomic<uint64_t> done{0};
        TRY(smem_limit(qb::ta::combine_kernel<QT, KT, COST, D, ROWS, ACROSS>, done, dev, 219 * 1024));
    }
    cfg.blockDim = dim3(qb::ta::kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CU(cudaLaunchKernelEx(&cfg, qb::ta::combine_kernel<QT, KT, COST, D, ROWS, ACROSS>, P));
    return QWEN_OK;
}
template <int QT, int STORE, int D, int MT>
int attention_launch(const qb::ta::Params& P, const Plan& plan, int dev, cudaStream_t st) {
    using L = qb::ta::Layout<STORE, D, MT>;
    static std::atomic<uint64_t> done{0};
    auto kernel = qb::ta::attention_kernel<QT, STORE, D, MT>;
    TRY(smem_limit(kernel, done, dev, L::kSmem));
    kernel<<<plan.shares, qb::ta::kThreads, L::kSmem, st>>>(P);
    CU(cudaGetLastError());
    return join_launch<QT, L::KT, qb::ta::kItemCost, D, L::kRows, false>(P, plan, dev, st);
}
template <int QT, int STORE, int D>
int attention_tc_launch(const qb::ta::Params& P, const Plan& plan, int dev, cudaStream_t st) {
    using L = qb::ta::TcLayout<STORE, D>;
    static std::atomic<uint64_t> done{0};
    auto kernel = qb::ta::attention_tc_kernel<QT, STORE, D>;
    TRY(smem_limit(kernel, done, dev, L::kSmem));
    kernel<<<plan.shares, qb::ta::kTcThreads, L::kSmem, st>>>(P);
    CU(cudaGetLastError());
    return join_launch<QT, qb::ta::kTcKT, qb::ta::kTcItemCost, D, qb::ta::kTcRows, true>(P, plan, dev, st);
}
template <int QT, int STORE, int D>
int attention_by_rows(const qb::ta::Params& P, const Plan& plan, int dev, cudaStream_t st) {
    switch (plan.rows) {
        case 16: return attention_launch<QT, STORE, D, 1>(P, plan, dev, st);
        case 32: return attention_launch<QT, STORE, D, 2>(P, plan, dev, st);
        default: return attention_tc_launch<QT, STORE, D>(P, plan, dev, st);
    }
}
template <int QT, int STORE>
int attention_by_shape(int dim, const qb::ta::Params& P, const Plan& plan, int dev, cudaStream_t st) {
    return dim == 64 ? attention_by_rows<QT, STORE, 64>(P, plan, dev, st) : attention_by_rows<QT, STORE, 128>(P, plan, dev, st);
}

// ---- verification --------------------------------------------------------------------
// CTAs for a sequence: as many as the SMs have for each of them, a run of 128
// tokens at least for each warp; 16 (more than every GPU must offer) where the
// device can hold that many such clusters.  Row buffers: two, one or none,
// whichever fits.
constexpr int kVerifySmem = 208 * 1024;
template <int T>
int verify_launch(qb::tv::Params& P, int n_seqs, int nsm, int dev, cudaStream_t st) {
    using namespace qb::tv;
    static std::atomic<uint64_t> done{0};
    static std::atomic<int> wide[64];   // clusters of 16 that fit at once, + 1
    const auto kernel = verify_kernel<T, true>;
    if (!((done.load() >> dev) & 1)) {
        CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        CU(cudaFuncSetAttribute(verify_kernel<T, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    }
    TRY(smem_limit(kernel, done, dev, kVerifySmem));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    int n16 = wide[dev].load();
    if (!n16) {
        cfg.gridDim = dim3(16);
        at[0].val.clusterDim.x = 16;
        cfg.dynamicSmemBytes = kVerifySmem;
        if (cudaOccupancyMaxActiveClusters(&n16, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n16 = 0; }
        wide[dev].store(++n16);
    }
    const int runs = (P.vocab + kRun - 1) / kRun;
    int cluster = 1;
    while (cluster < kMaxCluster && (long long)n_seqs * cluster * 2 <= nsm && runs >= cluster * 2 * kWarps) cluster *= 2;
    if (cluster == 16 && n_seqs > n16 - 1) cluster = 8;
    const int parts = cluster * kWarps;
    const int part_runs = (runs + parts - 1) / parts;
    P.part_bytes = (part_runs + 1) / 2 * 2 * kRun * (T == QWEN_FP32 ? 4 : 2);   // whole steps of two runs
    const long long row = (long long)kWarps * P.part_bytes;
    P.buffers = 2 * row <= kVerifySmem ? 2 : row <= kVerifySmem ? 1 : 0;
    at[0].val.clusterDim.x = cluster;
    cfg.gridDim = dim3((unsigned)n_seqs * cluster);
    cfg.dynamicSmemBytes = (size_t)(P.buffers * row);
    if (P.buffers) CU(cudaLaunchKernelEx(&cfg, kernel, P));
    else CU(cudaLaunchKernelEx(&cfg, verify_kernel<T, false>, P));
    return QWEN_OK;
}

}  // namespace

extern "C" int qwen_debug_draft_wait(unsigned long long wait_ns, int part) {
    if (part < -1 || part >= qb::tv::kMaxNodes) return fail(QWEN_E_ARG, "part out of [-1, 63]");
    if (wait_ns != 0 && wait_ns < 1000000ull) return fail(QWEN_E_ARG, "wait limit below 1 ms");
    g_wait_ns.store(wait_ns ? wait_ns : kWaitNs);
    g_withheld.store(part);
    return QWEN_OK;
}

extern "C" int qwen_kv_append(const qwen_kv_cache_t* cache, const void* k, const void* v, int src_dtype, long long ld, int n_tokens,
                              const int* start, const int* counts, void* stream) {
    TRY(check_rows(cache, k, v, src_dtype, ld, n_tokens, start, counts));
    return by_types<Append>(src_dtype, cache->dtype, cache->head_dim, cache, k, v, ld, n_tokens, start, counts, (cudaStream_t)stream);
}

extern "C" int qwen_kv_read(const qwen_kv_cache_t* cache, void* k, void* v, int dst_dtype, long long ld, int n_tokens, const int* start,
                            const int* counts, void* stream) {
    TRY(check_rows(cache, k, v, dst_dtype, ld, n_tokens, start, counts));
    return by_types<Read>(dst_dtype, cache->dtype, cache->head_dim, cache, k, v, ld, n_tokens, start, counts, (cudaStream_t)stream);
}

extern "C" int qwen_kv_keep(const qwen_kv_cache_t* cache, const int* start, const int* path, const int* n_path, int n_nodes, void* stream) {
    int dev = 0;
    TRY(check_view(cache));
    if (n_nodes < 1 || n_nodes > qb::kv::kMaxNodes) return fail(QWEN_E_ARG, "n_nodes out of [1, 64]");
    TRY(check_ptrs({QB_VIEW_PTRS(cache), {start, "start", 4, true}, {path, "path", 4, true}, {n_path, "n_path", 4, true}}, &dev));
    const dim3 grid((cache->n_kv_heads + qb::kv::kKeepHeads - 1) / qb::kv::kKeepHeads, cache->n_seqs);
    const auto c = device_view(cache);
    const cudaStream_t st = (cudaStream_t)stream;
    const bool k8 = is8(cache->dtype), wide = cache->head_dim == 128;
    if (k8 && wide) qb::kv::keep_kernel<128, true><<<grid, qb::kv::kKeepThreads, 0, st>>>(c, start, path, n_path, cache->n_kv_heads, n_nodes, 1);
    else if (k8) qb::kv::keep_kernel<64, true><<<grid, qb::kv::kKeepThreads, 0, st>>>(c, start, path, n_path, cache->n_kv_heads, n_nodes, 1);
    else if (wide) qb::kv::keep_kernel<256, false><<<grid, qb::kv::kKeepThreads, 0, st>>>(c, start, path, n_path, cache->n_kv_heads, n_nodes, 2);
    else qb::kv::keep_kernel<128, false><<<grid, qb::kv::kKeepThreads, 0, st>>>(c, start, path, n_path, cache->n_kv_heads, n_nodes, 2);
    CU(cudaGetLastError());
    return QWEN_OK;
}

extern "C" int qwen_tree_attention_workspace(const qwen_kv_cache_t* cache, int n_nodes, int n_heads, size_t* bytes) {
    if (!bytes) return fail(QWEN_E_ARG, "NULL argument");
    TRY(check_view(cache));
    TRY(check_tree(cache, n_nodes, n_heads));
    Plan p;
    attention_shape(cache, n_nodes, n_heads, &p);
    int dev = 0;
    if (!p.whole) CU(cudaGetDevice(&dev));
    TRY(attention_plan(cache, n_nodes, n_heads, dev, &p));
    *bytes = p.bytes;
    return QWEN_OK;
}

extern "C" int qwen_tree_attention(const qwen_kv_cache_t* cache, const void* q, void* out, int dtype, long long ldq, long long ldo, int n_nodes,
                                   int n_heads, const int* lens, const int* parents, float scale, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    TRY(check_view(cache));
    if (!is16(dtype)) return fail(QWEN_E_ARG, "q and out must be QWEN_BF16 or QWEN_FP16");
    if (is16(cache->dtype) && cache->dtype != dtype) return fail(QWEN_E_ARG, "q and a 16-bit cache must have the same type");
    TRY(check_tree(cache, n_nodes, n_heads));
    const long long width = (long long)n_heads * cache->head_dim;
    if (ldq % 8 || ldo % 8 || ldq < width || ldo < width) return fail(QWEN_E_ARG, "ldq and ldo must be multiples of 8 and hold every head");
    if (!(std::fabs(scale) < 0x1p127f)) return fail(QWEN_E_ARG, "scale must be finite and below 2^127 in magnitude");   // (times log2 e)
    if (q == out) return fail(QWEN_E_ARG, "out must not be q");
    int dev = 0;
    Plan plan;
    attention_shape(cache, n_nodes, n_heads, &plan);
    TRY(check_ptrs({QB_VIEW_PTRS(cache), {q, "q", 16, true}, {out, "out", 16, true}, {lens, "lens", 4, true}, {parents, "parents", 4, true},
                    {workspace, "workspace", 16, workspace || !plan.may_be_whole}}, &dev));
    TRY(attention_plan(cache, n_nodes, n_heads, dev, &plan));
    if (plan.bytes && !workspace) return fail(QWEN_E_ARG, "workspace is NULL");
    if (workspace_bytes < plan.bytes) return fail(QWEN_E_ARG, "workspace is smaller than qwen_tree_attention_workspace says");
    qb::ta::Params P;
    P.cache = device_view(cache);
    P.q = (const uint8_t*)q;
    P.out = (uint8_t*)out;
    P.lens = lens;
    P.parents = parents;
    P.work = (float*)workspace;
    P.ldq = ldq;
    P.ldo = ldo;
    P.n_seqs = cache->n_seqs;
    P.n_kv_heads = cache->n_kv_heads;
    P.group = n_heads / cache->n_kv_heads;
    P.per_group = 1.0f / (float)P.group;
    P.n_nodes = n_nodes;
    P.whole = plan.whole;
    P.row_blocks = plan.row_blocks;
    P.beside = plan.beside;
    P.groups = plan.shares / plan.beside;
    P.by_item = !plan.whole && (long long)P.n_seqs * P.n_kv_heads * (P.row_blocks / P.beside) <= P.groups;
    P.scale_log2 = scale * 1.4426950408889634f;
    P.wait_ns = g_wait_ns.load();
    P.withheld = g_withheld.load();
    const cudaStream_t st = (cudaStream_t)stream;
    const int dim = cache->head_dim;
    const bool bf = dtype == QWEN_BF16;
    switch (cache->dtype) {
        case QWEN_E4M3: return bf ? attention_by_shape<QWEN_BF16, QWEN_E4M3>(dim, P, plan, dev, st) : attention_by_shape<QWEN_FP16, QWEN_E4M3>(dim, P, plan, dev, st);
        case QWEN_INT8: return bf ? attention_by_shape<QWEN_BF16, QWEN_INT8>(dim, P, plan, dev, st) : attention_by_shape<QWEN_FP16, QWEN_INT8>(dim, P, plan, dev, st);
        default: return bf ? attention_by_shape<QWEN_BF16, QWEN_BF16>(dim, P, plan, dev, st) : attention_by_shape<QWEN_FP16, QWEN_FP16>(dim, P, plan, dev, st);
    }
}

extern "C" int qwen_tree_verify(const void* logits, int logits_dtype, long long ld, const float* draft, long long ld_draft, const int* tokens,
                                const int* parents, const float* uniforms, int n_seqs, int n_nodes, int vocab, float temperature, int* path,
                                int* n_path, int* next, void* stream) {
    if (!is16(logits_dtype) && logits_dtype != QWEN_FP32) return fail(QWEN_E_ARG, "logits must be QWEN_FP32, QWEN_BF16 or QWEN_FP16");
    if (n_seqs < 1 || n_seqs > 65535) return fail(QWEN_E_ARG, "n_seqs out of [1, 65535]");
    if (n_nodes < 1 || n_nodes > qb::tv::kMaxNodes) return fail(QWEN_E_ARG, "n_nodes out of [1, 64]");
    if (vocab < 1 || vocab > 1 << 30) return fail(QWEN_E_ARG, "vocab out of [1, 2^30]");
    if (ld < vocab || (draft && ld_draft < vocab)) return fail(QWEN_E_ARG, "ld and ld_draft must hold a row");
    if (!(temperature == 0.0f || (temperature >= 1e-6f && temperature <= 1e6f))) return fail(QWEN_E_ARG, "temperature must be 0 or within 1e-6 .. 1e6");
    const size_t elem = logits_dtype == QWEN_FP32 ? 4 : 2;
    const bool greedy = temperature == 0.0f;
    int dev = 0, nsm = 0;
    TRY(check_ptrs({{logits, "logits", elem, true}, {draft, "draft", 4, draft && !greedy}, {tokens, "tokens", 4, n_nodes > 1},
                    {parents, "parents", 4, true}, {uniforms, "uniforms", 4, !greedy}, {path, "path", 4, true}, {n_path, "n_path", 4, true},
                    {next, "next", 4, true}}, &dev));
    TRY(sm_count(dev, &nsm));
    qb::tv::Params P;
    P.logits = logits;
    P.draft = greedy ? nullptr : draft;
    P.tokens = tokens;
    P.parents = parents;
    P.uniforms = uniforms;
    P.path = path;
    P.n_path = n_path;
    P.next = next;
    P.ld = ld;
    P.ld_draft = ld_draft;
    P.n_nodes = n_nodes;
    P.vocab = vocab;
    const bool rows16 = ((uintptr_t)logits | (size_t)ld * elem) % 16 == 0;
    P.vec = rows16 && (!P.draft || ((uintptr_t)draft | (size_t)ld_draft * 4) % 16 == 0);
    P.temperature = temperature;
    P.wait_ns = g_wait_ns.load();
    P.withheld = g_withheld.load();
    const cudaStream_t st = (cudaStream_t)stream;
    switch (logits_dtype) {
        case QWEN_BF16: return verify_launch<QWEN_BF16>(P, n_seqs, nsm, dev, st);
        case QWEN_FP16: return verify_launch<QWEN_FP16>(P, n_seqs, nsm, dev, st);
        default: return verify_launch<QWEN_FP32>(P, n_seqs, nsm, dev, st);
    }
}
