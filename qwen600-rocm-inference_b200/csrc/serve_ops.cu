// serve_ops.cu — the C ABI of the operators of serving over a K/V cache in pages
// (qwen_qk_rope, qwen_prompt_attention, qwen_paged_attention, qwen_token_logprobs):
// argument checks, variant choice and launches.  No reference counterpart (the
// reference serves one sequence, token by token, main.cu:141-145).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <string>

#include "../../include/qwen_b200.h"
#include "attention_plan.cuh"
#include "kv_pages.cuh"
#include "op_checks.cuh"
#include "paged_attention.cuh"
#include "prompt_attention.cuh"
#include "token_logprobs.cuh"

unsigned long long qwen_internal_wait_ns();   // draft_ops.cu
int qwen_internal_withheld();

namespace {

// ---- argument checks -----------------------------------------------------------
bool is_rows(int t) { return is16(t) || t == QWEN_FP32; }
int check_heads(int n_heads, int n_kv_heads, int head_dim) {
    if (head_dim != 64 && head_dim != 128) return fail(QWEN_E_UNSUPPORTED, "head_dim must be 64 or 128");
    if (n_kv_heads < 1 || n_kv_heads > 65535) return fail(QWEN_E_ARG, "n_kv_heads out of [1, 65535]");
    if (n_heads < 1 || n_heads % n_kv_heads) return fail(QWEN_E_ARG, "n_heads must be a positive multiple of n_kv_heads");
    if (n_heads / n_kv_heads > 1 << 14) return fail(QWEN_E_UNSUPPORTED, "more than 2^14 query heads for each K/V head");
    return QWEN_OK;
}
int check_ld(long long ld, long long heads, int head_dim, const char* name) {
    if (ld % 8 || ld < heads * head_dim || ld > 1ll << 36) return fail(QWEN_E_ARG, std::string(name) + " must be a multiple of 8 (up to 2^36) and hold every head");
    return QWEN_OK;
}
int check_scale(float scale) {
    if (!(std::fabs(scale) < 0x1p127f)) return fail(QWEN_E_ARG, "scale must be finite and below 2^127 in magnitude");   // (times log2 e)
    return QWEN_OK;
}
int check_pages(const qwen_kv_pages_t* c) {
    if (!c) return fail(QWEN_E_ARG, "NULL view of pages");
    if (!is16(c->dtype) && !is8(c->dtype)) return fail(QWEN_E_ARG, "pages' dtype must be QWEN_BF16, QWEN_FP16, QWEN_E4M3 or QWEN_INT8");
    if (c->head_dim != 64 && c->head_dim != 128) return fail(QWEN_E_UNSUPPORTED, "head_dim must be 64 or 128");
    if (c->n_pages < 1) return fail(QWEN_E_ARG, "n_pages must be positive");
    if (c->n_seqs < 1 || c->n_seqs > 65535) return fail(QWEN_E_ARG, "n_seqs out of [1, 65535]");
    if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return fail(QWEN_E_ARG, "n_kv_heads out of [1, 65535]");
    if (c->page_size < 1 || c->page_size > 1 << 16 || (c->page_size & (c->page_size - 1))) return fail(QWEN_E_ARG, "page_size must be a power of two up to 2^16");
    if (c->max_pages < 1 || (long long)c->max_pages * c->page_size > 1 << 30) return fail(QWEN_E_ARG, "max_pages * page_size out of [1, 2^30]");
    if (c->page_stride < 0 || c->head_stride < 0 || c->page_stride % c->head_dim || c->head_stride % c->head_dim)
        return fail(QWEN_E_ARG, "strides must be multiples of head_dim and not negative");
    if (is16(c->dtype) && (c->k_scale || c->v_scale)) return fail(QWEN_E_ARG, "16-bit pages have no scales");
    // rows of heads and pages that begin at the same place, or inside one another's pages
    const long long row = (long long)c->page_size * c->head_dim;
    if ((c->n_kv_heads > 1 && c->head_stride < row) || (c->n_pages > 1 && c->page_stride < row))
        return fail(QWEN_E_ARG, "strides must be at least page_size * head_dim");
    return QWEN_OK;
}
// The view's pointers, as check_ptrs takes them.
#define QB_PAGES_PTRS(c, used)                                                                                                            \
    Ptr{(c)->k, "pages k", 16, used}, Ptr{(c)->v, "pages v", 16, used}, Ptr{(c)->k_scale, "pages k_scale", 4, (used) && is8((c)->dtype)}, \
        Ptr{(c)->v_scale, "pages v_scale", 4, (used) && is8((c)->dtype)}, Ptr{(c)->table, "table", 4, used}
qb::pg::Pages device_pages(const qwen_kv_pages_t* c) {
    int shift = 0;
    while (1 << shift < c->page_size) shift++;
    return qb::pg::Pages{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, c->table, c->page_stride, c->head_stride, c->n_pages, c->n_seqs, c->max_pages, shift};
}

// ---- norms, rotation, rows to pages ----------------------------------------------
template <int SRC, int D>
int rope_launch(const qb::pg::RopeParams& P, cudaStream_t st) {
    const int blocks = (P.n_rows - 1) / P.tokens + 1;
    if (is8(P.store)) qb::pg::qk_rope_kernel<SRC, D, true><<<blocks, qb::pg::kRopeThreads, 0, st>>>(P);
    else qb::pg::qk_rope_kernel<SRC, D, false><<<blocks, qb::pg::kRopeThreads, 0, st>>>(P);
    CU(cudaGetLastError());
    return QWEN_OK;
}

// ---- prompts -----------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;
// Rows of 64-element boxes in the 128-byte swizzle; rank 2 or 3, strides (bytes) of all but the first dimension.
int encode(CUtensorMap* m, int dtype, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    std::call_once(g_encode_once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    const cuuint32_t es[3] = {1, 1, 1};
    if (!g_encode || g_encode(m, dtype == QWEN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims,
                              strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return fail(QWEN_E_CUDA, "cuTensorMapEncodeTiled failed");
    return QWEN_OK;
}
template <int T, int D>
int prompt_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const qb::pr::Params& P, int grid, int dev, cudaStream_t st) {
    using L = qb::pr::Layout<D>;
    static std::atomic<uint64_t> done{0};
    auto kernel = qb::pr::prompt_kernel<T, D>;
    TRY(smem_limit(kernel, done, dev, L::kSmem));
    kernel<<<grid, qb::pr::kThreads, L::kSmem, st>>>(mq, mk, mv, P);
    CU(cudaGetLastError());
    return QWEN_OK;
}

// ---- attention over pages ------------------------------------------------------------
// A CTA for each item, a cluster of eight for each, or shares of the line of tiles.  A cluster needs one launch, its parts are joined through distributed
// shared memory, but eight CTAs an item leave others idle, and where lengths differ the longest sequence has no more than its eight.  So clusters
// where the items' CTAs all fit at once, for tables of up to 32 tiles, or of 96 where the items' CTAs are more than half of those that fit.  (The
// host knows the tables' width, not the lengths: short sequences in a wide table take the shares' two launches.)
// Measured, clusters / shares, 8 K/V heads of 128, rows in the L2.  bf16 (tiles of 64): 1 sequence of 1000 5.9 / 7.6 us, of 2000 7.4 / 9.5, of 4000
// 10.7 / 11.6, of 8000 17.1 / 14.0; 4 of 4000 13.6 / 15.8, of 6000 18.2 / 20.0, of 16000 49.1 / 51.4, but 4 of which three are half as long: 4000 12.2 /
// 13.1, 6000 16.2 / 15.3, 16000 38.7 / 35.1, and a sixteenth: 4000 11.3 / 12.0, 6000 14.7 / 13.3, 16000 30.8 / 18.5.  e4m3 (tiles of 128): 1 of
// 4000 8.1 / 10.1, of 8000 12.4 / 12.4; 4 of 8000 16.2 / 18.7, of 12000 22.2 / 24.6, three of them half as long 14.1 / 15.1 and 19.5 / 17.8, a
// sixteenth 13.0 / 13.4 and 17.3 / 14.8.
struct PagedPlan : Plan {
    int cluster;   // 0: none
};
int paged_plan(const qwen_kv_pages_t* c, int n_heads, int dev, PagedPlan* p) {
    const int group = n_heads / c->n_kv_heads, keys = qb::pa::tile_keys(c->head_dim * (is8(c->dtype) ? 1 : 2)), capacity = c->max_pages * c->page_size;
    p->rows = group <= 8 ? 8 : 16;
    p->row_blocks = (group + p->rows - 1) / p->rows;
    p->tiles = (capacity + keys - 1) / keys;
    p->blocks = (capacity + 63) / 64;
    p->items = (long long)c->n_seqs * c->n_kv_heads * p->row_blocks;
    p->spare = 7.0f;
    p->cluster = 0;
    p->whole = p->tiles <= 2 && p->items < 1 << 30;
    int nsm = 0, ctas = 0;
    if (!p->whole) {
        TRY(sm_count(dev, &nsm));
        ctas = 2 * nsm;
        const long long all = p->items * qb::pa::kCluster;
        if (all <= ctas && p->tiles >= qb::pa::kCluster && p->tiles <= (2 * all > ctas ? 96 : 32)) p->cluster = qb::pa::kCluster;
        p->whole = p->cluster != 0 || (p->blocks <= p->spare && p->items < 1 << 30) ||
                   (p->blocks <= 16 && p->items < 1 << 30 && (double)p->blocks * std::max(0ll, ctas - p->items) <= (double)p->spare * ctas);
    }
    return plan_shares(p, ctas, c->head_dim);
}
template <int QT, int STORE, int D, int NT>
int paged_launch(const qb::pa::Params& P, const PagedPlan& plan, int dev, cudaStream_t st) {
    using L = qb::pa::Layout<STORE, D, NT>;
    static std::atomic<uint64_t> done{0};
    auto kernel = qb::pa::paged_kernel<QT, STORE, D, NT>;
    TRY(smem_limit(kernel, done, dev, L::kSmem));
    if (plan.cluster) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = plan.cluster;
        at[0].val.clusterDim.y = 1;
        at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3((unsigned)(plan.items * plan.cluster));
        cfg.blockDim = dim3(qb::pa::kThreads);
        cfg.dynamicSmemBytes = L::kSmem;
        cfg.stream = st;
        CU(cudaLaunchKernelEx(&cfg, kernel, P));
        return QWEN_OK;
    }
    kernel<<<plan.shares, qb::pa::kThreads, L::kSmem, st>>>(P);
    CU(cudaGetLastError());
    return join_launch<QT, L::KT, qb::pa::kItemCost, D, L::kRows, false>(P.t, plan, dev, st);
}
template <int QT, int STORE>
int paged_by_shape(int dim, const qb::pa::Params& P, const PagedPlan& plan, int dev, cudaStream_t st) {
    if (dim == 64) return plan.rows == 8 ? paged_launch<QT, STORE, 64, 1>(P, plan, dev, st) : paged_launch<QT, STORE, 64, 2>(P, plan, dev, st);
    return plan.rows == 8 ? paged_launch<QT, STORE, 128, 1>(P, plan, dev, st) : paged_launch<QT, STORE, 128, 2>(P, plan, dev, st);
}

// ---- log probabilities -----------------------------------------------------------------
template <int T>
int logprobs_launch(const qb::lp::Params& P, int n_rows, int nsm, cudaStream_t st) {
    using namespace qb::lp;
    // Blocks for a row: no more in all than the SMs' two places hold, each with a piece a thread at least.  (Twice and four times as many: 64
    // rows of fp32 16.7 us instead of 11.7, 128 rows 21.9 and 31.9 instead of 17.1.)
    const int vec = T == QWEN_FP32 ? 4 : 8;
    int cluster = 1;
    while (cluster < kMaxCluster && (long long)n_rows * cluster * 2 <= 2 * nsm && P.vocab >= cluster * 2 * kThreads * vec) cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)n_rows * cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    CU(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, P));
    return QWEN_OK;
}

}  // namespace

extern "C" int qwen_qk_rope(const void* q, const void* k, const void* v, int dtype, long long ldq, long long ldk, long long ldv, int n_rows,
                            int n_heads, int n_kv_heads, int head_dim, const void* q_gain, const void* k_gain, int gain_dtype, float eps, double base,
                            const int* positions, void* q_out, void* k_out, int out_dtype, long long ldqo, long long ldko,
                            const qwen_kv_pages_t* pages, const int* seqs, void* stream) {
    if (!is_rows(dtype)) return fail(QWEN_E_ARG, "rows must be QWEN_BF16, QWEN_FP16 or QWEN_FP32");
    if (!is_rows(out_dtype)) return fail(QWEN_E_ARG, "out_dtype must be QWEN_BF16, QWEN_FP16 or QWEN_FP32");
    if (n_rows < 1) return fail(QWEN_E_ARG, "n_rows must be positive");
    TRY(check_heads(n_heads, n_kv_heads, head_dim));
    if (n_heads > 1 << 20) return fail(QWEN_E_UNSUPPORTED, "more than 2^20 query heads");
    TRY(check_ld(ldq, n_heads, head_dim, "ldq"));
    TRY(check_ld(ldk, n_kv_heads, head_dim, "ldk"));
    TRY(check_ld(ldqo, n_heads, head_dim, "ldqo"));
    if (k_out) TRY(check_ld(ldko, n_kv_heads, head_dim, "ldko"));
    if ((q_gain != nullptr) != (k_gain != nullptr)) return fail(QWEN_E_ARG, "q_gain and k_gain must both be given or both be NULL");
    if (q_gain && !is_rows(gain_dtype)) return fail(QWEN_E_ARG, "gain_dtype must be QWEN_BF16, QWEN_FP16 or QWEN_FP32");
    if (!(eps >= 0.f && std::isfinite(eps))) return fail(QWEN_E_ARG, "eps must be finite and not negative");
    if (!(base >= 1.0 && std::isfinite(base))) return fail(QWEN_E_ARG, "base must be finite and at least 1");
    static const qwen_kv_pages_t kNone = {};
    const qwen_kv_pages_t* c = pages ? pages : &kNone;
    if (pages) {
        TRY(check_pages(pages));
        TRY(check_ld(ldv, n_kv_heads, head_dim, "ldv"));
        if (pages->n_kv_heads != n_kv_heads || pages->head_dim != head_dim) return fail(QWEN_E_ARG, "the pages' heads are not the rows'");
    }
    int dev = 0, nsm = 0;
    const std::initializer_list<Ptr> ptrs = {{q, "q", 16, true}, {k, "k", 16, true}, {v, "v", 16, pages != nullptr}, {q_gain, "q_gain", 4, q_gain != nullptr},
                                             {k_gain, "k_gain", 4, k_gain != nullptr}, {positions, "positions", 4, true}, {q_out, "q_out", 16, true},
                                             {k_out, "k_out", 16, k_out != nullptr}, QB_PAGES_PTRS(c, pages != nullptr), {seqs, "seqs", 4, pages != nullptr}};
    TRY(check_places(ptrs));
    for (const void* out : {q_out, k_out})
        if (out && (out == q || out == k || (pages && out == v))) return fail(QWEN_E_ARG, "q_out and k_out must not be q, k or v");
    if (q_out == k_out) return fail(QWEN_E_ARG, "q_out must not be k_out");
    TRY(check_ptrs(ptrs, &dev));
    TRY(sm_count(dev, &nsm));
    qb::pg::RopeParams P;
    P.q = (const uint8_t*)q;
    P.k = (const uint8_t*)k;
    P.v = (const uint8_t*)v;
    P.ldq = ldq;
    P.ldk = ldk;
    P.ldv = ldv;
    P.ldqo = ldqo;
    P.ldko = ldko;
    P.q_gain = (const uint8_t*)q_gain;
    P.k_gain = (const uint8_t*)k_gain;
    P.positions = positions;
    P.seqs = seqs;
    P.q_out = (uint8_t*)q_out;
    P.k_out = (uint8_t*)k_out;
    P.pages = pages ? device_pages(pages) : qb::pg::Pages{};
    P.n_rows = n_rows;
    P.n_heads = n_heads;
    P.n_kv_heads = n_kv_heads;
    P.gain_type = gain_dtype;
    P.out_type = out_dtype;
    P.store = pages ? pages->dtype : -1;
    P.eps = eps;
    // base^0 / 2 pi is the largest: 0.16 turns.  Factor by factor, each rounding 2^-64: after 63 of them 2^-58, as far below 2^-53 as
    // the positions' 31 bits need to stay within 2^-22 of a turn at every position.
    const long double step = powl((long double)base, -2.0L / head_dim);
    long double turn = 0x1p63L / 3.14159265358979323846264338327950288L;
    for (int j = 0; j < head_dim / 2; j++, turn *= step) P.turn[j] = (unsigned long long)turn;
    P.tokens = std::min(std::max(n_rows / (4 * nsm), 1), qb::pg::kRopeTokens);   // (four blocks an SM at least)
    const cudaStream_t st = (cudaStream_t)stream;
    const bool wide = head_dim == 128;
    switch (dtype) {
        case QWEN_BF16: return wide ? rope_launch<QWEN_BF16, 128>(P, st) : rope_launch<QWEN_BF16, 64>(P, st);
        case QWEN_FP16: return wide ? rope_launch<QWEN_FP16, 128>(P, st) : rope_launch<QWEN_FP16, 64>(P, st);
        default: return wide ? rope_launch<QWEN_FP32, 128>(P, st) : rope_launch<QWEN_FP32, 64>(P, st);
    }
}

extern "C" int qwen_prompt_attention(const void* q, const void* k, const void* v, void* out, int dtype, long long ldq, long long ldk, long long ldv,
                                     long long ldo, const int* starts, const int* k_starts, int n_seqs, int n_rows, int n_keys, int n_heads,
                                     int n_kv_heads, int head_dim, float scale, void* stream) {
    if (!is16(dtype)) return fail(QWEN_E_ARG, "rows must be QWEN_BF16 or QWEN_FP16");
    if (n_seqs < 1 || n_seqs > 65535) return fail(QWEN_E_ARG, "n_seqs out of [1, 65535]");
    if (n_rows < 1 || n_rows > 1 << 30 || n_keys < 1 || n_keys > 1 << 30) return fail(QWEN_E_ARG, "n_rows and n_keys out of [1, 2^30]");
    TRY(check_heads(n_heads, n_kv_heads, head_dim));
    if (n_heads / n_kv_heads > 128) return fail(QWEN_E_UNSUPPORTED, "more than 128 query heads for each K/V head");
    TRY(check_ld(ldq, n_heads, head_dim, "ldq"));
    TRY(check_ld(ldk, n_kv_heads, head_dim, "ldk"));
    TRY(check_ld(ldv, n_kv_heads, head_dim, "ldv"));
    TRY(check_ld(ldo, n_heads, head_dim, "ldo"));
    TRY(check_scale(scale));
    if (out == q || out == k || out == v) return fail(QWEN_E_ARG, "out must not be q, k or v");
    int dev = 0, nsm = 0;
    TRY(check_ptrs({{q, "q", 16, true}, {k, "k", 16, true}, {v, "v", 16, true}, {out, "out", 16, true}, {starts, "starts", 4, true},
                    {k_starts, "k_starts", 4, k_starts != nullptr}}, &dev));
    TRY(sm_count(dev, &nsm));
    const int group = n_heads / n_kv_heads, tokens = 128 / group;
    CUtensorMap mq, mk, mv;
    {
        const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)n_heads, (cuuint64_t)n_rows}, strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)ldq * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tokens};
        TRY(encode(&mq, dtype, 3, q, dims, strides, box));
    }
    for (int i = 0; i < 2; i++) {
        const cuuint64_t dims[2] = {(cuuint64_t)n_kv_heads * head_dim, (cuuint64_t)n_keys}, strides[1] = {(cuuint64_t)(i ? ldv : ldk) * 2};
        const cuuint32_t box[2] = {64, qb::pr::kKT};
        TRY(encode(i ? &mv : &mk, dtype, 2, i ? v : k, dims, strides, box));
    }
    qb::pr::Params P;
    P.out = (uint8_t*)out;
    P.v = (const uint8_t*)v;
    P.starts = starts;
    P.k_starts = k_starts;
    P.ldv = ldv;
    P.ldo = ldo;
    P.n_seqs = n_seqs;
    P.n_rows = n_rows;
    P.n_keys = n_keys;
    P.n_kv_heads = n_kv_heads;
    P.group = group;
    P.tokens = tokens;
    P.out32 = ((uintptr_t)out | (size_t)ldo * 2) % 32 == 0;
    P.withheld = qwen_internal_withheld();
    P.wait_ns = qwen_internal_wait_ns();
    P.scale_log2 = scale * 1.4426950408889634f;
    P.items = ((long long)(n_rows + 2 * tokens - 1) / (2 * tokens) + n_seqs) * n_kv_heads;
    const int grid = (int)std::min((long long)nsm, P.items);
    const cudaStream_t st = (cudaStream_t)stream;
    if (head_dim == 64) return dtype == QWEN_BF16 ? prompt_launch<QWEN_BF16, 64>(mq, mk, mv, P, grid, dev, st) : prompt_launch<QWEN_FP16, 64>(mq, mk, mv, P, grid, dev, st);
    return dtype == QWEN_BF16 ? prompt_launch<QWEN_BF16, 128>(mq, mk, mv, P, grid, dev, st) : prompt_launch<QWEN_FP16, 128>(mq, mk, mv, P, grid, dev, st);
}

extern "C" int qwen_paged_attention_workspace(const qwen_kv_pages_t* pages, int n_heads, size_t* bytes) {
    if (!bytes) return fail(QWEN_E_ARG, "NULL argument");
    TRY(check_pages(pages));
    TRY(check_heads(n_heads, pages->n_kv_heads, pages->head_dim));
    int dev = 0;
    if ((long long)pages->max_pages * pages->page_size > 128) CU(cudaGetDevice(&dev));   // (shorter ones need none on any device)
    PagedPlan p;
    TRY(paged_plan(pages, n_heads, dev, &p));
    *bytes = p.bytes;
    return QWEN_OK;
}

extern "C" int qwen_paged_attention(const qwen_kv_pages_t* pages, const void* q, void* out, int dtype, long long ldq, long long ldo, int n_heads,
                                    const int* lens, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    TRY(check_pages(pages));
    if (!is16(dtype)) return fail(QWEN_E_ARG, "q and out must be QWEN_BF16 or QWEN_FP16");
    if (is16(pages->dtype) && pages->dtype != dtype) return fail(QWEN_E_ARG, "q and 16-bit pages must have the same type");
    TRY(check_heads(n_heads, pages->n_kv_heads, pages->head_dim));
    TRY(check_ld(ldq, n_heads, pages->head_dim, "ldq"));
    TRY(check_ld(ldo, n_heads, pages->head_dim, "ldo"));
    TRY(check_scale(scale));
    if (q == out) return fail(QWEN_E_ARG, "out must not be q");
    int dev = 0;
    TRY(check_ptrs({QB_PAGES_PTRS(pages, true), {q, "q", 16, true}, {out, "out", 16, true}, {lens, "lens", 4, true}, {workspace, "workspace", 16, workspace != nullptr}}, &dev));
    PagedPlan plan;
    TRY(paged_plan(pages, n_heads, dev, &plan));
    if (plan.bytes && !workspace) return fail(QWEN_E_ARG, "workspace is NULL");
    if (workspace_bytes < plan.bytes) return fail(QWEN_E_ARG, "workspace is smaller than qwen_paged_attention_workspace says");
    qb::pa::Params P;
    P.pages = device_pages(pages);
    P.cluster = plan.cluster;
    P.t = {};
    P.t.cache.capacity = pages->max_pages * pages->page_size;
    P.t.q = (const uint8_t*)q;
    P.t.out = (uint8_t*)out;
    P.t.lens = lens;
    P.t.work = (float*)workspace;
    P.t.ldq = ldq;
    P.t.ldo = ldo;
    P.t.n_seqs = pages->n_seqs;
    P.t.n_kv_heads = pages->n_kv_heads;
    P.t.group = n_heads / pages->n_kv_heads;
    P.t.per_group = 1.0f / (float)P.t.group;
    P.t.n_nodes = 1;
    P.t.whole = plan.whole;
    P.t.row_blocks = plan.row_blocks;
    P.t.beside = plan.beside;
    P.t.groups = plan.shares / plan.beside;
    P.t.by_item = !plan.whole && (long long)P.t.n_seqs * P.t.n_kv_heads * (P.t.row_blocks / P.t.beside) <= P.t.groups;
    P.t.scale_log2 = scale * 1.4426950408889634f;
    P.t.wait_ns = 0;
    P.t.withheld = -1;
    const cudaStream_t st = (cudaStream_t)stream;
    const int dim = pages->head_dim;
    const bool bf = dtype == QWEN_BF16;
    switch (pages->dtype) {
        case QWEN_E4M3: return bf ? paged_by_shape<QWEN_BF16, QWEN_E4M3>(dim, P, plan, dev, st) : paged_by_shape<QWEN_FP16, QWEN_E4M3>(dim, P, plan, dev, st);
        case QWEN_INT8: return bf ? paged_by_shape<QWEN_BF16, QWEN_INT8>(dim, P, plan, dev, st) : paged_by_shape<QWEN_FP16, QWEN_INT8>(dim, P, plan, dev, st);
        default: return bf ? paged_by_shape<QWEN_BF16, QWEN_BF16>(dim, P, plan, dev, st) : paged_by_shape<QWEN_FP16, QWEN_FP16>(dim, P, plan, dev, st);
    }
}

extern "C" int qwen_token_logprobs(const void* logits, int dtype, long long ld, int n_rows, int vocab, const int* tokens, float temperature, int n_top,
                                   float* logprob, float* entropy, int* top_ids, float* top_logprobs, void* stream) {
    if (!is_rows(dtype)) return fail(QWEN_E_ARG, "logits must be QWEN_FP32, QWEN_BF16 or QWEN_FP16");
    if (n_rows < 1 || n_rows > 1 << 24) return fail(QWEN_E_ARG, "n_rows out of [1, 2^24]");
    if (vocab < 1 || vocab > 1 << 30) return fail(QWEN_E_ARG, "vocab out of [1, 2^30]");
    if (ld < vocab || ld > 1ll << 36) return fail(QWEN_E_ARG, "ld must hold a row (up to 2^36)");
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(QWEN_E_ARG, "temperature must be within 1e-6 .. 1e6");
    if (n_top < 0 || n_top > qb::lp::kMaxTop) return fail(QWEN_E_ARG, "n_top out of [0, 64]");
    if ((tokens != nullptr) != (logprob != nullptr)) return fail(QWEN_E_ARG, "tokens and logprob must both be given or both be NULL");
    if (!tokens && !entropy && !n_top) return fail(QWEN_E_ARG, "nothing is asked for");
    int dev = 0, nsm = 0;
    const size_t elem = dtype == QWEN_FP32 ? 4 : 2;
    TRY(check_ptrs({{logits, "logits", elem, true}, {tokens, "tokens", 4, tokens != nullptr}, {logprob, "logprob", 4, logprob != nullptr},
                    {entropy, "entropy", 4, entropy != nullptr}, {top_ids, "top_ids", 4, n_top > 0}, {top_logprobs, "top_logprobs", 4, n_top > 0}}, &dev));
    TRY(sm_count(dev, &nsm));
    qb::lp::Params P;
    P.logits = (const uint8_t*)logits;
    P.ld = ld;
    P.vocab = vocab;
    P.n_top = n_top;
    P.c = (float)(1.4426950408889634 / (double)temperature);
    P.tokens = tokens;
    P.logprob = logprob;
    P.entropy = entropy;
    P.top_logprobs = top_logprobs;
    P.top_ids = top_ids;
    const cudaStream_t st = (cudaStream_t)stream;
    switch (dtype) {
        case QWEN_BF16: return logprobs_launch<QWEN_BF16>(P, n_rows, nsm, st);
        case QWEN_FP16: return logprobs_launch<QWEN_FP16>(P, n_rows, nsm, st);
        default: return logprobs_launch<QWEN_FP32>(P, n_rows, nsm, st);
    }
}
