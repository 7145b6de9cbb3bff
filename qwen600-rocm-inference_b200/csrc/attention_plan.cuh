// attention_plan.cuh — how an attention over a cache is divided among CTAs, and
// the kernel that joins what they leave, launched; for tree_attention.cuh's kernels and
// paged_attention.cuh's.
#pragma once
#include <algorithm>

#include "op_checks.cuh"
#include "tree_attention_tc.cuh"

namespace {

struct Plan {
    int rows, row_blocks, beside, shares;   // shares: CTAs, beside for each share of the line
    int tiles, blocks;                      // of a cache's capacity: the kernel's tiles; blocks of 64 keys (tensor-memory kernel: 128)
    long long items;                        // sequences, K/V heads and blocks of rows
    float spare;
    bool whole, may_be_whole;               // a CTA for each item, no joining
    size_t bytes;
};
// Of a plan that has rows, row_blocks, tiles, items and whole: the shares of the line for `ctas` CTAs, and the workspace.
int plan_shares(Plan* p, int ctas, int head_dim) {
    if (p->whole) {
        p->beside = p->row_blocks;
        p->shares = (int)p->items;
        p->bytes = 0;
        return QWEN_OK;
    }
    // shared out over the blocks of rows that walk side by side
    p->beside = p->row_blocks <= ctas ? p->row_blocks : 1;
    // no more shares than the line can have positions
    const double most = (double)p->items / p->beside * (p->tiles + qb::ta::kTcItemCost);
    p->shares = (int)std::min((double)(ctas / p->beside), most) * p->beside;
    if (most >= 2147483648.0) return fail(QWEN_E_UNSUPPORTED, "too many sequences, heads and positions for one call");
    p->bytes = (size_t)2 * p->shares * p->rows * (head_dim + 2) * sizeof(float);
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

}  // namespace
