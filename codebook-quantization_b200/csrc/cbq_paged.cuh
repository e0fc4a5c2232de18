// cbq_paged.cuh -- what the paged-cache kernels share: the device view of a
// cache and a batch, their host checks, and the lookup of a token's sequence.
#pragma once
#include "cbq_common.cuh"

namespace cbq {

// The cache and the batch as the kernels take them (by value).
struct PagedView {
    const void *k, *v;
    int64_t page_stride, head_stride, row_stride;      // elements
    int pages, kv_heads, ps_shift;                     // page_size = 1 << ps_shift
    int seqs, tokens, groups;
    const int32_t *cu, *lens, *table;
    int64_t table_stride;
    int cap;                                           // rows a table row can name
    const int32_t *gs, *plens, *ptable;
    int64_t ptable_stride;
    int pcap;
    uint32_t *status;
};

constexpr int kMaxSeqs = 65536;

// Largest i in [0, n) with a[i] <= x, for a never falling and a[0] <= x: a
// 32-way search by one warp (one load per lane and level).
__device__ __forceinline__ int warp_upper(const int32_t *a, int n, int x) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;                                // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5;
        const int i = lo + (lane + 1) * step;
        const unsigned le = __ballot_sync(0xffffffffu, i < hi && a[i] <= x);
        const int c = __popc(le);
        lo += c * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

}  // namespace cbq

namespace cbq_host {

// Checks what every entry point needs of a cache and a batch and fills the
// device view; CBQ_OK, CBQ_ERR_ARG or CBQ_ERR_UNSUPPORTED.
inline int paged_view(const cbq_paged_cache *c, const cbq_paged_batch *b, int64_t tokens, int64_t q_heads,
                      cbq::PagedView *out) {
    if (!c || !b) return CBQ_ERR_ARG;
    if (c->dtype != CBQ_F32 && c->dtype != CBQ_BF16) return CBQ_ERR_ARG;
    if (c->pages < 0 || c->kv_heads < 1 || tokens < 0 || b->seqs < 0 || b->groups < 0 || b->groups > b->seqs)
        return CBQ_ERR_ARG;
    if (q_heads < 1 || q_heads % c->kv_heads) return CBQ_ERR_ARG;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return CBQ_ERR_UNSUPPORTED;
    int shift = 4;
    while (shift <= 8 && (int64_t(1) << shift) != c->page_size) ++shift;
    if (shift > 8) return CBQ_ERR_UNSUPPORTED;
    if (q_heads / c->kv_heads > 64 || b->seqs > cbq::kMaxSeqs || c->pages > 0x7fffffff || tokens > 0x7fffffff / q_heads)
        return CBQ_ERR_UNSUPPORTED;
    if (b->seqs == 0 || tokens == 0) return CBQ_OK;      // nothing to do: the callers return before a launch
    const int64_t unit = c->dtype == CBQ_BF16 ? 8 : 4;   // elements in 16 bytes
    if (c->row_stride < c->head_dim || c->page_stride < 0 || c->head_stride < 0 || c->row_stride % unit ||
        c->page_stride % unit || c->head_stride % unit)
        return CBQ_ERR_ARG;
    if (c->pages > 0 && (!c->k_dev || !c->v_dev || (reinterpret_cast<uintptr_t>(c->k_dev) & 15) ||
                         (reinterpret_cast<uintptr_t>(c->v_dev) & 15)))
        return CBQ_ERR_ARG;
    // a table without columns (its address may be null) names no rows
    if (!b->kv_lens_dev || (!b->page_table_dev && b->table_width) || b->table_width < 0 || b->table_stride < b->table_width ||
        b->max_kv_len < 0)
        return CBQ_ERR_ARG;
    if ((!b->cu_tokens_dev && tokens != b->seqs)) return CBQ_ERR_ARG;
    if (b->groups && (!b->group_starts_dev || !b->prefix_lens_dev || (!b->prefix_table_dev && b->prefix_width) ||
                      b->prefix_width < 0 || b->prefix_stride < b->prefix_width || b->max_prefix_len < 0))
        return CBQ_ERR_ARG;
    if (b->table_width * c->page_size > 0x7fffff00 || (b->groups && b->prefix_width * c->page_size > 0x7fffff00))
        return CBQ_ERR_UNSUPPORTED;
    cbq::PagedView v{};
    v.k = c->k_dev; v.v = c->v_dev;
    v.page_stride = c->page_stride; v.head_stride = c->head_stride; v.row_stride = c->row_stride;
    v.pages = (int)c->pages; v.kv_heads = (int)c->kv_heads; v.ps_shift = shift;
    v.seqs = (int)b->seqs; v.tokens = (int)tokens; v.groups = (int)b->groups;
    v.cu = b->cu_tokens_dev; v.lens = b->kv_lens_dev; v.table = b->page_table_dev;
    v.table_stride = b->table_stride; v.cap = (int)(b->table_width * c->page_size);
    if (b->groups) {
        v.gs = b->group_starts_dev; v.plens = b->prefix_lens_dev; v.ptable = b->prefix_table_dev;
        v.ptable_stride = b->prefix_stride; v.pcap = (int)(b->prefix_width * c->page_size);
    }
    v.status = b->status_dev;
    *out = v;
    return CBQ_OK;
}

}  // namespace cbq_host
