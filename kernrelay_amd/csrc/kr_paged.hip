// Attention of new tokens over a paged key/value cache: one token, a tree of
// drafts, or a causal chunk per sequence. See kr_op_attention_paged.
//
// Row i (a new token and a query head) of a sequence with L cached tokens:
//   o = sum_j exp(s q.k_j - m) v_j / sum_j exp(s q.k_j - m), j over the
//   positions it sees: j < L, and new tokens by the causal order or the tree.
#include <cmath>

#include "kr_paged.h"

namespace kr {

namespace {

struct PagedParams {
    const uint16_t *q, *k, *v;
    uint16_t *o;
    const int32_t *table, *lens, *starts;
    const uint64_t *tree;
    int64_t ldq, ldo, ld_table, ld_tree, page_stride, token_stride, head_stride;
    int cap, pages, seqs, rows, max_new, tree_words, HQ, G;
    float scale;
    PageDiv div;
};

// One wave per row: lane j scores key j of each 64, then lanes hold columns.
template <int DT, int D>
__global__ void __launch_bounds__(256) PagedKernel(PagedParams p)
{
    const int lane = int(threadIdx.x) & 63;
    const int64_t item = int64_t(blockIdx.x) * 4 + (int(threadIdx.x) >> 6);
    if (item >= int64_t(p.rows) * p.HQ) return;
    const int r = int(item / p.HQ), h = int(item % p.HQ);
    int lo = 0, hi = p.seqs;  // last sequence that starts at or before r
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.starts[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int first = p.starts[lo];
    if (r < first || r >= p.starts[lo + 1] || r - first >= p.max_new) return;
    const int i = r - first;
    const int len = max(p.lens[lo], 0);
    const int64_t total = min(int64_t(len) + min(p.starts[lo + 1] - first, p.max_new), int64_t(p.cap));
    const int32_t *table = p.table + lo * p.ld_table;
    const uint16_t *q = p.q + int64_t(r) * p.ldq + int64_t(h) * D;
    const int64_t head = int64_t(h / p.G) * p.head_stride;
    float m = -INFINITY, l = 0.0f, acc[D / 64] = {};
    for (int64_t k0 = 0; k0 < total; k0 += 64) {
        const int64_t pos = k0 + lane;
        int64_t row = -1;
        if (pos < total) {
            const int pg = PageOf(p.div, int(pos));
            const int id = table[pg];
            const int64_t j = pos - len;
            bool sees = id >= 0 && id < p.pages;
            if (j >= 0) {
                if (p.tree == nullptr) sees = sees && j <= i;
                else sees = sees && j < 64 * int64_t(p.tree_words) &&
                            ((p.tree[r * p.ld_tree + j / 64] >> (j % 64)) & 1) != 0;
            }
            if (sees) row = id * p.page_stride + int64_t(int(pos) - pg * p.div.size) * p.token_stride + head;
        }
        float s = -INFINITY;
        if (row >= 0) {
            s = 0.0f;
            for (int c = 0; c < D; c += 8) {
                const U16x8 a = LoadU16x8(q + c), b = LoadU16x8(p.k + row + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) s += Elem<DT>::Load(a.v[e]) * Elem<DT>::Load(b.v[e]);
            }
            s *= p.scale;
        }
        const float mn = fmaxf(m, WaveMax(s));
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float alpha = FastExp(m - ms);
        const float w = row >= 0 ? FastExp(s - ms) : 0.0f;
        m = mn;
        l = l * alpha + WaveSum(w);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] *= alpha;
        for (int j = 0; j < 64; ++j) {
            const int64_t rj = __shfl(row, j, 64);
            const float wj = __shfl(w, j, 64);
            if (rj < 0) continue;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) acc[c] += wj * Elem<DT>::Load(p.v[rj + c * 64 + lane]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
        p.o[int64_t(r) * p.ldo + int64_t(h) * D + c * 64 + lane] = Elem<DT>::Store(acc[c] * inv);
}

}  // namespace

void PagedAttnNeeds(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes, int *counters)
{
    const kr_cache c = CheckCache(cache, "attention_paged");
    CheckSeqs(seqs, "attention_paged");
    if (HQ < 1 || HQ % c.heads != 0) 
        throw std::runtime_error("attention_paged: HQ must be a multiple of the cache's heads");
    *ws_bytes = 0;
    *counters = 0;
}

void PagedAttnLaunch(const PagedAttnDesc &d, hipStream_t stream)
{
    const char *who = "attention_paged";
    const kr_cache c = CheckCache(d.cache, who);
    CheckSeqs(d.seqs, who);
    const kr_seqs &s = *d.seqs;
    const auto refuse = [](const char *what) { throw std::runtime_error(std::string("attention_paged: ") + what); };
    if (d.HQ < 1 || d.HQ % c.heads != 0) refuse("HQ must be a multiple of the cache's heads");
    if (d.layer < 0 || d.layer >= c.layers) refuse("no such layer");
    if (!(d.scale > 0.0f) || std::isinf(d.scale)) refuse("scale must be positive");
    if (d.rows < 0) refuse("rows must not be negative");
    if (d.rows == 0 || s.seqs == 0 || s.max_new == 0) return;
    if (d.q == nullptr || d.out == nullptr) refuse("q or out is missing");
    if (((reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.out)) & 15) != 0)
        refuse("pointers must be 16-byte aligned");
    PagedParams p{};
    p.ldq = d.ldq > 0 ? d.ldq : int64_t(d.HQ) * c.head_dim;
    p.ldo = d.ldo > 0 ? d.ldo : int64_t(d.HQ) * c.head_dim;
    if (((p.ldq | p.ldo) % 8) != 0) refuse("row strides must be multiples of 8");
    const int64_t cap = int64_t(s.table_pages) * c.page_size;
    if (cap >= (int64_t(1) << 31) - 256) refuse("the page table spans too many tokens");
    p.q = static_cast<const uint16_t *>(d.q);
    p.k = static_cast<const uint16_t *>(c.k) + d.layer * c.layer_stride;
    p.v = static_cast<const uint16_t *>(c.v) + d.layer * c.layer_stride;
    p.o = static_cast<uint16_t *>(d.out);
    p.table = s.table;
    p.lens = s.lens;
    p.starts = s.starts;
    p.tree = s.tree;
    p.ld_table = s.ld_table;
    p.ld_tree = s.ld_tree;
    p.page_stride = c.page_stride;
    p.token_stride = c.token_stride;
    p.head_stride = c.head_stride;
    p.cap = int(cap);
    p.pages = c.pages;
    p.seqs = s.seqs;
    p.rows = d.rows;
    p.max_new = s.max_new;
    p.tree_words = s.tree_words;
    p.HQ = d.HQ;
    p.G = d.HQ / c.heads;
    p.scale = d.scale;
    p.div = MakePageDiv(c.page_size);
    const int64_t wg = (int64_t(d.rows) * d.HQ + 3) / 4;
    if (wg >= (int64_t(1) << 31)) refuse("too many rows for one launch");
    const dim3 grid{unsigned(wg)};
    const bool bf = c.dtype == kBF16;
    if (c.head_dim == 128) {
        if (bf) hipLaunchKernelGGL((PagedKernel<kBF16, 128>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((PagedKernel<kF16, 128>), grid, dim3(256), 0, stream, p);
    } else {
        if (bf) hipLaunchKernelGGL((PagedKernel<kBF16, 64>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((PagedKernel<kF16, 64>), grid, dim3(256), 0, stream, p);
    }
    Check(hipGetLastError(), "attention_paged launch");
}

}  // namespace kr
