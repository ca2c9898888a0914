// Writing and moving a paged key/value cache: q/k norm + RoPE in one pass (to
// plain tensors, or k and v to their cache slots), page copies, and the
// compaction of accepted drafts. No counterpart in the reference, whose path
// ends with the prompt's last row; the first stands for its EmitQkNorm and
// Rope (exec/qwen_main.cpp:1346-1357, 567-582).
#include <algorithm>
#include <cmath>
#include <vector>

#include "kr_paged.h"

namespace kr {

namespace {

[[noreturn]] void Refuse(const char *who, const char *what)
{
    throw std::runtime_error(std::string(who) + ": " + what);
}

bool Misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

bool Overlap(const RowSpan &a, const RowSpan &b)
{
    if (a.rows < 1 || b.rows < 1) return false;
    const int64_t pa = int64_t(reinterpret_cast<uintptr_t>(a.p) / 2), pb = int64_t(reinterpret_cast<uintptr_t>(b.p) / 2);
    if (pa + (a.rows - 1) * a.ld + a.width <= pb || pb + (b.rows - 1) * b.ld + b.width <= pa) return false;
    if (a.ld == b.ld && a.ld > 0) {
        // row i of a and i + t of b: -b.width < d + t ld < a.width
        const int64_t d = pb - pa, ld = a.ld;
        const auto floor_div = [](int64_t n, int64_t by) { return n / by - (n % by < 0); };
        const int64_t lo = std::max(-floor_div(d + b.width - 1, ld), 1 - a.rows);
        const int64_t hi = std::min(floor_div(a.width - 1 - d, ld), b.rows - 1);
        return lo <= hi;
    }
    for (int64_t i = 0, j = 0; i < a.rows && j < b.rows;) {
        const int64_t x = pa + i * a.ld, y = pb + j * b.ld;
        if (x + a.width <= y) ++i;
        else if (y + b.width <= x) ++j;
        else return true;
    }
    return false;
}

RowSpan LayerSpan(const kr_cache &c, const void *base, int layer)
{
    RowSpan s;
    s.p = static_cast<const uint16_t *>(base) + layer * c.layer_stride;
    s.rows = 1;
    s.width = (c.pages - 1) * c.page_stride + (c.page_size - 1) * c.token_stride + (c.heads - 1) * c.head_stride +
              c.head_dim;
    return s;
}

bool MeetsSeqs(const MemSpan &out, const kr_seqs &s, int64_t rows)
{
    return Meets(out, RowsSpan(s.table, s.seqs, s.ld_table, s.table_pages, 4)) ||
           Meets(out, RowsSpan(s.lens, 1, 0, s.seqs, 4)) || Meets(out, RowsSpan(s.starts, 1, 0, int64_t(s.seqs) + 1, 4)) ||
           (s.tree != nullptr && Meets(out, RowsSpan(s.tree, rows, s.ld_tree, s.tree_words, 8)));
}

kr_cache CheckCache(const kr_cache *c, const char *who)
{
    if (c == nullptr || c->k == nullptr || c->v == nullptr) Refuse(who, "needs a cache");
    kr_cache r = *c;
    if (r.dtype != kBF16 && r.dtype != kF16) Refuse(who, "the cache must be bf16 or f16");
    if (r.head_dim != 64 && r.head_dim != 128) Refuse(who, "head_dim must be 64 or 128");
    if (r.layers < 1 || r.pages < 1 || r.page_size < 1 || r.heads < 1) Refuse(who, "the cache is empty");
    if (Misaligned(r.k) || Misaligned(r.v)) Refuse(who, "cache pointers must be 16-byte aligned");
    if (r.layers == 1) r.layer_stride = 0;
    if (r.pages == 1) r.page_stride = 0;
    if (r.page_size == 1) r.token_stride = 0;
    if (r.heads == 1) r.head_stride = 0;
    const int64_t lim = int64_t(1) << 31;
    const auto bad = [&](int n, int64_t s) { return n > 1 && (s < r.head_dim || s % 8 != 0); };
    if (bad(r.layers, r.layer_stride) || bad(r.pages, r.page_stride) || bad(r.page_size, r.token_stride) ||
        bad(r.heads, r.head_stride))
        Refuse(who, "cache strides must be multiples of 8 and at least head_dim");
    if (r.page_stride >= lim || r.token_stride >= lim || r.head_stride >= lim)
        Refuse(who, "a cache stride is too large");
    return r;
}

void CheckSeqs(const kr_seqs *s, const char *who)
{
    // (arrays of no sequence may have no address)
    if (s == nullptr || (s->seqs > 0 && (s->table == nullptr || s->lens == nullptr || s->starts == nullptr)))
        Refuse(who, "needs a page table, lengths and starts");
    if (s->seqs < 0 || s->max_new < 0 || s->table_pages < 1) Refuse(who, "a negative or empty size");
    if (s->seqs > 1 && s->ld_table < s->table_pages) Refuse(who, "page table rows overlap");
    if (s->tree != nullptr) {
        if (s->tree_words < 1 || s->ld_tree < s->tree_words) Refuse(who, "tree rows overlap");
        if (int64_t(s->max_new) > 64 * int64_t(s->tree_words)) Refuse(who, "the tree has too few words for max_new");
    }
}

// ------------------------------------------------------------ q/k norm + RoPE
// Row (token r, head h), x of D values, at position p:
//   n = x g / sqrt(mean(x^2) + eps)  (or x),
//   y[i] = n[i] c[i] - n[i+D/2] s[i],  y[i+D/2] = n[i+D/2] c[i+D/2] + n[i] s[i+D/2].
// Bound by HBM: 4 D bytes a row (read and written once) against a few
// operations a value, so a row never leaves its lanes: D/16 lanes hold a row,
// each one 16-byte chunk of the first half and the chunk D/2 further on, its
// partner in the rotation. The sum of squares is the lane's own two chunks,
// then a butterfly over the row's lanes: the order of the standalone norm
// (kr_rowops.hip: 16 lanes of one chunk, partners 8 apart first), so `chain`
// gives the bits of the separate launches. Rows of q, k and (for the cache) v
// follow each other in one flat index: every lane has work whatever the head
// counts. The sums and the rotation are fp32; without `chain` the only
// rounding is the store. Measured: 4096 tokens of 32 + 8 heads of 128, 86 MB in
// 17.2 us (5.0 TB/s, what a large copy reaches), with `chain` 19.2 (the four
// separate launches: 37.2); 48 tokens of 28 + 2 x 4 heads 3.4 us.
namespace {

struct QkRopeParams {
    const uint16_t *q, *k, *v;
    uint16_t *qo, *ko;           // ko: k rows, or the cache's k
    uint16_t *vo;                // the cache's v
    const uint16_t *gq, *gk;
    const void *cos_t, *sin_t;
    const int64_t *positions, *slots;
    int64_t ldq, ldk, ldv, ldqo, ldko;
    int64_t page_stride, token_stride, head_stride, npos, nslots;
    int page_size, HQ, HKV, heads;  // heads: all of a token's rows
    int total;                      // tokens * heads
    float eps;
};

// The fp32 result itself, before it is rounded on: v_fma_mixlo_f16 would round
// a product or a fused sum to f16 at once, and a last bit now and then would
// not be the separate kernels'.
template <bool CHAIN>
__device__ __forceinline__ float InF32(float f)
{
    if constexpr (CHAIN) asm("" : "+v"(f));
    return f;
}

template <typename T>
__device__ __forceinline__ void LoadTable(const void *t, int64_t at, float (&o)[8])
{
    if constexpr (sizeof(T) == 4) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(t) + at);
        const float4 a = p[0], b = p[1];
        o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w;
        o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
    }
}

template <int DT, int D, bool CACHE, bool T32, bool CHAIN>
__global__ void __launch_bounds__(256) QkRopeKernel(QkRopeParams p)
{
    constexpr int LPR = D / 16;  // lanes per row
    const int i = (int(blockIdx.x) * 256 + int(threadIdx.x)) / LPR;
    const int c = int(threadIdx.x) % LPR;
    if (i >= p.total) return;    // a row's lanes leave together
    const int r = i / p.heads;
    const int h = i - r * p.heads;
    const bool is_q = h < p.HQ, is_v = CACHE && h >= p.HQ + p.HKV;
    const uint16_t *src;
    uint16_t *dst;
    if (is_q) {
        src = p.q + int64_t(r) * p.ldq + int64_t(h) * D;
        dst = p.qo + int64_t(r) * p.ldqo + int64_t(h) * D;
    } else {
        const int hk = is_v ? h - p.HQ - p.HKV : h - p.HQ;
        src = (is_v ? p.v + int64_t(r) * p.ldv : p.k + int64_t(r) * p.ldk) + int64_t(hk) * D;
        if constexpr (CACHE) {
            const int64_t slot = p.slots[r];
            if (slot < 0 || slot >= p.nslots) return;
            const int64_t page = slot / p.page_size;
            dst = (is_v ? p.vo : p.ko) + page * p.page_stride + (slot - page * p.page_size) * p.token_stride +
                  int64_t(hk) * p.head_stride;
        } else {
            dst = p.ko + int64_t(r) * p.ldko + int64_t(hk) * D;
        }
    }
    const int i0 = c * 8, i1 = i0 + D / 2;
    U16x8 a = LoadU16x8(src + i0), b = LoadU16x8(src + i1);
    if (!is_v) {
        const int64_t pos = p.positions != nullptr ? p.positions[r] : r;
        const bool there = pos >= 0 && pos < p.npos;
        const int64_t at = (there ? pos : 0) * D;
        float ca[8], cb[8], sa[8], sb[8], x1[8], x2[8];
        if constexpr (T32) {
            LoadTable<float>(p.cos_t, at + i0, ca);
            LoadTable<float>(p.cos_t, at + i1, cb);
            LoadTable<float>(p.sin_t, at + i0, sa);
            LoadTable<float>(p.sin_t, at + i1, sb);
        } else {
            const uint16_t *ct = static_cast<const uint16_t *>(p.cos_t), *st = static_cast<const uint16_t *>(p.sin_t);
            const U16x8 c0 = LoadU16x8(ct + at + i0), c1 = LoadU16x8(ct + at + i1);
            const U16x8 s0 = LoadU16x8(st + at + i0), s1 = LoadU16x8(st + at + i1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ca[e] = Elem<DT>::Load(c0.v[e]);
                cb[e] = Elem<DT>::Load(c1.v[e]);
                sa[e] = Elem<DT>::Load(s0.v[e]);
                sb[e] = Elem<DT>::Load(s1.v[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x1[e] = Elem<DT>::Load(a.v[e]);
            x2[e] = Elem<DT>::Load(b.v[e]);
        }
        const uint16_t *g = is_q ? p.gq : p.gk;
        if (g != nullptr) {
            const U16x8 g1 = LoadU16x8(g + i0), g2 = LoadU16x8(g + i1);
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s1 += x1[e] * x1[e];
                s2 += x2[e] * x2[e];
            }
            float ss = s1 + s2;
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const float rstd = 1.0f / sqrtf(ss / float(D) + p.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (CHAIN) {
                    x1[e] = RoundTo<DT>(InF32<true>(Elem<DT>::Load(g1.v[e]) * RoundTo<DT>(InF32<true>(x1[e] * rstd))));
                    x2[e] = RoundTo<DT>(InF32<true>(Elem<DT>::Load(g2.v[e]) * RoundTo<DT>(InF32<true>(x2[e] * rstd))));
                } else {
                    x1[e] = Elem<DT>::Load(g1.v[e]) * (x1[e] * rstd);
                    x2[e] = Elem<DT>::Load(g2.v[e]) * (x2[e] * rstd);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a.v[e] = there ? Elem<DT>::Store(InF32<CHAIN>(RopeFirst(x1[e], x2[e], ca[e], sa[e]))) : uint16_t(0);
            b.v[e] = there ? Elem<DT>::Store(InF32<CHAIN>(RopeSecond(x2[e], x1[e], cb[e], sb[e]))) : uint16_t(0);
        }
    }
    StoreU16x8(dst + i0, a);
    StoreU16x8(dst + i1, b);
}

template <int DT, int D, bool CACHE>
void QkRopeGo(const QkRopeParams &p, bool t32, bool chain, hipStream_t stream)
{
    const int64_t threads = int64_t(p.total) * (D / 16);
    const dim3 grid(unsigned((threads + 255) / 256));
    if (t32) {
        if (chain) hipLaunchKernelGGL((QkRopeKernel<DT, D, CACHE, true, true>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((QkRopeKernel<DT, D, CACHE, true, false>), grid, dim3(256), 0, stream, p);
    } else {
        if (chain) hipLaunchKernelGGL((QkRopeKernel<DT, D, CACHE, false, true>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((QkRopeKernel<DT, D, CACHE, false, false>), grid, dim3(256), 0, stream, p);
    }
}

}  // namespace

void QkRopeLaunch(const QkRopeDesc &d, hipStream_t stream)
{
    const char *who = d.cache != nullptr ? "qk_norm_rope_cache" : "qk_norm_rope";
    if (d.rows < 0) Refuse(who, "rows must not be negative");
    if (d.HQ < 1 || d.HKV < 1) Refuse(who, "needs at least one head of each kind");
    if (d.dtype != kBF16 && d.dtype != kF16) Refuse(who, "dtype must be bf16 or f16");
    if (d.D != 64 && d.D != 128 && d.D != 256) Refuse(who, "head_dim must be 64, 128 or 256");
    if (d.rope.cos_t == nullptr || d.rope.sin_t == nullptr || d.rope.positions < 1)
        Refuse(who, "needs rotation tables");
    if ((d.rope.q_gamma == nullptr) != (d.rope.k_gamma == nullptr)) Refuse(who, "one of the two gains is missing");
    if (d.rope.table_dtype != kF32 && d.rope.table_dtype != d.dtype)
        Refuse(who, "the tables must be fp32 or of the activations' type");
    if (d.rope.q_gamma != nullptr && !(d.rope.eps >= 0.0f)) Refuse(who, "eps must not be negative");
    if (d.rows == 0) return;
    QkRopeParams p{};
    p.HQ = d.HQ;
    p.HKV = d.HKV;
    p.heads = d.HQ + d.HKV;
    p.q = static_cast<const uint16_t *>(d.q);
    p.k = static_cast<const uint16_t *>(d.k);
    p.qo = static_cast<uint16_t *>(d.q_out);
    p.ko = static_cast<uint16_t *>(d.k_out);
    p.gq = static_cast<const uint16_t *>(d.rope.q_gamma);
    p.gk = static_cast<const uint16_t *>(d.rope.k_gamma);
    p.cos_t = d.rope.cos_t;
    p.sin_t = d.rope.sin_t;
    p.npos = d.rope.positions;
    p.eps = d.rope.eps;
    p.positions = d.positions;
    p.ldq = d.ldq > 0 ? d.ldq : int64_t(d.HQ) * d.D;
    p.ldk = d.ldk > 0 ? d.ldk : int64_t(d.HKV) * d.D;
    p.ldqo = d.ldqo > 0 ? d.ldqo : int64_t(d.HQ) * d.D;
    p.ldko = d.ldko > 0 ? d.ldko : int64_t(d.HKV) * d.D;
    if (d.cache != nullptr) {
        const kr_cache c = CheckCache(d.cache, who);
        if (d.layer < 0 || d.layer >= c.layers) Refuse(who, "no such layer");
        if (d.slots == nullptr || d.v == nullptr) Refuse(who, "needs slots and v");
        p.v = static_cast<const uint16_t *>(d.v);
        p.ldv = d.ldv > 0 ? d.ldv : int64_t(d.HKV) * d.D;
        p.ko = static_cast<uint16_t *>(c.k) + d.layer * c.layer_stride;
        p.vo = static_cast<uint16_t *>(c.v) + d.layer * c.layer_stride;
        p.page_stride = c.page_stride;
        p.token_stride = c.token_stride;
        p.head_stride = c.head_stride;
        p.page_size = c.page_size;
        p.nslots = int64_t(c.pages) * c.page_size;
        p.slots = d.slots;
        p.heads += d.HKV;
    }
    if (p.q == nullptr || p.k == nullptr || p.qo == nullptr || p.ko == nullptr) Refuse(who, "a tensor is missing");
    for (const void *x : {d.q, d.k, d.v, static_cast<const void *>(d.q_out), static_cast<const void *>(d.k_out),
                          d.rope.cos_t, d.rope.sin_t, d.rope.q_gamma, d.rope.k_gamma})
        if (Misaligned(x)) Refuse(who, "pointers must be 16-byte aligned");
    if (((p.ldq | p.ldk | p.ldv | p.ldqo | p.ldko) % 8) != 0) Refuse(who, "row strides must be multiples of 8");
    const int64_t total = int64_t(d.rows) * p.heads;
    if (total * (d.D / 16) > (int64_t(1) << 31) - 256) Refuse(who, "too many rows for one launch");
    // an output is its own input or no input at all
    const RowSpan q{d.q, p.ldq, d.rows, int64_t(d.HQ) * d.D}, k{d.k, p.ldk, d.rows, int64_t(d.HKV) * d.D};
    const RowSpan qo{d.q_out, p.ldqo, d.rows, q.width}, ko{d.k_out, p.ldko, d.rows, k.width};
    const auto same = [&](const RowSpan &a, const RowSpan &b) { return a.p == b.p && (d.rows == 1 || a.ld == b.ld); };
    if ((Overlap(qo, q) && !same(qo, q)) || Overlap(qo, k)) Refuse(who, "q_out overlaps an input");
    if (d.cache != nullptr) {
        if (Overlap(qo, RowSpan{d.v, p.ldv, d.rows, k.width})) Refuse(who, "q_out overlaps an input");
        const kr_cache c = CheckCache(d.cache, who);
        if (Overlap(qo, LayerSpan(c, c.k, d.layer)) || Overlap(qo, LayerSpan(c, c.v, d.layer)))
            Refuse(who, "q_out overlaps the cache");
    } else if ((Overlap(ko, k) && !same(ko, k)) || Overlap(ko, q) || Overlap(ko, qo)) {
        Refuse(who, "k_out overlaps an input or q_out");
    }
    p.total = int(total);
    const bool t32 = d.rope.table_dtype == kF32, chain = d.rope.chain != 0, bf = d.dtype == kBF16;
    const auto go = [&](auto bf16, auto f16) { bf ? bf16(p, t32, chain, stream) : f16(p, t32, chain, stream); };
    if (d.cache != nullptr) {
        if (d.D == 64) go(QkRopeGo<kBF16, 64, true>, QkRopeGo<kF16, 64, true>);
        else go(QkRopeGo<kBF16, 128, true>, QkRopeGo<kF16, 128, true>);
    } else if (d.D == 64) {
        go(QkRopeGo<kBF16, 64, false>, QkRopeGo<kF16, 64, false>);
    } else if (d.D == 128) {
        go(QkRopeGo<kBF16, 128, false>, QkRopeGo<kF16, 128, false>);
    } else {
        go(QkRopeGo<kBF16, 256, false>, QkRopeGo<kF16, 256, false>);
    }
    Check(hipGetLastError(), "qk_norm_rope launch");
}

// ---------------------------------------------------------------- page copies
// Bound by HBM: every byte of a page read and written once. A workgroup moves
// 16 KB of one page of one layer's k or v, each lane four 16-byte chunks in
// flight. The pairs travel with the launch, so nothing is copied to the
// device first and the host has seen every id. A page is (outer, mid, run): a
// run of contiguous values, merged as far as the strides allow (both usual
// layouts are one run). Measured: 239 MB in 48.0 us (5.0 TB/s), 14 MB in 3.9.
namespace {

constexpr int kCopyPairs = 384;  // of one launch: 3 KB of kernel arguments
constexpr int kCopyUnroll = 4;

struct CopyParams {
    uint16_t *k, *v;
    int64_t layer_stride, page_stride, outer_stride, mid_stride;
    int outer, mid, run8;  // run length in 16-byte chunks
    int chunks;            // of a page: outer * mid * run8
    int segs;              // workgroups per page
    int src[kCopyPairs], dst[kCopyPairs];
};

__device__ __forceinline__ int64_t PageChunk(const CopyParams &p, int c)
{
    if (p.outer == 1 && p.mid == 1) return int64_t(c) * 8;
    const int m = c / p.run8, o = m / p.mid;
    return o * p.outer_stride + int64_t(m - o * p.mid) * p.mid_stride + int64_t(c - m * p.run8) * 8;
}

__global__ void __launch_bounds__(256) CopyPagesKernel(CopyParams p)
{
    const int seg = int(blockIdx.x) % p.segs, pair = int(blockIdx.x) / p.segs;
    const int layer = int(blockIdx.y) >> 1;
    uint16_t *base = ((blockIdx.y & 1) != 0 ? p.v : p.k) + layer * p.layer_stride;
    const uint16_t *src = base + int64_t(p.src[pair]) * p.page_stride;
    uint16_t *dst = base + int64_t(p.dst[pair]) * p.page_stride;
    const int c0 = seg * 256 * kCopyUnroll + int(threadIdx.x);
    // chunks past the page's end repeat its last one: every load goes out
    // before the first store, with no branch between them
    typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
    int64_t at[kCopyUnroll];
    U32x4 x[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) at[u] = PageChunk(p, min(c0 + u * 256, p.chunks - 1));
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) x[u] = *reinterpret_cast<const U32x4 *>(src + at[u]);
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (c0 + u * 256 < p.chunks) *reinterpret_cast<U32x4 *>(dst + at[u]) = x[u];
}

}  // namespace

void CopyPagesLaunch(const kr_cache *cache, const int32_t *src, const int32_t *dst, int n, hipStream_t stream)
{
    const char *who = "cache_copy_pages";
    const kr_cache c = CheckCache(cache, who);
    if (n < 0) Refuse(who, "a negative number of pages");
    if (n == 0) return;
    if (src == nullptr || dst == nullptr) Refuse(who, "needs the pages' ids");
    std::vector<int32_t> to(dst, dst + n);
    for (int i = 0; i < n; ++i)
        if (src[i] < 0 || src[i] >= c.pages || dst[i] < 0 || dst[i] >= c.pages) Refuse(who, "no such page");
    std::sort(to.begin(), to.end());
    if (std::adjacent_find(to.begin(), to.end()) != to.end()) Refuse(who, "a page is written twice");
    for (int i = 0; i < n; ++i)
        if (std::binary_search(to.begin(), to.end(), src[i])) Refuse(who, "a page is both read and written");
    if (c.layers > 32767) Refuse(who, "too many layers");
    CopyParams p;
    p.k = static_cast<uint16_t *>(c.k);
    p.v = static_cast<uint16_t *>(c.v);
    p.layer_stride = c.layer_stride;
    p.page_stride = c.page_stride;
    // (count, stride) of tokens and heads, larger stride first; merge from the inside
    p.outer = c.page_size, p.outer_stride = c.token_stride;
    p.mid = c.heads, p.mid_stride = c.head_stride;
    if (p.outer == 1 || (p.mid > 1 && p.outer_stride < p.mid_stride)) {
        std::swap(p.outer, p.mid);
        std::swap(p.outer_stride, p.mid_stride);
    }
    int64_t run = c.head_dim;
    if (p.mid == 1 || p.mid_stride == run) {
        run *= p.mid;
        p.mid = 1;
        if (p.outer == 1 || p.outer_stride == run) {
            run *= p.outer;
            p.outer = 1;
        }
    }
    const int64_t chunks = int64_t(c.page_size) * c.heads * c.head_dim / 8;
    if (chunks >= (int64_t(1) << 30)) Refuse(who, "a page is too large");
    p.run8 = int(run / 8);
    p.chunks = int(chunks);
    p.segs = (p.chunks + 256 * kCopyUnroll - 1) / (256 * kCopyUnroll);
    for (int at = 0; at < n; at += kCopyPairs) {
        const int m = std::min(kCopyPairs, n - at);
        if (int64_t(m) * p.segs >= kMaxGrid) Refuse(who, "pages are too large");
        std::copy(src + at, src + at + m, p.src);
        std::copy(dst + at, dst + at + m, p.dst);
        std::fill(p.src + m, p.src + kCopyPairs, 0);
        std::fill(p.dst + m, p.dst + kCopyPairs, 0);
        hipLaunchKernelGGL(CopyPagesKernel, dim3(unsigned(m) * unsigned(p.segs), unsigned(2 * c.layers)), dim3(256), 0,
                           stream, p);
        Check(hipGetLastError(), "cache_copy_pages launch");
    }
}

// ----------------------------------------------------------------- compaction
// Bound by latency: a few rows of each layer move, and where they are takes a
// chain of loads (length, path, page ids). A workgroup takes LPR 16-byte
// chunks of every row of one sequence, in PL of the layers' k and v: the chain
// once, then PL planes in flight. It holds all of a plane in registers before
// it writes the first row (a row's new place may be another's old one): NS
// sweeps of 256 / LPR rows. Columns and planes are independent. 32 paths of up
// to 9 drafts, 28 layers of 4 heads: PL 1 9.6 us, 4 6.1 us.
namespace {

struct CompactParams {
    uint16_t *k, *v;
    int64_t layer_stride, page_stride, token_stride, head_stride;
    const int32_t *table, *lens, *path, *path_lens;
    int64_t ld_table, ld_path, cap;  // cap: table_pages * page_size
    int pages, heads, dch, width, slices, planes;
    PageDiv div;
};

template <int LPR, int NS, int PL>
__global__ void __launch_bounds__(256) CompactKernel(CompactParams p)
{
    constexpr int RPS = 256 / LPR;
    const int b = int(blockIdx.x) / p.slices;
    const int ch = (int(blockIdx.x) - b * p.slices) * LPR + int(threadIdx.x) % LPR;
    const int n = min(max(p.path_lens[b], 0), p.width);
    const int len = max(p.lens[b], 0);
    const int head = ch / p.dch;
    const int64_t col = int64_t(head) * p.head_stride + (ch - head * p.dch) * 8;
    const int32_t *table = p.table + b * p.ld_table;
    // element offset of the row at position pos; -1: not there
    const auto row = [&](int64_t pos) -> int64_t {
        if (pos >= p.cap) return -1;
        const int pg = PageOf(p.div, int(pos));
        const int id = table[pg];
        if (id < 0 || id >= p.pages) return -1;
        return id * p.page_stride + int64_t(int(pos) - pg * p.div.size) * p.token_stride + col;
    };
    const int plane0 = int(blockIdx.y) * PL;  // layer plane / 2, its k or v
    const auto base = [&](int i) {
        const int plane = min(plane0 + i, p.planes - 1);
        return ((plane & 1) != 0 ? p.v : p.k) + int64_t(plane >> 1) * p.layer_stride;
    };
    uint4 x[NS][PL];
    int64_t to[NS];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
        const int i = int(threadIdx.x) / LPR + u * RPS;
        const bool in = i < n && head < p.heads;
        const int from = in ? p.path[b * p.ld_path + i] : -1;
        const bool moves = from >= 0 && from != i;
        const int64_t src = moves ? row(int64_t(len) + from) : -1;
        to[u] = src >= 0 ? row(int64_t(len) + i) : -1;
#pragma unroll
        for (int q = 0; q < PL; ++q) {
            x[u][q] = make_uint4(0, 0, 0, 0);
            if (to[u] >= 0) x[u][q] = *reinterpret_cast<const uint4 *>(base(q) + src);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's rows are in registers
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int q = 0; q < PL; ++q)
            if (to[u] >= 0 && plane0 + q < p.planes) *reinterpret_cast<uint4 *>(base(q) + to[u]) = x[u][q];
}

}  // namespace

void CompactLaunch(const kr_cache *cache, const kr_seqs *s, const int32_t *path, int64_t ld_path, int width,
                   const int32_t *path_lens, hipStream_t stream)
{
    const char *who = "cache_compact";
    const kr_cache c = CheckCache(cache, who);
    CheckSeqs(s, who);
    if (width < 0 || width > 256) Refuse(who, "a path holds at most 256 drafts");
    if (s->seqs == 0 || width == 0) return;
    if (path == nullptr || path_lens == nullptr) Refuse(who, "needs the paths and their lengths");
    if (s->seqs > 1 && ld_path < width) Refuse(who, "path rows overlap");
    if (c.layers > 32767) Refuse(who, "too many layers");
    CompactParams p{};
    p.k = static_cast<uint16_t *>(c.k);
    p.v = static_cast<uint16_t *>(c.v);
    p.layer_stride = c.layer_stride;
    p.page_stride = c.page_stride;
    p.token_stride = c.token_stride;
    p.head_stride = c.head_stride;
    p.table = s->table;
    p.lens = s->lens;
    p.path = path;
    p.path_lens = path_lens;
    p.ld_table = s->ld_table;
    p.ld_path = ld_path;
    p.cap = int64_t(s->table_pages) * c.page_size;
    if (p.cap >= (int64_t(1) << 31) - 256) Refuse(who, "the page table spans too many tokens");
    p.pages = c.pages;
    p.heads = c.heads;
    p.dch = c.head_dim / 8;
    p.width = width;
    p.planes = 2 * c.layers;
    p.div = MakePageDiv(c.page_size);
    // lanes per row: as many as leave one sweep for a path of this width, so
    // that a short path keeps its workgroups full
    const int lpr = width <= 8 ? 32 : width <= 16 ? 16 : 8;
    p.slices = (c.heads * p.dch + lpr - 1) / lpr;
    if (int64_t(p.slices) * s->seqs >= kMaxGrid) Refuse(who, "too many sequences");
    const auto go = [&](auto kern, int pl) {
        const dim3 grid(unsigned(p.slices) * unsigned(s->seqs), unsigned((p.planes + pl - 1) / pl));
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p);
    };
    if (lpr == 32) go(CompactKernel<32, 1, 4>, 4);
    else if (lpr == 16) go(CompactKernel<16, 1, 4>, 4);
    else if (width <= 64) go(CompactKernel<8, 2, 4>, 4);
    else go(CompactKernel<8, 8, 1>, 1);
    Check(hipGetLastError(), "cache_compact launch");
}

}  // namespace kr
