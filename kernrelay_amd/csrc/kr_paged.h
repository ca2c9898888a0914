// Host interface of the paged key/value cache's kernels: q/k norm + RoPE into
// plain tensors or cache slots, page copies and draft compaction
// (kr_cache.hip), attention over the pages (kr_paged.hip), the weight it gives
// each cached token (kr_weigh.hip) and the tokens that go by it (kr_evict.hip),
// drafts against the target's logits (kr_verify.hip). The handles are the C
// ABI's own (include/kr_ops.h).
#pragma once

#include "../../include/kr_ops.h"

#include "kr_common.h"

namespace kr {

// Quotient by a page size d: n / d = mulhi(2n, mul) >> shift, 0 <= n < 2^31.
// With l = ceil(log2 d) and mul = floor(2^(31+l) / d) + 1 (below 2^32, since
// 2^l < 2d), n mul / 2^(31+l) exceeds n / d by at most n d / (d 2^(31+l)) <=
// n / (2^31 d) < 1 / d: too little to reach the next whole number.
struct PageDiv {
    uint32_t mul = 0;
    int32_t shift = 0;
    int32_t size = 1;
};

inline PageDiv MakePageDiv(int d)
{
    int l = 0;
    while ((int64_t(1) << l) < d) ++l;
    PageDiv p;
    p.mul = uint32_t((uint64_t(1) << (31 + l)) / uint64_t(d) + 1);
    p.shift = l;
    p.size = d;
    return p;
}

__device__ __forceinline__ int PageOf(const PageDiv &d, int n)
{
    return int(__umulhi(uint32_t(n) * 2u, d.mul) >> d.shift);
}

// Workgroups of up to 256 threads that a launch may have in x (the runtime
// counts its threads in 32 bits).
constexpr int64_t kMaxGrid = int64_t(1) << 23;

// Rows of 16-bit values: `width` of them every `ld` elements.
struct RowSpan {
    const void *p = nullptr;
    int64_t ld = 0, rows = 0, width = 0;
};

// Do two of them share memory (rows lying between the other's, the columns of
// one projection, do not)?
bool Overlap(const RowSpan &a, const RowSpan &b);

// Keys (or values) of a layer, the gaps between its rows included.
RowSpan LayerSpan(const kr_cache &c, const void *base, int layer);

// Throws unless the cache handle describes memory that the kernels can walk:
// known type, head size 64 or 128, 16-byte aligned rows, strides in range.
// Strides of dimensions of one element are not looked at (and set to 0).
kr_cache CheckCache(const kr_cache *c, const char *who);
// The same for a batch handle.
void CheckSeqs(const kr_seqs *s, const char *who);

// One pass over q [rows, HQ, D] and k [rows, HKV, D]: per-head RMSNorm (with
// gammas) and the rotation; see kr_op_qk_norm_rope.
struct QkRopeDesc {
    kr_rope rope{};
    int dtype = kBF16;
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    int64_t ldq = 0, ldk = 0, ldv = 0;
    void *q_out = nullptr, *k_out = nullptr;
    int64_t ldqo = 0, ldko = 0;
    const int64_t *positions = nullptr;  // nullptr: row r is at position r
    const int64_t *slots = nullptr;      // with `cache`: where row r's k and v go
    const kr_cache *cache = nullptr;
    int layer = 0;
    int rows = 0, HQ = 0, HKV = 0, D = 0;
};
void QkRopeLaunch(const QkRopeDesc &d, hipStream_t stream);

void CopyPagesLaunch(const kr_cache *c, const int32_t *src, const int32_t *dst, int n, hipStream_t stream);
void CompactLaunch(const kr_cache *c, const kr_seqs *s, const int32_t *path, int64_t ld_path, int width,
                   const int32_t *path_lens, hipStream_t stream);

void PagedAttnNeeds(const kr_cache *c, const kr_seqs *s, int HQ, size_t *ws_bytes, int *counters);
struct PagedAttnDesc {
    const kr_cache *cache = nullptr;
    const kr_seqs *seqs = nullptr;
    int layer = 0;
    const void *q = nullptr;
    void *out = nullptr;
    int64_t ldq = 0, ldo = 0;
    int rows = 0, HQ = 0;
    float scale = 1.0f;
    void *ws = nullptr;
    size_t ws_bytes = 0;
    int32_t *cnt = nullptr;
    int cnt_len = 0;
    bool with_lse = false;  // the logarithms of the rows' sums too
    float *lse = nullptr;
    int64_t ld_lse = 0;
};
void PagedAttnLaunch(const PagedAttnDesc &d, hipStream_t stream);

// Memory from p on, as far as a launch may touch it.
struct MemSpan {
    const void *p = nullptr;
    int64_t bytes = 0;
};
inline bool Meets(const MemSpan &a, const MemSpan &b)
{
    if (a.p == nullptr || b.p == nullptr || a.bytes < 1 || b.bytes < 1) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x < y + uintptr_t(b.bytes) && y < x + uintptr_t(a.bytes);
}
// Rows of `width` values of `size` bytes, every `ld` values.
inline MemSpan RowsSpan(const void *p, int64_t rows, int64_t ld, int64_t width, int64_t size)
{
    return MemSpan{p, rows < 1 ? 0 : ((rows - 1) * ld + width) * size};
}

// Does an output meet an array that a launch reads through its sequences' handle?
bool MeetsSeqs(const MemSpan &out, const kr_seqs &s, int64_t rows);

// Throws unless the weights' rows are apart; strides of dimensions of one element become 0.
kr_weights CheckWeights(const kr_weights *w, const kr_cache &c, const char *who);
MemSpan WeightsSpan(const kr_weights &w);

// Attention weight per cached token (kr_weigh.hip).
void WeighNeeds(const kr_cache *c, const kr_seqs *s, int HQ, size_t *ws_bytes);
struct WeighDesc {
    const kr_cache *cache = nullptr;
    const kr_seqs *seqs = nullptr;
    const kr_weights *weights = nullptr;
    int layer = 0;
    const void *q = nullptr;
    const float *lse = nullptr;
    int64_t ldq = 0, ld_lse = 0;
    int rows = 0, HQ = 0, last = 0;
    float scale = 1.0f, decay = 1.0f;
    const int32_t *path = nullptr, *path_lens = nullptr;
    int64_t ld_path = 0;
    int path_width = 0;
    void *ws = nullptr;
    size_t ws_bytes = 0;
};
void WeighLaunch(const WeighDesc &d, hipStream_t stream);

// Tokens that got least go (kr_evict.hip).
void EvictLaunch(const kr_cache *c, const kr_seqs *s, const kr_weights *w, int budget, int sinks, int recent,
                 int32_t *keep, hipStream_t stream);

// Drafts against the target's logits (kr_verify.hip).
void VerifyNeeds(const kr_drafts *d, const kr_seqs *s, size_t *ws_bytes, int *counters);
struct VerifyOut {
    int32_t *path = nullptr, *path_lens = nullptr;
    int64_t ld_path = 0;
    int width = 0;
    int64_t *next = nullptr;
};
void VerifyLaunch(const kr_drafts *d, const kr_seqs *s, const VerifyOut &o, void *ws, size_t ws_bytes, int32_t *cnt,
                  int cnt_len, hipStream_t stream);

// A value that is the same in every lane, as the scalar it is.
__device__ __forceinline__ int Uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int WaveScan(int v, int lane)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}

}  // namespace kr
