// Host interface of the paged key/value cache's kernels: q/k norm + RoPE into
// plain tensors or cache slots, page copies and draft compaction
// (kr_cache.hip), attention over the pages (kr_paged.hip). The handles are
// the C ABI's own (include/kr_ops.h).
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
};
void PagedAttnLaunch(const PagedAttnDesc &d, hipStream_t stream);

}  // namespace kr
