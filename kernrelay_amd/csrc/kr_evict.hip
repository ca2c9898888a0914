// Eviction from a paged key/value cache by accumulated attention weight: which
// tokens of a sequence stay, layer by layer and key head by key head, and their
// rows' move to the front. See kr_op_cache_evict. No counterpart in the
// reference, whose path ends with the prompt.
//
// Of n > budget tokens the first `sinks`, the last `recent` and, of those between
// (the middle), the K = budget - sinks - recent with the largest weights stay.
// With end = budget - recent: of the K, those that stand in [sinks, end) stay
// where they are; the free places there (holes) are as many as the others of
// the K (movers, all at end or behind), and the n-th hole takes the n-th mover.
// So only what has to move does, holes are nobody's source and movers nobody's
// destination: all of them can move at once. The recent tokens then come down
// to [end, budget), by a shift, in order.
//
// The first launch finds the K-th largest weight by its bits, 11 or 10 at a time
// from the top (a histogram of those that share the bits found so far), then
// lists holes and movers; the second and third move the rows.
#include <algorithm>

#include "kr_paged.h"

namespace kr {

namespace {

struct EvictParams {
    uint16_t *k, *v;
    float *w;
    int32_t *keep;
    const int32_t *table, *lens, *entry;
    int64_t layer_stride, page_stride, token_stride, head_stride;
    int64_t w_layer, w_entry, w_head, ld_table;
    int cap, pages, seqs, heads, layers, entries, width, budget, sinks, recent;
    PageDiv div;
};

// Tokens of sequence b; 0 if it is left alone (few enough, or no weights).
__device__ __forceinline__ int Evicted(const EvictParams &p, int b, int &entry)
{
    const int len = min(max(p.lens[b], 0), p.cap);
    entry = p.entry != nullptr ? p.entry[b] : b;
    return len > p.budget && len <= p.width && entry >= 0 && entry < p.entries ? len : 0;
}

// The order of the weights in that of whole numbers; 0 and -0 are equal, a NaN
// comes before everything.
__device__ __forceinline__ uint32_t KeyOf(float f)
{
    const uint32_t u = __float_as_uint(f + 0.0f);
    return f != f ? 0u : (u >> 31) != 0 ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;

// Sum of `v` over the threads before this one; `total` over all.
__device__ __forceinline__ int BlockScan(int v, int *part, int &total)
{
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
    const int incl = WaveScan(v, lane);
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
        const int x = part[i];
        before += i < wave ? x : 0;
        total += x;
    }
    __syncthreads();
    return before + incl - v;
}

__global__ void __launch_bounds__(kSelThreads) SelectKernel(EvictParams p)
{
    __shared__ int hist[2048];
    __shared__ int part[kSelWaves];
    __shared__ int found[3];
    const int tid = int(threadIdx.x);
    const int h = int(blockIdx.x) % p.heads, b = int(blockIdx.x) / p.heads, layer = int(blockIdx.y);
    int32_t *keep = p.keep + ((int64_t(layer) * p.seqs + b) * p.heads + h) * p.budget;
    int entry;
    const int len = Evicted(p, b, entry);
    if (len == 0) {
        const int n = min(min(max(p.lens[b], 0), p.cap), p.budget);
        for (int i = tid; i < p.budget; i += kSelThreads) keep[i] = i < n ? i : -1;
        return;
    }
    float *w = p.w + layer * p.w_layer + entry * p.w_entry + h * p.w_head;
    const int end = p.budget - p.recent, low = len - p.recent;
    const int K = end - p.sinks;
    // ---- the K-th largest key of the middle, how many of it are wanted and there
    uint32_t key = 0;
    int want = K, equal = 0;
    if (K > 0) {
        for (int step = 0; step < 3; ++step) {
            const int shift = step == 0 ? 21 : step == 1 ? 10 : 0;
            const int bins = step == 2 ? 1024 : 2048;
            for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int j = p.sinks + tid; j < low; j += kSelThreads) {
                const uint32_t x = KeyOf(w[j]);
                const bool in = step == 0 || (step == 1 ? (x >> 21) == (key >> 21) : (x >> 10) == (key >> 10));
                if (in) atomicAdd(&hist[(x >> shift) & uint32_t(bins - 1)], 1);
            }
            __syncthreads();
            // bins from the top: thread t has the two below 2048 - 2 t
            const int hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
            int total;
            const int above = BlockScan(hi + lo, part, total);
            if (above < want && above + hi + lo >= want) {
                const bool first = above + hi >= want;
                found[0] = first ? 2047 - 2 * tid : 2046 - 2 * tid;
                found[1] = want - above - (first ? 0 : hi);
                found[2] = first ? hi : lo;
            }
            __syncthreads();
            key |= uint32_t(found[0]) << shift;
            want = found[1];
            equal = found[2];
            __syncthreads();
        }
    }
    // of the `equal` tokens with exactly this weight the first `want` stay
    const bool ranked = want < equal;
    // ---- movers, in order, to keep[sinks..]; the equal ones before `end` come first
    int ties = 0, movers = 0;
    if (ranked) {
        for (int j0 = p.sinks; j0 < end; j0 += kSelThreads) {
            int total;
            const int j = j0 + tid;
            BlockScan(j < end && KeyOf(w[j]) == key ? 1 : 0, part, total);
            ties += total;
        }
    }
    const int ties_front = ties;
    if (K > 0) {
        for (int j0 = end; j0 < low; j0 += kSelThreads) {
            const int j = j0 + tid;
            const uint32_t x = j < low ? KeyOf(w[j]) : 0u;
            int total;
            bool wins = j < low && x > key;
            if (ranked) {
                const bool tie = j < low && x == key;
                const int rank = ties + BlockScan(tie ? 1 : 0, part, total);
                ties += total;
                wins = wins || (tie && rank < want);
            } else {
                wins = wins || (j < low && x == key);
            }
            const int at = movers + BlockScan(wins ? 1 : 0, part, total);
            movers += total;
            if (wins) keep[p.sinks + at] = j;
        }
    }
    __syncthreads();
    // ---- the holes, last to first: the one that comes n-th is at sinks + n or
    // behind it, so what is written over is no longer needed
    int left = movers;
    ties = ties_front;
    for (int j0 = p.sinks + (max(K - 1, 0) / kSelThreads) * kSelThreads; K > 0 && j0 >= p.sinks; j0 -= kSelThreads) {
        const int j = j0 + tid;
        const bool in = j < end;
        const uint32_t x = in ? KeyOf(w[j]) : 0u;
        int total;
        bool wins = in && x > key;
        if (ranked) {
            const bool tie = in && x == key;
            const int before = BlockScan(tie ? 1 : 0, part, total);
            ties -= total;
            wins = wins || (tie && ties + before < want);
        } else {
            wins = wins || (in && x == key);
        }
        const bool hole = in && !wins;
        const int before = BlockScan(hole ? 1 : 0, part, total);
        left -= total;
        const int of = hole ? keep[p.sinks + left + before] : j;
        __syncthreads();
        if (in) keep[j] = of;
    }
    for (int i = tid; i < p.sinks; i += kSelThreads) keep[i] = i;
    for (int i = end + tid; i < p.budget; i += kSelThreads) keep[i] = low + i - end;
    __syncthreads();
    // ---- the weights move as the rows will
    for (int i = p.sinks + tid; i < end; i += kSelThreads) {
        const int of = keep[i];
        if (of != i) w[i] = w[of];
    }
    __syncthreads();
    for (int i0 = end; i0 < p.budget; i0 += kSelThreads) {
        const int i = i0 + tid;
        const float x = i < p.budget ? w[low + i - end] : 0.0f;
        __syncthreads();
        if (i < p.budget) w[i] = x;
    }
}

// Element offset of column `col` of the row at position pos; -1: not there.
__device__ __forceinline__ int64_t RowAt(const EvictParams &p, const int32_t *table, int pos, int64_t col)
{
    const int pg = PageOf(p.div, pos);
    const int id = table[pg];
    if (id < 0 || id >= p.pages) return -1;
    return id * p.page_stride + int64_t(pos - pg * p.div.size) * p.token_stride + col;
}

constexpr int kMoveRows = 4;  // rows of a thread

// Rows to the holes: a workgroup has kMoveRows x 256 / LPR places of one
// sequence and head in one layer, K and V.
template <int LPR>
__global__ void __launch_bounds__(256) MoveKernel(EvictParams p, int slices)
{
    constexpr int RPS = 256 / LPR;
    const int slice = int(blockIdx.x) % slices, bh = int(blockIdx.x) / slices;
    const int h = bh % p.heads, b = bh / p.heads, layer = int(blockIdx.y);
    int entry;
    if (Evicted(p, b, entry) == 0) return;
    const int32_t *keep = p.keep + ((int64_t(layer) * p.seqs + b) * p.heads + h) * p.budget;
    const int32_t *table = p.table + b * p.ld_table;
    const int end = p.budget - p.recent;
    const int64_t col = h * p.head_stride + (int(threadIdx.x) % LPR) * 8;
    uint16_t *k = p.k + layer * p.layer_stride, *v = p.v + layer * p.layer_stride;
    uint4 x[kMoveRows][2];
    int64_t to[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
        const int i = p.sinks + (slice * kMoveRows + u) * RPS + int(threadIdx.x) / LPR;
        const int of = i < end ? keep[i] : i;
        const int64_t src = of != i ? RowAt(p, table, of, col) : -1;
        to[u] = src >= 0 ? RowAt(p, table, i, col) : -1;
        if (to[u] >= 0) {
            x[u][0] = *reinterpret_cast<const uint4 *>(k + src);
            x[u][1] = *reinterpret_cast<const uint4 *>(v + src);
        }
    }
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
        if (to[u] >= 0) {
            *reinterpret_cast<uint4 *>(k + to[u]) = x[u][0];
            *reinterpret_cast<uint4 *>(v + to[u]) = x[u][1];
        }
}

// The recent rows' shift: a workgroup has a sequence and head in one layer, K
// and V. Sweep by sweep: a later row's old place is behind all new ones so far.
template <int LPR>
__global__ void __launch_bounds__(256) ShiftKernel(EvictParams p)
{
    constexpr int RPS = 256 / LPR;
    const int h = int(blockIdx.x) % p.heads, b = int(blockIdx.x) / p.heads, layer = int(blockIdx.y);
    int entry;
    const int len = Evicted(p, b, entry);
    if (len == 0) return;
    const int32_t *table = p.table + b * p.ld_table;
    const int end = p.budget - p.recent;
    const int64_t col = h * p.head_stride + (int(threadIdx.x) % LPR) * 8;
    uint16_t *k = p.k + layer * p.layer_stride, *v = p.v + layer * p.layer_stride;
    for (int i0 = end; i0 < p.budget; i0 += kMoveRows * RPS) {
        uint4 x[kMoveRows][2];
        int64_t to[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int i = i0 + u * RPS + int(threadIdx.x) / LPR;
            const int64_t src = i < p.budget ? RowAt(p, table, len - p.budget + i, col) : -1;
            to[u] = src >= 0 ? RowAt(p, table, i, col) : -1;
            x[u][0] = x[u][1] = make_uint4(0, 0, 0, 0);
            if (to[u] >= 0) {
                x[u][0] = *reinterpret_cast<const uint4 *>(k + src);
                x[u][1] = *reinterpret_cast<const uint4 *>(v + src);
            }
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's rows are in registers
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u)
            if (to[u] >= 0) {
                *reinterpret_cast<uint4 *>(k + to[u]) = x[u][0];
                *reinterpret_cast<uint4 *>(v + to[u]) = x[u][1];
            }
        __syncthreads();
    }
}

}  // namespace

void EvictLaunch(const kr_cache *cache, const kr_seqs *s, const kr_weights *weights, int budget, int sinks, int recent,
                 int32_t *keep, hipStream_t stream)
{
    const char *who = "cache_evict";
    const auto refuse = [&](const char *what) { throw std::runtime_error(std::string(who) + ": " + what); };
    const kr_cache c = CheckCache(cache, who);
    CheckSeqs(s, who);
    const kr_weights w = CheckWeights(weights, c, who);
    if (budget < 1) refuse("a budget holds at least one token");
    if (sinks < 0 || recent < 0 || int64_t(sinks) + recent > budget) refuse("sinks and recent must fit the budget");
    if (s->seqs == 0) return;
    if (keep == nullptr || (reinterpret_cast<uintptr_t>(keep) & 3) != 0) refuse("keep is missing or misaligned");
    if (c.layers > 65535) refuse("too many layers");
    EvictParams p{};
    p.k = static_cast<uint16_t *>(c.k);
    p.v = static_cast<uint16_t *>(c.v);
    p.w = w.w;
    p.keep = keep;
    p.table = s->table;
    p.lens = s->lens;
    p.entry = w.entry;
    p.layer_stride = c.layer_stride;
    p.page_stride = c.page_stride;
    p.token_stride = c.token_stride;
    p.head_stride = c.head_stride;
    p.w_layer = w.layer_stride;
    p.w_entry = w.entry_stride;
    p.w_head = w.head_stride;
    p.ld_table = s->ld_table;
    const int64_t cap = int64_t(s->table_pages) * c.page_size;
    if (cap >= (int64_t(1) << 31) - 4096) refuse("the page table spans too many tokens");
    if (budget >= (1 << 30)) refuse("the budget is too large");
    p.cap = int(cap);
    p.pages = c.pages;
    p.seqs = s->seqs;
    p.heads = c.heads;
    p.layers = c.layers;
    p.entries = w.entries;
    p.width = w.width;
    p.budget = budget;
    p.sinks = sinks;
    p.recent = recent;
    p.div = MakePageDiv(c.page_size);
    const int64_t units = int64_t(s->seqs) * c.heads;
    const MemSpan list{keep, 4 * units * c.layers * budget}, ws = WeightsSpan(w);
    const int64_t all = 2 * ((c.layers - 1) * c.layer_stride + LayerSpan(c, c.k, 0).width);
    const MemSpan ks{c.k, all}, vs{c.v, all};
    if (Meets(list, ws) || Meets(list, ks) || Meets(list, vs) || Meets(ws, ks) || Meets(ws, vs))
        refuse("keep, the weights and the cache overlap");
    const int lpr = c.head_dim / 8, per = kMoveRows * (256 / lpr);
    const int slices = (budget - recent - sinks + per - 1) / per;
    if (units * std::max(slices, 1) >= (kMaxGrid >> 2)) refuse("too many sequences");
    hipLaunchKernelGGL(SelectKernel, dim3(unsigned(units), unsigned(c.layers)), dim3(kSelThreads), 0, stream, p);
    Check(hipGetLastError(), "cache_evict launch");
    if (slices > 0) {
        const dim3 grid(unsigned(units) * unsigned(slices), unsigned(c.layers));
        if (lpr == 8) hipLaunchKernelGGL((MoveKernel<8>), grid, dim3(256), 0, stream, p, slices);
        else hipLaunchKernelGGL((MoveKernel<16>), grid, dim3(256), 0, stream, p, slices);
    }
    if (recent > 0) {
        const dim3 grid(unsigned(units), unsigned(c.layers));
        if (lpr == 8) hipLaunchKernelGGL((ShiftKernel<8>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((ShiftKernel<16>), grid, dim3(256), 0, stream, p);
    }
    Check(hipGetLastError(), "cache_evict launch");
}

}  // namespace kr
