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
// The first launch finds the K-th largest weight by its bits from the top, then
// lists holes and movers; the second and third move the rows.
//
// What bounds it, on an MI355X, on states that were not trimmed before: the moves
// by HBM, the lists by the steps of their selection, one after the other. Eight
// sequences of 1500..3000 tokens down to 1000, 28 layers of 4 heads of 128: lists
// 17 us, holes 131, the 100 recent tokens 25. One of 32000 down to 4000, 36 layers
// of 8 heads: 60, 213 and (501) 33. Sixteen of 265..530 down to 512, the same
// heads: 18, 25 (16 MB; the rest is the reading of every place's list entry) and
// (128) 44. The rows at the holes are scattered, 256 bytes a key and head: 4.0 and
// 4.3 TB/s of them, where a large copy reaches 4.9. A sequence that was trimmed and
// is trimmed again with the weights that the first time left behind moves half of
// these rows and less.
#include <algorithm>

#include "kr_dma.h"
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

// Sum of `v` over the threads of the workgroup before this one; `total` over all.
template <int NT>
__device__ __forceinline__ int BlockScan(int v, int *part, int &total)
{
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
    const int incl = WaveScan(v, lane);
    if constexpr (NT == 64) {
        total = __shfl(incl, 63, 64);
        return incl - v;
    }
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        const int x = part[i];
        before += i < wave ? x : 0;
        total += x;
    }
    __syncthreads();
    return before + incl - v;
}

// The K-th largest of the keys that `each` goes through, by its bits from the
// top, and how many of that key are wanted and there.
struct Threshold {
    uint32_t key;
    int want, equal;
};

// By a histogram of 11, 11 and 10 bits. Weights have few exponents, so that a
// wave's lanes often add to the same bin, one after the other: many threads have
// CP copies of it, by the lane.
template <int NT, int CP, typename F>
__device__ __forceinline__ Threshold ByHistogram(int K, int *hist, int *part, int *found, F &&each)
{
    constexpr int PER = 2048 / NT;  // bins of a thread
    const int tid = int(threadIdx.x);
    Threshold t{0, K, 0};
    for (int step = 0; step < 3; ++step) {
        const int shift = step == 0 ? 21 : step == 1 ? 10 : 0;
        const uint32_t mask = step == 2 ? 1023 : 2047;
        for (int i = tid; i < 2048 * CP; i += NT) hist[i] = 0;
        __syncthreads();
        each([&](uint32_t x) {
            const bool in = step == 0 || (step == 1 ? (x >> 21) == (t.key >> 21) : (x >> 10) == (t.key >> 10));
            if (in) atomicAdd(&hist[((x >> shift) & mask) * CP + (tid & (CP - 1))], 1);
        });
        __syncthreads();
        // bins from the top: thread i has PER of them below 2048 - PER i
        int mine[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            mine[i] = 0;
#pragma unroll
            for (int c = 0; c < CP; ++c) mine[i] += hist[(2047 - PER * tid - i) * CP + c];
            sum += mine[i];
        }
        int total;
        int above = BlockScan<NT>(sum, part, total);
        if (above < t.want && above + sum >= t.want) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (above < t.want && above + mine[i] >= t.want) {
                    found[0] = 2047 - PER * tid - i;
                    found[1] = t.want - above;
                    found[2] = mine[i];
                }
                above += mine[i];
            }
        }
        __syncthreads();
        t.key |= uint32_t(found[0]) << shift;
        t.want = found[1];
        t.equal = found[2];
        __syncthreads();
    }
    return t;
}

__device__ __forceinline__ int32_t *KeepOf(const EvictParams &p, int layer, int b, int h)
{
    return p.keep + ((int64_t(layer) * p.seqs + b) * p.heads + h) * p.budget;
}

// Before the rest of a list: a sequence that is left alone.
__device__ __forceinline__ bool LeftAlone(const EvictParams &p, int b, int len, int32_t *keep, int nt)
{
    if (len > 0) return false;
    const int n = min(min(max(p.lens[b], 0), p.cap), p.budget);
    for (int i = int(threadIdx.x); i < p.budget; i += nt) keep[i] = i < n ? i : -1;
    return true;
}

// The rest of a list, and the recent tokens' weights: a shift, in order.
template <int NT>
__device__ __forceinline__ void Recent(const EvictParams &p, int len, int32_t *keep, float *w)
{
    const int tid = int(threadIdx.x);
    const int end = p.budget - p.recent, low = len - p.recent;
    for (int i = tid; i < p.sinks; i += NT) keep[i] = i;
    for (int i = end + tid; i < p.budget; i += NT) keep[i] = low + i - end;
    for (int i0 = end; i0 < p.budget; i0 += NT) {
        const int i = i0 + tid;
        const float x = i < p.budget ? w[low + i - end] : 0.0f;
        __syncthreads();
        if (i < p.budget) w[i] = x;
    }
}

// A list by NT threads that hold all of the middle: thread t tokens sinks + t +
// NT i. A wave alone finds the threshold bit by bit with ballots, more of them by
// histograms. Ranks come from one scan over the items' waves. The choice of NT and
// IT, measured on all lists of a launch (lists, tokens of the longest middle): 4608
// of 232: <64, 4> 41.6 us, <256, 4> 45.3; 4608 of 832: <256, 4> 136, <64, 16> 144;
// 896 of 3832: <256, 16> 48.5, <1024, 4> 67; 576 of 14900: <1024, 16> 72,
// SelectLongKernel 84.
template <int NT, int IT>
__global__ void __launch_bounds__(NT) SelectKernel(EvictParams p)
{
    constexpr int NW = NT / 64, CELLS = IT * NW, CP = NT == 1024 ? 4 : 1;
    __shared__ int hist[NT == 64 ? 1 : 2048 * CP];
    __shared__ int part[NW];
    __shared__ int found[3];
    __shared__ int cells[2][CELLS];
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int h = int(blockIdx.x) % p.heads, b = int(blockIdx.x) / p.heads, layer = int(blockIdx.y);
    int32_t *keep = KeepOf(p, layer, b, h);
    int entry;
    const int len = Evicted(p, b, entry);
    if (LeftAlone(p, b, len, keep, NT)) return;
    float *w = p.w + layer * p.w_layer + entry * p.w_entry + h * p.w_head;
    const int end = p.budget - p.recent, low = len - p.recent;
    const int K = end - p.sinks;
    if (K > 0) {
        uint32_t key[IT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int j = p.sinks + tid + NT * i;
            key[i] = KeyOf(w[uint32_t(min(j, low - 1))]);
        }
        const int items = (low - p.sinks - tid + NT - 1) / NT;
        const auto in = [&](int i) { return i < items; };
        Threshold t{0, K, 0};
        if constexpr (NT == 64) {
            // the largest key that K of them reach
            for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < IT; ++i) n += __popcll(__ballot(in(i) && key[i] >= (t.key | bit)));
                if (n >= K) t.key |= bit;
            }
            int above = 0;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                above += __popcll(__ballot(in(i) && key[i] > t.key));
                t.equal += __popcll(__ballot(in(i) && key[i] == t.key));
            }
            t.want = K - above;
        } else {
            t = ByHistogram<NT, CP>(K, hist, part, found, [&](auto &&add) {
#pragma unroll
                for (int i = 0; i < IT; ++i)
                    if (in(i)) add(key[i]);
            });
        }
        // how many tokens of an item's wave there are in front, for each of two kinds
        const uint64_t below = (1ull << lane) - 1;
        const auto scan = [&](auto &&kind, int kinds) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
                for (int k = 0; k < kinds; ++k) {
                    const int n = __popcll(__ballot(kind(i, k)));
                    if (lane == 0) cells[k][i * NW + wave] = n;
                }
            __syncthreads();
            for (int k = 0; k < kinds; ++k) {
                constexpr int PER = (CELLS + NT - 1) / NT;
                int mine[PER], sum = 0, total;
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    mine[c] = tid * PER + c < CELLS ? cells[k][tid * PER + c] : 0;
                    sum += mine[c];
                }
                int at = BlockScan<NT>(sum, part, total);
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    if (tid * PER + c < CELLS) cells[k][tid * PER + c] = at;
                    at += mine[c];
                }
            }
            __syncthreads();
        };
        uint32_t wins = 0;  // bit i
        static_assert(IT <= 32, "a bit an item");
        if (t.want < t.equal) {  // of the equal ones the first `want` stay
            scan([&](int i, int) { return in(i) && key[i] == t.key; }, 1);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const bool tie = in(i) && key[i] == t.key;
                const int rank = cells[0][i * NW + wave] + __popcll(__ballot(tie) & below);
                if (in(i) && (key[i] > t.key || (tie && rank < t.want))) wins |= 1u << i;
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < IT; ++i)
                if (in(i) && key[i] >= t.key) wins |= 1u << i;
        }
        const auto won = [&](int i) { return ((wins >> i) & 1) != 0; };
        const auto kind = [&](int i, int k) {
            const int j = p.sinks + tid + NT * i;
            return k == 0 ? won(i) && j >= end : !won(i) && j < end;
        };
        scan(kind, 2);
        // the movers, in order, to keep[sinks..]; then to the holes, which are as many
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const bool mover = kind(i, 0);
            const uint64_t all = __ballot(mover);
            if (mover) keep[uint32_t(p.sinks + cells[0][i * NW + wave] + __popcll(all & below))] = p.sinks + tid + NT * i;
        }
        __syncthreads();
        int of[IT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const bool hole = kind(i, 1);
            const uint64_t all = __ballot(hole);
            of[i] = hole ? keep[uint32_t(p.sinks + cells[1][i * NW + wave] + __popcll(all & below))] : -1;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int j = p.sinks + tid + NT * i;
            if (j >= end) continue;
            keep[uint32_t(j)] = of[i] >= 0 ? of[i] : j;
            if (of[i] >= 0) w[uint32_t(j)] = w[uint32_t(of[i])];  // (nobody's hole)
        }
        __syncthreads();
    }
    Recent<NT>(p, len, keep, w);
}

// Longer middles: tiles of 8192 tokens, read again for each step; two workgroups
// a CU. (288 middles of 31483: 70 us; in registers, 32 tokens a thread and one
// workgroup a CU, 66, but tiles of 16384 99.) What is read again may have changed
// where two sequences have the same entry, against the contract: places and tokens
// in the list are held within it.
__global__ void __attribute__((amdgpu_flat_work_group_size(1024, 1024), amdgpu_waves_per_eu(8)))
SelectLongKernel(EvictParams p)
{
    constexpr int NT = 1024, IT = 8, NW = NT / 64, TILE = NT * IT, CP = 4;
    __shared__ int hist[2048 * CP];
    __shared__ int part[NW];
    __shared__ int found[3];
    __shared__ int cells[IT * NW];
    static_assert(IT * NW <= NT, "a cell a thread");
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int h = int(blockIdx.x) % p.heads, b = int(blockIdx.x) / p.heads, layer = int(blockIdx.y);
    int32_t *keep = KeepOf(p, layer, b, h);
    int entry;
    const int len = Evicted(p, b, entry);
    if (LeftAlone(p, b, len, keep, NT)) return;
    float *w = p.w + layer * p.w_layer + entry * p.w_entry + h * p.w_head;
    const int end = p.budget - p.recent, low = len - p.recent;
    const int K = end - p.sinks;
    if (K > 0) {
        uint32_t key[IT];
        // (the next tile's on their way meanwhile: 73 us for 70)
        const auto load = [&](int j0, int last) {
#pragma unroll
            for (int i = 0; i < IT; ++i) key[i] = KeyOf(w[uint32_t(min(j0 + tid + NT * i, last - 1))]);
        };
        const Threshold t = ByHistogram<NT, CP>(K, hist, part, found, [&](auto &&add) {
            for (int j0 = p.sinks; j0 < low; j0 += TILE) {
                load(j0, low);
#pragma unroll
                for (int i = 0; i < IT; ++i)
                    if (j0 + tid + NT * i < low) add(key[i]);
            }
        });
        const uint64_t below = (1ull << lane) - 1;
        // how many of a tile's tokens of a kind are in front of each item's wave; returns how many there are
        const auto scan = [&](auto &&kind) {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int n = __popcll(__ballot(kind(i)));
                if (lane == 0) cells[i * NW + wave] = n;
            }
            __syncthreads();
            int total;
            const int at = BlockScan<NT>(tid < IT * NW ? cells[tid] : 0, part, total);
            if (tid < IT * NW) cells[tid] = at;
            __syncthreads();
            return total;
        };
        // which of a tile's tokens stay, as bits; `ties`: equal ones in front of the tile, of which the first `want` stay
        const bool ranked = t.want < t.equal;
        const auto winners = [&](int j0, int last, int ties, int &here) {
            uint32_t wins = 0;
            here = 0;
            if (ranked) here = scan([&](int i) { return j0 + tid + NT * i < last && key[i] == t.key; });
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const bool in = j0 + tid + NT * i < last, tie = in && key[i] == t.key;
                const uint64_t all = __ballot(tie);
                const bool stays = tie && (!ranked || ties + cells[i * NW + wave] + __popcll(all & below) < t.want);
                if (stays || (in && key[i] > t.key)) wins |= 1u << i;
            }
            if (ranked) __syncthreads();
            return wins;
        };
        // ---- movers, in order, to keep[sinks..]; the equal ones before `end` come first
        int ties = 0, movers = 0, here;
        if (ranked)
            for (int j0 = p.sinks; j0 < end; j0 += TILE) {
                load(j0, end);
                winners(j0, end, ties, here);
                ties += here;
            }
        const int ties_front = ties;
        for (int j0 = end; j0 < low; j0 += TILE) {
            load(j0, low);
            const uint32_t wins = winners(j0, low, ties, here);
            ties += here;
            const int all = scan([&](int i) { return ((wins >> i) & 1) != 0; });
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const bool mover = ((wins >> i) & 1) != 0;
                const uint64_t of = __ballot(mover);
                const int at = p.sinks + movers + cells[i * NW + wave] + __popcll(of & below);
                if (mover && at < end) keep[at] = j0 + tid + NT * i;
            }
            movers += all;
            __syncthreads();
        }
        // ---- the holes, last tile to first: the one that comes n-th is at sinks +
        // n or behind it, so what is written over is no longer needed
        int left = movers;
        ties = ties_front;
        for (int j0 = p.sinks + (K - 1) / TILE * TILE; j0 >= p.sinks; j0 -= TILE) {
            load(j0, end);
            if (ranked) ties -= scan([&](int i) { return j0 + tid + NT * i < end && key[i] == t.key; });
            if (ranked) __syncthreads();
            const uint32_t wins = winners(j0, end, ties, here);
            const auto hole = [&](int i) { return j0 + tid + NT * i < end && ((wins >> i) & 1) == 0; };
            left -= scan(hole);
            int of[IT];
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const bool is = hole(i);
                const uint64_t all = __ballot(is);
                const int at = p.sinks + left + cells[i * NW + wave] + __popcll(all & below);
                of[i] = is ? min(max(keep[min(max(at, p.sinks), end - 1)], 0), len - 1) : j0 + tid + NT * i;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < IT; ++i)
                if (j0 + tid + NT * i < end) keep[j0 + tid + NT * i] = of[i];
        }
        __syncthreads();
        // ---- the weights move as the rows will
        for (int i = p.sinks + tid; i < end; i += NT) {
            const int of = keep[i];
            if (of != i) w[i] = w[of];
        }
        __syncthreads();
    }
    Recent<NT>(p, len, keep, w);
}

// Element offset of column `col` of the row at position pos; -1: not there.
__device__ __forceinline__ int64_t RowAt(const EvictParams &p, const int32_t *table, int pos, int64_t col)
{
    const int pg = PageOf(p.div, pos);
    const int id = table[pg];
    if (id < 0 || id >= p.pages) return -1;
    return id * p.page_stride + int64_t(pos - pg * p.div.size) * p.token_stride + col;
}

typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
// All of the call, trims / the eight sequences / the long one above, on states that
// were not trimmed before: 91 / 175 / 303 us; 2 rows 98 / 180 / 306, 8 rows 89 / 176
// / 309; 2048 workgroups 92 / 188 / 319, 8192 92 / 169 / 298; stores that stay in
// the L2 90 / 162 / 282. The same states trimmed again and again, where few rows
// move: 83 / 67 / 126; 8 rows 83 / 66 / 131; 8192 workgroups 85 / 67 / 126; stores
// that stay 85 / 70 / 133. (Chosen on the latter, the only ones timed at first.)
constexpr int kMoveRows = 4;       // rows of a thread
constexpr int kMoveGroups = 4096;  // workgroups: 16 for each of 256 CUs

// The sequences that lose tokens, 64 at a time: body(b, unit) for this
// workgroup's share of the `per` units of each of them. (Most of a batch that is
// trimmed often has nothing to lose; a workgroup for each of its units would
// cost 1 ns a wave to start.)
template <typename F>
__device__ __forceinline__ void EachUnit(const EvictParams &p, int64_t per, F &&body)
{
    const int lane = int(threadIdx.x) & 63;
    int64_t u = blockIdx.x;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        int entry;
        const uint64_t some = __ballot(b0 + lane < p.seqs && Evicted(p, min(b0 + lane, p.seqs - 1), entry) > 0);
        const int64_t units = per * __popcll(some);
        for (; u < units; u += gridDim.x) {
            const int nth = int(u / per);
            uint64_t rest = some;
            for (int i = 0; i < nth; ++i) rest &= rest - 1;
            body(Uni(b0 + __builtin_ctzll(rest)), u - nth * per);
        }
        u -= units;
    }
}

// Rows of K and V of a sequence and head in one layer that move together: four
// a thread, LPR lanes a row. All loads go out before the first store, and the
// stores do not stay in the L2, which the reads need.
template <int LPR>
struct MoveRows {
    static constexpr int RPS = 256 / LPR, ROWS = kMoveRows * RPS;
    U32x4 x[kMoveRows][2];
    int64_t to[kMoveRows];
    // place i0 + n gets the row of token of(place); -1: stays
    template <typename F>
    __device__ __forceinline__ void Load(const EvictParams &p, int b, int layer, int h, int i0, F &&of)
    {
        const int32_t *table = p.table + b * p.ld_table;
        const int64_t col = h * p.head_stride + (int(threadIdx.x) % LPR) * 8;
        const uint16_t *k = p.k + layer * p.layer_stride, *v = p.v + layer * p.layer_stride;
        int64_t from[kMoveRows];
#pragma unroll
        for (int n = 0; n < kMoveRows; ++n) {
            const int i = i0 + n * RPS + int(threadIdx.x) / LPR;
            const int j = of(i);
            from[n] = j >= 0 ? RowAt(p, table, j, col) : -1;
            to[n] = from[n] >= 0 ? RowAt(p, table, i, col) : -1;
        }
#pragma unroll
        for (int n = 0; n < kMoveRows; ++n)
            if (to[n] >= 0) {
                x[n][0] = *reinterpret_cast<const U32x4 *>(k + from[n]);
                x[n][1] = *reinterpret_cast<const U32x4 *>(v + from[n]);
            }
        asm volatile("" ::: "memory");  // (a row's store would join its load)
    }
    __device__ __forceinline__ void Store(const EvictParams &p, int layer) const
    {
        uint16_t *k = p.k + layer * p.layer_stride, *v = p.v + layer * p.layer_stride;
#pragma unroll
        for (int n = 0; n < kMoveRows; ++n)
            if (to[n] >= 0) {
                __builtin_nontemporal_store(x[n][0], reinterpret_cast<U32x4 *>(k + to[n]));
                __builtin_nontemporal_store(x[n][1], reinterpret_cast<U32x4 *>(v + to[n]));
            }
    }
};

// Rows to the holes: a unit is a slice of the places of one sequence and head in one layer.
template <int LPR>
__global__ void __launch_bounds__(256) MoveKernel(EvictParams p, int slices)
{
    EachUnit(p, int64_t(slices) * p.heads * p.layers, [&](int b, int64_t unit) {
        const int slice = Uni(int(unit % slices)), lh = Uni(int(unit / slices));
        const int h = lh % p.heads, layer = lh / p.heads;
        const int32_t *keep = KeepOf(p, layer, b, h);
        const int end = p.budget - p.recent;
        MoveRows<LPR> r;
        r.Load(p, b, layer, h, p.sinks + slice * MoveRows<LPR>::ROWS, [&](int i) {
            const int j = i < end ? keep[i] : i;
            return j != i ? j : -1;
        });
        r.Store(p, layer);
    });
}

// The recent rows' shift. Where their new places are none of the old ones, a
// unit is a slice as above. Otherwise it is all of a sequence and head in one
// layer, slice by slice, each read before any of it is written: a slice's old
// places are behind all new ones so far. What that costs, 6000 recent tokens of one
// sequence that come down by 10: 48 lists of 64 values a row 103 us, 1.4 TB/s from
// 48 workgroups; 288 of 128 a row 475 us, 3.7 TB/s.
template <int LPR>
__global__ void __launch_bounds__(256) ShiftKernel(EvictParams p, int slices)
{
    constexpr int ROWS = MoveRows<LPR>::ROWS;
    EachUnit(p, int64_t(slices) * p.heads * p.layers, [&](int b, int64_t unit) {
        // (slice by slice: only the first of an overlapping shift has work)
        const int slice = Uni(int(unit / (p.heads * p.layers))), lh = Uni(int(unit % (p.heads * p.layers)));
        const int h = lh % p.heads, layer = lh / p.heads;
        const int by = min(p.lens[b], p.cap) - p.budget;
        const auto of = [&](int i) { return i < p.budget ? i + by : -1; };
        const int i0 = p.budget - p.recent;
        MoveRows<LPR> r;
        if (by >= p.recent) {
            r.Load(p, b, layer, h, i0 + slice * ROWS, of);
            r.Store(p, layer);
        } else if (slice == 0) {
            for (int n = 0; n < slices; ++n) {
                r.Load(p, b, layer, h, i0 + n * ROWS, of);
                __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's rows are in registers
                __syncthreads();
                r.Store(p, layer);
                __syncthreads();
            }
        }
    });
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
    const MemSpan entry = RowsSpan(w.entry, 1, 0, s->seqs, 4);
    if (Meets(list, ws) || Meets(list, ks) || Meets(list, vs) || Meets(ws, ks) || Meets(ws, vs))
        refuse("keep, the weights and the cache overlap");
    for (const MemSpan &out : {list, ws, ks, vs})
        if (MeetsSeqs(out, *s, 0) || Meets(out, entry)) refuse("an output overlaps what the handles read");
    if (units >= (kMaxGrid >> 2)) refuse("too many sequences");
    // the middle of the longest sequence that there is room for: lengths are on the
    // device, so that wide tables and weights choose kernels for longer sequences than
    // there are. (The calls at kMoveRows with room for 8192 tokens: trims 193 us for
    // 91, one of 700 tokens 29 for 24; the eight with room for 16384, 218 for 175.)
    const int64_t middle = std::min<int64_t>(cap, w.width) - sinks - recent;
    const dim3 lists(unsigned(units), unsigned(c.layers));
    const auto select = [&](auto kern, int nt) { hipLaunchKernelGGL(kern, lists, dim3(unsigned(nt)), 0, stream, p); };
    if (middle <= 256) select(SelectKernel<64, 4>, 64);
    else if (middle <= 1024) select(SelectKernel<256, 4>, 256);
    else if (middle <= 4096) select(SelectKernel<256, 16>, 256);
    else if (middle <= 16384) select(SelectKernel<1024, 16>, 1024);
    else select(SelectLongKernel, 1024);
    Check(hipGetLastError(), "cache_evict launch");
    const int lpr = c.head_dim / 8, per = kMoveRows * (256 / lpr);
    const auto move = [&](auto kern, int places) {
        const int slices = (places + per - 1) / per;
        const dim3 grid(unsigned(std::min<int64_t>(units * c.layers * slices, kMoveGroups)));
        if (slices > 0) hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p, slices);
    };
    lpr == 8 ? move(MoveKernel<8>, budget - recent - sinks) : move(MoveKernel<16>, budget - recent - sinks);
    lpr == 8 ? move(ShiftKernel<8>, recent) : move(ShiftKernel<16>, recent);
    Check(hipGetLastError(), "cache_evict launch");
}

}  // namespace kr
