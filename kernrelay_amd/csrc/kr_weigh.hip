// Attention weight per cached token: what each key of a paged cache gets from
// a launch's new tokens. See kr_op_attention_paged_weigh. No counterpart in the
// reference, whose path ends with the prompt.
//
// Key j of a sequence and key head, over the packed rows i (a new token and a
// query head of the key head's G) that see it:
//   w_j <- decay w_j + sum_i exp(s q_i.k_j - lse_i)   (a new token: the sum alone)
// The attention over the same rows has left lse, so one pass over K is enough
// and a key's sum belongs to one wave: no atomics.
//
// The scores are those of the attention (kr_paged.hip): S^T = K Q^T, a wave 32
// keys by 32 rows at a time, the keys in its registers. Lane l's row is l % 32,
// register v's key 8 (v / 4) + 4 (l / 32) + v % 4; the sums over rows stay in 16
// registers until the last row, and are then added up across lanes.
#include <algorithm>
#include <cmath>

#include "kr_attncore.h"
#include "kr_paged.h"

namespace kr {

kr_weights CheckWeights(const kr_weights *w, const kr_cache &c, const char *who)
{
    const auto refuse = [&](const char *what) { throw std::runtime_error(std::string(who) + ": " + what); };
    if (w == nullptr || w->w == nullptr) refuse("needs weights");
    kr_weights r = *w;
    if (r.layers != c.layers || r.heads != c.heads) refuse("the weights are of other layers or heads than the cache");
    if (r.entries < 1 || r.width < 1) refuse("the weights are empty");
    if ((reinterpret_cast<uintptr_t>(r.w) & 3) != 0 || (reinterpret_cast<uintptr_t>(r.entry) & 3) != 0)
        refuse("the weights are misaligned");
    if (r.layers == 1) r.layer_stride = 0;
    if (r.entries == 1) r.entry_stride = 0;
    if (r.heads == 1) r.head_stride = 0;
    // dimensions from the inside out: each steps past all that lies inside it
    struct Dim { int64_t n, stride; } d[3] = {{r.layers, r.layer_stride}, {r.entries, r.entry_stride}, {r.heads, r.head_stride}};
    std::sort(d, d + 3, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    int64_t extent = r.width;
    for (const Dim &x : d) {
        if (x.n == 1) continue;
        if (x.stride < extent || x.stride > (int64_t(1) << 40)) refuse("rows of the weights overlap");
        extent += (x.n - 1) * x.stride;
    }
    return r;
}

MemSpan WeightsSpan(const kr_weights &w)
{
    return MemSpan{w.w, 4 * ((w.layers - 1) * w.layer_stride + (w.entries - 1) * w.entry_stride +
                             (w.heads - 1) * w.head_stride + w.width)};
}

namespace {

struct WeighParams {
    const uint16_t *q, *k;
    const float *lse;
    float *w;
    const int32_t *table, *lens, *starts, *entry, *path, *path_lens;
    const uint64_t *tree;
    int64_t ldq, ld_lse, ld_table, ld_tree, ld_path;
    int64_t head_stride, w_entry, w_head;
    uint32_t page_stride, token_stride;
    int cap, pages, table_pages, seqs, rows, max_new, tree_words, HQ, HKV, G;
    int entries, width, path_width, last;
    float scale_log2, decay;
    PageDiv div;
};

// A sequence as the launch has it, every number within its bounds whatever
// the device arrays hold.
struct WeighSeq {
    int first, rows;      // its first row and how many it has
    int n, skip;          // new tokens (of the path, if there is one); those before `skip` do not count
    int len, total;       // cached tokens, and all
    int cols;             // columns that it has in the weights
    int entry;
};

__device__ __forceinline__ WeighSeq LoadSeq(const WeighParams &p, int b)
{
    WeighSeq s;
    s.first = min(max(p.starts[b], 0), p.rows);
    s.rows = min(min(max(p.starts[b + 1], s.first), p.rows) - s.first, p.max_new);
    s.n = p.path != nullptr ? min(max(p.path_lens[b], 0), min(p.path_width, s.rows)) : s.rows;
    s.skip = p.last > 0 ? max(s.n - p.last, 0) : 0;
    s.len = max(p.lens[b], 0);
    s.total = int(min(int64_t(s.len) + s.n, int64_t(p.cap)));
    s.len = min(s.len, p.cap);
    s.entry = p.entry != nullptr ? p.entry[b] : b;
    s.cols = s.n > 0 && s.entry >= 0 && s.entry < p.entries ? min(s.total, p.width) : 0;
    return s;
}

constexpr int kWeighKeys = 128;  // of a workgroup's tile: 32 a wave
constexpr int kWeighGroups = 2048;

template <int DT, int D>
__global__ void __launch_bounds__(256) WeighKernel(WeighParams p)
{
    const int lane = int(threadIdx.x) & 63, wave = Uni(int(threadIdx.x) >> 6);
    const int hf = lane >> 5;
    // tiles of all sequences in one line: key head by key head, 128 keys each
    const auto tiles_of = [&](const WeighSeq &s) { return p.HKV * ((s.cols + kWeighKeys - 1) / kWeighKeys); };
    int tiles = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        int u = b0 + lane < p.seqs ? tiles_of(LoadSeq(p, b0 + lane)) : 0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) u += __shfl_xor(u, o, 64);
        tiles += Uni(u);
    }
    const int share = (tiles + int(gridDim.x) - 1) / int(gridDim.x);
    int x = int(blockIdx.x) * share;
    const int x_end = min(x + share, tiles);
    if (x >= x_end) return;
    int b = 0, base = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        const int u = b0 + lane < p.seqs ? tiles_of(LoadSeq(p, b0 + lane)) : 0;
        const int incl = WaveScan(u, lane) + base;
        const uint64_t above = __ballot(incl > x);
        const int at = above != 0 ? __builtin_ctzll(above) : 63;
        base = Uni(__shfl(incl - (above != 0 ? u : 0), at, 64));
        if (above != 0) {
            b = b0 + at;
            break;
        }
    }
    WeighSeq sq = LoadSeq(p, b);
    for (; x < x_end; ++x) {
        while (x >= base + tiles_of(sq)) {
            base += tiles_of(sq);
            sq = LoadSeq(p, ++b);
        }
        const int per = (sq.cols + kWeighKeys - 1) / kWeighKeys;
        const int h = Uni((x - base) / per), t = x - base - h * per;
        const int j0 = Uni(t * kWeighKeys + wave * 32);
        if (j0 >= sq.cols) continue;
        // this wave's keys: lane l holds key l % 32's chunks of 8, every second one
        const int pos = j0 + (lane & 31);
        const int pg = PageOf(p.div, min(pos, sq.total - 1));
        const int id = p.table[b * p.ld_table + pg];
        const bool ok = pos < sq.total && uint32_t(id) < uint32_t(p.pages);
        const int64_t off = ok ? int64_t(uint64_t(uint32_t(id)) * p.page_stride +
                                         uint64_t(uint32_t(pos - pg * p.div.size)) * p.token_stride)
                               : 0;
        const uint16_t *kr = p.k + h * p.head_stride + off + hf * 8;
        uint4 kf[D / 16];
#pragma unroll
        for (int dc = 0; dc < D / 16; ++dc) kf[dc] = *reinterpret_cast<const uint4 *>(kr + dc * 16);
        const uint32_t there = uint32_t(__ballot(ok));
        float sum[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) sum[v] = 0.0f;
        const int R = (sq.n - sq.skip) * p.G;
        // rows whose token comes before the wave's first key see none of it
        int r0 = 0;
        if ((p.tree == nullptr || p.path != nullptr) && j0 - sq.len > sq.skip)
            r0 = (j0 - sq.len - sq.skip) * p.G / 32 * 32;
        for (; r0 < R; r0 += 32) {
            const int r = min(r0 + (lane & 31), R - 1);
            const int i = sq.skip + r / p.G;  // the new token
            const int g = r % p.G;
            int tok = i;                      // its row of the sequence
            if (p.path != nullptr) tok = p.path[b * p.ld_path + i];
            const bool live = r0 + (lane & 31) < R && tok >= 0 && tok < sq.rows;
            const int64_t row = sq.first + (live ? tok : 0);
            const uint16_t *qr = p.q + row * p.ldq + int64_t(h * p.G + g) * D + hf * 8;
            uint4 qf[D / 16];
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) qf[dc] = *reinterpret_cast<const uint4 *>(qr + dc * 16);
            const float lse = p.lse[row * p.ld_lse + h * p.G + g];
            const float nl = lse * -1.4426950408889634f;
            f32x16 s;
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) s = Mfma<DT>(kf[dc], qf[dc], s);
            uint32_t sees = live && lse != -INFINITY ? there : 0u;
            const int nj = j0 - sq.len;  // the first key as a new token
            if (p.tree != nullptr && p.path == nullptr) {
                if (nj + 31 >= 0) {
                    const uint64_t *tree = p.tree + row * p.ld_tree;
                    const auto word = [&](int w) { return w < p.tree_words ? tree[w] : 0ull; };
                    uint64_t w;
                    if (nj >= 0) {
                        w = word(nj >> 6) >> (nj & 63);
                        if ((nj & 63) != 0) w |= word((nj >> 6) + 1) << (64 - (nj & 63));
                    } else {
                        w = ((1ull << -nj) - 1) | (word(0) << -nj);
                    }
                    sees &= uint32_t(w);
                }
            } else {
                const int nb = i - nj + 1;
                sees &= nb >= 32 ? ~0u : nb <= 0 ? 0u : (1u << nb) - 1;
            }
            const uint32_t bits = sees >> (4 * hf);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], p.scale_log2, nl));
                sum[v] += ((bits >> (8 * (v >> 2) + (v & 3))) & 1) != 0 ? e : 0.0f;
            }
        }
        // over the 32 lanes of a half: each step halves the registers, a lane
        // keeps the half that its bit names
#pragma unroll
        for (int m = 8, o = 16; m > 0; m >>= 1, o >>= 1) {
            const bool up = (lane & o) != 0;
#pragma unroll
            for (int v = 0; v < m; ++v) {
                const float give = up ? sum[v] : sum[v + m], own = up ? sum[v + m] : sum[v];
                sum[v] = own + __shfl_xor(give, o, 64);
            }
        }
        const float got = sum[0] + __shfl_xor(sum[0], 1, 64);
        const int v = (lane >> 1) & 15;
        // bit 16 of the lane chose the registers' bit 3, 8 bit 2, 4 bit 1, 2 bit 0
        const int key = j0 + 8 * (v >> 2) + 4 * hf + (v & 3);
        if ((lane & 1) == 0 && key < sq.cols) {
            float *w = p.w + int64_t(sq.entry) * p.w_entry + int64_t(h) * p.w_head + key;
            float old = 0.0f;
            if (key < sq.len && p.decay != 0.0f) old = p.decay * *w;
            *w = old + got;
        }
    }
}

}  // namespace

void WeighNeeds(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes)
{
    const char *who = "attention_paged_weigh";
    const kr_cache c = CheckCache(cache, who);
    CheckSeqs(seqs, who);
    if (HQ < 1 || HQ % c.heads != 0) throw std::runtime_error(std::string(who) + ": HQ must be a multiple of the cache's heads");
    *ws_bytes = 0;
}

void WeighLaunch(const WeighDesc &d, hipStream_t stream)
{
    const char *who = "attention_paged_weigh";
    const auto refuse = [&](const char *what) { throw std::runtime_error(std::string(who) + ": " + what); };
    const kr_cache c = CheckCache(d.cache, who);
    CheckSeqs(d.seqs, who);
    const kr_seqs &s = *d.seqs;
    size_t need = 0;
    WeighNeeds(d.cache, d.seqs, d.HQ, &need);
    const kr_weights w = CheckWeights(d.weights, c, who);
    if (d.layer < 0 || d.layer >= c.layers) refuse("no such layer");
    if (!(d.scale > 0.0f) || std::isinf(d.scale)) refuse("scale must be positive");
    if (!(d.decay >= 0.0f) || std::isinf(d.decay)) refuse("decay must not be negative");
    if (d.rows < 0 || d.last < 0) refuse("rows and last must not be negative");
    if ((d.path == nullptr) != (d.path_lens == nullptr)) refuse("a path needs its lengths");
    if (d.path != nullptr && (d.path_width < 1 || (s.seqs > 1 && d.ld_path < d.path_width)))
        refuse("path rows are empty or overlap");
    if (d.rows == 0 || s.seqs == 0 || s.max_new == 0) return;
    if (d.q == nullptr || d.lse == nullptr) refuse("q or lse is missing");
    if ((reinterpret_cast<uintptr_t>(d.q) & 15) != 0 || (reinterpret_cast<uintptr_t>(d.lse) & 3) != 0)
        refuse("q must be 16-byte aligned, lse 4-byte");
    if (need > 0 && (d.ws == nullptr || d.ws_bytes < need || (reinterpret_cast<uintptr_t>(d.ws) & 15) != 0))
        refuse("the workspace is too small or misaligned");
    WeighParams p{};
    p.ldq = d.ldq > 0 ? d.ldq : int64_t(d.HQ) * c.head_dim;
    p.ld_lse = d.ld_lse > 0 ? d.ld_lse : d.HQ;
    if (p.ldq % 8 != 0) refuse("row strides must be multiples of 8");
    if (d.rows > 1 && (p.ldq < int64_t(d.HQ) * c.head_dim || p.ld_lse < d.HQ)) refuse("rows overlap");
    const int64_t cap = int64_t(s.table_pages) * c.page_size;
    if (cap >= (int64_t(1) << 31) - 1024) refuse("the page table spans too many tokens");
    if (int64_t(d.rows) * d.HQ >= (int64_t(1) << 31)) refuse("too many rows for one launch");
    p.q = static_cast<const uint16_t *>(d.q);
    p.k = static_cast<const uint16_t *>(c.k) + d.layer * c.layer_stride;
    p.lse = d.lse;
    p.w = w.w + d.layer * w.layer_stride;
    p.table = s.table;
    p.lens = s.lens;
    p.starts = s.starts;
    p.entry = w.entry;
    p.path = d.path;
    p.path_lens = d.path_lens;
    p.tree = s.tree;
    p.ld_table = s.ld_table;
    p.ld_tree = s.ld_tree;
    p.ld_path = d.ld_path;
    p.head_stride = c.head_stride;
    p.w_entry = w.entry_stride;
    p.w_head = w.head_stride;
    p.page_stride = uint32_t(c.page_stride);
    p.token_stride = uint32_t(c.token_stride);
    p.cap = int(cap);
    p.pages = c.pages;
    p.table_pages = s.table_pages;
    p.seqs = s.seqs;
    p.rows = d.rows;
    p.max_new = s.max_new;
    p.tree_words = s.tree_words;
    p.HQ = d.HQ;
    p.HKV = c.heads;
    p.G = d.HQ / c.heads;
    p.entries = w.entries;
    p.width = w.width;
    p.path_width = d.path_width;
    p.last = d.last;
    p.scale_log2 = d.scale * 1.4426950408889634f;
    p.decay = d.decay;
    p.div = MakePageDiv(c.page_size);
    const int64_t most = (std::min<int64_t>(cap, w.width) + kWeighKeys - 1) / kWeighKeys * c.heads * s.seqs;
    if (most >= (int64_t(1) << 31)) refuse("too many keys for one launch");
    const MemSpan out = WeightsSpan(w);
    const RowSpan k = LayerSpan(c, c.k, d.layer);
    if (Meets(out, RowsSpan(d.q, d.rows, p.ldq, int64_t(d.HQ) * c.head_dim, 2)) ||
        Meets(out, RowsSpan(d.lse, d.rows, p.ld_lse, d.HQ, 4)) || Meets(out, MemSpan{k.p, k.width * 2}) ||
        Meets(out, MemSpan{d.ws, int64_t(need)}))
        refuse("the weights overlap another tensor of the call");
    const dim3 grid(unsigned(std::min<int64_t>(most, kWeighGroups)));
    const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p); };
    if (c.head_dim == 64) c.dtype == kBF16 ? go(WeighKernel<kBF16, 64>) : go(WeighKernel<kF16, 64>);
    else c.dtype == kBF16 ? go(WeighKernel<kBF16, 128>) : go(WeighKernel<kF16, 128>);
    Check(hipGetLastError(), "attention_paged_weigh launch");
}

}  // namespace kr
