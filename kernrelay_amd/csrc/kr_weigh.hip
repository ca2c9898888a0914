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
// The scores S = Q K^T of a wave, 32 rows by 32 keys at a time: lane l's key is
// l % 32, register v's row 8 (v / 4) + 4 (l / 32) + v % 4. A key's sum stays in its
// two lanes until the last row, in fp32; the two are added at the end. (Row tiles
// are added one after the other: the weights of the chunk below are off by 1.4e-7
// relatively, in the root mean square, those of a sum in 32 bits by halves 0.5e-7.)
//
// What bounds it, on an MI355X:
//   few rows a head (StepKernel): K, once, and the weights, there and back. 64
//     sequences of 2000..4000 tokens, 28 heads of 128 over 4, a new token each: 203
//     MB in 44 us, 4.6 TB/s (a large copy: 4.9).
//   many rows (WeighKernel): products and vector work, which hardly overlap. 2048
//     new tokens behind 8000, the same heads: 168 us, 0.79 PFLOP/s; the matrix
//     cores are at work for 35% of the time, vector instructions for 57%. Without
//     the products it takes 129 us, without the exponentials 153, without the
//     rows' DMA 151, without reading the rows from LDS 163.
#include <algorithm>
#include <cmath>

#include "kr_attncore.h"
#include "kr_dma.h"
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
    int cap, pages, seqs, rows, max_new, tree_words, HQ, HKV, G;
    int entries, width, path_width, last;
    float scale_log2, decay;
    PageDiv div, group;  // by page_size, by G
    float *parts;        // [kWeighParts, 2, kWeighKeys]
};

constexpr float kLog2E = 1.4426950408889634f;

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

constexpr int kWeighKeys = 256;   // of a workgroup's tile: 64 a wave
constexpr int kWeighParts = 768;  // workgroups that share the line: three on each of 256 CUs (the chunk above,
                                  // early on: 512 238 us, 768 219, 1024 244)
constexpr int kWeighStages = 3;   // row tiles in LDS
constexpr int kWeighMasked = 1;   // quarters that a row tile counts for more where it needs masks (the chunk: 0 170.9
                                  // us, 1 167.5, 2 172.8; 512 tokens behind 40000: 190, 178.8, 178.7)

// Where in the line a workgroup stands: row tiles of the key tiles of all
// sequences, key head by key head. A key tile of new tokens begins with the
// first row tile that sees any of it: each of the `more` last ones has 8 G row
// tiles (its 256 tokens) less than the one before it.
struct WeighLine {
    int rt;           // row tiles of the sequence
    int full, more;   // key tiles of a key head with all row tiles, and the others
    int first, step;  // row tiles that the first of the others leaves out, and each after it more
    // The others' first `step` row tiles see a part of them, by masks, and count
    // for more than one: where a tile of so many row tiles ends in the line, and
    // the row tile that a place in it stands for.
    __device__ __forceinline__ int Places(int rows) const { return rows + min(rows, step) / 4 * kWeighMasked; }
    __device__ __forceinline__ int Row(int rows, int place) const
    {
        const int m = min(rows, step) / 4;
        return place < m * (4 + kWeighMasked) ? place * 4 / (4 + kWeighMasked) : place - m * kWeighMasked;
    }
    __device__ __forceinline__ WeighLine(const WeighParams &p, const WeighSeq &s)
    {
        const int tiles = (s.cols + kWeighKeys - 1) / kWeighKeys;
        rt = ((s.n - s.skip) * p.G + 31) / 32;
        full = tiles;
        if (p.tree == nullptr || p.path != nullptr) full = min(tiles, (s.len + s.skip) / kWeighKeys + 1);
        more = tiles - full;
        first = more > 0 ? (full * kWeighKeys - s.len - s.skip) * p.G / 32 : 0;
        step = 8 * p.G;
    }
    __device__ __forceinline__ int Head() const  // of a key head
    {
        // (of the others only the last can have fewer than `step`)
        const int few = more > 0 ? min(rt - first - step * (more - 1), step) / 4 : 0;
        return full * rt + more * (rt - first) - step * (more * (more - 1) / 2) +
               (max(more - 1, 0) * (step / 4) + few) * kWeighMasked;
    }
};

// A piece of a key tile: row tiles r_lo .. r_hi - 1.
struct WeighPiece {
    int b, h, t;
    int start, places;  // of the tile: where in the line it begins, and its places there
    int skip, rows;     // row tiles that it leaves out, and that it has
    bool masked;
};

// Position x of the line, in a sequence that begins at `base` of it.
__device__ __forceinline__ WeighPiece PieceAt(const WeighParams &p, const WeighLine &l, int b, int base, int x)
{
    WeighPiece w;
    const int head = l.Head();
    w.b = b;
    w.h = Uni((x - base) / head);
    int y = x - base - w.h * head;
    const int at = base + w.h * head;
    if (y < l.full * l.rt) {
        w.t = Uni(y / l.rt);
        w.start = at + w.t * l.rt;
        w.places = w.rows = l.rt;
        w.skip = 0;
        w.masked = false;
    } else {
        w.start = at + l.full * l.rt;
        w.t = l.full;
        w.skip = l.first;
        while (x >= w.start + l.Places(l.rt - w.skip)) {
            w.start += l.Places(l.rt - w.skip);
            w.skip += l.step;
            ++w.t;
        }
        w.rows = l.rt - w.skip;
        w.places = l.Places(w.rows);
        w.masked = true;
    }
    return w;
}

// All sequences' units one after the other, units(sequence) of each. Up to 64
// sequences are read once, one a lane, and looked up there.
constexpr int64_t kWeighLine = (int64_t(1) << 31) - 4096;
template <typename F>
struct WeighPlan {
    const WeighParams &p;
    const F units;
    const int lane;
    WeighSeq mine;
    int u, total;
    __device__ __forceinline__ int Units(const WeighSeq &s, int b) const { return b < p.seqs && s.cols > 0 ? units(s) : 0; }
    // Starts that ascend keep the total within what the host has checked; what is
    // longer all the same is not worked on.
    __device__ __forceinline__ WeighPlan(const WeighParams &p_, int lane_, F units_) : p(p_), units(units_), lane(lane_)
    {
        int64_t sum = 0;
        for (int b0 = 0; b0 < p.seqs; b0 += 64) {
            mine = LoadSeq(p, min(b0 + lane, p.seqs - 1));
            u = Units(mine, b0 + lane);
            uint32_t lo = uint32_t(u) & 0xffff, hi = uint32_t(u) >> 16;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                lo += uint32_t(__shfl_xor(int(lo), o, 64));
                hi += uint32_t(__shfl_xor(int(hi), o, 64));
            }
            sum += Uni(int(lo)) + (int64_t(Uni(int(hi))) << 16);
        }
        total = sum < kWeighLine ? int(sum) : 0;
    }
    // The sequence that holds unit x, which there is; `base`: the first of it.
    __device__ __forceinline__ int Find(int x, int &base, WeighSeq &s)
    {
        base = 0;
        for (int b0 = 0; b0 < p.seqs; b0 += 64) {
            if (p.seqs > 64) {
                mine = LoadSeq(p, min(b0 + lane, p.seqs - 1));
                u = Units(mine, b0 + lane);
            }
            const int incl = WaveScan(u, lane) + base;
            const uint64_t above = __ballot(incl > x);
            const int at = above != 0 ? __builtin_ctzll(above) : 63;
            base = Uni(__shfl(incl - (above != 0 ? u : 0), at, 64));
            if (above == 0) continue;
            const auto of = [&](int v) { return Uni(__shfl(v, at, 64)); };
            s = WeighSeq{of(mine.first), of(mine.rows), of(mine.n), of(mine.skip),
                         of(mine.len),   of(mine.total), of(mine.cols), of(mine.entry)};
            return b0 + at;
        }
        s = LoadSeq(p, 0);
        return 0;
    }
};

// A wave's own LDS writes before its other lanes' reads of them.
__device__ __forceinline__ void WaveLdsOrder()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A loaded value is needed here: the wait for it stands no further down.
__device__ __forceinline__ void Used(uint4 &x)
{
    typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
    U32x4 v = __builtin_bit_cast(U32x4, x);
    asm volatile("" : "+v"(v));
    x = __builtin_bit_cast(uint4, v);
}

// A key's sum to its column.
__device__ __forceinline__ void PutWeight(const WeighParams &p, const WeighSeq &s, int h, int key, float got)
{
    float *w = p.w + int64_t(s.entry) * p.w_entry + int64_t(h) * p.w_head + key;
    float old = 0.0f;
    if (key < s.len && p.decay != 0.0f) old = p.decay * *w;
    *w = old + got;
}

// Which of the 64 keys from nj on (as new tokens; negative: cached ones) row i of
// the sequence's new tokens sees: bit k for key nj + k. (Made once a row and tile,
// by the row's lane; looked up row by row and key by key the chunk above took 197
// us for 172, and 8 sequences of 1500 with trees of up to 60 drafts 44.7 for 30.7.)
template <bool PLAIN>
__device__ __forceinline__ uint64_t RowMask(const WeighParams &p, const WeighSeq &s, int b, int i, int nj, bool causal)
{
    if (!PLAIN && p.path != nullptr) {
        const int at = p.path[b * p.ld_path + i];
        if (at < 0 || at >= s.rows) return 0;
    }
    if (PLAIN || causal) {
        const int n = i - nj + 1;
        return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
    }
    const uint64_t *tree = p.tree + int64_t(s.first + i) * p.ld_tree;
    const auto word = [&](int w) { return w < 0 ? ~0ull : w < p.tree_words ? tree[w] : 0ull; };
    const int w = nj >> 6, by = nj & 63;
    const uint64_t lo = word(w);
    return by == 0 ? lo : (lo >> by) | (word(w + 1) << (64 - by));
}

// e where bit `key` of a row's mask is set, else 0, whatever e is.
__device__ __forceinline__ float Seen(float e, uint32_t mask, int key)
{
    return __uint_as_float(__float_as_uint(e) & uint32_t(__builtin_amdgcn_sbfe(int(mask), uint32_t(key), 1u)));
}

// PLAIN: causal, no path.
template <int DT, int D, bool PLAIN>
__global__ void __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2)))
WeighKernel(WeighParams p)
{
    constexpr int KB = 2;                 // 32-key blocks of a wave
    constexpr int NS = kWeighStages;
    constexpr int DCH = D / 8;            // 16-byte chunks per row
    constexpr int RPD = 64 / DCH;         // rows per 1 KB DMA block
    constexpr int DPW = 32 / RPD / 4;     // DMA blocks per wave and row tile
    __shared__ __attribute__((aligned(1024))) uint16_t qring[NS][32 * D];
    __shared__ __attribute__((aligned(256))) float lring[4][NS][64];  // a wave's own: lse of the tile's rows, twice
    __shared__ int64_t rows[4][32];                                  // and where its rows' queries are
    __shared__ __attribute__((aligned(16))) uint2 masks[4][32];      // and which of its keys they see
    const int lane = int(threadIdx.x) & 63, wave = Uni(int(threadIdx.x) >> 6);
    const int hf = lane >> 5;
    WeighPlan plan(p, lane, [&](const WeighSeq &s) { return p.HKV * WeighLine(p, s).Head(); });
    const int share = (plan.total + int(gridDim.x) - 1) / int(gridDim.x);
    int x = int(blockIdx.x) * share;
    const int x_end = min(x + share, plan.total);
    if (x >= x_end) return;
    int base;
    WeighSeq sq;
    int b = plan.Find(x, base, sq);
    WeighLine line(p, sq);
    const bool causal = PLAIN || p.tree == nullptr || p.path != nullptr;
    const int qaddr = (lane & 31) * D + KSlot<D>(lane & 31, hf) * 8;  // step dc: XOR 16 dc
    // 32 packed rows on: so many tokens and query heads
    const int step_tok = 32 / p.G, step_g = 32 - step_tok * p.G;
    const int64_t step_q = step_tok * p.ldq + step_g * D, step_qw = step_q + p.ldq - p.G * D;
    const int64_t step_l = step_tok * p.ld_lse + step_g, step_lw = step_l + p.ld_lse - p.G;
    while (x < x_end) {
        while (sq.cols == 0 || x >= base + p.HKV * line.Head()) {
            if (sq.cols > 0) base += p.HKV * line.Head();
            sq = LoadSeq(p, ++b);
            line = WeighLine(p, sq);
        }
        const WeighPiece pc = PieceAt(p, line, b, base, x);
        const int h = pc.h;
        const int y = x - pc.start, y_end = min(pc.places, x_end - pc.start);
        const int rt_lo = Uni(pc.skip + (pc.masked ? line.Row(pc.rows, y) : y));
        const int rt_hi = Uni(pc.skip + (pc.masked ? line.Row(pc.rows, y_end) : y_end));
        const int R = (sq.n - sq.skip) * p.G;
        const int j0 = Uni(pc.t * kWeighKeys + wave * (32 * KB));
        // ---- this wave's keys: lane l holds key l % 32 of each block, chunks of 8, every second one
        const uint16_t *kr[KB];
        uint32_t there = 0;  // bit kb: this lane's key is there
        bool all = true;     // so are all of the wave's
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int pos = j0 + kb * 32 + (lane & 31);
            const int pg = PageOf(p.div, min(pos, sq.total - 1));
            const int id = p.table[b * p.ld_table + pg];
            const bool ok = pos < sq.total && uint32_t(id) < uint32_t(p.pages);
            const int64_t off = ok ? int64_t(uint64_t(uint32_t(id)) * p.page_stride +
                                             uint64_t(uint32_t(pos - pg * p.div.size)) * p.token_stride)
                                   : 0;
            kr[kb] = p.k + h * p.head_stride + off + hf * 8;
            there |= ok ? 1u << kb : 0u;
            all = all && __ballot(!ok) == 0;
        }
        // packed row r of the unit, r = lane % 32 of a tile: where its query and lse
        // are; from tile to tile the addresses go on by as many tokens and heads
        int64_t qo = 0, lo = 0;  // elements
        int g = 0;
        bool out = false;  // of a path: does an entry of the tiles so far name no row?
        const auto point = [&](int r) {
            const int i = PageOf(p.group, r);
            g = r - i * p.G;
            int tok = sq.skip + i;
            if (!PLAIN && p.path != nullptr) {
                tok = p.path[b * p.ld_path + tok];
                const bool none = tok < 0 || tok >= sq.rows;
                out = out || __ballot(none) != 0;
                if (none) tok = 0;  // (counts nothing, see RowMask)
            }
            const int64_t row = sq.first + tok;
            qo = row * p.ldq + int64_t(h * p.G + g) * D;
            lo = row * p.ld_lse + h * p.G + g;
        };
        const auto fetch = [&](int st, int slot) {
            const int r0 = (rt_lo + st) * 32;
            if (!PLAIN || st == 0 || r0 + 32 > R) {
                point(min(r0 + (lane & 31), R - 1));
            } else {
                g += step_g;
                const bool wrap = g >= p.G;
                g -= wrap ? p.G : 0;
                qo += wrap ? step_qw : step_q;
                lo += wrap ? step_lw : step_l;
            }
            if (lane < 32) rows[wave][lane] = qo;
            WaveLdsOrder();
            const uint32_t dst = LdsAddr(&qring[slot][0]) + uint32_t(wave * DPW) * 1024u;
#pragma unroll
            for (int j = 0; j < DPW; ++j) {
                const int r = (wave * DPW + j) * RPD + lane / DCH;
                DmaLoad16(p.q + rows[wave][r] + KSlot<D>(r, lane % DCH) * 8, dst + uint32_t(j) * 1024u);
            }
            DmaTouch4(p.lse + lo, LdsAddr(&lring[wave][slot][0]));
        };
        const int ns = rt_hi - rt_lo;
        __syncthreads();  // (the rings are free)
        if (ns > 0) fetch(0, 0);
        if (ns > 1) fetch(1, 1);
        uint4 kf[KB][D / 16];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) kf[kb][dc] = *reinterpret_cast<const uint4 *>(kr[kb] + dc * 16);
        // (used here: a load that is still counted in the loop would have the compiler
        // wait there for everything in flight, the DMA of the tiles to come included)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) Used(kf[kb][dc]);
        float sum[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) sum[kb] = 0.0f;
        const int nj = j0 - sq.len;  // the first key as a new token
        static_assert(NS == 3, "slots");
        for (int st = 0, slot = 0; st < ns; ++st, slot = slot == NS - 1 ? 0 : slot + 1) {
            if (st + 1 < ns) KR_WAIT_VM(DPW + 1);
            else KR_WAIT_VM(0);
            __syncthreads();
            if (st + 2 < ns) fetch(st + 2, slot == 0 ? NS - 1 : slot - 1);
            const int r0 = (rt_lo + st) * 32;
            const uint16_t *Q = &qring[0][0] + slot * (32 * D);
            const float *ls = &lring[wave][0][0] + slot * 64;
            // rows that see nothing of the wave's keys, or all of them
            const int tok_lo = sq.skip + Uni(PageOf(p.group, r0));
            const int tok_hi = sq.skip + Uni(PageOf(p.group, min(r0 + 31, R - 1)));
            if (j0 >= sq.cols || (causal && nj > tok_hi)) continue;
            const bool dead = __ballot(ls[lane & 31] == -INFINITY) != 0;
            const bool whole = all && !dead && (PLAIN || !out) && r0 + 32 <= R &&
                               nj + 32 * KB <= (causal ? tok_lo + 1 : 0);
            if (!whole) {
                // a row's keys as 64 bits, made by the lane of that row
                const int rl = lane & 31, i32 = sq.skip + PageOf(p.group, min(r0 + rl, R - 1));
                const uint64_t m = r0 + rl < R && ls[rl] != -INFINITY ? RowMask<PLAIN>(p, sq, b, i32, nj, causal) : 0;
                if (lane < 32) masks[wave][lane] = make_uint2(uint32_t(m), uint32_t(m >> 32));
            }
            f32x16 s[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int v = 0; v < 16; ++v) s[kb][v] = 0.0f;
            {
                // the Q fragment of step dc is read QAH steps ahead of its MFMAs (of the
                // chunk above: 2 207 us, 4 204.7)
                constexpr int NP = D / 16, QAH = 4;
                uint4 qf[NP];
                const auto rd = [&](int dc) { qf[dc] = *reinterpret_cast<const uint4 *>(Q + (qaddr ^ (dc * 16))); };
#pragma unroll
                for (int dc = 0; dc < QAH; ++dc) rd(dc);
#pragma unroll
                for (int dc = 0; dc < NP; ++dc) {
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) s[kb] = Mfma<DT>(qf[dc], kf[kb][dc], s[kb]);
                    if (dc + QAH < NP) rd(dc + QAH);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, QAH, 0);  // 0x100 LDS read, 0x008 MFMA
#pragma unroll
                for (int i = 0; i < NP - QAH; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, KB, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, KB * QAH, 0);
            }
            // register v: row 8 (v / 4) + 4 hf + v % 4. The wave in its
            // exponentials goes first, as in the attention's kernels (without: 216 us
            // for 205).
            __builtin_amdgcn_s_setprio(2);
            if (whole) {
#pragma unroll
                for (int v4 = 0; v4 < 4; ++v4) {
                    const float4 l4 = *reinterpret_cast<const float4 *>(ls + 8 * v4 + 4 * hf);
                    const float nl[4] = {l4.x * -kLog2E, l4.y * -kLog2E, l4.z * -kLog2E, l4.w * -kLog2E};
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][4 * v4 + i], p.scale_log2, nl[i]));
                        sum[kb] += (e[0] + e[1]) + (e[2] + e[3]);
                    }
                }
            } else {
                WaveLdsOrder();
#pragma unroll
                for (int v4 = 0; v4 < 4; ++v4) {
                    const float4 l4 = *reinterpret_cast<const float4 *>(ls + 8 * v4 + 4 * hf);
                    const uint4 m01 = *reinterpret_cast<const uint4 *>(&masks[wave][8 * v4 + 4 * hf]);
                    const uint4 m23 = *reinterpret_cast<const uint4 *>(&masks[wave][8 * v4 + 4 * hf + 2]);
                    const float nl[4] = {l4.x * -kLog2E, l4.y * -kLog2E, l4.z * -kLog2E, l4.w * -kLog2E};
                    const uint32_t mm[4][KB] = {{m01.x, m01.y}, {m01.z, m01.w}, {m23.x, m23.y}, {m23.z, m23.w}};
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][4 * v4 + i], p.scale_log2, nl[i]));
                            e[i] = Seen(e[i], mm[i][kb], lane & 31);
                        }
                        const float of4 = (e[0] + e[1]) + (e[2] + e[3]);
                        sum[kb] += ((there >> kb) & 1) != 0 ? of4 : 0.0f;
                    }
                }
                WaveLdsOrder();
            }
            __builtin_amdgcn_s_setprio(0);
        }
        // ---- the two halves of a key's rows, and where its sum goes
        const bool cut = y > 0 || y_end < pc.places;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const float got = sum[kb] + __shfl_xor(sum[kb], 32, 64);
            const int key = j0 + kb * 32 + (lane & 31);
            if (hf != 0) continue;
            if (cut) p.parts[(2 * int(blockIdx.x) + (x > pc.start ? 0 : 1)) * kWeighKeys + wave * 32 * KB + kb * 32 + lane] = got;
            else if (key < sq.cols) PutWeight(p, sq, h, key, got);
        }
        x = pc.start + y_end;
    }
}

// ------------------------------------------------------- at most 32 rows a head
// A wave has a run of 32-key blocks, key head by key head. Keys go HBM -> LDS by
// the DMA, whole rows side by side, a lane for each 16 bytes of a row, a ring of
// kStepStages blocks for each wave, and nobody waits for another wave. The old
// weights come the same way, so that the loop holds no load that the compiler
// would wait for. Up to kStepRun blocks of a key head make a run, whose page ids
// are read at its start. (The step above, 203 MB: WeighKernel, whose loads go
// straight to the product's registers, 32 rows at a time, 53.4 us; this one 45,
// now 44.)
constexpr int kStepStages = 2;     // (45.0 us; 3 46.2, 4 47.3)
constexpr int kStepRun = 16;       // blocks (8 44.7 us, 16 45.0; 16 read the page table half as often)
constexpr int kStepGroups = 512;   // workgroups of four waves: two on each of 256 CUs (1024 46.3 us, 2048 50.8)

template <int DT, int D, bool PLAIN>
__global__ void __launch_bounds__(256) StepKernel(WeighParams p)
{
    constexpr int NS = kStepStages;
    constexpr int DCH = D / 8;       // 16-byte chunks per row
    constexpr int RPD = 64 / DCH;    // rows per 1 KB DMA block
    constexpr int NDMA = 32 / RPD;   // DMA blocks of a stage
    constexpr int VM = NDMA + 1;     // DMA instructions of a stage
    __shared__ __attribute__((aligned(1024))) uint16_t ring[4][NS][32 * D];
    __shared__ __attribute__((aligned(256))) float wring[4][NS][64];
    __shared__ int64_t offs[4][32];
    __shared__ __attribute__((aligned(16))) uint32_t masks[4][32];  // which keys of the block a row sees
    __shared__ int32_t tab[4][kStepRun * 32];
    const int lane = int(threadIdx.x) & 63, wave = Uni(int(threadIdx.x) >> 6);
    const int hf = lane >> 5, l32 = lane & 31;
    const auto blocks_of = [&](const WeighSeq &s) { return (s.cols + 31) / 32; };
    WeighPlan plan(p, lane, [&](const WeighSeq &s) { return p.HKV * blocks_of(s); });
    const int waves = 4 * int(gridDim.x), share = (plan.total + waves - 1) / waves;
    int x = (4 * int(blockIdx.x) + wave) * share;
    const int x_end = min(x + share, plan.total);
    if (x >= x_end) return;
    int base;
    WeighSeq sq;
    int b = plan.Find(x, base, sq);
    const bool causal = PLAIN || p.tree == nullptr || p.path != nullptr;
    const int kaddr = l32 * D + KSlot<D>(l32, hf) * 8;  // step dc: XOR 16 dc
    while (x < x_end) {
        while (x >= base + p.HKV * blocks_of(sq)) {
            base += p.HKV * blocks_of(sq);
            sq = LoadSeq(p, ++b);
        }
        // ---- a run: blocks t0 .. t0 + ns - 1 of key head h
        const int per = blocks_of(sq);
        const int h = Uni((x - base) / per), t0 = x - base - h * per;
        const int ns = Uni(min(min(per - t0, x_end - x), kStepRun));
        const int pg0 = Uni(PageOf(p.div, t0 * 32));
        const int npg = Uni(PageOf(p.div, min((t0 + ns) * 32, sq.total) - 1)) - pg0 + 1;
        for (int i = lane; i < npg; i += 64) tab[wave][i] = p.table[b * p.ld_table + pg0 + i];
        // rows: lane l has row l % 32, registers v row 8 (v / 4) + 4 hf + v % 4
        const int R = (sq.n - sq.skip) * p.G;
        const int i32 = sq.skip + PageOf(p.group, min(l32, R - 1));  // new token of row l % 32
        const int g = min(l32, R - 1) - (i32 - sq.skip) * p.G;
        int tok = i32;
        if (!PLAIN && p.path != nullptr) tok = p.path[b * p.ld_path + i32];
        const bool live = l32 < R && tok >= 0 && tok < sq.rows;
        const int64_t row = sq.first + (live ? tok : 0);
        uint4 qf[D / 16];
        {
            const uint16_t *q = p.q + row * p.ldq + int64_t(h * p.G + g) * D + hf * 8;
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) qf[dc] = *reinterpret_cast<const uint4 *>(q + dc * 16);
        }
        const float lse = live ? p.lse[row * p.ld_lse + h * p.G + g] : -INFINITY;
        const uint32_t counts = uint32_t(__ballot(lse != -INFINITY));  // rows that count
        float nl[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) nl[v] = __shfl(lse == -INFINITY ? -INFINITY : lse * -kLog2E, 8 * (v >> 2) + 4 * hf + (v & 3), 64);
#pragma unroll
        for (int dc = 0; dc < D / 16; ++dc) Used(qf[dc]);
        const uint16_t *kh = p.k + h * p.head_stride;
        float *wh = p.w + int64_t(sq.entry) * p.w_entry + int64_t(h) * p.w_head;
        KR_WAIT_VM(0);
        WaveLdsOrder();
        uint32_t there[NS];  // keys that are there: of the stage worked on and those in flight
        const auto fetch = [&](int st) -> uint32_t {
            const int pos = (t0 + st) * 32 + l32;
            const int pg = PageOf(p.div, min(pos, sq.total - 1));
            const int id = tab[wave][pg - pg0];
            const bool ok = pos < sq.total && uint32_t(id) < uint32_t(p.pages);
            const int64_t off = int64_t(uint64_t(uint32_t(id)) * p.page_stride +
                                        uint64_t(uint32_t(pos - pg * p.div.size)) * p.token_stride);
            offs[wave][l32] = ok ? off : 0;
            WaveLdsOrder();
            const uint32_t dst = LdsAddr(&ring[wave][st % NS][0]);
#pragma unroll
            for (int j = 0; j < NDMA; ++j) {
                const int r = j * RPD + lane / DCH;
                DmaLoad16(kh + offs[wave][r] + KSlot<D>(r, lane % DCH) * 8, dst + uint32_t(j) * 1024u);
            }
            DmaTouch4(wh + min(pos, sq.cols - 1), LdsAddr(&wring[wave][st % NS][0]));
            return uint32_t(__ballot(ok));
        };
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) there[i] = i < ns ? fetch(i) : 0u;
        for (int st = 0; st < ns; ++st) {
            if (st + NS - 1 < ns) {
                there[NS - 1] = fetch(st + NS - 1);
                KR_WAIT_VM((NS - 1) * VM);
            } else {
                KR_WAIT_VM(0);  // (the last stages of a run)
            }
            const uint16_t *K = &ring[wave][st % NS][0];
            const int j0 = (t0 + st) * 32, nj = j0 - sq.len;  // the first key, and as a new token
            f32x16 s;
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc)
                s = Mfma<DT>(qf[dc], *reinterpret_cast<const uint4 *>(K + (kaddr ^ (dc * 16))), s);
            const bool ok = ((there[0] >> l32) & 1) != 0;
            // do all rows count, and see every key? (Those past the last repeat it with weight 0.)
            const bool whole = there[0] == ~0u && nj + 32 <= (causal ? sq.skip + 1 : 0) && counts == (~0u >> (32 - min(R, 32)));
            if (!whole) {
                WaveLdsOrder();
                const uint32_t m = ((counts >> l32) & 1) != 0 ? uint32_t(RowMask<PLAIN>(p, sq, b, i32, nj, causal)) : 0u;
                if (lane < 32) masks[wave][lane] = m;
                WaveLdsOrder();
            }
            float sum = 0.0f;
#pragma unroll
            for (int v4 = 0; v4 < 4; ++v4) {
                if (8 * v4 >= R) break;
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * v4 + i], p.scale_log2, nl[4 * v4 + i]));
                if (!whole) {
                    const uint4 m = *reinterpret_cast<const uint4 *>(&masks[wave][8 * v4 + 4 * hf]);
                    const uint32_t mm[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = ok ? Seen(e[i], mm[i], l32) : 0.0f;
                }
                sum += (e[0] + e[1]) + (e[2] + e[3]);
            }
            sum += __shfl_xor(sum, 32, 64);
            const int key = j0 + l32;
            const float old = wring[wave][st % NS][lane];
            if (hf == 0 && key < sq.cols) wh[key] = (key < sq.len && p.decay != 0.0f ? p.decay * old : 0.0f) + sum;
#pragma unroll
            for (int i = 0; i + 1 < NS; ++i) there[i] = there[i + 1];
        }
        x += ns;
    }
}

// Tiles that came in pieces: workgroup i has the one that begins in part i and
// ends in a later one, slot 1 of that part and slot 0 of the next.
__global__ void __launch_bounds__(kWeighKeys) WeighJoinKernel(WeighParams p)
{
    const int lane = int(threadIdx.x) & 63;
    WeighPlan plan(p, lane, [&](const WeighSeq &s) { return p.HKV * WeighLine(p, s).Head(); });
    const int share = (plan.total + int(gridDim.x) - 1) / int(gridDim.x);
    const int x0 = int(blockIdx.x) * share, x1 = x0 + share;
    if (x1 >= plan.total) return;
    int base;
    WeighSeq sq;
    const int b = plan.Find(x1 - 1, base, sq);
    const WeighPiece pc = PieceAt(p, WeighLine(p, sq), b, base, x1 - 1);
    const int end = pc.start + pc.places;
    if (pc.start < x0 || end <= x1) return;
    const int key = pc.t * kWeighKeys + int(threadIdx.x);
    if (key >= sq.cols) return;
    float got = p.parts[(2 * int(blockIdx.x) + 1) * kWeighKeys + int(threadIdx.x)];
    const int last = (end - 1) / share;
    for (int i = int(blockIdx.x) + 1; i <= last; ++i) got += p.parts[2 * i * kWeighKeys + int(threadIdx.x)];
    PutWeight(p, sq, pc.h, key, got);
}

// Is every tile one row tile? Then none is cut, there is nothing to join, and a
// wave that holds all rows need not share them: StepKernel.
bool OneRowTile(int64_t tokens, int G) { return tokens * G <= 32; }

}  // namespace

void WeighNeeds(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes)
{
    const char *who = "attention_paged_weigh";
    const kr_cache c = CheckCache(cache, who);
    CheckSeqs(seqs, who);
    if (HQ < 1 || HQ % c.heads != 0) throw std::runtime_error(std::string(who) + ": HQ must be a multiple of the cache's heads");
    *ws_bytes = OneRowTile(seqs->max_new, HQ / c.heads) ? 0 : size_t(kWeighParts) * 2 * kWeighKeys * sizeof(float);
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
    p.group = MakePageDiv(p.G);
    p.parts = static_cast<float *>(d.ws);
    // the line: at most so many row tiles
    int64_t tokens = s.max_new;
    if (d.path != nullptr) tokens = std::min<int64_t>(tokens, d.path_width);
    if (d.last > 0) tokens = std::min<int64_t>(tokens, d.last);
    const int64_t tiles = (std::min<int64_t>(cap, w.width) + kWeighKeys - 1) / kWeighKeys;
    // (of all sequences together: no more than the rows fill, and one that is not full for each)
    const int64_t row_tiles = std::min((tokens * p.G + 31) / 32 * s.seqs, int64_t(d.rows) * p.G / 32 + s.seqs);
    if (tiles * c.heads >= kWeighLine / (row_tiles + row_tiles * kWeighMasked / 4) || 8 * tiles * c.heads >= kWeighLine / s.seqs)
        refuse("too many rows and keys for one launch");
    const RowSpan k = LayerSpan(c, c.k, d.layer);
    const MemSpan weights_span = WeightsSpan(w), ws{d.ws, int64_t(need)};
    const MemSpan ins[] = {RowsSpan(d.q, d.rows, p.ldq, int64_t(d.HQ) * c.head_dim, 2),
                           RowsSpan(d.lse, d.rows, p.ld_lse, d.HQ, 4), MemSpan{k.p, k.width * 2},
                           RowsSpan(w.entry, 1, 0, s.seqs, 4), RowsSpan(d.path, s.seqs, d.ld_path, d.path_width, 4),
                           RowsSpan(d.path_lens, 1, 0, s.seqs, 4)};
    if (Meets(weights_span, ws)) refuse("the weights and the workspace overlap");
    for (const MemSpan &in : ins) {
        if (Meets(weights_span, in)) refuse("the weights overlap another tensor of the call");
        if (Meets(ws, in)) refuse("the workspace overlaps another tensor of the call");
    }
    if (MeetsSeqs(weights_span, s, d.rows) || MeetsSeqs(ws, s, d.rows))
        refuse("the weights or the workspace overlap the sequences' arrays");
    if (OneRowTile(tokens, p.G)) {
        const int64_t blocks = (std::min<int64_t>(cap, w.width) + 31) / 32 * c.heads * s.seqs;
        const dim3 grid(unsigned(std::min<int64_t>((blocks + 3) / 4, kStepGroups)));
        const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p); };
        const bool bf = c.dtype == kBF16;
        if (s.tree == nullptr && d.path == nullptr) {
            if (c.head_dim == 64) bf ? go(StepKernel<kBF16, 64, true>) : go(StepKernel<kF16, 64, true>);
            else bf ? go(StepKernel<kBF16, 128, true>) : go(StepKernel<kF16, 128, true>);
        } else {
            if (c.head_dim == 64) bf ? go(StepKernel<kBF16, 64, false>) : go(StepKernel<kF16, 64, false>);
            else bf ? go(StepKernel<kBF16, 128, false>) : go(StepKernel<kF16, 128, false>);
        }
        Check(hipGetLastError(), "attention_paged_weigh launch");
        return;
    }
    const dim3 grid(kWeighParts);
    const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p); };
    const bool bf = c.dtype == kBF16;
    if (s.tree == nullptr && d.path == nullptr) {
        if (c.head_dim == 64) bf ? go(WeighKernel<kBF16, 64, true>) : go(WeighKernel<kF16, 64, true>);
        else bf ? go(WeighKernel<kBF16, 128, true>) : go(WeighKernel<kF16, 128, true>);
    } else {
        if (c.head_dim == 64) bf ? go(WeighKernel<kBF16, 64, false>) : go(WeighKernel<kF16, 64, false>);
        else bf ? go(WeighKernel<kBF16, 128, false>) : go(WeighKernel<kF16, 128, false>);
    }
    hipLaunchKernelGGL(WeighJoinKernel, grid, dim3(kWeighKeys), 0, stream, p);
    Check(hipGetLastError(), "attention_paged_weigh launch");
}

}  // namespace kr
