// Attention of new tokens over a paged key/value cache: one token, a tree of
// drafts, or a causal chunk per sequence. See kr_op_attention_paged. No
// counterpart in the reference, whose path ends with the prompt.
//
// Row i (a new token and a query head) of a sequence with L cached tokens:
//   o = sum_j exp(s q.k_j - m) v_j / sum_j exp(s q.k_j - m), j over the
//   positions it sees: j < L, and new tokens by the causal order or the tree.
//
// What bounds it: every visible key and value is read once, 4 D bytes a
// position and key head, against 4 D flops for each of the rows that share
// the head (new tokens x G query heads): HBM up to about a hundred rows, the
// matrix cores and the softmax's VALU work above. Measured (head size 128): 64
// single tokens over 2000 to 4000, 4 key heads, 394 MB in 87 us; one over
// 120001, 8 key heads, 492 MB in 100; 2048 tokens of a prompt over 8000, 28 query
// heads, 265 GFLOP in 295 to 317 (cards differ; 0.84 to 0.9 PFLOP/s). There the
// matrix cores are 44% busy: every K and V fragment is read from LDS for one
// MFMA, which at their full rate would take the whole of the LDS's (128 B a
// cycle).
// Each kernel spills 78 to 94 scalars into vector lanes, a dozen of which are
// read back in a stage.
//
// A unit of work is one key head of one sequence and RT = 32 QW packed rows
// (row r = new token r / G, query head r % G of the key head's G), so the
// heads that share keys share their read. A workgroup has QW x KW waves: QW
// of 32 rows each over the same keys, times KW key streams that take the
// 32 KB-key blocks of the unit in turn and are merged at its end.
//
// Keys and values go HBM -> LDS by the direct-to-LDS DMA into a ring of NS
// stages, each lane fetching 16 bytes of a row wherever the page table puts it.
// The table's entries travel the same way, further ahead (so nothing in the
// loop waits for a dependent load), and each wave turns a stage's into row
// offsets: lane l's key is l, its validity a ballot. A position past the
// sequence's end or on a page that is none is fetched from the cache's first
// row instead and seen by nobody.
// The products are those of the prompt's kernel (kr_attn.hip): S^T = K Q^T,
// softmax in base 2 with a lazily moved maximum, O^T += V^T P^T, fp32 state;
// P goes to the matrix cores in 16 bits, its sum is of the unrounded. Up to 32
// rows, where they have time to spare, it goes in two parts, the second what
// the first left over: a result is rounded once, at its store. Above, in one,
// which moves a result by at most half a step of sum p |v|, about what its own
// rounding does. Measured, one part / two, in us: 64 single tokens over 2000 to
// 4000, head size 128, 4 key heads, 86.7 / 87.1; one over 120001, 8 key heads,
// 103.4 / 103.7; head size 64, 2 key heads: 64 over 2000 to 4000 29.2 / 30.4, 64
// over 250 to 500 13.7 / 14.7; but two row blocks (8 trees of 16 over 2900, 8
// key heads) 33.6 / 35.4, and four (2048 rows of a prompt over 8000, 4 heads of
// 7) 317 / 405.
// fp16 weights carry a factor 2^7 through the sums.
// A block in which some row does not see some key goes the careful way: the
// scores are masked by 64 bits a row; value rows that are not there or hold a
// number that is not finite are zeroed in LDS (0 x NaN would reach everybody),
// and the latter added on the VALU to the rows that see them.
#include <algorithm>
#include <cmath>

#include "kr_attncore.h"
#include "kr_dma.h"
#include "kr_paged.h"
#include "kr_rowcore.h"

namespace kr {

namespace {

// What the second launch needs of a unit that came in pieces: they are slot 1
// of workgroup `part` and slot 0 of the next pieces - 1 ones.
struct PagedJoin {
    int32_t pieces, part;     // at most one: nothing to do
    int32_t first, r0, nrow;  // the sequence's first row; the unit's rows of it
    int32_t head;             // first query head
    int32_t pad[2];
};

struct PagedParams {
    const uint16_t *q, *k, *v;
    uint16_t *o;
    const int32_t *table, *lens, *starts;
    const uint64_t *tree;
    int64_t ldq, ldo, ld_table, ld_tree;
    int64_t head_stride;
    uint32_t page_stride, token_stride;
    int cap, pages, table_pages, seqs, rows, max_new, tree_words, HQ, HKV, G;
    float scale_log2;
    PageDiv div;
    int32_t *cnt;      // [max_units] arrival tickets, zero between launches; or NULL: a second launch sums
    float *ws;         // two partial slots per workgroup of the cut schedule
    PagedJoin *joins;  // [max_units], unit by unit as they come in the line; or NULL: tickets
    int max_units;
    int min_piece;     // stages of a piece, unless the units are shorter
    int slots;         // workgroups of the cut schedule; 0: whole units only
    float *lse;        // the rows' logarithms of sums [rows, HQ] (the kernels with LSE)
    int64_t ld_lse;
};

typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));

// A sequence as the launch has it, every number within its bounds whatever
// the device arrays hold.
struct PagedSeq {
    int first, n, len, total;  // first row, new tokens, cached tokens, keys
};

__device__ __forceinline__ PagedSeq LoadSeq(const PagedParams &p, int b)
{
    PagedSeq s;
    s.first = min(max(p.starts[b], 0), p.rows);
    s.n = min(min(max(p.starts[b + 1], s.first), p.rows) - s.first, p.max_new);
    s.len = max(p.lens[b], 0);
    s.total = int(min(int64_t(s.len) + s.n, int64_t(p.cap)));
    s.len = min(s.len, p.cap);
    return s;
}

// A wave's own LDS writes before its other lanes' reads of them.
__device__ __forceinline__ void WaveLdsOrder()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 8 bytes at byte offset `off` of a wave-uniform base, at device scope (as
// LoadU128Dev).
__device__ __forceinline__ uint2 LoadU64Dev(const void *base, int off)
{
    typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), short(0), 0x7fffffff, 0x00020000);
    const U32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 16 /* sc1 */);
    return make_uint2(v.x, v.y);
}

// A weight in two parts: the first its leading bits, the second what they left
// over and a little more (2^-23 of it; fp16: 2^-24, the smallest there is, as
// weights go to 2^7 and more), so that neither part of a weight that is not 0
// is 0 or negative: an infinite value times them is itself, and no NaN.
template <int DT>
__device__ __forceinline__ uint32_t Pack2Down(float lo, float hi)
{
    if constexpr (DT == kBF16) return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
}

template <int DT>
__device__ __forceinline__ float PartLeft(float p, float first)
{
    if constexpr (DT == kBF16) return __builtin_fmaf(p, 1.0f + 0x1p-23f, -first);
    else return (p - first) + fminf(p, 0x1p-24f);
}

// Any 16-bit value of the eight that is an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool AnyNonFinite(const uint4 &x)
{
    constexpr uint32_t E = DT == kBF16 ? 0x7f80u : 0x7c00u;
    bool bad = false;
    for (const uint32_t w : {x.x, x.y, x.z, x.w}) bad = bad || (w & E) == E || ((w >> 16) & E) == E;
    return bad;
}

// Sums pieces lo .. hi - 1 of a unit whose first piece is slot 1 of workgroup
// `part` (the others slot 0 of the next ones) for one chunk: 4 columns of a
// row, UN pieces in flight. DEV: written by workgroups of the running launch,
// so read at device scope.
struct PieceSum {
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
};

// Chunk ch of a unit's nrow rows: columns 4 cc.. of row ch % nrow, and where a
// slot has them: lane and store as d = cc / 8, g = cc / 2 % 4, half cc % 2.
template <int D> struct PieceChunk {
    int cc, row, at;
    __device__ __forceinline__ PieceChunk(int ch, int nrow)
    {
        cc = ch / nrow;
        row = ch - cc * nrow;
        at = ((row >> 5) * (D / 8) + (cc >> 1)) * 64 + (cc & 1) * 32 + (row & 31);
    }
};

template <int D, int QW, int UN, bool DEV>
__device__ __forceinline__ PieceSum SumPieces(const float *ws, int part, int lo, int hi, const PieceChunk<D> &c)
{
    constexpr int RT = 32 * QW, SLOT = RT * (D + 2);
    PieceSum s;
    for (int i0 = lo; i0 < hi; i0 += UN) {
        float ov[UN][4], mp[UN], lp[UN];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int pc = min(i0 + i, hi - 1);  // (past the end the last again, left out below)
            const float *slot = ws + int64_t(2 * (part + pc) + (pc == 0 ? 1 : 0)) * SLOT;
            uint4 o;
            uint2 ml;
            if constexpr (DEV) {
                o = LoadU128Dev(slot, c.at * 16);
                ml = LoadU64Dev(slot, (RT * D + 2 * c.row) * 4);
            } else {
                o = *reinterpret_cast<const uint4 *>(slot + c.at * 4);
                ml = *reinterpret_cast<const uint2 *>(slot + RT * D + 2 * c.row);
            }
            ov[i][0] = __uint_as_float(o.x);
            ov[i][1] = __uint_as_float(o.y);
            ov[i][2] = __uint_as_float(o.z);
            ov[i][3] = __uint_as_float(o.w);
            mp[i] = __uint_as_float(ml.x);
            lp[i] = __uint_as_float(ml.y);
        }
        float mn = s.m;
#pragma unroll
        for (int i = 0; i < UN; ++i) mn = __builtin_elementwise_maximum(mn, mp[i]);
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float a0 = __builtin_amdgcn_exp2f(s.m - ms);
        s.l *= a0;
#pragma unroll
        for (int e = 0; e < 4; ++e) s.acc[e] *= a0;
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const bool in = i0 + i < hi;
            const float a = __builtin_amdgcn_exp2f(mp[i] - ms);
            s.l = in ? __builtin_fmaf(lp[i], a, s.l) : s.l;
#pragma unroll
            for (int e = 0; e < 4; ++e) s.acc[e] = in ? __builtin_fmaf(ov[i][e], a, s.acc[e]) : s.acc[e];
        }
        s.m = mn;
    }
    return s;
}

// ln sum exp of a row from its base-2 maximum m and sum l.
template <int DT>
__device__ __forceinline__ float LseOf(float m, float l)
{
    // (fp16 weights carry 2^7: see the kernel)
    const float log2_sum = __builtin_amdgcn_logf(l) - (DT == kF16 ? 7.0f : 0.0f);
    return l == 0.0f ? -INFINITY : (m + log2_sum) * 0.6931471805599453f;
}

// A chunk's result to its row: row r of the unit's packed rows is new token
// r / G, query head `head` + r % G.
template <int DT>
__device__ __forceinline__ void StoreSum(const PieceSum &s, uint16_t *o, int64_t ldo, int first, int r, int head, int G,
                                         int D, int cc)
{
    const float inv = s.l == 0.0f ? 0.0f : 1.0f / s.l;
    const int tok = r / G;
    uint2 w;
    w.x = Pack2<DT>(s.acc[0] * inv, s.acc[1] * inv);
    w.y = Pack2<DT>(s.acc[2] * inv, s.acc[3] * inv);
    *reinterpret_cast<uint2 *>(o + int64_t(first + tok) * ldo + int64_t(head + r - tok * G) * D + cc * 4) = w;
}

template <int DT>
__device__ __forceinline__ void StoreLse(const PieceSum &s, float *lse, int64_t ld, int first, int r, int head, int G)
{
    const int tok = r / G;
    lse[int64_t(first + tok) * ld + head + r - tok * G] = LseOf<DT>(s.m, s.l);
}

// Workgroups of the cut schedule: two on each of 256 CUs (their rings fill 128
// of a CU's 160 KB at head size 128).
constexpr int kPagedSlots = 512;

// When units are cut. Whole, the launch lasts as long as its longest unit
// (`longest` stages of 64 keys; one workgroup alone on a CU has the CU's whole
// bandwidth and issue); cut, every workgroup has the same share, but a piece's
// rows are written and read once more (fp32), by a second launch of 6 to 18 us.
// So units are cut where the longest is more than a even shares and c stages.
// Measured, cut against whole, in us, at head size 128:
//   one row block: 1 sequence of 2000 tokens, 8 key heads: 14.5 / 46; 16 of up to
//   4000: 51 / 85; 64 of up to 500, 4 heads: 28 / 19; 64 of up to 1800, 8 heads:
//   86 / 79;
//   two: 8 trees of 16 over 3000, 8 heads: 34 / 52; 32: 91 / 82; 32 of 8 over
//   1000, 4 heads of 7: 30 / 24 (and cut, against the better);
//   four: 8 trees of 61 over 2900, 8 heads: 55 / 73; 16: 93 / 78; 1000 rows of a
//   prompt over 8000, 4 heads of 7: 169 / 185; 2048 rows: 330 / 309;
// and at 64, with 2 key heads of 7, where the shares are those of 128 though
// four workgroups would fit a CU:
//   one: 1 of 700: 14.4 / 15.2; 16 of up to 500: 14.4 / 12.7 (cut, against the
//   better); 1000: 14.8 / 19; 64 of up to 500: 14.8 / 13.2 (cut); 1800: 22 / 30;
//   128 of up to 4000: 53 / 48;
//   two: 8 trees of 9 over 800: 17 / 16 (cut); 3000: 19 / 40; 64: 30 / 40;
//   four: 8 trees of 61 over 1500: 25 / 31; 32 over 2900: 57 / 53 (cut); 2048
//   rows over 8000: 120 / 152; 2 of 1500 over 4000: 82 / 110 (whole).
template <int QW> struct CutRule {
    static constexpr float a = QW == 4 ? 2.0f : 2.6f;
    static constexpr int c = QW == 1 ? 6 : QW == 2 ? 8 : 16;
};

template <int DT, int D, int QW, int KW, int KB, int NS, bool LSE>
__global__ void __attribute__((amdgpu_flat_work_group_size(64 * QW * KW, 64 * QW * KW), amdgpu_waves_per_eu(2)))
PagedKernel(PagedParams p)
{
    static_assert(D == 64 || D == 128, "head_dim 64 or 128");
    constexpr int NW = QW * KW;
    constexpr int BLK = 32 * KB;            // keys of a stream's stage
    constexpr int SB = BLK * KW;            // keys of a workgroup's stage
    constexpr int RT = 32 * QW;             // rows of a unit
    constexpr int DCH = D / 8;              // 16-byte chunks per row
    constexpr int DBLK = D / 32;            // 32-wide d blocks of O^T
    constexpr int RPD = 64 / DCH;           // rows per 1 KB DMA block
    constexpr int DPW = BLK / RPD / QW;     // DMA blocks per wave, operand and stage
    constexpr int VAH = 4;                  // V fragments read ahead
    constexpr bool FINE = QW == 1;          // P in two parts (see the top)
    constexpr int VM = 2 * DPW + 1;         // DMA instructions of a wave's stage
    static_assert((NS - 1) * VM < 64, "vmcnt");
    static_assert(SB >= 64, "the host bounds the line by stages of 64 keys");
    constexpr uint64_t ALL = KB == 2 ? ~0ull : 0xffffffffull;
    __shared__ __attribute__((aligned(1024))) uint16_t kring[NS][KW][BLK * D];
    __shared__ __attribute__((aligned(1024))) uint16_t vring[NS][KW][BLK * D];
    __shared__ __attribute__((aligned(256))) int32_t tab[NW][NS][64];  // page ids of a stage's keys
    __shared__ int64_t offs[NW][64];                                  // and their rows' element offsets
    __shared__ uint64_t odd[NS][KW][QW];                               // keys whose values are not all finite
    __shared__ int last_piece;

    const int lane = int(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int wq = wave % QW, ks = wave / QW;  // row block, key stream
    const int hf = lane >> 5;

    // ---- which part of the work is this workgroup's
    // work of a sequence: its units (key heads x row blocks), each of `sb` stages
    const auto seq_units = [&](const PagedSeq &s) { return p.HKV * ((s.n * p.G + RT - 1) / RT); };
    const auto seq_stages = [&](const PagedSeq &s) { return (s.total + SB - 1) / SB; };
    int units = 0, stages = 0, longest = 0;
    PagedSeq mine{};  // lane's sequence of the first 64
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        int u = 0, w = 0, most = 0;
        if (b0 + lane < p.seqs) {
            const PagedSeq s = LoadSeq(p, b0 + lane);
            if (b0 == 0) mine = s;
            u = seq_units(s);
            most = u > 0 ? seq_stages(s) : 0;
            w = u * most;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            u += __shfl_xor(u, o, 64);
            w += __shfl_xor(w, o, 64);
            most = max(most, __shfl_xor(most, o, 64));
        }
        longest = max(longest, Uni(most));
        units += Uni(u);
        stages += Uni(w);
    }
    // sequence b, from the lane that has it
    const auto get_seq = [&](int b) {
        if (p.seqs > 64) return LoadSeq(p, b);
        PagedSeq s;
        s.first = __builtin_amdgcn_readlane(mine.first, b);
        s.n = __builtin_amdgcn_readlane(mine.n, b);
        s.len = __builtin_amdgcn_readlane(mine.len, b);
        s.total = __builtin_amdgcn_readlane(mine.total, b);
        return s;
    };
    // cut: `slots` workgroups share out the stages evenly, in one line through
    // all units; else a workgroup has one unit
    const bool cut = p.slots > 0 && float(longest) > CutRule<QW>::a * float(stages) / float(p.slots) +
                                                         float(CutRule<QW>::c * 64 / SB);
    int share = 1, parts = units;
    if (cut) {
        share = Uni(max((stages + p.slots - 1) / p.slots, min(p.min_piece, (stages + units - 1) / units)));
        parts = Uni((stages + share - 1) / share);
    }
    // notes past the units there are, by workgroups with a part of the line or
    // without: the workspace may hold anything, and the second launch reads
    // max_units notes (as many workgroups as there are at least)
    if (p.joins != nullptr && int(blockIdx.x) >= units && int(blockIdx.x) < p.max_units && threadIdx.x == 0)
        p.joins[blockIdx.x].pieces = 0;
    if (int(blockIdx.x) >= parts) return;
    const int part = XcdChunk(int(blockIdx.x), 0, parts);
    // this workgroup's stages (cut) or units, and the sequence that holds the
    // first: base <= x < base + its size, after `ubase` units
    int x = part * share, b = 0, base = 0, ubase = 0;
    const int x_end = cut ? min(x + share, stages) : x + 1;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        int u = 0, w = 0;
        if (b0 + lane < p.seqs) {
            const PagedSeq s = b0 == 0 ? mine : LoadSeq(p, b0 + lane);
            u = seq_units(s);
            w = u * (cut ? seq_stages(s) : 1);
        }
        const int incl = WaveScan(w, lane) + base, uincl = WaveScan(u, lane) + ubase;
        const uint64_t above = __ballot(incl > x);
        const int at = above != 0 ? __builtin_ctzll(above) : 63;
        base = Uni(__shfl(incl - (above != 0 ? w : 0), at, 64));
        ubase = Uni(__shfl(uincl - (above != 0 ? u : 0), at, 64));
        if (above != 0) {
            b = b0 + at;
            break;
        }
    }

    // fragment addresses (elements inside a K / V block), as in kr_attn.hip
    // (K's chunk 2 dc + hf of row lane % 32: the slot is an XOR, so step dc is
    // the first step's address XOR 16 dc)
    const int kaddr = (lane & 31) * D + KSlot<D>(lane & 31, hf) * 8;
    int vaddr[DBLK];
    {
        const int s16 = lane & 15, g1 = (lane >> 4) & 1, row = 4 * hf + (s16 >> 2);
#pragma unroll
        for (int d = 0; d < DBLK; ++d) {
            const int col = d * 32 + 16 * g1 + 4 * (s16 & 3);
            vaddr[d] = row * D + VSlot<D>(row, col / 8) * 8 + (col & 7);
        }
    }

    while (x < x_end) {
        // ---- one unit, or the part of it that is this workgroup's
        const PagedSeq sq = get_seq(b);
        const int qt = (sq.n * p.G + RT - 1) / RT;
        const int sb = seq_stages(sq);
        const int size = p.HKV * qt * (cut ? sb : 1);
        const int u = Uni(cut ? (x - base) / sb : x - base);
        const int s_lo = cut ? x - base - u * sb : 0;
        const int s_hi = cut ? min(sb, s_lo + (x_end - x)) : sb;
        const int h = Uni(u / qt), t = qt - 1 - (u - h * qt);  // a chunk's longest rows first
        const int unit0 = x - s_lo;  // the unit's first stage in the line
        const int first = cut ? Uni(unit0 / share) : 0;
        const int pieces = cut ? Uni((unit0 + sb - 1) / share) - first + 1 : 1;

        const int R = sq.n * p.G;
        const int r0 = t * RT;
        const int r = min(r0 + wq * 32 + (lane & 31), R - 1);  // (rows past the end repeat the last)
        const int tok = r / p.G;
        const bool live = r0 + wq * 32 < R;
        const int tok_lo = Uni(r0 / p.G);                              // of the unit
        const int wtok_hi = Uni(min(r0 + wq * 32 + 31, R - 1) / p.G);  // of this wave
        const int kend = p.tree != nullptr ? sq.total : min(sq.total, sq.len + Uni(min(r0 + RT - 1, R - 1) / p.G) + 1);
        const int ns = max(0, min(s_hi, (kend + SB - 1) / SB) - s_lo);
        const int32_t *table = p.table + b * p.ld_table;
        const uint16_t *kh0 = p.k + h * p.head_stride, *vh0 = p.v + h * p.head_stride;
        const uint64_t *tree = p.tree + (p.tree != nullptr ? int64_t(sq.first + tok) * p.ld_tree : 0);

        f32x16 oacc[DBLK];
#pragma unroll
        for (int d = 0; d < DBLK; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) oacc[d][v] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        // first key of stage st of this stream
        const auto key0 = [&](int st) { return ((s_lo + st) * KW + ks) * BLK; };
        // page ids of stage st's keys -> tab (one DMA instruction)
        const auto fetch_tab = [&](int st) {
            const int pg = min(PageOf(p.div, key0(st) + (lane & (BLK - 1))), p.table_pages - 1);
            DmaTouch4(table + pg, LdsAddr(&tab[wave][st % NS][0]));
        };
        // tab -> offs; returns which keys of stage st are there
        const auto rows_of = [&](int st) -> uint64_t {
            const int pos = key0(st) + (lane & (BLK - 1));
            const int id = tab[wave][st % NS][lane];
            const bool ok = pos < sq.total && uint32_t(id) < uint32_t(p.pages);
            const uint32_t in_page = uint32_t(pos - PageOf(p.div, pos) * p.div.size);
            const int64_t off = int64_t(uint64_t(uint32_t(id)) * p.page_stride + uint64_t(in_page) * p.token_stride);
            offs[wave][lane] = ok ? off : 0;
            WaveLdsOrder();
            return __ballot(ok) & ALL;
        };
        // keys and values of stage st -> ring (2 DPW DMA instructions)
        const auto fetch = [&](int st) {
            const uint32_t kdst = LdsAddr(&kring[st % NS][ks][0]) + uint32_t(wq * DPW) * 1024u;
            const uint32_t vdst = LdsAddr(&vring[st % NS][ks][0]) + uint32_t(wq * DPW) * 1024u;
#pragma unroll
            for (int j = 0; j < DPW; ++j) {
                const int row = (wq * DPW + j) * RPD + lane / DCH;
                const int64_t o = offs[wave][row];
                DmaLoad16(kh0 + o + KSlot<D>(row, lane % DCH) * 8, kdst + uint32_t(j) * 1024u);
                DmaLoad16(vh0 + o + VSlot<D>(row, lane % DCH) * 8, vdst + uint32_t(j) * 1024u);
            }
        };
        // does every row of the unit see every key of stage st
        const auto whole = [&](int st, uint64_t there) {
            return there == ALL && key0(st) + BLK <= (p.tree != nullptr ? sq.len : sq.len + tok_lo + 1);
        };
        // the values that this wave fetched for stage st: rows that are not
        // there or not all finite become 0; returns the latter
        const auto clean = [&](int st, uint64_t there) -> uint64_t {
            uint64_t bad = 0;
#pragma unroll 1
            for (int j = 0; j < DPW; ++j) {
                const int row = (wq * DPW + j) * RPD + lane / DCH;
                uint4 *a = reinterpret_cast<uint4 *>(&vring[st % NS][ks][(wq * DPW + j) * 512 + lane * 8]);
                const bool here = ((there >> row) & 1) != 0;
                uint64_t hit = __ballot(here && AnyNonFinite<DT>(*a));
                uint64_t odd_lanes = 0;
                while (hit != 0) {
                    const int g = __builtin_ctzll(hit) / DCH;
                    bad |= 1ull << ((wq * DPW + j) * RPD + g);
                    odd_lanes |= ((1ull << DCH) - 1) << (g * DCH);
                    hit &= ~odd_lanes;
                }
                if (!here || ((odd_lanes >> lane) & 1) != 0) *a = make_uint4(0, 0, 0, 0);
            }
            WaveLdsOrder();
            return bad;
        };
        // which keys of stage st this lane's row sees
        const auto seen = [&](int st, uint64_t there) -> uint64_t {
            const int j0 = key0(st) - sq.len;  // new token of the first key
            if (p.tree == nullptr) {
                const int nb = tok - j0 + 1;
                return there & (nb >= 64 ? ~0ull : nb <= 0 ? 0ull : (1ull << nb) - 1);
            }
            const auto word = [&](int i) { return i < p.tree_words ? tree[i] : 0ull; };
            uint64_t w;
            if (j0 >= 0) {
                const int sh = j0 & 63;
                w = word(j0 >> 6) >> sh;
                if (sh != 0) w |= word((j0 >> 6) + 1) << (64 - sh);
            } else {
                w = -j0 >= 64 ? ~0ull : ((1ull << -j0) - 1) | (word(0) << -j0);
            }
            return there & w;
        };

        // ---- the loop over stages: up to NS - 1 later ones are in flight while
        // one is worked; the page ids of a stage travel NS - 1 stages ahead of
        // its rows, so that they are older than every row still in flight
        uint4 qf[D / 16];
        {
            const uint16_t *qrow = p.q + int64_t(sq.first + tok) * p.ldq + int64_t(h * p.G + r - tok * p.G) * D;
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) qf[dc] = *reinterpret_cast<const uint4 *>(qrow + dc * 16 + hf * 8);
        }
        uint64_t there[NS];  // keys that are there: of the stage worked on and those in flight
#pragma unroll
        for (int i = 0; i < NS; ++i) there[i] = 0;
        if (ns > 0) {
#pragma unroll
            for (int i = 0; i < NS - 1; ++i) fetch_tab(i);
        }
        // q is used here, on every path: a load that the compiler still counts
        // in the loop would make it wait for the DMA there, stage by stage
#pragma unroll
        for (int dc = 0; dc < D / 16; ++dc) {
            U32x4 v = __builtin_bit_cast(U32x4, qf[dc]);
            asm volatile("" : "+v"(v));
            qf[dc] = __builtin_bit_cast(uint4, v);
        }
        KR_WAIT_VM(0);
        if (ns > 0) {
#pragma unroll
            for (int i = 0; i < NS - 1; ++i) {
                fetch_tab(NS - 1 + i);
                there[i] = rows_of(i);
                fetch(i);
            }
            if constexpr (QW > 1) {
                KR_WAIT_VM((NS - 2) * VM);
                if (!whole(0, there[0])) {
                    const uint64_t bad = clean(0, there[0]);
                    if (lane == 0) odd[0][ks][wq] = bad;
                }
                __syncthreads();
            }
        }
        for (int st = 0; st < ns; ++st) {
            // (past the last stage the fetches go on, into slots that nobody
            // reads: every stage issues the same count)
            fetch_tab(st + 2 * NS - 2);
            if constexpr (QW == 1) KR_WAIT_VM((NS - 1) * VM);  // the page ids of stage st + NS - 1
            there[NS - 1] = rows_of(st + NS - 1);
            fetch(st + NS - 1);
            if constexpr (QW == 1) KR_WAIT_VM((NS - 1) * VM);  // the rows of st
            const bool all = whole(st, there[0]);
            uint64_t bad = 0;
            if (!all) {
                if constexpr (QW == 1) {
                    bad = clean(st, there[0]);
                } else {
#pragma unroll
                    for (int i = 0; i < QW; ++i) bad |= odd[st % NS][ks][i];
                }
            }
            // skipped: no key is there, or all lie in this wave's future
            const bool future = p.tree == nullptr && key0(st) > sq.len + wtok_hi;
            if (live && there[0] != 0 && !future) {
                const uint16_t *K = &kring[st % NS][ks][0];
                const uint16_t *V = &vring[st % NS][ks][0];
                f32x16 sacc[KB];
#pragma unroll
                for (int kh = 0; kh < KB; ++kh)
#pragma unroll
                    for (int v = 0; v < 16; ++v) sacc[kh][v] = 0.0f;
                {
                    // the K fragments of step dc are read KAH steps ahead of
                    // their MFMAs, as in kr_attn.hip
                    constexpr int NP = D / 16, KAH = 3;
                    uint4 kf[KB][NP];
                    const auto rd = [&](int dc) {
#pragma unroll
                        for (int kh = 0; kh < KB; ++kh)
                            kf[kh][dc] = *reinterpret_cast<const uint4 *>(K + kh * 32 * D + (kaddr ^ (dc * 16)));
                    };
#pragma unroll
                    for (int dc = 0; dc < KAH; ++dc) rd(dc);
#pragma unroll
                    for (int dc = 0; dc < NP; ++dc) {
#pragma unroll
                        for (int kh = 0; kh < KB; ++kh) sacc[kh] = Mfma<DT>(kf[kh][dc], qf[dc], sacc[kh]);
                        if (dc + KAH < NP) rd(dc + KAH);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x100, KB * KAH, 0);  // 0x100 LDS read, 0x008 MFMA
#pragma unroll
                    for (int i = 0; i < NP - KAH; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, KB, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, KB, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x008, KB * KAH, 0);
                }
                // register v of half kh holds key kh*32 + 8 (v/4) + 4 hf + v%4
                uint64_t sees = ALL;
                if (!all) {
                    sees = seen(st, there[0]);
                    const uint64_t bits = sees >> (4 * hf);
                    const auto sees_key = [&](int i) { return ((uint32_t(bits >> (i & 32)) >> (i & 31)) & 1) != 0; };
#pragma unroll
                    for (int kh = 0; kh < KB; ++kh)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            sacc[kh][v] = sees_key(kh * 32 + 8 * (v >> 2) + (v & 3)) ? sacc[kh][v] : -INFINITY;
                }
                // two workgroups of four row blocks share a CU: the wave in its
                // softmax goes first (2048 rows over 8000: 311 -> 302 us), as
                // in kr_attn.hip
                if constexpr (QW == 4) __builtin_amdgcn_s_setprio(2);
                float mloc = sacc[0][0];
#pragma unroll
                for (int kh = 0; kh < KB; ++kh)
#pragma unroll
                    for (int v = 0; v < 16; ++v) mloc = __builtin_elementwise_maximum(mloc, sacc[kh][v]);
                {
                    const auto sw =
                        __builtin_amdgcn_permlane32_swap(__float_as_uint(mloc), __float_as_uint(mloc), false, false);
                    mloc = __builtin_elementwise_maximum(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * p.scale_log2;
                }
                // lazy maximum: moves only by more than 2^8 (kr_attn.hip); a
                // NaN moves it too, and stays
                const bool move = !(mloc <= m + 8.0f) && mloc != -INFINITY;
                const float mnew = move ? mloc : m;
                const float msub = mnew == -INFINITY ? 0.0f : mnew;
                const float alpha = move ? __builtin_amdgcn_exp2f(m - msub) : 1.0f;
                // fp16 holds its full precision down to 2^-14 only, and below
                // 2^-25 nothing: many small weights beside one of 1 would be
                // lost. So P is 2^7 2^(s - m): at most 2^15 with the lazy
                // maximum's 2^8, and full down to 2^-21; O and l both have the
                // factor, in every stream and piece, and lose it in O / l
                const float sub = DT == kF16 ? 7.0f - msub : -msub;
                uint4 pf[2 * KB], pl[FINE ? 2 * KB : 1];
                float ls[4];
#pragma unroll
                for (int c = 0; c < 2 * KB; ++c) {
                    const int kh = c >> 1, vb = (c & 1) * 8;
                    float pv[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[kh][vb + e], p.scale_log2, sub));
                        ls[e & 3] = c == 0 && e < 4 ? pv[e] : ls[e & 3] + pv[e];
                    }
                    if constexpr (FINE) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            hi[e] = Pack2Down<DT>(pv[2 * e], pv[2 * e + 1]);
                            lo[e] = Pack2<DT>(PartLeft<DT>(pv[2 * e], Elem<DT>::Load(uint16_t(hi[e]))),
                                              PartLeft<DT>(pv[2 * e + 1], Elem<DT>::Load(uint16_t(hi[e] >> 16))));
                        }
                        pf[c] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        pl[c] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    } else {
                        pf[c] = make_uint4(Pack2<DT>(pv[0], pv[1]), Pack2<DT>(pv[2], pv[3]), Pack2<DT>(pv[4], pv[5]),
                                           Pack2<DT>(pv[6], pv[7]));
                    }
                }
                l = l * alpha + ((ls[0] + ls[1]) + (ls[2] + ls[3]));
                m = mnew;
                if (__builtin_expect(__ballot(move) != 0, 0)) {
#pragma unroll
                    for (int d = 0; d < DBLK; ++d)
#pragma unroll
                        for (int v = 0; v < 16; ++v) oacc[d][v] *= alpha;
                }
                if constexpr (QW == 4) __builtin_amdgcn_s_setprio(0);
                {
                    // step i: 16 keys i / DBLK, d block i % DBLK; its V fragment
                    // is read VAH steps ahead of its MFMA
                    constexpr int NP = 2 * KB * DBLK;
                    const auto rd = [&](int i) {
                        const uint16_t *at = V + (i / DBLK) * 16 * D + vaddr[i % DBLK];
                        const AttnS4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(const_cast<uint16_t *>(at)));
                        const AttnS4 hi =
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(const_cast<uint16_t *>(at) + 8 * D));
                        const AttnU2 a = __builtin_bit_cast(AttnU2, lo), z = __builtin_bit_cast(AttnU2, hi);
                        return make_uint4(a.x, a.y, z.x, z.y);
                    };
                    uint4 vf[NP];
#pragma unroll
                    for (int i = 0; i < VAH; ++i) vf[i] = rd(i);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        oacc[i % DBLK] = Mfma<DT>(vf[i], pf[i / DBLK], oacc[i % DBLK]);
                        if (i + VAH < NP) vf[i + VAH] = rd(i + VAH);
                        if (FINE && i % DBLK == DBLK - 1) {
#pragma unroll
                            for (int d = 0; d < DBLK; ++d)
                                oacc[d] = Mfma<DT>(vf[i - DBLK + 1 + d], pl[FINE ? i / DBLK : 0], oacc[d]);
                        }
                    }
                    constexpr int PER = FINE ? 2 : 1;  // products of a fragment
                    __builtin_amdgcn_sched_group_barrier(0x100, 2 * VAH, 0);
#pragma unroll
                    for (int i = 0; i < NP - VAH; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x008, PER * VAH, 0);
                }
                // keys whose values are not all finite (zeroed in the ring):
                // added to the rows that see them, and to no others
                while (__builtin_expect(bad != 0, 0)) {
                    const int key = __builtin_ctzll(bad);
                    bad &= bad - 1;
                    // key 16 c + 8 e2 + 4 half + e: half word e % 2 of word 4 c + 2 e2 + e / 2 in that half's lanes
                    const int at = (key >> 4) * 4 + ((key >> 3) & 1) * 2 + ((key >> 1) & 1);
                    const auto weight = [&](const auto &pw) {
                        uint32_t w = 0;
#pragma unroll
                        for (int c = 0; c < 2 * KB; ++c) {
                            w = at == 4 * c ? pw[c].x : w;
                            w = at == 4 * c + 1 ? pw[c].y : w;
                            w = at == 4 * c + 2 ? pw[c].z : w;
                            w = at == 4 * c + 3 ? pw[c].w : w;
                        }
                        w = uint32_t(__shfl(int(w), (lane & 31) + 32 * ((key >> 2) & 1), 64));
                        return Elem<DT>::Load(uint16_t(w >> (16 * (key & 1))));
                    };
                    float pk = weight(pf);
                    if constexpr (FINE) pk += weight(pl);
                    const bool here = ((sees >> key) & 1) != 0;
                    const int pos = key0(st) + key, pg = PageOf(p.div, pos);
                    const uint16_t *row = vh0 + int64_t(uint64_t(uint32_t(table[pg])) * p.page_stride +
                                                        uint64_t(uint32_t(pos - pg * p.div.size)) * p.token_stride);
#pragma unroll
                    for (int d = 0; d < DBLK; ++d)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(row + d * 32 + 8 * g + 4 * hf);
                            const uint32_t half[4] = {x.x, x.x >> 16, x.y, x.y >> 16};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                oacc[d][4 * g + e] =
                                    here ? __builtin_fmaf(pk, Elem<DT>::Load(uint16_t(half[e])), oacc[d][4 * g + e])
                                         : oacc[d][4 * g + e];
                        }
                }
            }
#pragma unroll
            for (int i = 0; i + 1 < NS; ++i) there[i] = there[i + 1];
            if constexpr (QW > 1) {
                KR_WAIT_VM((NS - 2) * VM);  // this wave's part of stage st + 1 has landed
                if (st + 1 < ns && !whole(st + 1, there[0])) {
                    const uint64_t nf = clean(st + 1, there[0]);
                    if (lane == 0) odd[(st + 1) % NS][ks][wq] = nf;
                }
                __syncthreads();
            }
        }
        KR_WAIT_VM(0);  // (the fetches past the end too: the rings are used again)

        // ---- the key streams' states into stream 0's (through the rings)
        if constexpr (KW > 1) {
            constexpr int NE = DBLK * 16;
            static_assert((KW - 1) * QW * NE * 64 * 4 <= int(sizeof(kring)), "merge area");
            static_assert((KW - 1) * QW * 128 * 4 <= int(sizeof(vring)), "merge area");
            __syncthreads();
            float *og = reinterpret_cast<float *>(&kring[0][0][0]) + lane;
            float *mg = reinterpret_cast<float *>(&vring[0][0][0]) + lane;
            if (ks > 0) {
                const int at = (ks - 1) * QW + wq;
#pragma unroll
                for (int d = 0; d < DBLK; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) og[(at * NE + d * 16 + v) * 64] = oacc[d][v];
                mg[at * 128] = m;
                mg[at * 128 + 64] = l;
            }
            __syncthreads();
            if (ks == 0) {
#pragma unroll
                for (int o = 0; o < KW - 1; ++o) {
                    const int at = o * QW + wq;
                    const float m1 = mg[at * 128], l1 = mg[at * 128 + 64];
                    const float mn = __builtin_elementwise_maximum(m, m1);
                    const float ms = mn == -INFINITY ? 0.0f : mn;
                    const float a0 = __builtin_amdgcn_exp2f(m - ms), a1 = __builtin_amdgcn_exp2f(m1 - ms);
                    l = __builtin_fmaf(l1, a1, l * a0);
#pragma unroll
                    for (int d = 0; d < DBLK; ++d)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            oacc[d][v] = __builtin_fmaf(og[(at * NE + d * 16 + v) * 64], a1, oacc[d][v] * a0);
                    m = mn;
                }
            }
        }
        l += __shfl_xor(l, 32, 64);  // the two halves of a row's keys

        const bool out_row = live && ks == 0 && r0 + wq * 32 + (lane & 31) < R;
        if (pieces == 1) {
            if (out_row) {
                if constexpr (LSE) {
                    if (hf == 0) p.lse[int64_t(sq.first + tok) * p.ld_lse + h * p.G + r - tok * p.G] = LseOf<DT>(m, l);
                }
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                uint16_t *orow = p.o + int64_t(sq.first + tok) * p.ldo + int64_t(h * p.G + r - tok * p.G) * D;
#pragma unroll
                for (int d = 0; d < DBLK; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint2 w;
                        w.x = Pack2<DT>(oacc[d][4 * g] * inv, oacc[d][4 * g + 1] * inv);
                        w.y = Pack2<DT>(oacc[d][4 * g + 2] * inv, oacc[d][4 * g + 3] * inv);
                        *reinterpret_cast<uint2 *>(orow + d * 32 + 8 * g + 4 * hf) = w;
                    }
            }
        } else {
            // a piece of a cut unit: its (O, m, l) to a slot of this workgroup
            // (0: the unit began before the workgroup's part, 1: in it). With
            // tickets by device-scope stores, else for the second launch.
            const bool coh = p.cnt != nullptr;
            float *slot = p.ws + int64_t(2 * part + (s_lo == 0 ? 1 : 0)) * (RT * (D + 2));
            if (out_row) {
#pragma unroll
                for (int d = 0; d < DBLK; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        PutU128(slot + ((wq * DBLK * 4 + d * 4 + g) * 64 + lane) * 4,
                                make_uint4(__float_as_uint(oacc[d][4 * g]), __float_as_uint(oacc[d][4 * g + 1]),
                                           __float_as_uint(oacc[d][4 * g + 2]), __float_as_uint(oacc[d][4 * g + 3])),
                                coh);
                if (hf == 0) {
                    float *ml = slot + RT * D + 2 * (wq * 32 + lane);
                    PutU32(ml, __float_as_uint(m), coh);
                    PutU32(ml + 1, __float_as_uint(l), coh);
                }
            }
            if (coh && ubase + u < p.max_units) {
                // the last piece to arrive sums all of them, in the line's order
                __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's part is written
                __syncthreads();
                if (threadIdx.x == 0) {
                    int32_t *c = p.cnt + ubase + u;
                    const int32_t k = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    last_piece = k == pieces - 1;
                    if (last_piece) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (last_piece) {
                    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
                    const int nrow = min(RT, R - r0);
                    for (int ch = int(threadIdx.x); ch < nrow * (D / 4); ch += 64 * NW) {
                        const PieceChunk<D> c(ch, nrow);
                        const PieceSum s = SumPieces<D, QW, 8, true>(p.ws, first, 0, pieces, c);
                        StoreSum<DT>(s, p.o, p.ldo, sq.first, r0 + c.row, h * p.G, p.G, D, c.cc);
                        if constexpr (LSE) {
                            if (c.cc == 0) StoreLse<DT>(s, p.lse, p.ld_lse, sq.first, r0 + c.row, h * p.G, p.G);
                        }
                    }
                }
            }
        }
        if (p.joins != nullptr && s_lo == 0 && threadIdx.x == 0 && ubase + u < p.max_units) {
            PagedJoin &j = p.joins[ubase + u];
            j.pieces = pieces;
            j.part = part;
            j.first = sq.first;
            j.r0 = r0;
            j.nrow = min(RT, R - r0);
            j.head = h * p.G;
        }
        x += cut ? s_hi - s_lo : 1;
        if (x < x_end) {
            __syncthreads();  // the rings are free again
            if (x >= base + size) {  // on to the next sequence with new tokens
                base += size;
                ubase += p.HKV * qt;
                do {
                    ++b;
                } while (b < p.seqs && seq_units(get_seq(b)) == 0);
                if (b >= p.seqs) break;
            }
        }
    }
}

// The second launch: sums the pieces of the cut units, in the line's order.
// Workgroup (x, y) takes 256 / SP chunks of 4 columns of unit x, SP threads to
// a chunk with a share of its pieces each, UN of them in flight. A unit of
// few rows may come in nearly as many pieces as there are workgroups, one of many
// rows in a few. One sequence of 120001 tokens, head size 128, 8, 4, 2 and 1 key
// heads: 63, 126, 235 and 469 pieces a unit, 6, 7, 12 and 18 us beside 93, 52, 30
// and 18 of the first launch (head size 64, 2 heads: 10 beside 19).
template <int QW> struct JoinShape {
    static constexpr int SP = 4 / QW, UN = QW == 4 ? 4 : 8, CH = 256 / SP;
};

template <int DT, int D, int QW, bool LSE>
__global__ void __launch_bounds__(256)
PagedJoinKernel(const float *ws, const PagedJoin *joins, uint16_t *o, int64_t ldo, int G, float *lse, int64_t ld_lse)
{
    constexpr int SP = JoinShape<QW>::SP, CH = JoinShape<QW>::CH;
    __shared__ float part_sum[SP > 1 ? SP - 1 : 1][6][CH];
    const PagedJoin j = joins[blockIdx.x];
    const int chunks = j.nrow * (D / 4);
    if (j.pieces < 2 || int(blockIdx.y) * CH >= chunks) return;
    const int tx = int(threadIdx.x) % CH, sp = int(threadIdx.x) / CH;
    const int ch = int(blockIdx.y) * CH + tx;
    const PieceChunk<D> c(min(ch, chunks - 1), j.nrow);
    const int lo = j.pieces * sp / SP, hi = j.pieces * (sp + 1) / SP;
    PieceSum s = SumPieces<D, QW, JoinShape<QW>::UN, false>(ws, j.part, lo, hi, c);
    if constexpr (SP > 1) {
        if (sp > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) part_sum[sp - 1][e][tx] = s.acc[e];
            part_sum[sp - 1][4][tx] = s.m;
            part_sum[sp - 1][5][tx] = s.l;
        }
        __syncthreads();
        if (sp > 0) return;
#pragma unroll
        for (int i = 0; i < SP - 1; ++i) {
            const float m1 = part_sum[i][4][tx], mn = __builtin_elementwise_maximum(s.m, m1);
            const float ms = mn == -INFINITY ? 0.0f : mn;
            const float a0 = __builtin_amdgcn_exp2f(s.m - ms), a1 = __builtin_amdgcn_exp2f(m1 - ms);
            s.l = __builtin_fmaf(part_sum[i][5][tx], a1, s.l * a0);
#pragma unroll
            for (int e = 0; e < 4; ++e) s.acc[e] = __builtin_fmaf(part_sum[i][e][tx], a1, s.acc[e] * a0);
            s.m = mn;
        }
    }
    if (ch >= chunks) return;
    StoreSum<DT>(s, o, ldo, j.first, j.r0 + c.row, j.head, G, D, c.cc);
    if constexpr (LSE) {
        if (c.cc == 0) StoreLse<DT>(s, lse, ld_lse, j.first, j.r0 + c.row, j.head, G);
    }
}

// Rows a unit holds for this many rows of a sequence and key head.
int UnitWaves(int64_t rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

// The kernels: one row block with two key streams, or with four (the whole
// CU's rings in one workgroup); two with two streams; four with one, 64 keys a
// stage.
template <int DT, int D, bool LSE>
const void *PagedFor(int qw, bool wide)
{
    if (qw == 1 && wide) return reinterpret_cast<const void *>(&PagedKernel<DT, D, 1, 4, 1, 2, LSE>);
    if (qw == 1) return reinterpret_cast<const void *>(&PagedKernel<DT, D, 1, 2, 1, 2, LSE>);
    if (qw == 2) return reinterpret_cast<const void *>(&PagedKernel<DT, D, 2, 2, 1, 2, LSE>);
    return reinterpret_cast<const void *>(&PagedKernel<DT, D, 4, 1, 2, 2, LSE>);
}

template <bool LSE>
const void *PagedFor(int dtype, int D, int qw, bool wide)
{
    if (D == 64) return dtype == kBF16 ? PagedFor<kBF16, 64, LSE>(qw, wide) : PagedFor<kF16, 64, LSE>(qw, wide);
    return dtype == kBF16 ? PagedFor<kBF16, 128, LSE>(qw, wide) : PagedFor<kF16, 128, LSE>(qw, wide);
}

// Units from which the pieces of a cut one are summed by the last of them
// (tickets) instead of a second launch. That many units are cut only where
// their lengths differ a lot, and the launch costs 2 us all the same (64
// sequences of up to 500 tokens, 4 key heads, whole: 21.1 with it, 19.4 us
// without; of up to 1800, 8 heads: 81.3, 79.1); where cutting is the rule it is
// the faster (4 sequences of up to 2000, 2 key heads of 64: 14.3 us against 15.5).
constexpr int kTicketUnits = 192;
// A launch with notes has a workgroup for each unit, so that each writes its
// note whatever `starts` holds.
static_assert(kTicketUnits <= kPagedSlots, "units with notes");

// Units of one row block from which, and up to which, a workgroup has its CU to
// itself for the most part: it takes four key streams. Measured with two streams
// (the better of cut and whole) / with four, in us, head size 128, 4 key heads,
// lengths of up to 4000: 128 units 54 / 62, 160 68 / 68, 192 77 / 74, 256 93 / 87,
// 288 124 / 119; up to 500: 192 19.0 / 18.1, 256 19.3 / 19.3, 288 22 / 32 (more
// than one to a CU, and two do not fit). Head size 64, 2 heads, up to 4000: 160 38
// / 38, 192 41 / 40, 256 59 / 48, 288 75 / 66; up to 500: 256 14.9 / 13.7, 288 17.9
// / 16.8 (two fit: there four streams would go on being the better).
constexpr int kWideFrom = 192;
constexpr int kWideUnits = 256;

struct PagedShape {
    int qw;
    bool wide;
    int64_t units;  // at most
    bool tickets;
    size_t part_bytes, ws_bytes;
    int counters;
};

PagedShape ShapeOf(const kr_cache &c, const kr_seqs &s, int HQ)
{
    if (HQ < 1 || HQ % c.heads != 0)
        throw std::runtime_error("attention_paged: HQ must be a multiple of the cache's heads");
    const int G = HQ / c.heads;
    const int64_t most = int64_t(s.max_new) * G;
    PagedShape r;
    r.qw = UnitWaves(most);
    const int64_t qt = (most + 32 * r.qw - 1) / (32 * r.qw);
    r.units = qt * c.heads * s.seqs;
    if (r.units >= (int64_t(1) << 31)) throw std::runtime_error("attention_paged: too many rows for one launch");
    // nothing is cut where the table holds no unit long enough, or the line of
    // stages (64 keys each) and a share more would not fit 32 bits
    const int64_t most_stages = (int64_t(s.table_pages) * c.page_size + 63) / 64;
    const int at_least = r.qw == 1 ? CutRule<1>::c : r.qw == 2 ? CutRule<2>::c : CutRule<4>::c;
    const bool cuts = r.units > 0 && most_stages > at_least && r.units * most_stages < (int64_t(1) << 30);
    r.wide = r.qw == 1 && r.units >= kWideFrom && r.units <= kWideUnits;
    // a ticket, or a note for the second launch, per unit
    r.tickets = cuts && r.units >= kTicketUnits;
    r.part_bytes = cuts ? size_t(kPagedSlots) * 2 * 32 * r.qw * (c.head_dim + 2) * 4 : 0;
    r.ws_bytes = r.part_bytes + (cuts && !r.tickets ? size_t(r.units) * sizeof(PagedJoin) : 0);
    r.counters = r.tickets ? int(r.units) : 0;
    return r;
}

template <int DT, int D, bool LSE>
void JoinGo(int qw, const PagedParams &p, hipStream_t stream)
{
    const int64_t rows = std::min(int64_t(p.max_new) * p.G, int64_t(32 * qw));
    const int64_t per = qw == 1 ? JoinShape<1>::CH : qw == 2 ? JoinShape<2>::CH : JoinShape<4>::CH;
    const dim3 grid(unsigned(p.max_units), unsigned((rows * (D / 4) + per - 1) / per));
    const auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p.ws, p.joins, p.o, p.ldo, p.G, p.lse, p.ld_lse);
    };
    if (qw == 1) go(PagedJoinKernel<DT, D, 1, LSE>);
    else if (qw == 2) go(PagedJoinKernel<DT, D, 2, LSE>);
    else go(PagedJoinKernel<DT, D, 4, LSE>);
}

}  // namespace

void PagedAttnNeeds(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes, int *counters)
{
    const kr_cache c = CheckCache(cache, "attention_paged");
    CheckSeqs(seqs, "attention_paged");
    const PagedShape f = ShapeOf(c, *seqs, HQ);
    *ws_bytes = f.ws_bytes;
    *counters = f.counters;
}

void PagedAttnLaunch(const PagedAttnDesc &d, hipStream_t stream)
{
    const char *who = "attention_paged";
    const kr_cache c = CheckCache(d.cache, who);
    CheckSeqs(d.seqs, who);
    const kr_seqs &s = *d.seqs;
    const auto refuse = [](const char *what) { throw std::runtime_error(std::string("attention_paged: ") + what); };
    const PagedShape f = ShapeOf(c, s, d.HQ);
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
    if (cap >= (int64_t(1) << 31) - 1024) refuse("the page table spans too many tokens");
    if (int64_t(d.rows) * d.HQ >= (int64_t(1) << 31)) refuse("too many rows for one launch");
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
    p.page_stride = uint32_t(c.page_stride);
    p.token_stride = uint32_t(c.token_stride);
    p.head_stride = c.head_stride;
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
    p.scale_log2 = d.scale * 1.4426950408889634f;
    p.div = MakePageDiv(c.page_size);
    // a piece's cost grows with its rows (measured: 1 to 8 tokens of 4 heads best at 2 to 4, 32 and more at 8 to 12)
    p.min_piece = 2 + int(std::min<int64_t>(int64_t(s.max_new) * p.G, 128)) / 16;
    if (d.ws != nullptr && f.ws_bytes > 0) {
        if (d.ws_bytes < f.ws_bytes || (f.tickets && (d.cnt == nullptr || d.cnt_len < f.counters)) ||
            (reinterpret_cast<uintptr_t>(d.ws) & 15) != 0 || (reinterpret_cast<uintptr_t>(d.cnt) & 3) != 0)
            refuse("the workspace is too small or misaligned");
        p.ws = static_cast<float *>(d.ws);
        if (f.tickets) p.cnt = d.cnt;
        else p.joins = reinterpret_cast<PagedJoin *>(static_cast<char *>(d.ws) + f.part_bytes);
        p.slots = f.wide ? kPagedSlots / 2 : kPagedSlots;
    }
    // whole units: at most one more row block per sequence than its rows fill
    const int64_t units =
        std::min(f.units, int64_t(c.heads) * (int64_t(d.rows) * p.G / (32 * f.qw) + std::min(s.seqs, d.rows)));
    p.max_units = int(units);
    const int64_t wg = std::max<int64_t>(units, p.slots);
    if (wg >= kMaxGrid) refuse("too many rows for one launch");
    const int64_t width = int64_t(d.HQ) * c.head_dim;
    const RowSpan out{d.out, p.ldo, d.rows, width};
    if (Overlap(out, RowSpan{d.q, p.ldq, d.rows, width})) refuse("out overlaps q");
    if (Overlap(out, LayerSpan(c, c.k, d.layer)) || Overlap(out, LayerSpan(c, c.v, d.layer)))
        refuse("out overlaps the cache");
    if (d.with_lse) {
        p.lse = d.lse;
        p.ld_lse = d.ld_lse > 0 ? d.ld_lse : d.HQ;
        if (p.lse == nullptr || (reinterpret_cast<uintptr_t>(p.lse) & 3) != 0) refuse("lse is missing or misaligned");
        if (d.rows > 1 && p.ld_lse < d.HQ) refuse("lse rows overlap");
        const MemSpan lse = RowsSpan(p.lse, d.rows, p.ld_lse, d.HQ, 4);
        const RowSpan k = LayerSpan(c, c.k, d.layer), v = LayerSpan(c, c.v, d.layer);
        if (Meets(lse, RowsSpan(d.q, d.rows, p.ldq, width, 2)) || Meets(lse, RowsSpan(d.out, d.rows, p.ldo, width, 2)) ||
            Meets(lse, MemSpan{k.p, k.width * 2}) || Meets(lse, MemSpan{v.p, v.width * 2}) ||
            Meets(lse, MemSpan{p.ws, int64_t(f.ws_bytes)}) || Meets(lse, MemSpan{p.cnt, int64_t(f.counters) * 4}) ||
            MeetsSeqs(lse, s, d.rows))
            refuse("lse overlaps another tensor of the call");
    }
    void *args[] = {&p};
    const dim3 threads(f.qw == 1 && !f.wide ? 128 : 256);
    const void *kern = d.with_lse ? PagedFor<true>(c.dtype, c.head_dim, f.qw, f.wide)
                                  : PagedFor<false>(c.dtype, c.head_dim, f.qw, f.wide);
    Check(hipLaunchKernel(kern, dim3(unsigned(wg)), threads, args, 0, stream), "attention_paged launch");
    if (p.joins != nullptr) {
        const auto join = [&](auto bf16, auto f16) { c.dtype == kBF16 ? bf16(f.qw, p, stream) : f16(f.qw, p, stream); };
        if (c.head_dim == 64) {
            if (d.with_lse) join(JoinGo<kBF16, 64, true>, JoinGo<kF16, 64, true>);
            else join(JoinGo<kBF16, 64, false>, JoinGo<kF16, 64, false>);
        } else {
            if (d.with_lse) join(JoinGo<kBF16, 128, true>, JoinGo<kF16, 128, true>);
            else join(JoinGo<kBF16, 128, false>, JoinGo<kF16, 128, false>);
        }
    }
    Check(hipGetLastError(), "attention_paged launch");
}

}  // namespace kr
