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
// matrix cores and the softmax's VALU work above.
//
// A unit of work is one key head of one sequence and RT = 32 QW packed rows
// (row r = new token r / G, query head r % G of the key head's G), so the
// heads that share keys share their read. A workgroup has QW x KW waves: QW
// of 32 rows each over the same keys, times KW key streams that take the
// 32 KB-key blocks of the unit in turn and are merged at its end.
//
// Keys and values go HBM -> LDS by the direct-to-LDS DMA into a two-stage
// ring, each lane fetching 16 bytes of a row wherever the page table puts it.
// The table's entries travel the same way two stages ahead (so nothing in the
// loop waits for a dependent load), and each wave turns the next stage's into
// row offsets: lane l's key is l, its validity a ballot. A position past the
// sequence's end or on a page that is none is fetched from the cache's first
// row instead and seen by nobody.
// The products are those of the prompt's kernel (kr_attn.hip): S^T = K Q^T,
// softmax in base 2 with a lazily moved maximum, O^T += V^T P^T, fp32 state;
// P is rounded to 16 bits for the matrix cores, its sum is of the unrounded.
// A block in which some row does not see some key goes the careful way: the
// scores are masked by 64 bits a row, values of unseen rows are zeroed in LDS
// (0 x NaN would reach everybody), and where a seen draft's value is no
// finite number the block is summed on the VALU, row by row.
#include <algorithm>
#include <cmath>

#include "kr_attncore.h"
#include "kr_dma.h"
#include "kr_paged.h"
#include "kr_rowcore.h"

namespace kr {

namespace {

struct PagedParams {
    const uint16_t *q, *k, *v;
    uint16_t *o;
    const int32_t *table, *lens, *starts;
    const uint64_t *tree;
    int64_t ldq, ldo, ld_table, ld_tree;
    int64_t head_stride;
    uint32_t page_stride, token_stride;
    int cap, pages, table_pages, seqs, rows, max_new, tree_words, HQ, HKV, G, qt_max;
    float scale_log2;
    PageDiv div;
    float *ws;       // two partial slots per workgroup of the cut schedule
    int32_t *cnt;    // [seqs][HKV][qt_max] arrival tickets, zero between launches
    int slots;       // workgroups of the cut schedule; 0: whole units only
};

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

__device__ __forceinline__ int64_t WaveScan(int64_t v, int lane)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}

// A wave's own LDS writes before its other lanes' reads of them.
__device__ __forceinline__ void WaveLdsOrder()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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

// Smallest piece of the cut schedule, in stages of a workgroup: a piece costs
// its partial and a share of the sum at the unit's end.
constexpr int kMinPiece = 4;

template <int DT, int D, int QW, int KW, int KB>
__global__ void __attribute__((amdgpu_flat_work_group_size(64 * QW * KW, 64 * QW * KW), amdgpu_waves_per_eu(2)))
PagedKernel(PagedParams p)
{
    static_assert(D == 64 || D == 128, "head_dim 64 or 128");
    constexpr int NW = QW * KW;
    constexpr int THREADS = 64 * NW;
    constexpr int BLK = 32 * KB;            // keys of a stream's stage
    constexpr int SB = BLK * KW;            // keys of a workgroup's stage
    constexpr int RT = 32 * QW;             // rows of a unit
    constexpr int DCH = D / 8;              // 16-byte chunks per row
    constexpr int DBLK = D / 32;            // 32-wide d blocks of O^T
    constexpr int RPD = 64 / DCH;           // rows per 1 KB DMA block
    constexpr int DPW = BLK / RPD / QW;     // DMA blocks per wave, operand and stage
    constexpr uint64_t ALL = KB == 2 ? ~0ull : 0xffffffffull;
    __shared__ __attribute__((aligned(1024))) uint16_t kring[2][KW][BLK * D];
    __shared__ __attribute__((aligned(1024))) uint16_t vring[2][KW][BLK * D];
    __shared__ __attribute__((aligned(256))) int32_t tab[NW][2][64];  // page ids of a stage's keys
    __shared__ int64_t offs[NW][64];                                  // and their rows' element offsets
    __shared__ uint64_t odd[2][KW][QW];                               // keys whose values are not all finite
    __shared__ int last_piece;

    const int lane = int(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int wq = wave % QW, ks = wave / QW;  // row block, key stream
    const int hf = lane >> 5;

    // ---- which part of the work is this workgroup's
    // work of a sequence: its units (key heads x row blocks), each of `sb` stages
    const auto seq_units = [&](const PagedSeq &s) { return p.HKV * ((s.n * p.G + RT - 1) / RT); };
    const auto seq_stages = [&](const PagedSeq &s) { return (s.total + SB - 1) / SB; };
    int64_t units = 0, stages = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        int64_t u = 0, w = 0;
        if (b0 + lane < p.seqs) {
            const PagedSeq s = LoadSeq(p, b0 + lane);
            u = seq_units(s);
            w = u * seq_stages(s);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            u += __shfl_xor(u, o, 64);
            w += __shfl_xor(w, o, 64);
        }
        units += u;
        stages += w;
    }
    if (units == 0) return;
    // cut: `slots` workgroups share out the stages evenly, in one line through
    // all units; else a workgroup has one unit
    const bool cut = p.slots > 0 && units < 4 * int64_t(p.slots);
    int64_t share = 1, x, x_end;  // this workgroup's stages (cut) or units
    {
        int64_t parts = units;
        if (cut) {
            share = max((stages + p.slots - 1) / p.slots, min(int64_t(kMinPiece), (stages + units - 1) / units));
            parts = (stages + share - 1) / share;
        }
        if (int64_t(blockIdx.x) >= parts) return;
        x = XcdChunk(int(blockIdx.x), 0, int(parts)) * share;
        x_end = cut ? min(x + share, stages) : x + 1;
    }
    const int64_t part = cut ? x / share : 0;
    // the sequence that holds x: base <= x < base + its size
    int b = 0;
    int64_t base = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 64) {
        int64_t w = 0;
        if (b0 + lane < p.seqs) {
            const PagedSeq s = LoadSeq(p, b0 + lane);
            w = int64_t(seq_units(s)) * (cut ? seq_stages(s) : 1);
        }
        const int64_t incl = WaveScan(w, lane) + base;
        const uint64_t above = __ballot(incl > x);
        if (above != 0) {
            const int at = __builtin_ctzll(above);
            b = b0 + at;
            base = __shfl(incl - w, at, 64);
            break;
        }
        base = __shfl(incl, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);

    // fragment addresses (elements inside a K / V block), as in kr_attn.hip
    int kaddr[D / 16], vaddr[DBLK];
#pragma unroll
    for (int dc = 0; dc < D / 16; ++dc) kaddr[dc] = (lane & 31) * D + KSlot<D>(lane & 31, 2 * dc + hf) * 8;
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
        const PagedSeq sq = LoadSeq(p, b);
        const int qt = (sq.n * p.G + RT - 1) / RT;
        const int sb = seq_stages(sq);
        const int64_t size = int64_t(p.HKV) * qt * (cut ? sb : 1);
        const int64_t in = x - base;
        const int u = int(cut ? in / sb : in);
        const int s_lo = cut ? int(in - int64_t(u) * sb) : 0;
        const int s_hi = cut ? int(min(int64_t(sb), s_lo + (x_end - x))) : sb;
        const int h = u / qt, t = qt - 1 - u % qt;  // a chunk's longest rows first
        int pieces = 1;
        if (cut) {
            const int64_t u0 = x - s_lo, u1 = u0 + sb;  // the unit's stages in the line
            pieces = int((u1 - 1) / share - u0 / share) + 1;
        }
        const int64_t unit0 = cut ? x - s_lo : x;

        const int R = sq.n * p.G;
        const int r0 = t * RT;
        const int r = min(r0 + wq * 32 + (lane & 31), R - 1);  // (rows past the end repeat the last)
        const int tok = r / p.G;
        const bool live = r0 + wq * 32 < R;
        const int tok_lo = r0 / p.G;                            // of the unit
        const int wtok_hi = min(r0 + wq * 32 + 31, R - 1) / p.G;  // of this wave
        const int kend = p.tree != nullptr ? sq.total
                                           : int(min(int64_t(sq.total), int64_t(sq.len) + min(r0 + RT - 1, R - 1) / p.G + 1));
        const int ns = max(0, min(s_hi, (kend + SB - 1) / SB) - s_lo);
        const int32_t *table = p.table + b * p.ld_table;
        const uint16_t *kh0 = p.k + h * p.head_stride, *vh0 = p.v + h * p.head_stride;
        const uint64_t *tree = p.tree + (p.tree != nullptr ? int64_t(sq.first + tok) * p.ld_tree : 0);

        uint4 qf[D / 16];
        {
            const uint16_t *qrow = p.q + int64_t(sq.first + tok) * p.ldq + int64_t(h * p.G + r - tok * p.G) * D;
#pragma unroll
            for (int dc = 0; dc < D / 16; ++dc) qf[dc] = *reinterpret_cast<const uint4 *>(qrow + dc * 16 + hf * 8);
        }
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
            DmaTouch4(table + pg, LdsAddr(&tab[wave][st & 1][0]));
        };
        // tab -> offs; returns which keys of stage st are there
        const auto rows_of = [&](int st) -> uint64_t {
            const int pos = key0(st) + (lane & (BLK - 1));
            const int id = tab[wave][st & 1][lane];
            const bool ok = pos < sq.total && uint32_t(id) < uint32_t(p.pages);
            const uint32_t in_page = uint32_t(pos - PageOf(p.div, pos) * p.div.size);
            const int64_t off = int64_t(uint64_t(uint32_t(id)) * p.page_stride + uint64_t(in_page) * p.token_stride);
            offs[wave][lane] = ok ? off : 0;
            WaveLdsOrder();
            return __ballot(ok) & ALL;
        };
        // keys and values of stage st -> ring (2 DPW DMA instructions)
        const auto fetch = [&](int st) {
            const uint32_t kdst = LdsAddr(&kring[st & 1][ks][0]) + uint32_t(wq * DPW) * 1024u;
            const uint32_t vdst = LdsAddr(&vring[st & 1][ks][0]) + uint32_t(wq * DPW) * 1024u;
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
            const int64_t k0 = key0(st);
            return there == ALL && (p.tree != nullptr ? k0 + BLK <= sq.len : k0 + BLK - 1 <= int64_t(sq.len) + tok_lo);
        };
        // the values that this wave fetched for stage st: rows that are not
        // there become 0; returns the keys whose rows are not all finite
        const auto clean = [&](int st, uint64_t there) -> uint64_t {
            uint64_t bad = 0;
#pragma unroll
            for (int j = 0; j < DPW; ++j) {
                const int row = (wq * DPW + j) * RPD + lane / DCH;
                uint4 *a = reinterpret_cast<uint4 *>(&vring[st & 1][ks][(wq * DPW + j) * 512 + lane * 8]);
                const bool here = ((there >> row) & 1) != 0;
                const bool nf = here && AnyNonFinite<DT>(*a);
                if (!here) *a = make_uint4(0, 0, 0, 0);
                uint64_t hit = __ballot(nf);
                while (hit != 0) {
                    const int g = __builtin_ctzll(hit) / DCH;
                    bad |= 1ull << ((wq * DPW + j) * RPD + g);
                    hit &= ~(((1ull << DCH) - 1) << (g * DCH));
                }
            }
            WaveLdsOrder();
            return bad;
        };
        // which keys of stage st this lane's row sees
        const auto seen = [&](int st, uint64_t there) -> uint64_t {
            const int64_t j0 = int64_t(key0(st)) - sq.len;  // new token of the first key
            if (p.tree == nullptr) {
                const int64_t nb = tok - j0 + 1;
                return there & (nb >= 64 ? ~0ull : nb <= 0 ? 0ull : (1ull << nb) - 1);
            }
            const auto word = [&](int64_t i) { return i < p.tree_words ? tree[i] : 0ull; };
            uint64_t w;
            if (j0 >= 0) {
                const int sh = int(j0 & 63);
                w = word(j0 >> 6) >> sh;
                if (sh != 0) w |= word((j0 >> 6) + 1) << (64 - sh);
            } else {
                const int c = int(min(-j0, int64_t(64)));
                w = c >= 64 ? ~0ull : ((1ull << c) - 1) | (word(0) << c);
            }
            return there & w;
        };

        // ---- the loop over stages: stage st + 1 is fetched while st is worked
        uint64_t there = 0, next = 0;
        if (ns > 0) {
            fetch_tab(0);
            KR_WAIT_VM(0);
            there = rows_of(0);
            if (ns > 1) fetch_tab(1);
            fetch(0);
            if constexpr (QW > 1) {
                KR_WAIT_VM(0);
                if (!whole(0, there)) {
                    const uint64_t bad = clean(0, there);
                    if (lane == 0) odd[0][ks][wq] = bad;
                }
                __syncthreads();
            }
        }
        for (int st = 0; st < ns; ++st) {
            if (st + 1 < ns) {
                if constexpr (QW == 1) KR_WAIT_VM(2 * DPW);  // the table entries of st + 1 (before the rows of st)
                next = rows_of(st + 1);
                if (st + 2 < ns) fetch_tab(st + 2);
                fetch(st + 1);
                if constexpr (QW == 1) {
                    if (st + 2 < ns) KR_WAIT_VM(2 * DPW + 1);  // the rows of st
                    else KR_WAIT_VM(2 * DPW);
                }
            } else if constexpr (QW == 1) {
                KR_WAIT_VM(0);
            }
            const bool all = whole(st, there);
            uint64_t bad = 0;
            if (!all) {
                if constexpr (QW == 1) {
                    bad = clean(st, there);
                } else {
#pragma unroll
                    for (int i = 0; i < QW; ++i) bad |= odd[st & 1][ks][i];
                }
            }
            // skipped: no key is there, or all lie in this wave's future
            const bool future = p.tree == nullptr && key0(st) > int64_t(sq.len) + wtok_hi;
            if (live && there != 0 && !future) {
                const uint16_t *K = &kring[st & 1][ks][0];
                uint16_t *V = &vring[st & 1][ks][0];
                f32x16 sacc[KB];
#pragma unroll
                for (int kh = 0; kh < KB; ++kh)
#pragma unroll
                    for (int v = 0; v < 16; ++v) sacc[kh][v] = 0.0f;
#pragma unroll
                for (int dc = 0; dc < D / 16; ++dc)
#pragma unroll
                    for (int kh = 0; kh < KB; ++kh)
                        sacc[kh] = Mfma<DT>(*reinterpret_cast<const uint4 *>(K + kh * 32 * D + kaddr[dc]), qf[dc], sacc[kh]);
                // register v of half kh holds key kh*32 + 8 (v/4) + 4 hf + v%4
                uint64_t mine = ALL;
                if (!all) {
                    mine = seen(st, there);
                    const uint64_t bits = mine >> (4 * hf);
#pragma unroll
                    for (int kh = 0; kh < KB; ++kh)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            sacc[kh][v] = ((uint32_t(bits >> (32 * kh)) >> (8 * (v >> 2) + (v & 3))) & 1) != 0 ? sacc[kh][v]
                                                                                                          : -INFINITY;
                }
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
                uint4 pf[2 * KB];
                float ls[4];
#pragma unroll
                for (int c = 0; c < 2 * KB; ++c) {
                    const int kh = c >> 1, vb = (c & 1) * 8;
                    float pv[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[kh][vb + e], p.scale_log2, -msub));
                        ls[e & 3] = c == 0 && e < 4 ? pv[e] : ls[e & 3] + pv[e];
                    }
                    pf[c] = make_uint4(Pack2<DT>(pv[0], pv[1]), Pack2<DT>(pv[2], pv[3]), Pack2<DT>(pv[4], pv[5]),
                                       Pack2<DT>(pv[6], pv[7]));
                }
                l = l * alpha + ((ls[0] + ls[1]) + (ls[2] + ls[3]));
                m = mnew;
                if (__builtin_expect(__ballot(move) != 0, 0)) {
#pragma unroll
                    for (int d = 0; d < DBLK; ++d)
#pragma unroll
                        for (int v = 0; v < 16; ++v) oacc[d][v] *= alpha;
                }
                if (__builtin_expect(bad == 0, 1)) {
#pragma unroll
                    for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
                        for (int d = 0; d < DBLK; ++d) {
                            const AttnS4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(V + c * 16 * D + vaddr[d]));
                            const AttnS4 hi =
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(V + (c * 16 + 8) * D + vaddr[d]));
                            const AttnU2 a = __builtin_bit_cast(AttnU2, lo), z = __builtin_bit_cast(AttnU2, hi);
                            oacc[d] = Mfma<DT>(make_uint4(a.x, a.y, z.x, z.y), pf[c], oacc[d]);
                        }
                } else {
                    // a value that is no finite number, and rows that do not
                    // see it: only those that do may touch it
                    uint32_t w[8 * KB];
#pragma unroll
                    for (int c = 0; c < 2 * KB; ++c) {
                        w[4 * c] = pf[c].x;
                        w[4 * c + 1] = pf[c].y;
                        w[4 * c + 2] = pf[c].z;
                        w[4 * c + 3] = pf[c].w;
                    }
#pragma unroll 1
                    for (int i = 0; i < 8 * KB; ++i) {  // word i of the packed weights, rotated into w[0]
                        const uint32_t own = w[0], other = uint32_t(__shfl_xor(int(own), 32, 64));
#pragma unroll
                        for (int e = 0; e + 1 < 8 * KB; ++e) w[e] = w[e + 1];
#pragma unroll 1
                        for (int k4 = 0; k4 < 4; ++k4) {
                            const int e = 2 * (i & 3) + (k4 & 1), kf = k4 >> 1;
                            const int key = (i >> 2) * 16 + 8 * (e >> 2) + 4 * kf + (e & 3);
                            const float pk = Elem<DT>::Load(uint16_t((hf == kf ? own : other) >> (16 * (k4 & 1))));
                            const bool sees = ((mine >> key) & 1) != 0;
#pragma unroll
                            for (int d = 0; d < DBLK; ++d)
#pragma unroll
                                for (int v = 0; v < 16; ++v) {
                                    const int col = d * 32 + 8 * (v >> 2) + 4 * hf + (v & 3);
                                    const float val = Elem<DT>::Load(V[key * D + VSlot<D>(key, col / 8) * 8 + (col & 7)]);
                                    oacc[d][v] = sees ? __builtin_fmaf(pk, val, oacc[d][v]) : oacc[d][v];
                                }
                        }
                    }
                }
            }
            there = next;
            if constexpr (QW > 1) {
                KR_WAIT_VM(0);  // this wave's part of stage st + 1 has landed
                if (st + 1 < ns && !whole(st + 1, next)) {
                    const uint64_t nf = clean(st + 1, next);
                    if (lane == 0) odd[(st + 1) & 1][ks][wq] = nf;
                }
                __syncthreads();
            }
        }

        // ---- the key streams' states into stream 0's (through the rings)
        if constexpr (KW > 1) {
            constexpr int NE = DBLK * 16;
            static_assert((KW - 1) * QW * NE * 64 * 4 <= int(sizeof(kring)) && (KW - 1) * QW * 128 * 4 <= int(sizeof(vring)),
                          "merge area");
            __syncthreads();
            float *og = reinterpret_cast<float *>(&kring[0][0][0]) + lane, *mg = reinterpret_cast<float *>(&vring[0][0][0]) + lane;
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

        const bool mine = live && ks == 0 && r0 + wq * 32 + (lane & 31) < R;
        if (pieces == 1) {
            if (mine) {
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
            // (0: the unit began before the workgroup's part, 1: in it), with
            // device-scope stores; the last piece to arrive sums all of them
            // in the line's order
            constexpr int SLOT = RT * (D + 2);  // floats: O rows, then (m, l) pairs
            float *slot = p.ws + (2 * part + (s_lo == 0 ? 1 : 0)) * SLOT;
            if (mine) {
                const int row = wq * 32 + (lane & 31);
#pragma unroll
                for (int d = 0; d < DBLK; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        PutU128(slot + row * D + d * 32 + 8 * g + 4 * hf,
                                make_uint4(__float_as_uint(oacc[d][4 * g]), __float_as_uint(oacc[d][4 * g + 1]),
                                           __float_as_uint(oacc[d][4 * g + 2]), __float_as_uint(oacc[d][4 * g + 3])),
                                true);
                if (hf == 0) {
                    PutU32(slot + RT * D + 2 * row, __float_as_uint(m), true);
                    PutU32(slot + RT * D + 2 * row + 1, __float_as_uint(l), true);
                }
            }
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's part is written
            __syncthreads();
            if (threadIdx.x == 0) {
                int32_t *c = p.cnt + (int64_t(b) * p.HKV + h) * p.qt_max + t;
                const int32_t k = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last_piece = k == pieces - 1;
                if (last_piece) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (last_piece) {
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
                const int64_t p0 = unit0 / share;  // the unit's first workgroup
                const int nrow = min(RT, R - r0);
                for (int ch = int(threadIdx.x); ch < nrow * (D / 4); ch += THREADS) {
                    const int row = ch / (D / 4);
                    float acc[4] = {}, mm = -INFINITY, ll = 0.0f;
                    constexpr int UN = 8;  // pieces in flight
                    for (int i0 = 0; i0 < pieces; i0 += UN) {
                        uint4 ov[UN];
                        float mp[UN], lp[UN];
#pragma unroll
                        for (int i = 0; i < UN; ++i) {
                            mp[i] = -INFINITY;
                            lp[i] = 0.0f;
                            ov[i] = make_uint4(0, 0, 0, 0);
                            if (i0 + i < pieces) {
                                const int64_t pt = p0 + i0 + i;
                                const float *s = p.ws + (2 * pt + (pt * share <= unit0 ? 1 : 0)) * SLOT;
                                ov[i] = LoadU128Dev(s, ch * 16);
                                mp[i] = __hip_atomic_load(s + RT * D + 2 * row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                                lp[i] = __hip_atomic_load(s + RT * D + 2 * row + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                            }
                        }
                        float mn = mm;
#pragma unroll
                        for (int i = 0; i < UN; ++i) mn = __builtin_elementwise_maximum(mn, mp[i]);
                        const float ms = mn == -INFINITY ? 0.0f : mn;
                        const float a0 = __builtin_amdgcn_exp2f(mm - ms);
                        ll *= a0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[e] *= a0;
#pragma unroll
                        for (int i = 0; i < UN; ++i) {
                            const float a = __builtin_amdgcn_exp2f(mp[i] - ms);
                            ll = __builtin_fmaf(lp[i], a, ll);
                            acc[0] = __builtin_fmaf(__uint_as_float(ov[i].x), a, acc[0]);
                            acc[1] = __builtin_fmaf(__uint_as_float(ov[i].y), a, acc[1]);
                            acc[2] = __builtin_fmaf(__uint_as_float(ov[i].z), a, acc[2]);
                            acc[3] = __builtin_fmaf(__uint_as_float(ov[i].w), a, acc[3]);
                        }
                        mm = mn;
                    }
                    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                    const int tk = (r0 + row) / p.G, g = r0 + row - tk * p.G;
                    uint2 w;
                    w.x = Pack2<DT>(acc[0] * inv, acc[1] * inv);
                    w.y = Pack2<DT>(acc[2] * inv, acc[3] * inv);
                    *reinterpret_cast<uint2 *>(p.o + int64_t(sq.first + tk) * p.ldo + int64_t(h * p.G + g) * D +
                                               (ch - row * (D / 4)) * 4) = w;
                }
            }
        }
        x += cut ? s_hi - s_lo : 1;
        if (x < x_end) {
            __syncthreads();  // the rings and last_piece are free again
            if (x >= base + size) {  // on to the next sequence with new tokens
                base += size;
                do {
                    if (++b >= p.seqs) return;
                } while (seq_units(LoadSeq(p, b)) == 0);
            }
        }
    }
}

// Rows a unit holds for this many rows of a sequence and key head.
int UnitWaves(int64_t rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

template <int DT, int D, int QW>
const void *PagedFn()
{
    if constexpr (QW == 1) return reinterpret_cast<const void *>(&PagedKernel<DT, D, 1, 2, 1>);
    else if constexpr (QW == 2) return reinterpret_cast<const void *>(&PagedKernel<DT, D, 2, 2, 1>);
    else return reinterpret_cast<const void *>(&PagedKernel<DT, D, 4, 1, 2>);
}

int PagedThreads(int qw) { return qw == 1 ? 128 : 256; }

const void *PagedFor(int dtype, int D, int qw)
{
    const auto pick = [&](auto d64, auto d128) { return D == 64 ? d64() : d128(); };
    if (dtype == kBF16) {
        if (qw == 1) return pick(PagedFn<kBF16, 64, 1>, PagedFn<kBF16, 128, 1>);
        if (qw == 2) return pick(PagedFn<kBF16, 64, 2>, PagedFn<kBF16, 128, 2>);
        return pick(PagedFn<kBF16, 64, 4>, PagedFn<kBF16, 128, 4>);
    }
    if (qw == 1) return pick(PagedFn<kF16, 64, 1>, PagedFn<kF16, 128, 1>);
    if (qw == 2) return pick(PagedFn<kF16, 64, 2>, PagedFn<kF16, 128, 2>);
    return pick(PagedFn<kF16, 64, 4>, PagedFn<kF16, 128, 4>);
}

// Workgroups of the cut schedule: two on each of 256 CUs (their rings fill 128
// of a CU's 160 KB at head size 128).
constexpr int kPagedSlots = 512;

struct PagedShape {
    int qw, qt_max;
    size_t ws_bytes;
    int64_t counters;
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
    r.counters = qt * c.heads * s.seqs;
    if (r.counters >= (int64_t(1) << 31)) throw std::runtime_error("attention_paged: too many rows for one launch");
    r.qt_max = int(qt);
    r.ws_bytes = r.counters == 0 ? 0 : size_t(kPagedSlots) * 2 * 32 * r.qw * (c.head_dim + 2) * 4;
    return r;
}

}  // namespace

void PagedAttnNeeds(const kr_cache *cache, const kr_seqs *seqs, int HQ, size_t *ws_bytes, int *counters)
{
    const kr_cache c = CheckCache(cache, "attention_paged");
    CheckSeqs(seqs, "attention_paged");
    const PagedShape f = ShapeOf(c, *seqs, HQ);
    *ws_bytes = f.ws_bytes;
    *counters = int(f.counters);
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
    p.qt_max = f.qt_max;
    p.scale_log2 = d.scale * 1.4426950408889634f;
    p.div = MakePageDiv(c.page_size);
    if (d.ws != nullptr) {
        if (d.cnt == nullptr || d.ws_bytes < f.ws_bytes || d.cnt_len < f.counters ||
            (reinterpret_cast<uintptr_t>(d.ws) & 15) != 0)
            refuse("the workspace is too small or misaligned");
        p.ws = static_cast<float *>(d.ws);
        p.cnt = d.cnt;
        p.slots = kPagedSlots;
    }
    // whole units: at most one more row block per sequence than its rows fill
    const int64_t units =
        std::min(f.counters, int64_t(c.heads) * (int64_t(d.rows) * p.G / (32 * f.qw) + std::min(s.seqs, d.rows)));
    const int64_t wg = std::max<int64_t>(units, p.slots);
    if (wg >= (int64_t(1) << 31)) refuse("too many rows for one launch");
    void *args[] = {&p};
    Check(hipLaunchKernel(PagedFor(c.dtype, c.head_dim, f.qw), dim3(unsigned(wg)), dim3(unsigned(PagedThreads(f.qw))),
                          args, 0, stream),
          "attention_paged launch");
    Check(hipGetLastError(), "attention_paged launch");
}

}  // namespace kr
