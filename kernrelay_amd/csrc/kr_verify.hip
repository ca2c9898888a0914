// Drafted tokens against the target's logits: rejection sampling down a chain
// or tree of drafts. See kr_op_verify_drafts. No counterpart in the reference,
// whose path ends with the prompt's last row.
//
// With p = softmax(x / t) at a row and its drafts tried in order: token y is
// accepted iff u q(y) < p(y); else p <- max(p - q, 0) / sum. The token after
// the last accepted row is drawn from the p that is left there, by its
// cumulated sum. Kept tokens are then distributed as the target's own.
//
// Everything is computed in 64 bits, the exponentials too: with 150000 tokens a
// token's share of the cumulated sum is often below the 2^-24 that 32 bits
// leave of it.
//
// Launches: the largest logit and the sum of each row, in pieces of 8192
// values; a workgroup for each sequence walks down its drafts; sums of what is
// left at the row where the walk ended, in the same pieces; and the token.
#include <algorithm>

#include "kr_paged.h"

namespace kr {

namespace {

constexpr int kPiece = 8192;    // values of a piece: 32 a thread
constexpr int kMostNew = 1024;  // tokens of a sequence

struct RowPart {
    float top;  // largest logit of the piece
    int at;     // its first place
    double sum; // of exp((x - top) / t)
};
struct SeqEnd {
    int row;      // where the walk ended: a row of the launch, -1: the sequence has none
    int refused;  // drafts that were refused there
};
struct LeftPart {
    double left, was;  // sums of p after and before the last refusal
};

struct VerifyParams {
    const void *logits, *draft;
    const int64_t *tokens;
    const int32_t *parents, *starts;
    const float *u, *u_next, *temperature;
    int32_t *path, *path_lens;
    int64_t *next;
    int64_t ld_logits, ld_draft, ld_path;
    int dtype, draft_dtype, vocab, rows, seqs, max_new, width, pieces;
    bool wide, draft_wide;  // rows are 16-byte aligned
    RowPart *parts;         // [rows, pieces]
    RowPart *stats;         // [rows]
    double *totals;         // [rows]: of a sequence's end row, the sums after its refusals
    SeqEnd *ends;           // [seqs]
    LeftPart *lefts;        // [seqs, pieces]
};

struct VerifySeq {
    int first, n;
};

__device__ __forceinline__ VerifySeq LoadSeq(const VerifyParams &p, int b)
{
    VerifySeq s;
    s.first = min(max(p.starts[b], 0), p.rows);
    s.n = min(min(max(p.starts[b + 1], s.first), p.rows) - s.first, p.max_new);
    return s;
}

// -1 for a temperature that picks the first of the largest.
__device__ __forceinline__ double InvTemperature(const VerifyParams &p, int b)
{
    if (p.temperature == nullptr) return 1.0;
    const float t = p.temperature[b];
    return t > 0.0f ? 1.0 / double(t) : -1.0;
}

__device__ __forceinline__ float LoadAny(const void *base, int dtype, int64_t at)
{
    if (dtype == kF32) return static_cast<const float *>(base)[at];
    const uint16_t x = static_cast<const uint16_t *>(base)[at];
    return dtype == kBF16 ? BF16ToF32(x) : F16ToF32(x);
}

// Values at .. at + 7 of a row of n; past its end `none`.
__device__ __forceinline__ void Load8(const void *row, int dtype, bool wide, int at, int n, float none, float (&x)[8])
{
    if (wide && at + 8 <= n) {
        if (dtype == kF32) {
            const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(row) + at);
            const float4 c = *reinterpret_cast<const float4 *>(static_cast<const float *>(row) + at + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
            x[4] = c.x, x[5] = c.y, x[6] = c.z, x[7] = c.w;
        } else {
            const U16x8 v = LoadU16x8(static_cast<const uint16_t *>(row) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = dtype == kBF16 ? BF16ToF32(v.v[e]) : F16ToF32(v.v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = at + e < n ? LoadAny(row, dtype, at + e) : none;
    }
}

__device__ __forceinline__ const void *RowOf(const void *base, int dtype, int64_t at)
{
    return static_cast<const char *>(base) + at * (dtype == kF32 ? 4 : 2);
}

__device__ __forceinline__ float Logit(float x) { return x != x ? -INFINITY : x; }
__device__ __forceinline__ float Chance(float q) { return q > 0.0f ? q : 0.0f; }

// exp((x - top) / t), 1 at the top itself, also an infinite one; without a
// temperature 1 at place `at` alone. (Differences of infinities and their
// products with 1 / t = 0 are no numbers.)
__device__ __forceinline__ double Weight(float x, int i, float top, int at, double inv_t)
{
    if (inv_t < 0.0) return i == at ? 1.0 : 0.0;
    if (x == -INFINITY) return 0.0;
    if (x == top) return 1.0;
    return top == INFINITY ? 0.0 : exp((double(x) - double(top)) * inv_t);
}

__device__ __forceinline__ double WaveSumD(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Sum over the 256 threads, in every one of them.
__device__ __forceinline__ double BlockSumD(double v, double *part)
{
    v = WaveSumD(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ void __launch_bounds__(256) StatsKernel(VerifyParams p)
{
    __shared__ float top_of[4];
    __shared__ int at_of[4];
    __shared__ double part[4];
    const int piece = int(blockIdx.x) % p.pieces, row = int(blockIdx.x) / p.pieces;
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
    int b = -1;
    for (int b0 = 0; b0 < p.seqs && b < 0; b0 += 64) {
        bool mine = false;
        if (b0 + lane < p.seqs) {
            const VerifySeq s = LoadSeq(p, b0 + lane);
            mine = row >= s.first && row < s.first + s.n;
        }
        const uint64_t hit = __ballot(mine);
        if (hit != 0) b = b0 + __builtin_ctzll(hit);
    }
    if (b < 0) return;  // a row of no sequence
    const double inv_t = InvTemperature(p, b);
    const void *x_row = RowOf(p.logits, p.dtype, int64_t(row) * p.ld_logits);
    float x[32];
    const int i0 = piece * kPiece + int(threadIdx.x) * 8;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float y[8];
        Load8(x_row, p.dtype, p.wide, i0 + g * 2048, p.vocab, -INFINITY, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[g * 8 + e] = Logit(y[e]);
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, x[e]);
    top = WaveMax(top);
    if (lane == 0) top_of[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
    int at = INT32_MAX;
    double sum = 0.0;
#pragma unroll
    for (int g = 3; g >= 0; --g)
#pragma unroll
        for (int e = 7; e >= 0; --e) {
            if (x[g * 8 + e] == top) at = i0 + g * 2048 + e;
            if (inv_t >= 0.0) sum += Weight(x[g * 8 + e], 0, top, 0, inv_t);
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if (lane == 0) at_of[wave] = at;
    sum = BlockSumD(sum, part);
    if (threadIdx.x == 0) {
        RowPart r;
        r.top = top;
        r.at = min(min(at_of[0], at_of[1]), min(at_of[2], at_of[3]));
        r.sum = inv_t < 0.0 ? 1.0 : sum;
        p.parts[int64_t(row) * p.pieces + piece] = r;
    }
}

// What is left of value i's probability after `refused` refusals at a row with
// draft probabilities q: `totals` are the sums after each, the last one not
// needed. was: before the last refusal.
__device__ __forceinline__ double Left(double w, double q, const double *totals, int refused, double &was)
{
    double r = w;
    was = r;
    for (int k = 0; k < refused; ++k) {
        was = r;
        r = fmax(r - q, 0.0);
        if (k + 1 < refused) {
            const double t = totals[k];
            r = t > 0.0 ? r / t : was;
        }
    }
    return r;
}

__global__ void __launch_bounds__(256) WalkKernel(VerifyParams p)
{
    __shared__ double prob[kMostNew];      // of draft i at the row that it follows, before any refusal
    __shared__ double totals[kMostNew];
    __shared__ RowPart stats[kMostNew];
    __shared__ float chance[kMostNew], u[kMostNew];
    __shared__ int above[kMostNew], token[kMostNew];
    __shared__ double part[4];
    const int b = int(blockIdx.x), tid = int(threadIdx.x), lane = tid & 63;
    const VerifySeq sq = LoadSeq(p, b);
    const double inv_t = InvTemperature(p, b);
    for (int i = tid; i < p.width; i += 256) p.path[b * p.ld_path + i] = i == 0 && sq.n > 0 ? 0 : -1;
    if (sq.n == 0) {
        if (tid == 0) {
            p.path_lens[b] = 0;
            p.ends[b] = SeqEnd{-1, 0};
        }
        return;
    }
    // ---- rows: their pieces put together, eight lanes to a row
    for (int r0 = 0; r0 < sq.n; r0 += 32) {
        const int r = r0 + tid / 8, l8 = tid % 8;
        const RowPart *parts = p.parts + int64_t(sq.first + min(r, sq.n - 1)) * p.pieces;
        float top = -INFINITY;
        for (int c = l8; c < p.pieces; c += 8) top = fmaxf(top, parts[c].top);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        int at = INT32_MAX;
        double sum = 0.0;
        for (int c = l8; c < p.pieces; c += 8) {
            const RowPart x = parts[c];
            if (x.top == top) at = min(at, x.at);
            if (inv_t >= 0.0) sum += x.sum * Weight(x.top, 0, top, 0, inv_t);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            at = min(at, __shfl_xor(at, o, 64));
            sum += __shfl_xor(sum, o, 64);
        }
        if (l8 == 0 && r < sq.n) {
            RowPart x;
            x.top = top;
            x.at = at;
            x.sum = inv_t < 0.0 ? 1.0 : sum;
            stats[r] = x;
            p.stats[sq.first + r] = x;
        }
    }
    // ---- drafts: what they follow and how likely they are there
    for (int i = tid; i < sq.n; i += 256) {
        const int64_t tok = p.tokens[sq.first + i];
        const int par = p.parents != nullptr ? p.parents[sq.first + i] : i - 1;
        above[i] = i > 0 && par >= 0 && par < i ? par : -1;
        token[i] = tok >= 0 && tok < p.vocab ? int(tok) : -1;
        u[i] = p.u[sq.first + i];
    }
    __syncthreads();
    for (int i = tid; i < sq.n; i += 256) {
        const int par = above[i], tok = token[i];
        double w = 0.0;
        float q = 1.0f;
        if (par >= 0 && tok >= 0) {
            const RowPart s = stats[par];
            const int64_t row = sq.first + par;
            const float x = Logit(LoadAny(p.logits, p.dtype, row * p.ld_logits + tok));
            if (s.top != -INFINITY) w = Weight(x, tok, s.top, s.at, inv_t) / s.sum;
            if (p.draft != nullptr) {
                q = Chance(LoadAny(p.draft, p.draft_dtype, row * p.ld_draft + tok));
            } else {
                // a token that was refused there already has nothing left
                for (int j = par + 1; j < i; ++j)
                    if (above[j] == par && token[j] == tok) w = 0.0;
            }
        }
        prob[i] = w;
        chance[i] = q;
    }
    __syncthreads();
    // ---- down the drafts; every thread takes the same steps
    int cur = 0, len = 1, refused = 0;
    while (len < p.width) {
        refused = 0;
        double rest = 1.0;  // (drafts that were not drawn)
        int next = -1;
        for (int i0 = (cur + 1) / 64 * 64; i0 < sq.n && next < 0; i0 += 64) {
            uint64_t hit = __ballot(i0 + lane < sq.n && i0 + lane > cur && above[min(i0 + lane, sq.n - 1)] == cur);
            while (hit != 0 && next < 0) {
                const int i = Uni(i0 + __builtin_ctzll(hit));
                hit &= hit - 1;
                bool ok;
                if (p.draft == nullptr) {
                    ok = double(u[i]) * rest < prob[i];
                    rest = fmax(rest - prob[i], 0.0);
                } else {
                    if (refused > 0) {
                        // the sum after the last refusal, over the vocabulary
                        const RowPart s = stats[cur];
                        const int64_t row = sq.first + cur;
                        const void *xr = RowOf(p.logits, p.dtype, row * p.ld_logits);
                        const void *qr = RowOf(p.draft, p.draft_dtype, row * p.ld_draft);
                        double sum = 0.0;
                        for (int v = tid * 8; v < p.vocab; v += 2048) {
                            float x[8], q[8];
                            Load8(xr, p.dtype, p.wide, v, p.vocab, -INFINITY, x);
                            Load8(qr, p.draft_dtype, p.draft_wide, v, p.vocab, 0.0f, q);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                double was;
                                if (s.top != -INFINITY)
                                    sum += Left(Weight(Logit(x[e]), v + e, s.top, s.at, inv_t) / s.sum, Chance(q[e]),
                                                totals, refused, was);
                            }
                        }
                        sum = BlockSumD(sum, part);
                        if (tid == 0) totals[refused - 1] = sum;
                        __syncthreads();
                    }
                    double r = prob[i];
                    for (int k = 0; k < refused; ++k)
                        r = totals[k] > 0.0 ? fmax(r - double(chance[i]), 0.0) / totals[k] : r;
                    ok = double(u[i]) * double(chance[i]) < r;
                }
                if (ok) next = i;
                else ++refused;
            }
        }
        if (next < 0) break;
        if (tid == 0) p.path[b * p.ld_path + len] = next;
        refused = 0;
        cur = next;
        ++len;
    }
    if (tid == 0) {
        p.path_lens[b] = len;
        p.ends[b] = SeqEnd{sq.first + cur, refused};
    }
    if (p.draft != nullptr)
        for (int k = tid; k + 1 < refused; k += 256) p.totals[sq.first + k] = totals[k];
}

// What is left of the end row's values i .. i + 7 of a thread, before and after the last refusal.
struct EndRow {
    const void *x, *q;
    RowPart s;
    const double *totals;
    double inv_t;
    int refused, row;
};

__device__ __forceinline__ EndRow LoadEnd(const VerifyParams &p, int b, const SeqEnd &e)
{
    EndRow r;
    r.row = e.row;
    r.refused = e.refused;
    r.s = p.stats[e.row];
    r.inv_t = InvTemperature(p, b);
    r.x = RowOf(p.logits, p.dtype, int64_t(e.row) * p.ld_logits);
    r.q = p.draft != nullptr ? RowOf(p.draft, p.draft_dtype, int64_t(e.row) * p.ld_draft) : nullptr;
    r.totals = p.totals + LoadSeq(p, b).first;
    return r;
}

// Marks the tokens of a piece that were refused at the end row (drafts that were not drawn).
__device__ __forceinline__ void MarkRefused(const VerifyParams &p, int b, const EndRow &r, int v0, uint32_t *marks)
{
    for (int i = int(threadIdx.x); i < kPiece / 32; i += 256) marks[i] = 0;
    __syncthreads();
    if (p.draft == nullptr && r.refused > 0) {
        const VerifySeq sq = LoadSeq(p, b);
        for (int i = int(threadIdx.x); i < sq.n; i += 256) {
            const int par = p.parents != nullptr ? p.parents[sq.first + i] : i - 1;
            const int64_t tok = p.tokens[sq.first + i] - v0;
            if (i > 0 && par >= 0 && par < i && sq.first + par == r.row && tok >= 0 && tok < kPiece)
                atomicOr(&marks[tok >> 5], 1u << (tok & 31));
        }
    }
    __syncthreads();
}

__device__ __forceinline__ void Left8(const VerifyParams &p, const EndRow &r, int v, int v0, const uint32_t *marks,
                                      double (&left)[8], double (&was)[8])
{
    float x[8], q[8];
    Load8(r.x, p.dtype, p.wide, v, p.vocab, -INFINITY, x);
    if (p.draft != nullptr && r.refused > 0) Load8(r.q, p.draft_dtype, p.draft_wide, v, p.vocab, 0.0f, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const double w = r.s.top == -INFINITY || v + e >= p.vocab ? 0.0 : Weight(Logit(x[e]), v + e, r.s.top, r.s.at, r.inv_t);
        if (p.draft != nullptr) {
            left[e] = Left(w / r.s.sum, r.refused > 0 ? double(Chance(q[e])) : 0.0, r.totals, r.refused, was[e]);
        } else {
            was[e] = w;
            left[e] = ((marks[(v + e - v0) >> 5] >> ((v + e - v0) & 31)) & 1) != 0 ? 0.0 : w;
        }
    }
}

__global__ void __launch_bounds__(256) LeftKernel(VerifyParams p)
{
    __shared__ uint32_t marks[kPiece / 32];
    __shared__ double part[4];
    const int piece = int(blockIdx.x) % p.pieces, b = int(blockIdx.x) / p.pieces;
    const SeqEnd end = p.ends[b];
    if (end.row < 0) return;
    const EndRow r = LoadEnd(p, b, end);
    const int v0 = piece * kPiece;
    MarkRefused(p, b, r, v0, marks);
    double left = 0.0, was = 0.0;
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        double l8[8], w8[8];
        Left8(p, r, v0 + g * 2048 + int(threadIdx.x) * 8, v0, marks, l8, w8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            left += l8[e];
            was += w8[e];
        }
    }
    left = BlockSumD(left, part);
    was = BlockSumD(was, part);
    if (threadIdx.x == 0) p.lefts[int64_t(b) * p.pieces + piece] = LeftPart{left, was};
}

__global__ void __launch_bounds__(256) NextKernel(VerifyParams p)
{
    __shared__ uint32_t marks[kPiece / 32];
    __shared__ double wave_sum[4];
    const int b = int(blockIdx.x), tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const SeqEnd end = p.ends[b];
    if (end.row < 0) {
        if (tid == 0) p.next[b] = -1;
        return;
    }
    const EndRow r = LoadEnd(p, b, end);
    // ---- the piece: every thread adds up the pieces in order
    const LeftPart *lefts = p.lefts + int64_t(b) * p.pieces;
    double left = 0.0, was = 0.0;
    for (int c = 0; c < p.pieces; ++c) {
        left += lefts[c].left;
        was += lefts[c].was;
    }
    const bool stays = !(left > 0.0);  // nothing left: p as it was
    const double total = stays ? was : left;
    if (!(total > 0.0)) {
        if (tid == 0) p.next[b] = -1;
        return;
    }
    const double bar = double(p.u_next[b]) * total;
    double base = 0.0, sum = 0.0;
    int piece = -1;
    for (int c = 0; c < p.pieces; ++c) {
        const double x = stays ? lefts[c].was : lefts[c].left;
        if (x > 0.0) {
            piece = c;
            base = sum;
            if (sum + x > bar) break;
        }
        sum += x;
    }
    // ---- the value: thread t has 32 in a row
    const int v0 = piece * kPiece, i0 = tid * 32;
    MarkRefused(p, b, r, v0, marks);
    double mine[32], own = 0.0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        double l8[8], w8[8];
        Left8(p, r, v0 + i0 + g * 8, v0, marks, l8, w8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mine[g * 8 + e] = stays ? w8[e] : l8[e];
            own += mine[g * 8 + e];
        }
    }
    double incl = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(incl, o, 64);
        if (lane >= o) incl += x;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    for (int i = 0; i < wave; ++i) base += wave_sum[i];
    double at = base + (incl - own);
    int hit = INT32_MAX, tail = -1;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        at += mine[e];
        if (mine[e] > 0.0) {
            if (hit == INT32_MAX && at > bar) hit = v0 + i0 + e;
            tail = v0 + i0 + e;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        hit = min(hit, __shfl_xor(hit, o, 64));
        tail = max(tail, __shfl_xor(tail, o, 64));
    }
    __shared__ int hits[4], tails[4];
    if (lane == 0) hits[wave] = hit, tails[wave] = tail;
    __syncthreads();
    if (tid == 0) {
        hit = min(min(hits[0], hits[1]), min(hits[2], hits[3]));
        tail = max(max(tails[0], tails[1]), max(tails[2], tails[3]));
        p.next[b] = hit != INT32_MAX ? hit : tail;
    }
}

struct VerifyShape {
    int pieces;
    size_t parts, stats, totals, ends, lefts, bytes;
};

VerifyShape ShapeOf(const kr_drafts &d, const kr_seqs &s)
{
    VerifyShape f{};
    f.pieces = int((int64_t(d.vocab) + kPiece - 1) / kPiece);
    const size_t rows = size_t(d.rows), seqs = size_t(s.seqs);
    f.parts = 0;
    f.stats = f.parts + rows * f.pieces * sizeof(RowPart);
    f.totals = f.stats + rows * sizeof(RowPart);
    f.lefts = f.totals + (rows * sizeof(double) + 15) / 16 * 16;
    f.ends = f.lefts + seqs * f.pieces * sizeof(LeftPart);
    f.bytes = f.ends + (seqs * sizeof(SeqEnd) + 15) / 16 * 16;
    return f;
}

kr_drafts CheckDrafts(const kr_drafts *d, const kr_seqs *s)
{
    const auto refuse = [](const char *what) { throw std::runtime_error(std::string("verify_drafts: ") + what); };
    if (d == nullptr) refuse("needs drafts");
    CheckSeqs(s, "verify_drafts");
    const auto known = [](int t) { return t == kBF16 || t == kF16 || t == kF32; };
    if (!known(d->dtype) || (d->draft != nullptr && !known(d->draft_dtype)))
        refuse("logits and draft must be bf16, f16 or f32");
    if (d->rows < 0 || d->vocab < 1) refuse("a negative or empty size");
    if (s->max_new > kMostNew) refuse("a sequence has at most 1024 new tokens");
    if (d->rows > 1 && (d->ld_logits < d->vocab || (d->draft != nullptr && d->ld_draft < d->vocab)))
        refuse("rows of logits or draft overlap");
    if (d->ld_logits > (int64_t(1) << 40) || d->ld_draft > (int64_t(1) << 40)) refuse("a row stride is too large");
    if (d->vocab > (1 << 30)) refuse("the vocabulary is too large");
    const int64_t pieces = (int64_t(d->vocab) + kPiece - 1) / kPiece;
    if (pieces * d->rows >= kMaxGrid || pieces * s->seqs >= kMaxGrid) refuse("too many rows for one launch");
    return *d;
}

}  // namespace

void VerifyNeeds(const kr_drafts *drafts, const kr_seqs *s, size_t *ws_bytes, int *counters)
{
    const kr_drafts d = CheckDrafts(drafts, s);
    *ws_bytes = ShapeOf(d, *s).bytes;
    *counters = 0;
}

void VerifyLaunch(const kr_drafts *drafts, const kr_seqs *s, const VerifyOut &o, void *ws, size_t ws_bytes,
                  int32_t *, int, hipStream_t stream)
{
    const auto refuse = [](const char *what) { throw std::runtime_error(std::string("verify_drafts: ") + what); };
    const kr_drafts d = CheckDrafts(drafts, s);
    if (s->seqs == 0) return;
    if (o.width < 1 || (s->seqs > 1 && o.ld_path < o.width)) refuse("path rows are empty or overlap");
    if (o.path == nullptr || o.path_lens == nullptr || o.next == nullptr) refuse("an output is missing");
    if (d.u_next == nullptr ||
        (d.rows > 0 && (d.logits == nullptr || d.tokens == nullptr || d.u == nullptr)))
        refuse("logits, tokens or random numbers are missing");
    const auto off = [](const void *p, int by) { return (reinterpret_cast<uintptr_t>(p) & uintptr_t(by - 1)) != 0; };
    const int size = d.dtype == kF32 ? 4 : 2, dsize = d.draft_dtype == kF32 ? 4 : 2;
    if (off(d.logits, size) || off(d.draft, d.draft != nullptr ? dsize : 1) || off(d.tokens, 8) || off(o.next, 8) ||
        off(d.parents, 4) || off(d.u, 4) || off(d.u_next, 4) || off(d.temperature, 4) || off(o.path, 4) || off(o.path_lens, 4))
        refuse("a pointer is misaligned");
    const VerifyShape f = ShapeOf(d, *s);
    if (ws == nullptr || ws_bytes < f.bytes || off(ws, 16)) refuse("the workspace is too small or misaligned");
    const MemSpan outs[] = {RowsSpan(o.path, s->seqs, o.ld_path, o.width, 4), RowsSpan(o.path_lens, 1, 0, s->seqs, 4),
                            RowsSpan(o.next, 1, 0, s->seqs, 8), MemSpan{ws, int64_t(f.bytes)}};
    const MemSpan ins[] = {RowsSpan(d.logits, d.rows, d.ld_logits, d.vocab, size),
                           RowsSpan(d.draft, d.rows, d.ld_draft, d.vocab, dsize), RowsSpan(d.tokens, 1, 0, d.rows, 8),
                           RowsSpan(d.parents, 1, 0, d.rows, 4), RowsSpan(d.u, 1, 0, d.rows, 4),
                           RowsSpan(d.u_next, 1, 0, s->seqs, 4), RowsSpan(d.temperature, 1, 0, s->seqs, 4),
                           RowsSpan(s->starts, 1, 0, s->seqs + 1, 4)};
    for (int i = 0; i < 4; ++i) {
        for (int j = i + 1; j < 4; ++j)
            if (Meets(outs[i], outs[j])) refuse("outputs and workspace overlap");
        for (const MemSpan &in : ins)
            if (Meets(outs[i], in)) refuse("an output or the workspace overlaps an input");
    }
    VerifyParams p{};
    p.logits = d.logits;
    p.draft = d.draft;
    p.tokens = d.tokens;
    p.parents = d.parents;
    p.starts = s->starts;
    p.u = d.u;
    p.u_next = d.u_next;
    p.temperature = d.temperature;
    p.path = o.path;
    p.path_lens = o.path_lens;
    p.next = o.next;
    p.ld_logits = d.ld_logits;
    p.ld_draft = d.ld_draft;
    p.ld_path = o.ld_path;
    p.dtype = d.dtype;
    p.draft_dtype = d.draft_dtype;
    p.vocab = d.vocab;
    p.rows = d.rows;
    p.seqs = s->seqs;
    p.max_new = s->max_new;
    p.width = o.width;
    p.pieces = f.pieces;
    p.wide = !off(d.logits, 16) && (d.rows <= 1 || d.ld_logits * size % 16 == 0);
    p.draft_wide = !off(d.draft, 16) && (d.rows <= 1 || d.ld_draft * dsize % 16 == 0);
    char *base = static_cast<char *>(ws);
    p.parts = reinterpret_cast<RowPart *>(base + f.parts);
    p.stats = reinterpret_cast<RowPart *>(base + f.stats);
    p.totals = reinterpret_cast<double *>(base + f.totals);
    p.lefts = reinterpret_cast<LeftPart *>(base + f.lefts);
    p.ends = reinterpret_cast<SeqEnd *>(base + f.ends);
    if (d.rows > 0 && s->max_new > 0) {
        hipLaunchKernelGGL(StatsKernel, dim3(unsigned(d.rows) * unsigned(f.pieces)), dim3(256), 0, stream, p);
        Check(hipGetLastError(), "verify_drafts launch");
    }
    hipLaunchKernelGGL(WalkKernel, dim3(unsigned(s->seqs)), dim3(256), 0, stream, p);
    Check(hipGetLastError(), "verify_drafts launch");
    if (d.rows > 0 && s->max_new > 0) {
        hipLaunchKernelGGL(LeftKernel, dim3(unsigned(s->seqs) * unsigned(f.pieces)), dim3(256), 0, stream, p);
        Check(hipGetLastError(), "verify_drafts launch");
    }
    hipLaunchKernelGGL(NextKernel, dim3(unsigned(s->seqs)), dim3(256), 0, stream, p);
    Check(hipGetLastError(), "verify_drafts launch");
}

}  // namespace kr
