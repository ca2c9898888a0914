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
// Two launches. The first takes the largest logit and the sum of every row, in
// pieces of 8192 values; the last workgroup of a sequence to arrive walks down
// its drafts. In the second a workgroup adds up what is left of 2048 values of a
// sequence's last row, and the last of them to arrive finds the token: its
// piece, its thread's eight values, its place. Where several drafts were drawn
// after one row the walk needs sums over the vocabulary on its way, each after a
// refusal that it cannot foresee: it stops there, and the next launch makes the
// sums of the sequences that wait for one, by many workgroups each, and goes on
// (from the top: the steps up to there are a few hundred operations). After
// kSumRounds such launches a single workgroup makes what sums are left.
//
// What bounds it, on an MI355X: for many rows the first launch, and there no one
// thing: the start of its waves (about 1 ns each), the loads behind it and the
// 64-bit exponentials overlap little. 32 chains of up to 7 over 152064 tokens (bf16,
// 176 rows, 13 thousand waves): 35 us of 49; without the exponentials 26, without
// their sums too 26, without the maximum 24, without the loads as well, so that the
// waves start, find their sequence, arrive and the last of them walks, 16. The bytes
// alone are 11 at a copy's rate. 16 trees of up to 24 over 151936 (fp32, 301 rows,
// 23 thousand waves): 49 us of 61, 42, 42, 41 and 22; the bytes 37. (All of the call
// with bf16 logits, half the bytes: 65.) For one sequence of 5 rows the launches and
// the last workgroups' own steps (12 us and 10; the first without its logits 7.5).
#include <algorithm>

#include "kr_paged.h"

namespace kr {

namespace {

constexpr int kPiece = 8192;    // values of a piece of a row: 32 a thread (of the chains above: pieces of 4096
                                // 41 us for 33; 512 threads 38 for 34, 1024 57; of 16384 the whole call 53.6
                                // for 51.2, the trees 59.7 for 61.4)
constexpr int kEndPiece = 2048; // of a sequence's last row: 8 a thread
constexpr int kMostNew = 1024;  // tokens of a sequence
// Counters of a sequence, a line of memory: arrivals at one line wait for each
// other (32 sampled chains of up to 7, all on one line 90 us, on their own 49).
// The first counts the pieces of its rows, the second those of its end row; the
// third is 1 from the walk to the end of the call. Where `starts` does not
// ascend and two sequences claim a row, a walk may not come; the last launch
// sees that by it, and leaves all of them zero whatever came.
constexpr int kCounters = 32;
enum { kRowsDone, kEndDone, kWalked };
// Launches that make sums for sampled trees. One that finds nothing to do costs
// 2.5 us, one with work 9, a sum by a single workgroup 10 us (32003 tokens) to
// 45 (152064). Two trees of 25 over 151936 tokens: 148 us without these, 41 with.
constexpr int kSumRounds = 3;
constexpr int kNone = -1;       // the type of draft probabilities that are not there

struct RowPart {
    float top;   // largest logit
    int at;      // its first place
    double sum;  // of exp((x - top) / t)
};
struct SeqEnd {
    int row;      // where the walk ended: a row of the sequence
    int refused;  // drafts that were refused there
    int waits;    // the last of them, if the walk waits for the sum after it; else -1
    int pad;
    RowPart stats;
};
struct VerifyParams {
    const void *logits, *draft;
    const int64_t *tokens;
    const int32_t *parents, *starts;
    const float *u, *u_next, *temperature;
    int32_t *path, *path_lens;
    int64_t *next;
    int64_t ld_logits, ld_draft, ld_path;
    int vocab, rows, seqs, max_new, width, pieces, end_pieces;
    RowPart *parts;         // [rows, pieces]
    double *totals;         // [rows]: of a sequence's end row, the sums after its refusals
    double *after;          // [rows]: the sum after the refusal of this draft; -1: not known
    int32_t *refused;       // [rows]: the tokens refused there
    SeqEnd *ends;           // [seqs]
    double *sums;           // [seqs, end_pieces]: of what is left at the end row
    double *sums8;          // [seqs, end_pieces, 256]: of 8 values each
    int32_t *cnt;           // [seqs, kCounters]: arrivals, zero between launches
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

// log2(e) / t; -1 for a temperature that picks the first of the largest.
__device__ __forceinline__ double Slope(float t) { return t > 0.0f ? 1.4426950408889634 / double(t) : -1.0; }
__device__ __forceinline__ double SlopeOf(const VerifyParams &p, int b)
{
    return Slope(p.temperature != nullptr ? p.temperature[b] : 1.0f);
}

template <int DT> struct Val {
    typedef uint16_t T;
    static constexpr T kLow = DT == kBF16 ? 0xff80 : 0xfc00;  // -infinity
    __device__ static float Load(T x) { return Elem<DT>::Load(x); }
};
template <> struct Val<kF32> {
    typedef float T;
    static constexpr T kLow = -INFINITY;
    __device__ static float Load(T x) { return x; }
};

template <int DT>
__device__ __forceinline__ float At(const void *base, int64_t at)
{
    typedef typename Val<DT>::T T;
    return Val<DT>::Load(static_cast<const T *>(base)[at]);
}

// Eight values at `at` of a row of n, as they are; past its end `none`. A row may
// begin anywhere: the loads are 16 bytes wide and as aligned as the values.
template <int DT> struct Raw8 {
    typename Val<DT>::T v[8];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> Load8(const void *base, int64_t row, int at, int n, typename Val<DT>::T none)
{
    typedef typename Val<DT>::T T;
    const T *p = static_cast<const T *>(base) + row + at;
    Raw8<DT> r;
    if (at + 8 <= n) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = at + e < n ? p[e] : none;
    }
    return r;
}

__device__ __forceinline__ float Logit(float x) { return x != x ? -INFINITY : x; }
__device__ __forceinline__ double Chance(float q) { return q > 0.0f ? double(q) : 0.0; }

// 2^z for -1000 <= z <= 0, within 2^-44 of it: z = m / 64 + f with |f| <= 1/128,
// m from the last bits of a sum with 1.5 2^52; 2^f by its series to f^4 (the
// first term left out is below 2^-44), 2^(m % 64 / 64) from a table in LDS and
// the rest by the exponent's bits. 17 operations at the full rate with the
// difference and product that make z, where the series alone took 30, and the
// library's exp three times that.
constexpr int kTable = 64;
struct Pow2 {
    double of[kTable];
    // all threads of the workgroup (at least 64); a barrier follows before its use
    __device__ __forceinline__ void Fill()
    {
        if (threadIdx.x >= kTable) return;
        // sqrt(2) exp(r), r = (j - 32) ln(2) / 64
        const double r = double(int(threadIdx.x) - kTable / 2) * (0x1.62e42fefa39efp-1 / kTable);
        double e = 1.0 / 479001600.0;
        e = __builtin_fma(e, r, 1.0 / 39916800.0);
        e = __builtin_fma(e, r, 1.0 / 3628800.0);
        e = __builtin_fma(e, r, 1.0 / 362880.0);
        e = __builtin_fma(e, r, 1.0 / 40320.0);
        e = __builtin_fma(e, r, 1.0 / 5040.0);
        e = __builtin_fma(e, r, 1.0 / 720.0);
        e = __builtin_fma(e, r, 1.0 / 120.0);
        e = __builtin_fma(e, r, 1.0 / 24.0);
        e = __builtin_fma(e, r, 1.0 / 6.0);
        e = __builtin_fma(e, r, 0.5);
        e = __builtin_fma(e, r, 1.0);
        e = __builtin_fma(e, r, 1.0);
        of[threadIdx.x] = e * 1.4142135623730951;
    }
    __device__ __forceinline__ double operator()(double z) const
    {
        // (three-address sums, the constants in registers: the compiler would
        // move each constant into the sum's own register first)
        double t, s;
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(t) : "v"(z), "v"(double(kTable)), "v"(0x1.8p52));
        const double f = __builtin_fma(t - 0x1.8p52, -1.0 / kTable, z);
        const int m = __double2loint(t);
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(s) : "v"(f), "v"(0.009618129107628477),  // ln(2)^4 / 24
            "v"(0.05550410866482158));                                                        // ln(2)^3 / 6
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(s) : "v"(s), "v"(f), "v"(0.2402265069591007));  // ln(2)^2 / 2
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(s) : "v"(s), "v"(f), "v"(0.6931471805599453));
        const double b = of[m & (kTable - 1)];
        const double w = __builtin_fma(b, s * f, b);
        return __hiloint2double(__double2hiint(w) + ((m & -kTable) << 14), __double2loint(w));
    }
};

constexpr double kFar = -1000.0;  // log2 of a weight that is 0

// exp((x - top) / t), c = log2(e) / t: 1 at the top itself, also an infinite
// one; without a temperature (c < 0) 1 at place `at` alone. (Differences of
// infinities and their products with c = 0 are no numbers.)
__device__ __forceinline__ double Weight(const Pow2 &pow2, float x, int i, float top, int at, double c)
{
    if (c < 0.0) return i == at ? 1.0 : 0.0;
    const double z = (double(x) - double(top)) * c;
    const double w = pow2(fmax(z, kFar));
    return x == top && x != -INFINITY ? 1.0 : x == -INFINITY || top == INFINITY || z < kFar ? 0.0 : w;
}

__device__ __forceinline__ double WaveSumD(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Sum over the NT threads, in every one of them.
template <int NT>
__device__ __forceinline__ double BlockSumD(double v, double *part)
{
    v = WaveSumD(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) s += part[i];
    return s;
}

// 8 bytes to and from other workgroups of the running launch.
__device__ __forceinline__ void PutDev(double *p, double v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double GetDev(const double *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void PutPart(RowPart *p, const RowPart &x)
{
    const uint64_t head = uint64_t(__float_as_uint(x.top)) | (uint64_t(uint32_t(x.at)) << 32);
    PutDev(reinterpret_cast<double *>(p), __builtin_bit_cast(double, head));
    PutDev(&p->sum, x.sum);
}
__device__ __forceinline__ RowPart GetPart(const RowPart *p)
{
    const uint64_t head = __builtin_bit_cast(uint64_t, GetDev(reinterpret_cast<const double *>(p)));
    return RowPart{__uint_as_float(uint32_t(head)), int(head >> 32), GetDev(&p->sum)};
}
// One more of `all` arrivals, by one thread; is it the last? The counter is
// zero again then.
__device__ __forceinline__ bool Arrive(int32_t *cnt, int all)
{
    const bool last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
    if (last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return last;
}

// ---------------------------------------------------------------- the walk
// What is left of a value's probability w after `refused` refusals at a row
// with draft probability q: `totals` are the sums after each, the last one not
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

// Of a sequence's rows, in LDS that the launch sizes by max_new.
struct WalkLds {
    RowPart *stats;
    double *prob;    // of draft i at the row that it follows, before any refusal
    double *totals;  // at the row where the walk is, after each refusal
    float *chance, *u;
    int *above, *token;
    static constexpr int kBytes = sizeof(RowPart) + 2 * sizeof(double) + 4 * 4;
    __device__ __forceinline__ WalkLds(char *lds, int n)
    {
        stats = reinterpret_cast<RowPart *>(lds);
        prob = reinterpret_cast<double *>(stats + n);
        totals = prob + n;
        chance = reinterpret_cast<float *>(totals + n);
        u = chance + n;
        above = reinterpret_cast<int *>(u + n);
        token = above + n;
    }
};

#include "kr_walk.inc"

// Down the drafts of sequence b, by NT threads that all take the same steps.
template <int XT, int QT, int NT, int SUMS>
__device__ __forceinline__ void Walk(const VerifyParams &p, int b, const VerifySeq &sq, double c, const Pow2 &pow2,
                                       const WalkLds &l, double *part)
{
    constexpr int QL = QT == kNone ? kF32 : QT;
    const int tid = int(threadIdx.x), lane = tid & 63;
    // ---- drafts: what they follow
    for (int i = tid; i < sq.n; i += NT) {
        const int64_t tok = p.tokens[sq.first + i];
        const int par = p.parents != nullptr ? p.parents[sq.first + i] : i - 1;
        l.above[i] = i > 0 && par >= 0 && par < i ? par : -1;
        l.token[i] = tok >= 0 && tok < p.vocab ? int(tok) : -1;
        l.u[i] = p.u[sq.first + i];
        if (SUMS == kFirst) PutDev(p.after + sq.first + i, -1.0);
    }
    // ---- rows: their pieces put together, eight lanes to a row
    for (int r0 = 0; r0 < sq.n; r0 += NT / 8) {
        const int r = r0 + tid / 8, l8 = tid % 8;
        const RowPart *parts = p.parts + int64_t(sq.first + min(r, sq.n - 1)) * p.pieces;
        RowPart x{-INFINITY, INT32_MAX, 0.0};
        const auto add = [&](const RowPart &y) {
            // (a part of no logits adds nothing; of two infinite tops both count)
            const float top = fmaxf(x.top, y.top);
            const int ax = x.top == top ? x.at : INT32_MAX, ay = y.top == top ? y.at : INT32_MAX;
            if (c < 0.0) x.sum = 1.0;
            else x.sum = x.sum * Weight(pow2, x.top, 0, top, 0, c) + y.sum * Weight(pow2, y.top, 0, top, 0, c);
            x.top = top;
            x.at = min(ax, ay);
        };
        for (int k = l8; k < p.pieces; k += 32) {
            RowPart y[4];  // (all on their way before the first is used)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = GetPart(parts + min(k + 8 * i, p.pieces - 1));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k + 8 * i < p.pieces) add(y[i]);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            RowPart y;
            y.top = __shfl_xor(x.top, o, 64);
            y.at = __shfl_xor(x.at, o, 64);
            y.sum = __shfl_xor(x.sum, o, 64);
            add(y);
        }
        if (l8 == 0 && r < sq.n) l.stats[r] = x;
    }
    __syncthreads();
    // ---- and how likely they are there
    for (int i = tid; i < sq.n; i += NT) {
        const int par = l.above[i], tok = l.token[i];
        double w = 0.0;
        float q = 1.0f;
        if (par >= 0 && tok >= 0) {
            const RowPart s = l.stats[par];
            const int64_t row = sq.first + par;
            const float x = Logit(At<XT>(p.logits, row * p.ld_logits + tok));
            if (QT != kNone) q = float(Chance(At<QL>(p.draft, row * p.ld_draft + tok)));
            if (s.top != -INFINITY) w = Weight(pow2, x, tok, s.top, s.at, c) / s.sum;
            if (QT == kNone) {
                // a token that was refused there already has nothing left
                for (int j = par + 1; j < i; ++j)
                    if (l.above[j] == par && l.token[j] == tok) w = 0.0;
            }
        }
        l.prob[i] = w;
        l.chance[i] = q;
    }
    __syncthreads();
    const auto known = [&](int gone) { return GetDev(p.after + sq.first + gone); };
    const auto make = [&](int cur, int refused) {
        double sum = 0.0;
        if constexpr (SUMS == kMakes) {
            const RowPart s = l.stats[cur];
            const int64_t row = sq.first + cur;
            const double inv = 1.0 / s.sum;
            for (int v = tid * 8; v < p.vocab; v += NT * 8) {
                const Raw8<XT> x = Load8<XT>(p.logits, row * p.ld_logits, v, p.vocab, Val<XT>::kLow);
                const Raw8<QL> q = Load8<QL>(p.draft, row * p.ld_draft, v, p.vocab, 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (s.top == -INFINITY) continue;
                    double was;
                    const double w = Weight(pow2, Logit(Val<XT>::Load(x.v[e])), v + e, s.top, s.at, c) * inv;
                    sum += Left(w, Chance(Val<QL>::Load(q.v[e])), l.totals, refused, was);
                }
            }
            sum = BlockSumD<NT>(sum, part);
        }
        return sum;
    };
    const WalkEnd at = WalkDown<QT != kNone, SUMS>(l, sq.n, p.width, known, make,
                                                  [&](int len, int i) { p.path[b * p.ld_path + len] = i; });
    const int cur = at.cur, len = at.len, refused = at.refused;
    if (at.waits >= 0) {
        for (int k = tid; k + 1 < refused; k += NT) PutDev(p.totals + sq.first + k, l.totals[k]);
        if (tid == 0) p.ends[b] = SeqEnd{cur, refused, at.waits, 0, l.stats[cur]};
        return;
    }
    if (tid == 0) {
        p.path[b * p.ld_path] = 0;
        p.path_lens[b] = len;
        p.ends[b] = SeqEnd{cur, refused, -1, 0, l.stats[cur]};
    }
    for (int i = len + tid; i < p.width; i += NT) p.path[b * p.ld_path + i] = -1;
    if (QT != kNone) {
        for (int k = tid; SUMS != kNoSums && k + 1 < refused; k += NT) PutDev(p.totals + sq.first + k, l.totals[k]);
    } else if (refused > 0 && tid < 64) {  // (all that follow it)
        int at = 0;
        for (int i0 = (cur + 1) / 64 * 64; i0 < sq.n; i0 += 64) {
            const int i = min(i0 + lane, sq.n - 1);
            const bool is = i0 + lane < sq.n && i0 + lane > cur && l.above[i] == cur;
            const uint64_t hit = __ballot(is);
            if (is) p.refused[sq.first + at + __popcll(hit & ((1ull << lane) - 1))] = l.token[i];
            at += __popcll(hit);
        }
    }
}

__device__ __forceinline__ void NoRows(const VerifyParams &p, int b, int nt)
{
    for (int i = int(threadIdx.x); i < p.width; i += nt) p.path[b * p.ld_path + i] = -1;
    if (threadIdx.x == 0) {
        p.path_lens[b] = 0;
        p.next[b] = -1;
        p.cnt[b * kCounters + kRowsDone] = 0;
    }
}

// Sampled trees whose walk still waits: 1024 threads, as the sums are made by one workgroup.
template <int XT, int QT>
__global__ void __launch_bounds__(1024) WalkKernel(VerifyParams p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ Pow2 pow2;
    __shared__ double part[16];
    const int b = int(blockIdx.x);
    const VerifySeq sq = LoadSeq(p, b);
    if (sq.n == 0 || p.cnt[b * kCounters + kWalked] == 0 || p.ends[b].waits < 0) return;
    const double c = SlopeOf(p, b);
    pow2.Fill();
    __syncthreads();
    Walk<XT, QT, 1024, kMakes>(p, b, sq, c, pow2, WalkLds(lds, p.max_new), part);
}

// The sums that walks wait for: a workgroup has a piece of a row, as in the last
// launch; the last of them goes on with the walk.
template <int XT, int QT>
__global__ void __launch_bounds__(256) SumKernel(VerifyParams p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ Pow2 pow2;
    __shared__ double part[4];
    __shared__ int last;
    const int b = int(blockIdx.x) / p.end_pieces, mine = int(blockIdx.x) - b * p.end_pieces;
    const int tid = int(threadIdx.x);
    const VerifySeq sq = LoadSeq(p, b);
    if (sq.n == 0 || p.cnt[b * kCounters + kWalked] == 0) return;
    const SeqEnd end = p.ends[b];
    if (end.waits < 0) return;
    const double c = SlopeOf(p, b);
    pow2.Fill();
    const int64_t row = sq.first + end.row;
    const int v = mine * kEndPiece + tid * 8;
    const Raw8<XT> x = Load8<XT>(p.logits, row * p.ld_logits, v, p.vocab, Val<XT>::kLow);
    const Raw8<QT> q = Load8<QT>(p.draft, row * p.ld_draft, v, p.vocab, 0);
    __syncthreads();
    double sum = 0.0;
    if (end.stats.top != -INFINITY) {
        const double inv = 1.0 / end.stats.sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            double was;
            const double w = Weight(pow2, Logit(Val<XT>::Load(x.v[e])), v + e, end.stats.top, end.stats.at, c) * inv;
            sum += Left(w, Chance(Val<QT>::Load(q.v[e])), p.totals + sq.first, end.refused, was);
        }
    }
    sum = BlockSumD<256>(sum, part);
    double *sums = p.sums + int64_t(b) * p.end_pieces;
    if (tid == 0) {
        PutDev(sums + mine, sum);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): it is written
        last = Arrive(p.cnt + b * kCounters + kEndDone, p.end_pieces);
    }
    __syncthreads();
    if (!last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    sum = 0.0;
    for (int k = tid; k < p.end_pieces; k += 256) sum += GetDev(sums + k);
    sum = BlockSumD<256>(sum, part);
    if (tid == 0) {
        PutDev(p.after + sq.first + end.waits, sum);
        __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    __syncthreads();
    Walk<XT, QT, 256, kResume>(p, b, sq, c, pow2, WalkLds(lds, p.max_new), part);
}

// ---------------------------------------------------------------- rows
// The last workgroup of a sequence walks.
template <int XT, int QT, int SUMS>
__global__ void __launch_bounds__(256) StatsKernel(VerifyParams p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int last;
    __shared__ Pow2 pow2;
    __shared__ float top_of[4];
    __shared__ int at_of[4];
    __shared__ double part[4];
    const int piece = int(blockIdx.x) % p.pieces, row = int(blockIdx.x) / p.pieces;
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
    const int i0 = piece * kPiece + int(threadIdx.x) * 8;
    Raw8<XT> raw[4];  // (on their way while the row's sequence is looked up)
#pragma unroll
    for (int g = 0; g < 4; ++g) raw[g] = Load8<XT>(p.logits, int64_t(row) * p.ld_logits, i0 + g * 2048, p.vocab, Val<XT>::kLow);
    pow2.Fill();
    int b = -1;
    VerifySeq sq{0, 0};
    float t = 1.0f;
    for (int b0 = 0; b0 < p.seqs && b < 0; b0 += 64) {
        bool mine = false;
        float tb = 1.0f;
        VerifySeq s{0, 0};
        if (b0 + lane < p.seqs) {
            if (p.temperature != nullptr) tb = p.temperature[b0 + lane];
            s = LoadSeq(p, b0 + lane);
            mine = row >= s.first && row < s.first + s.n;
        }
        const uint64_t hit = __ballot(mine);
        if (hit != 0) {
            const int at = __builtin_ctzll(hit);
            b = b0 + at;
            t = __shfl(tb, at, 64);
            sq.first = Uni(__shfl(s.first, at, 64));
            sq.n = Uni(__shfl(s.n, at, 64));
        }
    }
    if (b < 0) return;  // a row of no sequence
    const double c = Slope(t);
    float x[32];
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[g * 8 + e] = Val<XT>::Load(raw[g].v[e]);
            top = fmaxf(top, x[g * 8 + e]);  // (passes a NaN by)
        }
    top = WaveMax(top);
    if (lane == 0) top_of[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
    int at = INT32_MAX;
    double sum = 1.0;
    if (c < 0.0) {
#pragma unroll
        for (int g = 3; g >= 0; --g)
#pragma unroll
            for (int e = 7; e >= 0; --e)
                if (x[g * 8 + e] == top) at = i0 + g * 2048 + e;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
        if (lane == 0) at_of[wave] = at;
        __syncthreads();
        at = min(min(at_of[0], at_of[1]), min(at_of[2], at_of[3]));
    } else {
        double s[2] = {0.0, 0.0};
        if (top == INFINITY) {
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e & 1] += x[e] == top ? 1.0 : 0.0;
        } else if (top != -INFINITY) {
            // (weights below 2^-1000 count as that, nothing beside the top's 1;
            // so do NaNs and -infinity times a slope of 0: fmax passes a NaN by)
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e & 1] += pow2(fmax((double(x[e]) - double(top)) * c, kFar));
        }
        sum = BlockSumD<256>(s[0] + s[1], part);
    }
    if (threadIdx.x == 0) {
        PutPart(&p.parts[int64_t(row) * p.pieces + piece], RowPart{top, at, sum});
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): it is written
        last = Arrive(p.cnt + b * kCounters + kRowsDone, sq.n * p.pieces);
        if (last) p.cnt[b * kCounters + kWalked] = 1;
    }
    __syncthreads();
    if (!last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    Walk<XT, QT, 256, SUMS>(p, b, sq, c, pow2, WalkLds(lds, p.max_new), part);
}

// ---------------------------------------------------------------- the token
// The first thread (of 256, in order) whose inclusive sum, from `base` on, is
// over the bar, else the last one with anything; -1 if none has. `before`: the
// sum ahead of it.
struct Pick {
    int at;
    double before;
    bool over;
};
__device__ __forceinline__ Pick PickThread(double v, double base, double bar, double *part, int *pick, double *ahead)
{
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    double incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(incl, o, 64);
        if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 63) part[wave] = incl;
    if (tid < 8) pick[tid] = -1;
    __syncthreads();
    for (int i = 0; i < wave; ++i) base += part[i];
    const double excl = base + (incl - v);
    const uint64_t over = __ballot(v > 0.0 && base + incl > bar), some = __ballot(v > 0.0);
    // slots 0..3: a wave's first over the bar; 4..7: its last with anything
    if (over != 0 && lane == __builtin_ctzll(over)) pick[wave] = tid, ahead[wave] = excl;
    if (some != 0 && lane == 63 - __builtin_clzll(some)) pick[4 + wave] = tid, ahead[4 + wave] = excl;
    __syncthreads();
    Pick r{-1, 0.0, false};
#pragma unroll
    for (int i = 4; i < 8; ++i)
        if (pick[i] >= 0) r = Pick{pick[i], ahead[i], false};
#pragma unroll
    for (int i = 3; i >= 0; --i)
        if (pick[i] >= 0) r = Pick{pick[i], ahead[i], true};
    return r;
}

template <int XT, int QT>
__global__ void __launch_bounds__(256) NextKernel(VerifyParams p)
{
    __shared__ Pow2 pow2;
    __shared__ uint32_t marks[kEndPiece / 32];  // refused tokens of a piece (drafts that were not drawn)
    __shared__ double part[4], ahead[8];
    __shared__ int pick[8];
    __shared__ int last;
    constexpr int QL = QT == kNone ? kF32 : QT;
    const int b = int(blockIdx.x) / p.end_pieces, mine = int(blockIdx.x) - b * p.end_pieces;
    const int tid = int(threadIdx.x), lane = tid & 63;
    const VerifySeq sq = LoadSeq(p, b);
    if (sq.n == 0 || p.cnt[b * kCounters + kWalked] == 0) {
        if (mine == 0) NoRows(p, b, 256);
        return;
    }
    const double c = SlopeOf(p, b);
    const SeqEnd end = p.ends[b];
    pow2.Fill();
    __syncthreads();
    const int64_t row = sq.first + end.row;
    const double inv = 1.0 / end.stats.sum;
    const double *totals = p.totals + sq.first;
    const auto mark = [&](int v0) {
        if constexpr (QT == kNone) {
            __syncthreads();
            if (tid < kEndPiece / 32) marks[tid] = 0;
            __syncthreads();
            for (int i = tid; i < end.refused; i += 256) {
                const int tok = p.refused[sq.first + i];
                if (tok >= v0 && tok < v0 + kEndPiece) atomicOr(&marks[(tok - v0) >> 5], 1u << (tok & 31));
            }
            __syncthreads();
        }
    };
    // what is left of value v, x its logit and q its draft probability; where
    // nothing is left at all, p before the last refusal (`stays`)
    const auto left_of = [&](int v, float x, float q, bool refused, bool stays) {
        const double w = Weight(pow2, Logit(x), v, end.stats.top, end.stats.at, c);
        if (QT == kNone) return refused && !stays ? 0.0 : w;
        double was;
        const double left = Left(w * inv, Chance(q), totals, end.refused, was);
        return stays ? was : left;
    };
    // a piece's values, 8 in a row for each thread: their sum
    const auto sum_of = [&](int piece, bool stays) {
        const int v0 = piece * kEndPiece, v = v0 + tid * 8;
        const Raw8<XT> x = Load8<XT>(p.logits, row * p.ld_logits, v, p.vocab, Val<XT>::kLow);
        Raw8<QL> q;
        if (QT != kNone) q = Load8<QL>(p.draft, row * p.ld_draft, v, p.vocab, 0);
        mark(v0);
        const uint32_t refused = QT == kNone ? marks[tid >> 2] >> (8 * (tid & 3)) : 0;
        double s = 0.0;
        if (end.stats.top != -INFINITY) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                s += left_of(v + e, Val<XT>::Load(x.v[e]), QT != kNone ? Val<QL>::Load(q.v[e]) : 0.0f,
                             ((refused >> e) & 1) != 0, stays);
        }
        return s;
    };
    double *sums = p.sums + int64_t(b) * p.end_pieces, *sums8 = p.sums8 + int64_t(b) * p.end_pieces * 256;
    // ---- this workgroup's piece; the last one of the sequence goes on
    {
        const double s = sum_of(mine, false);
        PutDev(sums8 + mine * 256 + tid, s);
        const double all = BlockSumD<256>(s, part);
        if (tid == 0) PutDev(sums + mine, all);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's sums are written
        __syncthreads();
        if (tid == 0) last = Arrive(p.cnt + b * kCounters + kEndDone, p.end_pieces);
        __syncthreads();
        if (!last) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        if (tid == 0) p.cnt[b * kCounters + kWalked] = 0;
    }
    const auto total_of = [&] {
        double s = 0.0;
        for (int k = tid; k < p.end_pieces; k += 256) s += GetDev(sums + k);
        return BlockSumD<256>(s, part);
    };
    double total = total_of();
    const bool stays = !(total > 0.0);
    if (stays) {  // nothing is left: all pieces again, by this workgroup
        for (int k = 0; k < p.end_pieces; ++k) {
            const double s = sum_of(k, true);
            PutDev(sums8 + k * 256 + tid, s);
            const double all = BlockSumD<256>(s, part);
            if (tid == 0) PutDev(sums + k, all);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
        total = total_of();
        if (!(total > 0.0)) {
            if (tid == 0) p.next[b] = -1;
            return;
        }
    }
    const double bar = double(p.u_next[b]) * total;
    // its piece
    int piece = 0;
    double base = 0.0, before = 0.0;
    for (int k0 = 0; k0 < p.end_pieces; k0 += 256) {
        const double v = k0 + tid < p.end_pieces ? GetDev(sums + k0 + tid) : 0.0;
        const Pick k = PickThread(v, before, bar, part, pick, ahead);
        if (k.at >= 0) {
            piece = k0 + k.at;
            base = k.before;
        }
        if (k.over || k0 + 256 >= p.end_pieces) break;
        before += BlockSumD<256>(v, part);
    }
    // its eight values
    const Pick t = PickThread(GetDev(sums8 + piece * 256 + tid), base, bar, part, pick, ahead);
    // its place: lanes 0 to 7
    const int v0 = piece * kEndPiece, v = v0 + max(t.at, 0) * 8 + (lane & 7);
    mark(v0);
    if (tid >= 64) return;
    double own = 0.0;
    if (lane < 8 && v < p.vocab)
        own = left_of(v, At<XT>(p.logits, row * p.ld_logits + v),
                      QT != kNone ? At<QL>(p.draft, row * p.ld_draft + v) : 0.0f,
                      QT == kNone && ((marks[(v - v0) >> 5] >> (v & 31)) & 1) != 0, stays);
    double incl = own;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const double x = __shfl_up(incl, o, 64);
        if (lane >= o) incl += x;
    }
    const uint64_t over = __ballot(own > 0.0 && t.before + incl > bar), some = __ballot(own > 0.0);
    if (lane == 0)
        p.next[b] = v + (over != 0 ? __builtin_ctzll(over) : some != 0 ? 63 - __builtin_clzll(some) : 0);
}

struct VerifyShape {
    int pieces, end_pieces;
    size_t parts, totals, after, refused, ends, sums, sums8, bytes;
};

VerifyShape ShapeOf(const kr_drafts &d, const kr_seqs &s)
{
    VerifyShape f{};
    f.pieces = int((int64_t(d.vocab) + kPiece - 1) / kPiece);
    const size_t rows = size_t(d.rows), seqs = size_t(s.seqs);
    f.end_pieces = int((int64_t(d.vocab) + kEndPiece - 1) / kEndPiece);
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 15) / 16 * 16;
        return from;
    };
    f.parts = take(rows * f.pieces * sizeof(RowPart));
    f.totals = take(rows * sizeof(double));
    f.after = take(rows * sizeof(double));
    f.refused = take(rows * sizeof(int32_t));
    f.ends = take(seqs * sizeof(SeqEnd));
    f.sums = take(seqs * f.end_pieces * sizeof(double));
    f.sums8 = take(seqs * f.end_pieces * 256 * sizeof(double));
    f.bytes = at;
    return f;
}

template <int XT, int QT>
void VerifyGo(const VerifyParams &p, hipStream_t stream)
{
    const dim3 rows(unsigned(p.rows) * unsigned(p.pieces)), ends(unsigned(p.seqs) * unsigned(p.end_pieces));
    const unsigned lds = unsigned(p.max_new) * WalkLds::kBytes;
    if (p.rows > 0 && p.max_new > 0) {
        if constexpr (QT != kNone) {
            if (p.parents != nullptr) {
                hipLaunchKernelGGL((StatsKernel<XT, QT, kFirst>), rows, dim3(256), lds, stream, p);
                for (int i = 0; i < kSumRounds; ++i)
                    hipLaunchKernelGGL((SumKernel<XT, QT>), ends, dim3(256), lds, stream, p);
                hipLaunchKernelGGL((WalkKernel<XT, QT>), dim3(unsigned(p.seqs)), dim3(1024), lds, stream, p);
            }
        }
        if (QT == kNone || p.parents == nullptr)
            hipLaunchKernelGGL((StatsKernel<XT, QT, kNoSums>), rows, dim3(256), lds, stream, p);
    }
    hipLaunchKernelGGL((NextKernel<XT, QT>), ends, dim3(256), 0, stream, p);
}

template <int XT>
void VerifyGo(const VerifyParams &p, int qt, hipStream_t stream)
{
    if (qt == kNone) VerifyGo<XT, kNone>(p, stream);
    else if (qt == kBF16) VerifyGo<XT, kBF16>(p, stream);
    else if (qt == kF16) VerifyGo<XT, kF16>(p, stream);
    else VerifyGo<XT, kF32>(p, stream);
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
    if (s->seqs > (1 << 24)) refuse("too many sequences");
    if (s->max_new > kMostNew) refuse("a sequence has at most 1024 new tokens");
    if (d->rows > 1 && (d->ld_logits < d->vocab || (d->draft != nullptr && d->ld_draft < d->vocab)))
        refuse("rows of logits or draft overlap");
    if (d->ld_logits > (int64_t(1) << 40) || d->ld_draft > (int64_t(1) << 40)) refuse("a row stride is too large");
    if (d->vocab > (1 << 30)) refuse("the vocabulary is too large");
    const int64_t pieces = (int64_t(d->vocab) + kPiece - 1) / kPiece;
    const int64_t end_pieces = (int64_t(d->vocab) + kEndPiece - 1) / kEndPiece;
    if (pieces * d->rows >= kMaxGrid || end_pieces * s->seqs >= kMaxGrid) refuse("too many rows for one launch");
    // (kMaxGrid is for workgroups of 256 threads, WalkKernel's have 1024)
    if (d->draft != nullptr && d->parents != nullptr && s->seqs >= (kMaxGrid >> 2)) refuse("too many sequences");
    return *d;
}

}  // namespace

void VerifyNeeds(const kr_drafts *drafts, const kr_seqs *s, size_t *ws_bytes, int *counters)
{
    const kr_drafts d = CheckDrafts(drafts, s);
    *ws_bytes = ShapeOf(d, *s).bytes;
    *counters = s->seqs * kCounters;
}

void VerifyLaunch(const kr_drafts *drafts, const kr_seqs *s, const VerifyOut &o, void *ws, size_t ws_bytes,
                  int32_t *cnt, int cnt_len, hipStream_t stream)
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
    if (ws == nullptr || ws_bytes < f.bytes || off(ws, 16) || cnt == nullptr || cnt_len < s->seqs * kCounters || off(cnt, 4))
        refuse("the workspace is too small or misaligned");
    const MemSpan outs[] = {RowsSpan(o.path, s->seqs, o.ld_path, o.width, 4), RowsSpan(o.path_lens, 1, 0, s->seqs, 4),
                            RowsSpan(o.next, 1, 0, s->seqs, 8), MemSpan{ws, int64_t(f.bytes)},
                            RowsSpan(cnt, 1, 0, s->seqs * kCounters, 4)};
    const MemSpan ins[] = {RowsSpan(d.logits, d.rows, d.ld_logits, d.vocab, size),
                           RowsSpan(d.draft, d.rows, d.ld_draft, d.vocab, dsize), RowsSpan(d.tokens, 1, 0, d.rows, 8),
                           RowsSpan(d.parents, 1, 0, d.rows, 4), RowsSpan(d.u, 1, 0, d.rows, 4),
                           RowsSpan(d.u_next, 1, 0, s->seqs, 4), RowsSpan(d.temperature, 1, 0, s->seqs, 4),
                           RowsSpan(s->starts, 1, 0, s->seqs + 1, 4)};
    for (int i = 0; i < 5; ++i) {
        for (int j = i + 1; j < 5; ++j)
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
    p.vocab = d.vocab;
    p.rows = d.rows;
    p.seqs = s->seqs;
    p.max_new = s->max_new;
    p.width = o.width;
    p.pieces = f.pieces;
    p.end_pieces = f.end_pieces;
    char *base = static_cast<char *>(ws);
    p.parts = reinterpret_cast<RowPart *>(base + f.parts);
    p.totals = reinterpret_cast<double *>(base + f.totals);
    p.after = reinterpret_cast<double *>(base + f.after);
    p.ends = reinterpret_cast<SeqEnd *>(base + f.ends);
    p.sums = reinterpret_cast<double *>(base + f.sums);
    p.sums8 = reinterpret_cast<double *>(base + f.sums8);
    p.refused = reinterpret_cast<int32_t *>(base + f.refused);
    p.cnt = cnt;
    const int qt = d.draft != nullptr ? d.draft_dtype : kNone;
    if (d.dtype == kBF16) VerifyGo<kBF16>(p, qt, stream);
    else if (d.dtype == kF16) VerifyGo<kF16>(p, qt, stream);
    else VerifyGo<kF32>(p, qt, stream);
    Check(hipGetLastError(), "verify_drafts launch");
}

}  // namespace kr
