// The walk down a tree of drafts (kr_walk.inc) on the CPU, a thread for each lane
// of two waves: its steps against a plain walk, and the order of what the lanes
// read and write at the sums that they share. Between two barriers of the
// workgroup a place that one wave writes is no other wave's: whether a run's
// timing shows the difference does not matter here. Prints what is wrong.
#include <pthread.h>
#include <unistd.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <map>
#include <mutex>
#include <random>
#include <set>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline

constexpr int kWaves = 2, kThreads = 64 * kWaves;
struct Index {
    int x;
};
thread_local Index threadIdx;
thread_local int epoch;  // barriers of the workgroup so far
pthread_barrier_t all_lanes, wave_lanes[kWaves];
std::atomic<uint64_t> votes[kWaves];

void __syncthreads()
{
    pthread_barrier_wait(&all_lanes);
    ++epoch;
}
uint64_t __ballot(bool mine)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (mine) votes[wave].fetch_or(1ull << lane);
    pthread_barrier_wait(&wave_lanes[wave]);
    const uint64_t r = votes[wave];
    pthread_barrier_wait(&wave_lanes[wave]);
    if (lane == 0) votes[wave] = 0;
    pthread_barrier_wait(&wave_lanes[wave]);
    return r;
}
int Uni(int v) { return v; }

#include "kr_walk.inc"

// A shared array that notes who reads and writes where, and between which barriers.
std::mutex noting;
struct Notes {
    std::set<int> readers, writers;
};
std::map<std::pair<int, int>, Notes> notes;  // (place, epoch)
struct Shared {
    double *v;
    struct Place {
        double *v;
        int at;
        void note(bool writes) const
        {
            std::lock_guard<std::mutex> hold(noting);
            Notes &n = notes[{at, epoch}];
            (writes ? n.writers : n.readers).insert(threadIdx.x >> 6);
        }
        operator double() const
        {
            note(false);
            return *v;
        }
        void operator=(double x) const
        {
            note(true);
            *v = x;
        }
    };
    Place operator[](int i) const { return Place{v + i, i}; }
};
struct Lds {
    const int *above;
    const double *prob;
    const float *chance, *u;
    Shared totals;
};

struct Tree {
    std::vector<int> above;
    std::vector<double> prob, after;  // after: the sum after the refusal of this draft
    std::vector<float> chance, u;
};

struct Steps {
    WalkEnd end;
    std::vector<int> path;
    int rows;  // that needed a sum
};

// Row by row, by one thread. known: the sums that are there (else -1).
Steps Plain(const Tree &t, int width, bool drawn, int sums, const std::vector<double> &known)
{
    Steps s{{0, 1, 0, -1}, {0}, 0};
    const int n = int(t.above.size());
    for (bool on = true; on && s.end.len < width;) {
        on = false;
        s.end.refused = 0;
        double rest = 1.0;
        std::vector<double> totals;
        for (int i = s.end.cur + 1, gone = -1; i < n && !on; ++i) {
            if (t.above[i] != s.end.cur) continue;
            bool ok;
            if (!drawn) {
                ok = double(t.u[i]) * rest < t.prob[i];
                rest = std::max(rest - t.prob[i], 0.0);
            } else {
                if (sums != kNoSums && s.end.refused > 0) {
                    if (sums == kFirst || (sums == kResume && known[gone] < 0.0)) {
                        s.end.waits = gone;
                        return s;
                    }
                    totals.push_back(t.after[gone]);
                    s.rows += totals.size() == 1;
                }
                double r = t.prob[i];
                for (double total : totals) r = total > 0.0 ? std::max(r - double(t.chance[i]), 0.0) / total : r;
                ok = double(t.u[i]) * double(t.chance[i]) < r;
            }
            if (ok) {
                on = true;
                s.path.push_back(i);
                s.end = WalkEnd{i, s.end.len + 1, 0, -1};
            } else {
                ++s.end.refused;
                gone = i;
            }
        }
    }
    return s;
}

template <bool DRAWN, int SUMS>
int Run(const Tree &t, int width, const std::vector<double> &known, const char *what, int seed, int &rows)
{
    const int n = int(t.above.size());
    std::vector<double> totals(n, 0.0);
    std::vector<int> path(n + 1, -1);
    std::vector<WalkEnd> ends(kThreads);
    std::vector<int> epochs(kThreads);
    const Lds l{t.above.data(), t.prob.data(), t.chance.data(), t.u.data(), Shared{totals.data()}};
    path[0] = 0;
    notes.clear();
    std::vector<std::thread> lanes;
    for (int x = 0; x < kThreads; ++x)
        lanes.emplace_back([&, x] {
            threadIdx.x = x;
            epoch = 0;
            const auto make = [&](int cur, int refused) {  // (reads as the sum over the vocabulary does)
                volatile double sink = 0.0;
                for (int k = 0; k + 1 < refused; ++k) sink = sink + l.totals[k];
                __syncthreads();
                __syncthreads();
                for (int i = cur + 1, nth = 0; i < n; ++i)
                    if (t.above[i] == cur && ++nth == refused) return t.after[i];
                return -1.0;
            };
            ends[x] = WalkDown<DRAWN, SUMS>(l, n, width, [&](int i) { return known[i]; }, make,
                                            [&](int len, int i) { path[len] = i; });
            epochs[x] = epoch;
        });
    for (std::thread &x : lanes) x.join();
    const Steps want = Plain(t, width, DRAWN, SUMS, known);
    int bad = 0;
    const auto wrong = [&](const char *text) {
        if (bad++ == 0) std::printf("%s, tree %d: %s\n", what, seed, text);
    };
    for (int x = 0; x < kThreads; ++x) {
        const WalkEnd &e = ends[x];
        if (e.cur != want.end.cur || e.len != want.end.len || e.refused != want.end.refused || e.waits != want.end.waits)
            wrong("a lane ended elsewhere than the plain walk");
        if (epochs[x] != epochs[0]) wrong("lanes met other numbers of barriers");
    }
    for (size_t i = 0; i < want.path.size(); ++i)
        if (path[i] != want.path[i]) wrong("another path");
    for (const auto &at : notes) {
        std::set<int> seen = at.second.readers;
        seen.insert(at.second.writers.begin(), at.second.writers.end());
        if (!at.second.writers.empty() && seen.size() > 1) wrong("a sum is written while another wave may read it");
    }
    rows = std::max(rows, want.rows);
    return bad;
}

int main()
{
    alarm(100);  // (lanes that wait at different barriers)
    pthread_barrier_init(&all_lanes, nullptr, kThreads);
    for (pthread_barrier_t &b : wave_lanes) pthread_barrier_init(&b, nullptr, 64);
    int bad = 0, rows = 0;
    for (int seed = 0; seed < 24; ++seed) {
        std::mt19937 g(seed);
        const auto real = [&] { return std::uniform_real_distribution<double>(0.0, 1.0)(g); };
        Tree t;
        const int n = seed % 3 == 0 ? 150 : 20 + 4 * seed;
        for (int i = 0; i < n; ++i) {
            t.above.push_back(i == 0 ? -1 : seed % 2 == 0 ? (i - 1) / 4 : std::max(0, i - 1 - int(real() * 5)));
            const bool good = real() < 0.4;  // (likely to pass, after a refusal too)
            t.prob.push_back(good ? 0.6 + 0.3 * real() : 0.05 * real());
            t.chance.push_back(float(good ? 0.2 * real() : 0.4 + 0.5 * real()));
            t.u.push_back(float(real()));
            t.after.push_back(0.2 + 0.8 * real());
        }
        std::vector<double> none(n, -1.0), some(t.after);
        for (double &x : some)
            if (real() < 0.3) x = -1.0;
        int unused = 0;
        bad += Run<true, kFirst>(t, n, none, "first", seed, unused);
        bad += Run<true, kResume>(t, n, t.after, "resumed", seed, rows);
        bad += Run<true, kResume>(t, n, some, "resumed in part", seed, unused);
        bad += Run<true, kMakes>(t, n, some, "makes some", seed, rows);
        bad += Run<true, kMakes>(t, n, none, "makes all", seed, rows);
        bad += Run<false, kNoSums>(t, 1 + seed, none, "not drawn", seed, unused);
        for (int i = 0; i < n; ++i) t.above[i] = i - 1;
        bad += Run<true, kNoSums>(t, n, none, "chain", seed, unused);
    }
    if (rows < 2) std::printf("no walk needed sums at two rows\n"), ++bad;
    std::printf(bad == 0 ? "ok\n" : "%d wrong\n", bad);
    return bad != 0;
}
