// Replay of the many-row attention kernel's barriers (hayai_b200/csrc/attn_many.cu) on the host.
//
// Every role of a block is a straight list of waits and arrivals, made from a random list of segments.  The
// roles are stepped in random orders, some of them with one role as far ahead as it gets.  A wait for the
// n-th phase of a barrier goes by the phase's parity, so it is sound only while n or n + 1 phases are
// complete: anything else is reported.  Prints the number of unsound waits found and of replays that stood still.
//
//     attn_phases <replays> <seed>       with -DEARLY=1: the first units look at V before their scores
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "attn_phases.h"

struct Step {
    int kind, bar, phase;  // 0: wait for the phase; 1: arrive; 2: arrive once all products so far are done
};
struct Bar {
    int count, pending, done;
};
struct Seg {
    int units, halves;
    std::vector<char> full;  // [unit][half]: no look at V
};

#ifdef EARLY
static bool early_look(int, int) { return true; }
#else
static bool early_look(int st, int lo) { return hc::many_early_look(st, lo); }
#endif

int main(int argc, char** argv) {
    const int replays = argc > 1 ? atoi(argv[1]) : 200;
    std::mt19937 rng(argc > 2 ? atoi(argv[2]) : 1);
    auto pick = [&](int n) { return (int)(rng() % n); };
    long unsound = 0, stuck = 0;
    for (int rep = 0; rep < replays; ++rep) {
        const bool i8 = rep % 3 == 0;
        const int NB = hc::many_ring(i8, pick(2) ? 64 : 128);
        std::vector<Seg> segs(1 + pick(12));
        for (Seg& s : segs) {
            s.units = 1 + (pick(3) ? pick(5) : pick(14));
            s.halves = 1 + pick(2);
            for (int i = 0; i < 2 * s.units; ++i) s.full.push_back(pick(3) == 0);
        }
        const int N = (int)segs.size();
        // barriers
        const int FULL = 0, EMPTY = NB, S = 2 * NB, P = S + 2, O = P + 2, Q = O + 2, QF = Q + 2, SEG = QF + 2, SEGE = SEG + 4, CHK = SEGE + 4;
        std::vector<Bar> bars(CHK + 2);
        auto init = [&](int at, int n, int count) { for (int i = 0; i < n; ++i) bars[at + i] = {count, count, 0}; };
        init(FULL, NB, 4), init(EMPTY, NB, 1), init(S, 2, 1), init(P, 2, 4), init(O, 2, 1), init(Q, 2, 2), init(QF, 2, 1);
        init(SEG, 4, 1), init(SEGE, 4, 15), init(CHK, 2, 4);
        std::vector<std::vector<Step>> roles;
        auto wait = [&](int bar, int phase) { if (phase >= 0) roles.back().push_back({0, bar, phase}); };
        auto arrive = [&](int bar) { roles.back().push_back({1, bar, 0}); };
        auto commit = [&](int bar) { roles.back().push_back({2, bar, 0}); };
        for (int w = 0; w < 8; ++w) {  // the rows' warps
            roles.emplace_back();
            const int h = w >> 2;
            int ph_s = 0, ph_o = 0, checks = 0, unit = 0;
            for (int n = 0; n < N; ++n) {
                wait(SEG + n % 4, n / 4);
                const int kvt = 2 * unit;
                unit += segs[n].units;
                arrive(SEGE + n % 4);
                if (h >= segs[n].halves) continue;
                for (int st = 0; st < segs[n].units; ++st) {
                    const int vt = kvt + 2 * st + 1;
                    if (!i8 && !segs[n].full[2 * st + h]) {
                        if (!early_look(st, 0)) wait(S + h, ph_s);
                        wait(FULL + vt % NB, vt / NB);
                        arrive(CHK + h);
                        wait(CHK + h, checks++);
                    }
                    wait(S + h, ph_s++);
                    if (i8) wait(FULL + vt % NB, vt / NB);
                    arrive(P + h);
                }
                wait(O + h, ph_o++);
            }
            wait(SEG + N % 4, N / 4);
        }
        for (int w = 0; w < 4; ++w) {  // keys and values in
            roles.emplace_back();
            int t_issue = 0, t_done = 0;
            auto hand_on = [&]() {
                const int t = t_done++;
                if (i8) wait(EMPTY + t % NB, t / NB - 1);
                arrive(FULL + t % NB);
            };
            for (int n = 0; n < N; ++n) {
                wait(SEG + n % 4, n / 4);
                arrive(SEGE + n % 4);
                for (int st = 0; st < 2 * segs[n].units; ++st) {
                    if (t_issue - t_done == 3) hand_on();
                    const int t = t_issue++;
                    if (!i8) wait(EMPTY + t % NB, t / NB - 1);
                }
            }
            wait(SEG + N % 4, N / 4);
            while (t_done < t_issue) hand_on();
        }
        {  // the products
            roles.emplace_back();
            int ph_p[2] = {0, 0}, ph_q[2] = {0, 0}, t = 0;
            for (int n = 0; n < N; ++n) {
                wait(SEG + n % 4, n / 4);
                arrive(SEGE + n % 4);
                const int nu = segs[n].units, halves = segs[n].halves;
                auto scores = [&](int h, bool last) {
                    commit(S + h);
                    if (last) commit(QF + h);
                };
                wait(FULL + t % NB, t / NB);
                for (int h = 0; h < halves; ++h) {
                    wait(Q + h, ph_q[h]++);
                    scores(h, nu == 1);
                }
                commit(EMPTY + t % NB);
                for (int u = 0; u < nu; ++u, t += 2) {
                    wait(FULL + (t + 1) % NB, (t + 1) / NB);
                    if (u + 1 < nu) wait(FULL + (t + 2) % NB, (t + 2) / NB);
                    for (int h = 0; h < halves; ++h) {
                        wait(P + h, ph_p[h]++);
                        if (u + 1 < nu) scores(h, u + 2 == nu);
                        else commit(O + h);
                    }
                    commit(EMPTY + (t + 1) % NB);
                    if (u + 1 < nu) commit(EMPTY + (t + 2) % NB);
                }
            }
            wait(SEG + N % 4, N / 4);
        }
        roles.emplace_back();  // the segments
        for (int n = 0; n <= N; ++n) {
            wait(SEGE + n % 4, n / 4 - 1);
            arrive(SEG + n % 4);
        }
        for (int w = 0; w < 2; ++w) {  // the queries
            roles.emplace_back();
            int ph_qf[2] = {-1, -1};
            for (int n = 0; n < N; ++n) {
                wait(SEG + n % 4, n / 4);
                arrive(SEGE + n % 4);
                for (int h = 0; h < segs[n].halves; ++h) {
                    wait(QF + h, ph_qf[h]++);
                    arrive(Q + h);
                }
            }
            wait(SEG + N % 4, N / 4);
        }

        std::vector<size_t> at(roles.size(), 0);
        std::vector<int> queue;  // the tensor cores' arrivals, in order
        size_t qat = 0;
        auto done_at = [&](int bar) {
            if (--bars[bar].pending == 0) bars[bar].pending = bars[bar].count, ++bars[bar].done;
        };
        const int R = (int)roles.size();
        const int ahead = pick(3) ? pick(R + 1) : -1;  // a role that runs whenever it can
        bool told = false;
        auto check = [&]() {  // every wait that a role stands at
            for (int r = 0; r < R; ++r) {
                if (at[r] >= roles[r].size()) continue;
                const Step& s = roles[r][at[r]];
                if (s.kind == 0 && (bars[s.bar].done < s.phase || bars[s.bar].done > s.phase + 1)) {
                    if (!told) ++unsound;
                    told = true;
                }
            }
        };
        for (;;) {
            auto can = [&](int r) {
                if (r == R) return qat < queue.size();
                if (at[r] >= roles[r].size()) return false;
                const Step& s = roles[r][at[r]];
                return s.kind != 0 || bars[s.bar].done > s.phase;
            };
            int r = -1;
            if (ahead >= 0 && can(ahead)) {
                r = ahead;
            } else {
                std::vector<int> free_roles;
                for (int i = 0; i <= R; ++i)
                    if (can(i)) free_roles.push_back(i);
                if (free_roles.empty()) break;
                r = free_roles[pick((int)free_roles.size())];
            }
            if (r == R) {
                done_at(queue[qat++]);
            } else {
                const Step s = roles[r][at[r]++];
                if (s.kind == 1) done_at(s.bar);
                if (s.kind == 2) queue.push_back(s.bar);
            }
            check();
        }
        for (int r = 0; r < R; ++r)
            if (at[r] < roles[r].size()) {
                ++stuck;
                break;
            }
    }
    printf("%ld %ld\n", unsound, stuck);
    return 0;
}
