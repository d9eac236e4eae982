// Every order of events of the tensor-core kernel over shared positions that copies its rows (bf16
// pages): loader warps, MMA warp, softmax warps and the tensor pipe, with the waits and
// arrivals as k_shared_tc.cu has them and the stages of csrc/shared_stages.h. A state is how far
// each of them is. In each that can be reached: whoever passes a wait finds what it waited for, no copy
// goes over what an MMA has still to read, every MMA reads its own step's rows, and somebody can go on.
// The last is done for one barrier for all stages too, which has to fail: the walk sees it.
#include <cstdio>
#include <map>
#include <set>
#include <vector>

#include "shared_stages.h"

namespace {

constexpr int kStages = 3;
using Stage = tie::Stages<kStages>;

enum Bar { Q_FULL, K_FULL, S_FULL, S_FREE, P_FULL, O_FULL, BARS = O_FULL + kStages };
// what a role does next: a wait for a phase, an arrival, or something that has a condition of its own
enum What { WAIT, ARRIVE, COPY, LAND, WRITE_Q, READ_S, WRITE_P, READ_O, ISSUE_S, ISSUE_PV };
struct Op {
    What what;
    int bar;
    int n;                             // phase, step or item
};

struct Walk {
    bool one_barrier;                  // the planted mistake
    std::vector<int> items;            // steps of each
    int loaders;
    std::vector<std::vector<Op>> roles;        // loaders, MMA, softmax
    std::vector<std::pair<bool, int>> pipe;    // (P V, step) in the order of issue
    std::vector<int> first;            // of an item
    const char* wrong = nullptr;

    int o_bar(int step) const { return O_FULL + (one_barrier ? 0 : (int)Stage::of(step)); }
    int o_phase(int step) const { return one_barrier ? step : (int)Stage::phase(step); }

    void programs() {
        int f = 0;
        std::vector<Op> load, mma, soft;
        for (size_t i = 0; i < items.size(); ++i) {
            const int n = items[i], end = f + n;
            first.push_back(f);
            auto copy = [&](int step) {
                if (step >= end) return;
                if (!one_barrier && Stage::used(step)) load.push_back({WAIT, o_bar(Stage::before(step)), o_phase(Stage::before(step))});
                load.push_back({COPY, 0, step});
            };
            auto landed = [&](int step) {
                load.push_back({LAND, 0, step});
                load.push_back({ARRIVE, S_FULL, 0});
                load.push_back({ARRIVE, K_FULL, 0});
            };
            copy(f);
            copy(f + 1);
            load.push_back({WRITE_Q, 0, (int)i});
            load.push_back({ARRIVE, Q_FULL, 0});
            landed(f);
            for (int g = f; g < end; ++g) {
                load.push_back({WAIT, S_FULL, g});
                if (g + 1 < end) landed(g + 1);
                if (g + 2 < end) {
                    if (one_barrier && g) load.push_back({WAIT, O_FULL, g - 1});
                    copy(g + 2);
                }
            }
            if (one_barrier) load.push_back({WAIT, O_FULL, end - 1});

            auto scores = [&](int g) {
                mma.push_back({WAIT, K_FULL, g});
                mma.push_back({ISSUE_S, 0, g});
                pipe.push_back({false, g});
            };
            mma.push_back({WAIT, Q_FULL, (int)i});
            scores(f);
            for (int g = f; g < end; ++g) {
                if (g + 1 < end) {
                    mma.push_back({WAIT, S_FREE, g});
                    scores(g + 1);
                }
                mma.push_back({WAIT, P_FULL, g});
                mma.push_back({ISSUE_PV, 0, g});
                pipe.push_back({true, g});
            }

            for (int g = f; g < end; ++g) {
                soft.push_back({WAIT, S_FULL, g});
                soft.push_back({READ_S, 0, g});
                soft.push_back({ARRIVE, S_FREE, 0});
                if (g > f) {
                    soft.push_back({WAIT, o_bar(g - 1), o_phase(g - 1)});
                    soft.push_back({READ_O, 0, g - 1});
                }
                soft.push_back({WRITE_P, 0, g});
                soft.push_back({ARRIVE, P_FULL, 0});
            }
            soft.push_back({WAIT, o_bar(end - 1), o_phase(end - 1)});
            soft.push_back({READ_O, 0, end - 1});
            f = end;
        }
        for (int i = 0; i < loaders; ++i) roles.push_back(load);
        roles.push_back(mma);
        roles.push_back(soft);
    }

    using State = std::vector<int>;    // each role's place, and how much the pipe has done

    int done(const State& s, int role, What what) const {      // how many of `what` the role has behind it
        int n = 0;
        for (int i = 0; i < s[role]; ++i) n += roles[role][i].what == what;
        return n;
    }
    bool piped(const State& s, bool pv, int step) const {
        for (int i = 0; i < s.back(); ++i)
            if (pipe[i].first == pv && pipe[i].second == step) return true;
        return false;
    }
    // phases that a barrier has behind it: its arrivals are a matter of the places
    int phases(const State& s, int bar) const {
        int n = 0, all = bar == S_FULL ? 1 + loaders : bar == Q_FULL || bar == K_FULL ? loaders : 1;
        for (size_t r = 0; r < roles.size(); ++r)
            for (int i = 0; i < s[r]; ++i) n += roles[r][i].what == ARRIVE && roles[r][i].bar == bar;
        for (int i = 0; i < s.back(); ++i) n += pipe[i].first ? o_bar(pipe[i].second) == bar : bar == S_FULL;
        return n / all;
    }

    // false: not yet
    bool may(const State& s, int role, const Op& op) {
        const int mma = loaders, soft = loaders + 1;
        switch (op.what) {
            case WAIT: {
                const int c = phases(s, op.bar);
                if ((c & 1) == (op.n & 1)) return false;       // (the phase that it is in has this parity)
                if (c <= op.n) wrong = "a wait is over before its phase";
                return true;
            }
            case COPY:
                if (op.n >= kStages) {
                    const int old = op.n - kStages;
                    if (!piped(s, false, old) || !piped(s, true, old)) wrong = "a copy over rows that an MMA has still to read";
                }
                return true;
            case WRITE_Q:
                if (op.n && !piped(s, false, first[op.n] - 1)) wrong = "Q written while it is read";
                return true;
            case READ_S:
                if (!piped(s, false, op.n)) wrong = "S read before it is computed";
                if (piped(s, false, op.n + 1) && done(s, mma, ISSUE_S) > op.n + 1) wrong = "S of another step read";
                return true;
            case WRITE_P:
                if (op.n && !piped(s, true, op.n - 1)) wrong = "P written while it is read";
                return true;
            case READ_O:
                if (!piped(s, true, op.n)) wrong = "O read before it is computed";
                if (done(s, mma, ISSUE_PV) > op.n + 1) wrong = "O of another step read";
                return true;
            case ISSUE_S:
                for (int l = 0; l < loaders; ++l)
                    if (done(s, l, LAND) <= op.n || done(s, l, COPY) > op.n + kStages) wrong = "S of rows that are not there";
                if (done(s, soft, READ_S) < op.n) wrong = "S written before it is read";
                return true;
            case ISSUE_PV:
                for (int l = 0; l < loaders; ++l)
                    if (done(s, l, COPY) > op.n + kStages) wrong = "P V of another step's rows";
                if (done(s, soft, WRITE_P) <= op.n) wrong = "P V before P";
                if (done(s, soft, READ_O) < op.n) wrong = "O written before it is read";
                return true;
            default:
                return true;
        }
    }

    // what goes wrong, or nullptr
    const char* run(size_t* states) {
        programs();
        std::set<State> seen;
        std::vector<State> open{State(roles.size() + 1, 0)};
        seen.insert(open[0]);
        while (!open.empty()) {
            const State s = open.back();
            open.pop_back();
            bool went = false, over = s.back() == (int)pipe.size();
            for (size_t r = 0; r <= roles.size(); ++r) {
                State next = s;
                ++next[r];
                if (r < roles.size()) {
                    if (s[r] == (int)roles[r].size()) continue;
                    over = false;
                    if (!may(s, (int)r, roles[r][s[r]])) continue;
                    if (wrong) return wrong;
                } else {                               // the pipe completes what was issued, in order
                    const int issued = done(s, loaders, ISSUE_S) + done(s, loaders, ISSUE_PV);
                    if (s.back() >= issued) continue;
                    for (int l = 0; l < loaders; ++l)
                        if (done(s, l, COPY) > pipe[s.back()].second + kStages) return "an MMA reads another step's rows";
                }
                went = true;
                if (seen.insert(next).second) open.push_back(next);
            }
            if (!went && !over) return "nobody can go on";
        }
        *states = seen.size();
        return nullptr;
    }
};

}  // namespace

int main() {
    size_t states = 0, all = 0;
    std::map<const char*, int> planted;
    for (int loaders = 1; loaders <= 2; ++loaders)
        for (int a = 1; a <= 5; ++a)
            for (int b = 0; b <= (loaders == 1 ? 5 : 4); ++b)
                for (int c = 0; c <= (b && loaders == 1 ? 3 : 0); ++c) {
                    std::vector<int> items{a};
                    if (b) items.push_back(b);
                    if (c) items.push_back(c);
                    Walk good{false, items, loaders, {}, {}, {}};
                    if (const char* wrong = good.run(&states)) {
                        std::printf("items %d %d %d, %d loaders: %s\n", a, b, c, loaders, wrong);
                        return 1;
                    }
                    all += states;
                    Walk bad{true, items, loaders, {}, {}, {}};
                    if (const char* wrong = bad.run(&states)) ++planted[wrong];
                }
    if (planted.empty()) {
        std::printf("the walk does not see one barrier for all stages fail\n");
        return 1;
    }
    std::fprintf(stderr, "%zu states\n", all);
    for (const auto& p : planted) std::fprintf(stderr, "one barrier: %s, %d times\n", p.first, p.second);
    std::printf("ok\n");
    return 0;
}
