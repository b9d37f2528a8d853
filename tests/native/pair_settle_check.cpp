// An SM pair's full barriers under random schedules that stop anywhere, settled by
// tpt_infer_b200/csrc/pair_settle.h: every stage's phase ends when its last copy has
// landed, neither before nor never.
//
//   g++ -O2 -o pair_settle_check pair_settle_check.cpp && ./pair_settle_check <schedules>
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <vector>

#include "../../tpt_infer_b200/csrc/pair_settle.h"

namespace {

constexpr int S = 6;

// an mbarrier of one arrival: `phases` of them have ended
struct Bar {
    int pending = 1, phases = 0;
    long long tx = 0;
    void step() {
        if (pending == 0 && tx == 0) {
            pending = 1;
            phases++;
        }
    }
    void arrive_expect(uint32_t bytes) {
        tx += bytes;
        pending--;
        step();
    }
    void complete(uint32_t bytes) {
        tx -= bytes;
        step();
    }
};

struct Copy {
    int stage;
    uint32_t bytes;
};

int run(unsigned seed) {
    std::mt19937 rng(seed);
    auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
    const int total = 1 + below(30), stop = below(150), kblocks = 1 + below(5);
    std::vector<uint32_t> tile_bytes(total);
    for (auto &b : tile_bytes) b = 16384u + (16384u >> below(3));
    auto bytes = [&](int i) { return tile_bytes[i / kblocks]; };
    Bar full[S];
    std::vector<Copy> flight;
    int issued[2] = {0, 0}, commits = 0;
    auto land = [&]() {
        const int at = below((int)flight.size());
        const Copy c = flight[at];
        flight.erase(flight.begin() + at);
        full[c.stage % S].complete(c.bytes);
    };
    for (int step = 0; step < stop; step++) {
        const int what = below(4);
        if (what < 2) {  // a producer, the leader's or the other's
            int &n = issued[what];
            if (n < total && n < commits + S) {
                if (what == 0) full[n % S].arrive_expect(2 * bytes(n));
                flight.push_back({n, bytes(n)});
                n++;
            }
        } else if (what == 2) {
            if (!flight.empty()) land();
        } else if (full[commits % S].phases > commits / S) {
            commits++;  // the MMAs have read the stage
        }
    }
    const int mine = issued[0], theirs = issued[1], last = mine > theirs ? mine : theirs;
    for (int i = last > S ? last - S : 0; i < last; i++) {
        const tpt::PairSettle p = tpt::pair_settle(i, mine, theirs, bytes(i));
        if (p.arrive) full[i % S].arrive_expect(p.expect);
        if (p.complete) full[i % S].complete(p.complete);
    }
    for (;;) {
        for (int i = last > S ? last - S : 0; i < last; i++) {
            int left = 0;
            for (const Copy &c : flight) left += c.stage == i;
            if ((full[i % S].phases == i / S + 1) != (left == 0) || full[i % S].phases > i / S + 1) {
                printf("schedule %u: stage %d of %d and %d, %d copies in flight, %d phases\n", seed, i, mine, theirs, left,
                       full[i % S].phases);
                return 1;
            }
        }
        if (flight.empty()) return 0;
        if (flight[0].stage < last - S) {
            printf("schedule %u: a copy of stage %d is not waited for\n", seed, flight[0].stage);
            return 1;
        }
        land();
    }
}

}  // namespace

int main(int argc, char **argv) {
    const int n = argc > 1 ? atoi(argv[1]) : 1000;
    int bad = 0;
    for (int i = 0; i < n; i++) bad += run((unsigned)i);
    printf("%d schedules, %d wrong\n", n, bad);
    return bad != 0;
}
