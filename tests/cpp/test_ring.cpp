// The way out of a warp that fills a ring itself and gives up in the middle (csrc/ring.h): the loads that it then waits for are those
// in flight, each by the phase that it completes. A wait for another phase passes while the load is still on its way (it would land in
// shared memory that belongs to somebody else by then), or runs until its limit.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "ring.h"

using namespace srhpm;

namespace {

struct Barrier {
    uint32_t armed = 0, complete = 0;  // phases
    bool     passes(uint32_t parity) const { return (complete & 1) != parity; }  // of a wait by parity
};

int fails = 0;
void want(bool x, const char * what, uint32_t n, uint32_t steps, uint32_t at) {
    if (!x) {
        if (fails++ < 10) std::printf("%s: %u slots, %u steps, gives up in step %u\n", what, n, steps, at);
    }
}

// a warp of `steps` steps whose loads from number `at` on do not land, so that it gives up in step `at`
void run(uint32_t n, uint32_t steps, uint32_t at) {
    std::vector<Barrier> bar(n);
    uint32_t             sent = 0;
    int                  idle = steps ? -1 : 0;
    auto                 issue = [&](uint32_t slot) {
        if (idle >= 0) {
            idle++;
            return;
        }
        want(slot == ring_slot(sent, n), "slot", n, steps, at);
        want(bar[slot].armed == bar[slot].complete, "a slot is armed twice", n, steps, at);
        bar[slot].armed++;
        sent++;
        if (sent == steps) idle = 0;
    };
    for (uint32_t s = 0; s < n; s++) issue(s);
    uint32_t stage = 0, use = 0;
    for (uint32_t step = 0; step < at; step++) {  // loads land in any order; one by one is the hardest case for the way out
        Barrier & b = bar[stage];
        want(!b.passes(use & 1), "the step's wait passes before its load", n, steps, at);
        b.complete++;
        want(b.passes(use & 1), "the step's wait does not pass", n, steps, at);
        issue(stage);
        if (++stage == n) {
            stage = 0;
            use++;
        }
    }
    const uint32_t done = use * n + stage, issued = ring_issued(done, n, idle);
    want(done == at && issued == sent, "loads sent", n, steps, at);
    std::vector<bool> seen(n, false);
    for (uint32_t c = done; c < issued; c++) {
        const uint32_t slot = ring_slot(c, n), parity = ring_parity(c, n);
        Barrier &      b = bar[slot];
        want(b.armed == b.complete + 1, "a slot without a load", n, steps, at);
        want(!b.passes(parity), "passes while the load is on its way", n, steps, at);
        b.complete++;
        want(b.passes(parity), "does not pass when it has landed", n, steps, at);
        seen[slot] = true;
    }
    for (uint32_t s = 0; s < n; s++) want(bar[s].armed == bar[s].complete, "a load is left", n, steps, at);
}

}  // namespace

int main() {
    for (uint32_t n = 2; n <= 6; n++) {
        for (uint32_t steps = 0; steps <= 5 * n; steps++) {
            for (uint32_t at = 0; at <= steps; at++) run(n, steps, at);
        }
    }
    std::printf(fails ? "FAILED\n" : "ok\n");
    return fails != 0;
}
