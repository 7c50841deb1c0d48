// One CTA, or a pair, of the lm_head's product as a model: copying, multiplying and adding warps, barriers with phases, copies and
// arrivals that take effect in any order, and warps that give up at any wait that is not ready.  After they stopped, the drain of
// rs_head_drain.cuh runs.  Every wait of the drain must end, and afterwards nothing may be on its way.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "rs_head_drain.cuh"

using namespace rs;
typedef std::mt19937 Rng;

struct Bar {
    int want = 1, pending = 1, tx = 0;
    uint32_t done = 0;      // phases completed
    void init(int n) { want = pending = n; }
    void check() {
        if (pending < 0) { printf("one arrival too many\n"); exit(1); }
        if (pending == 0 && tx == 0) { done++; pending = want; }
    }
    void arrive() { pending--; check(); }
    void arrive_expect(int bytes) { tx += bytes; arrive(); }
    void complete(int bytes) { tx -= bytes; check(); }
    bool ready(uint32_t parity) const { return (done & 1u) != parity; }
};
struct Event {      // a copy that lands, or an arrival of finished products, at CTA `at`
    Bar* bar;
    int bytes;      // 0: an arrival
};

struct Model {
    int ctas;
    uint32_t stages, bufs, steps;
    Bar full[16], empty[2][16], sfull[2][4], sempty[4];
    bool gave_up[2] = {false, false};
    uint32_t issued[2] = {0, 0}, products = 0, added[2] = {0, 0};
    bool copy_stopped[2] = {false, false}, mma_stopped = false, add_stopped[2] = {false, false};
    std::vector<Event> events;
    std::vector<Event> commits;      // of products, in the order of their steps: four arrivals each

    Model(int c, uint32_t s, uint32_t b, uint32_t n) : ctas(c), stages(s), bufs(b), steps(n) {
        for (auto& x : full) x.init(ctas);
        for (auto& x : sempty) x.init(ctas);
        if (ctas == 1) copy_stopped[1] = add_stopped[1] = true;
    }
    // one warp's next wait: 1 ready, 0 not yet, -1 gives up
    int wait(int cta, const Bar& b, uint32_t parity, double patience, Rng& rng) {
        if (b.ready(parity)) return 1;
        if (gave_up[cta]) return -1;
        if (std::uniform_real_distribution<>(0, 1)(rng) < patience) return 0;
        gave_up[cta] = true;
        return -1;
    }
    void copy(int r, double p, Rng& rng) {
        const uint32_t k = issued[r], s = k % stages;
        if (k == steps) { copy_stopped[r] = true; return; }
        if (k >= stages) {
            const int w = wait(r, empty[r][s], ((k / stages) & 1u) ^ 1u, p, rng);
            if (w < 0) copy_stopped[r] = true;
            if (w <= 0) return;
        }
        full[s].arrive_expect(2);
        events.push_back({&full[s], 1});      // weights and tokens
        events.push_back({&full[s], 1});
        issued[r]++;
    }
    void multiply(double p, Rng& rng) {
        const uint32_t k = products, s = k % stages;
        if (k == steps) { mma_stopped = true; return; }
        int w = wait(0, full[s], (k / stages) & 1u, p, rng);
        if (w > 0 && k >= bufs) w = wait(0, sempty[k % bufs], ((k / bufs) & 1u) ^ 1u, p, rng);
        if (w < 0) mma_stopped = true;
        if (w <= 0) return;
        for (int c = 0; c < ctas; c++) {
            commits.push_back({&sfull[c][k % bufs], 0});
            commits.push_back({&empty[c][s], 0});
        }
        products++;
    }
    void add(int r, double p, Rng& rng) {
        const uint32_t k = added[r];
        if (k == steps) { add_stopped[r] = true; return; }
        const int w = wait(r, sfull[r][k % bufs], (k / bufs) & 1u, p, rng);
        if (w < 0) add_stopped[r] = true;
        if (w <= 0) return;
        sempty[k % bufs].arrive();
        added[r]++;
    }
    bool happen(Rng& rng) {      // one thing that is on its way
        if (events.empty() && commits.empty()) return false;
        const bool products_end = !commits.empty() && (events.empty() || rng() % 2);
        std::vector<Event>& from = products_end ? commits : events;
        const size_t i = products_end ? rng() % std::min<size_t>(from.size(), 2 * ctas) : rng() % from.size();
        const Event e = from[i];
        from.erase(from.begin() + i);
        if (e.bytes) e.bar->complete(e.bytes); else e.bar->arrive();
        return true;
    }
    bool await(const Bar& b, uint32_t parity, Rng& rng) {
        while (!b.ready(parity))
            if (!happen(rng)) return false;
        return true;
    }
    const char* drain(Rng& rng) {
        for (int r = 0; r < 2 && ctas == 2; r++) {
            const DrainSteps owed = drain_owed(issued[r], issued[1 - r]);
            for (uint32_t k = owed.from; k < owed.to; k++) full[drain_slot(k, stages)].arrive();
        }
        for (int r = 0; r < ctas; r++) {
            DrainSteps d = drain_recent(products, stages);
            for (uint32_t k = d.from; k < d.to; k++)
                if (!await(empty[r][drain_slot(k, stages)], drain_parity(k, stages), rng)) return "a wait for products that never ends";
            d = drain_recent(products, bufs);
            for (uint32_t k = d.from; k < d.to; k++)
                if (!await(sfull[r][drain_slot(k, bufs)], drain_parity(k, bufs), rng)) return "a wait for sums that never ends";
        }
        const DrainSteps d = drain_recent(issued[0] > issued[1] ? issued[0] : issued[1], stages);
        for (uint32_t k = d.from; k < d.to; k++)
            if (!await(full[drain_slot(k, stages)], drain_parity(k, stages), rng)) return "a wait for copies that never ends";
        return events.empty() && commits.empty() ? nullptr : "something is still on its way";
    }
};

int main(int argc, char** argv) {
    const int runs = argc > 1 ? atoi(argv[1]) : 20000;
    Rng rng(1);
    int stopped = 0, apart = 0, plain = 0;
    for (int i = 0; i < runs; i++) {
        const int ctas = 1 + (int)(rng() % 2);
        Model p(ctas, 1 + rng() % 7, ctas == 2 || rng() % 2 ? 2 : 4, 1 + rng() % 40);
        const double patience = i % 4 == 0 ? 1.0 : 1.0 - 1.0 / (1 + rng() % 200);
        long long turns = 0;
        while (!(p.copy_stopped[0] && p.copy_stopped[1] && p.mma_stopped && p.add_stopped[0] && p.add_stopped[1])) {
            const uint32_t who = rng() % 9;
            if (who < 2) { if (!p.copy_stopped[who]) p.copy((int)who, patience, rng); }
            else if (who == 2) { if (!p.mma_stopped) p.multiply(patience, rng); }
            else if (who < 5) { if (!p.add_stopped[who - 3]) p.add((int)who - 3, patience, rng); }
            else p.happen(rng);
            if (++turns > 10000000) { printf("run %d: stuck\n", i); return 1; }
        }
        if (p.gave_up[0] || p.gave_up[1]) {
            stopped++;
            apart += p.issued[0] != p.issued[1];
        } else {
            plain++;
            if (p.products != p.steps || p.added[0] != p.steps) { printf("run %d: not all steps\n", i); return 1; }
        }
        if (const char* what = p.drain(rng)) {
            printf("run %d: %s (%d CTAs, stages %u, issued %u and %u, products %u)\n", i, what, ctas, p.stages, p.issued[0], p.issued[1], p.products);
            return 1;
        }
    }
    printf("%d runs to the end, %d stopped, %d of these with the CTAs at different steps\n", plain, stopped, apart);
    return stopped > runs / 4 && apart > runs / 50 && plain > 0 ? 0 : 1;
}
