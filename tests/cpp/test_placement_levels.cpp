// Regions of the HBM that measure at different levels (nabla_amd/csrc/host/nbo_placement_plan.hpp), on the CPU: two
// chunks of one region read 5.0-5.3 TB/s together, two of another 5.56-5.75, two of different ones 6.1.
#include <cstdio>
#include <cmath>
#include <vector>

#include "../../nabla_amd/csrc/host/nbo_placement_plan.hpp"

using namespace nbo::plan;

#define CHECK(cond)                                                                        \
    do {                                                                                   \
        if (!(cond)) {                                                                     \
            std::fprintf(stderr, "%s:%d: CHECK failed: %s\n", __FILE__, __LINE__, #cond);  \
            return 1;                                                                      \
        }                                                                                  \
    } while (0)

static bool matches(const RegionFinder &f, const std::vector<int> &truth)
{
    for (size_t a = 0; a < truth.size(); a++)
        for (size_t b = a + 1; b < truth.size(); b++)
            if ((f.region_of()[a] == f.region_of()[b]) != (truth[a] == truth[b])) return false;
    return true;
}

int main()
{
    // as measured: twelve chunks of the anchor's region, three of one whose pairs read above the middle between
    // the anchor's (5.07) and the pairs of both (6.12)
    {
        const std::vector<int> truth{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1};
        const double with0[] = {0, 5012, 5305, 5254, 5252, 5318, 5291, 5252, 4961, 5042, 5024, 4987, 6147, 6120, 6104};
        auto probe = [&](size_t a, size_t b) {
            if (a == 0) return with0[b];
            return truth[a] != truth[b] ? 6110.0 : truth[a] == 0 ? 5150.0 : a == 12 && b == 13 ? 5629.0 : 5560.0;
        };
        auto halves = [&](size_t a) { return truth[a] == 0 ? 5072.0 : 5603.0; };
        RegionFinder f;
        f.add_chunks(15, probe, halves);
        CHECK(f.anchor() == 0 && std::fabs(f.threshold() - 5614) < 40);
        CHECK(f.regions() == 2 && matches(f, truth));
        CHECK(f.threshold_between(0, 1) > 5700 && f.threshold_between(0, 1) < 6100);
    }
    // three regions, each at its own level, all of them apart
    {
        const std::vector<int> truth{0, 1, 2, 0, 1, 2, 0, 1, 2, 0, 1, 2};
        const double level[] = {5100, 5690, 5400};
        auto probe = [&](size_t a, size_t b) {
            const double w = 1.0 + 0.004 * (double)((int)((a * 7 + b * 13) % 11) - 5) / 5.0;
            return (truth[a] == truth[b] ? level[truth[a]] : 6150.0) * w;
        };
        RegionFinder f;
        f.add_chunks(12, probe, [&](size_t a) { return level[truth[a]]; });
        CHECK(f.regions() == 3 && matches(f, truth));
    }
    // a chunk pieced together from two regions does not raise the bar for its neighbours
    {
        const std::vector<int> truth{0, 0, 0, 7, 1, 1, 1, 0};
        auto probe = [&](size_t a, size_t b) {
            return truth[a] == 7 || truth[b] == 7 ? 5930.0 : truth[a] == truth[b] ? 5450.0 : 6150.0;
        };
        RegionFinder f;
        f.add_chunks(8, probe, [&](size_t a) { return truth[a] == 7 ? 5920.0 : 5450.0; });
        CHECK(f.regions() == 3 && matches(f, truth));
    }
    // reads_apart: a probe that is disturbed is slower, never faster, so a low reading is taken again, a high one not
    {
        size_t n = 0;
        const double reads[] = {5500, 5900, 6100, 9999};
        double last = 0.0;
        CHECK(reads_apart([&] { return reads[n++]; }, 6000.0, &last) && n == 3 && last == 6100);
        n = 0;
        CHECK(!reads_apart([&] { return reads[n++]; }, 7000.0, &last) && n == 3 && last == 6100);
        n = 0;
        CHECK(reads_apart([&] { return reads[n++]; }, 5400.0, &last) && n == 1 && last == 5500);
        CHECK(!reads_apart([&] { return std::nan(""); }, 5400.0, &last));
    }
    std::puts("placement levels: all checks passed");
    return 0;
}
