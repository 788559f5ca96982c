// window_split and window_part_units (csrc/hkv_plan.h): over many shapes of calls, the parts that a
// call's tiles are cut into never pass the units that an engine holds for them.
#include <cstdio>
#include <random>
#include <vector>

#include "hkv_plan.h"

int main() {
    std::mt19937 gen(17);
    auto upto = [&](int64_t hi) { return std::uniform_int_distribution<int64_t>(1, hi)(gen); };
    int64_t most_units = 0;
    for (int round = 0; round < 200000; ++round) {
        const int64_t sms = round % 5 == 0 ? upto(200) : 148;
        const int64_t G = round % 7 == 0 ? upto(300) : int64_t{1} << (upto(5) - 1);
        const int64_t n = upto(round % 3 == 0 ? 400 : 12);
        const int64_t longest = upto(round % 2 == 0 ? 3000 : 40);
        std::vector<int64_t> blocks;
        for (int64_t i = 0; i < n; ++i) {
            // all alike, any, or a few long ones among short ones
            blocks.push_back(round % 4 == 0 ? longest : round % 4 == 1 && i % 9 != 0 ? upto(2) : upto(longest));
        }
        const int64_t most = hkv::window_split(blocks, G, sms);
        int64_t parts = 0, ctas = 0, top = 0;
        for (const int64_t b : blocks) {
            const int64_t cuts = (b + most - 1) / most;
            parts += cuts > 1 ? cuts : 0;
            ctas += cuts;
            top = b > top ? b : top;
        }
        most_units = parts * G > most_units && sms == 148 ? parts * G : most_units;
        if (most < 1 || parts * G > hkv::window_part_units(sms) || (n * G <= sms && ctas * G > sms)) {
            std::fprintf(stderr, "round %d: sms %lld G %lld n %lld: %lld parts, at most %lld blocks\n", round,
                         (long long)sms, (long long)G, (long long)n, (long long)parts, (long long)most);
            return 1;
        }
    }
    std::printf("window plan ok, up to %lld units of %lld\n", (long long)most_units,
                (long long)hkv::window_part_units(148));
    return 0;
}
