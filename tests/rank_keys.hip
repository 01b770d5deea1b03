// Checks on the host of the keys by which log probabilities rank logits
// (tests/test_rank_keys.py): every key lies between 0 and kAboveKeys, keys
// order pairs as the operator documents it, and passes that take the largest
// key below the last one's find every logit once.  Prints one line per check:
// its name and how many cases broke it.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <map>
#include <random>
#include <string>
#include <vector>

#include "rq_rank.h"

namespace {

std::map<std::string, int> g_broken;
void check(const char* name, bool holds) { g_broken[name] += holds ? 0 : 1; }

float of_bits(uint32_t u) {
    float x;
    memcpy(&x, &u, 4);
    return x;
}

const float kValues[] = {NAN, -NAN, of_bits(0x7f800001u), of_bits(0xffffffffu), INFINITY, -INFINITY, 0.0f, -0.0f, 1.0f, -1.0f,
                         3.402823466e+38f, -3.402823466e+38f, 1e-45f, -1e-45f, 2.5f};

// The documented order: NaN first, then greater values, then lower indexes.
bool before(const std::vector<float>& x, uint32_t a, uint32_t b) {
    const bool nan_a = x[a] != x[a], nan_b = x[b] != x[b];
    if (nan_a != nan_b) return nan_a;
    if (!nan_a && x[a] != x[b]) return x[a] > x[b];
    return a < b;
}

void row(const std::vector<float>& x) {
    std::vector<uint32_t> want(x.size());
    for (uint32_t i = 0; i < x.size(); ++i) want[i] = i;
    std::sort(want.begin(), want.end(), [&](uint32_t a, uint32_t b) { return before(x, a, b); });
    uint64_t below = rq::kAboveKeys;
    for (uint32_t expected : want) {
        uint64_t best = 0;
        for (uint32_t i = 0; i < x.size(); ++i) best = rq::next_rank(best, rq::rank_key(x[i], i), below);
        check("passes", 0xffffffffu - (uint32_t)best == expected);
        below = best;
    }
}

}  // namespace

int main() {
    for (float x : kValues)
        for (uint32_t index : {0u, 1u, 2u, 49151u, 0x7ffffffeu}) {
            const uint64_t key = rq::rank_key(x, index);
            check("range", key > 0 && key < rq::kAboveKeys);
            check("index", 0xffffffffu - (uint32_t)key == index);
        }
    std::mt19937_64 rng(5);
    const int kinds = sizeof(kValues) / sizeof(kValues[0]);
    for (size_t size : {1, 2, 7, 32, 100}) {
        row(std::vector<float>(size, NAN));
        row(std::vector<float>(size, -INFINITY));
        for (int k = 0; k < 200; ++k) {
            std::vector<float> x;
            for (size_t i = 0; i < size; ++i) x.push_back(kValues[rng() % kinds]);
            row(x);
        }
    }
    for (const auto& [name, count] : g_broken) printf("%s %d\n", name.c_str(), count);
    return 0;
}
