// How attention's work is shared out (csrc/attention_plan.h), and the argument structures of the C header, without a GPU.
#include <cstdio>
#include <cstdlib>
#include <algorithm>
#include <cstddef>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "../../dlf_b200/csrc/attention_plan.h"
#include "../../include/dlf_b200.h"

using namespace dlfb200;

static void check(bool ok, const char* what) {
    if (!ok) {
        std::printf("failed: %s\n", what);
        std::exit(1);
    }
}

int main() {
    bool bad = false;
    check(plan_length(-3, 10, &bad) == 0 && !bad, "a length below zero counts as none");
    check(plan_length(10, 10, &bad) == 10 && !bad, "a full length");
    check(plan_length(11, 10, &bad) == 10 && bad, "a length beyond the room is cut and reported");
    check(plan_units(0, 64) == 1 && plan_units(1, 64) == 1 && plan_units(64, 64) == 1 && plan_units(65, 64) == 2, "units");
    check(plan_units(2147483647, 64) == 33554432, "units of the longest");
    check(plan_place(-1, 3, 8) < 0 && plan_place(8, 3, 8) < 0, "no such page");
    check((plan_place(7, 3, 8) >> 32) == 7 && static_cast<int>(plan_place(7, 3, 8)) == 3, "a place");
    check(plan_place(2147483646, 127, 2147483647) > 0, "the last page there can be");
    check(plan_per(2147483647, 592, 2) == 3627507, "no overflow in the share of a CTA");

    std::mt19937 rng(1);
    for (int round = 0; round < 4000; ++round) {
        const int batch = 1 + static_cast<int>(rng() % 9), heads = 1 + static_cast<int>(rng() % 6), unit = rng() % 2 ? 64 : 128;
        const int ctas = 1 + static_cast<int>(rng() % 40), least = 1 + static_cast<int>(rng() % 3);
        std::vector<int> units;
        int total = 0;
        for (int b = 0; b < batch; ++b) {
            units.push_back(plan_units(static_cast<int>(rng() % (rng() % 4 ? 900 : 20000)) - 5, unit));
            total += units.back() * heads;
        }
        const int per = plan_per(total, ctas, least);
        check(static_cast<long long>(per) * ctas >= total, "the shares cover the work");
        std::vector<int> seen(static_cast<size_t>(total), 0);
        std::map<int, std::vector<int>> slots;  // by first unit of the (sequence, head): slots in the order of the CTAs
        std::set<int> used;
        for (int c = 0; c < ctas; ++c) {
            for (long long at = static_cast<long long>(c) * per; at < total && at < (c + 1ll) * per;) {
                const int u = static_cast<int>(at);
                int first = 0, b = 0, h = 0;  // the (sequence, head) that u lies in
                while (first + units[static_cast<size_t>(b)] <= u) {
                    first += units[static_cast<size_t>(b)];
                    if (++h == heads) h = 0, ++b;
                }
                const int n = units[static_cast<size_t>(b)], end = static_cast<int>(std::min<long long>({first + n, (c + 1ll) * per, total}));
                for (int i = u; i < end; ++i) ++seen[static_cast<size_t>(i)];
                if (end - u < n) {
                    const int slot = plan_slot(u, per);
                    check(slot >= 0 && slot < 2 * ctas && used.insert(slot).second, "a slot of its own for every part");
                    slots[first].push_back(slot);
                }
                at = end;
            }
        }
        for (int n : seen) check(n == 1, "every unit once");
        int first = 0;
        for (int b = 0; b < batch; ++b)
            for (int h = 0; h < heads; ++h, first += units[static_cast<size_t>(b)]) {
                // what the joining kernels enumerate
                const int last = first + units[static_cast<size_t>(b)] - 1, c0 = first / per, c1 = last / per;
                std::vector<int> want;
                for (int c = c0; c0 != c1 && c <= c1; ++c) want.push_back(c == c0 ? plan_slot(first, per) : 2 * c);
                check(want == slots[first], "the parts that are joined are the ones that were written");
            }
    }
    std::printf("%zu %zu %zu %zu %zu %zu\n", offsetof(dlf_b200_attention_args, q), sizeof(dlf_b200_attention_args),
                offsetof(dlf_b200_paged_attention_args, q), sizeof(dlf_b200_paged_attention_args), offsetof(dlf_b200_paged_append_args, k),
                sizeof(dlf_b200_paged_append_args));
    return 0;
}
