// CPU check of the search that the embedding gradient makes for entries
// without a token (alphazero_b200/csrc/sorted_search.cuh): up to the largest
// number of tokens that a call accepts, it reads inside the tokens only and
// finds the first place that is not smaller.
#include "../../alphazero_b200/csrc/sorted_search.cuh"

#include <cstdio>

namespace {

int failures = 0;

// Token i of n sorted ones: i / run.
struct Keys {
    int n, run;
    mutable bool outside = false;
    uint32_t operator()(int i) const {
        if (i < 0 || i >= n) {
            outside = true;
            return ~0u;
        }
        return (uint32_t)(i / run);
    }
};

void look(int n, int run, uint32_t v) {
    const Keys keys{n, run};
    const int at = mgb::ops::lower_bound(keys, n, v);
    const int64_t first = (int64_t)v * run, want = first < n ? first : n;
    if (keys.outside || at != want) {
        std::printf("n %d run %d v %u: %d, expected %lld%s\n", n, run, v, at, (long long)want,
                    keys.outside ? " (read outside)" : "");
        ++failures;
    }
}

}  // namespace

int main() {
    const int sizes[] = {0, 1, 2, 3, 1000, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, 1500000007, INT32_MAX - 1025};
    int looked = 0;
    for (int n : sizes)
        for (int run : {1, 7, 1 << 20}) {
            const uint32_t top = n / run;
            for (uint32_t v : {0u, 1u, top / 3, top / 2, top / 2 + 1, top / 4 * 3, top, top + 1, 0x7fffffffu}) {
                look(n, run, v);
                ++looked;
            }
        }
    std::printf("%d searches, %d failures\n", looked, failures);
    return failures != 0;
}
