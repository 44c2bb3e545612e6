// Search in sorted tokens, callable on the host as well, where a CPU test
// checks it at lengths that fill 32 bits.
#pragma once

#include <cstdint>

namespace mgb {
namespace ops {

// First place in [0, n) whose key is at least v, n if there is none.
template <class KeyAt>
__host__ __device__ __forceinline__ int lower_bound(const KeyAt& key, int n, uint32_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;  // lo + hi may not fit
        if (key(mid) < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

}  // namespace ops
}  // namespace mgb
