// Trees of drafted tokens: what the kernels that verify them share.
//
// parents[j] is the index of token j's parent among the sequence's M <= 64 tokens, smaller than j, or -1: a child of the last committed
// token.  Anything else counts as -1.  A wavefront holds one token per lane, so a whole tree is one register.
#pragma once
#include "qt_common.h"

namespace qt {

constexpr int TREE_MAX = 64;

__device__ __forceinline__ int tree_parent(const int* __restrict__ parents, int j, int M) {
    const int p = j < M ? parents[j] : -1;
    return (unsigned)p < (unsigned)j ? p : -1;
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
    const unsigned lo = __shfl((unsigned)v, lane), hi = __shfl((unsigned)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
// bit i of the result: token i is the lane's token or one of its ancestors.  Doubling: each of the six rounds joins what a token has collected with
// what the nearest token beyond that has.
__device__ __forceinline__ uint64_t tree_ancestors(int parent, int lane) {
    uint64_t seen = 1ull << lane | (parent >= 0 ? 1ull << parent : 0);
    int a = parent;
#pragma unroll
    for (int i = 0; i < 6; i++) {
        const int from = a < 0 ? lane : a;
        const uint64_t s = shfl64(seen, from);
        const int up = __shfl(a, from);
        if (a >= 0) seen |= s, a = up;
    }
    return seen;
}
// the same, and v becomes the sum of v over the lane's token and its ancestors
__device__ __forceinline__ uint64_t tree_ancestors_sum(int parent, double& v, int lane) {
    uint64_t seen = 1ull << lane | (parent >= 0 ? 1ull << parent : 0);
    int a = parent;
#pragma unroll
    for (int i = 0; i < 6; i++) {
        const int from = a < 0 ? lane : a;
        const uint64_t s = shfl64(seen, from);
        const double d = __hiloint2double(__shfl(__double2hiint(v), from), __shfl(__double2loint(v), from));
        const int up = __shfl(a, from);
        if (a >= 0) seen |= s, v += d, a = up;
    }
    return seen;
}

}  // namespace qt
