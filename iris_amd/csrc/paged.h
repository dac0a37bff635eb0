// Shared pieces of the operators over a paged cache: argument checks, and the
// ancestors of a tree of drafted rows.
#pragma once

#include "../../include/iris_hip.h"
#include "layer_kernels.h"

// Rows of one request's drafted tree: a lane each, and a bit each of a mask.
constexpr uint32_t TREE_MAX_NODES = 64;
// Positions a request may hold: every sum of exp terms (2^32 at most each)
// stays exact in double, below 2^53.
constexpr uint32_t TREE_MAX_POSITIONS = 1u << 20;

// 0, or why the cache cannot be used (host checks).
int iris_paged_check(const IrisPagedKv* c);

inline bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

// Raises a kernel's dynamic LDS limit where a launch needs more than 64 KB.
// (Not a stream operation: it can precede a captured launch.)
inline hipError_t paged_lds_limit(const void* kernel, size_t bytes) {
    return bytes > 65536 ? hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : hipSuccess;
}

// The ancestors of row `lane` of a tree of n <= 64 rows, itself included, as
// a mask of rows (0 from row n on). parents[i] is row i's parent where it lies
// in [0, i), else i has none; null: i's parent is i - 1. Every lane of the
// wave takes part. After t rounds a lane's mask holds its 2^t nearest rows up
// the tree, and `up` the row 2^t above it.
__device__ __forceinline__ uint64_t tree_ancestors(const int32_t* parents, uint32_t n, uint32_t lane) {
    if (lane >= n) n = 0;
    uint64_t mask = n ? 1ull << lane : 0;
    if (!parents) return n ? mask | (mask - 1) : 0;
    int up = n ? parents[lane] : -1;
    if (up < 0 || up >= (int)lane) up = -1;
#pragma unroll
    for (int round = 0; round < 6; round++) {
        const int from = up < 0 ? (int)lane : up;
        const uint64_t above = __shfl((unsigned long long)mask, from);
        const int next = __shfl(up, from);
        if (up >= 0) {
            mask |= above;
            up = next;
        }
    }
    return mask;
}
