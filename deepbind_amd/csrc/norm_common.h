// Shared by the norms of a row's chunks (layernorm.hip, blocknorm.hip).
#pragma once
#include "rows_common.h"

namespace dbk {

// A chunk's mean and reciprocal deviation from its sum's mean `near`, the mean of the squared distances to that and the mean of the distances. The sum's
// roundings make `near` miss the mean by a few units in its last place, which is all there is where the values are equal, and more than their
// spread where they lie far from zero: the distances, of the spread's size, say by how much.
template <typename A> __device__ __forceinline__ void norm_stats(A near, A sq, A rest, A eps, A& mean, A& rstd)
{
    const A var = fma(-rest, rest, sq);
    mean = near + rest;
    rstd = A(1) / sqrt((var < A(0) ? A(0) : var) + eps);        // (a NaN stays)
}

// Chunks of `lanes` lanes side by side in a workgroup of 256: log2 of the power of two that costs least, counting the lanes whose chunk does not exist
// and, against short pieces of rows, 128 bytes more for every piece.
inline unsigned chunks_side_by_side(unsigned lanes, size_t nchunk)
{
    unsigned best = 0;
    double least = 1e300;
    for (unsigned c = 0; lanes && lanes << c <= 256u; ++c) {
        const size_t tiles = (nchunk + (size_t(1) << c) - 1) >> c;
        const double cost = (double)(tiles << c) * (1.0 + 128.0 / (double)((size_t)lanes * 16 << c));
        if (cost <= least) { least = cost; best = c; }
        if (tiles == 1) break;
    }
    return best;
}

}  // namespace dbk
