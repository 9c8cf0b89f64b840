// spans.hpp - rows of many requests in one tensor: who owns which. The lists are
// device memory that the host does not read, so the kernels hold every entry to
// the tensor's rows before they use it.
#pragma once

#include "sdh_internal.hpp"

namespace sdh {
namespace dev {

// [first, first + rows) cut to [0, total).
__device__ __forceinline__ void cut_span(int& first, int& rows, int total) {
    first = min(max(first, 0), total);
    rows = min(max(rows, 0), total - first);
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const int u = __shfl_up(v, s, 64);
        if (lane >= s) v += u;
    }
    return v;
}

// The entry of `list` (first row, rows, ...) that holds row `row` of `total`, or
// -1; the first of them where several do. Every lane of a wave gets the answer.
__device__ __forceinline__ int span_of_row(const int4* __restrict__ list, int n, int row, int total) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < n; s0 += 64) {
        int first = 0, rows = 0;
        if (s0 + lane < n) {
            const int4 e = list[s0 + lane];
            first = e.x, rows = e.y;
            cut_span(first, rows, total);
        }
        const unsigned long long m = __ballot(row >= first && row - first < rows);
        if (m) return s0 + (int)__ffsll(m) - 1;
    }
    return -1;
}

}  // namespace dev
}  // namespace sdh
