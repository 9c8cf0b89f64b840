// spans.hpp - rows of many requests in one tensor: who owns which. The lists are
// device memory that the host does not read, so the kernels hold every entry to
// the tensor's rows before they use it.
#pragma once

#include "sdh_internal.hpp"

namespace sdh {
namespace dev {

// Every workgroup walks the list, 64 entries at a time, which is why it has a limit.
constexpr int64_t kMaxSpans = 65536;

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

// A workgroup's place among the row tiles of all entries.
struct SpanTile {
    int index;        // the entry
    int first, rows;  // its rows, cut to the tensor
    int z, w;         // its other two words
    int row0;         // the tile's first row within it, in rows times `mult`
};
// Entries have ceil(rows * mult / tile_rows) tiles each, numbered through; false past
// the last one. Every lane of a wave gets the answer. rows * mult < 2^30 for all; no entry has more
// tiles than the grid has items, below 2^25, so that the sums, of 64 entries behind `before` <= item,
// stay inside 31 bits.
__device__ __forceinline__ bool find_tile(const int4* __restrict__ list, int n, int total, int mult, int tile_rows, int item,
                                          SpanTile& t) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0, before = 0; s0 < n; s0 += 64) {
        int4 e = make_int4(0, 0, 0, 0);
        if (s0 + lane < n) {
            e = list[s0 + lane];
            cut_span(e.x, e.y, total);
        }
        const int tiles = (e.y * mult + tile_rows - 1) / tile_rows;
        const int upto = before + wave_scan(tiles);
        const unsigned long long m = __ballot(item < upto);
        if (m) {
            const int at = (int)__ffsll(m) - 1;
            t.index = s0 + at;
            t.first = __builtin_amdgcn_readlane(e.x, at);
            t.rows = __builtin_amdgcn_readlane(e.y, at);
            t.z = __builtin_amdgcn_readlane(e.z, at);
            t.w = __builtin_amdgcn_readlane(e.w, at);
            t.row0 = (item - __builtin_amdgcn_readlane(upto - tiles, at)) * tile_rows;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

}  // namespace dev
}  // namespace sdh
