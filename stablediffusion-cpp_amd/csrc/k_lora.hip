// k_lora.hip - low-rank adapters of many requests beside a projection that they
// share: C[t] (+)= s_a (X[t] A_a^T) B_a^T for the rows t of each run of rows, a the
// run's adapter (no reference function; the projection itself is
// backend_cuda.h:38-43, gemm_nt_bf16 / gemm_nt_f32).
//
// fp32 throughout: X keeps its 24 bits (unlike the A of gemm_nt_bf16, which is
// rounded to bf16), the weights theirs, H = X A^T and the sums are fp32.
#include <algorithm>
#include <string>
#include <type_traits>

#include "spans.hpp"

namespace sdh {
namespace {

typedef unsigned short u16;

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(u16 b) { return __uint_as_float((unsigned)b << 16); }

// A run of rows: its adapter and rank, the rank 0 where it has none.
struct Run {
    int first, rows, adapter, rank;
};
__device__ __forceinline__ Run run_at(const int4* __restrict__ list, int s, int M, int adapters, int rank) {
    const int4 e = list[s];
    Run r{e.x, e.y, e.z, e.w};
    dev::cut_span(r.first, r.rows, M);
    r.rank = r.adapter < 0 || r.adapter >= adapters ? 0 : min(max(r.rank, 0), rank);
    return r;
}

constexpr int kRowWaves = 4;

// H[t, :] = s_a X[t] A_a^T, a wave per row.
template <class TX, class TW>
__global__ __launch_bounds__(64 * kRowWaves) void k_lora_down_rows(const TX* __restrict__ X, int64_t ldx, const TW* __restrict__ A,
                                                                   const float* __restrict__ scale, const int4* __restrict__ runs, int n,
                                                                   float* __restrict__ H, int M, int K, int rank, int adapters) {
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x * kRowWaves + (threadIdx.x >> 6);
    if (t >= M) return;
    const int s = dev::span_of_row(runs, n, t, M);
    if (s < 0) return;
    const Run r = run_at(runs, s, M, adapters, rank);
    if (!r.rank) return;
    const float f = scale ? scale[r.adapter] : 1.0f;
    const TX* x = X + (int64_t)t * ldx;
    for (int j = 0; j < r.rank; ++j) {
        const TW* a = A + ((int64_t)r.adapter * rank + j) * K;
        float v = 0.f;
        for (int k = lane; k < K; k += 64) v = fmaf(value(x[k]), value(a[k]), v);
        v = dev::wave_sum(v);
        if (lane == 0) H[(int64_t)t * rank + j] = v * f;
    }
}

// C[t, :] (+)= H[t] B_a^T, a thread per column.
template <class TW>
__global__ __launch_bounds__(256) void k_lora_up_rows(const float* __restrict__ H, const TW* __restrict__ B, const int4* __restrict__ runs,
                                                      int n, float* __restrict__ C, int64_t ldc, int M, int N, int rank, int adapters,
                                                      int accumulate) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    for (int t = blockIdx.y; t < M; t += gridDim.y) {
        const int s = dev::span_of_row(runs, n, t, M);
        if (s < 0) continue;
        const Run r = run_at(runs, s, M, adapters, rank);
        if (c >= N || (accumulate && !r.rank)) continue;
        float v = 0.f;
        const TW* b = B + ((int64_t)max(r.adapter, 0) * N + c) * rank;
        for (int j = 0; j < r.rank; ++j) v = fmaf(H[(int64_t)t * rank + j], value(b[j]), v);
        float* p = C + (int64_t)t * ldc + c;
        *p = accumulate ? *p + v : v;
    }
}

template <class TX, class TW>
void run_lora(const char* op, int64_t M, int64_t N, int64_t K, const TX* X, int64_t ldx, const TW* A, const TW* B, int64_t rank,
              int64_t adapters, const float* scale, const int32_t* segments, int64_t count, float* C, int64_t ldc, bool accumulate) {
    constexpr int64_t kMost = int64_t(1) << 30;
    need(M >= 0 && N >= 0 && K >= 0 && rank >= 0 && adapters >= 0 && count >= 0, op, "negative size");
    need(ldx >= K && ldc >= N, op, "leading dimension smaller than the row");
    need(M < kMost && N < kMost && K < kMost && adapters < kMost && count < kMost, op, "a size of 2^30 or more");
    need(rank <= 1024, op, "rank above 1024");
    if (M == 0 || N == 0 || count == 0) return;
    ensure_init();
    check_range(segments, (size_t)count * 16, op, "segments");
    need(aligned16(segments), op, "segments is not 16-byte aligned");
    const size_t cb = (size_t)((M - 1) * ldc + N) * 4;
    check_range(C, cb, op, "C");
    need(!overlaps(C, cb, segments, (size_t)count * 16), op, "C overlaps an input");
    const bool any = K > 0 && rank > 0 && adapters > 0;
    if (any) {
        const size_t xb = (size_t)((M - 1) * ldx + K) * sizeof(TX), ab = (size_t)(adapters * rank * K) * sizeof(TW),
                     bb = (size_t)(adapters * N * rank) * sizeof(TW);
        check_range(X, xb, op, "X");
        check_range(A, ab, op, "A");
        check_range(B, bb, op, "B");
        need(!overlaps(C, cb, X, xb) && !overlaps(C, cb, A, ab) && !overlaps(C, cb, B, bb), op, "C overlaps an input");
        if (scale) {
            check_range(scale, (size_t)adapters * 4, op, "scale");
            need(!overlaps(C, cb, scale, (size_t)adapters * 4), op, "C overlaps an input");
        }
    } else if (accumulate) {
        return;
    }
    const int r = any ? (int)rank : 0, na = any ? (int)adapters : 0;
    float* H = (float*)scratch(std::max<size_t>((size_t)(M * r) * 4, 4));
    need((M + kRowWaves - 1) / kRowWaves * 64 * kRowWaves <= kMaxGridItems && N <= kMaxGridItems - 256, op, "matrix too large for one launch");
    if (any)
        k_lora_down_rows<TX, TW><<<blocks_for(M, kRowWaves), 64 * kRowWaves, 0, stream()>>>(X, ldx, A, scale, (const int4*)segments, (int)count, H,
                                                                                         (int)M, (int)K, r, na);
    k_lora_up_rows<TW><<<dim3(blocks_for(N, 256), (unsigned)std::min<int64_t>(M, 65535)), 256, 0, stream()>>>(H, B, (const int4*)segments, (int)count, C, ldc, (int)M,
                                                                                   (int)N, r, na, accumulate ? 1 : 0);
    launched(op);
}

}  // namespace
}  // namespace sdh

using namespace sdh;

extern "C" {

int sdh_lora_nt_bf16(int64_t M, int64_t N, int64_t K, const float* X, int64_t ldx, const uint16_t* A, const uint16_t* B, int64_t rank,
                     int64_t adapters, const float* scale, const int32_t* segments, int64_t count, float* C, int64_t ldc, int accumulate) {
    return guarded([&] {
        run_lora<float, u16>("sdh_lora_nt_bf16", M, N, K, X, ldx, A, B, rank, adapters, scale, segments, count, C, ldc, accumulate != 0);
    });
}

int sdh_lora_nt_bf16_packed(int64_t M, int64_t N, int64_t K, const uint16_t* X, int64_t ldx, const uint16_t* A, const uint16_t* B,
                            int64_t rank, int64_t adapters, const float* scale, const int32_t* segments, int64_t count, float* C, int64_t ldc,
                            int accumulate) {
    return guarded([&] {
        run_lora<u16, u16>("sdh_lora_nt_bf16_packed", M, N, K, X, ldx, A, B, rank, adapters, scale, segments, count, C, ldc, accumulate != 0);
    });
}

int sdh_lora_nt_f32(int64_t M, int64_t N, int64_t K, const float* X, int64_t ldx, const float* A, const float* B, int64_t rank,
                    int64_t adapters, const float* scale, const int32_t* segments, int64_t count, float* C, int64_t ldc, int accumulate) {
    return guarded([&] {
        run_lora<float, float>("sdh_lora_nt_f32", M, N, K, X, ldx, A, B, rank, adapters, scale, segments, count, C, ldc, accumulate != 0);
    });
}

}  // extern "C"
