// k_lora.hip - low-rank adapters of many requests beside a projection that they
// share: C[t] (+)= s_a (X[t] A_a^T) B_a^T for the rows t of each run of rows, a the
// run's adapter (no reference function; the projection itself is
// backend_cuda.h:38-43, gemm_nt_bf16 / gemm_nt_f32).
//
// Two launches: down, H = s_a X A_a^T into scratch, and up, C (+)= H B_a^T, both on
// v_mfma_f32_32x32x16_bf16; one for few rows and a short K (k_lora_small). fp32 accuracy:
// a float is the exact sum of three bf16 values (24 bits in steps of 8, cut towards zero,
// so nothing overflows and the range is fp32's), a bf16 value its own; the products of the
// parts are exact in the fp32 accumulators. X keeps its 24 bits, unlike the A of
// gemm_nt_bf16. With fp32 weights the product of the two smallest parts (below 2^-28) is
// left out. An infinity has no such parts (inf - inf): sums of H that come out not finite are
// formed again from X and A as they are, and what such rows of H add to C in fp32.
//
// Bound by memory for many rows: X is read once (a workgroup has all ranks of its rows), C
// read and written once, while A, B and H come from the L2s. [12528,3840] bf16 to 10240
// columns, rank 64: 137 us, 4.5 TB/s (down 27, up 106; a kernel that only writes C takes
// 77); [8192,640] to 5120, fp32, rank 12: 78 us, 4.0 TB/s; 48 single rows of 2560 to 4096
// columns, rank 16: 10.4 us, the two launches' own length.
#include <algorithm>
#include <string>
#include <type_traits>

#include "spans.hpp"

namespace sdh {
namespace {

typedef unsigned short u16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));  // 8 bf16
using dev::f4;

constexpr int kLoraWaves = 4, kLoraThreads = 64 * kLoraWaves;

// Eight values of a row on their way, and as MFMA operands.
template <class T>
struct Eight;
template <>
struct Eight<float> {
    static constexpr int kParts = 3;
    f4 a, b;
    // The values p[at .. at + 7], zeros from `end` on. VEC: 16-byte aligned, and in memory all eight where the first is in
    // front of `end` (those behind it are then cut off by the caller).
    template <bool VEC>
    __device__ __forceinline__ void load(const float* p, int at, int end) {
        if constexpr (VEC) {
            const f4* q = (const f4*)(p + (at < end ? at : 0));
            a = q[0], b = q[1];
            if (at >= end) a = b = f4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = at + e < end ? p[at + e] : 0.f;
                b[e] = at + 4 + e < end ? p[at + 4 + e] : 0.f;
            }
        }
    }
    // Zeros behind the first `n`.
    __device__ __forceinline__ void cut(int n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e >= n) a[e] = 0.f;
            if (e + 4 >= n) b[e] = 0.f;
        }
    }
    __device__ __forceinline__ void parts(bf16x8* out) const {
        u32x4 hi, mid, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = i < 2 ? a[2 * i] : b[2 * i - 4], y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
            const unsigned xh = __float_as_uint(x) & 0xFFFF0000u, yh = __float_as_uint(y) & 0xFFFF0000u;
            const float xr = x - __uint_as_float(xh), yr = y - __uint_as_float(yh);
            const unsigned xm = __float_as_uint(xr) & 0xFFFF0000u, ym = __float_as_uint(yr) & 0xFFFF0000u;
            const float xl = xr - __uint_as_float(xm), yl = yr - __uint_as_float(ym);
            hi[i] = xh >> 16 | yh;
            mid[i] = xm >> 16 | ym;
            lo[i] = __float_as_uint(xl) >> 16 | (__float_as_uint(yl) & 0xFFFF0000u);
        }
        out[0] = __builtin_bit_cast(bf16x8, hi);
        out[1] = __builtin_bit_cast(bf16x8, mid);
        out[2] = __builtin_bit_cast(bf16x8, lo);
    }
};
template <>
struct Eight<u16> {
    static constexpr int kParts = 1;
    u32x4 a;
    template <bool VEC>
    __device__ __forceinline__ void load(const u16* p, int at, int end) {
        if constexpr (VEC) {
            a = *(const u32x4*)(p + (at < end ? at : 0));
            if (at >= end) a = u32x4{0u, 0u, 0u, 0u};
        } else {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const unsigned x = at + e < end ? p[at + e] : 0u, y = at + e + 1 < end ? p[at + e + 1] : 0u;
                a[e / 2] = x | y << 16;
            }
        }
    }
    __device__ __forceinline__ void cut(int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] &= 2 * i >= n ? 0u : 2 * i + 1 >= n ? 0xFFFFu : ~0u;
    }
    __device__ __forceinline__ void parts(bf16x8* out) const { out[0] = __builtin_bit_cast(bf16x8, a); }
};
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(u16 x) { return __uint_as_float((unsigned)x << 16); }
template <int PA, int PB>
__device__ __forceinline__ f32x16 multiply(const bf16x8* a, const bf16x8* b, f32x16 c) {
    // the smallest products first
#pragma unroll
    for (int s = PA + PB - 2 - (PA == 3 && PB == 3); s >= 0; --s)
#pragma unroll
        for (int i = 0; i < PA; ++i)
            if (s - i >= 0 && s - i < PB) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[s - i], c, 0, 0, 0);
    return c;
}

struct Lora {
    const void *x, *a, *b;
    const float* scale;
    const int4* runs;
    float *h, *c;
    int64_t ldx, ldc;
    int M, N, K, rank, adapters, count, splits, hrank, accumulate;  // hrank: H's row, rank up to the next 32
};

// The adapter of a run, -1 without one, and how many of its ranks count.
__device__ __forceinline__ int adapter_of(const Lora& P, const dev::SpanTile& t, int& rank) {
    const bool has = t.z >= 0 && t.z < P.adapters;
    rank = has ? min(max(t.w, 0), P.rank) : 0;
    return rank ? t.z : -1;
}

// ---------------------------------------------------------------------------
// H[part][t, :] = s_a X[t] A_a^T over a share of K. A workgroup takes 32 RF rows of a run
// and 32 RT ranks (blockIdx.z the block of ranks); K goes in blocks of a line of X (128
// bytes) to its four waves and to blockIdx.y's workgroups in turn (down_sums: a wave's
// sums). A lane's operands are the first or second half of a block, eight values an MFMA
// step, of X and of A alike: the sum does not mind the order.
// ---------------------------------------------------------------------------
template <class TX>
constexpr int kDownBlock = 128 / sizeof(TX);

// A wave's 32 rows of `BLOCK` values as they are loaded, neighbouring lanes along a row, and their way
// through the wave's 4 KB of LDS into MFMA operands. Loaded as operands, 16 bytes of each of 32 rows an
// instruction, a line came to the L1 four times, and three of those went on to the L2: 47 us, STAGED 27, for
// [12528,3840] bf16 to 64 ranks.
template <class T, int BLOCK>
struct Staged {
    static constexpr int kPieces = BLOCK * (int)sizeof(T) / 16, kLoads = kPieces / 2, kEach = 16 / (int)sizeof(T);
    static_assert(kPieces == 8 || kPieces == 4, "rows of 128 or 64 bytes");
    const T* row[kLoads];
    u32x4 raw[kLoads];

    // Every `stride`-th row from `first` to `last` of p, the lane's 16-byte piece of each.
    __device__ __forceinline__ void rows_of(const T* p, int64_t ld, int first, int stride, int last) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) row[i] = p + min(first + (i * (64 / kPieces) + lane / kPieces) * stride, last) * ld;
    }
    __device__ __forceinline__ void load(int k0, int end) {
        const int k = k0 + (threadIdx.x & (kPieces - 1)) * kEach;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            raw[i] = *(const u32x4*)(row[i] + (k < end ? k : 0));
            if (k >= end) raw[i] = u32x4{0u, 0u, 0u, 0u};
        }
    }
    static __device__ __forceinline__ int at(int row, int piece) {
        return row * (kPieces * 16) + ((piece ^ (kPieces == 8 ? row & 7 : (row >> 1) & 3)) << 4);
    }
    // The operands of the block's MFMA steps, a lane's half of the block (HALVES) or of each step; a wave's LDS
    // accesses keep their order.
    template <bool HALVES>
    __device__ __forceinline__ void deal(char* lds, Eight<T>* out) const {
        const int lane = threadIdx.x & 63, fr = lane & 31, fh = lane >> 5;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *(u32x4*)(lds + at(i * (64 / kPieces) + lane / kPieces, lane & (kPieces - 1))) = raw[i];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < BLOCK / 16; ++u) {
            const int e = HALVES ? fh * (BLOCK / 16) + u : u * 2 + fh;
            if constexpr (sizeof(T) == 2) {
                out[u].a = *(const u32x4*)(lds + at(fr, e));
            } else {
                out[u].a = *(const f4*)(lds + at(fr, 2 * e));
                out[u].b = *(const f4*)(lds + at(fr, 2 * e + 1));
            }
        }
    }
};

// How X and A come: value by value (odd addresses or lengths), as operands, or STAGED. Few rows, whose
// lines the L1 holds, come as operands, which saves the way through LDS: 48 single rows of 2560 bf16 10.6
// us, staged 11.5; [12528,3840] bf16 to 64 ranks and 10240 columns 166 us, staged 147.
enum { kValues, kOperands, kStaged };

// `lds`: the wave's own 4 KB, 16-byte aligned.
template <class TX, class TW, int RT, int RF, int MODE>
__device__ __forceinline__ void down_sums(const Lora& P, const dev::SpanTile& t, int adapter, int rank, int j0, int part, int parts, char* lds,
                                          f32x16 (&acc)[RF][RT]) {
    constexpr int BLOCK = kDownBlock<TX>, U = BLOCK / 16;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, fr = lane & 31, fh = lane >> 5;
    const TX* x0 = (const TX*)P.x + (t.first + t.row0) * P.ldx;
    const TW* a0 = (const TW*)P.a + ((int64_t)adapter * P.rank + j0) * P.K;
#pragma unroll
    for (int i = 0; i < RF; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int step = BLOCK * kLoraWaves * parts;
    int k = (part * kLoraWaves + w) * BLOCK;
    auto add = [&](const Eight<TX> (&x)[RF][U], const Eight<TW> (&a)[U], int j) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            bf16x8 ap[Eight<TW>::kParts];
            a[u].parts(ap);
#pragma unroll
            for (int i = 0; i < RF; ++i) {
                bf16x8 xp[Eight<TX>::kParts];
                x[i][u].parts(xp);
                acc[i][j] = multiply<Eight<TX>::kParts, Eight<TW>::kParts>(xp, ap, acc[i][j]);
            }
        }
    };
    if constexpr (MODE == kStaged) {
        Staged<TX, BLOCK> x[RF];
        Staged<TW, BLOCK> a[RT];
        // rows behind the run's, and ranks behind the adapter's, are its last one again
#pragma unroll
        for (int i = 0; i < RF; ++i) x[i].rows_of(x0, P.ldx, i * 32, 1, t.rows - 1 - t.row0);
#pragma unroll
        for (int j = 0; j < RT; ++j) a[j].rows_of(a0, P.K, j * 32, 1, rank - 1 - j0);
        auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < RF; ++i) x[i].load(k0, P.K);
#pragma unroll
            for (int j = 0; j < RT; ++j) a[j].load(k0, P.K);
        };
        if (k < P.K) load(k);
        for (; k < P.K; k += step) {
            Eight<TX> xf[RF][U];
            Eight<TW> af[RT][U];
#pragma unroll
            for (int i = 0; i < RF; ++i) x[i].template deal<true>(lds, xf[i]);
#pragma unroll
            for (int j = 0; j < RT; ++j) a[j].template deal<true>(lds, af[j]);
            if (k + step < P.K) load(k + step);
#pragma unroll
            for (int j = 0; j < RT; ++j) add(xf, af[j], j);
        }
    } else {
        constexpr bool VEC = MODE == kOperands;
        const TX* x[RF];
        const TW* a[RT];
#pragma unroll
        for (int i = 0; i < RF; ++i) x[i] = x0 + min(i * 32 + fr, t.rows - 1 - t.row0) * P.ldx;
#pragma unroll
        for (int j = 0; j < RT; ++j) a[j] = a0 + (int64_t)min(j * 32 + fr, rank - 1 - j0) * P.K;
        Eight<TX> xn[RF][U];
        Eight<TW> an[RT][U];
        auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = k0 + fh * (BLOCK / 2) + u * 8;
#pragma unroll
                for (int i = 0; i < RF; ++i) xn[i][u].template load<VEC>(x[i], at, P.K);
#pragma unroll
                for (int j = 0; j < RT; ++j) an[j][u].template load<VEC>(a[j], at, P.K);
            }
        };
        if (k < P.K) load(k);
        for (; k < P.K; k += step) {
            Eight<TX> xc[RF][U];
            Eight<TW> ac[RT][U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < RF; ++i) xc[i][u] = xn[i][u];
#pragma unroll
                for (int j = 0; j < RT; ++j) ac[j][u] = an[j][u];
            }
            if (k + step < P.K) load(k + step);
#pragma unroll
            for (int j = 0; j < RT; ++j) add(xc, ac[j], j);
        }
    }
}

// One of those sums, over the blocks of a part of K, in fp32.
template <class TX, class TW>
__device__ __forceinline__ float plain_sum(const Lora& P, const dev::SpanTile& t, int adapter, int row, int j, int part, int parts) {
    constexpr int STEP = kDownBlock<TX> * kLoraWaves;
    const TX* x = (const TX*)P.x + (t.first + t.row0 + row) * P.ldx;
    const TW* a = (const TW*)P.a + ((int64_t)adapter * P.rank + j) * P.K;
    float sum = 0.f;
    for (int64_t k0 = part * STEP; k0 < P.K; k0 += STEP * parts)
        for (int64_t k = k0, end = min(k0 + STEP, (int64_t)P.K); k < end && sum == sum; ++k) sum = fmaf(value(x[k]), value(a[k]), sum);
    return sum;
}

template <class TX, class TW, int RT, int RF, int MODE>
__global__ __launch_bounds__(kLoraThreads) void k_lora_down(Lora P) {
    __shared__ __attribute__((aligned(16))) float part[kLoraWaves][RF * 32][33];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, fr = lane & 31, fh = lane >> 5;
    dev::SpanTile t;
    if (!dev::find_tile(P.runs, P.count, P.M, 1, RF * 32, blockIdx.x, t)) return;
    int rank;
    const int adapter = adapter_of(P, t, rank), j0 = blockIdx.z * RT * 32;
    if (j0 >= rank) return;  // up reads none of them
    f32x16 acc[RF][RT];
    down_sums<TX, TW, RT, RF, MODE>(P, t, adapter, rank, j0, blockIdx.y, P.splits, (char*)part[w], acc);
    const float f = P.scale ? P.scale[adapter] : 1.0f;
    float* h = P.h + ((int64_t)blockIdx.y * P.M + t.first + t.row0) * P.hrank;
    const int left = t.rows - t.row0;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
#pragma unroll
        for (int i = 0; i < RF; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) part[w][i * 32 + (e >> 2) * 8 + fh * 4 + (e & 3)][fr] = acc[i][j][e];
        __syncthreads();
        for (int i = threadIdx.x; i < RF * 1024; i += kLoraThreads) {
            const int row = i >> 5, c = i & 31, at = j0 + j * 32 + c;
            float v = (part[0][row][c] + part[1][row][c]) + (part[2][row][c] + part[3][row][c]);
            if (!finite(v) && row < left && at < rank) v = plain_sum<TX, TW>(P, t, adapter, row, at, blockIdx.y, P.splits);
            if (row < left && at < P.hrank) h[(int64_t)row * P.hrank + at] = at < rank ? v * f : 0.f;
        }
        __syncthreads();
    }
}

// A row's share of H (eight ranks of each step of 16) as MFMA operands. Returns which of a wave's 32 rows have a value
// that is not finite: zeros here, for plain_columns.
template <int KS>
__device__ __forceinline__ unsigned operands_of_h(Eight<float> (&v)[KS], bf16x8 (&hp)[KS][3]) {
    float odd = 0.f;  // NaN then
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = fmaf(v[ks].a[e], 0.f, fmaf(v[ks].b[e], 0.f, odd));
    const unsigned long long m = __ballot(odd != 0.f);
    const unsigned rows = (unsigned)m | (unsigned)(m >> 32);
    if (rows) {
        const int n = rows >> (threadIdx.x & 31) & 1 ? 0 : 8;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) v[ks].cut(n);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) v[ks].parts(hp[ks]);
    return rows;
}

// The same from scratch, from j0 on, its parts of K summed.
template <int KS>
__device__ __forceinline__ unsigned parts_of_h(const Lora& P, int64_t row, int j0, int rank, int fh, bf16x8 (&hp)[KS][3]) {
    constexpr int AHEAD = KS >= 8 ? 1 : KS >= 4 ? 2 : 4;  // parts asked for at once
    const float* h = P.h + row * P.hrank + j0 + fh * 8;
    const int64_t next = (int64_t)P.M * P.hrank;
    Eight<float> v[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) v[ks].a = v[ks].b = f4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < P.splits; s += AHEAD) {
        f4 x[AHEAD][KS][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                x[u][ks][0] = x[u][ks][1] = f4{0.f, 0.f, 0.f, 0.f};
                if (s + u < P.splits && j0 + ks * 16 + fh * 8 < rank) {
                    const f4* q = (const f4*)(h + (s + u) * next + ks * 16);
                    x[u][ks][0] = q[0], x[u][ks][1] = q[1];
                }
            }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) v[ks].a += x[u][ks][0], v[ks].b += x[u][ks][1];
    }
    return operands_of_h<KS>(v, hp);
}

// A bit for each of the first `left` of 32 rows.
__device__ __forceinline__ unsigned rows_of(int left) { return left >= 32 ? ~0u : (1u << max(left, 0)) - 1u; }

// What the values of H at the ranks j0 .. j1 add to the columns n .. n1 of `rows` of the 32 from `first` on, in fp32, behind
// a wave's other work on them; h: H's rows, or null for those in scratch. Each lane takes the places of C that it has itself
// written there. A call, and P by the address of the kernel's arguments: inside the kernels it cost their loops 30 registers.
typedef const __attribute__((address_space(4))) Lora* LoraArgs;
__device__ __forceinline__ LoraArgs lora_args() { return (LoraArgs)__builtin_amdgcn_kernarg_segment_ptr(); }  // a kernel's first argument
template <class TW>
__device__ __attribute__((noinline)) void plain_columns(LoraArgs P, int adapter, int j0, int j1, unsigned rows, int64_t first, int n, int n1, const float* h,
                                                        int ldh) {
    const TW* b = (const TW*)P->b + (int64_t)adapter * P->N * P->rank;
    for (; rows; rows &= rows - 1) {
        const int row = __ffs(rows) - 1;
        if ((row >> 2 & 1) != (int)(threadIdx.x >> 5 & 1)) continue;
        for (int n0 = n; n0 < n1; n0 += 128)
            for (int col = n0 + (threadIdx.x & 31) * 4, end = min(col + 4, P->N); col < end; ++col) {
                float sum = 0.f;
                for (int r = j0; r < j1 && sum == sum; ++r) {
                    float x = 0.f;
                    if (h) x = h[row * ldh + r];
                    else
                        for (int s = 0; s < P->splits; ++s) x += P->h[((int64_t)s * P->M + first + row) * P->hrank + r];
                    sum = fmaf(x, value(b[(int64_t)col * P->rank + r]), sum);
                }
                P->c[(first + row) * P->ldc + col] += sum;
            }
    }
}

// ---------------------------------------------------------------------------
// C[t, :] (+)= H[t] B_a^T over the ranks j0 .. j0 + 16 KS. A wave keeps the parts of 32 rows
// of H in registers and goes through `columns` columns, 128 at a time: four products, the
// j-th with the columns 4 i + j, so that a lane's four results of a row are neighbours and a
// row of C moves in 512-byte pieces (CV; else by single values). The four waves of a
// workgroup have neighbouring rows and the same columns (their B comes from the L1), or,
// with FEW, the same rows and neighbouring columns.
// ---------------------------------------------------------------------------
// The columns n .. n1 of a wave's rows, `left` of them, from c on; hp null without an adapter: zeros.
template <class TW, int KS, bool VEC, bool CV>
__device__ __forceinline__ void up_columns(const Lora& P, int adapter, int rank, int j0, const bf16x8 (*hp)[3], int n, int n1, float* c, int left, char* lds) {
    const int lane = threadIdx.x & 63, fr = lane & 31, fh = lane >> 5;
    auto row_of = [&](int e) { return (e >> 2) * 8 + fh * 4 + (e & 3); };
    auto put = [&](int e, int col, const f4& v) __attribute__((always_inline)) {
        float* to = c + row_of(e) * P.ldc + col;
        if (row_of(e) >= left) return;
        if constexpr (CV) {
            if (col < P.N) dev::st_stream((f4*)to, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < P.N) to[j] = v[j];
        }
    };
    if (!hp) {
        for (; n < n1; n += 128)
#pragma unroll
            for (int e = 0; e < 16; ++e) put(e, n + fr * 4, f4{0.f, 0.f, 0.f, 0.f});
        return;
    }
    const TW* b = (const TW*)P.b + (int64_t)adapter * P.N * P.rank;
    for (; n < n1; n += 128) {
        const int col = n + fr * 4;
        f4 y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            y[e] = f4{0.f, 0.f, 0.f, 0.f};
            if (!P.accumulate || row_of(e) >= left) continue;
            const float* from = c + row_of(e) * P.ldc + col;
            if constexpr (CV) {
                if (col < P.N) y[e] = *(const f4*)from;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < P.N) y[e][j] = from[j];
            }
        }
        f32x16 acc[4];
        // bf16 rows of whole lines come STAGED: 48 single rows of 2560 to 4096 columns, rank 64, 19.1 -> 17.3 us. fp32 ones
        // do not: their parts leave no registers for a second stage (rank 128 58 -> 68).
        constexpr int BLOCK = 128 / sizeof(TW), BLOCKS = KS * 16 / BLOCK;
        constexpr bool STAGE = VEC && sizeof(TW) == 2 && BLOCKS > 0;
        Staged<TW, BLOCK> staged[2][STAGE ? BLOCKS : 1];
        auto ask = [&](int j) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) {
                staged[j & 1][k].rows_of(b, P.rank, n + j, 4, P.N - 1);
                staged[j & 1][k].load(j0 + k * BLOCK, rank);
            }
        };
        if constexpr (STAGE) ask(0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Eight<TW> bn[KS];
            if constexpr (STAGE) {
                if (j < 3) ask(j + 1);
#pragma unroll
                for (int k = 0; k < BLOCKS; ++k) staged[j & 1][k].template deal<false>(lds, bn + k * (BLOCK / 16));
            } else {
                const TW* row = b + (int64_t)min(col + j, P.N - 1) * P.rank;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) bn[ks].template load<VEC>(row, j0 + ks * 16 + fh * 8, rank);
            }
            if (VEC && rank % 8) {  // what lies behind the ranks that count may be anything
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) bn[ks].cut(rank - (j0 + ks * 16 + fh * 8));
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 bp[Eight<TW>::kParts];
                bn[ks].parts(bp);
                acc[j] = multiply<3, Eight<TW>::kParts>(hp[ks], bp, acc[j]);
            }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) put(e, col, y[e] + f4{acc[0][e], acc[1][e], acc[2][e], acc[3][e]});
    }
}

template <class TW, int KS, bool FEW, bool VEC, bool CV>
__global__ __launch_bounds__(kLoraThreads, KS <= 4 ? 2 : 1) void k_lora_up(Lora P, int j0, int columns) {
    __shared__ __attribute__((aligned(16))) char lds[VEC ? kLoraWaves : 1][4096];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 31, fh = lane >> 5;
    dev::SpanTile t;
    if (!dev::find_tile(P.runs, P.count, P.M, 1, FEW ? 32 : 32 * kLoraWaves, blockIdx.x, t)) return;
    int rank;
    const int adapter = adapter_of(P, t, rank);
    const int row0 = t.row0 + (FEW ? 0 : w * 32), left = t.rows - row0;
    const int n = (FEW ? blockIdx.y * kLoraWaves + w : blockIdx.y) * columns, n1 = min(n + columns, P.N);
    if (left <= 0 || n >= n1 || (P.accumulate && j0 >= rank)) return;
    const int64_t first = t.first + row0;
    float* c = P.c + first * P.ldc;
    if (adapter < 0) {  // only without accumulate; B may not be there at all
        up_columns<TW, KS, VEC, CV>(P, adapter, rank, j0, nullptr, n, n1, c, left, nullptr);
        return;
    }
    bf16x8 hp[KS][3];
    const unsigned odd = parts_of_h<KS>(P, first + min(fr, left - 1), j0, rank, fh, hp) & rows_of(left);
    up_columns<TW, KS, VEC, CV>(P, adapter, rank, j0, hp, n, n1, c, left, lds[VEC ? w : 0]);
    if (odd) plain_columns<TW>(lora_args(), adapter, j0, min(rank, j0 + KS * 16), odd, first, n, n1, nullptr, 0);
}

// Both in one launch, for few rows a run and a short K: every workgroup of a run forms H for
// itself, in LDS. A is then read once for each of them (from the L2), which costs less than
// the second launch's beginning as long as K is short (the rule stands at the launch).
template <class TX, class TW, int KS, bool XVEC, bool VEC, bool CV>
__global__ __launch_bounds__(kLoraThreads, 2) void k_lora_small(Lora P, int columns) {
    constexpr int RT = (KS + 1) / 2;
    __shared__ __attribute__((aligned(16))) float part[kLoraWaves][32][33];
    __shared__ __attribute__((aligned(16))) float h[32][RT * 32 + 4];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 31, fh = lane >> 5;
    dev::SpanTile t;
    if (!dev::find_tile(P.runs, P.count, P.M, 1, 32, blockIdx.x, t)) return;
    int rank;
    const int adapter = adapter_of(P, t, rank), left = t.rows - t.row0;
    const int n = (blockIdx.y * kLoraWaves + w) * columns, n1 = min(n + columns, P.N);
    if (P.accumulate && !rank) return;
    float* c = P.c + (int64_t)(t.first + t.row0) * P.ldc;
    if (adapter < 0) {
        up_columns<TW, KS, VEC, CV>(P, adapter, rank, 0, nullptr, n, n1, c, left, nullptr);
        return;
    }
    f32x16 acc[1][RT];
    down_sums<TX, TW, RT, 1, XVEC ? kOperands : kValues>(P, t, adapter, rank, 0, 0, 1, (char*)part[w], acc);
    const float f = P.scale ? P.scale[adapter] : 1.0f;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
#pragma unroll
        for (int e = 0; e < 16; ++e) part[w][(e >> 2) * 8 + fh * 4 + (e & 3)][fr] = acc[0][j][e];
        __syncthreads();
        for (int i = threadIdx.x; i < 1024; i += kLoraThreads) {
            const int row = i >> 5, col = i & 31;
            float v = (part[0][row][col] + part[1][row][col]) + (part[2][row][col] + part[3][row][col]);
            if (!finite(v) && row < left && j * 32 + col < rank) v = plain_sum<TX, TW>(P, t, adapter, row, j * 32 + col, 0, 1);
            h[row][j * 32 + col] = j * 32 + col < rank ? v * f : 0.f;
        }
        __syncthreads();
    }
    bf16x8 hp[KS][3];
    Eight<float> v[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        v[ks].a = *(const f4*)&h[fr][ks * 16 + fh * 8];
        v[ks].b = *(const f4*)&h[fr][ks * 16 + fh * 8 + 4];
    }
    const unsigned odd = operands_of_h<KS>(v, hp) & rows_of(left);
    up_columns<TW, KS, VEC, CV>(P, adapter, rank, 0, hp, n, n1, c, left, (char*)part[w]);
    if (odd) plain_columns<TW>(lora_args(), adapter, 0, rank, odd, t.first + t.row0, n, n1, &h[0][0], RT * 32 + 4);
}

// Up for runs of many rows: the waves of a workgroup have neighbouring rows and share
// each 128 columns of B through LDS. Read from memory by its rows, a fragment (32 rows of B,
// 16 bytes each a lane) costs the L1 an access a lane: 60 million of them took 112 of 185 us
// at [12528,64] x [10240,64]^T. The copies to LDS are of whole rows, 16 bytes a lane, two
// stages; LDS row j*32 + i holds column 4 i + j, its 16-byte piece c at c ^ swizzle(row), so
// that 16 neighbouring rows are read from 16 different pieces of a 256-byte window.
template <class TW, int KS, bool ACC, bool CV>
__global__ __launch_bounds__(kLoraThreads, KS <= 4 ? 2 : 1) void k_lora_up_shared(Lora P, int j0, int columns) {
    constexpr int PER = 16 / sizeof(TW), PIECES = KS * 16 / PER, ROW = PIECES * 16, STAGE = 128 * ROW;  // pieces a row, bytes
    constexpr int TURN = PIECES >= 16 ? 1 : 16 / PIECES;  // rows in 256 bytes
    __shared__ __attribute__((aligned(1024))) char stage0[STAGE], stage1[STAGE];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 31, fh = lane >> 5;
    dev::SpanTile t;
    if (!dev::find_tile(P.runs, P.count, P.M, 1, 32 * kLoraWaves, blockIdx.x, t)) return;
    int rank;
    const int adapter = adapter_of(P, t, rank);
    const int n0 = blockIdx.y * columns, n1 = min(n0 + columns, P.N);
    if (ACC && j0 >= rank) return;
    const int row0 = t.row0 + w * 32, left = t.rows - row0;
    const int64_t first = t.first + row0;
    float* c = P.c + first * P.ldc;
    auto row_of = [&](int e) { return (e >> 2) * 8 + fh * 4 + (e & 3); };
    auto put = [&](int e, int col, const f4& v) __attribute__((always_inline)) {
        float* to = c + row_of(e) * P.ldc + col;
        if (row_of(e) >= left) return;
        if constexpr (CV) {
            if (col < P.N) dev::st_stream((f4*)to, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < P.N) to[j] = v[j];
        }
    };
    if (adapter < 0) {  // only without accumulate; B may not be there at all
        for (int n = n0; n < n1; n += 128)
#pragma unroll
            for (int e = 0; e < 16; ++e) put(e, n + fr * 4, f4{0.f, 0.f, 0.f, 0.f});
        return;
    }
    const TW* b = (const TW*)P.b + (int64_t)adapter * P.N * P.rank;
    auto swizzle = [](int row) { return (row / TURN) & (PIECES - 1); };
    auto copy = [&](int n, char* to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < STAGE / (kLoraThreads * 16); ++i) {
            const int chunk = (i * kLoraWaves + w) * 64, at = chunk + lane, row = at / PIECES, c = (at % PIECES) ^ swizzle(row);
            const int col = min(n + (row & 31) * 4 + (row >> 5), P.N - 1), k = j0 + c * PER;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(b + (int64_t)col * P.rank + (k < P.rank ? k : 0)),
                                             (__attribute__((address_space(3))) void*)(to + chunk * 16), 16, 0, 0);
        }
    };
    copy(n0, stage0);
    bf16x8 hp[KS][3];
    const unsigned odd = parts_of_h<KS>(P, t.first + min(row0 + fr, t.rows - 1), j0, rank, fh, hp) & rows_of(left);
    auto landed = [] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
    landed();
    auto step = [&](int n, const char* from, char* to) __attribute__((always_inline)) {
        // This stage has landed (waited for in front of the last stores of C, which have a whole
        // step to leave) and nobody reads the other one any more.
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (n + 128 < n1) copy(n + 128, to);
        if (left <= 0) {
            landed();
            return;
        }
        const int col = n + fr * 4;
        f4 y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            y[e] = f4{0.f, 0.f, 0.f, 0.f};
            if (!ACC || row_of(e) >= left) continue;
            const float* at = c + row_of(e) * P.ldc + col;
            if constexpr (CV) {
                if (col < P.N) y[e] = dev::ld_stream((const f4*)at);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < P.N) y[e][j] = at[j];
            }
        }
        f32x16 acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int row = j * 32 + fr;
                Eight<TW> v;
                if constexpr (sizeof(TW) == 2) {
                    v.a = *(const u32x4*)(from + row * ROW + (((ks * 2 + fh) ^ swizzle(row)) << 4));
                } else {
                    v.a = *(const f4*)(from + row * ROW + (((ks * 4 + fh * 2) ^ swizzle(row)) << 4));
                    v.b = *(const f4*)(from + row * ROW + (((ks * 4 + fh * 2 + 1) ^ swizzle(row)) << 4));
                }
                if (j0 + ks * 16 + 16 > rank) v.cut(rank - (j0 + ks * 16 + fh * 8));  // what lies behind the ranks that count may be anything
                bf16x8 bp[Eight<TW>::kParts];
                v.parts(bp);
                acc[j] = multiply<3, Eight<TW>::kParts>(hp[ks], bp, acc[j]);
            }
        }
        landed();
#pragma unroll
        for (int e = 0; e < 16; ++e) put(e, col, y[e] + f4{acc[0][e], acc[1][e], acc[2][e], acc[3][e]});
    };
    for (int n = n0; n < n1; n += 256) {
        step(n, stage0, stage1);
        if (n + 128 < n1) step(n + 128, stage1, stage0);
    }
    if (odd) plain_columns<TW>(lora_args(), adapter, j0, min(rank, j0 + KS * 16), odd, first, n0, n1, nullptr, 0);
}

template <class TX, class TW>
void launch_lora(Lora P, int64_t M, bool vec) {
    using std::integral_constant;
    using T_ = std::true_type;
    using F_ = std::false_type;
    const int cus = num_cus();
    // Few rows a run: 32-row tiles.
    const bool few = M <= 32 * (int64_t)P.count;
    const int rt = P.rank <= 32 ? 1 : P.rank <= 64 ? 2 : 4, rf = few || rt > 2 || !vec ? 1 : 2;
    const int64_t down = M / (32 * rf) + std::min<int64_t>(P.count, M);
    const int64_t tiles = M / (few ? 32 : 128) + std::min<int64_t>(P.count, M);
    const bool bvec = P.rank % 8 == 0 && aligned16(P.b), cvec = P.N % 4 == 0 && P.ldc % 4 == 0 && aligned16(P.c);
    // Columns of a workgroup's wave: as many as leave four workgroups a CU (with few rows, soon
    // done, six), since each begins with H and its parts. Measured, us, for two / four a CU:
    // [8192,640] -> 5120 rank 12 87 / 79, [12528,3840] -> 10240 rank 64 168 / 167.
    int64_t columns = 4096;
    while (columns > 128 && tiles * ((P.N + columns * (few ? kLoraWaves : 1) - 1) / (columns * (few ? kLoraWaves : 1))) < (few ? 6 : 4) * (int64_t)cus)
        columns /= 2;
    // One launch or two, for few rows a run: by K and the bytes of a row of B. Measured, us, one / two, 48 single rows to
    // 4096 columns: bf16 K 320 rank 8 7.4 / 9.3, rank 64 11.9 / 13.9; K 640 rank 8 8.4 / 9.3, rank 64 14.1 / 14.4; K 1280
    // rank 8 11.7 / 9.5; fp32 rank 64 K 320 24.0 / 23.7, K 640 28.6 / 24.6.
    if (few && P.rank > 0 && P.rank * sizeof(TW) <= 128 && P.K <= 640) {
        const dim3 grid((unsigned)tiles, (unsigned)((P.N + columns * kLoraWaves - 1) / (columns * kLoraWaves)));
        auto go = [&](auto k, auto x, auto v) {
            constexpr int KS = decltype(k)::value;
            constexpr bool X = decltype(x)::value, V = decltype(v)::value;
            if (cvec) k_lora_small<TX, TW, KS, X, V, true><<<grid, kLoraThreads, 0, stream()>>>(P, (int)columns);
            else k_lora_small<TX, TW, KS, X, V, false><<<grid, kLoraThreads, 0, stream()>>>(P, (int)columns);
        };
        auto with = [&](auto x, auto v) {
            if (P.rank <= 16) go(integral_constant<int, 1>(), x, v);
            else if (P.rank <= 32) go(integral_constant<int, 2>(), x, v);
            else if constexpr (sizeof(TW) == 2) go(integral_constant<int, 4>(), x, v);
        };
        if (vec && bvec) with(T_(), T_());
        else with(F_(), F_());
        return;
    }
    if (P.rank > 0) {
        // Parts of K until the chip has two workgroups a CU, as many as fit, while each wave keeps two
        // blocks, and at most four, which up has to sum: [2480,2560] -> 4096 takes 42 us with two, 38 with
        // four, 44 with eight; [12528,3840] bf16 -> 10240 rank 64 137 us with two (this rule), 145 with four,
        // 150 with one.
        const int64_t most = std::max<int64_t>(1, P.K / (64 * kLoraWaves));
        P.splits = (int)std::max<int64_t>(1, std::min<int64_t>({most, 2 * cus / std::max<int64_t>(1, M / (32 * rf) + 1), 4}));
    }
    P.hrank = (P.rank + 31) / 32 * 32;
    P.h = (float*)scratch(std::max<size_t>((size_t)P.splits * M * P.hrank * 4, 4));
    if (P.rank > 0) {
        const dim3 grid((unsigned)down, (unsigned)P.splits, (unsigned)((P.rank + rt * 32 - 1) / (rt * 32)));
        auto go = [&](auto r, auto f, auto v) {
            k_lora_down<TX, TW, decltype(r)::value, decltype(f)::value, decltype(v)::value><<<grid, kLoraThreads, 0, stream()>>>(P);
        };
        using One = integral_constant<int, 1>;
        using Two = integral_constant<int, 2>;
        using Four = integral_constant<int, 4>;
        using Values = integral_constant<int, kValues>;
        using Operands = integral_constant<int, kOperands>;
        using Staged = integral_constant<int, kStaged>;
        auto with = [&](auto r) {  // four tiles of ranks go with one of rows
            if (!vec) go(r, One(), Values());
            else if (few) go(r, One(), Operands());
            else if constexpr (decltype(r)::value > 2) go(r, One(), Staged());
            else go(r, Two(), Staged());
        };
        if (rt == 1) with(One());
        else if (rt == 2) with(Two());
        else with(Four());
    }
    // Ranks of a launch: 128, for whose parts of B and H a wave of few rows has no registers. 48 single rows of 2560 to
    // 4096 columns, rank 128, us, one launch / two of 64: bf16 35.7 / 30.0, fp32 58 / 52; eight runs of four to 1000
    // columns 21.7 / 23.5, 40 / 45.
    const int per = few ? 64 : 128;
    for (int j0 = 0; j0 == 0 || j0 < P.rank; j0 += per) {
        const int ks = std::min(P.rank - j0, per);
        const dim3 grid((unsigned)tiles, (unsigned)((P.N + columns * (few ? kLoraWaves : 1) - 1) / (columns * (few ? kLoraWaves : 1))));
        auto go = [&](auto k, auto f, auto v) {
            constexpr int KS = decltype(k)::value;
            constexpr bool F = decltype(f)::value, V = decltype(v)::value;
            // pieces of 16 bytes, whole ones a row
            if constexpr (!F)
                if (P.rank % (16 / sizeof(TW)) == 0 && aligned16(P.b)) {
                    auto shared = P.accumulate ? (cvec ? k_lora_up_shared<TW, KS, true, true> : k_lora_up_shared<TW, KS, true, false>)
                                               : (cvec ? k_lora_up_shared<TW, KS, false, true> : k_lora_up_shared<TW, KS, false, false>);
                    shared<<<grid, kLoraThreads, 0, stream()>>>(P, j0, (int)columns);
                    return;
                }
            if (cvec) k_lora_up<TW, KS, F, V, true><<<grid, kLoraThreads, 0, stream()>>>(P, j0, (int)columns);
            else k_lora_up<TW, KS, F, V, false><<<grid, kLoraThreads, 0, stream()>>>(P, j0, (int)columns);
        };
        auto with = [&](auto f, auto v) {
            if (ks <= 16) go(integral_constant<int, 1>(), f, v);
            else if (ks <= 32) go(integral_constant<int, 2>(), f, v);
            else if (ks <= 64) go(integral_constant<int, 4>(), f, v);
            else if constexpr (!decltype(f)::value) go(integral_constant<int, 8>(), f, v);
        };
        if (few) bvec ? with(T_(), T_()) : with(T_(), F_());
        else with(F_(), F_());
        P.accumulate = 1;
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
    need(count <= dev::kMaxSpans, op, "more than 65536 segments");
    need(std::max(ldx, ldc) <= (int64_t(1) << 46) / std::max<int64_t>(M, 1) &&
             adapters * std::max<int64_t>(rank, 1) <= (int64_t(1) << 46) / std::max<int64_t>({N, K, 1}),
         op, "matrix too large");
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
    need((N + 31) / 32 <= 65535 && (M / 32 + std::min(count, M) + 1) * kLoraThreads <= kMaxGridItems, op, "matrix too large for one launch");
    Lora P{X, A, B, scale, (const int4*)segments, nullptr, C, ldx, ldc, (int)M, (int)N, (int)K, any ? (int)rank : 0, any ? (int)adapters : 0,
           (int)count, 1, 0, accumulate ? 1 : 0};
    const bool vec = K % 8 == 0 && ldx % (16 / sizeof(TX)) == 0 && aligned16(X) && aligned16(A);
    launch_lora<TX, TW>(P, M, vec);
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
