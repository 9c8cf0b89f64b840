// k_attn_packed.hip - attention over sequences packed into one tensor: the rows of
// many requests, each attending the keys of its own, under a causal, window or
// prefix mask, with scores capped by a tanh or biased by distance (no reference
// function; backend_cuda.h:57-59 attention() takes batches of one length).
//
// Query i of a sequence with lq queries and lk keys stands at position
// p = i + lk - lq among its keys: the last query at the last key. It sees key j when
// j < prefix, or when (not causal or j <= p) and (no window or |p - j| < window): the
// union of [0, prefix) and one interval [lo, hi). Its scores are
// x = scale q.k, then cap tanh(x / cap), then + bias[h, clamp(j - p, -R, R) + R]; a row
// that sees nothing, or only keys biased by -inf, gives zeros.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "fp16_pair.hpp"
#include "spans.hpp"

namespace sdh {
namespace {

typedef unsigned short u16;
typedef float f2 __attribute__((ext_vector_type(2)));
using dev::f4;
constexpr float kLog2e = 1.44269504088896341f;

struct Packed {
    const float *q, *k, *v;
    void* out;
    const int4* spans;
    const int* prefix;
    const float* bias;
    int Tq, Tk, seqs, heads, kv_heads, d, causal, window, radius;  // window 0: none
    float scale, cap;
};

// The keys that a query sees: [0, pre) and [lo, hi), the latter behind the former.
struct Seen {
    int pre, lo, hi;
};
__device__ __forceinline__ Seen seen_from(const Packed& P, int p, int lk, int pre) {
    int lo = 0, hi = lk;
    if (P.window) {
        lo = p - P.window + 1;
        hi = min(hi, p + P.window);
    }
    if (P.causal) hi = min(hi, p + 1);
    lo = max(lo, pre);
    return Seen{pre, lo, max(hi, lo)};
}

// tanh to about 3e-7 of itself. Near zero 1 - e would cancel: a polynomial (its next
// term is below 2e-8 of the sum at 0.35).
__device__ __forceinline__ float tanh_near(float x) {
    const float a = fabsf(x), x2 = x * x;
    const float e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * a);
    const float far = copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), x);
    const float p = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1382.0f / 155925.0f, 62.0f / 2835.0f), -17.0f / 315.0f), 2.0f / 15.0f),
                         -1.0f / 3.0f);
    return a < 0.35f ? fmaf(x * x2, p, x) : far;
}

// ---------------------------------------------------------------------------
// Any head dimension: fp32 products, one wave per (query, head). Lanes take 64 keys at a
// time for the scores, then 64 columns at a time for the weighted sum.
// ---------------------------------------------------------------------------
constexpr int kRowWaves = 4, kMaxD = 1024;

template <bool OUT16>
__global__ __launch_bounds__(64 * kRowWaves) void k_attn_packed_rows(Packed P) {
    __shared__ float sq[kRowWaves][kMaxD];
    __shared__ float sp[kRowWaves][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int t = blockIdx.x * kRowWaves + w, h = blockIdx.y, d = P.d;
    if (t >= P.Tq) return;  // whole wave; no block-level barrier below
    const int s = dev::span_of_row(P.spans, P.seqs, t, P.Tq);
    if (s < 0) return;
    int4 e = P.spans[s];
    dev::cut_span(e.x, e.y, P.Tq);
    dev::cut_span(e.z, e.w, P.Tk);
    const int lk = e.w, p = t - e.x + lk - e.y;
    const Seen r = seen_from(P, p, lk, P.prefix ? min(max(P.prefix[s], 0), lk) : 0);
    const int64_t inner = (int64_t)P.heads * d, kv_inner = (int64_t)P.kv_heads * d;
    const int64_t at = (int64_t)t * inner + (int64_t)h * d;
    const int64_t kv0 = e.z * kv_inner + (int64_t)(h / (P.heads / P.kv_heads)) * d;
    for (int c = lane; c < d; c += 64) sq[w][c] = P.q[at + c];
    __builtin_amdgcn_wave_barrier();
    constexpr int kAcc = kMaxD / 64;
    float acc[kAcc];
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i] = 0.f;
    float m = -INFINITY, sum = 0.f;
    auto keys = [&](int from, int to) {
        for (int k0 = from; k0 < to; k0 += 64) {
            const int j = k0 + lane;
            float x = -INFINITY;
            if (j < to) {
                const float* kp = P.k + kv0 + j * kv_inner;
                float a = 0.f;
                for (int c = 0; c < d; ++c) a = fmaf(sq[w][c], kp[c], a);
                x = a * P.scale;
                if (P.cap > 0.f) x = P.cap * tanh_near(x / P.cap);
                if (P.bias) x += P.bias[(int64_t)h * (2 * P.radius + 1) + min(max(j - p, -P.radius), P.radius) + P.radius];
            }
            const float mnew = fmaxf(m, dev::wave_max(x));
            const float ref = mnew == -INFINITY ? 0.f : mnew;  // nothing but -inf so far
            const float alpha = __builtin_amdgcn_exp2f((m - ref) * kLog2e);
            m = mnew;
            const float weight = __builtin_amdgcn_exp2f((x - ref) * kLog2e);
            sum = sum * alpha + dev::wave_sum(weight);
            __builtin_amdgcn_wave_barrier();
            sp[w][lane] = weight;
            __builtin_amdgcn_wave_barrier();
            const int nk = min(64, to - k0);
#pragma unroll
            for (int i = 0; i < kAcc; ++i) {
                const int c = i * 64 + lane;
                if (i * 64 >= d) break;
                float a = acc[i] * alpha;
                if (c < d)
                    for (int u = 0; u < nk; ++u) a = fmaf(sp[w][u], P.v[kv0 + (k0 + u) * kv_inner + c], a);
                acc[i] = a;
            }
        }
    };
    keys(0, r.pre);
    keys(r.lo, r.hi);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kAcc; ++i) {
        const int c = i * 64 + lane;
        if (i * 64 >= d) break;
        if (c < d) {
            if constexpr (OUT16) ((u16*)P.out)[at + c] = dev::bf16_rne(acc[i] * inv);
            else ((float*)P.out)[at + c] = acc[i] * inv;
        }
    }
}

// ---------------------------------------------------------------------------
// Head dimensions up to 128 (padded to DP = 64 or 128), on the MFMA units.
//
// A workgroup takes kTileRows rows of one sequence and key/value head, a row being a
// (query, head of the group) pair, heads fastest: the heads that share a key/value head
// share its tiles. It walks the 64-key tiles that any of its rows sees. The eight waves
// bring a tile in together, eight keys each, from fp32 in memory to fp16 pairs in LDS,
// and each wave then takes 32 rows against it.
//
// Operands are fp16 pairs hi + lo in block floating point, products hi hi + hi lo +
// lo hi with fp32 sums (2^-21 of each product). A block is a row of q, or the eight keys
// that a wave brought in: with k or v scaled by 2^-e to at most 2^14, a score is
// s 2^(e_q + e_k), and a weight is formed as p 2^(14 + e_v - E), E the largest e_v that the
// lane's row has seen, so that the sums of all blocks share the scale 2^(14 - E).
// Rows in LDS are ordered so that the eight scores of a lane's half of a 16-key step are
// eight neighbouring keys: one block, one exponent. Tiles at the border of what the rows
// see have an exponent for each key: an unseen key, whatever its size, then has no say
// in the others'. Values that are not finite go into the tiles as zeros, since 0 * inf would
// reach the rows that do not see them, and are added at the end; a key that is not finite
// makes the scores of the rows that see it NaN, and only those.
//
// S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_32x32x16_f16: lane l holds row l % 32 of
// the wave in both, its statistics are its own, and its weights are the second product's
// operand as they lie.
// ---------------------------------------------------------------------------
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Where the keys of a row are cut into parts (S.n of them, by blockIdx.y): each part's
// sum of weighted values, and its reference and sum of weights, for k_attn_packed_join.
struct Parts {
    int n, stride;  // floats of a cell: d up to the next 4
    float* o;       // [Tq, heads, n, stride]
    f2* ml;         // [Tq, heads, n]
};

constexpr int kKT = 64, kWaves = 8, kThreads = 64 * kWaves, kTileRows = 32 * kWaves;
// The reference m of the weights is raised when a tile's largest score passes it by more
// than this (in units of log2): weights stay below 2^(14 + kLazy), inside fp16.
constexpr float kLazy = 1.5f;
constexpr int kUnsetE = -1000;  // no values seen yet
constexpr int kFarE = -40;      // weights' exponents relative to E are not taken below this (2^-40 of the largest sum)

__device__ __forceinline__ int swz_v(int r) { return (r >> 1) & 7; }
template <int DP>
__device__ __forceinline__ int swz_k(int r) {
    return DP == 128 ? (r & 15) : ((r >> 1) & 7);
}
__device__ __forceinline__ int row_of_key(int j) { return (j & ~12) | ((j & 4) << 1) | ((j & 8) >> 1); }

template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
// Largest non-negative int over aligned groups of W lanes (8, 16 or 64).
template <int W>
__device__ __forceinline__ int group_imax(int v) {
    v = max(v, dpp_i<0xB1>(v));
    v = max(v, dpp_i<0x4E>(v));
    v = max(v, dpp_i<0x141>(v));
    if constexpr (W >= 16) v = max(v, dpp_i<0x140>(v));
    if constexpr (W == 64) {
        const int a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16), c = __builtin_amdgcn_readlane(v, 32),
                  d = __builtin_amdgcn_readlane(v, 48);
        v = max(max(a, b), max(c, d));
    }
    return v;
}
__device__ __forceinline__ int abs_bits(float x) { return (int)(__float_as_uint(x) & 0x7FFFFFFFu); }
constexpr int kInfBits = 0x7F800000;
// The exponent that brings a block's largest magnitude into [2^13, 2^14); zero and
// subnormal blocks the least there is.
__device__ __forceinline__ int block_exp(int bits) { return min(max((bits >> 23) - 140, -126), 126); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }  // e in [-126, 127]

template <int DP, bool OUT16, bool EXTRA, bool VEC>
__global__ __launch_bounds__(kThreads, 1) void k_attn_packed_tiles(Packed P, int items, Parts S) {
    constexpr int DS = DP / 16, DT = DP / 32, KU = DP / 64, PART = kKT * DP;
    // [K hi][K lo][V^T hi][V^T lo] of two tiles
    __shared__ __attribute__((aligned(1024))) u16 buf[2][4 * PART];
    __shared__ __attribute__((aligned(16))) int exps[2][2][8];      // of k, v, eight keys each
    __shared__ __attribute__((aligned(16))) int key_exps[2][2][kKT];  // at a border: of each key
    __shared__ __attribute__((aligned(16))) int bads[2][8];         // values that are not finite
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 31, fh = lane >> 5;
    const int group = P.heads / P.kv_heads;
    // Workgroups are dealt to the 8 XCDs in turn; renumbered so that an XCD has
    // neighbouring row tiles of a sequence and head, whose keys its L2 then holds.
    const int per = gridDim.x >> 3, rem = gridDim.x & 7, xcd = blockIdx.x & 7;
    const int lb = xcd * per + min(xcd, rem) + (blockIdx.x >> 3);
    const int kh = lb / items;
    dev::SpanTile T;
    if (!dev::find_tile(P.spans, P.seqs, P.Tq, group, kTileRows, lb - kh * items, T)) return;
    dev::cut_span(T.z, T.w, P.Tk);
    const int d = P.d, rows = T.rows * group, lk = T.w, pre = P.prefix ? min(max(P.prefix[T.index], 0), lk) : 0;
    const int64_t inner = (int64_t)P.heads * d, kv_inner = (int64_t)P.kv_heads * d;
    const int r = T.row0 + w * 32 + fr;
    const int rc = min(r, rows - 1), qi = rc / group, h = kh * group + (rc - qi * group);
    const int shift = lk - T.rows;
    const int p = qi + shift;
    const Seen see = seen_from(P, p, lk, pre);
    const Seen wg_first = seen_from(P, T.row0 / group + shift, lk, pre),
               wg_last = seen_from(P, (min(T.row0 + kTileRows, rows) - 1) / group + shift, lk, pre);
    const int wg_lo = wg_first.lo, wg_hi = wg_last.hi;
    const bool active = T.row0 + w * 32 < rows;
    const int first_lo = __builtin_amdgcn_readlane(see.lo, 0), last_hi = __builtin_amdgcn_readlane(see.hi, 31);
    const int npre = (pre + kKT - 1) / kKT, next = max(npre, wg_lo / kKT);
    const int all = npre + (wg_hi > wg_lo ? max(0, (wg_hi + kKT - 1) / kKT - next) : 0);
    const int n0 = (int)((int64_t)all * blockIdx.y / S.n), nt = (int)((int64_t)all * (blockIdx.y + 1) / S.n);
    auto key_of = [&](int n) { return (n < npre ? n : next + n - npre) * kKT; };

    // Q: the B operand of S^T, row qi of head h, dims ds*16 + fh*8 .. +7
    const float* qp = P.q + (T.first + qi) * inner + (int64_t)h * d;
    h8 qh[DS], ql[DS];
    int eq;
    {
        float x[DS][8];
        int top = 0;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            const int c0 = ds * 16 + fh * 8;
            if constexpr (VEC) {
                const float* a = qp + min(c0, d - 8);
                const f4 u = *(const f4*)a, v = *(const f4*)(a + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[ds][e] = c0 < d ? (e < 4 ? u[e & 3] : v[e & 3]) : 0.f;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[ds][e] = c0 + e < d ? qp[c0 + e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[ds][e]));
        }
        top = max(top, __shfl_xor(top, 32, 64));
        eq = block_exp(top);
        const float sc = copysignf(pow2(-eq), P.scale);  // a negative scale turns q's sign
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                h2 hi, lo;
                split_pair(x[ds][e] * sc, x[ds][e + 1] * sc, hi, lo);
                qh[ds][e] = hi[0], qh[ds][e + 1] = hi[1];
                ql[ds][e] = lo[0], ql[ds][e + 1] = lo[1];
            }
    }
    const float scale = fabsf(P.scale);

    // A tile on its way: this wave's eight keys. k: 16-byte chunks of their rows; v: the
    // lane's columns of all eight.
    constexpr int KCH = DP / 8;  // chunks of a row
    const int kch = lane & (KCH - 1), krow = lane / KCH;
    constexpr int KROWS = 64 / KCH;
    float kx[KU][8], vx[8][KU];
    const float* kbase = P.k + T.z * kv_inner + (int64_t)kh * d;
    const float* vbase = P.v + T.z * kv_inner + (int64_t)kh * d;
    // a tile that some of the workgroup's rows see in part
    auto border = [&](int k0) { return !(k0 + kKT <= pre || (k0 >= wg_last.lo && k0 + kKT <= wg_first.hi)); };
    auto wanted = [&](int j) { return j < lk && (j < pre || (j >= wg_lo && j < wg_hi)); };
    auto fetch = [&](int n) __attribute__((always_inline)) {
        const int j0 = key_of(n) + w * 8;
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const float* a = kbase + (int64_t)min(j0 + u * KROWS + krow, lk - 1) * kv_inner;
            if constexpr (VEC) {
                a += min(kch * 8, d - 8);
                const f4 x = *(const f4*)a, y = *(const f4*)(a + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) kx[u][e] = e < 4 ? x[e & 3] : y[e & 3];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) kx[u][e] = a[min(kch * 8 + e, d - 1)];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float* a = vbase + (int64_t)min(j0 + i, lk - 1) * kv_inner;
            if constexpr (VEC && KU == 2) {
                const f2 x = *(const f2*)(a + min(lane * 2, d - 2));
                vx[i][0] = x.x, vx[i][1] = x.y;
            } else {
#pragma unroll
                for (int u = 0; u < KU; ++u) vx[i][u] = a[min(lane * KU + u, d - 1)];
            }
        }
    };
    // Into LDS: scaled, split, in the order of the fragments' reads.
    auto store = [&](int n, int b) __attribute__((always_inline)) {
        const int k0 = key_of(n), j0 = k0 + w * 8;
        int ktop = 0, vtop = 0;
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const bool ok = wanted(j0 + u * KROWS + krow);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!ok || kch * 8 + e >= d) kx[u][e] = 0.f;
                ktop = max(ktop, abs_bits(kx[u][e]));
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool ok = wanted(j0 + i);
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                if (!ok || lane * KU + u >= d) vx[i][u] = 0.f;
                vtop = max(vtop, abs_bits(vx[i][u]));
            }
        }
        ktop = group_imax<64>(ktop);
        vtop = group_imax<64>(vtop);
        const bool bad = vtop >= kInfBits;
        if (bad) {
            vtop = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int u = 0; u < KU; ++u) {
                    if (abs_bits(vx[i][u]) >= kInfBits) vx[i][u] = 0.f;
                    vtop = max(vtop, abs_bits(vx[i][u]));
                }
            vtop = group_imax<64>(vtop);
        }
        const int ek = block_exp(ktop), ev = block_exp(vtop);
        if (lane == 0) {
            exps[b][0][w] = ek;
            exps[b][1][w] = ev;
            bads[b][w] = bad;
        }
        float ks[KU], vs[8];
#pragma unroll
        for (int u = 0; u < KU; ++u) ks[u] = pow2(-ek);
#pragma unroll
        for (int i = 0; i < 8; ++i) vs[i] = pow2(-ev);
        if (border(k0)) {
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                int top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, abs_bits(kx[u][e]));
                const int e = block_exp(group_imax<KCH>(top));
                ks[u] = pow2(-e);
                if (kch == 0) key_exps[b][0][w * 8 + u * KROWS + krow] = e;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                int top = 0;
#pragma unroll
                for (int u = 0; u < KU; ++u) top = max(top, abs_bits(vx[i][u]));
                const int e = block_exp(group_imax<64>(top));
                vs[i] = pow2(-e);
                if (lane == 0) key_exps[b][1][w * 8 + i] = e;
            }
        }
        u16 *kd = buf[b], *vd = buf[b] + 2 * PART;
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int row = row_of_key(w * 8 + u * KROWS + krow);
            h8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                h2 a, c;
                split_pair(kx[u][e] * ks[u], kx[u][e + 1] * ks[u], a, c);
                hi[e] = a[0], hi[e + 1] = a[1];
                lo[e] = c[0], lo[e + 1] = c[1];
            }
            const int at = row * DP + ((kch ^ swz_k<DP>(row)) << 3);
            *(h8*)(kd + at) = hi;
            *(h8*)(kd + PART + at) = lo;
        }
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int row = lane * KU + u;
            h8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                h2 a, c;
                split_pair(vx[i][u] * vs[i], vx[i + 1][u] * vs[i + 1], a, c);
                hi[i] = a[0], hi[i + 1] = a[1];
                lo[i] = c[0], lo[i + 1] = c[1];
            }
            const int at = row * kKT + ((w ^ swz_v(row)) << 3);
            *(h8*)(vd + at) = hi;
            *(h8*)(vd + PART + at) = lo;
        }
    };

    f32x16 o[DT], s[2];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float m = -INFINITY, sum = 0.f;  // the reference (log2 units without EXTRA), this lane's keys' sum of weights
    int E = kUnsetE;

    auto scores = [&](const u16* kd) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[j][i] = 0.f;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            h8 kf[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = j * 32 + fr, at = row * DP + (((ds * 2 + fh) ^ swz_k<DP>(row)) << 3);
                kf[j][0] = *(const h8*)(kd + at);
                kf[j][1] = *(const h8*)(kd + PART + at);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j][0], qh[ds], s[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j][0], ql[ds], s[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j][1], qh[ds], s[j], 0, 0, 0);
        }
    };
    // Score register i of half j is key k0 + j*32 + (i/8)*16 + fh*8 + i%8.
    auto key_at = [&](int j, int i) { return j * 32 + (i >> 3) * 16 + fh * 8 + (i & 7); };
    auto visible = [&](int j) { return (j < pre) | ((j >= see.lo) & (j < see.hi)); };

    // s -> weights in place, the statistics and the scale of o brought up to date
    auto softmax = [&](int k0, int b) __attribute__((always_inline)) {
        const bool edge = border(k0);
        int ek[4], ev[4], emax = kUnsetE;
        if (edge) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                ek[u] = ev[u] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int j = u * 16 + fh * 8 + i;
                    const bool ok = visible(k0 + j);
                    s[u >> 1][(u & 1) * 8 + i] = ldexpf(s[u >> 1][(u & 1) * 8 + i], key_exps[b][0][j]);
                    if (ok) emax = max(emax, key_exps[b][1][j]);
                }
            }
            emax = max(emax, __shfl_xor(emax, 32, 64));
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                ek[u] = exps[b][0][u * 2 + fh];
                ev[u] = exps[b][1][u * 2 + fh];
                emax = max(emax, max(exps[b][1][u * 2], exps[b][1][u * 2 + 1]));
            }
        }
        float ct[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)  // kept normal: -inf stays -inf, zero zero
            ct[u] = fminf(fmaxf(ldexpf(EXTRA ? scale : scale * kLog2e, eq + ek[u]), 1.17549435e-38f), 3.40282347e38f);
        if constexpr (EXTRA) {
            const float* bp = P.bias + (int64_t)h * (2 * P.radius + 1) + P.radius;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x = s[j][i] * ct[j * 2 + (i >> 3)];
                    if (P.cap > 0.f) x = P.cap * tanh_near(x / P.cap);
                    if (P.bias) x += bp[min(max(k0 + key_at(j, i) - p, -P.radius), P.radius)];
                    s[j][i] = x;
                }
        }
        if (edge) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!visible(k0 + key_at(j, i))) s[j][i] = -INFINITY;
        }
        float mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float mx = s[u >> 1][(u & 1) * 8];
#pragma unroll
            for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[u >> 1][(u & 1) * 8 + i]);
            mt = fmaxf(mt, EXTRA ? mx : mx * ct[u]);
        }
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float mnew = mt > m + (EXTRA ? kLazy / kLog2e : kLazy) ? mt : m;
        float alpha = 1.0f;
        if (mnew != m) alpha = __builtin_amdgcn_exp2f(EXTRA ? (m - mnew) * kLog2e : m - mnew);
        m = mnew;
        const float ref = m == -INFINITY ? 0.f : m;
        float ao = alpha;
        if (emax > E) {
            const int up = min(emax + 1, 126);  // a little ahead: the next tiles' are alike
            ao = E == kUnsetE ? 0.f : ldexpf(alpha, max(E - up, -300));
            E = up;
        }
        float total = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int by = 14 + (edge ? 0 : max(ev[u] - E, kFarE));
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = s[u >> 1][(u & 1) * 8 + i];
                if constexpr (EXTRA) x = __builtin_amdgcn_exp2f(fmaf(x - ref, kLog2e, (float)by));
                else x = __builtin_amdgcn_exp2f(fmaf(x, ct[u], (float)by - ref));
                s[u >> 1][(u & 1) * 8 + i] = x;
                part += x;
            }
            total += ldexpf(part, -by);
        }
        sum = fmaf(sum, alpha, total);
        if (edge) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i)  // an unseen key's weight is zero, its exponent may be above E
                    s[u >> 1][(u & 1) * 8 + i] = ldexpf(s[u >> 1][(u & 1) * 8 + i],
                                                        min(max(key_exps[b][1][u * 16 + fh * 8 + i] - E, kFarE), 0));
        }
        if (__ballot(ao != 1.0f)) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= ao;
        }
    };
    auto values = [&](const u16* vd) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            h8 ph, pl;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                h2 hi, lo;
                split_pair(s[ks >> 1][(ks & 1) * 8 + e], s[ks >> 1][(ks & 1) * 8 + e + 1], hi, lo);
                ph[e] = hi[0], ph[e + 1] = hi[1];
                pl[e] = lo[0], pl[e + 1] = lo[1];
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const int row = dt * 32 + fr, at = row * kKT + (((ks * 2 + fh) ^ swz_v(row)) << 3);
                const h8 vh = *(const h8*)(vd + at), vl = *(const h8*)(vd + PART + at);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph, o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl, o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph, o[dt], 0, 0, 0);
            }
        }
    };

    int bad_first = nt, bad_last = -1;  // the tiles that hold values that are not finite
    if (n0 < nt) {
        fetch(n0);
        store(n0, n0 & 1);
    }
    for (int n = n0; n < nt; ++n) {
        const int b = n & 1, k0 = key_of(n);
        if (n + 1 < nt) fetch(n + 1);
        // tile n is in LDS, and nobody reads tile n - 1 any more
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (active && (k0 < pre || (k0 < last_hi && k0 + kKT > first_lo))) {
            scores(buf[b]);
            softmax(k0, b);
            values(buf[b] + 2 * PART);
        }
        int any = 0;
#pragma unroll
        for (int g = 0; g < 8; ++g) any |= bads[b][g];
        if (__builtin_amdgcn_readfirstlane(any)) {
            bad_first = min(bad_first, n);
            bad_last = n;
        }
        if (n + 1 < nt) store(n + 1, b ^ 1);
    }

    if (r >= rows) return;
    sum += __shfl_xor(sum, 32, 64);
    const int64_t cell = ((int64_t)(T.first + qi) * P.heads + h) * S.n + blockIdx.y;
    // a part of the keys: the sums as they are, on the scale of the reference
    const float inv = sum == 0.f ? 0.f : ldexpf(S.n > 1 ? 1.0f : 1.0f / sum, E - 14);
    for (int n = bad_first; n <= bad_last; ++n)
        for (int j = key_of(n), end = min(j + kKT, lk); j < end; ++j) {
            if (!visible(j)) continue;
            const float* vp = vbase + j * kv_inner;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {  // columns past d are not stored
                    const float x = vp[min(dt * 32 + (i >> 2) * 8 + fh * 4 + (i & 3), d - 1)];
                    if (abs_bits(x) >= kInfBits) o[dt][i] += x;
                }
        }
    if (S.n > 1) {
        if (fh == 0) S.ml[cell] = f2{m, sum};
        float* to = S.o + cell * S.stride;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = dt * 32 + g * 8 + fh * 4;
                if (c < d) *(f4*)(to + c) = f4{o[dt][g * 4] * inv, o[dt][g * 4 + 1] * inv, o[dt][g * 4 + 2] * inv, o[dt][g * 4 + 3] * inv};
            }
        return;
    }
    const int64_t at = (T.first + qi) * inner + (int64_t)h * d;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = dt * 32 + g * 8 + fh * 4;
            const f4 v = {o[dt][g * 4] * inv, o[dt][g * 4 + 1] * inv, o[dt][g * 4 + 2] * inv, o[dt][g * 4 + 3] * inv};
            if constexpr (VEC) {
                if (c >= d) continue;
                if constexpr (OUT16) *(uint2*)((u16*)P.out + at + c) = dev::bf16x4(v);
                else *(f4*)((float*)P.out + at + c) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < d) {
                        if constexpr (OUT16) ((u16*)P.out)[at + c + e] = dev::bf16_rne(v[e]);
                        else ((float*)P.out)[at + c + e] = v[e];
                    }
            }
        }
}

// ---------------------------------------------------------------------------
// Few rows a sequence (single tokens): fp32 on the vector ALUs, R rows of one
// key/value head a workgroup, each key and value read once for all of them.
//
// DP / 4 lanes have a key, four of its values each (whole rows of 64 or 128 values a load,
// 2 or 4 keys), a wave kLoads loads of keys and as many of values at once. Every group of
// lanes keeps a softmax of its own keys; they are put together at the end.
// ---------------------------------------------------------------------------
constexpr int kLoads = 8, kFewWaves = 4;

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {  // over aligned groups of 16 or 32
    v = dev::group_sum<16>(v);
    if constexpr (LANES == 32) {
        const unsigned b = __float_as_uint(v);
        const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);  // the two 16-lane rows side by side
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

template <int DP, int R, bool EXTRA>
__global__ __launch_bounds__(64 * kFewWaves) void k_attn_packed_few(Packed P, int out16, Parts S) {
    constexpr int LANES = DP / 4, KEYS = 64 / LANES, CHUNK = kLoads * KEYS, GROUPS = kFewWaves * KEYS;
    __shared__ float so[GROUPS][R][DP];
    __shared__ float sm[GROUPS][R], sl[GROUPS][R];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = lane / LANES, c4 = lane % LANES * 4, d = P.d;
    const int group = P.heads / P.kv_heads, kh = blockIdx.x % P.kv_heads;
    dev::SpanTile T;
    if (!dev::find_tile(P.spans, P.seqs, P.Tq, group, R, blockIdx.x / P.kv_heads, T)) return;
    dev::cut_span(T.z, T.w, P.Tk);
    const int lk = T.w, rows = T.rows * group, left = min(rows - T.row0, R), shift = lk - T.rows;
    const int pre = P.prefix ? min(max(P.prefix[T.index], 0), lk) : 0;
    const int64_t inner = (int64_t)P.heads * d, kv_inner = (int64_t)P.kv_heads * d;
    f4 q[R], o[R];
    float m[R], sum[R];
    int place[R], lo[R], hi[R], head[R];
    const float f = EXTRA ? P.scale : P.scale * kLog2e;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int rr = T.row0 + min(r, left - 1), qi = rr / group;
        head[r] = kh * group + rr - qi * group;
        place[r] = qi + shift;
        const Seen see = seen_from(P, place[r], lk, pre);
        lo[r] = see.lo, hi[r] = see.hi;
        const float* a = P.q + (T.first + qi) * inner + (int64_t)head[r] * d;
        q[r] = c4 < d ? *(const f4*)(a + c4) * f : f4{0.f, 0.f, 0.f, 0.f};
        o[r] = f4{0.f, 0.f, 0.f, 0.f};
        m[r] = -INFINITY, sum[r] = 0.f;
    }
    const int npre = (pre + CHUNK - 1) / CHUNK, next = max(npre, lo[0] / CHUNK);
    const int all = npre + (hi[R - 1] > lo[0] ? max(0, (hi[R - 1] + CHUNK - 1) / CHUNK - next) : 0);
    const int n0 = (int)((int64_t)all * blockIdx.y / S.n), n1 = (int)((int64_t)all * (blockIdx.y + 1) / S.n);
    const int64_t base = T.z * kv_inner + (int64_t)kh * d + (c4 < d ? c4 : 0);
    for (int n = n0 + w; n < n1; n += kFewWaves) {
        const int k0 = (n < npre ? n : next + n - npre) * CHUNK;
        f4 kx[kLoads], vx[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) kx[u] = *(const f4*)(P.k + base + min(k0 + u * KEYS + sub, lk - 1) * kv_inner);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) vx[u] = *(const f4*)(P.v + base + min(k0 + u * KEYS + sub, lk - 1) * kv_inner);
        const bool full = k0 + CHUNK <= pre || (k0 >= lo[R - 1] && k0 + CHUNK <= hi[0]);
        auto visible = [&](int u, int r) {
            const int j = k0 + u * KEYS + sub;
            return (j < pre) | ((j >= lo[r]) & (j < hi[r]));
        };
        float s[kLoads][R];
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r)
                s[u][r] = lanes_sum<LANES>(fmaf(q[r].x, kx[u].x, q[r].y * kx[u].y) + fmaf(q[r].z, kx[u].z, q[r].w * kx[u].w));
        if constexpr (EXTRA) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (P.cap > 0.f) s[u][r] = P.cap * tanh_near(s[u][r] / P.cap);
                    if (P.bias)
                        s[u][r] += P.bias[(int64_t)head[r] * (2 * P.radius + 1) + P.radius +
                                          min(max(k0 + u * KEYS + sub - place[r], -P.radius), P.radius)];
                }
        }
        if (!full) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (!visible(u, r)) s[u][r] = -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = s[0][r];
#pragma unroll
            for (int u = 1; u < kLoads; ++u) mx = fmaxf(mx, s[u][r]);
            const float mnew = fmaxf(m[r], mx), ref = mnew == -INFINITY ? 0.f : mnew;
            const float alpha = __builtin_amdgcn_exp2f(EXTRA ? (m[r] - ref) * kLog2e : m[r] - ref);
            m[r] = mnew;
            sum[r] *= alpha;
            o[r] *= alpha;
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
                s[u][r] = __builtin_amdgcn_exp2f(EXTRA ? (s[u][r] - ref) * kLog2e : s[u][r] - ref);
                sum[r] += s[u][r];
            }
        }
        if (full) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) o[r] += s[u][r] * vx[u];
        } else {
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (visible(u, r)) o[r] += s[u][r] * vx[u];  // 0 * inf is not zero
        }
    }
    const int g0 = w * KEYS + sub;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        *(f4*)&so[g0][r][c4] = o[r];
        if (c4 == 0) sm[g0][r] = m[r], sl[g0][r] = sum[r];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < left * LANES; i += 64 * kFewWaves) {
        const int r = i / LANES, c = i % LANES * 4;
        float top = sm[0][r];
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) top = fmaxf(top, sm[g][r]);
        const float ref = top == -INFINITY ? 0.f : top;
        f4 v = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const float x = __builtin_amdgcn_exp2f(EXTRA ? (sm[g][r] - ref) * kLog2e : sm[g][r] - ref);
            l = fmaf(x, sl[g][r], l);
            v += x * *(const f4*)&so[g][r][c];
        }
        if (c >= d) continue;
        const int rr = T.row0 + r, qi = rr / group, h = kh * group + rr - qi * group;
        const int64_t row = (int64_t)(T.first + qi) * P.heads + h;
        if (S.n > 1) {
            const int64_t cell = row * S.n + blockIdx.y;
            if (c == 0) S.ml[cell] = f2{top, l};
            *(f4*)(S.o + cell * S.stride + c) = v;
        } else {
            v *= l == 0.f ? 0.f : 1.0f / l;
            if (out16) *(uint2*)((u16*)P.out + row * d + c) = dev::bf16x4(v);
            else *(f4*)((float*)P.out + row * d + c) = v;
        }
    }
}

// out from the parts: a workgroup of eight 32-lane groups per (query row, head), each taking
// every eighth part. `unit`: log2(e) where the references are not in log2 units.
__global__ __launch_bounds__(256) void k_attn_packed_join(Packed P, int out16, Parts S, float unit) {
    __shared__ float so[8][128];
    __shared__ float sm[8], sl[8];
    const int t = blockIdx.x, h = blockIdx.y, c = (threadIdx.x & 31) * 4, g = threadIdx.x >> 5;
    if (dev::span_of_row(P.spans, P.seqs, t, P.Tq) < 0) return;
    const int64_t row = (int64_t)t * P.heads + h, cell = row * S.n;
    float top = -INFINITY, l = 0.f;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = g; s < S.n; s += 8) {
        const f2 ml = S.ml[cell + s];
        const float mnew = fmaxf(top, ml.x), ref = mnew == -INFINITY ? 0.f : mnew;
        const float keep = __builtin_amdgcn_exp2f((top - ref) * unit), add = __builtin_amdgcn_exp2f((ml.x - ref) * unit);
        l = l * keep + ml.y * add;
        if (c < P.d) v = v * keep + *(const f4*)(S.o + (cell + s) * S.stride + c) * add;
        top = mnew;
    }
    *(f4*)&so[g][c] = v;
    if (c == 0) sm[g] = top, sl[g] = l;
    __syncthreads();
    if (g || c >= P.d) return;
    top = sm[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, sm[i]);
    const float ref = top == -INFINITY ? 0.f : top;
    v = f4{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = __builtin_amdgcn_exp2f((sm[i] - ref) * unit);
        l = fmaf(x, sl[i], l);
        v += x * *(const f4*)&so[i][c];
    }
    v *= l == 0.f ? 0.f : 1.0f / l;
    const int64_t at = row * P.d + c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < P.d) {
            if (out16) ((u16*)P.out)[at + e] = dev::bf16_rne(v[e]);
            else ((float*)P.out)[at + e] = v[e];
        }
}

// The parts' memory, in scratch; the keys uncut where it cannot be had.
Parts make_parts(const Packed& P, int64_t n) {
    Parts S{(int)n, (P.d + 3) / 4 * 4, nullptr, nullptr};
    const size_t cells = (size_t)P.Tq * P.heads * n, ob = (cells * S.stride * 4 + 255) / 256 * 256;
    char* base = n > 1 ? (char*)try_scratch(ob + cells * sizeof(f2)) : nullptr;
    if (!base) S.n = 1;
    S.o = (float*)base;
    S.ml = base ? (f2*)(base + ob) : nullptr;
    return S;
}

void join_parts(const Packed& P, bool out16, const Parts& S, bool log2_units) {
    if (S.n > 1)
        k_attn_packed_join<<<dim3((unsigned)P.Tq, (unsigned)P.heads), 256, 0, stream()>>>(P, out16, S, log2_units ? 1.0f : kLog2e);
}

template <int DP>
void run_few(const Packed& P, bool out16, int64_t items, int rows) {
    const bool extra = P.cap > 0.f || P.bias;
    // Parts of the keys until there are eight workgroups a CU, each wave with two chunks of an average sequence.
    const int64_t wgs = items * P.kv_heads, keys = P.Tk / std::max(1, P.seqs);
    const Parts S = make_parts(P, std::max<int64_t>(1, std::min<int64_t>({8 * num_cus() / wgs, keys / (kFewWaves * 64), 256})));
    auto go = [&](auto r, auto ex) {
        k_attn_packed_few<DP, decltype(r)::value, decltype(ex)::value>
            <<<dim3((unsigned)wgs, (unsigned)S.n), 64 * kFewWaves, 0, stream()>>>(P, out16, S);
    };
    auto with = [&](auto ex) {
        using std::integral_constant;
        if (rows <= 1) go(integral_constant<int, 1>(), ex);
        else if (rows <= 4) go(integral_constant<int, 4>(), ex);
        else go(integral_constant<int, 8>(), ex);
    };
    if (extra) with(std::true_type());
    else with(std::false_type());
    join_parts(P, out16, S, !extra);
}

template <int DP>
void run_tiles(const Packed& P, bool out16, int64_t items) {
    const bool vec = P.d % 8 == 0 && aligned16(P.q) && aligned16(P.k) && aligned16(P.v) && (out16 ? ((uintptr_t)P.out & 7) == 0 : aligned16(P.out));
    const bool extra = P.cap > 0.f || P.bias;
    using T_ = std::true_type;
    using F_ = std::false_type;
    // Parts of the keys while the workgroups do not fill the chip, of eight tiles of an average sequence at least.
    const int64_t wgs = items * P.kv_heads, keys = P.Tk / std::max(1, P.seqs);
    const Parts S = make_parts(P, std::max<int64_t>(1, std::min<int64_t>(num_cus() / wgs, keys / (8 * kKT))));
    auto go = [&](auto o16, auto ex, auto ve) {
        k_attn_packed_tiles<DP, decltype(o16)::value, decltype(ex)::value, decltype(ve)::value>
            <<<dim3((unsigned)wgs, (unsigned)S.n), kThreads, 0, stream()>>>(P, (int)items, S);
    };
    auto with = [&](auto o16) {
        if (extra) vec ? go(o16, T_(), T_()) : go(o16, T_(), F_());
        else vec ? go(o16, F_(), T_()) : go(o16, F_(), F_());
    };
    if (out16) with(T_());
    else with(F_());
    join_parts(P, out16, S, !extra);
}

void run_attention_packed(const float* q, const float* k, const float* v, void* out, bool out16, int64_t Tq, int64_t Tk, int heads,
                          int kv_heads, int64_t d, const int32_t* spans, int64_t seqs, float scale, bool causal, int64_t window,
                          const int32_t* prefix, float cap, const float* bias, int64_t radius) {
    const char* op = "sdh_attention_packed";
    constexpr int64_t kMost = int64_t(1) << 30;
    if (kv_heads <= 0) kv_heads = heads;
    need(Tq >= 0 && Tk >= 0 && seqs >= 0 && window >= 0 && radius >= 0, op, "negative size");
    need(heads > 0 && d > 0, op, "heads and d must be positive");
    need(heads % kv_heads == 0, op, "heads mismatch");
    need(d <= kMaxD, op, "head dimension above 1024");
    need(heads <= 65535, op, "too many heads for one launch");
    need(Tq < kMost && Tk < kMost && seqs < kMost && radius < kMost, op, "a size of 2^30 or more");
    need(std::isfinite(scale) && std::isfinite(cap) && cap >= 0.f, op, "scale and cap must be finite, cap not negative");
    if (Tq == 0 || seqs == 0) return;
    ensure_init();
    const size_t qb = (size_t)(Tq * heads * d) * 4, ob = out16 ? qb / 2 : qb, kb = (size_t)(Tk * kv_heads * d) * 4;
    const size_t sb = (size_t)seqs * 16, pb = (size_t)seqs * 4, bb = (size_t)heads * (2 * radius + 1) * 4;
    check_range(q, qb, op, "q");
    check_range(out, ob, op, "out");
    check_range(spans, sb, op, "spans");
    need(aligned16(spans), op, "spans is not 16-byte aligned");
    if (Tk > 0) {
        check_range(k, kb, op, "k");
        check_range(v, kb, op, "v");
    }
    if (prefix) check_range(prefix, pb, op, "prefix");
    if (bias) check_range(bias, bb, op, "bias");
    need(!overlaps(out, ob, q, qb) && !(Tk > 0 && (overlaps(out, ob, k, kb) || overlaps(out, ob, v, kb))) && !overlaps(out, ob, spans, sb) &&
             !(prefix && overlaps(out, ob, prefix, pb)) && !(bias && overlaps(out, ob, bias, bb)),
         op, "out overlaps an input");
    Packed P{q,    k,   v,   out, (const int4*)spans, prefix, bias, (int)Tq, (int)Tk, (int)seqs, heads, kv_heads, (int)d, causal ? 1 : 0,
             window < kMost ? (int)window : 0,  // a wider one hides nothing
             bias ? (int)radius : 0, scale, cap};
    // A sequence's rows at one key/value head are few: see k_attn_packed_few.
    const int64_t group = heads / kv_heads, live = std::min(seqs, Tq), mean = (Tq + live - 1) / live * group;
    if (d <= 128 && d % 4 == 0 && mean <= 8 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out)) {
        const int r = mean <= 1 ? 1 : mean <= 4 ? 4 : 8;
        const int64_t n = Tq * group / r + live;
        if (Tq * group < kMost && n * kv_heads * 64 * kFewWaves <= kMaxGridItems) {
            if (d <= 64) run_few<64>(P, out16, n, r);
            else run_few<128>(P, out16, n, r);
            launched(op);
            return;
        }
    }
    const int64_t rows = Tq * group, items = rows / kTileRows + live;
    if (d <= 128 && rows < kMost && items * kv_heads * kThreads <= kMaxGridItems) {
        if (d <= 64) run_tiles<64>(P, out16, items);
        else run_tiles<128>(P, out16, items);
        launched(op);
        return;
    }
    const int64_t gx = (Tq + kRowWaves - 1) / kRowWaves;
    need(gx * 64 * kRowWaves <= kMaxGridItems, op, "too many queries for one launch");
    const dim3 grid((unsigned)gx, (unsigned)heads);
    if (out16) k_attn_packed_rows<true><<<grid, 64 * kRowWaves, 0, stream()>>>(P);
    else k_attn_packed_rows<false><<<grid, 64 * kRowWaves, 0, stream()>>>(P);
    launched(op);
}

}  // namespace
}  // namespace sdh

using namespace sdh;

extern "C" {

int sdh_attention_packed(const float* q, const float* k, const float* v, void* out, int out_bf16, int64_t Tq, int64_t Tk, int heads,
                         int kv_heads, int64_t d, const int32_t* spans, int64_t seqs, float scale, int causal, int64_t window,
                         const int32_t* prefix, float cap, const float* bias, int64_t radius) {
    return guarded([&] {
        run_attention_packed(q, k, v, out, out_bf16 != 0, Tq, Tk, heads, kv_heads, d, spans, seqs, scale, causal != 0, window, prefix, cap,
                             bias, radius);
    });
}

}  // extern "C"
