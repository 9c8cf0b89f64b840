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

// tanh to about 3e-7 of itself. Near zero 1 - e would cancel: x + x^3 p(x^2), p the polynomial
// of degree two whose largest error on [0, kTanhNear^2] is least (4e-8 of tanh x, found by weighted
// least squares; the Taylor series needs two terms more). `last`: a loop may hold it in a register.
constexpr float kTanhNear = 0.35f, kTanhLast = -0.0491593033f;
__device__ __forceinline__ float tanh_small(float x, float last = kTanhLast) {
    const float x2 = x * x;
    return fmaf(x * x2, fmaf(x2, fmaf(x2, last, 0.133000106f), -0.333326697f), x);
}
__device__ __forceinline__ float tanh_near(float x) {
    const float a = fabsf(x);
    const float e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * a);
    const float far = copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), x);
    return a < kTanhNear ? tanh_small(x) : far;
}

__device__ __forceinline__ int abs_bits(float x) { return (int)(__float_as_uint(x) & 0x7FFFFFFFu); }
constexpr int kInfBits = 0x7F800000;
__device__ __forceinline__ bool finite(float x) { return abs_bits(x) < kInfBits; }
__device__ __forceinline__ bool finite(const f4& x) { return finite(x.x) && finite(x.y) && finite(x.z) && finite(x.w); }
// A sum of weighted values at another reference: what is not finite stays so, however far the reference has risen.
__device__ __forceinline__ float scaled(float sum, float by) { return by == 0.f && !finite(sum) ? sum : sum * by; }
__device__ __forceinline__ f4 scaled(const f4& sum, float by) {
    return f4{scaled(sum.x, by), scaled(sum.y, by), scaled(sum.z, by), scaled(sum.w, by)};
}
// A bias of -inf hides its key, whatever the key holds.
__device__ __forceinline__ float biased(float x, float b) { return b == -INFINITY ? b : x + b; }

// ---------------------------------------------------------------------------
// Any head dimension: fp32 products, one wave per (query, head). Lanes take 64 keys at a
// time for the scores, then 64 columns at a time for the weighted sum. Takes heads of more
// than 128 dims, and calls whose tiles find no scratch.
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
                if (P.bias) x = biased(x, P.bias[(int64_t)h * (2 * P.radius + 1) + min(max(j - p, -P.radius), P.radius) + P.radius]);
            }
            const float mnew = fmaxf(m, dev::wave_max(x));
            const float ref = mnew == -INFINITY ? 0.f : mnew;  // nothing but -inf so far
            const float alpha = __builtin_amdgcn_exp2f((m - ref) * kLog2e);
            m = mnew;
            const float weight = __builtin_amdgcn_exp2f((x - ref) * kLog2e);
            sum = sum * alpha + dev::wave_sum(weight);
            __builtin_amdgcn_wave_barrier();
            sp[w][lane] = weight;
            const unsigned long long count = __ballot(x != -INFINITY);
            __builtin_amdgcn_wave_barrier();
            const int nk = min(64, to - k0);
#pragma unroll
            for (int i = 0; i < kAcc; ++i) {
                const int c = i * 64 + lane;
                if (i * 64 >= d) break;
                float a = acc[i] * alpha;
                if (c < d)
                    for (int u = 0; u < nk; ++u) a = fmaf(sp[w][u], P.v[kv0 + (k0 + u) * kv_inner + c], a);
                if (__ballot(!finite(a)) && c < d) {  // 0 * inf is neither zero nor inf: keys that do not count, weights that underflow
                    a = scaled(acc[i], alpha);
                    for (int u = 0; u < nk; ++u) {
                        if (!(count >> u & 1)) continue;
                        const float x = P.v[kv0 + (k0 + u) * kv_inner + c];
                        a = finite(x) ? fmaf(sp[w][u], x, a) : a + x;
                    }
                }
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
// Head dimensions up to 128 (padded to DP = 64 or 128), on the MFMA units, in two launches.
//
// k_attn_packed_split cuts k and v of a key/value head into tiles of 64 rows (of the
// tensor: a tile may hold rows of several sequences) in library scratch, as fp16 pairs in
// the order of the fragments' reads; a tile that no sequence reads is left out.
// k_attn_packed_tiles takes 32 rows a wave of one sequence and key/value head a workgroup,
// a row being a (query, head of the group) pair, heads fastest: the heads that share a
// key/value head share its tiles. It copies the tiles that any of its rows sees to LDS, and
// each of its waves takes 32 rows against them.
//
// Operands are fp16 pairs hi + lo in block floating point, products hi hi + hi lo +
// lo hi with fp32 sums (2^-21 of each product). A block is a row of q, or a tile of k or
// v: scaled by 2^-e to at most 2^14, a score is s 2^(e_q + e_k), and a weight is formed as
// p 2^(14 + e_v - E), so that the sums of all tiles share the scale 2^(14 - E). The pair
// holds 22 bits down to 2^-16 of its block's largest value.
//   E goes by the weighted values: the largest log2(p) + e_v of a row's tiles, p relative to
// the row's reference, with which E sinks as the reference rises. A value that is large but
// has no weight, hidden or far below in score, then costs the others nothing, and the largest
// that has weight is near 2^28 in its sum. A tile whose values are more than 2^kSpread apart, or
// that has rows of zeros among them, has an exponent for each key: p 2^e_v of the tile says
// nothing there about any one key. So it has for keys that far apart, whose largest need not be
// one that a row sees. Rows that no sequence reads are zeros that do not count.
//   Values that are not finite go into the tiles as zeros, since 0 * inf would reach the rows
// that do not see them, and are added at the end. An infinity in q or k would be inf - inf in a
// pair: a wave one of whose rows sees such a key, or has such a query, takes the tile's scores
// in fp32 (fp32_scores). So it does where values far below their block's largest, whose pairs
// are off by up to 2^-25, could move a score by more than 2^-21: by 2^-25 (sum|q| + sum|k|) of
// the scaled values in units of 2^(e_q + e_k) scale, and, where that says so, by how many such
// values there are against a largest of 2^14. Heads of 128 whose largest q and k meet at scores
// of 2^15 are far from that; a channel of q or k that is 2^12 above the others is not. Such
// tiles, and those with exponents of their keys, go through a second loop, one at a time.
//
// S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_32x32x16_f16: lane l holds row l % 32 of
// the wave in both, its statistics are its own. K's rows are ordered so that the eight
// scores of a lane's half of a 16-key step are eight neighbouring keys: its weights
// are the second product's operand as they lie, V^T in the keys' own order.
//
// Long sequences are bound by the three products: two images of 4200 rows, 30 heads of 128,
// 1.45 ms, 369 TFLOP/s of 4 d a visible pair, near k_attention.hip's kernel on that shape; the split 0.1
// ms of it. Short ones by their workgroups' starts (the list, q): 24 prompts of up to 203
// rows, 32/8 heads of 128, 63 us, 16 of them their bytes at the rate of a copy. The rules for
// unlike and infinite values cost 1 % of the former and 2 to 3 % of the latter.
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

constexpr int kKT = 64, kSplitWaves = 4;
// The reference m of the weights is raised when a tile's largest score passes it by more
// than this (in units of log2): weights stay below 2^(14 + kLazy), inside fp16.
constexpr float kLazy = 1.5f;
constexpr float kFarRef = 1e4f;  // rounded by less than 2^-10
// The bias of a head in LDS goes on at both ends with its end values, as far as a wave's 32 rows and a
// tile's 64 keys reach past the radius unless all of them are beyond it: no index is held to the radius
// (ten instructions a score; the rows and tiles at the band's edges took half the softmax' time).
constexpr int kBiasPad = 96;
constexpr float kMostLost = 16.0f;  // 2^25 times 2^-21
constexpr int kInfinite = 1 << 16;  // values that are not finite, in a count of others
constexpr int kBadKey = 1000;   // the exponent of a key that is not finite
constexpr int kUnsetE = -2000;  // no weighted values yet, or next to nothing beside the reference
constexpr int kSpread = 8;
// A tile's weights are scaled by no less than this, which keeps their sum in range. At that scale they are below 2^(14 + kLazy - 42),
// less than half of fp16's least: the pairs are zero, as they are to be, since the tile's values are below 2^-42 of the largest.
constexpr int kFarE = -42;

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
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
// The larger of each half over the wave's lanes.
__device__ __forceinline__ unsigned wave_max_halves(unsigned v) {
    auto larger = [](unsigned a, unsigned b) {
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
    };
    v = larger(v, dpp_i<0xB1>(v));
    v = larger(v, dpp_i<0x4E>(v));
    v = larger(v, dpp_i<0x141>(v));
    v = larger(v, dpp_i<0x140>(v));
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = larger(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return larger(b[0], b[1]);
}
// The exponent that brings a block's largest magnitude into [2^13, 2^14); zero and
// subnormal blocks the least there is.
__device__ __forceinline__ int block_exp(int bits) { return min(max((bits >> 23) - 140, -126), 126); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }  // e in [-126, 127]

// A tile's exponents of k and v, and what is special about it.
enum { kKeyExps = 1, kValueExps = 2, kNotFinite = 4 };
struct Tiles {
    u16* data;   // [kv_heads, n, 4 * 64 DP]: K hi, K lo, V^T hi, V^T lo
    int4* info;  // [kv_heads, n]: e_k, e_v, flags, the largest sum of a scaled key's magnitudes (a float)
    int* exps;   // [kv_heads, n, 2, 64]: of the keys, where the flags say so
    int n;
};

template <int DP, bool VEC>
__global__ __launch_bounds__(64 * kSplitWaves) void k_attn_packed_split(Packed P, Tiles X) {
    constexpr int PART = kKT * DP, KCH = DP / 8, KROWS = 64 / KCH, KU = 16 / KROWS;  // 16-byte chunks of a K row, rows of a wave's load, loads
    constexpr int VU = DP / 64;                                                     // columns of v a lane has
    __shared__ __attribute__((aligned(16))) u16 vt[2 * PART];
    __shared__ int tops[2][kSplitWaves], flags[kSplitWaves];
    __shared__ float sums[kSplitWaves];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x, kh = blockIdx.y, j0 = tile * kKT + w * 16, d = P.d;
    const int64_t kv_inner = (int64_t)P.kv_heads * d;
    const int kch = lane & (KCH - 1), krow = lane / KCH;
    // sixteen keys a wave; k: 16-byte chunks of their rows, v: the lane's columns of all of them
    float kx[KU][8], vx[16][VU];
#pragma unroll
    for (int u = 0; u < KU; ++u) {
        const float* a = P.k + min(j0 + u * KROWS + krow, P.Tk - 1) * kv_inner + (int64_t)kh * d;
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
    for (int i = 0; i < 16; ++i) {
        const float* a = P.v + min(j0 + i, P.Tk - 1) * kv_inner + (int64_t)kh * d;
        if constexpr (VEC && VU == 2) {
            const f2 x = *(const f2*)(a + min(lane * 2, d - 2));
            vx[i][0] = x.x, vx[i][1] = x.y;
        } else {
#pragma unroll
            for (int u = 0; u < VU; ++u) vx[i][u] = a[min(lane * VU + u, d - 1)];
        }
    }
    // The tile's rows that sequences read. What the others hold does not matter, and is not to cost them anything: behind the
    // sequences in their slots a cache may have zeros, or anything.
    unsigned long long used = 0;
    for (int s0 = 0; s0 < P.seqs && ~used; s0 += 64) {
        int4 e = make_int4(0, 0, 0, 0);
        if (s0 + lane < P.seqs) {
            e = P.spans[s0 + lane];
            dev::cut_span(e.z, e.w, P.Tk);
        }
        const int from = max(e.z - tile * kKT, 0), to = min(e.z + e.w - tile * kKT, kKT);
        for (unsigned long long m = __ballot(e.y > 0 && from < to); m && ~used; m &= m - 1) {
            const int at = (int)__ffsll(m) - 1, lo = __builtin_amdgcn_readlane(from, at), hi = __builtin_amdgcn_readlane(to, at);
            used |= ~0ull >> (kKT - (hi - lo)) << lo;
        }
    }
    if (!used) return;
    const unsigned mine = (unsigned)(used >> (w * 16)) & 0xFFFFu;
    // a key's largest magnitudes, rows of no sequence and columns past d zero, and what is not finite
    int ktop[KU], vtop[16], kmost = 0, vmost = 0, flag = 0;
#pragma unroll
    for (int u = 0; u < KU; ++u) {
        ktop[u] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!(mine >> (u * KROWS + krow) & 1) || kch * 8 + e >= d) kx[u][e] = 0.f;
            ktop[u] = max(ktop[u], abs_bits(kx[u][e]));
        }
        ktop[u] = group_imax<KCH>(ktop[u]);
        if (ktop[u] < kInfBits) kmost = max(kmost, ktop[u]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        vtop[i] = 0;
#pragma unroll
        for (int u = 0; u < VU; ++u) {
            if (!(mine >> i & 1) || lane * VU + u >= d) vx[i][u] = 0.f;
            if (abs_bits(vx[i][u]) >= kInfBits) vx[i][u] = 0.f, flag = kNotFinite;
            vtop[i] = max(vtop[i], abs_bits(vx[i][u]));
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {  // the upper halves order as the values do
        const unsigned both = wave_max_halves(((unsigned)vtop[i] >> 16) | ((unsigned)vtop[i + 1] & 0xFFFF0000u));
        vtop[i] = (int)(both << 16);
        vtop[i + 1] = (int)(both & 0xFFFF0000u);
        vmost = max(vmost, max(vtop[i], vtop[i + 1]));
    }
    kmost = group_imax<64>(kmost);
    if (lane == 0) tops[0][w] = kmost, tops[1][w] = vmost;
    __syncthreads();
    kmost = max(max(tops[0][0], tops[0][1]), max(tops[0][2], tops[0][3]));
    vmost = max(max(tops[1][0], tops[1][1]), max(tops[1][2], tops[1][3]));
#pragma unroll
    for (int u = 0; u < KU; ++u)
        if (ktop[u] >= kInfBits || (ktop[u] && abs((kmost >> 23) - (ktop[u] >> 23)) > kSpread)) flag |= kKeyExps;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if ((mine >> i & 1) && (vmost >> 23) - (vtop[i] >> 23) > kSpread) flag |= kValueExps;
    flag = (__ballot(flag & kKeyExps) ? kKeyExps : 0) | (__ballot(flag & kValueExps) ? kValueExps : 0) | (__ballot(flag & kNotFinite) ? kNotFinite : 0);
    if (lane == 0) flags[w] = flag;
    __syncthreads();
    flag = flags[0] | flags[1] | flags[2] | flags[3];
    const int ek = block_exp(kmost), ev = block_exp(vmost);
    const int64_t at = (int64_t)kh * X.n + tile;
    int* exps = X.exps + at * 2 * kKT;
    u16 *kd = X.data + at * 4 * PART, *vd = kd + 2 * PART;
    float ksum = 0.f;
#pragma unroll
    for (int u = 0; u < KU; ++u) {
        const int key = w * 16 + u * KROWS + krow, e = flag & kKeyExps ? block_exp(ktop[u]) : ek;
        if ((flag & kKeyExps) && kch == 0) exps[key] = ktop[u] >= kInfBits ? kBadKey : e;
        const float sc = pow2(-e);
        h8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; ++i) kx[u][i] *= sc;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += fabsf(kx[u][i]);
        sum = dev::group_sum<KCH>(sum);
        if (ktop[u] < kInfBits) ksum = fmaxf(ksum, sum);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            h2 a, c;
            split_pair(kx[u][i], kx[u][i + 1], a, c);
            hi[i] = a[0], hi[i + 1] = a[1];
            lo[i] = c[0], lo[i + 1] = c[1];
        }
        const int row = row_of_key(key), to = row * DP + ((kch ^ swz_k<DP>(row)) << 3);
        *(h8*)(kd + to) = hi;
        *(h8*)(kd + PART + to) = lo;
    }
    float vs[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int e = flag & kValueExps ? block_exp(vtop[i]) : ev;
        if ((flag & kValueExps) && lane == 0) exps[kKT + w * 16 + i] = e;
        vs[i] = pow2(-e);
    }
#pragma unroll
    for (int u = 0; u < VU; ++u)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            h8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                h2 a, c;
                split_pair(vx[b * 8 + i][u] * vs[b * 8 + i], vx[b * 8 + i + 1][u] * vs[b * 8 + i + 1], a, c);
                hi[i] = a[0], hi[i + 1] = a[1];
                lo[i] = c[0], lo[i + 1] = c[1];
            }
            const int row = lane * VU + u, to = row * kKT + (((w * 2 + b) ^ swz_v(row)) << 3);
            *(h8*)(vt + to) = hi;
            *(h8*)(vt + PART + to) = lo;
        }
    ksum = dev::wave_max(ksum);
    if (lane == 0) sums[w] = ksum;
    __syncthreads();  // whole lines of V^T, of which a wave has a quarter
    if (threadIdx.x == 0) X.info[at] = make_int4(ek, ev, flag, (int)__float_as_uint(fmaxf(fmaxf(sums[0], sums[1]), fmaxf(sums[2], sums[3]))));
#pragma unroll
    for (int i = 0; i < 2 * PART / (8 * 64 * kSplitWaves); ++i) {
        const int to = (i * 64 * kSplitWaves + threadIdx.x) * 8;
        *(h8*)(vd + to) = *(const h8*)(vt + to);
    }
}

// Eight waves a workgroup, one workgroup a CU; for DP = 64, whose tiles are half the size and
// whose sequences are mostly shorter, four and two.
template <int DP>
constexpr int kWaves = DP == 128 ? 8 : 4;

// table: the values of bias that the group's heads have, kept in LDS; 0 where they are read from memory.
template <int DP, bool EXTRA, bool VEC>
__global__ __launch_bounds__(64 * kWaves<DP>, 2 / (kWaves<DP> / 4)) void k_attn_packed_tiles(Packed P, Tiles X, int out16, int items, int table,
                                                                                          Parts S) {
    constexpr int WAVES = kWaves<DP>, kThreads = 64 * WAVES, kTileRows = 32 * WAVES;
    constexpr int DS = DP / 16, DT = DP / 32, PART = kKT * DP;
    // Rows of K, hi and lo, of two tiles, and of V^T. Objects of their own, so that the compiler
    // knows which copy a read has to wait for.
    __shared__ __attribute__((aligned(1024))) u16 kbuf0[2 * PART], kbuf1[2 * PART], vbuf0[2 * PART], vbuf1[2 * PART];
    __shared__ f2 q_waves[WAVES];
    extern __shared__ float biases[];
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
    // A sequence's last rows, which see most keys, come first: the short ones fill the end. Measured, us,
    // first / last rows first, 32/8 heads of 128, causal: one sequence of 2048 to 4096 231 / 198, four of
    // 500 to 1000 125 / 118, eight of 250 to 500 77 / 79.
    if (P.causal) T.row0 = (T.rows * group - 1) / kTileRows * kTileRows - T.row0;
    const int d = P.d, rows = T.rows * group, lk = T.w, pre = P.prefix ? min(max(P.prefix[T.index], 0), lk) : 0;
    const int64_t inner = (int64_t)P.heads * d;
    const int r = T.row0 + w * 32 + fr;
    const int rc = min(r, rows - 1), qi = rc / group, h = kh * group + (rc - qi * group);
    const int shift = lk - T.rows;
    const int p = qi + shift;
    const Seen see = seen_from(P, p, lk, pre);
    const int wg_lo = seen_from(P, T.row0 / group + shift, lk, pre).lo,
              wg_hi = seen_from(P, (min(T.row0 + kTileRows, rows) - 1) / group + shift, lk, pre).hi;
    const bool active = T.row0 + w * 32 < rows;
    const int first_lo = __builtin_amdgcn_readlane(see.lo, 0), last_lo = __builtin_amdgcn_readlane(see.lo, 31);
    const int first_p = __builtin_amdgcn_readlane(p, 0), last_p = __builtin_amdgcn_readlane(p, 31);
    const int first_hi = __builtin_amdgcn_readlane(see.hi, 0), last_hi = __builtin_amdgcn_readlane(see.hi, 31);
    // The tensor's tiles with a key of the prefix, then those with a key of the intervals; this part's share of them.
    const int t0 = T.z / kKT, npre = pre ? (T.z + pre + kKT - 1) / kKT - t0 : 0;
    const int next = max(t0 + npre, (T.z + wg_lo) / kKT);
    const int all = npre + (wg_hi > wg_lo ? max(0, (T.z + wg_hi + kKT - 1) / kKT - next) : 0);
    const int n0 = (int)((int64_t)all * blockIdx.y / S.n), nt = (int)((int64_t)all * (blockIdx.y + 1) / S.n);
    auto tile_of = [&](int n) { return n < npre ? t0 + n : next + n - npre; };
    const u16* data = X.data + (int64_t)kh * X.n * 4 * PART;
    const int4* info = X.info + (int64_t)kh * X.n;
    auto copy = [&](int tile, int part, u16* to) __attribute__((always_inline)) {
        // Buffer loads, not global_load_lds: the compiler counts a FLAT-encoded copy into LDS as
        // pending on the LDS counter too, and then waits for every LDS read in full.
        const __amdgpu_buffer_rsrc_t rsrc =
            __builtin_amdgcn_make_buffer_rsrc((void*)(data + (int64_t)tile * 4 * PART + part * 2 * PART), (short)0, 4 * PART, 0x00020000);
#pragma unroll
        for (int i = 0; i < 4 * PART / (kThreads * 16); ++i) {
            const int chunk = (i * WAVES + w) * 64;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(to + chunk * 8), 16, lane * 16, chunk * 16, 0,
                                                     0);
        }
    };
    if (n0 < nt) {
        copy(tile_of(n0), 0, kbuf0);
        copy(tile_of(n0), 1, vbuf0);
    }
    const int row_of_bias = 2 * P.radius + 1 + 2 * kBiasPad;
    if (EXTRA && table)  // [group, row_of_bias]
        for (int i = threadIdx.x; i < table; i += kThreads) {
            const int hh = i / row_of_bias, c = min(max(i - hh * row_of_bias - kBiasPad, 0), 2 * P.radius);
            biases[i] = P.bias[(int64_t)(kh * group + hh) * (2 * P.radius + 1) + c];
        }

    // Q: the B operand of S^T, row qi of head h, dims ds*16 + fh*8 .. +7. Whole rows
    // come in 64 dims at a time and are dealt out through a share of the LDS that no tile is in
    // yet, the 16-byte piece c of row i at c ^ (i & 15).
    const float* qp = P.q + (int64_t)(T.first + qi) * inner + (int64_t)h * d;
    float qx[DS][8];
    if constexpr (VEC) {
        char* mine = (char*)(w < WAVES / 2 ? kbuf1 : vbuf1) + (w % (WAVES / 2)) * (32 * 256);
        static_assert(WAVES / 2 * 32 * 256 <= 4 * PART, "Q's rows in LDS");
#pragma unroll
        for (int half = 0; half < DP / 64; ++half) {
            f4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // four rows a load
                const int row = i * 4 + (lane >> 4), rr = min(T.row0 + w * 32 + row, rows - 1), qr = rr / group;
                const float* from = P.q + (int64_t)(T.first + qr) * inner + (int64_t)(kh * group + rr - qr * group) * d;
                x[i] = *(const f4*)(from + min(half * 64 + (lane & 15) * 4, d - 4));
            }
            __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses keep their order
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = i * 4 + (lane >> 4);
                *(f4*)(mine + row * 256 + (((lane & 15) ^ (row & 15)) << 4)) = x[i];
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int ds = half * 4 + k;
                const f4 u = *(const f4*)(mine + fr * 256 + (((k * 4 + fh * 2) ^ (fr & 15)) << 4)),
                         v = *(const f4*)(mine + fr * 256 + (((k * 4 + fh * 2 + 1) ^ (fr & 15)) << 4));
#pragma unroll
                for (int e = 0; e < 8; ++e) qx[ds][e] = ds * 16 + fh * 8 < d ? (e < 4 ? u[e & 3] : v[e & 3]) : 0.f;
            }
        }
    } else {
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int e = 0; e < 8; ++e) qx[ds][e] = ds * 16 + fh * 8 + e < d ? qp[ds * 16 + fh * 8 + e] : 0.f;
    }
    h8 qh[DS], ql[DS];
    int eq;
    {
        int top = 0;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(qx[ds][e]));
        top = max(top, __shfl_xor(top, 32, 64));
        eq = block_exp(top);
        const float sc = copysignf(pow2(-eq), P.scale);  // a negative scale turns q's sign
        float all = 0.f;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                h2 hi, lo;
                const float x = qx[ds][e] * sc, y = qx[ds][e + 1] * sc;
                all += fabsf(x) + fabsf(y);
                split_pair(x, y, hi, lo);
                qh[ds][e] = hi[0], qh[ds][e + 1] = hi[1];
                ql[ds][e] = lo[0], ql[ds][e + 1] = lo[1];
            }
        // of the wave's rows: the largest block, and the largest sum of magnitudes
        all += __shfl_xor(all, 32, 64);
        const float block = pow2(eq), most = dev::wave_max(block), sum = dev::wave_max(all < INFINITY ? block * all : INFINITY);
        if (lane == 0) q_waves[w] = f2{most, sum};
    }
    const float scale = EXTRA ? fabsf(P.scale) : fabsf(P.scale) * kLog2e;

    f32x16 o[DT];     // O^T
    f32x16 s[2];      // S^T of the newest tile: s[i / 16][i % 16] of the lane is the tile's key (i/8)*16 + fh*8 + i%8
    h8 ph[4], pl[4];  // its weights
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float m = -INFINITY, sum = 0.f;  // the reference (log2 units without EXTRA), this lane's keys' sum of weights
    int E = kUnsetE;

    auto scores = [&](const u16* kbuf) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[j][i] = 0.f;
        int row0 = fr;
        asm volatile("" : "+v"(row0));  // the addresses are formed here, not kept in registers through the loop
        h8 kf[2][2][2];  // [step % 2][half][hi, lo]: a step's fragments are read ahead of the MFMAs before it
        auto fetch = [&](int ds) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = j * 32 + row0, at = row * DP + (((ds * 2 + fh) ^ swz_k<DP>(row)) << 3);
                kf[ds & 1][j][0] = *(const h8*)(kbuf + at);
                kf[ds & 1][j][1] = *(const h8*)(kbuf + PART + at);
            }
        };
        fetch(0);
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            if (ds + 1 < DS) fetch(ds + 1);
            __builtin_amdgcn_sched_barrier(0);
            const int b = ds & 1;
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[b][j][0], qh[ds], s[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[b][j][0], ql[ds], s[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[b][j][1], qh[ds], s[j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto visible = [&](int j) { return ((unsigned)j < (unsigned)pre) | ((unsigned)(j - see.lo) < (unsigned)(see.hi - see.lo)); };
    // Keeps the compiler from working on all 32 scores at once, for which there are no registers.
    auto few = [](int i) __attribute__((always_inline)) {
        if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
    };
    // P for code that hardly ever runs, read from the kernel's arguments there: kept in registers it would push others out.
    auto args = []() __attribute__((always_inline)) {
        auto R = (const __attribute__((address_space(4))) Packed*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(R));
        return R;
    };
    auto hidden = [&](auto R, int j) {  // by a bias of -inf
        return EXTRA && R->bias && R->bias[(int64_t)h * (2 * R->radius + 1) + R->radius + min(max(j - p, -R->radius), R->radius)] == -INFINITY;
    };
    // s = scale q.k of a tile, whatever q and k hold, -inf where a bias hides the key. Eight keys at a time, in
    // little code and few registers.
    auto fp32_scores = [&](int k0) __attribute__((always_inline)) {
        const auto R = args();
        const int d = R->d;
        const int64_t kv_inner = (int64_t)R->kv_heads * d;
        const float *qr = R->q + ((int64_t)(T.first + qi) * R->heads + h) * d, *kr = R->k + T.z * kv_inner + (int64_t)kh * d;
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
            const int j = k0 + u * 16 + fh * 8;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
#pragma unroll 1
            for (int c = 0; c < d; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = fmaf(qr[c], kr[min(max(j + i, 0), lk - 1) * kv_inner + c], x[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = hidden(R, j + i) ? -INFINITY : x[i] * R->scale;
#pragma unroll
                for (int to = 0; to < 4; ++to)
                    if (u == to) s[to >> 1][(to & 1) * 8 + i] = x[i];
            }
        }
    };
    // How many values of a row of q, and of a key of the tile in kbuf, at most have pairs of fewer than 22 bits, down to none; a
    // query that is not finite counts kInfinite. For tiles that may lose some by their sums of magnitudes.
    auto few_bits = [&](const u16* kbuf) __attribute__((always_inline)) {
        auto lost = [](unsigned hi) {  // of two values
            const unsigned a = hi & 0x7FFFu, b = hi >> 16 & 0x7FFFu;
            return (int)(a < 0x3000u) + (int)(b < 0x3000u) + ((a >= 0x7C00u) + (b >= 0x7C00u)) * kInfinite;
        };
        auto of_row = [&](int n) { return n == DP ? 0 : n - (DP - P.d); };  // rows of zeros lose nothing, nor do the columns past d
        int nq = 0, nk = 0;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int e = 0; e < 8; e += 2) nq += lost(__builtin_bit_cast(unsigned, h2{qh[ds][e], qh[ds][e + 1]}));
#pragma unroll 1
        for (int i = 0; i < DP / 2; ++i)  // a key a lane, from a bank each
            nk += lost(((const unsigned*)kbuf)[lane * (DP / 2) + ((i + lane) & (DP / 2 - 1))]) % kInfinite;
        return group_imax<64>(of_row(nq + __shfl_xor(nq, 32, 64))) + group_imax<64>(of_row(nk));
    };
    f2 q_most = {0.f, 0.f};  // of the workgroup's rows, as q_waves
    auto loses = [&](int ek, float ksum) { return !(ldexpf(scale * fmaf(q_most[0], ksum, q_most[1]), ek) <= kMostLost); };
    // s -> weights in place, the statistics and the scale of o brought up to date. k0: the
    // sequence's key at the tile's first row (below zero in front of the sequence). `odd`: what the
    // first loop leaves to the second.
    auto softmax = [&](auto odd, int k0, int tile, int tile_ek, int tile_ev, int flag, float ksum) __attribute__((always_inline)) {
        constexpr bool ODD = decltype(odd)::value;
        const int* exps = X.exps + ((int64_t)kh * X.n + tile) * 2 * kKT;
        const bool edge = !((k0 >= 0 && k0 + kKT <= pre) || (k0 >= last_lo && k0 + kKT <= first_hi));  // of this wave
        int ek = tile_ek;
        if (ODD && (flag & kKeyExps)) {
            ek = -126;
#pragma unroll 1
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = exps[u * 16 + fh * 8 + i];
                    ek = max(ek, visible(k0 + u * 16 + fh * 8 + i) ? e : -126);
                }
            ek = max(ek, __shfl_xor(ek, 32, 64));
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i)  // an unseen key's may be larger
                    s[u >> 1][(u & 1) * 8 + i] = ldexpf(s[u >> 1][(u & 1) * 8 + i], min(exps[u * 16 + fh * 8 + i] - ek, 0));
        }
        // kept normal: -inf stays -inf, zero zero
        float unit = fminf(fmaxf(ldexpf(scale, eq + ek), 1.17549435e-38f), 3.40282347e38f);  // of s
        if (ODD && __ballot(ek == kBadKey || loses(ek, ksum))) {
            const int n = few_bits(kbuf0);
            if (n >= kInfinite || __ballot(ek == kBadKey || !(unit * (float)n <= kMostLost * 0x1p-14f))) {
                fp32_scores(k0);
                unit = EXTRA ? 1.0f : kLog2e;
            }
        }
        if constexpr (EXTRA) {
            const float* near = biases + (h - kh * group) * row_of_bias + kBiasPad + P.radius;
            const float* bp = P.bias + (int64_t)h * (2 * P.radius + 1) + P.radius;
            if (P.cap > 0.f) {
                const float in = fminf(unit / P.cap, 3.40282347e38f);
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    s[i >> 4][i & 15] *= in;
                    top = fmaxf(top, fabsf(s[i >> 4][i & 15]));
                }
                unit = P.cap;
                // Scores well inside the cap, as most are, take the polynomial alone (half the
                // instructions, no exponential).
                const bool small = !__ballot(!(top < kTanhNear));
                if (small) {
                    float last = kTanhLast;
                    asm volatile("" : "+v"(last));
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        s[i >> 4][i & 15] = tanh_small(s[i >> 4][i & 15], last);
                        few(i);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float y = s[i >> 4][i & 15];
                        asm volatile("" : "+v"(y));  // the polynomials are not to be formed in front of the branch
                        s[i >> 4][i & 15] = tanh_near(y);
                        few(i);
                    }
                }
            }
            if (P.bias) {
                const int from = k0 - last_p, to = k0 + kKT - 1 - first_p;  // the wave's distances
                const int at = k0 + fh * 8 - p;
                if (to <= -P.radius || from >= P.radius) {  // one value for all
                    const int c = from >= P.radius ? P.radius : -P.radius;
                    float v;
                    if (table) {
                        v = near[c];
                        asm volatile("" : "+v"(v));  // not one load by a chosen address: it would wait for the copies
                    } else {
                        v = bp[c];
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) s[i >> 4][i & 15] = fmaf(s[i >> 4][i & 15], unit, v);
                } else if (table) {  // beyond the radius by less than kBiasPad
                    const float* b = near + at;
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            s[u >> 1][(u & 1) * 8 + i] = fmaf(s[u >> 1][(u & 1) * 8 + i], unit, b[u * 16 + i]);
                            few(i);
                        }
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            s[u >> 1][(u & 1) * 8 + i] = fmaf(s[u >> 1][(u & 1) * 8 + i], unit, bp[min(max(at + u * 16 + i, -P.radius), P.radius)]);
                            few(i);
                        }
                }
                unit = 1.0f;
            }
        }
        if (edge && (k0 >= pre || !pre)) {
            const int c = k0 + fh * 8 - see.lo;
            const unsigned n = see.hi - see.lo;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if ((unsigned)(c + u * 16 + i) >= n) s[u >> 1][(u & 1) * 8 + i] = -INFINITY;
                    few(i);
                }
        } else if (edge) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (!visible(k0 + u * 16 + fh * 8 + i)) s[u >> 1][(u & 1) * 8 + i] = -INFINITY;
                    few(i);
                }
        }
        float mt = s[0][0];
#pragma unroll
        for (int i = 0; i < 32; ++i) mt = fmaxf(mt, s[i >> 4][i & 15]);
        mt *= unit;
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float mnew = mt > m + (EXTRA ? kLazy / kLog2e : kLazy) ? mt : m;
        float alpha = 1.0f, ao = 1.0f;  // of the sum of weights, of o
        if (mnew != m) {
            const float rise = EXTRA ? (mnew - m) * kLog2e : mnew - m;
            const float whole = fminf(floorf(rise), 1024.0f);  // taken off E, the rest off o
            ao = __builtin_amdgcn_exp2f(whole - rise);
            alpha = ldexpf(ao, -(int)whole);
            E = max(E - (int)whole, kUnsetE);
        }
        m = mnew;
        const float ref = m == -INFINITY ? 0.f : m;
        float f = EXTRA ? unit * kLog2e : unit, off = EXTRA ? ref * kLog2e : ref;
        float most, total = 0.f;  // log2 of the tile's largest weighted value, the sum of its weights
        const bool own = ODD && (flag & kValueExps);
        if (own) {  // s to log2 units above the reference, with the key's exponent
            most = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = fmaf(s[u >> 1][(u & 1) * 8 + i], unit, -ref) * (EXTRA ? kLog2e : 1.0f);
                    total += __builtin_amdgcn_exp2f(x);
                    s[u >> 1][(u & 1) * 8 + i] = x + (float)(exps[kKT + u * 16 + fh * 8 + i] - tile_ev);
                    most = fmaxf(most, s[u >> 1][(u & 1) * 8 + i]);
                    few(i);
                }
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            f = 1.0f, off = 0.f;
        } else {
            most = fminf(EXTRA ? (mt - ref) * kLog2e : mt - ref, 0.0f);
        }
        const int need = (int)fmaxf(ceilf(most), 2.0f * kUnsetE) + tile_ev;
        if (need > E) {
            ao = ldexpf(ao, max(E - need - 1, -300));
            E = need + 1;  // a little ahead: the next tiles' are alike
        }
        const int above = tile_ev - E, by = 14 + (own ? above : max(above, kFarE));
        float weights = 0.f;
        // A reference far out (biases of the type's lowest value, for one) is taken off before the product, which could overflow.
        // It was rounded, as the scores here are not: their weights are held to what the others may reach.
        if (!own && __ballot(!(fabsf(ref) < kFarRef))) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float x = fmaf(s[i >> 4][i & 15], unit, -ref) * (EXTRA ? kLog2e : 1.0f);
                s[i >> 4][i & 15] = __builtin_amdgcn_exp2f((x > kLazy ? kLazy : x) + (float)by);  // NaN stays
            }
        } else {
            const float up = (float)by - off;
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i >> 4][i & 15] = __builtin_amdgcn_exp2f(fmaf(s[i >> 4][i & 15], f, up));
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) weights += s[i >> 4][i & 15];
        asm volatile("" : "+v"(weights));  // not behind the branch below, for which they would be copied
        if (!own) total = ldexpf(weights, -by);
        sum = fmaf(sum, alpha, total);
        if (__ballot(ao != 1.0f)) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= ao;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                h2 hi, lo;
                split_pair(s[u >> 1][(u & 1) * 8 + i], s[u >> 1][(u & 1) * 8 + i + 1], hi, lo);
                ph[u][i] = hi[0], ph[u][i + 1] = hi[1];
                pl[u][i] = lo[0], pl[u][i + 1] = lo[1];
            }
    };
    // 2 DT steps of two (16 keys, 32 columns), columns fastest; the two accumulators in turn.
    auto values = [&](const u16* vbuf) __attribute__((always_inline)) {
        int row0 = fr;
        asm volatile("" : "+v"(row0));
        h8 vf[2][2][2];  // [step % 2][of the two][hi, lo]
        auto fetch = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int ks = (i * 2 + u) / DT, row = (i * 2 + u) % DT * 32 + row0, at = row * kKT + (((ks * 2 + fh) ^ swz_v(row)) << 3);
                vf[i & 1][u][0] = *(const h8*)(vbuf + at);
                vf[i & 1][u][1] = *(const h8*)(vbuf + PART + at);
            }
        };
        fetch(0);
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
            if (i + 1 < 2 * DT) fetch(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            const int b = i & 1, ks = i * 2 / DT, dt = i * 2 % DT;
#pragma unroll
            for (int u = 0; u < 2; ++u) o[dt + u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[b][u][0], ph[ks], o[dt + u], 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) o[dt + u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[b][u][0], pl[ks], o[dt + u], 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) o[dt + u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[b][u][1], ph[ks], o[dt + u], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Meeting n: K of tile n and V of tile n - 1 have landed, and nobody reads K of n - 1 or V of
    // n - 2 any more, whose buffers then take K of n + 1 and V of n. The two waves of a SIMD (w and
    // w + 4) meet at different places of their work, the first in front of the weighted values,
    // the other in front of the softmax: one's MFMAs run while the other takes exponentials.
    auto meet = [&](int n, u16* kn, u16* vn) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (n + 1 < nt) copy(tile_of(n + 1), 0, kn);
        if (n > n0 && n < nt) copy(tile_of(n), 1, vn);  // the first one came with its K
    };
    const bool late = w < WAVES / 2;
    // Tiles with exponents of their keys, and those whose scores may need fp32, are behind everything that a row
    // sees in this loop and wait for a second one: branches for them here made the compiler copy the scores around
    // each (17 of 400 instructions a tile, distance 84 -> 88 us), ways around their products made it spill.
    bool some_odd = false;
    auto is_odd = [&](int ek, int flag, float ksum) { return (flag & (kKeyExps | kValueExps)) || loses(ek, ksum); };
    auto sees = [&](int k0) { return active && ((k0 < pre && k0 + kKT > 0) || (k0 < last_hi && k0 + kKT > first_lo)); };
    int bad_first = nt, bad_last = -1;  // the tiles that hold values that are not finite
    // kc, vc: this tile's; vn: the next one's V (the next but one's K goes into kc)
    auto step = [&](int n, u16* kc, u16* vc, u16* vn) __attribute__((always_inline)) {
        const int tile = tile_of(n), k0 = tile * kKT - T.z;
        // asked for here, so that the answer is there after the products
        const int4 about = info[tile];
        const int tile_ek = __builtin_amdgcn_readfirstlane(about.x), tile_ev = __builtin_amdgcn_readfirstlane(about.y),
                  flag = __builtin_amdgcn_readfirstlane(about.z), sum_bits = __builtin_amdgcn_readfirstlane(about.w);
        if (flag & kNotFinite) {
            bad_first = min(bad_first, n);
            bad_last = n;
        }
        const bool odd = is_odd(tile_ek, flag, __uint_as_float(sum_bits));
        some_odd |= odd;
        if (!sees(k0)) {
            meet(n + 1, kc, vn);
            return;
        }
        scores(kc);
        if (!late) meet(n + 1, kc, vn);
        softmax(std::false_type(), odd ? lk + kKT : k0, tile, tile_ek, tile_ev, flag, 0.f);
        if (late) meet(n + 1, kc, vn);
        values(vc);
    };
    if (n0 < nt) meet(n0, kbuf1, vbuf0);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) q_most = f2{fmaxf(q_most[0], q_waves[i][0]), fmaxf(q_most[1], q_waves[i][1])};
    q_most = f2{dev::readlane(q_most[0], 0), dev::readlane(q_most[1], 0)};
    for (int n = n0; n < nt; n += 2) {
        step(n, kbuf0, vbuf0, vbuf1);
        if (n + 1 < nt) step(n + 1, kbuf1, vbuf1, vbuf0);
    }
    if (some_odd) {  // of all waves alike
        auto together = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
        for (int n = n0; n < nt; n += 64) {
            const int4 about = n + lane < nt ? info[tile_of(n + lane)] : make_int4(0, 0, 0, 0);
            for (unsigned long long left = __ballot(n + lane < nt && is_odd(about.x, about.z, __uint_as_float(about.w))); left; left &= left - 1) {
                const int i = (int)__ffsll(left) - 1, tile = tile_of(n + i), k0 = tile * kKT - T.z;
                together();  // nobody reads the buffers any more
                copy(tile, 0, kbuf0);
                copy(tile, 1, vbuf0);
                together();
                if (!sees(k0)) continue;
                scores(kbuf0);
                softmax(std::true_type(), k0, tile, __builtin_amdgcn_readlane(about.x, i), __builtin_amdgcn_readlane(about.y, i),
                        __builtin_amdgcn_readlane(about.z, i), dev::readlane(__uint_as_float(about.w), i));
                values(vbuf0);
            }
        }
    }

    if (r >= rows) return;
    sum += __shfl_xor(sum, 32, 64);
    // a part of the keys: the sums as they are, on the scale of the reference
    const float inv = sum == 0.f ? 0.f : S.n > 1 ? 1.0f : 1.0f / sum;
    for (int n = bad_first; n <= bad_last; ++n)
        for (int j = max(tile_of(n) * kKT - T.z, 0), end = min(tile_of(n) * kKT - T.z + kKT, lk); j < end; ++j) {
            if (!visible(j)) continue;
            const auto R = args();
            const int d = R->d;
            const int64_t key = ((int64_t)(T.z + j) * R->kv_heads + kh) * d;
            const float *qr = R->q + ((int64_t)(T.first + qi) * R->heads + h) * d, *kr = R->k + key, *vr = R->v + key;
            bool any = false;
            for (int c = 0; c < d; ++c) any |= abs_bits(vr[c]) >= kInfBits;
            if (!any || hidden(R, j)) continue;
            float x = 0.f;
            for (int c = 0; c < d; ++c) x = fmaf(qr[c], kr[c], x);
            if (x * R->scale == -INFINITY && !(R->cap > 0.f)) continue;  // no weight
            int c0 = fh * 4;
            asm volatile("" : "+v"(c0));
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {  // columns past d are not stored
                    const float y = vr[min(dt * 32 + (i >> 2) * 8 + c0 + (i & 3), d - 1)];
                    if (abs_bits(y) >= kInfBits) o[dt][i] += y;
                    few(i);
                }
        }
    const int64_t row = (int64_t)(T.first + qi) * P.heads + h, cell = row * S.n + blockIdx.y, at = row * d;
    if (S.n > 1 && fh == 0) S.ml[cell] = f2{m, sum};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = dt * 32 + g * 8 + fh * 4;
            if (c >= d) continue;
            f4 v;  // two steps: 2^(E - 14) / sum may be subnormal where the results are not
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = ldexpf(o[dt][g * 4 + e] * inv, E - 14);
            if (S.n > 1) {
                *(f4*)(S.o + cell * S.stride + c) = v;
            } else if constexpr (VEC) {
                if (out16) *(uint2*)((u16*)P.out + at + c) = dev::bf16x4(v);
                else *(f4*)((float*)P.out + at + c) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < d) {
                        if (out16) ((u16*)P.out)[at + c + e] = dev::bf16_rne(v[e]);
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
//
// Bound by the cache's bytes: 32 tokens of 40 to 4096 keys, 32/8 heads of 128, 102 us with the
// join, 5.4 TB/s. Four loads instead of eight, two or eight waves instead of four: all slower.
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
    // The weighted values of a chunk some of which are not finite, a key at a time: 0 * inf is neither zero nor inf, where a
    // key does not count or its weight underflows. What is not finite waits in the lane's place of so for the end.
    bool had_odd = false;
    const int g0 = w * KEYS + sub;
    auto odd_values = [&](int k0) __attribute__((always_inline)) {
        if (!had_odd) {
#pragma unroll
            for (int r = 0; r < R; ++r) *(f4*)&so[g0][r][c4] = f4{0.f, 0.f, 0.f, 0.f};
        }
        had_odd = true;
#pragma unroll 1
        for (int u = 0; u < kLoads; ++u) {
            const int j = k0 + u * KEYS + sub;
            const int64_t at = base + min(j, lk - 1) * kv_inner;
            f4 k = *(const f4*)(P.k + at);
            const f4 v = *(const f4*)(P.v + at);
            if (c4 >= d) k = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = lanes_sum<LANES>(fmaf(q[r].x, k.x, q[r].y * k.y) + fmaf(q[r].z, k.z, q[r].w * k.w));
                if constexpr (EXTRA) {
                    if (P.cap > 0.f) x = P.cap * tanh_near(x / P.cap);
                    if (P.bias) x = biased(x, P.bias[(int64_t)head[r] * (2 * P.radius + 1) + P.radius + min(max(j - place[r], -P.radius), P.radius)]);
                }
                if (!((j < pre) | ((j >= lo[r]) & (j < hi[r]))) || x == -INFINITY) continue;
                const float weight = __builtin_amdgcn_exp2f((x - m[r]) * (EXTRA ? kLog2e : 1.0f));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (finite(v[e])) o[r][e] = fmaf(weight, v[e], o[r][e]);
                    else so[g0][r][c4 + e] += v[e];
                }
            }
        }
    };
    for (int n = n0 + w; n < n1; n += kFewWaves) {
        const int k0 = (n < npre ? n : next + n - npre) * CHUNK;
        f4 kx[kLoads], vx[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) kx[u] = dev::ld_stream((const f4*)(P.k + base + min(k0 + u * KEYS + sub, lk - 1) * kv_inner));
#pragma unroll
        for (int u = 0; u < kLoads; ++u) vx[u] = dev::ld_stream((const f4*)(P.v + base + min(k0 + u * KEYS + sub, lk - 1) * kv_inner));
        if (d < DP) {  // lanes past d: their zeros of q times an infinity would be NaN
#pragma unroll
            for (int u = 0; u < kLoads; ++u) kx[u] = c4 < d ? kx[u] : f4{0.f, 0.f, 0.f, 0.f};
        }
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
                        s[u][r] = biased(s[u][r], P.bias[(int64_t)head[r] * (2 * P.radius + 1) + P.radius +
                                                         min(max(k0 + u * KEYS + sub - place[r], -P.radius), P.radius)]);
                }
        }
        if (!full) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (!visible(u, r)) s[u][r] = -INFINITY;
        }
        float odd = 0.f;  // NaN with a value that is not finite
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd = fmaf(vx[u][e], 0.f, odd);
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
        if (__ballot(odd != 0.f)) {
            odd_values(k0);
        } else {
#pragma unroll
            for (int u = 0; u < kLoads; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) o[r] += s[u][r] * vx[u];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        *(f4*)&so[g0][r][c4] = had_odd ? o[r] + *(const f4*)&so[g0][r][c4] : o[r];
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
        if (!finite(v)) {  // a group's infinity times its weight of zero
            v = f4{0.f, 0.f, 0.f, 0.f};
            for (int g = 0; g < GROUPS; ++g)
                v += scaled(*(const f4*)&so[g][r][c], __builtin_amdgcn_exp2f(EXTRA ? (sm[g][r] - ref) * kLog2e : sm[g][r] - ref));
        }
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

// out from the parts: a workgroup of sixteen 32-lane groups per (query row, head), each taking
// every sixteenth part, once the parts' weights are known. `unit`: log2(e) where the references
// are not in log2 units.
constexpr int kMaxParts = 256, kJoin = 16;
__global__ __launch_bounds__(32 * kJoin) void k_attn_packed_join(Packed P, int out16, Parts S, float unit) {
    __shared__ float so[kJoin][128], weight[kMaxParts], tops[kJoin / 2], sums[kJoin / 2];
    const int t = blockIdx.x, h = blockIdx.y, c = (threadIdx.x & 31) * 4, g = threadIdx.x >> 5;
    if (dev::span_of_row(P.spans, P.seqs, t, P.Tq) < 0) return;
    const int64_t row = (int64_t)t * P.heads + h, cell = row * S.n;
    const int i = threadIdx.x;
    const f2 ml = i < S.n ? S.ml[cell + i] : f2{-INFINITY, 0.f};
    const float mine = dev::wave_max(ml.x);
    if ((i & 63) == 0) tops[i >> 6] = mine;
    __syncthreads();
    float top = tops[0];
#pragma unroll
    for (int k = 1; k < kJoin / 2; ++k) top = fmaxf(top, tops[k]);
    const float ref = top == -INFINITY ? 0.f : top;
    const float x = __builtin_amdgcn_exp2f((ml.x - ref) * unit);
    if (i < kMaxParts) weight[i] = x;
    const float part = dev::wave_sum(i < S.n ? x * ml.y : 0.f);
    if ((i & 63) == 0) sums[i >> 6] = part;
    __syncthreads();
    f4 v = {0.f, 0.f, 0.f, 0.f};
    if (c < P.d) {
#pragma unroll 4
        for (int s = g; s < S.n; s += kJoin) v += weight[s] * *(const f4*)(S.o + (cell + s) * S.stride + c);
        if (!finite(v)) {  // a part's infinity times its weight of zero
            v = f4{0.f, 0.f, 0.f, 0.f};
            for (int s = g; s < S.n; s += kJoin) v += scaled(*(const f4*)(S.o + (cell + s) * S.stride + c), weight[s]);
        }
    }
    *(f4*)&so[g][c] = v;
    __syncthreads();
    if (g || c >= P.d) return;
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < kJoin / 2; ++k) l += sums[k];
#pragma unroll
    for (int k = 1; k < kJoin; ++k) v += *(const f4*)&so[k][c];
    v *= l == 0.f ? 0.f : 1.0f / l;
    const int64_t at = row * P.d + c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < P.d) {
            if (out16) ((u16*)P.out)[at + e] = dev::bf16_rne(v[e]);
            else ((float*)P.out)[at + e] = v[e];
        }
}

// The parts' memory; where it cannot be had the keys stay uncut. `behind`: bytes that the
// caller needs in front of it, whose address is put into `front` (null with nothing to be had).
Parts make_parts(const Packed& P, int64_t n, size_t behind, char*& front) {
    Parts S{(int)n, (P.d + 3) / 4 * 4, nullptr, nullptr};
    const size_t cells = (size_t)P.Tq * P.heads * n, ob = (cells * S.stride * 4 + 255) / 256 * 256;
    behind = (behind + 255) / 256 * 256;
    front = n > 1 ? (char*)try_scratch(behind + ob + cells * sizeof(f2)) : nullptr;
    if (front) {
        S.o = (float*)(front + behind);
        S.ml = (f2*)(front + behind + ob);
    } else {
        S.n = 1;
        if (behind) front = (char*)try_scratch(behind);
    }
    return S;
}

void join_parts(const Packed& P, bool out16, const Parts& S, bool log2_units) {
    if (S.n > 1)
        k_attn_packed_join<<<dim3((unsigned)P.Tq, (unsigned)P.heads), 32 * kJoin, 0, stream()>>>(P, out16, S, log2_units ? 1.0f : kLog2e);
}

template <int DP>
void run_few(const Packed& P, bool out16, int64_t items, int rows) {
    const bool extra = P.cap > 0.f || P.bias;
    // Parts of the keys until there are sixteen workgroups a CU, which evens out sequences of unlike
    // length, but of 256 keys of an average one at least. Measured, us, with eight / sixteen: 32
    // sequences of up to 4096 keys, 32/8 heads of 128: 127 / 116; one of 30001 in 256 / 128 parts 73 / 67.
    const int64_t wgs = items * P.kv_heads, keys = P.Tk / std::max(1, P.seqs);
    char* none;
    const Parts S = make_parts(P, std::max<int64_t>(1, std::min<int64_t>({16 * num_cus() / wgs, keys / 256, (int64_t)kMaxParts})), 0, none);
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

// `rows` rows (queries times the heads of a group) of `live` sequences; false where the tiles'
// scratch cannot be had.
template <int DP>
bool run_tiles(const Packed& P, bool out16, int64_t rows, int64_t live) {
    const bool kvec = P.d % 8 == 0 && aligned16(P.k) && aligned16(P.v),
               qvec = P.d % 8 == 0 && aligned16(P.q) && (out16 ? ((uintptr_t)P.out & 7) == 0 : aligned16(P.out));
    // Parts of the keys while the workgroups do not fill the chip, of eight tiles of an average sequence at least.
    const int64_t items = rows / (32 * kWaves<DP>) + live, wgs = items * P.kv_heads, keys = P.Tk / std::max(1, P.seqs), ntiles = (P.Tk + kKT - 1) / kKT;
    if (wgs * 64 * kWaves<DP> > kMaxGridItems) return false;
    const size_t cells = (size_t)ntiles * P.kv_heads, tb = cells * 4 * kKT * DP * 2;
    char* front;
    const Parts S = make_parts(P, std::max<int64_t>(1, std::min<int64_t>({num_cus() * (8 / kWaves<DP>) / wgs, keys / (8 * kKT), (int64_t)kMaxParts})),
                               tb + cells * (sizeof(int4) + 2 * kKT * sizeof(int)), front);
    if (!front) return false;
    const Tiles X{(u16*)front, (int4*)(front + tb), (int*)(front + tb + cells * sizeof(int4)), (int)ntiles};
    const dim3 sg((unsigned)ntiles, (unsigned)P.kv_heads);
    if (kvec) k_attn_packed_split<DP, true><<<sg, 64 * kSplitWaves, 0, stream()>>>(P, X);
    else k_attn_packed_split<DP, false><<<sg, 64 * kSplitWaves, 0, stream()>>>(P, X);
    // What the tiles leave of a CU's LDS takes the bias of a group's heads, if it fits.
    const int64_t values = P.bias ? (int64_t)(P.heads / P.kv_heads) * (2 * P.radius + 1 + 2 * kBiasPad) : 0;
    const int table = values * 4 <= 14 * 1024 * (kWaves<DP> / 4) ? (int)values : 0;
    const bool extra = P.cap > 0.f || P.bias;
    using T_ = std::true_type;
    using F_ = std::false_type;
    auto go = [&](auto ex, auto ve) {
        k_attn_packed_tiles<DP, decltype(ex)::value, decltype(ve)::value>
            <<<dim3((unsigned)wgs, (unsigned)S.n), 64 * kWaves<DP>, (unsigned)table * 4, stream()>>>(P, X, out16, (int)items, table, S);
    };
    if (extra) qvec ? go(T_(), T_()) : go(T_(), F_());
    else qvec ? go(F_(), T_()) : go(F_(), F_());
    join_parts(P, out16, S, !extra);
    return true;
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
    need(seqs <= dev::kMaxSpans, op, "more than 65536 sequences");
    need(d <= kMaxD, op, "head dimension above 1024");
    need(heads <= 65535, op, "too many heads for one launch");
    need(Tq < kMost && Tk < kMost && radius < kMost, op, "a size of 2^30 or more");
    need(!bias || (int64_t)heads * (2 * radius + 1) < 2 * kMost, op, "a bias of 2^31 values or more");
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
    // An average sequence's rows at one key/value head: up to sixteen go to k_attn_packed_few. Measured, us, there /
    // in tiles, 32/8 heads of 128: 32 sequences of up to 4096 keys, 8 rows 158 / 406, 16 rows 261 / 420, 40 rows 568 /
    // 434; four sequences, 16 rows 64 / 79, 40 rows 112 / 80; 32 of up to 256 keys, 16 rows 32 / 37, 40 rows 66 / 38.
    const int64_t group = heads / kv_heads, live = std::min(seqs, Tq), mean = (Tq + live - 1) / live * group;
    if (d <= 128 && d % 4 == 0 && mean <= 16 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out)) {
        const int r = mean <= 1 ? 1 : mean <= 4 ? 4 : 8;
        const int64_t n = Tq * group / r + live;
        if (Tq * group < kMost && n * kv_heads * 64 * kFewWaves <= kMaxGridItems) {
            if (d <= 64) run_few<64>(P, out16, n, r);
            else run_few<128>(P, out16, n, r);
            launched(op);
            return;
        }
    }
    if (d <= 128 && Tq * group < kMost && (Tk + kKT) * 4 <= kMaxGridItems) {
        if (d <= 64 ? run_tiles<64>(P, out16, Tq * group, live) : run_tiles<128>(P, out16, Tq * group, live)) {
            launched(op);
            return;
        }
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
