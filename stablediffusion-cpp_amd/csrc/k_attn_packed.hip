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

#include "spans.hpp"

namespace sdh {
namespace {

typedef unsigned short u16;
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
