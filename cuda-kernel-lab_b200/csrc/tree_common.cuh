// tree_common.cuh -- what the draft-tree attention and the cache-weight kernels share: the
// launch arguments, the geometry of a sequence and its new tokens, the scores and who sees what.
#pragma once

#include "attn_common.cuh"

namespace ckl {
namespace tree {

using namespace attn;

struct Args {
    const __half* q;
    const __half* v;          // the V cache (the streamed reads go through tensor maps)
    const int* indptr;
    const int* indices;
    const int* last;
    const int* q_indptr;      // NULL: one token per sequence
    const uint32_t* mask;     // NULL: chain
    const int* positions;     // NULL: cache places
    const float* slopes;      // NULL: no bias
    float* part_o;            // [N*Hq][num_chunks][128], NULL with one chunk
    float* part_lse;          // [N*Hq][num_chunks]
    __half* out;
    float* lse;
    unsigned* err;
    unsigned long long timeout_ns;
    int B, N, Hq, Hkv, G, max_q, mask_words, num_chunks, chunk_tokens, window, num_pages;
    float scale_log2;         // sm_scale * log2(e)
    float cap_log2;           // softcap * log2(e), 0: no cap
    float cap_in;             // 2 log2(e) sm_scale / softcap
    float cap_k;              // sm_scale / softcap
    float cap_lim;            // greatest |q.k| that cap_factor2 is for (-1: none)
    float cap_poly[4];        // of a capped score / q.k in (q.k)^2, see cap_factor2
    int q_tma;                // the tcgen05 kernel reads Q tiles through a tensor map
};

// Length of sequence b from the page table; a last page outside [0, 16] is taken as full/empty.
__device__ __forceinline__ int seq_len(const int* indptr, const int* last, int b, int* page0) {
    *page0 = __ldg(indptr + b);
    const int np = __ldg(indptr + b + 1) - *page0;
    return np > 0 ? (np - 1) * PAGE + min(max(__ldg(last + b), 0), PAGE) : 0;
}

struct Seq {
    int page0;      // first entry of the page list
    int len;        // cached tokens, new ones included
    int q0, T;      // first row and count of the new tokens
    int ctx;        // cache place of new token 0 (negative when the table is too short)
    __device__ __forceinline__ Seq() : page0(0), len(0), q0(0), T(0), ctx(0) {}
    __device__ __forceinline__ Seq(const Args& a, int b) {
        len = seq_len(a.indptr, a.last, b, &page0);
        q0 = a.q_indptr ? __ldg(a.q_indptr + b) : b;
        T = a.q_indptr ? __ldg(a.q_indptr + b + 1) - q0 : 1;
        if (q0 < 0 || q0 + T > a.N || T < 0) T = 0;      // rows outside the tensors: none
        ctx = len - T;
    }
    // Position of cached token p (p itself behind the sequence).
    __device__ __forceinline__ int pos(const Args& a, int p) const {
        return a.positions && p >= ctx && p < len ? __ldg(a.positions + q0 + (p - ctx)) : p;
    }
};

// Least and greatest position of the sequence's tokens (one warp; all lanes get both).
__device__ __forceinline__ void pos_range(const Args& a, const Seq& s, int lane, int* lo, int* hi) {
    if (!a.positions) {
        *lo = s.ctx;
        *hi = s.len - 1;
        return;
    }
    int l = 0x7fffffff, h = -0x7fffffff - 1;
    for (int i = lane; i < s.T; i += 32) {
        const int p = __ldg(a.positions + s.q0 + i);
        l = min(l, p);
        h = max(h, p);
    }
    *lo = __reduce_min_sync(0xffffffffu, l);
    *hi = __reduce_max_sync(0xffffffffu, h);
}

// First cache place that any token of the sequence can see, rounded down to a page: context
// keys at or below (least position - window) are out of every window. 64-bit: positions span
// all of int32.
__device__ __forceinline__ int first_key(const Args& a, const Seq& s, int pos_lo) {
    if (a.window <= 0) return 0;
    const long long f = (long long)pos_lo - a.window + 1;
    const int lim = max(min(s.ctx, s.len), 0);           // drafted keys have their own positions
    const int k = f <= 0 ? 0 : (f >= lim ? lim : (int)f);
    return k & ~(PAGE - 1);
}

// W blocks over n CTAs: the first W % n take one more than the others.
struct Share {
    long long each;
    int n, more;
    __device__ __forceinline__ Share(long long W, int n_) : n(n_) {
        each = W >> 31 ? W / n : (long long)((unsigned)W / (unsigned)n);
        more = (int)(W - each * n);
    }
    __device__ __forceinline__ long long first(int c) const { return each * c + min(c, more); }   // block of CTA c
    __device__ __forceinline__ int owner(long long u) const {                                      // CTA of block u
        const long long big = (each + 1) * more, x = u < big ? u : u - big, d = u < big ? each + 1 : each;
        return (u < big ? 0 : more) + (int)(x >> 31 ? x / d : (long long)((unsigned)x / (unsigned)d));
    }
};

// One query row's view of the keys.
struct Row {
    int i = -1;           // new token (-1: padding)
    int pos = 0;
    float slope2 = 0.f;   // slope * log2(e)
    __device__ __forceinline__ void set(const Args& a, const Seq& s, int row, int nrows, int kvh) {
        if (row >= nrows) return;
        i = row / a.G;
        pos = a.positions ? __ldg(a.positions + s.q0 + i) : s.ctx + i;
        if (a.slopes) slope2 = __ldg(a.slopes + kvh * a.G + row % a.G) * LOG2E;
    }
    // Is cached token p (at position kpos) seen?
    __device__ __forceinline__ bool sees(const Args& a, const Seq& s, int p, int kpos) const {
        if (i < 0 || p >= s.len) return false;
        if (a.window > 0 && (long long)pos - kpos >= a.window) return false;
        const int j = p - s.ctx;
        if (j < 0) return true;
        if (!a.mask) return j <= i;
        if (j >= 32 * a.mask_words) return false;
        return (__ldg(a.mask + (size_t)(s.q0 + i) * a.mask_words + (j >> 5)) >> (j & 31)) & 1u;
    }
};

// P goes to its product in fp16 (2^-11 of each weight, as V's own rounding). The reference that it is
// taken against stays 2^P_LIFT below the running maximum: weights reach 2^15 with RESCALE_THRESHOLD
// on top, and one is lost from 2^-32 of the greatest down, where without it a long row of weights
// below 2^-25 would count in the sum but not in the result.
constexpr float P_LIFT = 7.f;

// tanh(y)/y in y^2 for |y| <= CAP_SMALL: fitted to it by weighted least squares, off by at most 2^-21.9
// of it.
constexpr float TANH_0 = 0.99999976f, TANH_1 = -0.33329466f, TANH_2 = 0.13236369f, TANH_3 = -0.04602819f;
constexpr float CAP_SMALL = 0.45f;
// A capped score in the log2 domain from the raw product q.k, y = q.k sm_scale / softcap. Up to
// CAP_SMALL the polynomial, off by 2^-21.9 of the score however loose the cap. Beyond it tanh(y) =
// 1 - 2/(1 + e^2y), off by ~2^-23 of the cap, which the score is 0.42 of at least (tanh.approx would
// lose 2^-11). Each value by its own size: what else a warp holds has no part in it.
__device__ __forceinline__ float2 cap_small2(const Args& a, float2 qk) {
    const float2 y = mul2(qk, make_float2(a.cap_k, a.cap_k)), t = mul2(y, y);
    float2 p = fma2(make_float2(TANH_3, TANH_3), t, make_float2(TANH_2, TANH_2));
    p = fma2(p, t, make_float2(TANH_1, TANH_1));
    p = fma2(p, t, make_float2(TANH_0, TANH_0));
    return mul2(mul2(qk, make_float2(a.scale_log2, a.scale_log2)), p);
}
__device__ __forceinline__ float cap_exact(const Args& a, float qk) {
    return fmaf(-2.f * a.cap_log2, rcp(1.f + ex2(qk * a.cap_in)), a.cap_log2);
}
// Scores in the log2 domain of the M products that a thread holds. The exponential form is only made
// in warps that need it.
template <int M>
__device__ __forceinline__ void cap_all(const Args& a, float (&x)[M]) {
    float m4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < M; c++) m4[c & 3] = fmaxf(m4[c & 3], fabsf(x[c]));
    const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    if (__any_sync(0xffffffffu, !(top * a.cap_k <= CAP_SMALL))) {
#pragma unroll
        for (int c = 0; c < M; c += 2) {
            const float2 v = make_float2(x[c], x[c + 1]), s = cap_small2(a, v);
            const float e0 = cap_exact(a, v.x), e1 = cap_exact(a, v.y);
            x[c] = fabsf(v.x) * a.cap_k <= CAP_SMALL ? s.x : e0;
            x[c + 1] = fabsf(v.y) * a.cap_k <= CAP_SMALL ? s.y : e1;
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < M; c += 2) {
        const float2 s = cap_small2(a, make_float2(x[c], x[c + 1]));
        x[c] = s.x;
        x[c + 1] = s.y;
    }
}
template <bool EXT, int M>
__device__ __forceinline__ void score_all(const Args& a, float (&x)[M]) {
    if (EXT && a.cap_log2 > 0.f) {
        cap_all(a, x);
        return;
    }
#pragma unroll
    for (int c = 0; c < M; c += 2) {
        const float2 v = mul2(make_float2(x[c], x[c + 1]), make_float2(a.scale_log2, a.scale_log2));
        x[c] = v.x;
        x[c + 1] = v.y;
    }
}
// Capped scores are nearly always far below the cap. In the main loop of the tcgen05 kernel, the terms
// scaled by the launch so that the polynomial is one in (q.k)^2: five operations on two values each
// where the exponential form takes two of the special-function unit, which the exponentials already
// fill. For |q.k| up to cap_lim, that is CAP_SMALL of the cap where the scaled terms are normal numbers.
// A fourth degree would reach to 0.6 of the cap: 16 x 24 drafts 128 us against 118.
// -> score / q.k, log2 domain
__device__ __forceinline__ float2 cap_factor2(const Args& a, float2 qk) {
    const float2 t = mul2(qk, qk);
    float2 p = fma2(make_float2(a.cap_poly[3], a.cap_poly[3]), t, make_float2(a.cap_poly[2], a.cap_poly[2]));
    p = fma2(p, t, make_float2(a.cap_poly[1], a.cap_poly[1]));
    return fma2(p, t, make_float2(a.cap_poly[0], a.cap_poly[0]));
}
template <bool EXT>
__device__ __forceinline__ float bias(const Args& a, float slope2, int pos, int kpos) {
    return EXT ? slope2 * (float)(kpos - pos) : 0.f;
}

// tree_attention.cu: checks the parameters that the attention and the weights share.
ckl_status check_params(const ckl_tree_params* p, const char* who);
ckl_status fill_args(const ckl_tree_params* p, Args* a);

}  // namespace tree
}  // namespace ckl
