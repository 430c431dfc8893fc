// rope_append.cu -- rotary positions on q and k, and the append of k and v to the paged cache,
// in one pass: every input element is read once and every output written once (HBM-bound for
// many tokens, launch latency for few).
//
// The angle of pair i at position p is 2 pi frac(p * f_i / 2 pi). f_i / 2 pi is kept as a 64-bit
// binary fraction, so the integer product p * turns[i] mod 2^64 is the wrapped turn itself: no
// table of positions to read, and far positions lose nothing (p * 2^-64 turns from the fraction's
// own rounding, where p * f_i in fp32 is off by p * 2^-25 radians and more). The top 32 bits go to
// sincospi. One CTA per token: 64 threads make the token's sines once for all of its heads.

#include <algorithm>
#include <cmath>

#include "ckl_internal.h"
#include "tree_common.cuh"

namespace ckl {
namespace rope {

using attn::D;
using attn::PAGE;

struct Args {
    const __half* q;
    const __half* k;
    const __half* v;
    __half* q_out;
    __half* k_cache;
    __half* v_cache;
    const int* indptr;
    const int* indices;
    const int* last;
    const int* q_indptr;
    const int* positions;
    long long q_stride, k_stride, v_stride;
    int B, N, Hq, Hkv, num_pages;
    int qheads;               // Hq, or 0 when q is NULL
    ckl_rope rope;            // rot_dim 0: copy
};

// Number of entries of ptr[0..n] (ascending, n + 1 of them) that are <= x: 32 probes a round.
__device__ __forceinline__ int count_le(const int* ptr, int n, int x, int lane) {
    int lo = 0, hi = n + 1;                          // the count is in [lo, hi]
    while (hi - lo > 32) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + (lane + 1) * step - 1;   // last entry of this lane's piece
        const bool le = at < hi && __ldg(ptr + at) <= x;
        const int pieces = __popc(__ballot_sync(0xffffffffu, le));
        lo += pieces * step;
        hi = min(hi, lo + step - 1);
    }
    const bool le = lo + lane < hi && __ldg(ptr + lo + lane) <= x;
    return lo + __popc(__ballot_sync(0xffffffffu, le));
}

__device__ __forceinline__ void rotate(float& a, float& b, float2 cs) {
    const float x = a * cs.x - b * cs.y;
    b = a * cs.y + b * cs.x;
    a = x;
}
__device__ __forceinline__ void unpack(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
        f[2 * i] = __low2float(h);
        f[2 * i + 1] = __high2float(h);
    }
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
}

// LAYOUT 0: halves in 16-byte chunks (rot_dim a multiple of 16): a unit is chunk c and its
//           partner chunk c + rot_dim/16, or one chunk of the copied rest;
//        1: interleaved in 16-byte chunks (rot_dim a multiple of 8): a unit is one chunk;
//        2: any even rot_dim: a unit is one chunk, its partners read one by one.
// grid = (N, splits of a token's units).
// A thread's first two units are fetched before the token's sequence, page and angles are known, so
// that those loads overlap the chain of lookups (12,500 tokens: 57.0 -> 50.4 us).
template <int LAYOUT>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ Args a) {
    __shared__ float2 cs[D / 2];
    pdl_wait();
    pdl_trigger();
    const int n = blockIdx.x, lane = threadIdx.x & 31;
    const int rot = a.rope.rot_dim, pairs = rot >> 1;
    const int rc = rot >> 3;                               // 16-byte chunks that are rotated (layouts 0, 1)
    const int per = LAYOUT == 0 ? 16 - (rc >> 1) : 16;     // units of a rotated head
    const int nrot = (a.qheads + a.Hkv) * per, units = nrot + a.Hkv * 16;
    const int stride = gridDim.y * blockDim.x, u0 = blockIdx.y * blockDim.x + threadIdx.x;
    // first chunk of unit u, in chunks of 16 bytes, and its head (q, then k; v from nrot on)
    auto source = [&](int u, int* head, int* c) -> const __half* {
        if (u >= nrot) {
            *head = (u - nrot) >> 4;
            *c = (u - nrot) & 15;
            return a.v + n * a.v_stride + *head * D;
        }
        *head = u / per;
        *c = u - *head * per;
        return *head < a.qheads ? a.q + n * a.q_stride + *head * D : a.k + n * a.k_stride + (*head - a.qheads) * D;
    };
    auto fetch = [&](int u, uint4* x, uint4* y) {
        if (u >= units) return;
        int h, c;
        const uint4* s4 = reinterpret_cast<const uint4*>(source(u, &h, &c));
        const bool pair = LAYOUT == 0 && u < nrot && c < (rc >> 1);
        *x = __ldg(s4 + (LAYOUT == 0 && u < nrot && !pair ? c + (rc >> 1) : c));
        if (pair) *y = __ldg(s4 + c + (rc >> 1));
    };
    uint4 x0, y0, x1, y1;
    fetch(u0, &x0, &y0);
    fetch(u0 + stride, &x1, &y1);

    int b = n, i = 0, T = 1;
    if (a.q_indptr) {
        const int c = count_le(a.q_indptr, a.B, n, lane);
        if (c == 0 || c > a.B) return;                     // not a token of any sequence
        b = c - 1;
        const int q0 = __ldg(a.q_indptr + b);
        i = n - q0;
        T = __ldg(a.q_indptr + b + 1) - q0;
    }
    int page0;
    const int place = tree::seq_len(a.indptr, a.last, b, &page0) - T + i;
    const int pos = a.positions ? __ldg(a.positions + n) : place;
    long long crow = -1;                                   // row of this token in the cache
    if (place >= 0) {
        const int page = __ldg(a.indices + page0 + place / PAGE);
        if (page >= 0 && page < a.num_pages) crow = (long long)page * PAGE + place % PAGE;
    }
    if (threadIdx.x < pairs) {
        const uint64_t turn = (uint64_t)(long long)pos * a.rope.turns[threadIdx.x];
        float sn, c;
        sincospif((float)(int)(uint32_t)(turn >> 32) * 0x1p-31f, &sn, &c);
        cs[threadIdx.x] = make_float2(c * a.rope.scale, sn * a.rope.scale);
    }
    __syncthreads();

    auto emit = [&](int u, uint4 v, uint4 w) {
        int h, c;
        const __half* src = source(u, &h, &c);
        if (u >= nrot) {                                   // v: copied
            if (crow >= 0) reinterpret_cast<uint4*>(a.v_cache + (crow * a.Hkv + h) * D)[c] = v;
            return;
        }
        const bool isq = h < a.qheads;
        if (!isq && crow < 0) return;
        uint4* d4 = reinterpret_cast<uint4*>(isq ? a.q_out + ((size_t)n * a.Hq + h) * D
                                                 : a.k_cache + (crow * a.Hkv + (h - a.qheads)) * D);
        if (LAYOUT == 0) {
            const int hc = rc >> 1;
            if (c < hc) {
                float x[8], y[8];
                unpack(v, x);
                unpack(w, y);
#pragma unroll
                for (int e = 0; e < 8; e++) rotate(x[e], y[e], cs[8 * c + e]);
                d4[c] = pack(x);
                d4[c + hc] = pack(y);
            } else {
                d4[c + hc] = v;
            }
        } else if (LAYOUT == 1) {
            if (c < rc) {
                float x[8];
                unpack(v, x);
#pragma unroll
                for (int e = 0; e < 4; e++) rotate(x[2 * e], x[2 * e + 1], cs[4 * c + e]);
                v = pack(x);
            }
            d4[c] = v;
        } else {
            float x[8];
            unpack(v, x);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = 8 * c + e;
                if (d >= rot) continue;
                const bool first = a.rope.interleaved ? !(d & 1) : d < pairs;
                const int mate = a.rope.interleaved ? d ^ 1 : (first ? d + pairs : d - pairs);
                const float2 t = cs[a.rope.interleaved ? d >> 1 : (first ? d : d - pairs)];
                const float y = __half2float(__ldg(src + mate));
                x[e] = first ? x[e] * t.x - y * t.y : y * t.y + x[e] * t.x;
            }
            d4[c] = pack(x);
        }
    };
    if (u0 < units) emit(u0, x0, y0);
    if (u0 + stride < units) emit(u0 + stride, x1, y1);
    for (int u = u0 + 2 * stride; u < units; u += stride) {
        fetch(u, &x0, &y0);
        emit(u, x0, y0);
    }
}

}  // namespace rope
}  // namespace ckl

using namespace ckl;
using namespace ckl::rope;

extern "C" {

ckl_status ckl_rope_plan_freqs(const double* inv_freq, int rot_dim, int interleaved, double scale,
                               ckl_rope* rope) {
    if (!rope || !inv_freq) return fail(CKL_INVALID_ARG, "rope_plan: NULL");
    if (rot_dim < 2 || rot_dim > D || rot_dim % 2)
        return fail(CKL_INVALID_ARG, "rope_plan: rot_dim=%d (even, 2..%d)", rot_dim, D);
    if (!std::isfinite(scale) || std::fabs(scale) > 1e30)
        return fail(CKL_INVALID_ARG, "rope_plan: scale must be finite");
    ckl_rope r{};
    r.rot_dim = rot_dim;
    r.interleaved = interleaved ? 1 : 0;
    r.scale = (float)scale;
    for (int i = 0; i < rot_dim / 2; i++) {
        if (!(inv_freq[i] >= 0.0 && inv_freq[i] <= M_PI))
            return fail(CKL_INVALID_ARG, "rope_plan: inv_freq[%d] = %g outside [0, pi]", i, inv_freq[i]);
        // f / 2 pi <= 1/2: below 2^63 after scaling
        r.turns[i] = (uint64_t)std::llrint(std::ldexp(inv_freq[i] / (2.0 * M_PI), 63)) << 1;
    }
    *rope = r;
    return CKL_OK;
}

ckl_status ckl_rope_plan(int rot_dim, int interleaved, double base, int scaling, double factor,
                         int original_len, double beta_fast, double beta_slow, ckl_rope* rope) {
    if (rot_dim < 2 || rot_dim > D || rot_dim % 2)
        return fail(CKL_INVALID_ARG, "rope_plan: rot_dim=%d (even, 2..%d)", rot_dim, D);
    if (!(base > 1.0) || !std::isfinite(base)) return fail(CKL_INVALID_ARG, "rope_plan: base must be finite and above 1");
    if (scaling < CKL_ROPE_NONE || scaling > CKL_ROPE_BY_PARTS)
        return fail(CKL_INVALID_ARG, "rope_plan: unknown scaling %d", scaling);
    if (scaling != CKL_ROPE_NONE && !(factor >= 1.0 && std::isfinite(factor)))
        return fail(CKL_INVALID_ARG, "rope_plan: factor must be finite and at least 1");
    if (scaling == CKL_ROPE_BY_PARTS &&
        !(original_len > 0 && beta_slow > 0.0 && beta_fast > beta_slow && std::isfinite(beta_fast)))
        return fail(CKL_INVALID_ARG, "rope_plan: by parts needs original_len > 0 and beta_fast > beta_slow > 0");
    const double r = rot_dim;
    if (scaling == CKL_ROPE_NTK && rot_dim > 2) base *= std::pow(factor, r / (r - 2.0));
    double f[D / 2];
    for (int i = 0; i < rot_dim / 2; i++) {
        f[i] = std::pow(base, -2.0 * i / r);
        if (scaling == CKL_ROPE_LINEAR) f[i] /= factor;
    }
    double scale = 1.0;
    if (scaling == CKL_ROPE_BY_PARTS) {
        // pair index that turns `beta` times over original_len tokens
        auto index = [&](double beta) { return r * std::log(original_len / (beta * 2.0 * M_PI)) / (2.0 * std::log(base)); };
        const double low = std::max(std::floor(index(beta_fast)), 0.0);
        const double high = std::min(std::ceil(index(beta_slow)), r - 1.0);
        for (int i = 0; i < rot_dim / 2; i++) {
            const double ramp = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
            f[i] = f[i] / factor * ramp + f[i] * (1.0 - ramp);
        }
        scale = 0.1 * std::log(factor) + 1.0;
    }
    return ckl_rope_plan_freqs(f, rot_dim, interleaved, scale, rope);
}

ckl_status ckl_rope_append(const ckl_append_params* p, const ckl_rope* rope, void* stream) {
    if (!p) return fail(CKL_INVALID_ARG, "rope_append: params is NULL");
    if (p->B < 0 || p->N < 0 || p->Hq < 0 || p->Hkv <= 0 || (p->q && p->Hq == 0))
        return fail(CKL_INVALID_ARG, "rope_append: bad counts B=%d N=%d Hq=%d Hkv=%d", p->B, p->N, p->Hq, p->Hkv);
    if (rope && (rope->rot_dim < 2 || rope->rot_dim > D || rope->rot_dim % 2))
        return fail(CKL_INVALID_ARG, "rope_append: rope is not a plan (rot_dim=%d)", rope->rot_dim);
    if (p->Hq > 65535 || p->Hkv > 65535) return fail(CKL_UNSUPPORTED_SHAPE, "rope_append: more than 65535 heads");
    if (p->B == 0 || p->N == 0) return CKL_OK;
    if (!p->k || !p->v || !p->k_cache || !p->v_cache || !p->kv_indptr || !p->kv_indices || !p->kv_last_page_len ||
        (p->q && !p->q_out))
        return fail(CKL_INVALID_ARG, "rope_append: NULL tensor pointer");
    if (!p->q_indptr && p->N != p->B)
        return fail(CKL_INVALID_ARG, "rope_append: without q_indptr there is one token per sequence (N=%d, B=%d)", p->N, p->B);
    if (p->num_pages <= 0) return fail(CKL_INVALID_ARG, "rope_append: num_pages must be > 0");
    if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->q_out | (uintptr_t)p->k_cache |
         (uintptr_t)p->v_cache) & 15)
        return fail(CKL_INVALID_ARG, "rope_append: tensors must be 16-byte aligned");
    const long long hq = p->q ? p->Hq : 0;
    if ((p->q && (p->q_stride % 8 || p->q_stride < hq * D)) || p->k_stride % 8 || p->v_stride % 8 ||
        p->k_stride < (long long)p->Hkv * D || p->v_stride < (long long)p->Hkv * D)
        return fail(CKL_INVALID_ARG, "rope_append: strides %lld/%lld/%lld must be multiples of 8 that hold a token's row",
                    p->q_stride, p->k_stride, p->v_stride);
    // every output against every input
    const size_t row = D * sizeof(__half), cache = (size_t)p->num_pages * PAGE * p->Hkv * row;
    auto bytes = [&](long long stride, long long heads) { return ((size_t)(p->N - 1) * stride) * sizeof(__half) + heads * row; };
    const Span in[3] = {{p->q, p->q ? bytes(p->q_stride, hq) : 0}, {p->k, bytes(p->k_stride, p->Hkv)},
                        {p->v, bytes(p->v_stride, p->Hkv)}};
    const Span out[3] = {{p->q_out, p->q ? (size_t)p->N * hq * row : 0}, {p->k_cache, cache}, {p->v_cache, cache}};
    for (int i = 0; i < 3; i++)
        for (int o = 0; o < 3; o++)
            if (overlap(in[i], out[o]))
                return fail(CKL_INVALID_ARG, "rope_append: an output overlaps an input");
    for (int o = 0; o < 3; o++)
        if (overlap(out[o], out[(o + 1) % 3]))
            return fail(CKL_INVALID_ARG, "rope_append: two outputs overlap");
    const DeviceInfo* di = device_info();
    if (!di) return CKL_CUDA_ERROR;

    Args a{};
    a.q = static_cast<const __half*>(p->q);
    a.k = static_cast<const __half*>(p->k);
    a.v = static_cast<const __half*>(p->v);
    a.q_out = static_cast<__half*>(p->q_out);
    a.k_cache = static_cast<__half*>(p->k_cache);
    a.v_cache = static_cast<__half*>(p->v_cache);
    a.indptr = p->kv_indptr;
    a.indices = p->kv_indices;
    a.last = p->kv_last_page_len;
    a.q_indptr = p->q_indptr;
    a.positions = p->positions;
    a.q_stride = p->q_stride;
    a.k_stride = p->k_stride;
    a.v_stride = p->v_stride;
    a.B = p->B;
    a.N = p->N;
    a.Hq = p->Hq;
    a.Hkv = p->Hkv;
    a.num_pages = p->num_pages;
    a.qheads = (int)hq;
    if (rope) a.rope = *rope;
    const int rot = a.rope.rot_dim;
    const int layout = a.rope.interleaved ? (rot % 8 ? 2 : 1) : (rot % 16 ? 2 : 0);
    const int per = layout == 0 ? 16 - rot / 16 : 16;
    const long long units = (hq + p->Hkv) * per + (long long)p->Hkv * 16;
    // one CTA per token when the tokens fill the GPU; few tokens are split so that a thread has
    // one unit (a decode step is latency: the loads of one token go out at once)
    const int threads = units <= 128 ? 128 : 256;
    const long long all = (units + threads - 1) / threads;
    const unsigned split = (unsigned)std::min(std::max(1LL, std::min(all, 4LL * di->sms / p->N)), 65535LL);
    const void* fn = layout == 0 ? (const void*)append_kernel<0>
                   : layout == 1 ? (const void*)append_kernel<1> : (const void*)append_kernel<2>;
    void* args[] = {&a};
    CKL_CUDA_TRY(launch(fn, dim3((unsigned)p->N, split), dim3(threads), 0, (cudaStream_t)stream, args, true));
    return CKL_OK;
}

}  // extern "C"
