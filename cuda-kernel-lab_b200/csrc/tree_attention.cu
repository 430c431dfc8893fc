// tree_attention.cu -- attention of drafted tokens (a tree, a chain, or one token) over the
// paged cache, with capped scores, a distance bias and a sliding window.
//
// The T drafted tokens x G query heads that share a kv head are stacked into rows, so K and V
// are read once for all of them. Per (sequence, kv head, chunk of keys) a CTA streams pages
// through a TMA ring, computes S = Q K^T, an online softmax in the log2 domain and O += P V;
// split sequences are joined by their log-sum-exps in a second kernel.
//
//   up to 16 rows (few drafts, single-token decode): mma.sync, four warps that take pages in
//   turn (`rows_kernel` here);
//   more rows: tcgen05 on 128-row tiles (tree_tile.cu).

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <mutex>

#include "tree_tile.cuh"

namespace ckl {
namespace tree {

constexpr int CONSUMERS = 4;
constexpr int THREADS = (CONSUMERS + 1) * 32;
constexpr int STAGES = 8;
static_assert(STAGES % CONSUMERS == 0, "every stage must belong to one consumer warp");
constexpr int RING_BYTES = STAGES * STAGE_BYTES;

constexpr int R = 16;                              // rows of the MMA tile
constexpr int ROWS_SMEM = 1024 + RING_BYTES + KV_TILE + 2 * STAGES * 8 + 2 * CONSUMERS * R * 4;

// The keys of this CTA: [beg, end), beg a multiple of 16.
struct Keys {
    int beg, end;
    __device__ __forceinline__ Keys(const Args& a, const Seq& s, int first, int chunk) {
        const long long b = first + (long long)chunk * a.chunk_tokens;
        beg = b < s.len ? (int)b : s.len;
        // the last chunk takes what is left: a sequence longer than planned for loses no key
        end = chunk + 1 == a.num_chunks ? s.len : (int)min((long long)s.len, b + a.chunk_tokens);
    }
};

// ------------------------------------------------------------------ up to 16 rows: mma.sync
// Online-softmax state of one warp for a tile of 16 rows. Lane (g = lane/4, t = lane%4) holds rows
// g and g+8, dims 8j + 2t + {0,1} of o[j], and the fragments of Q.
// KIND: plain scores (0), a distance bias (1), a cap (2), with or without a bias.
template <int KIND>
struct State {
    float o[16][4];
    float m[2], l[2];
    Row row[2];
    uint32_t q[8][4];

    __device__ __forceinline__ void reset(uint32_t qb, int lane) {
        // A fragments of Q: matrices rows 0-7 / 8-15 x dims 16kk.. / +8
        const int q_row = (lane & 7) + (((lane >> 3) & 1) << 3), q_hi = lane >> 4;
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
            ldmatrix_x4(qb + tile_off(q_row, 2 * kk + q_hi), q[kk][0], q[kk][1], q[kk][2], q[kk][3]);
#pragma unroll
        for (int j = 0; j < 16; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // Attend the page at shared address kb (K; V at kb + KV_TILE) that holds cached tokens
    // [kbase, kbase + 16). `whole`: every row sees every key of it. A warp has its page to itself
    // and nothing to overlap it with but its own instructions: fragments are loaded well ahead of
    // the products, S is summed in two chains, one vote covers both rows' maxima, and branches stay
    // out of the loops over scores (a page took 1.45 us with the loops written plainly).
    __device__ __forceinline__ void page(const Args& a, const Seq& s, uint32_t kb, int kbase, bool whole, int lane) {
        const int t = lane & 3;
        const int k_key = (lane & 7) + ((lane >> 4) << 3), k_hi = (lane >> 3) & 1;
        const int v_key = (lane & 7) + (((lane >> 3) & 1) << 3), v_hi = lane >> 4;
        const uint32_t vb = kb + KV_TILE;
        float sc[2][4], sd[2][4];
#pragma unroll
        for (int c = 0; c < 8; c++) sc[c >> 2][c & 3] = sd[c >> 2][c & 3] = 0.f;
        {
            uint32_t kf[8][4];
#pragma unroll
            for (int i = 0; i < 8; i++)
                ldmatrix_x4(kb + tile_off(k_key, 2 * i + k_hi), kf[i][0], kf[i][1], kf[i][2], kf[i][3]);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                mma_16816(sc[0], q[i][0], q[i][1], q[i][2], q[i][3], kf[i][0], kf[i][1]);
                mma_16816(sc[1], q[i][0], q[i][1], q[i][2], q[i][3], kf[i][2], kf[i][3]);
                mma_16816(sd[0], q[i + 1][0], q[i + 1][1], q[i + 1][2], q[i + 1][3], kf[i + 1][0], kf[i + 1][1]);
                mma_16816(sd[1], q[i + 1][0], q[i + 1][1], q[i + 1][2], q[i + 1][3], kf[i + 1][2], kf[i + 1][3]);
            }
        }
        uint32_t vf[8][4];
#pragma unroll
        for (int i = 0; i < 8; i++)
            ldmatrix_x4_trans(vb + tile_off(v_key, 2 * i + v_hi), vf[i][0], vf[i][1], vf[i][2], vf[i][3]);
#pragma unroll
        for (int c = 0; c < 8; c++) sc[c >> 2][c & 3] += sd[c >> 2][c & 3];
        if (KIND == 2) {
            cap_all(a, reinterpret_cast<float (&)[8]>(sc));
        } else {
#pragma unroll
            for (int c = 0; c < 8; c++) sc[c >> 2][c & 3] *= a.scale_log2;
        }
        if (KIND == 1 || (KIND == 2 && a.slopes)) {
            int kp[4] = {kbase + 2 * t, kbase + 2 * t + 1, kbase + 8 + 2 * t, kbase + 9 + 2 * t};
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; i++) kp[i] = s.pos(a, kp[i]);
            }
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) sc[i >> 1][2 * r + (i & 1)] += bias<true>(a, row[r].slope2, row[r].pos, kp[i]);
        }
        bool odd = false;                                // masked V rows hold inf or NaN
        if (!whole) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int p = kbase + 8 * h + 2 * t + (c & 1);
                    if (p >= s.len || !row[c >> 1].sees(a, s, p, s.pos(a, p))) sc[h][c] = -INFINITY;
                }
            // 0 * inf is NaN in the product: rows behind the sequence are zeroed, and where another
            // row is not finite the page is summed row by row below
            const int left = s.len - kbase;
            auto keep = [&](int k) { return (k < left ? 0xffffu : 0u) | (k + 1 < left ? 0xffff0000u : 0u); };
            const uint32_t vm0 = keep(2 * t), vm1 = keep(8 + 2 * t);
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                vf[i][0] &= vm0;
                vf[i][1] &= vm1;
                vf[i][2] &= vm0;
                vf[i][3] &= vm1;
                bad |= not_finite(vf[i][0]) | not_finite(vf[i][1]) | not_finite(vf[i][2]) | not_finite(vf[i][3]);
            }
            odd = __any_sync(0xffffffffu, bad != 0);
        }
        float mx[2];
#pragma unroll
        for (int r = 0; r < 2; r++)
            mx[r] = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
#pragma unroll
        for (int w = 1; w <= 2; w <<= 1)
#pragma unroll
            for (int r = 0; r < 2; r++) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], w));
        mx[0] -= P_LIFT;
        mx[1] -= P_LIFT;
        if (__any_sync(0xffffffffu, mx[0] > m[0] + RESCALE_THRESHOLD || mx[1] > m[1] + RESCALE_THRESHOLD)) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float mn = fmaxf(m[r], mx[r]);
                const float cf = mn == -INFINITY ? 1.f : ex2(m[r] - mn);
                m[r] = mn;
                l[r] *= cf;
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    o[j][2 * r] *= cf;
                    o[j][2 * r + 1] *= cf;
                }
            }
        }
        uint32_t pa[4];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const float ms = m[r] == -INFINITY ? 0.f : m[r];     // a row that saw nothing yet
            float p[2][2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                p[h][0] = ex2(sc[h][2 * r] - ms);
                p[h][1] = ex2(sc[h][2 * r + 1] - ms);
            }
            l[r] += (p[0][0] + p[0][1]) + (p[1][0] + p[1][1]);
            // l sums the unrounded weights
            pa[r] = pack_half2(p[0][0], p[0][1]);
            pa[2 + r] = pack_half2(p[1][0], p[1][1]);
        }
        if (odd) {
            by_row(s, sc, kb, kbase, lane);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            mma_16816(o[2 * i], pa[0], pa[1], pa[2], pa[3], vf[i][0], vf[i][1]);
            mma_16816(o[2 * i + 1], pa[0], pa[1], pa[2], pa[3], vf[i][2], vf[i][3]);
        }
    }

    // O += P V of a masked page whose V is not finite everywhere, key by key: a key that a row
    // does not see (score -inf) is skipped for it.
    __device__ __forceinline__ void by_row(const Seq& s, const float (&sc)[2][4], uint32_t kb, int kbase, int lane) {
        const int t = lane & 3;
#pragma unroll 1
        for (int k = 0; k < PAGE && kbase + k < s.len; k++) {
            const int src = (lane & ~3) | ((k & 7) >> 1);
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int c = 2 * r;
                const float mine = k < 8 ? ((k & 1) ? sc[0][c + 1] : sc[0][c]) : ((k & 1) ? sc[1][c + 1] : sc[1][c]);
                const float x = __shfl_sync(0xffffffffu, mine, src);
                if (x == -INFINITY) continue;
                const float p = ex2(x - m[r]);
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    uint32_t v;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(kb + KV_TILE + tile_off(k, j) + 4 * t));
                    const __half2 hv = *reinterpret_cast<__half2*>(&v);
                    o[j][c] = fmaf(p, __low2float(hv), o[j][c]);
                    o[j][c + 1] = fmaf(p, __high2float(hv), o[j][c + 1]);
                }
            }
        }
    }

    static __device__ __forceinline__ uint32_t not_finite(uint32_t h2) {
        return ((h2 & 0x7c00u) == 0x7c00u) | ((h2 & 0x7c000000u) == 0x7c000000u);
    }
};

// Bound by HBM for many sequences: 64 with a window of 2000 keys over 8 kv heads, one token each, 85-97
// us by run for 483 MB, the last wave of CTAs not full; by latency for few (one token over 1 x 1000 keys:
// 10.4 us with the merge). grid = (B * Hkv, num_chunks).
template <int KIND>
__global__ void __launch_bounds__(THREADS, 2)
rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = align_ptr<1024>(smem_raw);
    uint8_t* qs = ring + RING_BYTES;                                    // swizzled like a page
    uint64_t* full = reinterpret_cast<uint64_t*>(qs + KV_TILE);
    uint64_t* empty = full + STAGES;
    float* m_red = reinterpret_cast<float*>(empty + STAGES);            // [CONSUMERS][R]
    float* l_red = m_red + CONSUMERS * R;

    const int b = blockIdx.x / a.Hkv, kvh = blockIdx.x - b * a.Hkv, chunk = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        fence_barrier_init();
    }
    if (warp == CONSUMERS && lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const Seq s(a, b);
    if (s.T > a.max_q && chunk == 0 && threadIdx.x == 0) atomicOr(a.err, DEVERR_BOUND);
    const int nrows = min(s.T, a.max_q) * a.G;
    if (nrows == 0) return;                                             // the whole CTA
    int pos_lo = 0, pos_hi = 0;
    if (a.window > 0) pos_range(a, s, lane, &pos_lo, &pos_hi);
    const Keys keys(a, s, first_key(a, s, pos_lo), chunk);
    const int p0 = keys.beg / PAGE;
    const int npg = keys.end > keys.beg ? (keys.end - keys.beg + PAGE - 1) / PAGE : 0;

    State<KIND> st;
    const int g = lane >> 2, t = lane & 3;
    if (warp == CONSUMERS) {
        const uint64_t pol = policy_evict_first();
        int ok = 1, issued = 0;
        for (int base = 0; base < npg && ok; base += 32) {
            const int cnt = min(32, npg - base);
            const int my_page = lane < cnt ? __ldg(a.indices + s.page0 + p0 + base + lane) : 0;
            for (int j = 0; j < cnt; j++) {
                const int page = __shfl_sync(0xffffffffu, my_page, j);
                if (elect_one()) {
                    const int i = base + j, sg = i % STAGES;
                    if (i >= STAGES) ok = mbar_wait_for(&empty[sg], ((i / STAGES) - 1) & 1, a.timeout_ns, a.err);
                    if (ok) {
                        mbar_arrive_expect_tx(&full[sg], STAGE_BYTES);
                        load_page(ring + sg * STAGE_BYTES, &tmK, &tmV, kvh, page, &full[sg], pol);
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                issued = base + j + 1;
            }
        }
        // every issued copy must land before the CTA reuses the ring or exits
        if (lane == 0)
            for (int sg = 0; sg < STAGES && sg < issued; sg++) {
                const int last = sg + ((issued - 1 - sg) / STAGES) * STAGES;
                mbar_wait_for(&full[sg], (last / STAGES) & 1, DRAIN_NS, a.err);
            }
    } else {
        // stage the Q rows (zeros behind the rows in use), 16 chunks of 16 bytes each
        for (int c = threadIdx.x; c < R * 16; c += CONSUMERS * 32) {
            const int rr = c >> 4, cd = c & 15;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (rr < nrows)
                v = __ldg(reinterpret_cast<const uint4*>(
                        a.q + ((size_t)(s.q0 + rr / a.G) * a.Hq + kvh * a.G + rr % a.G) * D) + cd);
            *reinterpret_cast<uint4*>(qs + tile_off(rr, cd)) = v;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS * 32) : "memory");
#pragma unroll
        for (int r = 0; r < 2; r++) st.row[r].set(a, s, 8 * r + g, nrows, kvh);
        st.reset(smem_u32(qs), lane);
        bool ok = true;
        for (int i = warp; i < npg; i += CONSUMERS) {
            const int sg = i % STAGES;
            const bool got = mbar_wait_for(&full[sg], (i / STAGES) & 1, a.timeout_ns, a.err);
            if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
            const int kbase = (p0 + i) * PAGE;
            const bool whole = kbase + PAGE <= s.ctx && (a.window <= 0 || (long long)pos_hi - kbase < a.window);
            st.page(a, s, smem_u32(ring + sg * STAGE_BYTES), kbase, whole, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[sg]);
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            float l = st.l[r];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (t == 0) {
                m_red[warp * R + 8 * r + g] = ok ? st.m[r] : -INFINITY;
                l_red[warp * R + 8 * r + g] = ok ? l : 0.f;
            }
        }
    }
    // all consumers are done with the ring and every copy has landed: it holds the warps' O now
    __syncthreads();
    if (warp < CONSUMERS) {
        float* ost = reinterpret_cast<float*>(ring);   // [CONSUMERS][R][128]
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int j = 0; j < 16; j++)
                *reinterpret_cast<float2*>(ost + ((size_t)warp * R + 8 * r + g) * D + 8 * j + 2 * t) =
                    make_float2(st.o[j][2 * r], st.o[j][2 * r + 1]);
    }
    __syncthreads();
    // join the four warps: 16 threads a row, 8 dims each
    const float* ost = reinterpret_cast<const float*>(ring);
    if (warp == CONSUMERS) return;
#pragma unroll
    for (int i = 0; i < R / 8; i++) {
        const int r = i * 8 + (threadIdx.x >> 4), d = (threadIdx.x & 15) * 4;
        if (r >= nrows) break;
        float M = -INFINITY, L = 0.f, sw[CONSUMERS];
#pragma unroll
        for (int w = 0; w < CONSUMERS; w++) M = fmaxf(M, m_red[w * R + r]);
        if (M == -INFINITY) M = 0.f;             // no key seen (or only NaN scores, which stay NaN)
        float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
        for (int w = 0; w < CONSUMERS; w++) {
            sw[w] = ex2(m_red[w * R + r] - M);
            L += l_red[w * R + r] * sw[w];
        }
#pragma unroll
        for (int w = 0; w < CONSUMERS; w++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float4 v = *reinterpret_cast<const float4*>(ost + ((size_t)w * R + r) * D + 64 * h + d);
                o[h].x += v.x * sw[w];
                o[h].y += v.y * sw[w];
                o[h].z += v.z * sw[w];
                o[h].w += v.w * sw[w];
            }
        const float inv = L != 0.f ? 1.f / L : 0.f;
        const float lse_v = L != 0.f ? (M + lg2(L)) * LN2 : -INFINITY;
        const size_t row = (size_t)(s.q0 + r / a.G) * a.Hq + kvh * a.G + r % a.G;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            o[h].x *= inv;
            o[h].y *= inv;
            o[h].z *= inv;
            o[h].w *= inv;
            if (a.num_chunks == 1)
                *reinterpret_cast<uint2*>(a.out + row * D + 64 * h + d) = make_uint2(pack_half2(o[h].x, o[h].y), pack_half2(o[h].z, o[h].w));
            else if (L != 0.f)                   // a chunk without keys for this row leaves only its
                                                 // lse: the merge skips it
                *reinterpret_cast<float4*>(a.part_o + (row * a.num_chunks + chunk) * D + 64 * h + d) = o[h];
        }
        if (d == 0) {
            if (a.num_chunks == 1) a.lse[row] = lse_v;
            else a.part_lse[row * a.num_chunks + chunk] = lse_v;
        }
    }
}

// ------------------------------------------------------------------ merge
// Joins a row's chunks: m = max lse_c, out = sum e^(lse_c - m) o_c / sum e^(lse_c - m). A row
// gets W warps (slots c = w mod W, summed in warp order): 1 when there are rows enough to fill
// the GPU, 8 when few rows have many slots to walk. grid = (ceil(max_q * Hq * W / 8), B); rows
// of tokens that a sequence does not have are left alone.
template <int W>
__global__ void __launch_bounds__(256) merge_kernel(const Args a) {
    __shared__ float4 s_acc[8][32];
    __shared__ float s_w[8];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q0 = a.q_indptr ? __ldg(a.q_indptr + blockIdx.y) : blockIdx.y;
    int T = a.q_indptr ? __ldg(a.q_indptr + blockIdx.y + 1) - q0 : 1;
    if (q0 < 0 || q0 + T > a.N || T < 0) T = 0;
    const long long r = (long long)blockIdx.x * (8 / W) + warp / W;
    if (r >= (long long)min(T, a.max_q) * a.Hq) return;      // whole rows: all W warps or none
    const size_t row = (size_t)q0 * a.Hq + r;
    const int S = a.num_chunks, w0 = warp % W;
    const float* L = a.part_lse + row * S;
    float m = -INFINITY;
    bool nan = false;
    for (int c = lane; c < S; c += 32) {
        const float x = L[c];
        nan |= x != x;
        m = fmaxf(m, x);
    }
    m = warp_max(m);
    nan = __any_sync(0xffffffffu, nan);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float ws = 0.f;
    if (m != -INFINITY || nan) {
        const float4* po = reinterpret_cast<const float4*>(a.part_o + row * S * D) + lane;
#pragma unroll 4
        for (int c = w0; c < S; c += W) {
            const float x = L[c];
            if (x == -INFINITY) continue;                     // nothing was written there
            const float w = ex2((x - m) * LOG2E);
            const float4 v = po[(size_t)c * (D / 4)];
            ws += w;
            acc.x += w * v.x;
            acc.y += w * v.y;
            acc.z += w * v.z;
            acc.w += w * v.w;
        }
    }
    if (W > 1) {
        s_acc[warp][lane] = acc;
        if (lane == 0) s_w[warp] = ws;
        __syncthreads();
        if (warp != 0) return;
#pragma unroll
        for (int w = 1; w < W; w++) {
            const float4 v = s_acc[w][lane];
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
            ws += s_w[w];
        }
    }
    const float inv = ws != 0.f ? 1.f / ws : 0.f;
    uint2 pk;
    pk.x = pack_half2(acc.x * inv, acc.y * inv);
    pk.y = pack_half2(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>(a.out + row * D)[lane] = pk;
    if (lane == 0) a.lse[row] = ws != 0.f ? m + logf(ws) : -INFINITY;
}

// ------------------------------------------------------------------ ancestor masks
// One thread per drafted token: walks up its parents. Each step goes to a lower index, so the
// walk ends.
__global__ void __launch_bounds__(128)
mask_kernel(const int* parents, const int* q_indptr, const int* indptr, const int* last, int B, int N,
            int words, uint32_t* mask, int* positions) {
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y;
    const int q0 = __ldg(q_indptr + b);
    int T = __ldg(q_indptr + b + 1) - q0;
    if (q0 < 0 || q0 + T > N || T < 0) T = 0;
    int page0;
    const int len = seq_len(indptr, last, b, &page0);
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < T; i += gridDim.x * blockDim.x) {
        uint32_t* row = mask + (size_t)(q0 + i) * words;
        for (int w = 0; w < words; w++) row[w] = 0u;
        int depth = 0;
        for (int j = i;; depth++) {
            if (j < 32 * words) row[j >> 5] |= 1u << (j & 31);
            const int p = __ldg(parents + q0 + j);
            if (p < 0 || p >= j) break;
            j = p;
        }
        if (positions) positions[q0 + i] = len - T + depth;
    }
}

// ------------------------------------------------------------------ host
const void* rows_fn(int kind) {
    return kind == 0 ? (const void*)rows_kernel<0> : kind == 1 ? (const void*)rows_kernel<1> : (const void*)rows_kernel<2>;
}

struct Setup {
    ckl_status st = CKL_OK;
};
const Setup* setup(const DeviceInfo* di) {
    static Setup ks[64];
    static std::once_flag once[64];
    std::call_once(once[di->device], [di] {
        Setup& k = ks[di->device];
        cudaError_t e = cudaSuccess;
        for (int kind = 0; kind < 3 && e == cudaSuccess; kind++)
            e = cudaFuncSetAttribute(rows_fn(kind), cudaFuncAttributeMaxDynamicSharedMemorySize, ROWS_SMEM);
        if (e != cudaSuccess) k.st = cuda_status(e, "tree attention setup");
    });
    return &ks[di->device];
}

ckl_status check_params(const ckl_tree_params* p, const char* who) {
    if (!p) return fail(CKL_INVALID_ARG, "%s: params is NULL", who);
    if (p->B < 0 || p->N < 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv)
        return fail(CKL_INVALID_ARG, "%s: bad counts B=%d N=%d Hq=%d Hkv=%d", who, p->B, p->N, p->Hq, p->Hkv);
    if (p->Hq / p->Hkv > 128)
        return fail(CKL_UNSUPPORTED_SHAPE, "%s: %d query heads per kv head (at most 128)", who, p->Hq / p->Hkv);
    if (p->B == 0 || p->N == 0) return CKL_OK;
    if (!p->q || !p->k_cache || !p->v_cache || !p->kv_indptr || !p->kv_indices || !p->kv_last_page_len)
        return fail(CKL_INVALID_ARG, "%s: NULL tensor pointer", who);
    if (((uintptr_t)p->k_cache | (uintptr_t)p->v_cache | (uintptr_t)p->q) & 15)
        return fail(CKL_INVALID_ARG, "%s: q, k_cache and v_cache must be 16-byte aligned", who);
    if (p->num_pages <= 0) return fail(CKL_INVALID_ARG, "%s: num_pages must be > 0", who);
    if (p->max_q <= 0) return fail(CKL_INVALID_ARG, "%s: max_q=%d must be > 0", who, p->max_q);
    if (!p->q_indptr && (p->N != p->B))
        return fail(CKL_INVALID_ARG, "%s: without q_indptr there is one token per sequence (N=%d, B=%d)", who, p->N, p->B);
    if (p->tree_mask && p->mask_words <= 0)
        return fail(CKL_INVALID_ARG, "%s: mask_words=%d", who, p->mask_words);
    if (p->tree_mask && (long long)p->mask_words * 32 < p->max_q)
        return fail(CKL_INVALID_ARG, "%s: %d mask words do not cover max_q=%d tokens", who, p->mask_words, p->max_q);
    if (p->window < 0) return fail(CKL_INVALID_ARG, "%s: window=%d", who, p->window);
    if (!(p->softcap >= 0.f) || p->softcap > 1e30f) return fail(CKL_INVALID_ARG, "%s: softcap must be >= 0 and finite", who);
    if (!(p->sm_scale > 0.f) || p->sm_scale > 1e30f)
        return fail(CKL_INVALID_ARG, "%s: sm_scale must be positive and finite", who);
    if ((long long)p->B * p->Hkv > 0x7fffffffLL || p->B > 65535 || (long long)p->N * p->Hq > 0x7fffffffLL ||
        (long long)p->max_q * p->Hq > 0x7fffffffLL)
        return fail(CKL_UNSUPPORTED_SHAPE, "%s: too many rows (B at most 65535, N*Hq below 2^31)", who);
    return CKL_OK;
}

ckl_status fill_args(const ckl_tree_params* p, Args* a) {
    const DeviceInfo* di = device_info();
    if (!di) return CKL_CUDA_ERROR;
    *a = Args{};
    a->q = static_cast<const __half*>(p->q);
    a->v = static_cast<const __half*>(p->v_cache);
    a->indptr = p->kv_indptr;
    a->indices = p->kv_indices;
    a->last = p->kv_last_page_len;
    a->q_indptr = p->q_indptr;
    a->mask = p->tree_mask;
    a->positions = p->positions;
    a->slopes = p->slopes;
    a->err = di->err_word;
    a->timeout_ns = spin_timeout_ns();
    a->B = p->B;
    a->N = p->N;
    a->Hq = p->Hq;
    a->Hkv = p->Hkv;
    a->G = p->Hq / p->Hkv;
    a->max_q = p->max_q;
    a->mask_words = p->mask_words;
    a->num_chunks = p->num_chunks;
    a->chunk_tokens = p->chunk_tokens;
    a->window = p->window;
    a->num_pages = p->num_pages;
    a->scale_log2 = p->sm_scale * LOG2E;
    if (p->softcap > 0.f) {
        // finite whatever the cap, so that a product of 0 is a score of 0
        const double k = (double)p->sm_scale / p->softcap;
        auto finite = [](double x) { return (float)std::min(x, (double)FLT_MAX); };
        a->cap_log2 = p->softcap * LOG2E;
        a->cap_in = finite(2.0 * LOG2E * k);
        a->cap_k = finite(k);
        a->cap_lim = finite(CAP_SMALL / k);
        const double poly[4] = {TANH_0, TANH_1, TANH_2, TANH_3};
        double term = a->scale_log2;
        for (int i = 0; i < 4; i++, term *= k * k) {
            const double c = poly[i] * term;
            if (!(std::fabs(c) >= FLT_MIN && std::fabs(c) <= FLT_MAX)) a->cap_lim = -1.f;
            a->cap_poly[i] = (float)c;
        }
    }
    return CKL_OK;
}

ckl_status check_split(const ckl_tree_params* p) {
    if (p->num_chunks <= 0 || p->num_chunks > 65535 || p->chunk_tokens <= 0 || p->chunk_tokens % PAGE)
        return fail(CKL_INVALID_ARG, "tree_attention: num_chunks=%d chunk_tokens=%d (must be > 0, multiple of 16)",
                    p->num_chunks, p->chunk_tokens);
    return CKL_OK;
}

// More rows than an m16 tile holds go to the tcgen05 kernel, which spends a 128-row tile on any
// number. At 24 rows a second m16 tile per warp (32 rows) against it, in us: 1 x 1000 keys 17.9 / 14.6,
// 1 x 4000 17.2 / 20.7, 1 x 30000 45.6 / 41.3, 8 x 4000 54.6 / 40.7, 8 x 16384 167 / 106: the tiles lose
// at one sequence of a few thousand keys, where each CTA has little to do, and gain at the other sizes.
bool use_tiles(long long rows) { return rows > R; }

// CTAs of the tcgen05 kernel: num_chunks for each unit (sequence, kv head, row group), one wave
// at most.
int tile_ctas(const ckl_tree_params* p, int sms) {
    const long long rows = (long long)p->max_q * (p->Hq / p->Hkv), per = 128LL * tile_count(rows);
    return (int)std::min((long long)sms, (long long)p->B * p->Hkv * ((rows + per - 1) / per) * p->num_chunks);
}

size_t part_o_size(const ckl_tree_params* p) {
    return align_up((size_t)p->N * p->Hq * p->num_chunks * D * sizeof(float), 256);
}

}  // namespace tree
}  // namespace ckl

using namespace ckl;
using namespace ckl::tree;

extern "C" {

ckl_status ckl_tree_plan(int G, int B, int Hkv, int max_q, int max_len, int window, int force_chunks,
                         int* num_chunks, int* chunk_tokens) {
    if (!num_chunks || !chunk_tokens || G <= 0 || B <= 0 || Hkv <= 0 || max_q <= 0 || max_len < 0 || window < 0)
        return fail(CKL_INVALID_ARG, "tree_plan: bad arguments");
    if (G > 128) return fail(CKL_UNSUPPORTED_SHAPE, "tree_plan: %d query heads per kv head (at most 128)", G);
    // keys a sequence's tokens can see, rounded out to pages
    long long len = max_len;
    if (window > 0) len = std::min(len, (long long)window + max_q + 2 * PAGE);
    len = std::max(len, 1LL);
    long long chunks, unit_keys = PAGE;
    if (force_chunks > 0) {
        chunks = force_chunks;
    } else {
        const DeviceInfo* di = device_info();
        if (!di) return CKL_CUDA_ERROR;
        const long long rows = (long long)max_q * G;
        const bool tiles = use_tiles(rows);
        const long long per = tiles ? 128LL * tile_count(rows) : R;
        const long long units = (long long)B * Hkv * ((rows + per - 1) / per);
        if (tiles) {
            // One CTA per SM. In blocks of 128 keys: the CTA's share, 2 more for a join, 2 more
            // where the shares do not end with the units (a second segment's start and end). All
            // SMs are taken when the work is long; short work is cut where units divide evenly (at
            // 24 rows, 1 x 1000 keys: 8 x 1 blocks 14.4 us, 4 x 2 16.5 us; 4 x 600 keys: 1 x 5
            // blocks 17.8 us, 3 pieces 21 us; 8 x 8000 keys: 2 pieces 61 us, 148 shares 58.8 us).
            const long long blocks = (len + 127) / 128, most = std::min(di->sms / units, blocks);
            double best = (double)blocks * units / di->sms + 4.0;
            chunks = (di->sms + units - 1) / units;
            for (long long n = 1; n <= std::max(most, 1LL); n++) {
                const double cost = (double)((blocks + n - 1) / n) + (blocks % n ? 2.0 : 0.0) + (n > 1 ? 2.0 : 0.0);
                if (units * n <= di->sms && cost < best) {
                    best = cost;
                    chunks = n;
                }
            }
        } else {
            // two resident CTAs per SM, about one wave; a page per warp at least
            chunks = std::min(std::max(1LL, 2LL * di->sms / units), (len + 4 * PAGE - 1) / (4 * PAGE));
            unit_keys = 4 * PAGE;
        }
    }
    chunks = std::min(chunks, 65535LL);
    const long long tok = (((len + chunks - 1) / chunks) + unit_keys - 1) / unit_keys * unit_keys;
    *chunk_tokens = (int)std::min(tok, (long long)(INT_MAX / PAGE) * PAGE);
    *num_chunks = (int)((len + *chunk_tokens - 1) / *chunk_tokens);
    return CKL_OK;
}

size_t ckl_tree_workspace_size(const ckl_tree_params* p) {
    if (!p || p->N <= 0 || p->B <= 0) return 0;
    if (p->Hq > 0 && p->Hkv > 0 && p->max_q > 0 && p->num_chunks > 0 && use_tiles((long long)p->max_q * (p->Hq / p->Hkv))) {
        const DeviceInfo* di = device_info();
        if (!di) return SIZE_MAX;
        return tile_workspace(tile_ctas(p, di->sms), (long long)p->max_q * (p->Hq / p->Hkv));
    }
    if (p->num_chunks == 1) return 0;
    // shapes the launch would reject: report a size no caller can provide
    if (p->Hq <= 0 || p->num_chunks <= 0 || p->num_chunks > 65535 || (long long)p->N * p->Hq > 0x7fffffffLL)
        return SIZE_MAX;
    return part_o_size(p) + align_up((size_t)p->N * p->Hq * p->num_chunks * sizeof(float), 256);
}

ckl_status ckl_tree_attention(const ckl_tree_params* p, void* out, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream) {
    ckl_status st = check_params(p, "tree_attention");
    if (st != CKL_OK) return st;
    if (p->B == 0 || p->N == 0) return CKL_OK;
    st = check_split(p);
    if (st != CKL_OK) return st;
    if (!out || !lse) return fail(CKL_INVALID_ARG, "tree_attention: out/lse are NULL");
    if ((uintptr_t)out & 15) return fail(CKL_INVALID_ARG, "tree_attention: out must be 16-byte aligned");
    const size_t need = ckl_tree_workspace_size(p);
    if (need) {
        if (!workspace || workspace_bytes < need)
            return fail(CKL_WORKSPACE_TOO_SMALL, "tree_attention needs %zu workspace bytes, got %zu", need,
                        workspace ? workspace_bytes : (size_t)0);
        if ((uintptr_t)workspace & 255)
            return fail(CKL_INVALID_ARG, "tree_attention: workspace must be 256-byte aligned");
    }
    Args a;
    st = fill_args(p, &a);
    if (st != CKL_OK) return st;
    const DeviceInfo* di = device_info();
    const Setup* ks = setup(di);
    if (ks->st != CKL_OK) return ks->st;
    a.out = static_cast<__half*>(out);
    a.lse = lse;
    if (need) {
        a.part_o = static_cast<float*>(workspace);
        a.part_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + part_o_size(p));
    }
    const cudaStream_t s = (cudaStream_t)stream;
    if (use_tiles((long long)p->max_q * (p->Hq / p->Hkv))) return launch_tiles(p, a, workspace, tile_ctas(p, di->sms), s);
    const int kind = p->softcap > 0.f ? 2 : p->slopes ? 1 : 0;
    CUtensorMap tmK, tmV;
    st = encode_page_maps(p->k_cache, p->v_cache, p->Hkv, p->num_pages, &tmK, &tmV);
    if (st != CKL_OK) return st;
    void* args[] = {&tmK, &tmV, &a};
    CKL_CUDA_TRY(launch(rows_fn(kind), dim3((unsigned)(p->B * p->Hkv), (unsigned)p->num_chunks),
                        dim3(THREADS), ROWS_SMEM, s, args, true));
    if (p->num_chunks == 1) return CKL_OK;
    void* margs[] = {&a};
    const long long mrows = (long long)p->max_q * p->Hq;
    if (p->num_chunks >= 16 && mrows * p->B < 4 * di->sms)
        CKL_CUDA_TRY(launch((const void*)merge_kernel<8>, dim3((unsigned)mrows, (unsigned)p->B), dim3(256), 0, s,
                            margs, true));
    else
        CKL_CUDA_TRY(launch((const void*)merge_kernel<1>, dim3((unsigned)((mrows + 7) / 8), (unsigned)p->B),
                            dim3(256), 0, s, margs, true));
    return CKL_OK;
}

ckl_status ckl_tree_mask(const int* parents, const int* q_indptr, const int* kv_indptr,
                         const int* kv_last_page_len, int B, int N, int mask_words, uint32_t* mask,
                         int* positions, void* stream) {
    if (B < 0 || N < 0 || mask_words <= 0) return fail(CKL_INVALID_ARG, "tree_mask: B=%d N=%d mask_words=%d", B, N, mask_words);
    if (B > 65535) return fail(CKL_UNSUPPORTED_SHAPE, "tree_mask: B=%d (at most 65535)", B);
    if (B == 0 || N == 0) return CKL_OK;
    if (!parents || !q_indptr || !kv_indptr || !kv_last_page_len || !mask)
        return fail(CKL_INVALID_ARG, "tree_mask: NULL tensor pointer");
    // a thread walks parents that other threads' results would replace
    const size_t ints = (size_t)B * sizeof(int), rows = (size_t)N * sizeof(int);
    const Span out[] = {{mask, rows * mask_words}, {positions, rows}};
    const Span in[] = {{parents, rows}, {q_indptr, ints + sizeof(int)}, {kv_indptr, ints + sizeof(int)}, {kv_last_page_len, ints}};
    if (overlap(out[0], out[1])) return fail(CKL_INVALID_ARG, "tree_mask: mask and positions overlap");
    for (const Span& o : out)
        for (const Span& i : in)
            if (overlap(o, i)) return fail(CKL_INVALID_ARG, "tree_mask: an output overlaps an input");
    if (!device_info()) return CKL_CUDA_ERROR;
    void* args[] = {&parents, &q_indptr, &kv_indptr, &kv_last_page_len, &B, &N, &mask_words, &mask, &positions};
    const unsigned gx = (unsigned)std::min(std::max(1, ceil_div(N, 128)), 8);
    CKL_CUDA_TRY(launch((const void*)mask_kernel, dim3(gx, (unsigned)B), dim3(128), 0, (cudaStream_t)stream, args, true));
    return CKL_OK;
}

}  // extern "C"
