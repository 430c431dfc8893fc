// cache_evict.cu -- trimming the paged cache: the attention weight every cached token received
// (ckl_cache_weights), the choice of the tokens to keep (ckl_cache_select) and the move of the
// kept rows to the front, in place (ckl_cache_compact).

#include <algorithm>
#include <climits>
#include <mutex>

#include "tree_common.cuh"

namespace ckl {
namespace evict {

using namespace attn;
using tree::Row;
using tree::Seq;

// ------------------------------------------------------------------ weights
// acc[b][p] += sum over rows r (tokens x heads) of exp(s_rp - lse_r): one pass over K (half the
// bytes of an attention call), bound by HBM for few rows. A warp owns whole pages, all kv heads
// of them, so a token's sum stays in its registers and is added in a fixed order: no atomics,
// no second kernel. S = K Q^T tiles by mma.sync as in the attention; the softmax is already
// normalised by the caller's lse, so there is no running maximum.
constexpr int W_WARPS = 8;
constexpr int W_THREADS = W_WARPS * 32;
constexpr int W_STAGES = 3;                    // K tiles (one page, one head: 4 KB) in flight per warp
constexpr int W_PAGES = 2 * W_WARPS;           // pages of a CTA's chunk, at most
constexpr int W_RING = W_WARPS * W_STAGES * KV_TILE;

struct WArgs {
    tree::Args t;
    const float* lse_in;
    float* acc;
    long long acc_stride;
    float decay;
    int q_tiles;                               // row tiles of 16 that fit in the Q buffer
};

constexpr int w_smem(int q_tiles) { return 1024 + W_RING + q_tiles * (KV_TILE + 16 * 4) + W_WARPS * W_STAGES * 8; }

// grid = (CTAs per sequence, B): a CTA takes chunks of pages blockIdx.x, + gridDim.x, ...
template <bool EXT>
__global__ void __launch_bounds__(W_THREADS) weights_kernel(const __grid_constant__ CUtensorMap tmK, const WArgs w) {
    extern __shared__ uint8_t smem_raw[];
    const tree::Args& a = w.t;
    uint8_t* ring = align_ptr<1024>(smem_raw);
    uint8_t* qs = ring + W_RING;                                          // [q_tiles] swizzled like a page
    float* ls = reinterpret_cast<float*>(qs + (size_t)w.q_tiles * KV_TILE);   // [q_tiles][16] lse, log2
    uint64_t* full = reinterpret_cast<uint64_t*>(ls + w.q_tiles * 16);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < W_WARPS * W_STAGES; i++) mbar_init(&full[i], 1);
        fence_barrier_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const uint64_t deadline = globaltimer() + a.timeout_ns;
    const Seq s(a, blockIdx.y);
    const int npages = (s.len + PAGE - 1) / PAGE;
    if (npages == 0) return;
    if (s.T > a.max_q && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, DEVERR_BOUND);
    const int nrows = min(s.T, a.max_q) * a.G;
    int pos_lo = 0, pos_hi = 0;
    if (a.window > 0) pos_range(a, s, lane, &pos_lo, &pos_hi);
    const int first = nrows > 0 ? tree::first_key(a, s, pos_lo) / PAGE : npages;   // pages before: nobody sees them
    const int cp = min(W_PAGES, max(1, (npages + gridDim.x - 1) / gridDim.x));   // even chunks

    const int tiles = (nrows + 15) / 16;
    const int tb = min(max(tiles, 1), w.q_tiles);              // row tiles per block
    const int hb = max(1, w.q_tiles / max(tiles, 1));          // heads per block (1 when rows are split)
    uint8_t* myring = ring + warp * W_STAGES * KV_TILE;
    uint64_t* myfull = full + warp * W_STAGES;
    const uint64_t pol = policy_evict_first();
    int nload = 0, nuse = 0;                                   // this warp's tiles, since the start
    bool ok = true;

    for (int chunk = blockIdx.x; (long long)chunk * cp < npages; chunk += gridDim.x) {
        const int pg0 = chunk * cp, pg1 = min(npages, pg0 + cp);
        float sum[2][2][2];                                    // [page of this warp][8-key half][key]
#pragma unroll
        for (int i = 0; i < 2; i++) sum[i][0][0] = sum[i][0][1] = sum[i][1][0] = sum[i][1][1] = 0.f;
        // this warp's pages of the chunk that somebody can see: pg0 + warp + 8 i
        int mine[2], ids[2], np = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int pg = pg0 + warp + 8 * i;
            mine[i] = pg;
            ids[i] = pg < pg1 ? __ldg(a.indices + s.page0 + pg) : 0;
            if (pg < pg1) np = i + 1;
        }
        for (int h0 = 0; h0 < a.Hkv; h0 += hb)
            for (int t0 = 0; t0 < tiles; t0 += tb) {
                const int nh = min(hb, a.Hkv - h0), nt = min(tb, tiles - t0);
                // the units of this block: pages x heads, in order; issue the first ones now
                const int units = np * nh;
                auto issue = [&](int u) {
                    const int i = u / nh, h = h0 + u - i * nh, sg = nload % W_STAGES;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&myfull[sg], KV_TILE);
                        tma_load_5d(myring + sg * KV_TILE, &tmK, 0, 0, h, 0, ids[i], &myfull[sg], pol);
                    }
                    nload++;
                };
                // pages that nobody sees keep a sum of 0
                const int u0 = np > 0 && mine[0] < first ? (np > 1 && mine[1] < first ? units : nh) : 0;
                int next = u0;
                for (; ok && next < units && next < u0 + W_STAGES; next++) issue(next);
                __syncthreads();                               // the previous block's Q is done with
                for (int c = threadIdx.x; c < nh * nt * 256; c += W_THREADS) {
                    const int tile = c >> 8, r = (c >> 4) & 15, cd = c & 15;
                    const int h = tile / nt, rr = (t0 + tile - h * nt) * 16 + r;
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    const size_t row = (size_t)(s.q0 + rr / a.G) * a.Hq + (h0 + h) * a.G + rr % a.G;
                    if (rr < nrows) v = __ldg(reinterpret_cast<const uint4*>(a.q + row * D) + cd);
                    *reinterpret_cast<uint4*>(qs + tile * KV_TILE + tile_off(r, cd)) = v;
                    if (cd == 0) {
                        // padding rows and rows that saw nothing: exp2(s - inf) = 0
                        const float l = rr < nrows ? w.lse_in[row] : -INFINITY;
                        ls[tile * 16 + r] = l == -INFINITY ? INFINITY : l * LOG2E;
                    }
                }
                __syncthreads();
                for (int u = u0; u < units && ok; u++) {
                    const int i = u / nh, hh = u - i * nh, sg = nuse % W_STAGES;
                    ok = __all_sync(0xffffffffu, mbar_wait(&myfull[sg], (nuse / W_STAGES) & 1, deadline, a.err));
                    if (ok) {
                        nuse++;
                        const uint32_t kb = smem_u32(myring + sg * KV_TILE);
                        const int k_key = (lane & 7) + ((lane >> 4) << 3), k_hi = (lane >> 3) & 1;
                        const int q_row = (lane & 7) + (((lane >> 3) & 1) << 3), q_hi = lane >> 4;
                        uint32_t kf[8][4];
#pragma unroll
                        for (int kk = 0; kk < 8; kk++)
                            ldmatrix_x4(kb + tile_off(k_key, 2 * kk + k_hi), kf[kk][0], kf[kk][1], kf[kk][2], kf[kk][3]);
                        const int g = lane >> 2, t = lane & 3;
                        const int kbase = mine[i] * PAGE;
                        const bool whole = kbase + PAGE <= s.ctx &&
                                           (a.window <= 0 || (long long)pos_hi - kbase < a.window);
                        float add[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
                        for (int n = 0; n < nt; n++) {
                            const int tile = hh * nt + n;
                            const uint32_t qb = smem_u32(qs + tile * KV_TILE);
                            float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                            for (int kk = 0; kk < 8; kk++) {
                                uint32_t a0, a1, a2, a3;
                                ldmatrix_x4(qb + tile_off(q_row, 2 * kk + q_hi), a0, a1, a2, a3);
                                mma_16816(sc[0], a0, a1, a2, a3, kf[kk][0], kf[kk][1]);
                                mma_16816(sc[1], a0, a1, a2, a3, kf[kk][2], kf[kk][3]);
                            }
#pragma unroll
                            for (int r = 0; r < 2; r++) {
                                const float l2 = ls[tile * 16 + 8 * r + g];
                                Row row;
                                if ((EXT && a.slopes) || !whole)
                                    row.set(a, s, (t0 + n) * 16 + 8 * r + g, nrows, h0 + hh);
#pragma unroll
                                for (int h = 0; h < 2; h++)
#pragma unroll
                                    for (int c = 0; c < 2; c++) {
                                        const int p = kbase + 8 * h + 2 * t + c;
                                        float x = tree::score<EXT>(a, sc[h][2 * r + c]);
                                        if (EXT && a.slopes)
                                            x += tree::bias<EXT>(a, row.slope2, row.pos, whole ? p : s.pos(a, p));
                                        if (!whole && (p >= s.len || !row.sees(a, s, p, s.pos(a, p)))) x = -INFINITY;
                                        add[h][c] += ex2(x - l2);
                                    }
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int c = 0; c < 2; c++) {
                                if (i == 0) sum[0][h][c] += add[h][c];
                                else sum[1][h][c] += add[h][c];
                            }
                    }
                    __syncwarp();                              // every lane has read the stage
                    if (next < units && ok) {
                        issue(next);
                        next++;
                    }
                }
                if (!ok) {
                    // copies still in flight must land before the CTA exits
                    for (; nuse < nload; nuse++)
                        if (lane == 0) mbar_wait(&myfull[nuse % W_STAGES], (nuse / W_STAGES) & 1, deadline, a.err);
                }
            }
        // the eight lanes of a key hold its rows g, g+8 of every tile
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float x = sum[i][h][c];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    const int p = mine[i] * PAGE + 8 * h + 2 * (lane & 3) + c;
                    if (lane < 4 && mine[i] < pg1 && p < s.len && p < w.acc_stride) {
                        float* dst = w.acc + blockIdx.y * w.acc_stride + p;
                        *dst = w.decay != 0.f ? fmaf(w.decay, *dst, x) : x;
                    }
                }
    }
}

// ------------------------------------------------------------------ select
// Order of the weights as unsigned integers: NaN lowest, then -inf .. +inf, -0 = +0.
__device__ __forceinline__ uint32_t rank_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int S_THREADS = 1024;
constexpr int S_WARPS = S_THREADS / 32;
constexpr int S_BINS = 2048;               // radix passes over 11, 11 and 10 bits
constexpr int S_MAX_KEYS = 47 << 10;       // keys of a CTA's slice kept in shared memory, at most
constexpr int S_SLICE = 4096;              // places per CTA that a cluster is sized for

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A 32-bit word of shared memory of CTA `rank` of the cluster, at this CTA's address `p`.
__device__ __forceinline__ int cluster_load(const int* p, int rank) {
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

struct SArgs {
    const float* acc;
    const int* indptr;
    const int* last;
    int* keep_idx;
    int* keep_count;
    long long stride;
    int keep, sink, recent, cluster, max_keys;
};

// Keeps the `want` greatest of a sequence's middle places. A cluster of CTAs (one for short
// sequences) shares the sequence: each loads its slice once, as ordered integers in shared
// memory; three radix passes narrow the threshold, each a histogram per CTA that all CTAs of the
// cluster add up from one another's shared memory; then every warp counts and writes its part of
// the list in order. Bound by latency: per pass one cluster barrier, two block barriers. A pass
// whose bin is taken whole ends the search (the usual case after two passes unless values tie).
// grid = (cluster, B).
__global__ void __launch_bounds__(S_THREADS) select_kernel(const SArgs a) {
    extern __shared__ uint32_t keys[];                       // [max_keys]
    __shared__ int hist[3][S_BINS];
    __shared__ int warp_sum[S_WARPS], warp_eq[S_WARPS];
    __shared__ int s_bin, s_left, s_in;
    __shared__ int total[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int i = tid; i < 3 * S_BINS; i += S_THREADS) (&hist[0][0])[i] = 0;
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y, rank = blockIdx.x;
    int page0;
    const int len = tree::seq_len(a.indptr, a.last, b, &page0);
    int* out = a.keep_idx + (size_t)b * a.keep;
    const int step = a.cluster * S_THREADS, me = rank * S_THREADS + tid;
    if (me == 0) a.keep_count[b] = min(len, a.keep);
    if (len <= a.keep) {                                     // the same for the whole cluster
        for (int i = me; i < a.keep; i += step) out[i] = i < len ? i : -1;
        return;
    }
    const int hi = len - a.recent, mid = hi - a.sink;
    int want = a.keep - a.sink - a.recent;                   // of the places [sink, hi); mid > want
    for (int i = me; i < a.sink; i += step) out[i] = i;
    for (int i = me; i < a.recent; i += step) out[a.keep - a.recent + i] = hi + i;
    if (want == 0) return;
    // this CTA's slice of the middle, a multiple of a warp's 32 places per warp
    const int slice = ((mid + a.cluster - 1) / a.cluster + 31) & ~31;
    const int beg = a.sink + min(mid, rank * slice), n = a.sink + min(mid, (rank + 1) * slice) - beg;
    const float* row = a.acc + b * a.stride + beg;
    const long long have = a.stride - beg;                   // places of the row that exist
    auto load = [&](int i) { return i < have ? rank_key(__ldg(row + i)) : 0u; };
    const bool held = n <= a.max_keys;                       // longer slices are read again from L2
    if (held)
        for (int i = tid; i < n; i += S_THREADS) keys[i] = load(i);
    auto key = [&](int i) { return held ? keys[i] : load(i); };
    __syncthreads();

    uint32_t prefix = 0, known = 0;
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t field = pass == 2 ? 1023u : 2047u;
        int* h = hist[pass];
        for (int i = tid; i < n; i += S_THREADS) {
            const uint32_t k = key(i);
            if ((k & known) == prefix) atomicAdd(&h[(k >> shift) & field], 1);
        }
        if (a.cluster > 1) cluster_sync();
        else __syncthreads();
        // bins from the greatest down, two per thread
        const int bin = S_BINS - 1 - 2 * tid;
        int c0 = 0, c1 = 0;
        if (a.cluster > 1) {
            for (int r = 0; r < a.cluster; r++) {
                c0 += cluster_load(&h[bin], r);
                c1 += cluster_load(&h[bin - 1], r);
            }
        } else {
            c0 = h[bin];
            c1 = h[bin - 1];
        }
        int x = c0 + c1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        int before = lane < warp ? warp_sum[lane] : 0;
        before = __reduce_add_sync(0xffffffffu, before);
        const int up0 = before + x - c0 - c1, up1 = up0 + c0;     // keys above each bin
        if (up0 < want && want <= up1) { s_bin = bin; s_left = want - up0; s_in = c0; }
        if (up1 < want && want <= up1 + c1) { s_bin = bin - 1; s_left = want - up1; s_in = c1; }
        __syncthreads();
        prefix |= (uint32_t)s_bin << shift;
        known |= field << shift;
        want = s_left;
        if (s_in == want) break;                             // the whole bin is kept
    }
    // keys above `prefix` in the known bits are kept, and the first `want` of those equal to it
    const int per = ((n + S_WARPS - 1) / S_WARPS + 31) & ~31;
    const int w0 = min(n, warp * per), w1 = min(n, w0 + per);
    int gt = 0, eq = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t k = key(i) & known;
        gt += k > prefix;
        eq += k == prefix;
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        warp_sum[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    int g = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
    int e = __reduce_add_sync(0xffffffffu, lane < warp ? warp_eq[lane] : 0);
    if (a.cluster > 1) {
        if (warp == S_WARPS - 1 && lane == 0) {
            total[0] = g + gt;
            total[1] = e + eq;
        }
        cluster_sync();
        for (int r = 0; r < rank; r++) {
            g += cluster_load(&total[0], r);
            e += cluster_load(&total[1], r);
        }
        cluster_sync();                                      // nobody leaves while it is read
    }
    out += a.sink;
    for (int base = w0; base < w1; base += 32) {
        const int i = base + lane;
        const uint32_t k = i < w1 ? key(i) & known : 0u;
        const bool is_gt = i < w1 && k > prefix, is_eq = i < w1 && k == prefix;
        const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
        const uint32_t below = (1u << lane) - 1u;
        const int ei = e + __popc(be & below);
        if (is_gt || (is_eq && ei < want)) out[g + __popc(bg & below) + min(ei, want)] = beg + i;
        g += __popc(bg);
        e += __popc(be);
    }
}

// ------------------------------------------------------------------ compact
constexpr int C_THREADS = 256;
constexpr int C_U = 8;           // 16-byte pieces per thread and tile

struct CArgs {
    uint4* k;
    uint4* v;
    const int* indptr;
    const int* indices;
    const int* last;
    const int* idx;
    const int* count;
    const int* start;
    float* acc;
    int* new_len;
    unsigned* err;
    long long acc_stride;
    int Hkv, num_pages, keep_stride;
    int pieces;                  // 16-byte pieces of a row per CTA: a power of two, at most 16
};

// In place and in order: rows move towards the front (keep[i] >= start + i, ascending), so the
// rows that a tile of the list overwrites are read by this tile or an earlier one only. A CTA
// owns a column of the rows -- `pieces` 16-byte pieces of one head -- for all of a sequence's
// list: per tile every thread loads, the CTA meets, and every thread stores; the next tile's
// loads need not wait for the stores. No CTA waits for another.
// grid = (Hkv * 16 / pieces (+ 1 for acc and the lengths), B, 2).
__global__ void __launch_bounds__(C_THREADS) compact_kernel(const CArgs a) {
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y, tid = threadIdx.x;
    int page0;
    const int len = tree::seq_len(a.indptr, a.last, b, &page0);
    const int start = a.start ? __ldg(a.start + b) : 0;
    const int n = max(0, min(__ldg(a.count + b), a.keep_stride));
    const int* idx = a.idx + (size_t)b * a.keep_stride;
    // the list ascends strictly from `start` and ends below len; i0 = its first moved entry
    // (entries before it are in their places already: idx[i] - i never falls)
    int bad = start < 0 || start > len, i0 = n;
    for (int i = tid; i < n; i += C_THREADS) {
        const int x = __ldg(idx + i), before = i ? __ldg(idx + i - 1) : start - 1;
        bad |= x <= before || x >= len;
        if (x != start + i) i0 = min(i0, i);
    }
    __shared__ int s_first;
    if (tid == 0) s_first = n;
    bad = __syncthreads_or(bad);
    const bool side = blockIdx.x == gridDim.x - 1;           // acc and the lengths
    if (side && blockIdx.z) return;
    if (bad) {
        if (side && tid == 0) {
            atomicOr(a.err, DEVERR_BOUND);
            if (a.new_len) a.new_len[b] = len;
        }
        return;
    }
    if (i0 < n) atomicMin(&s_first, i0);
    __syncthreads();
    i0 = s_first;
    if (side) {
        if (tid == 0 && a.new_len) a.new_len[b] = start + n;
        if (!a.acc) return;
        float* row = a.acc + b * a.acc_stride;
        for (int base = i0; base < n; base += C_THREADS * C_U) {
            float x[C_U];
#pragma unroll
            for (int u = 0; u < C_U; u++) {
                const int i = base + u * C_THREADS + tid;
                const int src = i < n ? __ldg(idx + i) : 0;
                x[u] = i < n && src < a.acc_stride ? row[src] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < C_U; u++) {
                const int i = base + u * C_THREADS + tid;
                if (i < n && start + i < a.acc_stride) row[start + i] = x[u];
            }
        }
        __syncthreads();
        for (long long p = (long long)start + n + tid; p < len && p < a.acc_stride; p += C_THREADS) row[p] = 0.f;
        return;
    }
    uint4* cache = blockIdx.z ? a.v : a.k;
    const int per_head = 16 / a.pieces;
    const int head = blockIdx.x / per_head, col = (blockIdx.x - head * per_head) * a.pieces;
    const int rows = C_THREADS / a.pieces, r = tid / a.pieces, c = col + tid % a.pieces;
    auto at = [&](int p) -> uint4* {                          // nullptr: a page outside the cache
        const int page = __ldg(a.indices + page0 + p / PAGE);
        if (page < 0 || page >= a.num_pages) return nullptr;
        return cache + (((size_t)page * PAGE + p % PAGE) * a.Hkv + head) * 16 + c;
    };
    for (int base = i0; base < n; base += rows * C_U) {
        uint4 x[C_U];
#pragma unroll
        for (int u = 0; u < C_U; u++) {
            const int i = base + u * rows + r;
            const uint4* src = i < n ? at(__ldg(idx + i)) : nullptr;
            x[u] = src ? *src : make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < C_U; u++) {
            const int i = base + u * rows + r;
            uint4* dst = i < n ? at(start + i) : nullptr;
            if (dst) *dst = x[u];
        }
    }
}

struct Setup {
    ckl_status st = CKL_OK;
};
constexpr int Q_SMALL = 3, Q_BIG = 28;         // 16-row tiles of Q per block: two CTAs an SM, or one
const Setup* setup(const DeviceInfo* di) {
    static Setup ks[64];
    static std::once_flag once[64];
    std::call_once(once[di->device], [di] {
        cudaError_t e = cudaFuncSetAttribute(weights_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, w_smem(Q_BIG));
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(weights_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, w_smem(Q_BIG));
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S_MAX_KEYS * 4);
        if (e != cudaSuccess) ks[di->device].st = cuda_status(e, "cache kernels setup");
    });
    return &ks[di->device];
}

}  // namespace evict
}  // namespace ckl

using namespace ckl;
using namespace ckl::evict;

extern "C" {

ckl_status ckl_cache_weights(const ckl_tree_params* p, const float* lse, float* acc, long long acc_stride,
                             float decay, void* stream) {
    ckl_status st = tree::check_params(p, "cache_weights");
    if (st != CKL_OK) return st;
    if (acc_stride <= 0) return fail(CKL_INVALID_ARG, "cache_weights: acc_stride=%lld", acc_stride);
    if (!(decay >= 0.f && decay <= 1.f)) return fail(CKL_INVALID_ARG, "cache_weights: decay outside [0, 1]");
    if (p->B == 0) return CKL_OK;
    if (p->N == 0) return fail(CKL_INVALID_ARG, "cache_weights: no tokens");
    if (!lse || !acc) return fail(CKL_INVALID_ARG, "cache_weights: lse/acc are NULL");
    const DeviceInfo* di = device_info();
    if (!di) return CKL_CUDA_ERROR;
    const Setup* ks = setup(di);
    if (ks->st != CKL_OK) return ks->st;
    WArgs w{};
    st = tree::fill_args(p, &w.t);
    if (st != CKL_OK) return st;
    w.lse_in = lse;
    w.acc = acc;
    w.acc_stride = acc_stride;
    w.decay = decay;
    // rows of one head in one small Q block: two CTAs per SM; more rows: one CTA with a large
    // block, so that K is read again as seldom as can be
    const bool small = (long long)p->max_q * w.t.G <= 16 * Q_SMALL;
    w.q_tiles = small ? Q_SMALL : Q_BIG;
    const long long chunks = (acc_stride + PAGE - 1) / PAGE;
    const unsigned gx = (unsigned)std::max(1LL, std::min(chunks, (long long)di->sms * (small ? 2 : 1) / p->B));
    CUtensorMap tmK, tmV;
    st = encode_page_maps(p->k_cache, p->v_cache, p->Hkv, p->num_pages, &tmK, &tmV);
    if (st != CKL_OK) return st;
    void* args[] = {&tmK, &w};
    const bool ext = p->softcap > 0.f || p->slopes;
    CKL_CUDA_TRY(launch(ext ? (const void*)weights_kernel<true> : (const void*)weights_kernel<false>,
                        dim3(gx, (unsigned)p->B), dim3(W_THREADS), w_smem(w.q_tiles), (cudaStream_t)stream, args, true));
    return CKL_OK;
}

ckl_status ckl_cache_select(const float* acc, long long acc_stride, const int* kv_indptr,
                            const int* kv_last_page_len, int B, int keep, int sink, int recent,
                            int* keep_idx, int* keep_count, void* stream) {
    if (B < 0 || keep <= 0 || sink < 0 || recent < 0 || (long long)sink + recent > keep || acc_stride <= 0)
        return fail(CKL_INVALID_ARG, "cache_select: B=%d keep=%d sink=%d recent=%d acc_stride=%lld", B, keep, sink,
                    recent, acc_stride);
    if (B == 0) return CKL_OK;
    if (!acc || !kv_indptr || !kv_last_page_len || !keep_idx || !keep_count)
        return fail(CKL_INVALID_ARG, "cache_select: NULL tensor pointer");
    if (B > 65535) return fail(CKL_UNSUPPORTED_SHAPE, "cache_select: B=%d (at most 65535)", B);
    const DeviceInfo* di = device_info();
    if (!di) return CKL_CUDA_ERROR;
    const Setup* ks = setup(di);
    if (ks->st != CKL_OK) return ks->st;
    // a CTA per S_SLICE places, as long as the clusters of all sequences fit the GPU at once
    int cluster = 1;
    while (cluster < 8 && (long long)cluster * S_SLICE < acc_stride && (long long)B * cluster * 2 <= di->sms) cluster *= 2;
    const long long slice = ((acc_stride + cluster - 1) / cluster + 31) & ~31LL;
    SArgs a{acc, kv_indptr, kv_last_page_len, keep_idx, keep_count, acc_stride, keep, sink, recent, cluster,
            (int)std::min(slice, (long long)S_MAX_KEYS)};
    void* args[] = {&a};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster, (unsigned)B);
    cfg.blockDim = dim3(S_THREADS);
    cfg.dynamicSmemBytes = (size_t)a.max_keys * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CKL_CUDA_TRY(cudaLaunchKernelExC(&cfg, (const void*)select_kernel, args));
    return CKL_OK;
}

ckl_status ckl_cache_compact(void* k_cache, void* v_cache, const int* kv_indptr, const int* kv_indices,
                             const int* kv_last_page_len, int B, int Hkv, int num_pages,
                             const int* keep_idx, int keep_stride, const int* keep_count,
                             const int* dst_start, float* acc, long long acc_stride, int* new_len,
                             void* stream) {
    if (B < 0 || Hkv <= 0 || num_pages <= 0 || keep_stride <= 0 || (acc && acc_stride <= 0))
        return fail(CKL_INVALID_ARG, "cache_compact: B=%d Hkv=%d num_pages=%d keep_stride=%d acc_stride=%lld", B, Hkv,
                    num_pages, keep_stride, acc_stride);
    if (B > 65535 || Hkv > 65535) return fail(CKL_UNSUPPORTED_SHAPE, "cache_compact: B=%d Hkv=%d (at most 65535)", B, Hkv);
    if (B == 0) return CKL_OK;
    if (!k_cache || !v_cache || !kv_indptr || !kv_indices || !kv_last_page_len || !keep_idx || !keep_count)
        return fail(CKL_INVALID_ARG, "cache_compact: NULL tensor pointer");
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15)
        return fail(CKL_INVALID_ARG, "cache_compact: k_cache and v_cache must be 16-byte aligned");
    if (k_cache == v_cache) return fail(CKL_INVALID_ARG, "cache_compact: k_cache and v_cache are the same");
    const DeviceInfo* di = device_info();
    if (!di) return CKL_CUDA_ERROR;
    CArgs a{};
    a.k = static_cast<uint4*>(k_cache);
    a.v = static_cast<uint4*>(v_cache);
    a.indptr = kv_indptr;
    a.indices = kv_indices;
    a.last = kv_last_page_len;
    a.idx = keep_idx;
    a.count = keep_count;
    a.start = dst_start;
    a.acc = acc;
    a.new_len = new_len;
    a.err = di->err_word;
    a.acc_stride = acc_stride;
    a.Hkv = Hkv;
    a.num_pages = num_pages;
    a.keep_stride = keep_stride;
    // whole heads (256 bytes) per CTA, halved while the columns leave SMs idle, down to 64
    // bytes: two 32-byte sectors, the least that HBM serves
    a.pieces = 16;
    while (a.pieces > 4 && (long long)B * Hkv * 2 * (16 / a.pieces) < di->sms) a.pieces /= 2;
    void* args[] = {&a};
    CKL_CUDA_TRY(launch((const void*)compact_kernel, dim3((unsigned)(Hkv * (16 / a.pieces) + 1), (unsigned)B, 2),
                        dim3(C_THREADS), 0, (cudaStream_t)stream, args, true));
    return CKL_OK;
}

}  // extern "C"
