// cache_evict.cu -- trimming the paged cache: the attention weight every cached token received
// (ckl_cache_weights), the choice of the tokens to keep (ckl_cache_select) and the move of the
// kept rows to the front, in place (ckl_cache_compact).

#include <algorithm>
#include <climits>
#include <mutex>
#include <type_traits>

#include "tree_tile.cuh"

namespace ckl {
namespace evict {

using namespace attn;
using tree::Row;
using tree::Seq;

// ------------------------------------------------------------------ weights
// acc[b][p] += sum over rows r (tokens x heads) of exp(s_rp - lse_r): one pass over K (half the
// bytes of an attention call), bound by HBM for few rows and by the exponentials for many.
//
// S^T = K Q^T on tcgen05 with the keys as M: 128 keys are the lanes of tensor memory and the rows
// of a kv head its columns, so a thread owns a key and its sum over rows and heads stays with it:
// no atomics and no second kernel, and additions in the same order whatever the batch. The lse of the
// attention call already normalises, so there is no running maximum either.
//
// The blocks of all sequences, end to end, are divided evenly over one wave of CTAs (by whole
// blocks: the ring turns over a part of a block no faster than a whole one). A CTA's run of
// a sequence is taken W_SEG blocks at a time: for each kv head (and each W_ROWS of its rows) Q is
// staged once and the blocks' K tiles stream past it. Warp 0 loads K (TMA), warp 1 issues the MMAs,
// warps 2-3 stage Q and the rows' lse, position and slope, and two groups of four warps turn S into
// weights: for many rows each takes half of the columns of every tile, for few rows, where a tile
// is mostly waiting, the tiles of every other kv head. One token of 32 heads over 8 x 8192 keys: 28.1
// us for 134.8 MB (4.8 TB/s in all, the start and the end of the stream a third of it; 148 CTAs share 512
// blocks, so the longest run is 4 against 3.46 on average); 32 tokens over 3 sequences of up to 7001 keys
// and 4 kv heads, 256 rows of S a key: 19.6 us (24 with a masked block's columns tested one by one, for
// every head): 104 blocks leave 44 SMs without one, and the others take the kv heads one after another.
constexpr int W_THREADS = 384;
constexpr int W_BLK = 128;                     // keys of a tile
constexpr int W_BLK_PAGES = W_BLK / PAGE;
constexpr int W_TILE = W_BLK * D * 2;          // 32 KB: dims 0-63 of 128 keys, then 64-127
constexpr int W_ROWS = 256;                    // rows per staged Q, at most (N of the MMA)
constexpr int W_SEG = 16;                      // blocks of a segment
constexpr int W_MAX_STAGES = 6;
constexpr int W_NARROW = 32;                   // up to so many rows a tile is one group of warps' work
constexpr int W_BUFS = 8;                      // S buffers of a group then: 2 * 8 * 32 columns
constexpr int W_QS = 8;                        // staged Qs then (2 otherwise): short segments change Q often

struct WArgs {
    tree::Args t;
    const float* lse_in;
    float* acc;
    long long acc_stride, acc_cols;            // a row's distance and its places
    float decay;
    int rows;                                  // rows per staged Q: a multiple of 16, at most W_ROWS
    int stages;                                // K tiles in flight
};
// Of the columns of a staged Q, rows words each: lse in log2 (+inf: adds nothing), slope, position,
// the sequence's token (-1 behind the rows).
struct RowInfo {
    float* base;
    int rows;
    __device__ __forceinline__ float* lse2(int c) const { return base + c; }
    __device__ __forceinline__ float* slope2(int c) const { return base + rows + c; }
    __device__ __forceinline__ int* pos(int c) const { return reinterpret_cast<int*>(base + 2 * rows + c); }
    __device__ __forceinline__ int* i(int c) const { return reinterpret_cast<int*>(base + 3 * rows + c); }
};
constexpr size_t W_FIXED = 1024 + 2 * W_SEG * W_BLK * 4 + (2 * W_MAX_STAGES + 4 * W_QS + 4 * W_BUFS + 1) * 8 + 16;
constexpr int w_qbufs(int rows) { return rows <= W_NARROW ? W_QS : 2; }
constexpr int w_ibufs(int rows) { return rows <= W_NARROW ? W_QS : 4; }   // row infos: staged further ahead
constexpr size_t w_smem(int rows, int stages) {
    return W_FIXED + (size_t)rows * (w_qbufs(rows) * D * 2 + w_ibufs(rows) * 16) + (size_t)stages * W_TILE;
}

struct WSeg {
    int b, pg0, pg1;                           // pages of the sequence, whole blocks but for its end
};
// A CTA's run of blocks, a segment of at most W_SEG at a time.
struct WWalk {
    long long left, off;
    int b;
    __device__ __forceinline__ bool next(const tree::Args& a, WSeg* g) {
        while (left > 0 && b < a.B) {
            int page0;
            const int np = (tree::seq_len(a.indptr, a.last, b, &page0) + PAGE - 1) / PAGE;
            const int blocks = (np + W_BLK_PAGES - 1) / W_BLK_PAGES;
            if (off >= blocks) {
                off -= blocks;
                b++;
                continue;
            }
            const int b1 = (int)min(min((long long)blocks, off + left), off + W_SEG);
            g->b = b;
            g->pg0 = (int)off * W_BLK_PAGES;
            g->pg1 = min(np, b1 * W_BLK_PAGES);
            left -= b1 - off;
            off = b1;
            return true;
        }
        return false;
    }
};

// Bits [at, at + 32) of the 128-bit set v3 v2 v1 v0 (at >= 0). By value: a choice between
// variables must not become one between addresses, which would put them in local memory.
__device__ __forceinline__ uint32_t bits32(uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3, int at) {
    const int w = at >> 5;
    const uint32_t lo = w == 0 ? v0 : w == 1 ? v1 : w == 2 ? v2 : w == 3 ? v3 : 0u;
    const uint32_t hi = w == 0 ? v1 : w == 1 ? v2 : w == 2 ? v3 : 0u;
    return __funnelshift_r(lo, hi, at & 31);
}

// Of 32 columns, of which the first is `skip` rows into its token, those whose token's bit in `see` (the
// first column's is bit 0) is set, and only the first `valid`: a token at a time, not a column.
__device__ __forceinline__ uint32_t columns(uint32_t see, int G, int skip, int valid) {
    uint32_t v = 0u;
    for (int lo = -skip; lo < 32 && see; lo += G, see >>= 1) {
        const uint32_t from = 0xffffffffu << max(lo, 0), upto = lo + G < 32 ? ~(0xffffffffu << (lo + G)) : 0xffffffffu;
        v |= see & 1u ? from & upto : 0u;
    }
    return valid < 32 ? v & ~(0xffffffffu << max(valid, 0)) : v;
}

// Sum of the weights of M <= 32 columns from `col` on; x holds their scores (bias excluded). Where
// not every column is a row that sees the key (`full`), bit i of `cols` says whether column col + i
// does.
template <bool EXT, int M>
__device__ __forceinline__ float weigh(const tree::Args& a, const RowInfo& in, bool full, int kpos, uint32_t cols, int col,
                                       float (&x)[M]) {
    if (EXT && a.slopes) {
#pragma unroll
        for (int i = 0; i < M; i++) x[i] += tree::bias<EXT>(a, *in.slope2(col + i), *in.pos(col + i), kpos);
    }
    if (!full) {
#pragma unroll
        for (int i = 0; i < M; i++) x[i] = (cols >> i) & 1u ? x[i] : -INFINITY;
    }
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
    for (int i = 0; i < M; i += 4) {
        const float4 l = *reinterpret_cast<const float4*>(in.lse2(col + i));
        s0 += ex2(x[i] - l.x);
        s1 += ex2(x[i + 1] - l.y);
        s2 += ex2(x[i + 2] - l.z);
        s3 += ex2(x[i + 3] - l.w);
    }
    return (s0 + s1) + (s2 + s3);
}

__device__ __forceinline__ uint32_t w_sw(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

template <bool EXT>
__global__ void __launch_bounds__(W_THREADS, 1)
weights_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ, const WArgs w) {
    extern __shared__ uint8_t smem_raw[];
    const tree::Args& a = w.t;
    const int N = w.rows, KST = w.stages, q_bytes = N * D * 2;
    // S buffers: two of 256 columns, or W_BUFS narrow ones for each group of warps
    const bool narrow = N <= W_NARROW;
    const int d_cols = narrow ? W_NARROW : 256, bufs = narrow ? W_BUFS : 2;
    const int qbufs = w_qbufs(N), ibufs = w_ibufs(N);
    uint8_t* kring = align_ptr<1024>(smem_raw);
    uint8_t* qs = kring + KST * W_TILE;                              // [qbufs] staged Q: dims 0-63, then 64-127
    float* infos = reinterpret_cast<float*>(qs + qbufs * q_bytes);   // [ibufs] row infos, 4 N words each
    float* sums = infos + ibufs * 4 * N;                             // [2 groups][W_SEG][128]
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sums + 2 * W_SEG * W_BLK);
    uint64_t* k_empty = k_full + W_MAX_STAGES;
    uint64_t* q_full = k_empty + W_MAX_STAGES;   // [qbufs] staged
    uint64_t* q_empty = q_full + W_QS;           // [qbufs] its MMAs are done
    uint64_t* i_full = q_empty + W_QS;           // [ibufs] row infos are there
    uint64_t* i_empty = i_full + W_QS;           // [ibufs] the row infos have been used
    uint64_t* d_full = i_empty + W_QS;              // [2 groups][W_BUFS] S written
    uint64_t* d_empty = d_full + 2 * W_BUFS;     // [2 groups][W_BUFS] S read
    uint64_t* done = d_empty + 2 * W_BUFS;                // every issued MMA finished
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    __shared__ long long s_left, s_off;
    __shared__ int s_b;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < KST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < qbufs; i++) {
            mbar_init(&q_full[i], a.q_tma ? 1 : 64);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < ibufs; i++) {
            mbar_init(&i_full[i], 64);
            mbar_init(&i_empty[i], 256);
        }
        for (int i = 0; i < 2 * W_BUFS; i++) {
            mbar_init(&d_full[i], 1);
            mbar_init(&d_empty[i], narrow ? 128 : 256);
        }
        mbar_init(done, 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) tma_prefetch_desc(&tmK);
    pdl_wait();
    if (warp == 2) {
        // this CTA's blocks: two sweeps over the lengths
        auto blocks = [&](int b) {
            int p;
            return b < a.B ? (tree::seq_len(a.indptr, a.last, b, &p) + W_BLK - 1) / W_BLK : 0;
        };
        const int first = blocks(lane);                              // of sequences 0 .. 31
        long long total = first;
        for (int b0 = 32; b0 < a.B; b0 += 32) total += blocks(b0 + lane);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const tree::Share sh(total, gridDim.x);
        const long long beg = sh.first(blockIdx.x);
        long long before = 0;
        int b = a.B;
        for (int b0 = 0; b0 < a.B && b == a.B; b0 += 32) {
            const int mine = b0 ? blocks(b0 + lane) : first;
            long long x = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned over = __ballot_sync(0xffffffffu, before + x > beg);
            const int l = over ? __ffs(over) - 1 : 31;
            if (over) b = b0 + l;
            before += __shfl_sync(0xffffffffu, over ? x - mine : x, l);
        }
        if (lane == 0) {
            s_left = sh.first(blockIdx.x + 1) - beg;
            s_off = beg - before;
            s_b = b;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_trigger();
    const uint32_t tmem = *tmem_slot;
    auto d_col = [&](int d) { return (uint32_t)((d / W_BUFS * bufs + d % W_BUFS) * d_cols); };   // of S buffer d
    WWalk walk{s_left, s_off, s_b};
    WSeg g;
    bool ok = true;
    int chunk = 0, n = 0;                        // staged Qs and K tiles so far
    // every role walks the same segments, chunks (kv head, rows) and blocks; pages before the
    // first key in anyone's window are not loaded
    auto plan = [&](const Seq& s, int* first, int* nrows, int* pos_hi) {
        int lo = 0;
        *pos_hi = s.len - 1;
        *nrows = min(s.T, a.max_q) * a.G;
        if (a.window > 0) tree::pos_range(a, s, lane, &lo, pos_hi);
        *first = tree::first_key(a, s, lo) / PAGE;
    };

    if (warp == 0) {
        // ---------------------------------------------------------------- K producer
        const uint64_t pol = policy_evict_first();
        while (ok && walk.next(a, &g)) {
            const Seq s(a, g.b);
            int first, nrows, pos_hi;
            plan(s, &first, &nrows, &pos_hi);
            const int pg0 = max(g.pg0, first);
            int ids[W_SEG / 4];                              // the segment's page ids, 32 per register
#pragma unroll
            for (int i = 0; i < W_SEG / 4; i++) {
                const int pg = pg0 + 32 * i + lane;
                ids[i] = pg < g.pg1 ? __ldg(a.indices + s.page0 + pg) : 0;
            }
            for (int h = 0; h < a.Hkv && ok; h++)
                for (int r0 = 0; r0 < nrows && ok; r0 += N, chunk++) {
                    for (int pg = pg0; pg < g.pg1 && ok; pg += W_BLK_PAGES, n++) {
                        const int np = min(W_BLK_PAGES, g.pg1 - pg), st = n % KST, j = (pg - pg0) / W_BLK_PAGES;
                        int id = ids[0];
#pragma unroll
                        for (int i = 1; i < W_SEG / 4; i++) id = (j >> 2) == i ? ids[i] : id;
                        int page[W_BLK_PAGES];
#pragma unroll
                        for (int i = 0; i < W_BLK_PAGES; i++) page[i] = __shfl_sync(0xffffffffu, id, (j & 3) * 8 + i);
                        if (n >= KST) ok = __all_sync(0xffffffffu, mbar_wait_for(&k_empty[st], (n / KST - 1) & 1, a.timeout_ns, a.err));
                        if (!ok) break;
                        if (elect_one()) {
                            mbar_arrive_expect_tx(&k_full[st], np * KV_TILE);
                            uint8_t* dst = kring + st * W_TILE;
#pragma unroll
                            for (int i = 0; i < W_BLK_PAGES; i++)
                                if (i < np) {
                                    tma_load_5d(dst + i * HALF_TILE, &tmK, 0, 0, 0, h, page[i], &k_full[st], pol);
                                    tma_load_5d(dst + W_TILE / 2 + i * HALF_TILE, &tmK, 0, 0, 1, h, page[i], &k_full[st], pol);
                                }
                        }
                    }
                }
        }
        // every issued copy must land before the CTA exits
        if (lane == 0)
            for (int i = 0; i < KST && i < n; i++)
                mbar_wait_for(&k_full[i], ((i + (n - 1 - i) / KST * KST) / KST) & 1, DRAIN_NS, a.err);
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const uint32_t idesc = umma_idesc_f16(W_BLK, N, false, false);
        const uint64_t kd = umma_desc_sw128(smem_u32(kring), 16, 1024), qd = umma_desc_sw128(smem_u32(qs), 16, 1024);
        int tiles[2] = {0, 0};                       // of each group
        while (ok && walk.next(a, &g)) {
            const Seq s(a, g.b);
            int first, nrows, pos_hi;
            plan(s, &first, &nrows, &pos_hi);
            const int pg0 = max(g.pg0, first), nb = max(0, (g.pg1 - pg0 + W_BLK_PAGES - 1) / W_BLK_PAGES);
            const int chunks = nb > 0 ? a.Hkv * ((nrows + N - 1) / N) : 0;
            if (elect_one()) {
                int t0 = tiles[0], t1 = tiles[1];
                for (int c = 0; c < chunks && ok; c++) {
                    const int qb = (chunk + c) % qbufs;
                    ok = mbar_wait_for(&q_full[qb], ((chunk + c) / qbufs) & 1, a.timeout_ns, a.err);
                    for (int j = 0; j < nb && ok; j++) {
                        const int m = n + c * nb + j, st = m % KST, gr = narrow ? c & 1 : 0;
                        const int t = gr ? t1++ : t0++, d = gr * W_BUFS + t % bufs;
                        ok = mbar_wait_for(&k_full[st], (m / KST) & 1, a.timeout_ns, a.err);
                        if (ok && t >= bufs) ok = mbar_wait_for(&d_empty[d], (t / bufs - 1) & 1, a.timeout_ns, a.err);
                        if (!ok) break;
                        tc_fence_after_sync();
#pragma unroll
                        for (int kk = 0; kk < 8; kk++)
                            umma_f16(tmem + d_col(d), kd + st * (W_TILE / 16) + ((kk >> 2) * (W_TILE / 2) + (kk & 3) * 32) / 16,
                                     qd + (qb * q_bytes + (kk >> 2) * (q_bytes / 2) + (kk & 3) * 32) / 16, idesc, kk != 0);
                        umma_commit(&d_full[d]);
                        umma_commit(&k_empty[st]);
                        if (j == nb - 1) umma_commit(&q_empty[qb]);
                    }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            chunk += chunks;
            n += chunks * nb;
            tiles[0] += nb * (narrow ? (chunks + 1) / 2 : chunks);
            tiles[1] += nb * (narrow ? chunks / 2 : 0);
        }
        if (elect_one()) umma_commit(done);
        __syncwarp();
    } else if (warp < 4) {
        // ---------------------------------------------------------------- Q and the rows' infos
        const int tid = threadIdx.x - 64;
        while (ok && walk.next(a, &g)) {
            const Seq s(a, g.b);
            int first, nrows, pos_hi;
            plan(s, &first, &nrows, &pos_hi);
            if (s.T > a.max_q && g.pg0 == 0 && tid == 0) atomicOr(a.err, DEVERR_BOUND);
            if (max(g.pg0, first) >= g.pg1) continue;
            for (int h = 0; h < a.Hkv && ok; h++)
                for (int r0 = 0; r0 < nrows && ok; r0 += N, chunk++) {
                    const int qb = chunk % qbufs, ib = chunk % ibufs;
                    if (chunk >= qbufs)
                        ok = __all_sync(0xffffffffu, mbar_wait_for(&q_empty[qb], (chunk / qbufs - 1) & 1, a.timeout_ns, a.err));
                    if (!ok) break;
                    uint8_t* dst = qs + qb * q_bytes;
                    if (a.q_tma) {
                        // rows are tokens x heads of the group: a box per 64-dim half; rows behind
                        // the sequence's may be another's, and weigh nothing
                        if (tid == 0) {
                            const int i0 = s.q0 + r0 / a.G;
                            mbar_arrive_expect_tx(&q_full[qb], q_bytes);
                            tma_load_3d(dst, &tmQ, 0, h * a.G, i0, &q_full[qb]);
                            tma_load_3d(dst + q_bytes / 2, &tmQ, 64, h * a.G, i0, &q_full[qb]);
                        }
                    } else {
#pragma unroll 8
                        for (int c = tid; c < N * 16; c += 64) {
                            const int r = c >> 4, cd = c & 15, rr = r0 + r;
                            uint4 v = make_uint4(0u, 0u, 0u, 0u);
                            if (rr < nrows) {
                                const int i = rr / a.G;
                                v = __ldg(reinterpret_cast<const uint4*>(
                                        a.q + ((size_t)(s.q0 + i) * a.Hq + h * a.G + (rr - i * a.G)) * D) + cd);
                            }
                            *reinterpret_cast<uint4*>(dst + (cd >> 3) * (q_bytes / 2) + w_sw(r, cd & 7)) = v;
                        }
                        fence_proxy_async_smem();
                        mbar_arrive(&q_full[qb]);
                    }
                    if (chunk >= ibufs)
                        ok = __all_sync(0xffffffffu, mbar_wait_for(&i_empty[ib], (chunk / ibufs - 1) & 1, a.timeout_ns, a.err));
                    if (!ok) { chunk++; break; }
                    const RowInfo in{infos + ib * 4 * N, N};
                    for (int r = tid; r < N; r += 64) {
                        Row row;
                        row.set(a, s, r0 + r, nrows, h);
                        float l = -INFINITY;
                        if (row.i >= 0) l = w.lse_in[(size_t)(s.q0 + row.i) * a.Hq + h * a.G + (r0 + r - row.i * a.G)];
                        // padding rows and rows that saw nothing: exp2(s - inf) = 0
                        *in.lse2(r) = l == -INFINITY ? INFINITY : l * LOG2E;
                        *in.slope2(r) = row.slope2;
                        *in.pos(r) = row.pos;
                        *in.i(r) = row.i;
                    }
                    mbar_arrive(&i_full[ib]);
                }
        }
        // a copied Q that nobody waited for (after a timeout) must still land
        if (a.q_tma && tid == 0)
            for (int c = max(0, chunk - qbufs); c < chunk; c++)
                mbar_wait_for(&q_full[c % qbufs], (c / qbufs) & 1, DRAIN_NS, a.err);
    } else {
        // ---------------------------------------------------------------- weights
        const int quarter = warp & 3, hf = (warp - 4) >> 2;
        const int key = quarter * 32 + lane;
        const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16);
        const int c0 = narrow ? 0 : hf * (N / 2), c1 = narrow ? N : c0 + N / 2;   // this thread's columns
        const int gr = narrow ? hf : 0;                              // narrow: the heads of that parity
        int tile = 0;                                                // of this group
        while (walk.next(a, &g)) {
            const Seq s(a, g.b);
            int first, nrows, pos_hi;
            plan(s, &first, &nrows, &pos_hi);
            const int pg0 = max(g.pg0, first), nb = max(0, (g.pg1 - pg0 + W_BLK_PAGES - 1) / W_BLK_PAGES);
            const int rchunks = (nrows + N - 1) / N, chunks = nb > 0 ? a.Hkv * rchunks : 0;
            for (int j = 0; j < nb; j++) sums[(hf * W_SEG + j) * W_BLK + key] = 0.f;
            // the old weights are on their way while the scores are made
            const bool keeps = hf == 0 && w.decay != 0.f;
            auto has = [&](int j) {                              // block j's key of this thread has an entry
                const int p = (pg0 + j * W_BLK_PAGES) * PAGE + key;
                return j < nb && p < s.len && p < g.pg1 * PAGE && p < w.acc_cols;
            };
            float* acc_row = w.acc + g.b * w.acc_stride + pg0 * PAGE + key;
            float old[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (keeps && has(j)) old[j] = acc_row[j * W_BLK];
            // columns of a masked tile that count, 32 a word: the same for every head, kept from one to the next
            uint32_t m0 = 0u, m1 = 0u, m2 = 0u, m3 = 0u;
            int masked = -1;                                     // the tile they are of
            for (int c = 0; c < chunks; c++, chunk++) {
                const int ib = chunk % ibufs;
                const RowInfo in{infos + ib * 4 * N, N};
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait_for(&i_full[ib], (chunk / ibufs) & 1, a.timeout_ns, a.err));
                const int r0 = c % rchunks * N;                      // first row of this chunk
                const int t_lo = (r0 + c0) / a.G;                    // tokens of this thread's columns
                const int nt = r0 + c0 < nrows ? (min(nrows, r0 + c1) - 1) / a.G - t_lo + 1 : 0;
                const int valid = nrows - r0;                        // columns that are rows: the others may hold
                                                                     // another sequence's, and are left out
                const bool mine = !narrow || (c & 1) == gr;
                for (int j = 0; mine && j < nb; j++, tile++) {
                    const int d = gr * W_BUFS + tile % bufs;
                    const uint32_t d_at = d_col(d);
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_for(&d_full[d], (tile / bufs) & 1, a.timeout_ns, a.err));
                    if (!ok) continue;
                    tc_fence_after_sync();
                    const int kbase = (pg0 + j * W_BLK_PAGES) * PAGE, p = kbase + key;
                    const bool whole = kbase + W_BLK <= s.ctx && (a.window <= 0 || (long long)pos_hi - kbase < a.window);
                    const bool full = whole && c1 <= valid;          // every column counts
                    const int kpos = whole ? p : s.pos(a, p);
                    const int id = c % rchunks * W_SEG + j;
                    if (!whole && id != masked) {
                        masked = id;
                        uint32_t v0 = 0u, v1 = 0u, v2 = 0u, v3 = 0u;     // tokens t_lo .. + 127 that see the key
                        if (p < s.len) {
                            const int k = p - s.ctx;                     // drafted index of the key
                            const bool bits = k >= 0 && k < 32 * a.mask_words;
                            const uint32_t* mw = a.mask + (size_t)(s.q0 + t_lo) * a.mask_words + (k >> 5);
                            // tokens t_lo + 32 q .. that see the key
                            auto seen = [&](int q) {
                                const int n32 = min(nt - 32 * q, 32);
                                if (n32 <= 0) return 0u;
                                uint32_t v = 0xffffffffu;
                                if (a.mask) {
                                    if (k >= 0) v = 0u;
                                    if (bits) {
#pragma unroll 8
                                        for (int i = 0; i < n32; i++)
                                            v |= ((__ldg(mw + (size_t)(32 * q + i) * a.mask_words) >> (k & 31)) & 1u) << i;
                                    }
                                } else {
                                    const int f = k - t_lo - 32 * q;      // a chain: tokens from k on
                                    v = f <= 0 ? 0xffffffffu : f >= 32 ? 0u : 0xffffffffu << f;
                                }
                                if (a.window > 0) {
                                    for (int i = 0; i < n32; i++) {
                                        const int t = t_lo + 32 * q + i;
                                        const int tp = a.positions ? __ldg(a.positions + s.q0 + t) : s.ctx + t;
                                        if ((long long)tp - kpos >= a.window) v &= ~(1u << i);
                                    }
                                }
                                return v;
                            };
                            v0 = seen(0);
                            v1 = seen(1);
                            v2 = seen(2);
                            v3 = seen(3);
                        }
                        auto of = [&](int col) {
                            if (col >= min(c1, valid)) return 0u;
                            const int i = *in.i(col);
                            return columns(bits32(v0, v1, v2, v3, i - t_lo), a.G, r0 + col - i * a.G, valid - col);
                        };
                        m0 = of(c0);
                        m1 = of(c0 + 32);
                        m2 = of(c0 + 64);
                        m3 = of(c0 + 96);
                    }
                    auto cols_of = [&](int col) {
                        if (whole) return valid - col < 32 ? ~(0xffffffffu << (valid - col)) : 0xffffffffu;
                        const int q = (col - c0) >> 5;
                        return (q == 0 ? m0 : q == 1 ? m1 : q == 2 ? m2 : m3) >> ((col - c0) & 31);
                    };
                    float add = 0.f;
                    int col = c0;
                    for (; col + 32 <= c1 && col < valid; col += 32) {
                        float x[32];
                        tmem_ld32(trow + d_at + col, reinterpret_cast<uint32_t(&)[32]>(x));
                        tmem_ld_wait();
                        tree::score_all<EXT>(a, x);
                        add += weigh<EXT, 32>(a, in, full, kpos, cols_of(col), col, x);
                    }
                    for (; col < min(c1, valid); col += 8) {
                        float x[8];
                        tmem_ld8(trow + d_at + col, reinterpret_cast<uint32_t(&)[8]>(x));
                        tmem_ld_wait();
                        tree::score_all<EXT>(a, x);
                        add += weigh<EXT, 8>(a, in, full, kpos, cols_of(col), col, x);
                    }
                    tc_fence_before_sync();
                    mbar_arrive(&d_empty[d]);
                    sums[(hf * W_SEG + j) * W_BLK + key] += add;
                }
                if (ok) mbar_arrive(&i_empty[ib]);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");           // both column halves are summed
            if (hf == 0 && ok) {
                // pages that nobody sees only decay
                for (int p = g.pg0 * PAGE + key; p < min(s.len, pg0 * PAGE); p += W_BLK)
                    if (p < w.acc_cols && p < g.pg1 * PAGE) {
                        float* dst = w.acc + g.b * w.acc_stride + p;
                        *dst = w.decay != 0.f ? w.decay * *dst : 0.f;
                    }
                auto put = [&](int j, float before) {
                    const float x = sums[j * W_BLK + key] + sums[(W_SEG + j) * W_BLK + key];
                    acc_row[j * W_BLK] = w.decay != 0.f ? fmaf(w.decay, before, x) : x;
                };
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (has(j)) put(j, old[j]);
                for (int j = 4; j < nb; j++)
                    if (has(j)) put(j, keeps ? acc_row[j * W_BLK] : 0.f);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");           // before the sums are cleared
        }
    }
    // every MMA must have finished before tensor memory is released
    if (threadIdx.x == 0) mbar_wait_for(done, 0, DRAIN_NS, a.err);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, 512);
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
constexpr int S_BINS = 2048;               // words of a pass's histogram
constexpr int S_KEYS = 16;                 // keys a thread holds in registers
constexpr int S_CLUSTER = 8;               // CTAs of a sequence, at most
constexpr int S_SLICE = 8192;              // places per CTA that a cluster is sized for

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
    long long stride, cols;
    int keep, sink, recent, cluster;
};
struct SShared {
    int hist[3][S_BINS];                   // three passes of 2048 bins, or four of 256
    int warp_gt[S_WARPS], warp_eq[S_WARPS];
    int part[4][256];
    int bin, left, in;
    int total[2];
};

// Keeps the `want` greatest of the places [a.sink, a.sink + mid): radix passes over the ordered
// keys narrow the threshold, then every warp counts and writes its part of the list in order. A
// warp owns a run of 32-place rows of the CTA's slice; HELD: a thread has its keys in registers,
// otherwise (slices beyond 16K places) they are read again each time.
// CLUSTERED: the CTAs of a cluster share the sequence and add up one another's histograms, in 8-bit
// digits (one remote pair of words per thread and pass; 11-bit digits would move 64 KB per CTA);
// a single CTA takes 11 bits a pass. A pass whose bin is taken whole ends the search.
template <bool CLUSTERED, bool HELD>
__device__ __forceinline__ void select_part(const SArgs& a, SShared& sh, const float* acc_row, int mid, int want,
                                            int* out, int tid, int rank) {
    constexpr int PASSES = CLUSTERED ? 4 : 3;
    const int warp = tid >> 5, lane = tid & 31;
    // this CTA's slice of the middle, a warp's rows of it
    const int slice = CLUSTERED ? ((mid + a.cluster - 1) / a.cluster + 31) & ~31 : mid;
    const int beg = a.sink + min(mid, rank * slice), n = a.sink + min(mid, (rank + 1) * slice) - beg;
    const int per = ((n + S_WARPS - 1) / S_WARPS + 31) & ~31;
    const int w0 = min(n, warp * per), w1 = min(n, w0 + per);
    const float* row = acc_row + beg;
    const long long have = a.cols - beg;                    // places of the row that exist
    auto load = [&](int i) { return i < have ? rank_key(__ldg(row + i)) : 0u; };
    uint32_t held[HELD ? S_KEYS : 1];
    if (HELD) {
#pragma unroll
        for (int r = 0; r < S_KEYS; r++) {
            const int i = w0 + r * 32 + lane;
            held[HELD ? r : 0] = i < w1 ? load(i) : 0u;
        }
    }
    // f(first place of the row, this lane's key, whether it has one) for every row of the warp
    auto rows = [&](auto f) {
        if (HELD) {
#pragma unroll
            for (int r = 0; r < S_KEYS; r++)
                if (w0 + r * 32 < w1) f(w0 + r * 32, held[HELD ? r : 0], w0 + r * 32 + lane < w1);
        } else {
            for (int i = w0; i < w1; i += 32) f(i, i + lane < w1 ? load(i + lane) : 0u, i + lane < w1);
        }
    };

    uint32_t prefix = 0, known = 0;
    for (int pass = 0; pass < PASSES; pass++) {
        const int shift = CLUSTERED ? 24 - 8 * pass : pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t field = CLUSTERED ? 255u : pass == 2 ? 1023u : 2047u;
        int* h = CLUSTERED ? sh.hist[0] + pass * 256 : sh.hist[pass];
        rows([&](int, uint32_t k, bool in) {
            if (in && (k & known) == prefix) atomicAdd(&h[(k >> shift) & field], 1);
        });
        // bins from the greatest down: two per thread, or one each in the first 256
        int bin, c0 = 0, c1 = 0;
        if (CLUSTERED) {
            cluster_sync();
            const int r = (tid >> 8) * 2;
            bin = 255 - (tid & 255);
            if (r < a.cluster) c0 = cluster_load(&h[bin], r);
            if (r + 1 < a.cluster) c0 += cluster_load(&h[bin], r + 1);
            sh.part[tid >> 8][bin] = c0;
            __syncthreads();
            c0 = tid < 256 ? sh.part[0][bin] + sh.part[1][bin] + sh.part[2][bin] + sh.part[3][bin] : 0;
        } else {
            __syncthreads();
            bin = S_BINS - 1 - 2 * tid;
            c0 = h[bin];
            c1 = h[bin - 1];
        }
        int x = c0 + c1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sh.warp_gt[warp] = x;
        __syncthreads();
        const int before = __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_gt[lane] : 0);
        const int up0 = before + x - c0 - c1, up1 = up0 + c0;     // keys above each bin
        if (up0 < want && want <= up1) { sh.bin = bin; sh.left = want - up0; sh.in = c0; }
        if (up1 < want && want <= up1 + c1) { sh.bin = bin - 1; sh.left = want - up1; sh.in = c1; }
        __syncthreads();
        prefix |= (uint32_t)sh.bin << shift;
        known |= field << shift;
        want = sh.left;
        if (sh.in == want) break;                            // the whole bin is kept
    }
    // keys above `prefix` in the known bits are kept, and the first `want` of those equal to it
    int gt = 0, eq = 0;
    rows([&](int, uint32_t k, bool in) {
        gt += in && (k & known) > prefix;
        eq += in && (k & known) == prefix;
    });
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        sh.warp_gt[warp] = gt;
        sh.warp_eq[warp] = eq;
    }
    __syncthreads();
    int g = __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_gt[lane] : 0);
    int e = __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_eq[lane] : 0);
    if (CLUSTERED) {
        if (warp == S_WARPS - 1 && lane == 0) {
            sh.total[0] = g + gt;
            sh.total[1] = e + eq;
        }
        cluster_sync();
        g += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_load(&sh.total[0], lane) : 0);
        e += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_load(&sh.total[1], lane) : 0);
        cluster_sync();                                      // nobody leaves while it is read
    }
    const uint32_t below = (1u << lane) - 1u;
    rows([&](int i0, uint32_t k, bool in) {
        const bool is_gt = in && (k & known) > prefix, is_eq = in && (k & known) == prefix;
        const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
        const int ei = e + __popc(be & below);
        if (is_gt || (is_eq && ei < want)) out[g + __popc(bg & below) + min(ei, want)] = beg + i0 + lane;
        g += __popc(bg);
        e += __popc(be);
    });
}

// grid = (cluster, B): bound by latency. 1 x 131072 places: 18.7 us, against 34 with the keys in
// shared memory and 11-bit digits across the cluster.
template <bool CLUSTERED>
__global__ void __launch_bounds__(S_THREADS) select_kernel(const SArgs a) {
    __shared__ SShared sh;
    const int tid = threadIdx.x;
    for (int i = tid; i < (CLUSTERED ? 4 * 256 : 3 * S_BINS); i += S_THREADS) (&sh.hist[0][0])[i] = 0;
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y, rank = CLUSTERED ? blockIdx.x : 0;
    int page0;
    const int len = tree::seq_len(a.indptr, a.last, b, &page0);
    int* out = a.keep_idx + (size_t)b * a.keep;
    const int step = gridDim.x * S_THREADS, me = rank * S_THREADS + tid;
    if (me == 0) a.keep_count[b] = min(len, a.keep);
    if (len <= a.keep) {                                     // the same for the whole cluster
        for (int i = me; i < a.keep; i += step) out[i] = i < len ? i : -1;
        return;
    }
    const int hi = len - a.recent, mid = hi - a.sink;
    const int want = a.keep - a.sink - a.recent;             // of the places [sink, hi); mid > want
    for (int i = me; i < a.sink; i += step) out[i] = i;
    for (int i = me; i < a.recent; i += step) out[a.keep - a.recent + i] = hi + i;
    if (want == 0) return;
    __syncthreads();                                         // the histograms are zero
    const float* row = a.acc + b * a.stride;
    const int slice = CLUSTERED ? (mid + a.cluster - 1) / a.cluster : mid;
    if (slice <= S_KEYS * S_THREADS - 31)                    // a slice is rounded up to a warp's 32 places
        select_part<CLUSTERED, true>(a, sh, row, mid, want, out + a.sink, tid, rank);
    else
        select_part<CLUSTERED, false>(a, sh, row, mid, want, out + a.sink, tid, rank);
}

// ------------------------------------------------------------------ compact
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
    long long acc_stride, acc_cols;
    int Hkv, num_pages, keep_stride;
    int pieces;                  // 16-byte pieces of a row per CTA: a power of two, at most 16
};

// In place and in order: rows move towards the front (keep[i] >= start + i, ascending), so the
// rows that a tile of the list overwrites are read by this tile or an earlier one only. A CTA
// owns a column of the rows -- `pieces` 16-byte pieces of one head -- for all of a sequence's
// list: every thread loads its pieces of tile t + 1, the CTA meets (tile t has been read), and
// every thread stores tile t: 64 KB are on their way while 64 KB are written. The places are
// translated to cache rows ahead of time, so that no load waits for an index. No CTA waits for
// another. 8 x 4096 rows of 8 heads: 55.8 us, 4.8 TB/s of pieces of 128 bytes that lie 2 KB apart: 256
// columns, one CTA an SM (512 threads of 101 registers), so some SMs take a second turn.
// ROWS: list entries translated at a time. The accepted paths of drafts are a few rows a
// sequence: small CTAs, so that all of them are resident (512 threads: 10.3 us at 32 x 5 rows,
// 128: 3.3 us). grid = (Hkv * 16 / pieces (+ 1 for acc and the lengths), B, 2).
template <int C_THREADS, int C_ROWS>
__global__ void __launch_bounds__(C_THREADS) compact_kernel(const CArgs a) {
    __shared__ int s_src[C_ROWS], s_dst[C_ROWS];              // cache rows, -1: none
    __shared__ int s_first;
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
#pragma unroll 4
    for (int i = tid; i < n; i += C_THREADS) {
        const int x = __ldg(idx + i), before = i ? __ldg(idx + i - 1) : start - 1;
        bad |= x <= before || x >= len;
        if (x != start + i) i0 = min(i0, i);
    }
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
                x[u] = i < n && src < a.acc_cols ? row[src] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < C_U; u++) {
                const int i = base + u * C_THREADS + tid;
                if (i < n && start + i < a.acc_cols) row[start + i] = x[u];
            }
        }
        __syncthreads();
        for (long long p = (long long)start + n + tid; p < len && p < a.acc_cols; p += C_THREADS) row[p] = 0.f;
        return;
    }
    uint4* cache = blockIdx.z ? a.v : a.k;
    const int per_head = 16 / a.pieces;
    const int head = blockIdx.x / per_head, col = (blockIdx.x - head * per_head) * a.pieces;
    const int rows = C_THREADS / a.pieces, r = tid / a.pieces;
    const int tile = rows * C_U;
    cache += head * 16 + col + tid % a.pieces;
    auto row_of = [&](int p) {                               // -1: a page outside the cache
        const int page = __ldg(a.indices + page0 + p / PAGE);
        return page < 0 || page >= a.num_pages ? -1 : page * PAGE + p % PAGE;
    };
    for (int base = i0; base < n; base += C_ROWS) {
        const int m = min(C_ROWS, n - base);
        __syncthreads();                                     // the rows before have been used
#pragma unroll 4
        for (int i = tid; i < m; i += C_THREADS) {
            s_src[i] = row_of(__ldg(idx + base + i));
            s_dst[i] = row_of(start + base + i);
        }
        __syncthreads();
        auto load = [&](int t, uint4 (&x)[C_U]) {
#pragma unroll
            for (int u = 0; u < C_U; u++) {
                const int i = t + u * rows + r, src = i < m ? s_src[i] : -1;
                x[u] = src >= 0 ? cache[(size_t)src * a.Hkv * 16] : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        auto store = [&](int t, const uint4 (&x)[C_U]) {
#pragma unroll
            for (int u = 0; u < C_U; u++) {
                const int i = t + u * rows + r, dst = i < m ? s_dst[i] : -1;
                if (dst >= 0) cache[(size_t)dst * a.Hkv * 16] = x[u];
            }
        };
        uint4 x[C_U], y[C_U];
        load(0, x);
        for (int t = 0; t < m; t += 2 * tile) {
            load(t + tile, y);
            __syncthreads();
            store(t, x);
            if (t + tile >= m) break;
            load(t + 2 * tile, x);
            __syncthreads();
            store(t + tile, y);
        }
    }
}

struct Setup {
    ckl_status st = CKL_OK;
};
const Setup* setup(const DeviceInfo* di) {
    static Setup ks[64];
    static std::once_flag once[64];
    std::call_once(once[di->device], [di] {
        cudaError_t e = cudaFuncSetAttribute(weights_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, di->smem_optin - 1024);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(weights_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, di->smem_optin - 1024);
        if (e != cudaSuccess) ks[di->device].st = cuda_status(e, "cache kernels setup");
    });
    return &ks[di->device];
}

}  // namespace evict
}  // namespace ckl

using namespace ckl;
using namespace ckl::evict;

extern "C" {

ckl_status ckl_cache_weights_ex(const ckl_tree_params* p, const float* lse, float* acc, long long acc_stride,
                                long long acc_cols, float decay, void* stream) {
    ckl_status st = tree::check_params(p, "cache_weights");
    if (st != CKL_OK) return st;
    if (acc_cols <= 0 || acc_cols > acc_stride)
        return fail(CKL_INVALID_ARG, "cache_weights: acc_stride=%lld acc_cols=%lld", acc_stride, acc_cols);
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
    w.acc_cols = acc_cols;
    w.decay = decay;
    // the rows of a kv head in one staged Q where they fit; the rest of shared memory streams K
    const long long rows = (long long)p->max_q * w.t.G;
    w.rows = (int)std::min((rows + 15) / 16 * 16, (long long)W_ROWS);
    w.stages = 2;
    while (w.stages < W_MAX_STAGES && w_smem(w.rows, w.stages + 1) <= (size_t)di->smem_optin - 1024) w.stages++;
    const long long blocks = (acc_cols + W_BLK - 1) / W_BLK;    // of a sequence, at most (longer ones take longer)
    const unsigned grid = (unsigned)std::min((long long)di->sms, blocks * p->B);
    CUtensorMap tmK, tmQ;
    st = tree::encode_half_map(p->k_cache, p->Hkv, p->num_pages, 1, &tmK);
    if (st != CKL_OK) return st;
    w.t.q_tma = w.rows % w.t.G == 0;
    st = tree::encode_q_map(p->q, p->N, p->Hq, w.t.q_tma ? w.t.G : 1, w.t.q_tma ? w.rows / w.t.G : 1, &tmQ);
    if (st != CKL_OK) return st;
    void* args[] = {&tmK, &tmQ, &w};
    const bool ext = p->softcap > 0.f || p->slopes;
    CKL_CUDA_TRY(launch(ext ? (const void*)weights_kernel<true> : (const void*)weights_kernel<false>, dim3(grid),
                        dim3(W_THREADS), w_smem(w.rows, w.stages), (cudaStream_t)stream, args, true));
    return CKL_OK;
}

ckl_status ckl_cache_weights(const ckl_tree_params* p, const float* lse, float* acc, long long acc_stride,
                             float decay, void* stream) {
    return ckl_cache_weights_ex(p, lse, acc, acc_stride, acc_stride, decay, stream);
}

ckl_status ckl_cache_select_ex(const float* acc, long long acc_stride, long long acc_cols, const int* kv_indptr,
                               const int* kv_last_page_len, int B, int keep, int sink, int recent,
                               int* keep_idx, int* keep_count, void* stream) {
    if (B < 0 || keep <= 0 || sink < 0 || recent < 0 || (long long)sink + recent > keep || acc_cols <= 0 ||
        acc_cols > acc_stride)
        return fail(CKL_INVALID_ARG, "cache_select: B=%d keep=%d sink=%d recent=%d acc_stride=%lld acc_cols=%lld", B,
                    keep, sink, recent, acc_stride, acc_cols);
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
    while (cluster < S_CLUSTER && (long long)cluster * S_SLICE < acc_cols && (long long)B * cluster * 2 <= di->sms) cluster *= 2;
    SArgs a{acc, kv_indptr, kv_last_page_len, keep_idx, keep_count, acc_stride, acc_cols, keep, sink, recent, cluster};
    void* args[] = {&a};
    if (cluster == 1) {
        CKL_CUDA_TRY(launch((const void*)select_kernel<false>, dim3(1, (unsigned)B), dim3(S_THREADS), 0,
                            (cudaStream_t)stream, args, true));
        return CKL_OK;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster, (unsigned)B);
    cfg.blockDim = dim3(S_THREADS);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CKL_CUDA_TRY(cudaLaunchKernelExC(&cfg, (const void*)select_kernel<true>, args));
    return CKL_OK;
}

ckl_status ckl_cache_select(const float* acc, long long acc_stride, const int* kv_indptr,
                            const int* kv_last_page_len, int B, int keep, int sink, int recent,
                            int* keep_idx, int* keep_count, void* stream) {
    return ckl_cache_select_ex(acc, acc_stride, acc_stride, kv_indptr, kv_last_page_len, B, keep, sink, recent,
                               keep_idx, keep_count, stream);
}

ckl_status ckl_cache_compact_ex(void* k_cache, void* v_cache, const int* kv_indptr, const int* kv_indices,
                                const int* kv_last_page_len, int B, int Hkv, int num_pages,
                                const int* keep_idx, int keep_stride, const int* keep_count,
                                const int* dst_start, float* acc, long long acc_stride, long long acc_cols,
                                int* new_len, void* stream) {
    if (B < 0 || Hkv <= 0 || num_pages <= 0 || keep_stride <= 0 || (acc && (acc_cols <= 0 || acc_cols > acc_stride)))
        return fail(CKL_INVALID_ARG, "cache_compact: B=%d Hkv=%d num_pages=%d keep_stride=%d acc_stride=%lld "
                    "acc_cols=%lld", B, Hkv, num_pages, keep_stride, acc_stride, acc_cols);
    if (B > 65535 || Hkv > 65535) return fail(CKL_UNSUPPORTED_SHAPE, "cache_compact: B=%d Hkv=%d (at most 65535)", B, Hkv);
    if (B == 0) return CKL_OK;
    if (!k_cache || !v_cache || !kv_indptr || !kv_indices || !kv_last_page_len || !keep_idx || !keep_count)
        return fail(CKL_INVALID_ARG, "cache_compact: NULL tensor pointer");
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15)
        return fail(CKL_INVALID_ARG, "cache_compact: k_cache and v_cache must be 16-byte aligned");
    if (num_pages > INT_MAX / PAGE) return fail(CKL_UNSUPPORTED_SHAPE, "cache_compact: num_pages=%d", num_pages);
    // what a CTA writes, others still read: each output stands alone. (Of kv_indices the host knows
    // no more than its first entry.)
    const size_t cache = (size_t)num_pages * PAGE * Hkv * D * sizeof(__half), ints = (size_t)B * sizeof(int);
    const Span out[] = {{k_cache, cache}, {v_cache, cache}, {new_len, ints},
                        {acc, ((size_t)(B - 1) * acc_stride + acc_cols) * sizeof(float)}};
    const Span in[] = {{kv_indptr, ints + sizeof(int)}, {kv_indices, sizeof(int)}, {kv_last_page_len, ints},
                       {keep_idx, ints * keep_stride}, {keep_count, ints}, {dst_start, ints}};
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < i; j++)
            if (overlap(out[i], out[j])) return fail(CKL_INVALID_ARG, "cache_compact: two of k_cache, v_cache, new_len and acc overlap");
        for (const Span& x : in)
            if (overlap(out[i], x)) return fail(CKL_INVALID_ARG, "cache_compact: k_cache, v_cache, new_len or acc overlaps an input");
    }
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
    a.acc_cols = acc_cols;
    a.Hkv = Hkv;
    a.num_pages = num_pages;
    a.keep_stride = keep_stride;
    // whole heads (256 bytes) per CTA, halved while the columns leave SMs idle, down to 64
    // bytes: two 32-byte sectors, the least that HBM serves
    a.pieces = 16;
    while (a.pieces > 4 && (long long)B * Hkv * 2 * (16 / a.pieces) < di->sms) a.pieces /= 2;
    void* args[] = {&a};
    const bool few = keep_stride <= 128;
    CKL_CUDA_TRY(launch(few ? (const void*)compact_kernel<128, 128> : (const void*)compact_kernel<512, 4096>,
                        dim3((unsigned)(Hkv * (16 / a.pieces) + 1), (unsigned)B, 2), dim3(few ? 128 : 512), 0,
                        (cudaStream_t)stream, args, true));
    return CKL_OK;
}

ckl_status ckl_cache_compact(void* k_cache, void* v_cache, const int* kv_indptr, const int* kv_indices,
                             const int* kv_last_page_len, int B, int Hkv, int num_pages,
                             const int* keep_idx, int keep_stride, const int* keep_count,
                             const int* dst_start, float* acc, long long acc_stride, int* new_len,
                             void* stream) {
    return ckl_cache_compact_ex(k_cache, v_cache, kv_indptr, kv_indices, kv_last_page_len, B, Hkv, num_pages, keep_idx,
                                keep_stride, keep_count, dst_start, acc, acc_stride, acc_stride, new_len, stream);
}

}  // extern "C"
