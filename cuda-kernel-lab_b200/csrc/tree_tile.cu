// tree_tile.cu -- the draft-tree attention for more than 16 stacked rows (drafted tokens x query
// heads of a kv head) on the 5th-generation tensor cores.
//
// A CTA holds 128 * MT rows of one (sequence, kv head) as MT tiles, the M of tcgen05.mma, and
// streams keys in blocks of 8 pages, taken in parts of 128 keys (one tile) or 64 (two):
//   S = Q K^T   M=128, N=a part: Q and K (both K-major) in shared memory, S in tensor memory, two
//               buffers a tile;
//   softmax     one thread per row: the row of S from tensor memory, online max and sum in
//               registers, P = exp2(S - m) as fp16 back into tensor memory, over S;
//   O += P V    M=128, N=128, K=16 a page: P from tensor memory, V (MN-major) from shared
//               memory, O in tensor memory for the whole run.
// Both tiles use the same K and V block: with 256 rows the stream is read once where the tensor
// cores still keep up with it (512 flops per byte of K and V against the card's ~256).
//
// Tensor memory is what the parts are cut to: 512 columns hold two tiles' O and twice 64 columns of S
// each. With one buffer of 128 the softmax waited for P V and the next S in turn (16 x 24 drafts,
// capped: 118 us, with two 109; 8 x 64 drafts, where the SM clock falls to 1.5 GHz under the products:
// 147 us and 149, as a product of N = 64 reads Q twice as often: 49 cycles per K = 16 step, of N =
// 128 65).
//
// V pages arrive as one 4 KB box each, [64-dim half][16 tokens][64 dims]. K pages take a 2 KB box
// per half, so that a part's keys of a half lie together and S is one product. For 256 rows bound by
// the chain of S, softmax and P V of a part (no unit is busy more than 36 % of the time), at the clock that
// the power cap leaves: 8 x 64 drafts over 16,384 keys 152-168 us in short runs (0.82-0.90 PFLOP/s), 184 us
// at 1.52 GHz in a long one. By HBM for up to 128 (8 x 32 drafts: 7 TB/s in the main loop), by start, masked
// block and join for short ones.
//
// Work is divided exactly: the key blocks of all (sequence, row group, kv head) units, end to
// end, over one wave of CTAs. A unit that lies within one CTA is written out directly; where a
// CTA's run of blocks crosses a unit's border it leaves a partial (at most two per CTA) and a
// second kernel joins them.

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "tree_tile.cuh"

namespace ckl {
namespace tree {
namespace tile {

constexpr int BLK_PAGES = 8;
constexpr int BLK = BLK_PAGES * PAGE;              // 128 keys
constexpr int KV_BLK = BLK_PAGES * KV_TILE;        // 32 KB of K or V
constexpr int Q_TILE = 128 * D * 2;                // 32 KB: dims 0-63 of 128 rows, then 64-127
constexpr int VST = 2;                             // V blocks in flight
template <int MT> struct Cfg {
    static constexpr int KST = MT == 1 ? 4 : 3;    // K blocks in flight
    static constexpr int SW = MT == 1 ? 128 : 64;  // keys of an S buffer: tensor memory holds two a tile
    static constexpr int U = BLK / SW;             // parts of a block
    static constexpr int PH = SW / 64;             // halves of P, 4 pages each
    static constexpr int TILE_COLS = 2 * SW + 128; // tensor memory of a tile: S (and P) twice, then O
    static constexpr int THREADS = 128 + 128 * MT; // warps 0-3: TMA, MMA, two that look V over; then a thread per row
    static constexpr int ROWS = 128 * MT;
    static constexpr int OFF_K = MT * Q_TILE;
    static constexpr int OFF_V = OFF_K + KST * KV_BLK;
    static constexpr int OFF_BAR = OFF_V + VST * KV_BLK;
    static constexpr int NBAR = 2 * KST + 3 * VST + (5 + 2 * PH) * MT + 2;
    static constexpr int SMEM = 1024 + OFF_BAR + NBAR * 8 + 32;
    static constexpr uint32_t TMEM_COLS = 512;
};
static_assert(Cfg<1>::SMEM <= 232448 && Cfg<2>::SMEM <= 232448, "shared memory of a CTA");

__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Blocks of keys of a unit of sequence s whose keys start at `first`: at least one, so that rows
// that see nothing are written too.
__device__ __forceinline__ int blocks_of(const Seq& s, int first) {
    return s.len > first ? (s.len - first + BLK - 1) / BLK : 1;
}
struct Work {                                       // of one sequence
    int first = 0, nblk = 0, nrows = 0, units = 0;
    __device__ __forceinline__ long long blocks() const { return (long long)nblk * units; }
};
template <int ROWS>
__device__ __forceinline__ Work work_of(const Args& a, const Seq& s, int pos_lo) {
    Work w;
    w.nrows = min(s.T, a.max_q) * a.G;
    if (w.nrows == 0) return w;
    w.first = first_key(a, s, pos_lo);
    w.nblk = blocks_of(s, w.first);
    w.units = (w.nrows + ROWS - 1) / ROWS * a.Hkv;
    return w;
}
// The same by one lane alone.
template <int ROWS>
__device__ __forceinline__ long long blocks_lane(const Args& a, int b) {
    if (b >= a.B) return 0;
    const Seq s(a, b);
    int lo = s.ctx;
    if (a.window > 0 && a.positions) {
        lo = 0x7fffffff;
        for (int i = 0; i < s.T; i++) lo = min(lo, __ldg(a.positions + s.q0 + i));
    }
    return work_of<ROWS>(a, s, lo).blocks();
}
// Blocks of sequences [0, upto) (one warp, all lanes get the sum).
template <int ROWS>
__device__ __forceinline__ long long blocks_before(const Args& a, int upto, int lane) {
    long long sum = 0;
    for (int b0 = 0; b0 < upto; b0 += 32) sum += b0 + lane < upto ? blocks_lane<ROWS>(a, b0 + lane) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
// A CTA's run of blocks, unit by unit. All lanes of a warp hold the same state.
struct Seg {
    int b, kvh, row0, rows;      // rows of this unit: [row0, row0 + rows) of the sequence's
    int blk0, blk1, nblk;
};
template <int ROWS>
struct Walk {
    long long left;              // blocks of this CTA not handed out yet
    long long off;               // next block within sequence b
    int b;
    __device__ __forceinline__ Walk(long long left_, long long off_, int b_)
        : left(left_), off(off_), b(b_) {}
    // The next segment, its sequence and work; false at the end.
    __device__ __forceinline__ bool next(const Args& a, Seg* g, Seq* s, Work* w, int* pos_hi, int lane) {
        while (left > 0 && b < a.B) {
            *s = Seq(a, b);
            int lo = s->ctx;
            *pos_hi = s->len - 1;
            if (a.window > 0) pos_range(a, *s, lane, &lo, pos_hi);
            *w = work_of<ROWS>(a, *s, lo);
            if (off >= w->blocks()) {
                off -= w->blocks();
                b++;
                continue;
            }
            const int unit = off >> 31 ? (int)(off / w->nblk) : (int)((unsigned)off / (unsigned)w->nblk), z = unit / a.Hkv;
            g->b = b;
            g->kvh = unit - z * a.Hkv;
            g->row0 = z * ROWS;
            g->rows = min(ROWS, w->nrows - g->row0);
            g->nblk = w->nblk;
            g->blk0 = (int)(off - (long long)unit * w->nblk);
            g->blk1 = (int)min((long long)w->nblk, g->blk0 + left);
            off += g->blk1 - g->blk0;
            left -= g->blk1 - g->blk0;
            return true;
        }
        return false;
    }
};

// Which of the keys [p, p + 32) row r sees, as bits.
__device__ __forceinline__ uint32_t seen32(const Args& a, const Seq& s, const Row& r, int p) {
    if (r.i < 0) return 0u;
    const int in = s.len - p;                                     // keys within the sequence
    uint32_t v = in >= 32 ? 0xffffffffu : in <= 0 ? 0u : (1u << in) - 1u;
    const int j0 = p - s.ctx;                                     // drafted index of the first key
    if (j0 > -32) {
        uint32_t d;                                               // bits of drafted keys j0 .. j0 + 31
        if (a.mask) {
            const uint32_t* m = a.mask + (size_t)(s.q0 + r.i) * a.mask_words;
            auto word = [&](int w) { return w >= 0 && w < a.mask_words ? __ldg(m + w) : 0u; };
            const int w = j0 >> 5;                                // floor
            d = __funnelshift_r(word(w), word(w + 1), j0 & 31);
        } else {
            const int n = r.i - j0 + 1;                           // j <= i
            d = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
        }
        if (j0 < 0) d |= (1u << -j0) - 1u;                        // context keys
        v &= d;
    }
    if (a.window > 0) {
        for (uint32_t m = v; m; m &= m - 1) {
            const int k = __ffs(m) - 1;
            if ((long long)r.pos - s.pos(a, p + k) >= a.window) v &= ~(1u << k);
        }
    }
    return v;
}

template <int MT, bool EXT>
__global__ void __launch_bounds__(Cfg<MT>::THREADS, 1)
tile_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
            const __grid_constant__ CUtensorMap tmQ, const Args a) {
    using C = Cfg<MT>;
    constexpr int KST = C::KST, SW = C::SW, U = C::U, PH = C::PH, COLS = C::TILE_COLS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = align_ptr<1024>(smem_raw);
    uint8_t* qs = sm;
    uint8_t* kring = sm + C::OFF_K;
    uint8_t* vring = sm + C::OFF_V;
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* k_empty = k_full + KST;
    uint64_t* v_full = k_empty + KST;
    uint64_t* v_empty = v_full + VST;
    uint64_t* v_ready = v_empty + VST;       // V looked over, where some row does not see it all
    uint64_t* q_empty = v_ready + VST;       // every S of a segment done: Q may be replaced
    uint64_t* q_full = q_empty + 1;          // [MT] Q of a segment is there
    uint64_t* s_full = q_full + MT;          // [MT][2] S written (MMA -> softmax)
    // [MT][2][PH] P of four pages written (softmax -> MMA): one per S buffer, since the softmax may
    // end the next part before the MMA warp has seen this one
    uint64_t* p_full = s_full + MT * 2;
    // [MT][2] O holds the part, its P has been read (MMA -> all): one per S buffer too, since the last
    // part's P may be written before O holds the part before it
    uint64_t* o_done = p_full + MT * 2 * PH;
    uint64_t* done = o_done + MT * 2;          // every issued MMA finished
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* odd = reinterpret_cast<volatile int*>(tmem_slot + 1);   // unseen V held inf or NaN
    long long* range = reinterpret_cast<long long*>(tmem_slot + 2);       // {left, offset}, sequence
    int* range_b = reinterpret_cast<int*>(range + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < KST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < VST; i++) {
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&v_ready[i], 64);
        }
        for (int t = 0; t < MT; t++) {
            mbar_init(&q_full[t], a.q_tma ? 1 : 128);
            for (int i = 0; i < 2; i++) {
                mbar_init(&s_full[t * 2 + i], 1);
                mbar_init(&o_done[t * 2 + i], 1);
            }
            for (int i = 0; i < 2 * PH; i++) mbar_init(&p_full[t * 2 * PH + i], 128);
        }
        mbar_init(q_empty, 1);
        mbar_init(done, 1);
        fence_barrier_init();
        *odd = 0;
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    pdl_wait();
    if (warp == 2) {
        const long long first = blocks_lane<C::ROWS>(a, lane);         // of sequences 0 .. 31
        long long W = first;
        for (int b0 = 32; b0 < a.B; b0 += 32) W += blocks_lane<C::ROWS>(a, b0 + lane);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(0xffffffffu, W, o);
        const Share sh(W, gridDim.x);
        const long long beg = sh.first(blockIdx.x), end = sh.first(blockIdx.x + 1);
        long long before = 0;
        int b = a.B;
        for (int b0 = 0; b0 < a.B && b == a.B; b0 += 32) {
            const long long mine = b0 ? blocks_lane<C::ROWS>(a, b0 + lane) : first;
            long long x = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned over = __ballot_sync(0xffffffffu, before + x > beg);
            if (over) {
                const int l = __ffs(over) - 1;
                b = b0 + l;
                before += __shfl_sync(0xffffffffu, x - mine, l);
            } else {
                before += __shfl_sync(0xffffffffu, x, 31);
            }
        }
        if (lane == 0) {
            range[0] = end - beg;
            range[1] = beg - before;
            *range_b = b;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    pdl_trigger();
    const uint32_t tmem = *tmem_slot;
    Walk<C::ROWS> walk(range[0], range[1], *range_b);
    Seg g;
    Seq s;
    Work w;
    int pos_hi;

    if (warp < 4) {
    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        const uint64_t pol = policy_evict_first();
        int qn[MT];                                     // Q loads issued into each tile
#pragma unroll
        for (int t = 0; t < MT; t++) qn[t] = 0;
        int ok = 1, n = 0, seg = 0;
        int nk = 0, nv = 0;                             // blocks of K and of V issued
        while (ok && walk.next(a, &g, &s, &w, &pos_hi, lane)) {
            const int p0 = w.first / PAGE, npg = (s.len + PAGE - 1) / PAGE;
            int ids_at = 0, my_id = 0;
            for (int j = g.blk0; j < g.blk1 && ok; j++, n++) {
                const int at = p0 + j * BLK_PAGES;
                // page ids, 32 per load; a page behind the sequence reads as zeros (its
                // coordinate is past the tensor map's extent)
                if (j == g.blk0 || at >= ids_at + 32) {
                    ids_at = at;
                    my_id = at + lane < npg ? __ldg(a.indices + s.page0 + at + lane) : a.num_pages;
                }
                int page[BLK_PAGES];
#pragma unroll
                for (int i = 0; i < BLK_PAGES; i++) page[i] = __shfl_sync(0xffffffffu, my_id, at - ids_at + i);
                const int ks = n % KST, vs = n % VST;
                // one elected lane issues: a box per lane would be serialised at ~50 ns each
                if (elect_one()) {
                    if (n >= KST) ok = mbar_wait_for(&k_empty[ks], ((n / KST) - 1) & 1, a.timeout_ns, a.err);
                    if (ok) {
                        uint8_t* dst = kring + ks * KV_BLK;
                        mbar_arrive_expect_tx(&k_full[ks], KV_BLK);
#pragma unroll
                        for (int i = 0; i < BLK_PAGES; i++) {
                            tma_load_5d(dst + i * HALF_TILE, &tmK, 0, 0, 0, g.kvh, page[i], &k_full[ks], pol);
                            tma_load_5d(dst + KV_BLK / 2 + i * HALF_TILE, &tmK, 0, 0, 1, g.kvh, page[i], &k_full[ks], pol);
                        }
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                nk = n + 1;
                if (elect_one()) {
                    if (n >= VST) ok = mbar_wait_for(&v_empty[vs], ((n / VST) - 1) & 1, a.timeout_ns, a.err);
                    if (ok) {
                        uint8_t* dst = vring + vs * KV_BLK;
                        mbar_arrive_expect_tx(&v_full[vs], KV_BLK);
#pragma unroll
                        for (int i = 0; i < BLK_PAGES; i++)
                            tma_load_5d(dst + i * KV_TILE, &tmV, 0, 0, 0, g.kvh, page[i], &v_full[vs], pol);
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                nv = n + 1;
                if (j == g.blk0 && a.q_tma) {
                    // the segment's Q, behind its first block: the earlier segment still reads its own
                    if (lane == 0) {
                        if (seg > 0) ok = mbar_wait_for(q_empty, (seg - 1) & 1, a.timeout_ns, a.err);
#pragma unroll
                        for (int t = 0; t < MT; t++) {
                            if (!ok || t * 128 >= g.rows) break;
                            uint8_t* dst = qs + t * Q_TILE;
                            const int tok = s.q0 + (g.row0 + t * 128) / a.G;
                            mbar_arrive_expect_tx(&q_full[t], Q_TILE);
                            tma_load_3d(dst, &tmQ, 0, g.kvh * a.G, tok, &q_full[t]);
                            tma_load_3d(dst + Q_TILE / 2, &tmQ, 64, g.kvh * a.G, tok, &q_full[t]);
                            qn[t]++;
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) break;
                }
            }
            seg++;
        }
        // every issued copy must land before the CTA exits
        if (lane == 0) {
            for (int i = 0; i < KST && i < nk; i++)
                mbar_wait_for(&k_full[i], ((i + (nk - 1 - i) / KST * KST) / KST) & 1, DRAIN_NS, a.err);
            for (int i = 0; i < VST && i < nv; i++)
                mbar_wait_for(&v_full[i], ((i + (nv - 1 - i) / VST * VST) / VST) & 1, DRAIN_NS, a.err);
#pragma unroll
            for (int t = 0; t < MT; t++)
                if (qn[t] > 0) mbar_wait_for(&q_full[t], (qn[t] - 1) & 1, DRAIN_NS, a.err);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        // S runs up to two parts ahead of P V, in the other buffer than the softmax reads: neither waits
        // for the other
        const uint32_t idesc_s = umma_idesc_f16(128, SW, false, false);
        const uint32_t idesc_o = umma_idesc_f16(128, D, false, true);
        const uint64_t qd = umma_desc_sw128(smem_u32(qs), 16, 1024);
        const uint64_t kd = umma_desc_sw128(smem_u32(kring), 16, 1024);
        const uint64_t vd = umma_desc_sw128(smem_u32(vring), HALF_TILE, 1024);
        bool ok = true;
        int n = 0;                                      // blocks before this segment
        int done_parts[MT], q_seen[MT];                 // of each tile, before this segment
#pragma unroll
        for (int t = 0; t < MT; t++) done_parts[t] = q_seen[t] = 0;
        while (ok && walk.next(a, &g, &s, &w, &pos_hi, lane)) {
            const int nt = (g.rows + 127) / 128, nb = g.blk1 - g.blk0, parts = nb * U;
            if (elect_one()) {
                auto wait = [&](uint64_t* bar, int phase) { return mbar_wait_for(bar, phase & 1, a.timeout_ns, a.err); };
                // S of part x (of this segment), tile t (offsets in descriptors: 16 bytes)
                auto qk = [&](int x, int t, int buf) {
                    const int kn = n + x / U;
                    const uint64_t kb = kd + (uint64_t)(kn % KST * (KV_BLK / 16) + x % U * (SW * 128 / 16));
                    const uint64_t qb = qd + (uint64_t)(t * (Q_TILE / 16));
                    const uint32_t d = tmem + t * COLS + buf * SW;
#pragma unroll
                    for (int kk = 0; kk < 8; kk++)
                        umma_f16(d, qb + ((kk >> 2) * (Q_TILE / 2) + (kk & 3) * 32) / 16,
                                 kb + ((kk >> 2) * (KV_BLK / 2) + (kk & 3) * 32) / 16, idesc_s, kk != 0);
                    umma_commit(&s_full[t * 2 + buf]);
                    if (t == nt - 1 && x % U == U - 1) {
                        umma_commit(&k_empty[kn % KST]);
                        if (x == parts - 1) umma_commit(q_empty);
                    }
                };
                // S of part x for every tile; its buffer's P belongs to part x - 2, or to the earlier
                // segment, all of whose P has been read when its last has
                auto qk_all = [&](int x) {
                    if (x >= parts) return;
                    if (x % U == 0) ok = wait(&k_full[(n + x / U) % KST], (n + x / U) / KST);
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        if (t >= nt || !ok) break;
                        const int c = done_parts[t] + x, before = x < 2 ? done_parts[t] - 1 : c - 2;
                        if (x == 0) ok = wait(&q_full[t], q_seen[t]);
                        if (ok && before >= 0) ok = wait(&o_done[t * 2 + (before & 1)], before >> 1);
                        if (!ok) break;
                        tc_fence_after_sync();
                        qk(x, t, c & 1);
                    }
                };
                qk_all(0);
                if (ok) qk_all(1);
                for (int x = 0; x < parts && ok; x++) {
                    const int vn = n + x / U, vs = vn % VST;
                    const uint64_t vb = vd + (uint64_t)(vs * (KV_BLK / 16) + x % U * (SW / PAGE * KV_TILE / 16));
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        if (t >= nt || !ok) break;
                        const int c = done_parts[t] + x, buf = c & 1;
                        const uint32_t sb = tmem + t * COLS + buf * SW, o = tmem + t * COLS + 2 * SW;
#pragma unroll
                        for (int h = 0; h < PH; h++) {
                            if (ok) ok = wait(&p_full[(t * 2 + buf) * PH + h], c >> 1);
                            if (ok && t == 0 && h == 0 && x % U == 0) ok = wait(&v_full[vs], vn / VST) && wait(&v_ready[vs], vn / VST);
                            if (!ok) break;
                            tc_fence_after_sync();
#pragma unroll
                            for (int pg = 4 * h; pg < 4 * h + 4; pg++)
                                umma_f16_ts(o, sb + pg * 8, vb + pg * (KV_TILE / 16), idesc_o, pg != 0 || x != 0);
                        }
                        if (!ok) break;
                        umma_commit(&o_done[t * 2 + buf]);
                        if (t == nt - 1 && x % U == U - 1) umma_commit(&v_empty[vs]);
                    }
                    if (ok) qk_all(x + 2);
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            n += nb;
#pragma unroll
            for (int t = 0; t < MT; t++)
                if (t < nt) {
                    done_parts[t] += parts;
                    q_seen[t]++;
                }
        }
        if (elect_one()) umma_commit(done);
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- V of masked blocks
        // 0 * inf is NaN in the product: V rows behind the sequence and values that are not finite
        // are zeroed before P V; the latter are made up for where they are seen (epilogue). Every
        // block passes here, in order, so that no phase of v_ready can be mistaken for another.
        bool ok = true;
        int n = 0;
        while (ok && walk.next(a, &g, &s, &w, &pos_hi, lane)) {
            for (int j = g.blk0; j < g.blk1 && ok; j++, n++) {
                const int vs = n % VST, kbase = w.first + j * BLK;
                ok = __all_sync(0xffffffffu, mbar_wait_for(&v_full[vs], (n / VST) & 1, a.timeout_ns, a.err));
                if (!ok) break;
                if (!(kbase + BLK <= s.ctx && (a.window <= 0 || (long long)pos_hi - kbase < a.window))) {
                    uint8_t* vb = vring + vs * KV_BLK;
                    bool found = false;
                    // pages that every row sees whole are left; a window reaches all of them
                    const int pg0 = a.window > 0 ? 0 : max(0, min(BLK_PAGES, (s.ctx - kbase) / PAGE));
#pragma unroll 4
                    for (int c = pg0 * 256 + threadIdx.x - 64; c < BLK * 16; c += 64) {
                        // chunk c: page c / 256, half, token, 16-byte piece (swizzled; all pieces of
                        // a 128-byte row are treated alike)
                        const int key = (c >> 8) * PAGE + ((c >> 3) & 15);
                        uint4* at = reinterpret_cast<uint4*>(vb + c * 16);
                        uint4 v = *at;
                        bool f = false;
                        auto fix = [&](uint32_t& x) {
                            uint32_t keep = 0xffffffffu;
                            if ((x & 0x7c00u) == 0x7c00u) keep &= 0xffff0000u;
                            if ((x & 0x7c000000u) == 0x7c000000u) keep &= 0x0000ffffu;
                            x &= keep;
                            f |= keep != 0xffffffffu;
                        };
                        fix(v.x);
                        fix(v.y);
                        fix(v.z);
                        fix(v.w);
                        const bool out = kbase + key >= s.len;
                        if (out) v = make_uint4(0u, 0u, 0u, 0u);
                        if (f || out) *at = v;
                        found |= f && !out;
                    }
                    if (found) *odd = 1;
                    fence_proxy_async_smem();
                }
                mbar_arrive(&v_ready[vs]);
            }
        }
    }
    } else {
        // ---------------------------------------------------------------- softmax: a row per thread
        const int t = (warp - 4) >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;              // row of the tile
        const uint32_t trow = tmem + t * COLS + ((uint32_t)(quarter * 32) << 16);
        const uint32_t orow_t = trow + 2 * SW;        // this thread's row of O
        bool ok = true;
        int cnt = 0;                                    // parts of this tile
        auto o_wait = [&](int c) {
            return __all_sync(0xffffffffu, mbar_wait_for(&o_done[t * 2 + (c & 1)], (c >> 1) & 1, a.timeout_ns, a.err));
        };
        while (walk.next(a, &g, &s, &w, &pos_hi, lane)) {
            const int nt = (g.rows + 127) / 128, parts = (g.blk1 - g.blk0) * U;
            if (t < nt) {
                const int rr = g.row0 + t * 128 + r;
                Row row;
                row.set(a, s, rr, g.row0 + g.rows, g.kvh);
                const size_t orow = (size_t)(s.q0 + max(row.i, 0)) * a.Hq + g.kvh * a.G + (rr - max(row.i, 0) * a.G);
                if (!a.q_tma) {
                    // a group size that does not divide the tile: every thread brings its row. The
                    // tile's earlier S are done: its last o_done was waited for in the epilogue
                    const uint4* src = reinterpret_cast<const uint4*>(a.q + orow * D);
#pragma unroll
                    for (int c = 0; c < 16; c++) {
                        const uint4 v = row.i >= 0 ? __ldg(src + c) : make_uint4(0u, 0u, 0u, 0u);
                        *reinterpret_cast<uint4*>(qs + t * Q_TILE + (c >> 3) * (Q_TILE / 2) + sw128(r, c & 7)) = v;
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(&q_full[t]);
                }

                const bool idle = t * 128 + quarter * 32 >= g.rows;   // only padding rows: no softmax
                float m = -INFINITY, l = 0.f;
                // One part of the row: S from tensor memory, P back. Where every row sees every key S is
                // held in registers, with a version each for plain scores (1), capped ones (2), a
                // distance bias (3) and both (4). Other blocks -- the last one or two, a window's
                // border, scores beyond the polynomial of the cap -- go through rolled loops (0), scores
                // back into tensor memory in between: little code to fetch. (16 x 24 drafts with a cap of 2,
                // scores beyond 0.45 of it in every part: 210 us, with a cap of 30 111.)
                auto soft = [&](auto kind_, int x, int kbase, uint32_t srow) {
                    constexpr int KIND = decltype(kind_)::value;
                    constexpr bool HELD = KIND != 0, CAP = KIND == 2 || KIND == 4, BIAS = KIND >= 3;
                    const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
                    // the scores of columns 32 q .., -inf where unseen
                    uint32_t see0 = ~0u, see1 = ~0u, see2 = ~0u, see3 = ~0u;
                    if (!HELD) {
                        auto seen = [&](int q) {
                            const int p = kbase + 32 * q;
                            return p + 32 <= s.ctx && a.window <= 0 ? ~0u : seen32(a, s, row, p);
                        };
                        see0 = seen(0);
                        see1 = seen(1);
                        if (SW == 128) {
                            see2 = seen(2);
                            see3 = seen(3);
                        }
                    }
                    auto scored = [&](int q, float (&x)[32]) {
                        score_all<EXT>(a, x);
                        if (EXT && a.slopes) {
#pragma unroll
                            for (int c = 0; c < 32; c++) x[c] += bias<true>(a, row.slope2, row.pos, s.pos(a, kbase + 32 * q + c));
                        }
                        const uint32_t v = q == 0 ? see0 : q == 1 ? see1 : q == 2 ? see2 : see3;
#pragma unroll
                        for (int c = 0; c < 32; c++) x[c] = (v >> c) & 1u ? x[c] : -INFINITY;
                    };
                    float row_s[HELD ? SW / 32 : 1][32];
                    float mx = -INFINITY;
                    if (HELD) {
#pragma unroll
                        for (int q = 0; q < SW / 32; q++)
                            tmem_ld32(srow + q * 32, reinterpret_cast<uint32_t(&)[32]>(row_s[HELD ? q : 0]));
                        tmem_ld_wait();
                    }
                    if (CAP) {
                        float lo = INFINITY;
#pragma unroll
                        for (int q = 0; q < SW / 32; q++)
#pragma unroll
                            for (int c = 0; c < 32; c += 2) {
                                const float x0 = row_s[HELD ? q : 0][c], x1 = row_s[HELD ? q : 0][c + 1];
                                mx = fmaxf(mx, fmaxf(x0, x1));
                                lo = fminf(lo, fminf(x0, x1));
                            }
                        // padding rows may be another sequence's: they have no vote, here or below
                        if (__any_sync(0xffffffffu, row.i >= 0 && !(fmaxf(mx, -lo) <= a.cap_lim))) return false;
                    }
#pragma unroll(HELD ? SW / 32 : 1)
                    for (int q = 0; q < SW / 32; q++) {
                        float (&x)[32] = row_s[HELD ? q : 0];
                        if (!HELD) {
                            tmem_ld32(srow + q * 32, reinterpret_cast<uint32_t(&)[32]>(x));
                            tmem_ld_wait();
                            scored(q, x);
                            tmem_st32(srow + q * 32, reinterpret_cast<uint32_t(&)[32]>(x));
                        }
                        if (BIAS) {
                            // slope (kpos - qpos), key by key from the first
                            const float b0 = row.slope2 * (float)(kbase + 32 * q - row.pos);
                            const float2 s2 = make_float2(row.slope2, row.slope2), b2 = make_float2(b0, b0);
#pragma unroll
                            for (int c = 0; c < 32; c += 2) {
                                const float2 v = make_float2(x[c], x[c + 1]);
                                const float2 e = fma2(v, CAP ? cap_factor2(a, v) : sc2, fma2(s2, make_float2(c, c + 1), b2));
                                x[c] = e.x;
                                x[c + 1] = e.y;
                            }
                        }
                        if (KIND != 2) {
                            float m4[4] = {x[0], x[1], x[2], x[3]};
                            if (q == 0 && KIND == 4) mx = -INFINITY;
#pragma unroll
                            for (int c = 4; c < 32; c++) m4[c & 3] = fmaxf(m4[c & 3], x[c]);
                            mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                        }
                    }
                    if (!HELD) tmem_st_wait();
                    // plain and capped scores grow with the product: the greatest is enough
                    mx = KIND == 1 ? fmaf(mx, a.scale_log2, -P_LIFT)
                       : KIND == 2 ? fmaf(mx, cap_factor2(a, make_float2(mx, mx)).x, -P_LIFT) : mx - P_LIFT;
                    if (__any_sync(0xffffffffu, row.i >= 0 && mx > m + RESCALE_THRESHOLD)) {
                        const float mn = fmaxf(m, mx);
                        const float cf = mn == -INFINITY ? 1.f : ex2(m - mn);
                        if (x > 0 && !(ok = o_wait(cnt - 1)))
                            return true;
                        if (x > 0) {                    // O holds the parts before this one now
                            tc_fence_after_sync();
#pragma unroll
                            for (int c0 = 0; c0 < D; c0 += 32) {
                                uint32_t v[32];
                                tmem_ld32(orow_t + c0, v);
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * cf);
                                tmem_st32(orow_t + c0, v);
                            }
                        }
                        l *= cf;
                        m = mn;
                    }
                    const float ms = m == -INFINITY ? 0.f : m;   // a row that saw nothing yet
                    const float2 ms2 = make_float2(-ms, -ms);
                    // l sums the unrounded weights
                    float2 l4[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) l4[i] = make_float2(0.f, 0.f);
#pragma unroll(HELD ? PH : 1)
                    for (int h = 0; h < PH; h++) {        // pages 4h .. 4h + 3
                        uint32_t pk[32];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            float (&x)[32] = row_s[HELD ? 2 * h + u : 0];
                            if (!HELD) {
                                tmem_ld32(srow + (2 * h + u) * 32, reinterpret_cast<uint32_t(&)[32]>(x));
                                tmem_ld_wait();
                            }
#pragma unroll
                            for (int c = 0; c < 32; c += 2) {
                                const float2 v = make_float2(x[c], x[c + 1]);
                                // plain and capped: the score is a factor in the exponent
                                const float2 e = KIND == 1 ? fma2(v, sc2, ms2)
                                               : KIND == 2 ? fma2(v, cap_factor2(a, v), ms2) : add2(v, ms2);
                                const float2 p = make_float2(ex2(e.x), ex2(e.y));
                                l4[(c >> 1) & 3] = add2(l4[(c >> 1) & 3], p);
                                pk[u * 16 + (c >> 1)] = pack_half2(p.x, p.y);
                            }
                        }
                        // P of pages 0-3 goes over S columns 0-31, pages 4-7 over 32-63: those are in
                        // registers by now
                        tmem_st32(srow + h * 32, pk);
                        tmem_st_wait();
                        tc_fence_before_sync();
                        mbar_arrive(&p_full[(t * 2 + (cnt & 1)) * PH + h]);
                    }
                    const float2 l2 = add2(add2(l4[0], l4[1]), add2(l4[2], l4[3]));
                    l += l2.x + l2.y;
                    return true;
                };
                const bool capped = EXT && a.cap_log2 > 0.f, biased = EXT && a.slopes;
                for (int x = 0; x < parts; x++) {
                    const int kbase = w.first + g.blk0 * BLK + x * SW;
                    const bool whole = kbase + SW <= s.ctx && (a.window <= 0 || (long long)pos_hi - kbase < a.window);
                    const uint32_t srow = trow + (cnt & 1) * SW;
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_for(&s_full[t * 2 + (cnt & 1)], (cnt >> 1) & 1, a.timeout_ns, a.err));
                    if (!ok) continue;
                    if (idle) {                         // their P is whatever S held: no other row reads it
                        for (int h = 0; h < PH; h++) mbar_arrive(&p_full[(t * 2 + (cnt & 1)) * PH + h]);
                        cnt++;
                        continue;
                    }
                    tc_fence_after_sync();
                    if (kbase >= s.len) {               // a part behind the sequence: weights of 0 (2 us less
                                                        // than masking it: 16 x 24 drafts 106 us)
                        uint32_t zero[32];
#pragma unroll
                        for (int c = 0; c < 32; c++) zero[c] = 0u;
#pragma unroll
                        for (int h = 0; h < PH; h++) {
                            tmem_st32(srow + h * 32, zero);
                            tmem_st_wait();
                            tc_fence_before_sync();
                            mbar_arrive(&p_full[(t * 2 + (cnt & 1)) * PH + h]);
                        }
                        cnt++;
                        continue;
                    }
                    bool did = false;
                    if (whole && !EXT) did = soft(std::integral_constant<int, 1>{}, x, kbase, srow);
                    if (EXT && whole && capped && !biased) did = soft(std::integral_constant<int, EXT ? 2 : 1>{}, x, kbase, srow);
                    if (EXT && whole && !capped && biased) did = soft(std::integral_constant<int, EXT ? 3 : 1>{}, x, kbase, srow);
                    if (EXT && whole && capped && biased) did = soft(std::integral_constant<int, EXT ? 4 : 1>{}, x, kbase, srow);
                    if (!did) soft(std::integral_constant<int, 0>{}, x, kbase, srow);
                    cnt++;
                }
                // epilogue: the last P V has landed
                if (ok) ok = o_wait(cnt - 1);
                if (ok) {
                    tc_fence_after_sync();
                    const bool full = g.blk0 == 0 && g.blk1 == g.nblk;
                    const float inv = l != 0.f ? 1.f / l : 0.f;
                    const float lse_v = l != 0.f ? ((m == -INFINITY ? 0.f : m) + lg2(l)) * LN2 : -INFINITY;
                    const size_t slot0 = ((size_t)blockIdx.x * 2 + (g.blk0 == 0)) * C::ROWS;
#pragma unroll
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld32(orow_t + c0, v);
                        tmem_ld_wait();
                        float o[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __uint_as_float(v[i]) * inv;
                        if (*odd) {
                            // values of seen keys that were zeroed above: an infinity or NaN that
                            // meets a weight is the result
                            const int e = min(s.len, w.first + g.blk1 * BLK);
                            for (int p = w.first + g.blk0 * BLK; p < e; p++) {
                                const int k0 = w.first + (p - w.first) / BLK * BLK;
                                if (k0 + BLK <= s.ctx && (a.window <= 0 || (long long)pos_hi - k0 < a.window)) {
                                    p = k0 + BLK - 1;             // a whole block: nothing was zeroed
                                    continue;
                                }
                                if (!row.sees(a, s, p, s.pos(a, p))) continue;
                                const int pg = __ldg(a.indices + s.page0 + p / PAGE);
                                if (pg < 0 || pg >= a.num_pages) continue;
                                const __half* vr = a.v + (((size_t)pg * PAGE + p % PAGE) * a.Hkv + g.kvh) * D + c0;
#pragma unroll
                                for (int i = 0; i < 32; i++) {
                                    const float y = __half2float(vr[i]);
                                    if (!(fabsf(y) <= 65504.f)) o[i] += y;
                                }
                            }
                        }
                        if (row.i >= 0) {
                            if (full) {
                                uint4* dst = reinterpret_cast<uint4*>(a.out + orow * D + c0);
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    dst[i] = make_uint4(pack_half2(o[8 * i], o[8 * i + 1]), pack_half2(o[8 * i + 2], o[8 * i + 3]),
                                                        pack_half2(o[8 * i + 4], o[8 * i + 5]), pack_half2(o[8 * i + 6], o[8 * i + 7]));
                            } else {
                                // [dims / 4][rows]: the threads of a warp write side by side
                                float4* dst = reinterpret_cast<float4*>(a.part_o) + (slot0 * (D / 4) + (c0 / 4) * C::ROWS) + t * 128 + r;
#pragma unroll
                                for (int i = 0; i < 8; i++)
                                    dst[i * C::ROWS] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                            }
                        }
                    }
                    if (row.i >= 0) {
                        if (full) a.lse[orow] = lse_v;
                        else a.part_lse[slot0 + t * 128 + r] = lse_v;
                    }
                    tc_fence_before_sync();
                }
            }
        }
    }
    // every MMA must have finished before tensor memory is released
    if (threadIdx.x == 0) mbar_wait_for(done, 0, DRAIN_NS, a.err);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
}

// Joins the units that more than one CTA worked on. A CTA takes 32 rows of a unit at a time: the
// lanes are the rows (a partial's rows lie side by side), and the result goes through shared memory
// so that whole rows are written. Its eight warps have 16 of the dims each; with SPLIT (few rows,
// each in many pieces) they share the pieces of one such 16 between them, and a row's dims are
// eight CTAs' work. grid = (row parts (* 8), B).
template <int MT, bool SPLIT>
__global__ void __launch_bounds__(256) tile_merge_kernel(const Args a, int ctas) {
    constexpr int ROWS = Cfg<MT>::ROWS;
    __shared__ long long s_before, s_all;
    __shared__ uint2 s_out[SPLIT ? 1 : 32][D / 4 + 1];
    __shared__ float4 s_acc[SPLIT ? 8 : 1][4][32];
    __shared__ float s_w[8][32];
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < 2) {
        const long long x = blocks_before<ROWS>(a, warp ? a.B : b, lane);
        if (lane == 0) (warp ? s_all : s_before) = x;
    }
    const Seq s(a, b);
    int lo = 0, hi;
    if (a.window > 0) pos_range(a, s, lane, &lo, &hi);
    const Work w = work_of<ROWS>(a, s, lo);
    if (s.T > a.max_q && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, DEVERR_BOUND);
    __syncthreads();
    const Share sh(s_all, ctas);
    const int parts = (w.nrows + 31) / 32, total = parts * a.Hkv * (SPLIT ? 8 : 1);   // 32 rows of one kv head
    const int c_first = SPLIT ? warp : 0, c_step = SPLIT ? 8 : 1;
    for (int y = blockIdx.x; y < total; y += gridDim.x) {
        const int x = SPLIT ? y >> 3 : y, dims = SPLIT ? y & 7 : warp;
        const int kvh = x / parts, row0 = (x - kvh * parts) * 32, z = row0 / ROWS;
        const long long u0 = s_before + (long long)(z * a.Hkv + kvh) * w.nblk;
        const int c0 = sh.owner(u0), c1 = sh.owner(u0 + w.nblk - 1);
        if (c0 == c1) continue;                                   // written by the CTA itself
        const int rr = row0 + lane, r = rr - z * ROWS;
        auto slot = [&](int c) { return ((size_t)c * 2 + (c == c0)) * ROWS; };
        float m = -INFINITY;
        bool nan = false;
#pragma unroll 8
        for (int c = c0; c <= c1; c++) {
            const float v = rr < w.nrows ? a.part_lse[slot(c) + r] : -INFINITY;
            nan |= v != v;
            m = fmaxf(m, v);
        }
        const bool any = m != -INFINITY || nan;
        float4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        float ws = 0.f;
#pragma unroll 4
        for (int c = c0 + c_first; c <= c1; c += c_step) {
            const float v = rr < w.nrows ? a.part_lse[slot(c) + r] : -INFINITY;
            const float e = any && v != -INFINITY ? ex2((v - m) * LOG2E) : 0.f;
            ws += e;
            const float4* po = reinterpret_cast<const float4*>(a.part_o) + slot(c) * (D / 4) + (dims * 4) * ROWS + r;
            if (e != 0.f) {                                       // nothing to add, and maybe nothing written
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 o = po[i * ROWS];
                    acc[i].x += e * o.x;
                    acc[i].y += e * o.y;
                    acc[i].z += e * o.z;
                    acc[i].w += e * o.w;
                }
            }
        }
        auto orow = [&](int row) {
            const int i = row / a.G;
            return (size_t)(s.q0 + i) * a.Hq + kvh * a.G + (row - i * a.G);
        };
        __syncthreads();                                          // the rows before are written
        if (SPLIT) {
#pragma unroll
            for (int i = 0; i < 4; i++) s_acc[SPLIT ? warp : 0][i][lane] = acc[i];
            s_w[warp][lane] = ws;
            __syncthreads();
            if (warp < 4) {                                       // four of the dims each, warps in order
                float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
                ws = 0.f;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float4 o = s_acc[SPLIT ? k : 0][warp][lane];
                    t.x += o.x;
                    t.y += o.y;
                    t.z += o.z;
                    t.w += o.w;
                    ws += s_w[k][lane];
                }
                const float inv = ws != 0.f ? 1.f / ws : 0.f;
                if (rr < w.nrows) {
                    reinterpret_cast<uint2*>(a.out + orow(rr) * D)[dims * 4 + warp] =
                        make_uint2(pack_half2(t.x * inv, t.y * inv), pack_half2(t.z * inv, t.w * inv));
                    if (dims == 0 && warp == 0) a.lse[orow(rr)] = ws != 0.f ? m + logf(ws) : -INFINITY;
                }
            }
            continue;
        }
        const float inv = ws != 0.f ? 1.f / ws : 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            s_out[SPLIT ? 0 : lane][warp * 4 + i] = make_uint2(pack_half2(acc[i].x * inv, acc[i].y * inv),
                                                               pack_half2(acc[i].z * inv, acc[i].w * inv));
        if (warp == 0 && rr < w.nrows) a.lse[orow(rr)] = ws != 0.f ? m + logf(ws) : -INFINITY;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int q = warp * 4 + i;
            if (row0 + q < w.nrows) reinterpret_cast<uint2*>(a.out + orow(row0 + q) * D)[lane] = s_out[SPLIT ? 0 : q][lane];
        }
    }
}

const void* tile_fn(int MT, bool ext) {
    if (MT == 1) return ext ? (const void*)tile_kernel<1, true> : (const void*)tile_kernel<1, false>;
    return ext ? (const void*)tile_kernel<2, true> : (const void*)tile_kernel<2, false>;
}

ckl_status setup_tiles(const DeviceInfo* di) {
    static ckl_status st[64];
    static std::once_flag once[64];
    std::call_once(once[di->device], [di] {
        cudaError_t e = cudaSuccess;
        for (int MT = 1; MT <= 2 && e == cudaSuccess; MT++)
            for (int ext = 0; ext < 2 && e == cudaSuccess; ext++)
                e = cudaFuncSetAttribute(tile_fn(MT, ext), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         MT == 1 ? Cfg<1>::SMEM : Cfg<2>::SMEM);
        st[di->device] = cuda_status(e, "tree attention setup");
    });
    return st[di->device];
}

size_t part_bytes(int ctas, int rows, size_t* o_bytes) {
    // at most two segments of a CTA are partial
    *o_bytes = align_up((size_t)ctas * 2 * rows * D * sizeof(float), 256);
    return *o_bytes + align_up((size_t)ctas * 2 * rows * sizeof(float), 256);
}

}  // namespace tile

ckl_status encode_half_map(const void* cache, int Hkv, int num_pages, int halves, CUtensorMap* tm) {
    const uint64_t dims[5] = {64, (uint64_t)PAGE, 2, (uint64_t)Hkv, (uint64_t)num_pages};
    const uint64_t strides[4] = {(uint64_t)Hkv * D * 2, 128, (uint64_t)D * 2, (uint64_t)PAGE * Hkv * D * 2};
    const uint32_t box[5] = {64, (uint32_t)PAGE, (uint32_t)halves, 1, 1};
    return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(cache), dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B);
}

ckl_status encode_q_map(const void* q, int N, int Hq, int heads, int tokens, CUtensorMap* tm) {
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)N};
    const uint64_t strides[2] = {(uint64_t)D * 2, (uint64_t)Hq * D * 2};
    const uint32_t box[3] = {64, (uint32_t)heads, (uint32_t)tokens};
    return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B);
}

int tile_count(long long rows) { return rows <= 128 ? 1 : 2; }

size_t tile_workspace(int ctas, long long rows) {
    size_t o;
    return tile::part_bytes(ctas, 128 * tile_count(rows), &o);
}

ckl_status launch_tiles(const ckl_tree_params* p, Args a, void* workspace, int ctas, cudaStream_t s) {
    using namespace tile;
    const DeviceInfo* di = device_info();
    if (!di) return CKL_CUDA_ERROR;
    ckl_status st = setup_tiles(di);
    if (st != CKL_OK) return st;
    const int MT = tile_count((long long)p->max_q * a.G);
    size_t o;
    part_bytes(ctas, 128 * MT, &o);
    a.part_o = static_cast<float*>(workspace);
    a.part_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + o);
    CUtensorMap tmK, tmV;
    st = encode_half_map(p->k_cache, p->Hkv, p->num_pages, 1, &tmK);
    if (st != CKL_OK) return st;
    st = encode_half_map(p->v_cache, p->Hkv, p->num_pages, 2, &tmV);
    if (st != CKL_OK) return st;
    // Q tiles by tensor map: [tokens][heads of the group][64 dims] are the stacked rows in order
    a.q_tma = 128 % a.G == 0;
    CUtensorMap tmQ;
    st = encode_q_map(p->q, p->N, p->Hq, a.q_tma ? a.G : 1, a.q_tma ? 128 / a.G : 1, &tmQ);
    if (st != CKL_OK) return st;
    void* args[] = {&tmK, &tmV, &tmQ, &a};
    const bool ext = p->softcap > 0.f || p->slopes;
    CKL_CUDA_TRY(launch(tile_fn(MT, ext), dim3((unsigned)ctas), dim3(128 + 128 * MT), MT == 1 ? Cfg<1>::SMEM : Cfg<2>::SMEM,
                        s, args, true));
    void* margs[] = {&a, &ctas};
    const long long parts = ((long long)p->max_q * a.G + 31) / 32 * p->Hkv;
    // few rows in many pieces each: split the pieces too
    const bool split = parts * p->B < di->sms;
    const long long want = split ? parts * 8 : parts;
    const unsigned gx = (unsigned)std::max(1LL, std::min(want, (long long)(8 * di->sms + p->B - 1) / p->B));
    const void* fn = MT == 1 ? (split ? (const void*)tile_merge_kernel<1, true> : (const void*)tile_merge_kernel<1, false>)
                             : (split ? (const void*)tile_merge_kernel<2, true> : (const void*)tile_merge_kernel<2, false>);
    CKL_CUDA_TRY(launch(fn, dim3(gx, (unsigned)p->B), dim3(256), 0, s, margs, true));
    return CKL_OK;
}

}  // namespace tree
}  // namespace ckl
