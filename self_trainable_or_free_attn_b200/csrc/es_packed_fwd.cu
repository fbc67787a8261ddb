// Forward attention of packed sequences, and of new tokens to a paged cache, on the 5th-generation tensor cores: one pass over the keys
// with the running maximum and sum of the softmax.
//
//   S = scale Q K^T, P = exp(S - m), l = sum P, O = P V / l, LSE = m + log l
//
// A CTA has two tiles of 128 query rows and walks the keys 128 at a time. The rows of a tile are (token, head) pairs, the `pack` query heads
// of a key head next to one another: all of them read the same K and V, a tile covers 128 / pack tokens, and the causal diagonal
// wastes that much less. One new token of a request still fills `pack` rows.
//   warps 0-3, 4-7  softmax of tile 0 and of tile 1, a thread per row
//   warp 8          issues the MMAs; warp 9 issues the TMA loads; warp 10 finds out what the CTA does next
// Tensor memory: S of tile 0, of tile 1 (128 columns each; P overwrites the first 64 of its S as 16-bit pairs and is the MMA's A operand from
// there), O of tile 0, of tile 1 (D columns each). The MMAs of an iteration are P V of tile 0, Q K^T of tile 0 for the next keys, the same two of
// tile 1: while one tile's softmax runs the tensor cores work for the other. K and V go through one ring in the order of use.
//
// A row's reference m is raised only when its maximum has grown by more than a factor 2^8 since (P stays below 2^8, rounded relative to
// itself): O, in tensor memory, is then rescaled by the row's own thread.
//
// What is hidden must not reach the row, but P = 0 times NaN or infinity is NaN. In the iterations that a mask cuts (the diagonal, the end of the
// keys) the softmax warps of one row tile therefore look through V in shared memory; what is not finite is set to 0 there and added at the end, from
// global memory, to the rows that do see it.
//
// Bound by the exponentials and what surrounds them: an iteration (two tiles, 128 keys) takes 3,430 clocks, of which its MMAs are 2,051. Of a tile's
// turn, 1,870 are softmax, 300 the way from P to the MMA warp, 1,065 the two products, 195 the way back; polynomial exponentials on the FMA
// pipes and P handed over in halves were no faster. fp16, causal, 32,760 tokens, 12 heads on 2: 2.75 ms cold = 1,198 TFLOP/s, 3.06 ms = 1,075
// when it runs on end and the power limit takes the clock down. 24 ragged prompts, 16,383 tokens, 40 heads on 8: 325 us = 780 TFLOP/s.
#include "es_packed_tc.cuh"

namespace es {
namespace packed {

namespace {
constexpr float RAISE = 8.f;                                 // log2 of the factor

template <int D> struct Cfg {
    static constexpr uint32_t TILE = TM * D * 2;             // [d half][128 rows][128 B]
    static constexpr int NSLOT = D == 128 ? 5 : 10;
    static constexpr uint32_t Q = 0, RING = 2 * TILE, CTL = RING + NSLOT * TILE, BYTES = CTL + 768;
};
// What a CTA does next.
struct Work {
    int q0, n_tok;       // first token, tokens (up to two tiles); n_tok <= 0: nothing more
    int base, nk;        // token t sees keys 0 .. base + t (causal), 0 .. nk - 1
    int k0;              // first key row
    int vh, split;
    int i0, end0, end1;  // key tiles of the two row tiles: i0 .. end - 1 (none where end = i0)
    __host__ __device__ __forceinline__ int end(int s) const { return s ? end1 : end0; }
    __host__ __device__ __forceinline__ int last() const { return end0 > end1 ? end0 : end1; }
};
struct Ctl {
    uint64_t qfull[2], qempty[2], full[10], empty[10], sfull[2], pfull[2], ofull[2], drain, wfull[2], wempty[2], want, next;
    alignas(16) uint32_t answer[4];
    uint32_t tmem_base;
    int abort, not_finite[2];
    volatile uint32_t moved[2];  // see mbar_wait_moving
    Work work[2], held;          // held: the last one taken, which a wait that gave up may have kept from being handed on
};
static_assert(sizeof(Ctl) <= 768, "control block");

struct FwdArgs {
    Batch b;
    int64_t slots;                                           // row tile pairs, some of them empty (paged: tiles, with heads and splits)
    int pack, tokens, splits;                                // heads per row group, tokens per 128 rows, CTAs that share a tile's keys
    int vheads;                                              // kv_heads * (G / pack)
    void* o;
    float* lse;
    float *part_o, *part_lse;                                // [split][token][head][D], log2-domain [split][token][head] (splits > 1)
    void* o_rest;                                            // what rounding O left, for the backward's delta; may be null
    const void* v;                                           // for what is not finite
    Rows rv;
    int* status;
    // paged keys: all queries see the first nk tokens of the pages in `list`
    const int* list;
    int nk, pages, log_page;
    int64_t v_page;
};

__device__ __forceinline__ int seen_by(const FwdArgs& a, const Work& w, int t) { return a.b.causal ? min(max(w.base + t + 1, 0), w.nk) : w.nk; }
// Whether row tile s is one of training with rows that see few keys (and one tile of keys in all): what rounding P left is multiplied with V as
// well. delta = rowsum(dO o O) stands against sums over these few keys, where P's roundings do not average out: dQ and dK of sequences of up to
// 32 tokens were off by 1.5 to 1.7 times what their own rounding is (in the norm), and are by 1.00 times with it (and with the same of the backward's P
// and dS). Longer rows go without: full attention 1.41 to 1.47 times from 33 keys on, causal 1.01 at 33, 1.20 at 64, 1.40 at 1,500.
__device__ __forceinline__ bool is_fine(const FwdArgs& a, const Work& w, int s) { return w.i0 == 0 && w.end(s) == 1 && seen_by(a, w, s * a.tokens) <= FEW; }
}  // namespace

// The grid's tile t: split and heads go fastest, and the last tiles of a causal sequence, which see the most keys, first.
template <bool PAGED> __device__ __forceinline__ Work work_of(const FwdArgs& a, int64_t t, int lane) {
    const int wide = a.vheads * a.splits, span = 2 * a.tokens;
    const int64_t x = t / wide;
    const int hs = (int)(t - x * wide);
    Work w{};
    w.vh = hs % a.vheads;
    w.split = hs / a.vheads;
    if (PAGED) {
        w.q0 = (int)x * span;
        w.n_tok = min(span, a.b.Tq - w.q0);
        w.nk = a.nk;
    } else {
        const Piece at = find_piece<true>(a.b.cu_q, a.b.B, a.b.Tq, a.slots, x, span, lane);
        w.q0 = at.first;
        w.n_tok = at.n;
        if (at.n > 0 && at.seq >= 0) {
            w.k0 = a.b.k_at(at.seq);
            w.nk = max(a.b.k_at(at.seq + 1) - w.k0, 0);
            w.base = at.offset + w.nk - at.length;
        }
    }
    auto key_tiles = [&](int s) {
        const int last = min((s + 1) * a.tokens, w.n_tok) - 1;
        return last >= s * a.tokens ? (seen_by(a, w, last) + TN - 1) / TN : 0;
    };
    const int n0 = key_tiles(0), n1 = key_tiles(1), all = max(n0, n1), i1 = (int)((int64_t)all * (w.split + 1) / a.splits);
    w.i0 = (int)((int64_t)all * w.split / a.splits);
    w.end0 = min(max(n0, w.i0), i1);
    w.end1 = min(max(n1, w.i0), i1);
    return w;
}

// FINE: in training.
template <typename T, int D, bool PAGED, bool FINE>
__global__ void __launch_bounds__(THREADS, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ FwdArgs a) {
    using C = Cfg<D>;
    constexpr uint32_t O_COL = 256;
    constexpr int USERS = 10;                                // warps that take each tile's work
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    launch_dependents();                                     // what follows waits for all of this, or (paged) has nothing to do with it
    const uint32_t base = smem_u32(smem);
    Ctl* ctl = reinterpret_cast<Ctl*>(smem + C::CTL);
    volatile int* abort_flag = &ctl->abort;
    if (tid == 0) {
        const int earlier = *reinterpret_cast<volatile int*>(a.status);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->qfull[i]), 1);
            mbar_init(smem_u32(&ctl->qempty[i]), 1);
            mbar_init(smem_u32(&ctl->sfull[i]), 1);
            mbar_init(smem_u32(&ctl->pfull[i]), 128);
            mbar_init(smem_u32(&ctl->ofull[i]), 1);
            mbar_init(smem_u32(&ctl->wfull[i]), 1);
            mbar_init(smem_u32(&ctl->wempty[i]), USERS);
            ctl->work[i].n_tok = 0;
        }
        for (int i = 0; i < C::NSLOT; ++i) {
            mbar_init(smem_u32(&ctl->full[i]), 1);
            mbar_init(smem_u32(&ctl->empty[i]), 1);
        }
        mbar_init(smem_u32(&ctl->drain), 1);
        mbar_init(smem_u32(&ctl->next), 1);
        mbar_init(smem_u32(&ctl->want), 1);
        ctl->held.n_tok = 0;
        ctl->moved[0] = ctl->moved[1] = 0;
        ctl->abort = (base & 1023u) || earlier ? 1 : 0;      // the swizzled tiles need a 1024-byte aligned base
        if (base & 1023u) atomicCAS(a.status, 0, 910);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(&ctl->tmem_base), 512);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(ctl->tmem_base);
    const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
    bool ok = *abort_flag == 0;
    // the CTA's n-th tile, for the warps that work on it; `leave` once they have read all they need of it
    auto enter = [&](int n, Work& w) {
        ok = ok && mbar_wait_moving(smem_u32(&ctl->wfull[n & 1]), (n >> 1) & 1, ctl->moved, abort_flag, a.status, 610);
        if (ok) w = ctl->work[n & 1];
        return ok && w.n_tok > 0;
    };
    auto leave = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->wempty[n & 1]));
    };
    uint32_t issued = 0, q_loads[2] = {0, 0};

    if (warp >= 8) {
        reg_dec<REGS_REST>();
        if (warp == 10) {
            // -------------------------------------------------------- which tiles
            // Paged tiles are all alike: every SM has as many, one more at most. (Taken as CTAs came, some runs had one that did another: 585 us instead of
            // 500 for 256 requests. After a wait that gave up the join writes NaN whatever the parts hold.)
            hand_out<PAGED>(ctl, [&](int64_t t) { return t >= 0 ? work_of<PAGED>(a, t, lane) : Work{}; }, a.slots, ok, lane, abort_flag, a.status, 611);
        } else if (warp == 9) {
            // -------------------------------------------------------- loads: Q, then K(i), V(i) for every i
            const int box = min(TN, PAGED ? 1 << a.log_page : TN), boxes = TN / box;
            const uint32_t qbytes = (uint32_t)(a.tokens * a.pack * D * 2);
            const int per_kv = a.b.G / a.pack;
            if (lane == 0) {
                tma_prefetch_desc(&tmQ);
                tma_prefetch_desc(&tmK);
                tma_prefetch_desc(&tmV);
            }
            uint32_t slot = 0, par = 1;
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                const int kh = w.vh / per_kv, head0 = w.vh * a.pack, i1 = w.last();
                for (int s = 0; s < 2 && ok; ++s) {
                    if (w.end(s) <= w.i0) continue;          // nobody would wait for it
                    ok = mbar_wait_warp(smem_u32(&ctl->qempty[s]), (q_loads[s] & 1) ^ 1, abort_flag, a.status, 600);
                    if (ok && lane == 0) {
                        mbar_arrive_expect_tx(smem_u32(&ctl->qfull[s]), qbytes);
                        for (int d = 0; d < D / 64; ++d)
                            tma_load_3d(base + C::Q + s * C::TILE + d * HALF, &tmQ, smem_u32(&ctl->qfull[s]), 64 * d, head0, w.q0 + s * a.tokens);
                    }
                    __syncwarp();
                    if (ok) ++q_loads[s];
                }
                for (int i = w.i0; i < i1 && ok; ++i) {
                    // paged: a lane per box; a page that is not of the cache, or behind the keys, is loaded as zeros
                    int page = a.pages;
                    if (PAGED && lane < boxes && i * TN + lane * box < w.nk) {
                        const int p = __ldg(a.list + ((i * TN + lane * box) >> a.log_page));
                        if (p >= 0 && p < a.pages) page = p;
                    }
                    for (int x = 0; x < 2 && ok; ++x) {
                        ok = mbar_wait_warp(empty0 + 8 * slot, par, abort_flag, a.status, 601);
                        if (!ok) break;
                        const uint32_t bar = full0 + 8 * slot, dst = base + C::RING + slot * C::TILE;
                        if (lane == 0) {
                            mbar_arrive_expect_tx(bar, C::TILE);
                            if (!PAGED)
                                for (int d = 0; d < D / 64; ++d) tma_load_3d(dst + d * HALF, x ? &tmV : &tmK, bar, 64 * d, kh, w.k0 + i * TN);
                        }
                        __syncwarp();
                        if (PAGED && lane < boxes)
                            for (int d = 0; d < D / 64; ++d)
                                tma_load_4d(dst + d * HALF + lane * box * 128, x ? &tmV : &tmK, bar, 64 * d, kh, (i * TN) & ((1 << a.log_page) - 1), page);
                        __syncwarp();
                        ++issued;
                        if (lane == 0) ctl->moved[0] = issued;
                        if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
                    }
                }
                if (!PAGED && lane == 0) mbar_arrive(smem_u32(&ctl->want));
            }
        } else if (warp == 8) {
            // -------------------------------------------------------- MMAs
            constexpr uint32_t ID_QK = umma_idesc<T>(128, TN, 0, 0), ID_PV = umma_idesc<T>(128, D, 0, 1);
            const uint64_t dk0 = umma_desc_sw128(0, 16, 1024), dv0 = umma_desc_sw128(0, HALF, 1024);
            const uint32_t k_hi = (uint32_t)(dk0 >> 32), k_lo = (uint32_t)dk0, v_hi = (uint32_t)(dv0 >> 32), v_lo = (uint32_t)dv0;
            uint32_t first = 0, products[2] = {0, 0}, tiles[2] = {0, 0};         // K / V tiles, P's and row tiles before this work
            auto slot_of = [&](uint32_t seq) { return seq % C::NSLOT; };
            auto take = [&](uint32_t seq) { ok = ok && mbar_wait_warp(full0 + 8 * slot_of(seq), (seq / C::NSLOT) & 1, abort_flag, a.status, 603); };
            auto issue_qk = [&](int s, uint32_t seq, bool last) {
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t qa = k_lo + ((base + C::Q + s * C::TILE) >> 4), kb = k_lo + ((base + C::RING + slot_of(seq) * C::TILE) >> 4);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = ((ks >> 2) * HALF + (ks & 3) * 32) >> 4;
                        umma_ss_lohi(tmem + s * 128, qa + off, k_hi, kb + off, k_hi, ID_QK, ks > 0);
                    }
                    umma_commit(smem_u32(&ctl->sfull[s]));
                    if (last) umma_commit(smem_u32(&ctl->qempty[s]));
                }
                __syncwarp();
            };
            auto release = [&](uint32_t seq) {
                if (elect_one()) umma_commit(empty0 + 8 * slot_of(seq));
                __syncwarp();
            };
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                w.i0 = uniform(w.i0);
                w.end0 = uniform(w.end0);
                w.end1 = uniform(w.end1);
                const int nt = w.last() - w.i0;
                if (nt <= 0) continue;
                take(first);
                for (int s = 0; s < 2; ++s)
                    if (w.end(s) > w.i0) {
                        ok = ok && mbar_wait_warp(smem_u32(&ctl->qfull[s]), tiles[s] & 1, abort_flag, a.status, 602);
                        if (ok) issue_qk(s, first, w.i0 + 1 == w.end(s));
                        ++tiles[s];
                    }
                if (ok) release(first);
                for (int i = 0; i < nt && ok; ++i) {
                    // (the tiles of K and V are there long before P as a rule: nothing but P is waited for between the products)
                    const uint32_t vseq = first + 2 * i + 1, kseq = vseq + 1;
                    take(vseq);
                    if (i + 1 < nt) take(kseq);
#pragma unroll 1
                    for (int s = 0; s < 2; ++s) {
                        if (w.i0 + i >= w.end(s)) continue;
                        ok = ok && mbar_wait_warp(smem_u32(&ctl->pfull[s]), products[s] & 1, abort_flag, a.status, 604);
                        if (!ok) break;
                        ++products[s];
                        tc_fence_after();
                        const int left = w.end(s) - (w.i0 + i);          // iterations of this row tile, with this one
                        const bool last = s == 1 || w.i0 + i >= w.end(1);    // no other row tile reads these K and V
                        if (elect_one()) {
                            const uint32_t vb = v_lo + ((base + C::RING + slot_of(vseq) * C::TILE) >> 4);
#pragma unroll
                            for (int ks = 0; ks < 8; ++ks)
                                umma_ts_lohi(tmem + O_COL + s * D, tmem + s * 128 + ks * 8, vb + ((ks * 2048) >> 4), v_hi, ID_PV, (i > 0 || ks > 0) ? 1u : 0u);
                            if (FINE && is_fine(a, w, s))
#pragma unroll
                                for (int ks = 0; ks < 8; ++ks)
                                    umma_ts_lohi(tmem + O_COL + s * D, tmem + s * 128 + 64 + ks * 8, vb + ((ks * 2048) >> 4), v_hi, ID_PV, 1u);
                            if (left == 1) umma_commit(smem_u32(&ctl->ofull[s]));
                            if (last) umma_commit(empty0 + 8 * slot_of(vseq));
                            if (left > 1) {
                                // over P, which has been read by then: MMAs run in their order
                                const uint32_t qa = k_lo + ((base + C::Q + s * C::TILE) >> 4), kb = k_lo + ((base + C::RING + slot_of(kseq) * C::TILE) >> 4);
#pragma unroll
                                for (int ks = 0; ks < D / 16; ++ks) {
                                    const uint32_t off = ((ks >> 2) * HALF + (ks & 3) * 32) >> 4;
                                    umma_ss_lohi(tmem + s * 128, qa + off, k_hi, kb + off, k_hi, ID_QK, ks > 0);
                                }
                                umma_commit(smem_u32(&ctl->sfull[s]));
                                if (left == 2) umma_commit(smem_u32(&ctl->qempty[s]));
                            }
                            if (last && i + 1 < nt) umma_commit(empty0 + 8 * slot_of(kseq));
                        }
                        __syncwarp();
                    }
                }
                first += 2 * nt;
            }
            // every MMA issued above has finished before tensor memory is freed
            if (elect_one()) umma_commit(smem_u32(&ctl->drain));
            __syncwarp();
            mbar_wait(smem_u32(&ctl->drain), 0, abort_flag, a.status, 606);
        }
    } else {
        // ------------------------------------------------------------ softmax and epilogue
        reg_inc<REGS_MATH>();
        const int s = warp >> 2, r = tid & 127, row_tok = s * a.tokens + r / a.pack, row_head = r % a.pack;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16), scol = tl + s * 128, ocol = tl + O_COL + s * D;
        const float c = a.b.scale * kLog2e;
        const int box = min(TN, PAGED ? 1 << a.log_page : TN);
        uint32_t first = 0, products = 0, tiles = 0;         // K / V tiles, P's and row tiles before this work
        Work w;
        for (int n = 0; enter(n, w); ++n) {
            const int head = w.vh * a.pack + row_head, end = w.end(s);
            const bool valid = r / a.pack < a.tokens && row_tok < w.n_tok;
            const int vis = valid ? seen_by(a, w, row_tok) : 0;
            const int whole = seen_by(a, w, s * a.tokens) / TN;      // tiles before this one are seen by every row (its first sees the fewest keys)
            float m = -INFINITY, l = 0.f;
            // paged: a bit per box of tile i whose page is not of the cache; looked up a tile ahead
            auto bad_pages = [&](int i) -> uint32_t {
                const int k = i * TN + lane * box;
                const int p = lane * box < TN && k < w.nk ? __ldg(a.list + (k >> a.log_page)) : 0;
                return __ballot_sync(0xffffffffu, p < 0 || p >= a.pages);
            };
            uint32_t bad = 0, bad_next = PAGED && w.i0 < end ? bad_pages(w.i0) : 0u;
            for (int i = w.i0; i < end && ok; ++i) {
                if (PAGED) {
                    bad = bad_next;
                    if (i + 1 < end) bad_next = bad_pages(i + 1);
                }
                ok = mbar_wait_warp(smem_u32(&ctl->sfull[s]), products & 1, abort_flag, a.status, 607);
                if (!ok) break;
                ++products;
                tc_fence_after();
                if (FINE && is_fine(a, w, s)) {
                    // the only tile of these rows, in quarters. (Apart from the rest: its registers are all taken.)
                    const int lim = vis - i * TN;
                    auto quarter = [&](int h, uint32_t* x) {
                        tmem_ld32(scol + 32 * h, x);
                        tmem_wait_ld_regs(x);
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * h + j >= lim) x[j] = 0xff800000u;
                    };
                    float top = -INFINITY;
#pragma unroll 1
                    for (int h = 0; h < 4; ++h) {
                        uint32_t x[32];
                        quarter(h, x);
#pragma unroll
                        for (int j = 0; j < 32; ++j) top = fmaxf(top, __uint_as_float(x[j]));
                    }
                    m = top * c;
                    const float off = m == -INFINITY ? 0.f : -m;
                    uint32_t p[64];
                    // from the last to the first: what is left goes where S has been read, P over S when all of it has
#pragma unroll
                    for (int h = 3; h >= 0; --h) {
                        uint32_t x[32], rest[16];
                        quarter(h, x);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float e0 = ex2_approx(__uint_as_float(x[2 * j]) * c + off), e1 = ex2_approx(__uint_as_float(x[2 * j + 1]) * c + off);
                            l += e0 + e1;
                            p[16 * h + j] = pack2<T>(e0, e1);
                            rest[j] = rest2<T>(e0, e1, p[16 * h + j]);
                        }
                        tmem_st16(scol + 64 + 16 * h, rest);
                    }
#pragma unroll
                    for (int h = 0; h < 4; ++h) tmem_st16(scol + 16 * h, p + 16 * h);
                } else {
                uint32_t x[128];
#pragma unroll
                for (int j = 0; j < 4; ++j) tmem_ld32(scol + 32 * j, x + 32 * j);
#pragma unroll
                for (int j = 0; j < 4; ++j) tmem_wait_ld_regs(x + 32 * j);
                if (i >= whole) {
                    const int lim = vis - i * TN;
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        if (j >= lim) x[j] = 0xff800000u;
                }
                if (PAGED && bad) {
                    // (their keys and values are zeros: nothing of them can reach the row but the logit 0)
                    const int shift = min(a.log_page, 7);
#pragma unroll
                    for (int j = 0; j < TN; j += 16)
                        if ((bad >> (j >> shift)) & 1)
#pragma unroll
                            for (int jj = 0; jj < 16; ++jj) x[j + jj] = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < TN; j += 2) top[(j >> 1) & 3] = fmaxf(fmaxf(top[(j >> 1) & 3], __uint_as_float(x[j])), __uint_as_float(x[j + 1]));
                const float y = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
                const bool raise = m == -INFINITY ? y > -INFINITY : y > m + RAISE;
                if (__any_sync(0xffffffffu, raise)) {
                    const float next = raise ? y : m, shrink = raise ? (m == -INFINITY ? 0.f : ex2_approx(m - next)) : 1.f;
                    m = next;
                    l *= shrink;
                    if (i > w.i0) {
                        // (P V of the iteration before was issued before this S: it has written O)
#pragma unroll 1
                        for (int h = 0; h < D / 32; ++h) {
                            uint32_t o[32];
                            tmem_ld32(ocol + 32 * h, o);
                            tmem_wait_ld_regs(o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                            tmem_st32(ocol + 32 * h, o);
                        }
                    }
                }
                const float off = m == -INFINITY ? 0.f : -m;
                const float2 cc = make_float2(c, c), oo = make_float2(off, off);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    uint32_t p[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 z = __ffma2_rn(make_float2(__uint_as_float(x[32 * h + 2 * j]), __uint_as_float(x[32 * h + 2 * j + 1])), cc, oo);
                        const float2 e = make_float2(ex2_approx(z.x), ex2_approx(z.y));
                        sum = __fadd2_rn(sum, e);
                        // the product takes 16 bits; the sum is of what was not rounded. Each key's weight is off by u at most and as often up as down: O is off by
                        // 1.06 (4 keys) to 1.40 times (1,500) what its own rounding to the type is
                        p[j] = pack2<T>(e.x, e.y);
                    }
                    tmem_st16(scol + 16 * h, p);
                }
                l += sum.x + sum.y;
                }
                if (i >= whole && (s == 0 || i >= w.end0)) {
                    // V rows that some rows of the tile may not see. One owner for both row tiles: tile 0 where it has these keys (it is cut wherever tile 1
                    // is), and its P is waited for before either product is issued
                    const uint32_t vseq = first + 2 * (i - w.i0) + 1, slot = vseq % C::NSLOT;
                    ok = mbar_wait_warp(full0 + 8 * slot, (vseq / C::NSLOT) & 1, abort_flag, a.status, 608);
                    if (!ok) break;
                    if (clean_row<T, D>(smem + C::RING + slot * C::TILE, r)) *reinterpret_cast<volatile int*>(&ctl->not_finite[n & 1]) = 1;
                    fence_proxy_async_smem();
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(smem_u32(&ctl->pfull[s]));
            }
            const bool any = end > w.i0;
            if (any) {
                ok = ok && mbar_wait_warp(smem_u32(&ctl->ofull[s]), tiles & 1, abort_flag, a.status, 609);
                ++tiles;
            }
            if (!ok) break;
            tc_fence_after();
            first += 2 * (w.last() - w.i0);
            const bool fix = any && *reinterpret_cast<volatile int*>(&ctl->not_finite[n & 1]) != 0;
            const float inv = l != 0.f ? 1.f / l : 0.f;      // l = 0: a row without a key; NaN stays NaN
            const int64_t row = (int64_t)(w.q0 + row_tok) * a.b.H + head, part = (int64_t)w.split * a.b.Tq * a.b.H + row;
#pragma unroll 1
            for (int h = 0; h < D / 32; ++h) {
                uint32_t o[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = 0;
                if (any) {
                    tmem_ld32(ocol + 32 * h, o);
                    tmem_wait_ld_regs(o);
                }
                if (!valid) continue;
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(l != 0.f ? __uint_as_float(o[j]) * inv : 0.f);
                if (fix) {
                    const int kh = w.vh / (a.b.G / a.pack);
                    const int from = max(w.i0, seen_by(a, w, 0) / TN) * TN, to = min(vis, w.last() * TN);
                    for (int k = from; k < to; ++k) {
                        const T* vr = static_cast<const T*>(a.v) + (int64_t)kh * a.rv.head + 32 * h;
                        if (PAGED) {
                            const int p = __ldg(a.list + (k >> a.log_page));
                            if (p < 0 || p >= a.pages) continue;
                            vr += p * a.v_page + (int64_t)(k & ((1 << a.log_page) - 1)) * a.rv.token;
                        } else {
                            vr += (int64_t)(w.k0 + k) * a.rv.token;
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float e = to_float(vr[j]);
                            if (!(fabsf(e) < INFINITY)) o[j] = __float_as_uint(__uint_as_float(o[j]) + e);
                        }
                    }
                }
                if (PAGED || a.splits > 1) {
                    if (any)
#pragma unroll
                        for (int j = 0; j < 4; ++j) store8(a.part_o + part * D + 32 * h + 8 * j, o + 8 * j);
                } else {
                    uint32_t p[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) p[j] = pack2<T>(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
                    store8(static_cast<T*>(a.o) + row * D + 32 * h, p);
                    store8(static_cast<T*>(a.o) + row * D + 32 * h + 16, p + 8);
                    if (a.o_rest) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) p[j] = rest2<T>(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]), p[j]);
                        store8(static_cast<T*>(a.o_rest) + row * D + 32 * h, p);
                        store8(static_cast<T*>(a.o_rest) + row * D + 32 * h + 16, p + 8);
                    }
                }
            }
            leave(n);
            if (valid) {
                const float z = l != 0.f ? m + log2f(l) : -INFINITY;
                if (PAGED || a.splits > 1) a.part_lse[part] = z;
                else a.lse[(int64_t)head * a.b.Tq + w.q0 + row_tok] = z * kLn2;
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    if (warp == 9 && lane == 0 && *abort_flag) {
        // a wait gave up: give the loads a moment (100 us in all) to land before shared memory goes away
        const uint64_t t_end = global_timer_ns() + 100000ull;
        for (int s = 0; s < 2; ++s)
            while (q_loads[s] && !mbar_try_wait(smem_u32(&ctl->qfull[s]), (q_loads[s] - 1) & 1) && global_timer_ns() < t_end) {}
        for (uint32_t back = 1; back <= (uint32_t)C::NSLOT && back <= issued; ++back) {
            const uint32_t sq = issued - back;
            while (!mbar_try_wait(full0 + 8 * (sq % C::NSLOT), (sq / C::NSLOT) & 1) && global_timer_ns() < t_end) {}
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (*abort_flag) {
        // NaN in the tiles that the CTA had taken and may not have finished: the caller's memory is not initialised
        for (int x = 0; x < 3; ++x) {
            const Work w = x < 2 ? ctl->work[x] : ctl->held;
            for (int e = tid; e < w.n_tok * a.pack; e += THREADS) {
                const int head = w.vh * a.pack + e % a.pack;
                const int64_t row = (int64_t)(w.q0 + e / a.pack) * a.b.H + head;
                if (PAGED || a.splits > 1) {
                    a.part_lse[(int64_t)w.split * a.b.Tq * a.b.H + row] = __uint_as_float(kNaN32);
                    for (int d = 0; d < D; ++d) a.part_o[((int64_t)w.split * a.b.Tq * a.b.H + row) * D + d] = __uint_as_float(kNaN32);
                } else {
                    a.lse[(int64_t)head * a.b.Tq + w.q0 + e / a.pack] = __uint_as_float(kNaN32);
                    for (int d = 0; d < D / 2; ++d) reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + row * D)[d] = kNaN16x2;
                }
            }
        }
    }
}

// o = sum_p 2^(z_p - M) o_p / sum_p 2^(z_p - M), a warp per row, a lane per part's LSE (at most 32 parts). What a part without a key (z =
// -inf) holds was not written and does not count.
template <typename T, int D>
__global__ void __launch_bounds__(256) merge_kernel(const float* part_o, const float* part_lse, T* o, T* o_rest, float* lse, int parts, int Tq, int H) {
    constexpr int C = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)Tq * H, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    wait_prerequisites();
    if (row >= rows) return;
    const float z = lane < parts ? part_lse[lane * rows + row] : -INFINITY;
    float top = z;
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float w = z == -INFINITY ? 0.f : z != z ? z : exp2f(z - top);
    float acc[C] = {}, sum = w;
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float* src = part_o + row * D + C * lane;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
        const float wp = __shfl_sync(0xffffffffu, w, p);
        float v[C];
        load_floats<C>(src + p * rows * D, v);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] += wp == 0.f ? 0.f : v[c] * wp;
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int c = 0; c < C / 2; ++c) {
        const float x = sum != 0.f ? acc[2 * c] * inv : 0.f, y = sum != 0.f ? acc[2 * c + 1] * inv : 0.f;
        const uint32_t p = pack2<T>(x, y);
        reinterpret_cast<uint32_t*>(o + row * D + C * lane)[c] = p;
        if (o_rest) reinterpret_cast<uint32_t*>(o_rest + row * D + C * lane)[c] = rest2<T>(x, y, p);
    }
    if (lane == 0) lse[(row % H) * Tq + row / H] = sum != 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

template <typename T, int D>
static int launch(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, FwdArgs a, cudaStream_t st) {
    CUtensorMap tq, tk, tv;
    // (a batch without keys loads none, but a map needs an extent)
    const long long tk_rows = a.b.Tk ? a.b.Tk : a.b.Tq;
    if (!a.b.Tk) { k = v = q; rk = rv = rq; }
    if (int rc = make_rows_map<T>(&tq, q, D, a.b.H, a.b.Tq, rq, a.pack, a.tokens)) return rc;
    if (int rc = make_rows_map<T>(&tk, k, D, a.b.Hk, tk_rows, rk, 1, TN)) return rc;
    if (int rc = make_rows_map<T>(&tv, v, D, a.b.Hk, tk_rows, rv, 1, TN)) return rc;
    auto kern = a.o_rest ? packed_fwd_kernel<T, D, false, true> : packed_fwd_kernel<T, D, false, false>;
    if (int rc = opt_in_shared_memory((const void*)kern, (int)Cfg<D>::BYTES)) return rc;
    a.slots = piece_slots(a.b.Tq, 2 * a.tokens, a.b.B);
    const int64_t grid = (int64_t)a.vheads * a.splits * a.slots;
    if (grid > 0x7FFFFFFF) return set_error(-1, "es_packed_attn_fwd: too many tiles");
    kern<<<(unsigned)grid, THREADS, Cfg<D>::BYTES, st>>>(tq, tk, tv, a);
    ES_CHECK_LAUNCH("packed_fwd_kernel");
    if (a.splits > 1) {
        const cudaError_t e = launch_dependent(merge_kernel<T, D>, dim3((unsigned)(((int64_t)a.b.Tq * a.b.H + 7) / 8)), dim3(256), 0, st, (const float*)a.part_o,
                                               (const float*)a.part_lse, static_cast<T*>(a.o), static_cast<T*>(a.o_rest), a.lse, a.splits, a.b.Tq, a.b.H);
        if (e != cudaSuccess) return set_error(-2, cudaGetErrorString(e));
        ES_CHECK_LAUNCH("merge_kernel");
    }
    return 0;
}

// CTAs that share the keys of a pair of row tiles: as many as make the launch shortest, in iterations of 128 keys. What is known of the
// lengths is their mean; START: a tile's start and end; the longest walk is taken for twice the mean of uneven sequences.
static int fwd_splits(int B, int Tq, int Tk, int H, int Hk, int D) {
    constexpr double START = 4, LAUNCH = 3, BYTES = 8e6;     // a launch, and the bytes of the parts that move, in the time of an iteration
    const int sms = sm_count(), pack = rows_pack(H / Hk), span = 2 * (TM / pack);
    const double tiles = H / pack * (Tq / (double)span + 0.5 * B), walk = (double)Tk / std::max(1, B) / TN, longest = B > 1 ? 2 * walk : walk;
    int best = 1;
    double least = 0;
    for (int n = 1; n <= 32; ++n) {
        const double cost = std::max(rounds(tiles * n / sms) * (walk / n + START), longest / n + START) + (n > 1 ? LAUNCH + 8.0 * n * Tq * H * D / BYTES : 0);
        if (n == 1 || cost < 0.9 * least) { best = n; least = cost; }
    }
    return best;
}

long long packed_fwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D) {
    const int n = fwd_splits(B, Tq, Tk, H, Hk, D);
    return n > 1 ? (long long)n * Tq * H * (D + 1) * 4 : 0;
}

// The caller has checked sizes and pointers. ws: packed_fwd_workspace bytes.
int packed_fwd_tc(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, void* o, void* o_rest,
                  float* lse, const Batch& b, int D, int dtype, void* ws, cudaStream_t st) {
    FwdArgs a{};
    a.b = b;
    a.pack = rows_pack(b.G);
    a.tokens = TM / a.pack;
    a.splits = fwd_splits(b.B, b.Tq, b.Tk, b.H, b.Hk, D);
    a.vheads = b.H / a.pack;
    a.part_o = static_cast<float*>(ws);
    a.part_lse = a.part_o + (int64_t)a.splits * b.Tq * b.H * D;
    a.o = o;
    a.o_rest = o_rest;
    a.lse = lse;
    a.v = v;
    a.rv = rv;
    a.status = device_status_ptr();
    if (!a.status) return set_error(-2, "es_packed_attn_fwd: the device status word is not available on this device");
    if (D == 64)
        return dtype == 0 ? launch<__nv_bfloat16, 64>(q, rq, k, rk, v, rv, a, st) : launch<__half, 64>(q, rq, k, rk, v, rv, a, st);
    return dtype == 0 ? launch<__nv_bfloat16, 128>(q, rq, k, rk, v, rv, a, st) : launch<__half, 128>(q, rq, k, rk, v, rv, a, st);
}

// The part of a batch's new tokens that sees a prefix in pages: `parts` fp32 partial results and log2-domain LSEs, [part][token][head]. The caller has
// checked sizes and pointers.
template <typename T, int D>
static int launch_prefix(const void* q, const void* k, CacheRows rk, const void* v, CacheRows rv, FwdArgs a, cudaStream_t st) {
    CUtensorMap tq, tk, tv;
    if (int rc = make_rows_map<T>(&tq, q, D, a.b.H, a.b.Tq, {(int64_t)a.b.H * D, D}, a.pack, a.tokens)) return rc;
    if (int rc = make_pages_map<T>(&tk, k, D, a.b.Hk, 1 << a.log_page, a.pages, rk, TN)) return rc;
    if (int rc = make_pages_map<T>(&tv, v, D, a.b.Hk, 1 << a.log_page, a.pages, rv, TN)) return rc;
    a.slots = (int64_t)a.vheads * a.splits * ((a.b.Tq + 2 * a.tokens - 1) / (2 * a.tokens));
    const int64_t grid = std::min<int64_t>(a.slots, sm_count());
    auto kern = packed_fwd_kernel<T, D, true, false>;
    if (int rc = opt_in_shared_memory((const void*)kern, (int)Cfg<D>::BYTES)) return rc;
    kern<<<(unsigned)grid, THREADS, Cfg<D>::BYTES, st>>>(tq, tk, tv, a);
    ES_CHECK_LAUNCH("packed_fwd_kernel (paged)");
    return 0;
}

int prefix_fwd_tc(const void* q, const void* k, CacheRows rk, const void* v, CacheRows rv, float* part_o, float* part_lse, int parts, const int* list, int prefix_len,
                  int tokens, int H, int Hk, int pages, int log_page, float scale, int D, int dtype, cudaStream_t st) {
    FwdArgs a{};
    a.b = Batch{nullptr, nullptr, 0, tokens, 0, H, Hk, H / Hk, scale, 0};
    a.pack = rows_pack(a.b.G);
    a.tokens = TM / a.pack;
    a.splits = parts;
    a.vheads = H / a.pack;
    a.part_o = part_o;
    a.part_lse = part_lse;
    a.v = v;
    a.rv = Rows{rv.token, rv.head};
    a.v_page = rv.page;
    a.list = list;
    a.nk = prefix_len;
    a.pages = pages;
    a.log_page = log_page;
    a.status = device_status_ptr();
    if (!a.status) return set_error(-2, "es_prefix_attn: the device status word is not available on this device");
    if (D == 64)
        return dtype == 0 ? launch_prefix<__nv_bfloat16, 64>(q, k, rk, v, rv, a, st) : launch_prefix<__half, 64>(q, k, rk, v, rv, a, st);
    return dtype == 0 ? launch_prefix<__nv_bfloat16, 128>(q, k, rk, v, rv, a, st) : launch_prefix<__half, 128>(q, k, rk, v, rv, a, st);
}

}  // namespace packed
}  // namespace es
