// Backward attention of packed sequences on the 5th-generation tensor cores, in two passes with one owner per output row: no atomics, the
// same inputs give the same bits.
//
//   P = exp(scale Q K^T - LSE), dS = P o (dO V^T - delta)
//   dK / dV pass: a CTA owns 128 keys and walks the query rows that see them, 128 (token, head) rows of all heads of the key's group at a time:
//                 S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//   dQ pass:      a CTA owns 128 (token, head) rows and walks their keys, 128 at a time: S = Q K^T, dP = dO V^T, dQ += dS K
// P and dS are written over S and dP in tensor memory, as 16-bit pairs, and are the A operands of the second products from there. (One
// pass instead would save two of seven products, S and dP again, and need dQ added with atomics in the order in which CTAs happen to run.)
//
// What rounding P and dS to 16 bits leaves is off by u at most per pair, as often up as down: dQ, dK and dV of long rows are off by 1.3 to 1.5 times what
// their own rounding to the type is. Tiles with rows that see few keys multiply what these roundings left as well, from the tensor memory that S and dP no
// longer need: there they do not average out, neither in P and dS nor in the forward's O, which delta is summed from.
//
//   warps 0-7  P and dS: a thread has row 32 (warp % 4) + lane and 64 columns, those of warps 4-7 the upper half
//   warp 8     issues the MMAs; warp 9 issues the TMA loads; warp 10 (dK / dV) brings LSE and delta of the walked rows; the next one
//              finds out what the CTA does next
//
// What a mask hides, or what lies in the walked tile behind the sequence, has P = dS = 0, and 0 times NaN or infinity would be NaN: in tiles
// that a mask cuts, values of the walked tiles that are not finite are set to 0 in shared memory once S and dP are there. dS is NaN already
// where they are seen; dV alone gets what is not finite in dO at the end, from global memory.
//
// Bound by the chain S -> P -> dP -> dS of an iteration, which one set of 128 x 128 tiles cannot hide (tensor pipe 56 % busy, exponentials 22 to 28 %). At
// D = 128 accumulators and scores fill tensor memory, the tiles shared memory; at D = 64 (tensor pipe 30 and 34 %) the dK / dV pass leaves 128 columns free,
// the dQ pass 64, and nothing uses them. (Sixteen math warps instead of eight were no faster.) bf16, causal, 32,768 tokens in 8 sequences, 12 heads: dQ 0.91 ms =
// 1,060 TFLOP/s, dK / dV 1.18 ms = 1,090. A CTA that takes tile after tile saves setting up and tearing down: 3 to 10 % of both passes.
#include "es_packed_tc.cuh"

#include <climits>

namespace es {
namespace packed {

namespace {
template <int D> struct Cfg {
    static constexpr uint32_t TILE = TM * D * 2;             // [d half][128 rows][128 B]
    static constexpr int NSLOT = D == 128 ? 5 : 10;
    static constexpr uint32_t Y1 = 0, Y2 = TILE, RING = 2 * TILE, ROWS = RING + NSLOT * TILE;
    static constexpr int NROW = 2;                           // stages of LSE and delta
    static constexpr uint32_t CTL = ROWS + NROW * 2 * TM * 4, BYTES = CTL + 768;
};
static_assert(Cfg<128>::BYTES <= 232448, "shared memory");
// What a CTA does next.
struct Work {
    int first, n_tok;    // the owner's first token, its tokens; n_tok <= 0: nothing more
    int w0, nw;          // first token and tokens of the other side of its sequence, which is walked
    int diag;            // dK / dV: query t sees the owner's keys 0 .. t + diag; dQ: token t of the owner sees keys 0 .. t + diag
    int nt;              // walked tiles
    int head, split;     // key head; dQ: first query head
    int from, per, tile0;        // dK / dV: first query that sees one of the keys, tiles from it to the end, the first of them in this split
    int ones, fine;      // see below
};
struct Ctl {
    uint64_t yfull, yempty, full[10], empty[10], sfull[2], dpfull, pfull, dsfull, rfull[2], rempty[2], gfull, drain, wfull[2], wempty[2], want, next;
    alignas(16) uint32_t answer[4];
    uint32_t tmem_base;
    int abort, not_finite[2];
    volatile uint32_t moved[2];  // see mbar_wait_moving
    Work work[2], held;          // held: the last one taken, which a wait that gave up may have kept from being handed on
};
static_assert(sizeof(Ctl) <= 768, "control block");

struct BwdArgs {
    Batch b;
    int pack, tokens;                                        // heads per row group, tokens per 128 rows
    const float *lse, *delta;
    void *d0, *d1;                                           // dQ, or dK and dV
    int splits;                                              // CTAs that share the rows a key tile is walked by
    float* part;                                             // their sums: [split][dV, dK][key][head][D]
    const void* dout;                                        // for what is not finite
    int64_t slots;                                           // owner tiles, some of them empty
    int behind_q;                                            // the dK / dV pass runs behind the dQ pass, not behind the row sums
    Rows rdo;
    int* status;
};

// A thread's row of an accumulator in tensor memory, columns 32 from .. 32 to - 1, times a factor: to dst, or as it is to part.
template <typename T, int D>
__device__ __forceinline__ void store_row(T* dst, float* part, uint32_t tcol, int from, int to, bool any, bool valid, float factor) {
#pragma unroll 1
    for (int h = from; h < to; ++h) {
        uint32_t g[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) g[j] = 0;
        if (any) {
            tmem_ld32(tcol + 32 * h, g);
            tmem_wait_ld_regs(g);
        }
        if (!valid) continue;
#pragma unroll
        for (int j = 0; j < 32; ++j) g[j] = __float_as_uint(__uint_as_float(g[j]) * factor);
        if (part) {
#pragma unroll
            for (int j = 0; j < 4; ++j) store8(part + 32 * h + 8 * j, g + 8 * j);
        } else {
            uint32_t p[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) p[j] = pack2<T>(__uint_as_float(g[2 * j]), __uint_as_float(g[2 * j + 1]));
            store8(dst + 32 * h, p);
            store8(dst + 32 * h + 16, p + 8);
        }
    }
}

// The wait of a CTA that gives up for the loads in flight (100 us in all), before shared memory goes away.
template <int NSLOT> __device__ __forceinline__ void land(Ctl* ctl, uint32_t owners, uint32_t issued) {
    const uint64_t t_end = global_timer_ns() + 100000ull;
    while (owners && !mbar_try_wait(smem_u32(&ctl->yfull), (owners - 1) & 1) && global_timer_ns() < t_end) {}
    for (uint32_t back = 1; back <= (uint32_t)NSLOT && back <= issued; ++back) {
        const uint32_t sq = issued - back;
        while (!mbar_try_wait(smem_u32(&ctl->full[sq % NSLOT]), (sq / NSLOT) & 1) && global_timer_ns() < t_end) {}
    }
}
}  // namespace

// ---------------------------------------------------------------------------------------------- dK, dV
// Tile t of the grid: splits and heads go fastest; the first keys of a causal sequence, which the most queries see, first.
__device__ __forceinline__ Work kv_work(const BwdArgs& a, int64_t t, int lane) {
    const int wide = a.b.Hk * a.splits;
    const int64_t x = t / wide;
    const int hs = (int)(t - x * wide);
    const Piece at = find_piece<false>(a.b.cu_k, a.b.B, a.b.Tk, a.slots, x, TN, lane);
    Work w{};
    w.head = hs % a.b.Hk;
    w.split = hs / a.b.Hk;
    w.first = at.first;
    w.n_tok = at.n;
    if (at.n <= 0 || at.seq < 0) return w;
    w.w0 = a.b.q_at(at.seq);
    w.nw = max(a.b.q_at(at.seq + 1) - w.w0, 0);
    w.diag = a.b.causal ? at.length - w.nw - at.offset : TN;
    w.from = min(max(-w.diag, 0), w.nw);
    w.per = (w.nw - w.from + a.tokens - 1) / a.tokens;
    const int64_t all = (int64_t)(a.b.G / a.pack) * w.per;
    w.tile0 = (int)(all * w.split / a.splits);
    w.nt = (int)(all * (w.split + 1) / a.splits) - w.tile0;
    // Rows that see one key: their P is 1 whatever the logit, and dS is 0 and not what rounding leaves of a difference (where it is a number). They
    // are the first columns of the first walked tile in causal attention, all rows (more than TM) where the sequence has one key.
    w.ones = at.length == 1 ? TM + 1 : a.b.causal && at.offset == 0 && w.nw >= at.length ? a.pack : 0;
    // Walked tiles that start at query `fine` or before have rows that see few keys, all of them in this tile. What rounding their P and dS left is
    // multiplied as well: such roundings do not average out (es_packed_fwd.cu).
    w.fine = at.offset > 0 ? -1 : a.b.causal ? FEW - 1 - w.diag : at.length <= FEW ? INT_MAX : -1;
    return w;
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
packed_bwd_kv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ BwdArgs a) {
    using C = Cfg<D>;
    constexpr uint32_t DP_COL = 128, DV_COL = 256, DK_COL = 256 + D;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int USERS = 11;                                // warps that take each tile's work
    const uint32_t base = smem_u32(smem);
    Ctl* ctl = reinterpret_cast<Ctl*>(smem + C::CTL);
    volatile int* abort_flag = &ctl->abort;
    if (tid == 0) {
        const int earlier = *reinterpret_cast<volatile int*>(a.status);
        mbar_init(smem_u32(&ctl->yfull), 1);
        mbar_init(smem_u32(&ctl->yempty), 1);
        for (int i = 0; i < C::NSLOT; ++i) {
            mbar_init(smem_u32(&ctl->full[i]), 1);
            mbar_init(smem_u32(&ctl->empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->sfull[i]), 1);
            mbar_init(smem_u32(&ctl->rfull[i]), 32);
            mbar_init(smem_u32(&ctl->rempty[i]), 8);
            mbar_init(smem_u32(&ctl->wfull[i]), 1);
            mbar_init(smem_u32(&ctl->wempty[i]), USERS);
            ctl->work[i].n_tok = 0;
        }
        ctl->held.n_tok = 0;
        ctl->moved[0] = ctl->moved[1] = 0;
        mbar_init(smem_u32(&ctl->want), 1);
        mbar_init(smem_u32(&ctl->dpfull), 1);
        mbar_init(smem_u32(&ctl->pfull), 8);
        mbar_init(smem_u32(&ctl->dsfull), 8);
        mbar_init(smem_u32(&ctl->gfull), 1);
        mbar_init(smem_u32(&ctl->drain), 1);
        mbar_init(smem_u32(&ctl->next), 1);
        ctl->abort = (base & 1023u) || earlier ? 1 : 0;      // the swizzled tiles need a 1024-byte aligned base
        if (base & 1023u) atomicCAS(a.status, 0, 911);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    // rows of the ring's tiles that no load writes (128 is not a multiple of the heads) take part in the products, times 0
    const int loaded = a.tokens * a.pack;
    if (loaded < TM) {
        const int chunks = (TM - loaded) * 8, all = chunks * (D / 64) * C::NSLOT;
        for (int e = tid; e < all; e += THREADS) {
            const int t = e / chunks, c = e % chunks;        // t: (slot, d half)
            *reinterpret_cast<uint4*>(smem + C::RING + t * HALF + loaded * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(&ctl->tmem_base), 512);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (!a.behind_q) wait_prerequisites();                   // (the row sums; behind the dQ pass they are there)
    launch_dependents();
    const uint32_t tmem = uniform(ctl->tmem_base);
    const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
    float* row_lse = reinterpret_cast<float*>(smem + C::ROWS);        // [stage][128]: minus LSE in log2; then minus delta
    float* row_delta = row_lse + C::NROW * TM;
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
    uint32_t issued = 0, owners = 0;
    // walked tile i: query heads head0 .., first token
    auto head_of = [&](const Work& w, int i) { return w.head * a.b.G + (w.tile0 + i) / w.per * a.pack; };
    auto is_fine = [&](const Work& w, int t0) { return t0 <= w.fine; };
    auto token_of = [&](const Work& w, int i) { return w.from + (w.tile0 + i) % w.per * a.tokens; };

    if (warp >= 8) {
        reg_dec<REGS_REST>();
        if (warp == 11) {
            // -------------------------------------------------------- which tiles
            hand_out<false>(ctl, [&](int64_t t) { return t >= 0 ? kv_work(a, t, lane) : Work{}; }, 0, ok, lane, abort_flag, a.status, 611);
        } else if (warp == 9) {
            // -------------------------------------------------------- loads: K, V, then Q(i), dO(i)
            const uint32_t bytes = (uint32_t)(loaded * D * 2);
            uint32_t slot = 0, par = 1;
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                if (w.nt <= 0) {
                    if (lane == 0) mbar_arrive(smem_u32(&ctl->want));
                    continue;
                }
                ok = mbar_wait_warp(smem_u32(&ctl->yempty), (owners & 1) ^ 1, abort_flag, a.status, 620);
                if (!ok) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(smem_u32(&ctl->yfull), 2 * C::TILE);
                    for (int d = 0; d < D / 64; ++d) {
                        tma_load_3d(base + C::Y1 + d * HALF, &tmK, smem_u32(&ctl->yfull), 64 * d, w.head, w.first);
                        tma_load_3d(base + C::Y2 + d * HALF, &tmV, smem_u32(&ctl->yfull), 64 * d, w.head, w.first);
                    }
                }
                __syncwarp();
                ++owners;
                for (int i = 0; i < w.nt && ok; ++i) {
                    const int h0 = head_of(w, i), t0 = w.w0 + token_of(w, i);
                    for (int x = 0; x < 2 && ok; ++x) {
                        ok = mbar_wait_warp(empty0 + 8 * slot, par, abort_flag, a.status, 621);
                        if (!ok) break;
                        if (lane == 0) {
                            const uint32_t bar = full0 + 8 * slot, dst = base + C::RING + slot * C::TILE;
                            mbar_arrive_expect_tx(bar, bytes);
                            for (int d = 0; d < D / 64; ++d) tma_load_3d(dst + d * HALF, x ? &tmDO : &tmQ, bar, 64 * d, h0, t0);
                        }
                        __syncwarp();
                        ++issued;
                        if (lane == 0) ctl->moved[0] = issued;
                        if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
                    }
                }
                if (lane == 0) mbar_arrive(smem_u32(&ctl->want));
            }
        } else if (warp == 10) {
            // -------------------------------------------------------- LSE and delta of each walked tile, once those of two tiles before have been read
            uint32_t seq = 0;
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                for (int i = 0; i < w.nt && ok; ++i, ++seq) {
                    float l[4], d[4];
                    const int h0 = head_of(w, i), t0 = token_of(w, i);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int r = lane + 32 * x, t = t0 + r / a.pack;
                        const bool valid = r < loaded && t < w.nw;
                        const int64_t g = (int64_t)(h0 + r % a.pack) * a.b.Tq + w.w0 + t;
                        const float z = valid ? __ldg(a.lse + g) : -INFINITY;
                        l[x] = z == -INFINITY ? -INFINITY : -z * kLog2e;   // (added to the logit: P of a row without keys, or of none, is 0)
                        d[x] = valid ? -__ldg(a.delta + g) : 0.f;
                    }
                    const uint32_t stage = seq % C::NROW;
                    ok = mbar_wait_warp(smem_u32(&ctl->rempty[stage]), ((seq / C::NROW) & 1) ^ 1, abort_flag, a.status, 622);
                    if (!ok) break;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        row_lse[stage * TM + lane + 32 * x] = l[x];
                        row_delta[stage * TM + lane + 32 * x] = d[x];
                    }
                    mbar_arrive(smem_u32(&ctl->rfull[stage]));
                }
            }
        } else if (warp == 8) {
            // -------------------------------------------------------- MMAs
            constexpr uint32_t ID_S = umma_idesc<T>(128, TM, 0, 0), ID_G = umma_idesc<T>(128, D, 0, 1);
            const uint64_t dk0 = umma_desc_sw128(0, 16, 1024), dx0 = umma_desc_sw128(0, HALF, 1024);
            const uint32_t k_hi = (uint32_t)(dk0 >> 32), k_lo = (uint32_t)dk0, x_hi = (uint32_t)(dx0 >> 32), x_lo = (uint32_t)dx0;
            uint32_t done = 0, tiles = 0;                        // walked tiles and owners before this work
            auto slot_of = [&](uint32_t seq) { return seq % C::NSLOT; };
            auto take = [&](uint32_t seq) { ok = ok && mbar_wait_warp(full0 + 8 * slot_of(seq), (seq / C::NSLOT) & 1, abort_flag, a.status, 623); };
            auto first_product = [&](int x, uint32_t i, bool last) {         // x = 0: S(i) = K Q^T, x = 1: dP(i) = V dO^T; i counts over all works
                take(2 * i + x);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t ya = k_lo + ((base + (x ? C::Y2 : C::Y1)) >> 4), xb = k_lo + ((base + C::RING + slot_of(2 * i + x) * C::TILE) >> 4);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = ((ks >> 2) * HALF + (ks & 3) * 32) >> 4;
                        umma_ss_lohi(tmem + x * DP_COL, ya + off, k_hi, xb + off, k_hi, ID_S, ks > 0);
                    }
                    umma_commit(x ? smem_u32(&ctl->dpfull) : smem_u32(&ctl->sfull[0]));
                    if (x && last) umma_commit(smem_u32(&ctl->yempty));
                }
                __syncwarp();
            };
            auto second_product = [&](int x, uint32_t i, uint32_t more, bool fine) {     // x = 0: dK += dS^T Q, x = 1: dV += P^T dO
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t xb = x_lo + ((base + C::RING + slot_of(2 * i + x) * C::TILE) >> 4), p = tmem + (x ? 0u : DP_COL);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        umma_ts_lohi(tmem + (x ? DV_COL : DK_COL), p + (ks < 4 ? ks * 8 : 64 + (ks - 4) * 8), xb + ((ks * 2048) >> 4), x_hi, ID_G,
                                     ks > 0 ? 1u : more);
                    if (fine)
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            umma_ts_lohi(tmem + (x ? DV_COL : DK_COL), p + 32 + (ks < 4 ? ks * 8 : 64 + (ks - 4) * 8), xb + ((ks * 2048) >> 4), x_hi, ID_G, 1u);
                    umma_commit(empty0 + 8 * slot_of(2 * i + x));
                }
                __syncwarp();
            };
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                const int nt = uniform(w.nt);
                if (nt <= 0) continue;
                ok = ok && mbar_wait_warp(smem_u32(&ctl->yfull), tiles & 1, abort_flag, a.status, 624);
                ++tiles;
                if (ok) first_product(0, done, false);
                if (ok) first_product(1, done, nt == 1);
                const int stop = w.from + w.per * a.tokens;
                int t0 = token_of(w, 0);
                for (int i = 0; i < nt && ok; ++i, ++done) {
                    const bool fine = uniform((int)is_fine(w, t0));
                    t0 = t0 + a.tokens < stop ? t0 + a.tokens : w.from;
                    ok = mbar_wait_warp(smem_u32(&ctl->pfull), done & 1, abort_flag, a.status, 625);
                    if (!ok) break;
                    second_product(1, done, i > 0, fine);
                    if (i + 1 < nt) first_product(0, done + 1, false);           // (over P, which dV has read: MMAs run in their order)
                    ok = ok && mbar_wait_warp(smem_u32(&ctl->dsfull), done & 1, abort_flag, a.status, 626);
                    if (!ok) break;
                    second_product(0, done, i > 0, fine);
                    if (i + 1 < nt) first_product(1, done + 1, i + 2 == nt);
                }
                if (ok && elect_one()) umma_commit(smem_u32(&ctl->gfull));
                __syncwarp();
            }
            // every MMA issued above has finished before tensor memory is freed
            if (elect_one()) umma_commit(smem_u32(&ctl->drain));
            __syncwarp();
            mbar_wait(smem_u32(&ctl->drain), 0, abort_flag, a.status, 627);
        }
    } else {
        // ------------------------------------------------------------ P, dS and epilogue
        reg_inc<REGS_MATH>();
        const int r = tid & 127, ch = warp >> 2;             // key row, half of the columns
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16), scol = tl + 64 * ch, dpcol = tl + DP_COL + 64 * ch;
        const float c = a.b.scale * kLog2e;
        uint32_t done = 0, tiles = 0;                        // walked tiles and owners before this work
        Work w;
        for (int n = 0; enter(n, w); ++n) {
        const int nt = w.nt, nw = w.nw, diag = w.diag, first = w.from, stop = first + w.per * a.tokens, last = w.n_tok - 1, ones = w.ones, fine_to = w.fine;
        int t0 = nt > 0 ? token_of(w, 0) : 0;
        for (int i = 0; i < nt && ok; ++i, ++done) {
            const uint32_t stage = done % C::NROW;
            // the first of the tile's tokens sees the fewest keys; the rows behind the last token are of other sequences
            const bool cut = t0 + diag < last, masked = cut || t0 + a.tokens > nw, fine = t0 <= fine_to;
            ok = mbar_wait_warp(smem_u32(&ctl->rfull[stage]), (done / C::NROW) & 1, abort_flag, a.status, 628) &&
                 mbar_wait_warp(smem_u32(&ctl->sfull[0]), done & 1, abort_flag, a.status, 629);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[64];
            tmem_ld32(scol, x);
            tmem_ld32(scol + 32, x + 32);
            tmem_wait_ld_regs(x);
            tmem_wait_ld_regs(x + 32);
            const int lim = cut ? max(r - diag - t0, 0) * a.pack - 64 * ch : 0;      // columns before it do not see the key
            const int end = min(nw - t0, a.tokens) * a.pack - 64 * ch;               // columns from here on are not rows of the sequence
            const float4* rl = reinterpret_cast<const float4*>(row_lse + stage * TM + 64 * ch);
            // P; one pair in four on the FMA pipes, as many as take no longer than the others take the 16 exponentials a clock of an SM
            auto probabilities = [&](auto cut_tile) {
                const float2 cc = make_float2(c, c);
                uint32_t p[32];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float4 z = rl[j];
                    const float2 z0 = __ffma2_rn(make_float2(__uint_as_float(x[4 * j]), __uint_as_float(x[4 * j + 1])), cc, make_float2(z.x, z.y));
                    const float2 z1 = __ffma2_rn(make_float2(__uint_as_float(x[4 * j + 2]), __uint_as_float(x[4 * j + 3])), cc, make_float2(z.z, z.w));
                    float2 e0 = make_float2(ex2_approx(z0.x), ex2_approx(z0.y));
                    float2 e1 = !decltype(cut_tile)::value && j % 2 == 1 ? ex2_poly(z1) : make_float2(ex2_approx(z1.x), ex2_approx(z1.y));
                    if (decltype(cut_tile)::value) {
                        if (4 * j < lim || 4 * j >= end) e0.x = 0.f;
                        if (4 * j + 1 < lim || 4 * j + 1 >= end) e0.y = 0.f;
                        if (4 * j + 2 < lim || 4 * j + 2 >= end) e1.x = 0.f;
                        if (4 * j + 3 < lim || 4 * j + 3 >= end) e1.y = 0.f;
                    }
                    x[4 * j] = __float_as_uint(e0.x); x[4 * j + 1] = __float_as_uint(e0.y);
                    x[4 * j + 2] = __float_as_uint(e1.x); x[4 * j + 3] = __float_as_uint(e1.y);
                    p[2 * j] = pack2<T>(e0.x, e0.y);
                    p[2 * j + 1] = pack2<T>(e1.x, e1.y);
                }
                tmem_st32(scol, p);
            };
            if (masked) {
                probabilities(std::true_type{});
                // dP of this tile is there too: from here on its Q and dO are read by the second products only
                ok = mbar_wait_warp(smem_u32(&ctl->dpfull), done & 1, abort_flag, a.status, 630);
                if (!ok) break;
                const uint32_t slot = (2 * done + ch) % C::NSLOT;             // half of the threads Q, half dO
                if (clean_row<T, D>(smem + C::RING + slot * C::TILE, r)) *reinterpret_cast<volatile int*>(&ctl->not_finite[n & 1]) = 1;
                fence_proxy_async_smem();
            } else {
                probabilities(std::false_type{});
            }
            if (fine) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t rest[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float p0 = __uint_as_float(x[32 * h + 2 * j]), p1 = __uint_as_float(x[32 * h + 2 * j + 1]);
                        rest[j] = rest2<T>(p0, p1, pack2<T>(p0, p1));
                    }
                    tmem_st16(scol + 32 + 16 * h, rest);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->pfull));
            if (ones && (ones > TM || t0 == first)) {
#pragma unroll
                for (int j = 0; j < 64; ++j)
                    if (j < ones - 64 * ch && fabsf(__uint_as_float(x[j])) < INFINITY) x[j] = 0;
            }
            ok = mbar_wait_warp(smem_u32(&ctl->dpfull), done & 1, abort_flag, a.status, 631);
            if (!ok) break;
            tc_fence_after();
            const float4* rd = reinterpret_cast<const float4*>(row_delta + stage * TM + 64 * ch);
            if (fine) {
                // in halves: dS over dP where that has been read
                uint32_t y[64];
                tmem_ld32(dpcol, y);
                tmem_ld32(dpcol + 32, y + 32);
                tmem_wait_ld_regs(y);
                tmem_wait_ld_regs(y + 32);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t ds[16], rest[16];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float4 z = rd[8 * h + j / 4];
                        const float nd = j % 4 == 0 ? z.x : j % 4 == 1 ? z.y : j % 4 == 2 ? z.z : z.w;
                        const float g = __uint_as_float(x[32 * h + j]) * (__uint_as_float(y[32 * h + j]) + nd);
                        y[32 * h + j] = 32 * h + j < lim || 32 * h + j >= end ? 0u : __float_as_uint(g);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float g0 = __uint_as_float(y[32 * h + 2 * j]), g1 = __uint_as_float(y[32 * h + 2 * j + 1]);
                        ds[j] = pack2<T>(g0, g1);
                        rest[j] = rest2<T>(g0, g1, ds[j]);
                    }
                    tmem_st16(dpcol + 16 * h, ds);
                    tmem_st16(dpcol + 32 + 16 * h, rest);
                }
            } else {
            uint32_t y[64];
            tmem_ld32(dpcol, y);
            tmem_ld32(dpcol + 32, y + 32);
            tmem_wait_ld_regs(y);
            tmem_wait_ld_regs(y + 32);
            auto differences = [&](auto cut_tile) {
                uint32_t ds[32];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float4 z = rd[j];                  // minus delta
                    float2 g0 = __fmul2_rn(make_float2(__uint_as_float(x[4 * j]), __uint_as_float(x[4 * j + 1])),
                                           __fadd2_rn(make_float2(__uint_as_float(y[4 * j]), __uint_as_float(y[4 * j + 1])), make_float2(z.x, z.y)));
                    float2 g1 = __fmul2_rn(make_float2(__uint_as_float(x[4 * j + 2]), __uint_as_float(x[4 * j + 3])),
                                           __fadd2_rn(make_float2(__uint_as_float(y[4 * j + 2]), __uint_as_float(y[4 * j + 3])), make_float2(z.z, z.w)));
                    if (decltype(cut_tile)::value) {         // (0 times what a hidden row holds)
                        if (4 * j < lim || 4 * j >= end) g0.x = 0.f;
                        if (4 * j + 1 < lim || 4 * j + 1 >= end) g0.y = 0.f;
                        if (4 * j + 2 < lim || 4 * j + 2 >= end) g1.x = 0.f;
                        if (4 * j + 3 < lim || 4 * j + 3 >= end) g1.y = 0.f;
                    }
                    ds[2 * j] = pack2<T>(g0.x, g0.y);
                    ds[2 * j + 1] = pack2<T>(g1.x, g1.y);
                }
                tmem_st32(dpcol, ds);
            };
            if (masked) differences(std::true_type{});
            else differences(std::false_type{});
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&ctl->rempty[stage]));
                mbar_arrive(smem_u32(&ctl->dsfull));
            }
            t0 += a.tokens;
            if (t0 >= stop) t0 = first;
        }
        if (nt > 0) ok = ok && mbar_wait_warp(smem_u32(&ctl->gfull), tiles++ & 1, abort_flag, a.status, 632);
        if (!ok) break;
        tc_fence_after();
        w = ctl->work[n & 1];                                // (read again: the loop's registers are few)
        const int64_t row = (int64_t)(w.first + r) * a.b.Hk + w.head;
        const bool valid = r < w.n_tok;
        // warps 0-3 write dV, warps 4-7 dK
        T* dst = static_cast<T*>(ch ? a.d0 : a.d1) + row * D;
        float* part = a.splits > 1 ? a.part + ((int64_t)(2 * w.split + ch) * a.b.Tk * a.b.Hk + row) * D : nullptr;
        store_row<T, D>(dst, part, tl + (ch ? DK_COL : DV_COL), 0, D / 32, w.nt > 0, valid, ch ? a.b.scale : 1.f);
        if (ch == 0 && valid && w.nt > 0 && *reinterpret_cast<volatile int*>(&ctl->not_finite[n & 1])) {
            // what is not finite in dO of the rows of cut tiles that see this key
            for (int i = 0; i < w.nt; ++i) {
                const int t0 = token_of(w, i);
                if (!(t0 + w.diag < w.n_tok - 1 || t0 + a.tokens > w.nw)) continue;
                for (int t = max(t0, r - w.diag); t < min(t0 + a.tokens, w.nw); ++t)
                    for (int h = head_of(w, i); h < head_of(w, i) + a.pack; ++h) {
                        const T* src = static_cast<const T*>(a.dout) + (int64_t)(w.w0 + t) * a.rdo.token + (int64_t)h * a.rdo.head;
                        for (int d = 0; d < D; ++d) {
                            const float e = to_float(src[d]);
                            if (fabsf(e) < INFINITY) continue;
                            if (part) part[d] += e;
                            else dst[d] = from_float<T>(to_float(dst[d]) + e);
                        }
                    }
            }
        }
        leave(n);
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    if (warp == 9 && lane == 0 && *abort_flag) land<C::NSLOT>(ctl, owners, issued);
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
            const int64_t all = (int64_t)a.b.Tk * a.b.Hk * D;
            for (int e = tid; e < w.n_tok * D; e += THREADS) {
                const int64_t at = ((int64_t)(w.first + e / D) * a.b.Hk + w.head) * D + e % D;
                if (a.splits > 1) a.part[2 * w.split * all + at] = a.part[(2 * w.split + 1) * all + at] = __uint_as_float(kNaN32);
                else static_cast<uint16_t*>(a.d0)[at] = static_cast<uint16_t*>(a.d1)[at] = (uint16_t)kNaN16x2;
            }
        }
    }
    wait_prerequisites();                                    // what comes next waits for this kernel, and so for the dQ pass too
}

// ---------------------------------------------------------------------------------------------- dQ
// Tile t of the grid: heads go fastest; the last rows of a causal sequence, which see the most keys, first.
__device__ __forceinline__ Work q_work(const BwdArgs& a, int64_t t, int lane) {
    const int vheads = a.b.H / a.pack;
    const int64_t x = t / vheads;
    const Piece at = find_piece<true>(a.b.cu_q, a.b.B, a.b.Tq, a.slots, x, a.tokens, lane);
    Work w{};
    w.head = (int)(t - x * vheads) * a.pack;
    w.first = at.first;
    w.n_tok = at.n;
    if (at.n <= 0 || at.seq < 0) return w;
    w.w0 = a.b.k_at(at.seq);
    w.nw = max(a.b.k_at(at.seq + 1) - w.w0, 0);
    w.diag = w.nw - at.length + at.offset;
    const int last = at.n - 1;
    // (rows that see few keys, see kv_work; one walked tile)
    w.nt = ((a.b.causal ? min(max(last + w.diag + 1, 0), w.nw) : w.nw) + TN - 1) / TN;
    w.fine = w.nt == 1 && (a.b.causal ? w.diag + 1 : w.nw) <= FEW;
    return w;
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
packed_bwd_q_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ BwdArgs a) {
    using C = Cfg<D>;
    constexpr uint32_t DP_COL = 256, DQ_COL = 384;           // S of even and of odd tiles: columns 0 and 128
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int USERS = 10;                                // warps that take each tile's work
    const uint32_t base = smem_u32(smem);
    Ctl* ctl = reinterpret_cast<Ctl*>(smem + C::CTL);
    volatile int* abort_flag = &ctl->abort;
    if (tid == 0) {
        const int earlier = *reinterpret_cast<volatile int*>(a.status);
        mbar_init(smem_u32(&ctl->yfull), 1);
        mbar_init(smem_u32(&ctl->yempty), 1);
        for (int i = 0; i < C::NSLOT; ++i) {
            mbar_init(smem_u32(&ctl->full[i]), 1);
            mbar_init(smem_u32(&ctl->empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->sfull[i]), 1);
            mbar_init(smem_u32(&ctl->rfull[i]), 32);
            mbar_init(smem_u32(&ctl->rempty[i]), 8);
            mbar_init(smem_u32(&ctl->wfull[i]), 1);
            mbar_init(smem_u32(&ctl->wempty[i]), USERS);
            ctl->work[i].n_tok = 0;
        }
        ctl->held.n_tok = 0;
        ctl->moved[0] = ctl->moved[1] = 0;
        mbar_init(smem_u32(&ctl->want), 1);
        mbar_init(smem_u32(&ctl->dpfull), 1);
        mbar_init(smem_u32(&ctl->pfull), 8);
        mbar_init(smem_u32(&ctl->dsfull), 8);
        mbar_init(smem_u32(&ctl->gfull), 1);
        mbar_init(smem_u32(&ctl->drain), 1);
        mbar_init(smem_u32(&ctl->next), 1);
        ctl->abort = (base & 1023u) || earlier ? 1 : 0;      // the swizzled tiles need a 1024-byte aligned base
        if (base & 1023u) atomicCAS(a.status, 0, 912);
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
    wait_prerequisites();                                    // the row sums
    launch_dependents();
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
    uint32_t issued = 0, owners = 0;

    if (warp >= 8) {
        reg_dec<REGS_REST>();
        if (warp == 10) {
            // -------------------------------------------------------- which tiles
            hand_out<false>(ctl, [&](int64_t t) { return t >= 0 ? q_work(a, t, lane) : Work{}; }, 0, ok, lane, abort_flag, a.status, 611);
        } else if (warp == 9) {
            // -------------------------------------------------------- loads: Q, dO, then K(i), V(i)
            const uint32_t bytes = (uint32_t)(a.tokens * a.pack * D * 2);
            uint32_t slot = 0, par = 1;
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                if (w.nt <= 0) {
                    if (lane == 0) mbar_arrive(smem_u32(&ctl->want));
                    continue;
                }
                ok = mbar_wait_warp(smem_u32(&ctl->yempty), (owners & 1) ^ 1, abort_flag, a.status, 640);
                if (!ok) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(smem_u32(&ctl->yfull), 2 * bytes);
                    for (int d = 0; d < D / 64; ++d) {
                        tma_load_3d(base + C::Y1 + d * HALF, &tmQ, smem_u32(&ctl->yfull), 64 * d, w.head, w.first);
                        tma_load_3d(base + C::Y2 + d * HALF, &tmDO, smem_u32(&ctl->yfull), 64 * d, w.head, w.first);
                    }
                }
                __syncwarp();
                ++owners;
                const int kh = w.head / a.b.G;
                for (int i = 0; i < w.nt && ok; ++i)
                    for (int x = 0; x < 2 && ok; ++x) {
                        ok = mbar_wait_warp(empty0 + 8 * slot, par, abort_flag, a.status, 641);
                        if (!ok) break;
                        if (lane == 0) {
                            const uint32_t bar = full0 + 8 * slot, dst = base + C::RING + slot * C::TILE;
                            mbar_arrive_expect_tx(bar, C::TILE);
                            for (int d = 0; d < D / 64; ++d) tma_load_3d(dst + d * HALF, x ? &tmV : &tmK, bar, 64 * d, kh, w.w0 + i * TN);
                        }
                        __syncwarp();
                        ++issued;
                        if (lane == 0) ctl->moved[0] = issued;
                        if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
                    }
                if (lane == 0) mbar_arrive(smem_u32(&ctl->want));
            }
        } else if (warp == 8) {
            // -------------------------------------------------------- MMAs
            constexpr uint32_t ID_S = umma_idesc<T>(128, TN, 0, 0), ID_G = umma_idesc<T>(128, D, 0, 1);
            const uint64_t dk0 = umma_desc_sw128(0, 16, 1024), dx0 = umma_desc_sw128(0, HALF, 1024);
            const uint32_t k_hi = (uint32_t)(dk0 >> 32), k_lo = (uint32_t)dk0, x_hi = (uint32_t)(dx0 >> 32), x_lo = (uint32_t)dx0;
            uint32_t done = 0, tiles = 0;                        // walked tiles and owners before this work
            auto slot_of = [&](uint32_t seq) { return seq % C::NSLOT; };
            auto first_product = [&](int x, uint32_t i, bool last) {         // x = 0: S(i) = Q K^T, x = 1: dP(i) = dO V^T; i counts over all works
                const uint32_t seq = 2 * i + x;
                ok = ok && mbar_wait_warp(full0 + 8 * slot_of(seq), (seq / C::NSLOT) & 1, abort_flag, a.status, 643);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t ya = k_lo + ((base + (x ? C::Y2 : C::Y1)) >> 4), xb = k_lo + ((base + C::RING + slot_of(seq) * C::TILE) >> 4);
                    const uint32_t d = tmem + (x ? DP_COL : (i & 1) * 128);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = ((ks >> 2) * HALF + (ks & 3) * 32) >> 4;
                        umma_ss_lohi(d, ya + off, k_hi, xb + off, k_hi, ID_S, ks > 0);
                    }
                    umma_commit(x ? smem_u32(&ctl->dpfull) : smem_u32(&ctl->sfull[i & 1]));
                    if (x) umma_commit(empty0 + 8 * slot_of(seq));       // V is needed no more
                    if (x && last) umma_commit(smem_u32(&ctl->yempty));
                }
                __syncwarp();
            };
            Work w;
            for (int n = 0; enter(n, w); ++n) {
                leave(n);
                const int nt = uniform(w.nt);
                if (nt <= 0) continue;
                ok = ok && mbar_wait_warp(smem_u32(&ctl->yfull), tiles & 1, abort_flag, a.status, 644);
                ++tiles;
                if (ok) first_product(0, done, false);
                if (ok) first_product(1, done, nt == 1);
                for (int i = 0; i < nt && ok; ++i, ++done) {
                    if (i + 1 < nt) first_product(0, done + 1, false);           // (over dS of tile i - 1, which dQ has read: MMAs run in their order)
                    ok = ok && mbar_wait_warp(smem_u32(&ctl->dsfull), done & 1, abort_flag, a.status, 646);
                    if (!ok) break;
                    if (i + 1 < nt) first_product(1, done + 1, i + 2 == nt);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t xb = x_lo + ((base + C::RING + slot_of(2 * done) * C::TILE) >> 4), p = tmem + (done & 1) * 128;
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            umma_ts_lohi(tmem + DQ_COL, p + (ks < 4 ? ks * 8 : 64 + (ks - 4) * 8), xb + ((ks * 2048) >> 4), x_hi, ID_G, (i > 0 || ks > 0) ? 1u : 0u);
                        if (w.fine)
#pragma unroll
                            for (int ks = 0; ks < 8; ++ks)
                                umma_ts_lohi(tmem + DQ_COL, p + 32 + (ks < 4 ? ks * 8 : 64 + (ks - 4) * 8), xb + ((ks * 2048) >> 4), x_hi, ID_G, 1u);
                        umma_commit(empty0 + 8 * slot_of(2 * done));
                        if (i + 1 == nt) umma_commit(smem_u32(&ctl->gfull));
                    }
                    __syncwarp();
                }
            }
            // every MMA issued above has finished before tensor memory is freed
            if (elect_one()) umma_commit(smem_u32(&ctl->drain));
            __syncwarp();
            mbar_wait(smem_u32(&ctl->drain), 0, abort_flag, a.status, 647);
        }
    } else {
        // ------------------------------------------------------------ P, dS and epilogue
        reg_inc<REGS_MATH>();
        const int r = tid & 127, ch = warp >> 2;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16), dpcol = tl + DP_COL + 64 * ch;
        const float c = a.b.scale * kLog2e;
        const int tok = r / a.pack, lane_head = r % a.pack;
        uint32_t done = 0, tiles = 0;                        // walked tiles and owners before this work
        Work w;
        for (int n = 0; enter(n, w); ++n) {
        const bool valid = tok < a.tokens && tok < w.n_tok;
        auto seen_by = [&](int t) { return a.b.causal ? min(max(t + w.diag + 1, 0), w.nw) : w.nw; };
        const int vis = valid ? seen_by(tok) : 0, whole = seen_by(0) / TN;
        const int64_t g = (int64_t)(w.head + lane_head) * a.b.Tq + w.first + tok;
        const float z = valid ? a.lse[g] : -INFINITY, off = z == -INFINITY ? -INFINITY : -z * kLog2e, delta = valid ? a.delta[g] : 0.f;
        const int nt = w.nt;
        for (int i = 0; i < nt && ok; ++i, ++done) {
            const uint32_t scol = tl + (done & 1) * 128 + 64 * ch;
            ok = mbar_wait_warp(smem_u32(&ctl->sfull[done & 1]), (done >> 1) & 1, abort_flag, a.status, 649);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[64];
            tmem_ld32(scol, x);
            tmem_ld32(scol + 32, x + 32);
            tmem_wait_ld_regs(x);
            tmem_wait_ld_regs(x + 32);
            const bool masked = i >= whole;
            const int lim = vis - i * TN - 64 * ch;
            // P; one pair in four on the FMA pipes (of tiles that no mask cuts)
            auto probabilities = [&](auto mixed) {
                const float2 cc = make_float2(c, c), oo = make_float2(off, off);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float2 z = __ffma2_rn(make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), cc, oo);
                    const float2 e = decltype(mixed)::value && j % 4 == 3 ? ex2_poly(z) : make_float2(ex2_approx(z.x), ex2_approx(z.y));
                    x[2 * j] = __float_as_uint(e.x);
                    x[2 * j + 1] = __float_as_uint(e.y);
                }
            };
            if (masked) {
                probabilities(std::false_type{});
                // S has read K by now; what is left is dQ, where hidden keys have dS = 0. A half of d for each half of the threads
                uint8_t* tile = smem + C::RING + (2 * done) % C::NSLOT * C::TILE;
                if (64 * ch < D) clean_row<T, 64>(tile + ch * HALF, r);
                fence_proxy_async_smem();
            } else {
                probabilities(std::true_type{});
            }
            ok = mbar_wait_warp(smem_u32(&ctl->dpfull), done & 1, abort_flag, a.status, 651);
            if (!ok) break;
            tc_fence_after();
            if (w.fine) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t y[32], ds[16], rest[16];
                    tmem_ld32(dpcol + 32 * h, y);
                    tmem_wait_ld_regs(y);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float g[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int k = 32 * h + 2 * j + e;
                            g[e] = k >= lim ? 0.f : __uint_as_float(x[k]) * (__uint_as_float(y[2 * j + e]) - delta);
                        }
                        // (a row that sees one key: P is 1 whatever the logit, and dS is 0 and not what rounding leaves; NaN stays)
                        if (h == 0 && j == 0 && vis == 1 && g[0] == g[0]) g[0] = 0.f;
                        ds[j] = pack2<T>(g[0], g[1]);
                        rest[j] = rest2<T>(g[0], g[1], ds[j]);
                    }
                    tmem_st16(scol + 16 * h, ds);
                    tmem_st16(scol + 32 + 16 * h, rest);
                }
            } else {
            uint32_t y[64];
            tmem_ld32(dpcol, y);
            tmem_ld32(dpcol + 32, y + 32);
            tmem_wait_ld_regs(y);
            tmem_wait_ld_regs(y + 32);
            auto differences = [&](auto cut_tile) {
                uint32_t ds[32];
                const float2 nd = make_float2(-delta, -delta);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float2 g = __fmul2_rn(make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])),
                                          __fadd2_rn(make_float2(__uint_as_float(y[2 * j]), __uint_as_float(y[2 * j + 1])), nd));
                    if (decltype(cut_tile)::value) {
                        // (a row that sees one key: P is 1 whatever the logit, and dS is 0 and not what rounding leaves; NaN stays)
                        if (2 * j >= lim || (vis == 1 && g.x == g.x)) g.x = 0.f;
                        if (2 * j + 1 >= lim) g.y = 0.f;
                    }
                    ds[j] = pack2<T>(g.x, g.y);
                }
                tmem_st32(scol, ds);
            };
            if (masked) differences(std::true_type{});
            else differences(std::false_type{});
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->dsfull));
        }
        if (nt > 0) ok = ok && mbar_wait_warp(smem_u32(&ctl->gfull), tiles++ & 1, abort_flag, a.status, 652);
        if (!ok) break;
        tc_fence_after();
        w = ctl->work[n & 1];                                // (read again: the loop's registers are few)
        T* dst = static_cast<T*>(a.d0) + ((int64_t)(w.first + tok) * a.b.H + w.head + lane_head) * D;
        store_row<T, D>(dst, nullptr, tl + DQ_COL, ch * (D / 64), (ch + 1) * (D / 64), nt > 0, valid, a.b.scale);
        leave(n);
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    if (warp == 9 && lane == 0 && *abort_flag) land<C::NSLOT>(ctl, owners, issued);
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
            for (int e = tid; e < w.n_tok * a.pack * (D / 2); e += THREADS) {
                const int row = e / (D / 2);
                static_cast<uint32_t*>(a.d0)[((int64_t)(w.first + row / a.pack) * a.b.H + w.head + row % a.pack) * (D / 2) + e % (D / 2)] = kNaN16x2;
            }
        }
    }
}

// dK, dV = the sums of their parts in the order of the CTAs; four values a thread.
template <typename T> __global__ void __launch_bounds__(256) sum_kernel(const float4* part, T* dk, T* dv, int splits, int64_t n4) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    wait_prerequisites();
    if (i >= 2 * n4) return;
    float4 s = part[i];
    for (int p = 1; p < splits; ++p) {
        const float4 x = part[2 * p * n4 + i];
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    T* dst = i < n4 ? dv + 4 * i : dk + 4 * (i - n4);
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

// CTAs that share the rows that walk a key tile: as many as make the pass shortest, in walked tiles. What is known of the lengths is
// their mean; START: a CTA's start and end; the longest walk is taken for twice the mean of uneven sequences.
static int kv_splits(int B, int Tq, int Tk, int H, int Hk, int D) {
    constexpr double START = 6, LAUNCH = 4, BYTES = 8e6;     // a launch, and the bytes of the parts that move, in the time of a tile
    const int sms = sm_count(), pack = rows_pack(H / Hk), tokens = TM / pack;
    const double tiles = Hk * (Tk / (double)TN + 0.5 * B), walk = (double)Tq / std::max(1, B) / tokens * (H / Hk / pack), longest = B > 1 ? 2 * walk : walk;
    int best = 1;
    double least = 0;
    for (int n = 1; n <= 16; ++n) {
        const double cost = std::max(rounds(tiles * n / sms) * (0.5 * walk / n + START), longest / n + START) + (n > 1 ? LAUNCH + 16.0 * n * Tk * Hk * D / BYTES : 0);
        if (n == 1 || cost < 0.9 * least) { best = n; least = cost; }
    }
    return best;
}

template <typename T, int D>
static int launch(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, const void* dout, Rows rdo, BwdArgs a, void* dq, void* dk, void* dv,
                  cudaStream_t st) {
    CUtensorMap tq, tk, tv, tdo;
    // (a batch without queries or without keys loads none, but a map needs an extent)
    long long nq = a.b.Tq, nk = a.b.Tk;
    if (!nq) { q = dout = k; rq = rdo = rk; nq = nk; }
    if (!nk) { k = v = q; rk = rv = rq; nk = nq; }
    const int qh = a.b.Tq ? a.b.H : a.b.Hk, qbox = a.b.Tq ? a.pack : 1, kvh = a.b.Tk ? a.b.Hk : 1;
    if (int rc = make_rows_map<T>(&tq, q, D, qh, nq, rq, qbox, a.tokens)) return rc;
    if (int rc = make_rows_map<T>(&tdo, dout, D, qh, nq, rdo, qbox, a.tokens)) return rc;
    if (int rc = make_rows_map<T>(&tk, k, D, kvh, nk, rk, 1, TN)) return rc;
    if (int rc = make_rows_map<T>(&tv, v, D, kvh, nk, rv, 1, TN)) return rc;
    for (int kv = 0; kv < 2; ++kv) {
        if (!(kv ? dk : dq)) continue;
        a.slots = kv ? piece_slots(a.b.Tk, TN, a.b.B) : piece_slots(a.b.Tq, a.tokens, a.b.B);
        const int64_t grid = a.slots * (kv ? a.b.Hk * a.splits : a.b.H / a.pack);
        if (grid > 0x7FFFFFFF) return set_error(-1, "es_packed_attn_bwd: too many tiles");
        auto kern = kv ? packed_bwd_kv_kernel<T, D> : packed_bwd_q_kernel<T, D>;
        if (int rc = opt_in_shared_memory((const void*)kern, (int)Cfg<D>::BYTES)) return rc;
        a.d0 = kv ? dk : dq;
        a.d1 = dv;
        a.behind_q = kv && dq;
        // either pass may set up while the kernel before it ends, and dK / dV start on the SMs that dQ has left
        const cudaError_t e = launch_dependent(kern, dim3((unsigned)grid), dim3(THREADS), Cfg<D>::BYTES, st, tq, tk, tv, tdo, a);
        if (e != cudaSuccess) return set_error(-2, cudaGetErrorString(e));
        ES_CHECK_LAUNCH("packed_bwd_kernel");
    }
    if (dk && a.splits > 1) {
        const int64_t n4 = (int64_t)a.b.Tk * a.b.Hk * D / 4, blocks = (2 * n4 + 255) / 256;
        if (blocks > 0x7FFFFFFF) return set_error(-1, "es_packed_attn_bwd: too many rows");
        const cudaError_t e = launch_dependent(sum_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const float4*>(a.part), static_cast<T*>(dk),
                                               static_cast<T*>(dv), a.splits, n4);
        if (e != cudaSuccess) return set_error(-2, cudaGetErrorString(e));
        ES_CHECK_LAUNCH("sum_kernel");
    }
    return 0;
}

long long packed_bwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D) {
    const int n = kv_splits(B, Tq, Tk, H, Hk, D);
    return n > 1 ? 2ll * n * Tk * Hk * D * 4 : 0;
}

// The caller has checked sizes and pointers; dq, or dk and dv, may be null. ws: packed_bwd_workspace bytes.
int packed_bwd_tc(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, const void* dout, Rows rdo, const float* lse, const float* delta, void* dq,
                  void* dk, void* dv, const Batch& b, int D, int dtype, void* ws, cudaStream_t st) {
    BwdArgs a{};
    a.b = b;
    a.pack = rows_pack(b.G);
    a.tokens = TM / a.pack;
    a.lse = lse;
    a.delta = delta;
    a.splits = kv_splits(b.B, b.Tq, b.Tk, b.H, b.Hk, D);
    a.part = static_cast<float*>(ws);
    a.dout = dout;
    a.rdo = rdo;
    a.status = device_status_ptr();
    if (!a.status) return set_error(-2, "es_packed_attn_bwd: the device status word is not available on this device");
    if (D == 64)
        return dtype == 0 ? launch<__nv_bfloat16, 64>(q, rq, k, rk, v, rv, dout, rdo, a, dq, dk, dv, st) : launch<__half, 64>(q, rq, k, rk, v, rv, dout, rdo, a, dq, dk, dv, st);
    return dtype == 0 ? launch<__nv_bfloat16, 128>(q, rq, k, rk, v, rv, dout, rdo, a, dq, dk, dv, st) : launch<__half, 128>(q, rq, k, rk, v, rv, dout, rdo, a, dq, dk, dv, st);
}

}  // namespace packed
}  // namespace es
