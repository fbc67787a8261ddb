// Attention of a batch's newest tokens to a shared prefix and to each request's own tokens, both in pages of a cache.
//
// The keys of a row are two sets, the prefix and its request's own; each gives a partial result O_p = softmax(S_p) V_p with its LSE z_p (log2),
// and they are joined by O = sum_p 2^(z_p - M) O_p / sum_p 2^(z_p - M).
//   prefix       all rows of the batch that read a key head see the same keys. More than ROWS of them: the tcgen05 kernel of es_packed_fwd.cu,
//                128 rows to a tile, the keys shared out over the SMs. Fewer: as one more item of the kernel below.
//   own tokens   `own_kernel`: tokens x heads of a group rows against each request's pages. Every key is read once and multiplied with a few
//                rows: bound by HBM. Warps with m16n8k16 MMAs, 64 keys at a time, scores and P in registers: the tensor cores are idle most of the
//                time at any shape (16 FLOP a byte; tcgen05 with its 128 rows would compute eight times as much for the same bytes).
// Work of own_kernel: the (request, heads, block of new tokens) items, each ITEM + its 64-key units long, one behind the other; CTA c of C has
// the stretch c W / C .. (c + 1) W / C of W whatever the lengths are. (ITEM: what starting and storing an item costs, in units.) An item's first
// share is stored by its rows (part A), one that starts inside an item by its CTA (part B; a CTA has at most one). The join finds them by
// the same arithmetic.
#include "es_packed_tc.cuh"
#include "es_vsa_mma.cuh"

namespace es {
namespace packed {

int prefix_fwd_tc(const void* q, const void* k, CacheRows rk, const void* v, CacheRows rv, float* part_o, float* part_lse, int parts, const int* list, int prefix_len,
                  int tokens, int H, int Hk, int pages, int log_page, float scale, int D, int dtype, cudaStream_t st);

namespace {
constexpr int UNIT = 64, WARPS = 4, OWN_THREADS = 32 * (WARPS + 1), ROWS = 64;
constexpr int ITEM = 2;
// A CTA whose stretch holds two requests passes those without tokens between them while its other warps wait: 13 ns each, 0.1 s of the wait's limit of 0.5.
constexpr int MOST_REQUESTS = 1 << 23;

__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

struct PrefixArgs {
    const int *prefix_pages, *table, *lengths;
    int prefix_len, width, B, N, H, Hk, pages, log_page;
    float scale;
    int pack, per_block, blocks;     // heads of a row group; new tokens of an item; items along a request's tokens
    int vheads;                      // H / pack
    int prefix_item;                 // the prefix is an item of own_kernel
    int ctas;
    const void *q, *v;
    CacheRows rv;
    float *a_o, *a_lse;              // part A of the requests [token][head][D], [token][head]
    float *p_o, *p_lse;              // of the prefix: parts [part][token][head][D], or part A of its item
    int p_parts;
    float *b_o, *b_lse;              // part B [cta][ROWS][D], [cta][ROWS]
    long long* first;                // [B + 1] where each request starts: written by CTA 0
    int* status;
};

__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) { return min(max(__ldg(a.lengths + b), 0), a.width << a.log_page); }
__device__ __forceinline__ int units_of(int keys) { return (int)(((long long)keys + UNIT - 1) / UNIT); }
// The stretch of a set of keys: of all its items.
__device__ __forceinline__ long long stretch(int keys, int items) { return keys > 0 ? (long long)(units_of(keys) + ITEM) * items : 0; }
__device__ __forceinline__ long long prefix_stretch(const PrefixArgs& a) { return a.prefix_item ? stretch(a.prefix_len, a.vheads) : 0; }

template <int D, int MT> struct Own {
    static constexpr uint32_t HALF = UNIT * 128, TILE = UNIT * D * 2;
    static constexpr int NSLOT = D == 64 ? 8 : MT == 2 ? 3 : 4;        // two CTAs per SM
    static constexpr uint32_t QPITCH = D * 2 + 16, QTILE = 16 * MT * QPITCH;
    static constexpr uint32_t RING = 0, Q = NSLOT * TILE, SUM = Q + 2 * QTILE, CTL = SUM + (MT < 4 ? WARPS * 16 * D * 4 : 0), BYTES = CTL + 1536;
};
// A unit as the load warp hands it to the others.
struct UnitDesc {
    int k0;              // first key in its set, -1: no more units
    int n;               // keys of the set
    int b;               // request, -1: the prefix
    int head0, t0, tq;   // first head, first new token of the item: in the batch, in the request
    int rows;
    int flags;           // FIRST, LAST unit of the CTA's share of the item; STARTS: the item's first share
    uint32_t bad;        // a bit per box whose page is not of the cache
};
enum { FIRST = 1, LAST = 2, STARTS = 4 };
struct OwnCtl {
    uint64_t full[8], empty[8], qfull[2], qempty[2], joined;
    int abort, not_finite, first_b;
    long long first_x, warp_sum[WARPS + 1];
    UnitDesc desc[4];
    float ml[WARPS][32];             // maxima and sums of warps that are joined
};
static_assert(sizeof(OwnCtl) <= 1536, "control block");

// MT: 16-row tiles of an item. One: every warp has them and a quarter of a unit's keys; two: two warps each and half; four: all keys.
// Bound by HBM: 256 requests of 4,096 tokens at most on 8 heads, 560 MB in 115 us = 4.8 TB/s; 64 samples of 1,024 at most, 27 MB in 14.5 us. What
// is missing to a copy's rate are the items' ends (a row's sums joined over warps, O stored) with two CTAs to an SM to hide them.
template <typename T, int D, int MT>
__global__ void __launch_bounds__(OWN_THREADS, 2)
own_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PrefixArgs a) {
    using C = Own<D, MT>;
    using E = vsa::Elt<T>;
    constexpr int WK = WARPS / MT, KW = UNIT / WK;            // warps that share a row tile, keys of a warp in a unit
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(smem);
    OwnCtl* ctl = reinterpret_cast<OwnCtl*>(smem + C::CTL);
    volatile int* abort_flag = &ctl->abort;
    launch_dependents();
    if (tid == 0) {
        const int earlier = *reinterpret_cast<volatile int*>(a.status);
        for (int i = 0; i < C::NSLOT; ++i) {
            mbar_init(smem_u32(&ctl->full[i]), 1);
            mbar_init(smem_u32(&ctl->empty[i]), WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->qfull[i]), 1);
            mbar_init(smem_u32(&ctl->qempty[i]), WARPS);
        }
        mbar_init(smem_u32(&ctl->joined), WARPS);
        ctl->not_finite = 0;
        ctl->first_b = -1;
        ctl->abort = (base & 1023u) || earlier ? 1 : 0;      // the swizzled tiles need a 1024-byte aligned base
        if (base & 1023u) atomicCAS(a.status, 0, 913);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    // where the requests start: a running sum over all of them, a run of requests to a thread
    const int items = a.vheads * a.blocks, run = (a.B + OWN_THREADS - 1) / OWN_THREADS, b0 = min(a.B, tid * run), b1 = min(a.B, b0 + run);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += stretch(own_length(a, b), items);
    long long x = mine;
    for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) ctl->warp_sum[warp] = x;
    __syncthreads();
    long long W = prefix_stretch(a);
    x += W - mine;
    for (int w = 0; w <= WARPS; ++w) {
        if (w < warp) x += ctl->warp_sum[w];
        W += ctl->warp_sum[w];
    }
    // (a CTA's stretch is never empty: no more CTAs than W)
    const long long ctas = min((long long)a.ctas, W);
    const bool busy = blockIdx.x < ctas;
    const long long beg = busy ? W * blockIdx.x / ctas : 0, end = busy ? W * (blockIdx.x + 1) / ctas : 0;
    if (blockIdx.x == 0 || (busy && x <= beg && beg < x + mine))
        for (int b = b0; b < b1; ++b) {
            const long long w = stretch(own_length(a, b), items);
            if (blockIdx.x == 0) a.first[b] = x;
            if (busy && x <= beg && beg < x + w) { ctl->first_b = b; ctl->first_x = beg - x; }
            x += w;
        }
    if (blockIdx.x == 0 && tid == 0) a.first[a.B] = W;
    __syncthreads();
    const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
    bool ok = *abort_flag == 0;

    if (warp == WARPS) {
        // ------------------------------------------------------------ loads: Q of every item, K and V of every unit, a lane per row or box
        const int box = min(UNIT, 1 << a.log_page), boxes = UNIT / box;
        uint32_t slot = 0, par = 1, issued = 0, unit = 0, item_no = 0;
        if (lane == 0) {
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
        }
        long long left = end - beg;
        int b = ctl->first_b;                                 // -1: in the prefix
        int n = b < 0 ? a.prefix_len : own_length(a, b), units = units_of(n), item, y;
        {
            const long long at = b < 0 ? beg : ctl->first_x;
            item = left > 0 ? (int)(at / (units + ITEM)) : 0;
            y = left > 0 ? (int)(at - (long long)item * (units + ITEM)) : 0;
        }
        while (left > 0 && ok) {
            const int y1 = (int)min((long long)units + ITEM, y + left), u0 = max(0, y - ITEM), u1 = max(0, y1 - ITEM);
            if (u1 > u0) {
                const int blk = b < 0 ? 0 : item / a.vheads, head0 = (item - blk * a.vheads) * a.pack;
                const int tq = blk * a.per_block, t0 = b < 0 ? 0 : b * a.N + tq;
                const int rows = (b < 0 ? a.B * a.N : min(a.per_block, a.N - tq)) * a.pack;
                const int* list = b < 0 ? a.prefix_pages : a.table + (size_t)b * a.width;
                const int kh = head0 / (a.H / a.Hk), qs = item_no & 1;
                ok = mbar_wait_warp(smem_u32(&ctl->qempty[qs]), ((item_no >> 1) & 1) ^ 1, abort_flag, a.status, 664);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(smem_u32(&ctl->qfull[qs]), (uint32_t)(rows * D * 2));
                __syncwarp();
                for (int r = lane; r < rows; r += 32)
                    bulk_load(base + C::Q + qs * C::QTILE + r * C::QPITCH, static_cast<const T*>(a.q) + ((int64_t)(t0 + r / a.pack) * a.H + head0 + r % a.pack) * D,
                              D * 2, smem_u32(&ctl->qfull[qs]));
                ++item_no;
                int win = 0, wbase = -1;                      // pages of the next 32 boxes
                for (int i = u0; i < u1 && ok; ++i) {
                    const int bx = i * boxes, w = bx & ~31;   // (8, 4, 2 or 1 boxes to a unit: a unit's are in one window)
                    if (w != wbase) {
                        wbase = w;
                        const long long k = (long long)(w + lane) * box;
                        win = k < n ? __ldg(list + (k >> a.log_page)) : -1;
                    }
                    const int p = __shfl_sync(0xffffffffu, win, (bx & 31) + (lane & (boxes - 1)));
                    const bool good = p >= 0 && p < a.pages, needed = (long long)(bx + lane) * box < n;
                    // a page that is not of the cache, or behind the keys, is loaded as zeros
                    const int page = lane < boxes && needed && good ? p : a.pages;
                    const uint32_t bad = __ballot_sync(0xffffffffu, lane < boxes && needed && !good);
                    for (int x_ = 0; x_ < 2 && ok; ++x_) {
                        ok = mbar_wait_warp(empty0 + 8 * slot, par, abort_flag, a.status, 661);
                        if (!ok) break;
                        const uint32_t bar = full0 + 8 * slot, dst = base + C::RING + slot * C::TILE;
                        if (lane == 0) {
                            // (the slot's last tenant was at least NSLOT tiles ago, its unit's copy of the descriptor long taken)
                            if (x_ == 0)
                                ctl->desc[unit & 3] = UnitDesc{i * UNIT, n, b, head0, t0, tq, rows, (i == u0 ? FIRST : 0) | (i + 1 == u1 ? LAST : 0) | (u0 == 0 ? STARTS : 0), bad};
                            mbar_arrive_expect_tx(bar, C::TILE);
                        }
                        __syncwarp();
                        if (lane < boxes)
                            for (int d = 0; d < D / 64; ++d)
                                tma_load_4d(dst + d * C::HALF + lane * box * 128, x_ ? &tmV : &tmK, bar, 64 * d, kh, (i * UNIT) & ((1 << a.log_page) - 1), page);
                        __syncwarp();
                        ++issued;
                        if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
                    }
                    ++unit;
                }
            }
            left -= y1 - y;
            y = 0;
            if (++item == (b < 0 ? a.vheads : items)) {
                item = 0;
                // the next request with tokens, sought 32 at a time: the other warps wait meanwhile
                int len = 0;
                uint32_t some = 0;
                for (++b; b < a.B; b += 32) {
                    len = b + lane < a.B ? own_length(a, b + lane) : 0;
                    some = __ballot_sync(0xffffffffu, len > 0);
                    if (some) break;
                }
                if (b >= a.B) break;
                const int first = __ffs(some) - 1;
                b += first;
                n = __shfl_sync(0xffffffffu, len, first);
                units = units_of(n);
            }
        }
        if (ok) ok = mbar_wait_warp(empty0 + 8 * slot, par, abort_flag, a.status, 665);
        if (ok && lane == 0) {
            ctl->desc[unit & 3].k0 = -1;
            mbar_arrive(full0 + 8 * slot);
        }
        __syncwarp();
        if (lane == 0 && *abort_flag) {
            // a wait gave up: give the loads a moment (100 us in all) to land before shared memory goes away
            const uint64_t t_end = global_timer_ns() + 100000ull;
            for (uint32_t q = 0; q < 2 && q < item_no; ++q) {
                const uint32_t it = item_no - 1 - q;
                while (!mbar_try_wait(smem_u32(&ctl->qfull[it & 1]), (it >> 1) & 1) && global_timer_ns() < t_end) {}
            }
            for (uint32_t back = 1; back <= (uint32_t)C::NSLOT && back <= issued; ++back) {
                const uint32_t sq = issued - back;
                while (!mbar_try_wait(full0 + 8 * (sq % C::NSLOT), (sq / C::NSLOT) & 1) && global_timer_ns() < t_end) {}
            }
        }
    } else {
        const int mt = warp / WK, wk = warp % WK;             // row tile, share of the keys
        const int r0 = 16 * mt + (lane >> 2), r1 = r0 + 8;
        const float c = a.scale * kLog2e;
        const int box = min(UNIT, 1 << a.log_page), box_log = 31 - __clz(box);
        uint32_t slot = 0, par = 0, unit = 0, item_no = 0;
        uint32_t qf[D / 16][4];
        float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        int from = 0;                                         // first unit's first key of the share
        uint32_t join_par = 0;
        // a barrier of the four warps whose wait is bounded: one that gave up elsewhere comes no more
        auto together = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->joined));
            ok = mbar_wait_warp(smem_u32(&ctl->joined), join_par, abort_flag, a.status, 667);
            join_par ^= 1;
            return ok;
        };
        while (ok) {
            ok = mbar_wait_warp(full0 + 8 * slot, par, abort_flag, a.status, 662);
            if (!ok) break;
            const UnitDesc u = ctl->desc[unit++ & 3];
            if (u.k0 < 0) break;
            // keys that the thread's two rows see, and the fewest and most that any row of the item sees
            auto seen = [&](int row) { return u.b < 0 ? u.n : max(u.n - a.N + u.tq + row / a.pack + 1, 0); };
            const int v0 = r0 < u.rows ? seen(r0) : 0, v1 = r1 < u.rows ? seen(r1) : 0, least = seen(0);
            if (u.flags & FIRST) {
                const int qs = item_no & 1;
                ok = mbar_wait_warp(smem_u32(&ctl->qfull[qs]), (item_no >> 1) & 1, abort_flag, a.status, 666);
                if (!ok) break;
                // 16 rows x 16 d: lanes 0-15 rows 0-15 of d 0-7, lanes 16-31 of d 8-15
                const uint32_t qa = base + C::Q + qs * C::QTILE + (16 * mt + (lane & 15)) * C::QPITCH + (lane >> 4) * 16;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) vsa::ldsm4(qa + 32 * ks, qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3]);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->qempty[qs]));
                ++item_no;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
                m0 = m1 = -INFINITY;
                l0 = l1 = 0.f;
                from = u.k0;
            }
            const int k0 = u.k0 + wk * KW;                    // this warp's keys k0 .. k0 + KW - 1
            float x[KW / 8][4];
            const uint32_t kb = base + C::RING + slot * C::TILE;
#pragma unroll
            for (int j = 0; j < KW / 8; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                for (int j = 0; j < KW / 16; ++j) {
                    // 16 keys x 16 d: lanes 0-7, 8-15 keys 0-7 (d 0-7, 8-15), lanes 16-31 keys 8-15
                    const int row = wk * KW + 16 * j + (lane & 7) + ((lane >> 4) << 3), ch = 2 * (ks & 3) + ((lane >> 3) & 1);
                    uint32_t f0, f1, f2, f3;
                    vsa::ldsm4(kb + (ks >> 2) * C::HALF + row * 128 + ((ch ^ (row & 7)) << 4), f0, f1, f2, f3);
                    E::mma(x[2 * j], qf[ks], f0, f1);
                    E::mma(x[2 * j + 1], qf[ks], f2, f3);
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * slot);
            if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
            if (u.k0 + UNIT > least) {
#pragma unroll
                for (int j = 0; j < KW / 8; ++j) {
                    const int k = k0 + 8 * j + 2 * (lane & 3);
                    if (k >= v0) x[j][0] = -INFINITY;
                    if (k + 1 >= v0) x[j][1] = -INFINITY;
                    if (k >= v1) x[j][2] = -INFINITY;
                    if (k + 1 >= v1) x[j][3] = -INFINITY;
                }
            }
            if (u.bad)
#pragma unroll
                for (int j = 0; j < KW / 8; ++j)
                    if ((u.bad >> ((wk * KW + 8 * j) >> box_log)) & 1) x[j][0] = x[j][1] = x[j][2] = x[j][3] = -INFINITY;
            float y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < KW / 8; ++j) {
                y0 = fmaxf(y0, fmaxf(x[j][0], x[j][1]));
                y1 = fmaxf(y1, fmaxf(x[j][2], x[j][3]));
            }
            y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, 1));
            y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, 1));
            y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, 2)) * c;
            y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, 2)) * c;
            if (__any_sync(0xffffffffu, y0 > m0 || y1 > m1)) {
                const float n0 = fmaxf(m0, y0), n1 = fmaxf(m1, y1);
                const float f0 = n0 == -INFINITY ? 1.f : ex2_approx(m0 - n0), f1 = n1 == -INFINITY ? 1.f : ex2_approx(m1 - n1);
                m0 = n0; m1 = n1;
                l0 *= f0; l1 *= f1;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) { o[j][0] *= f0; o[j][1] *= f0; o[j][2] *= f1; o[j][3] *= f1; }
            }
            const float z0 = m0 == -INFINITY ? 0.f : -m0, z1 = m1 == -INFINITY ? 0.f : -m1;
#pragma unroll
            for (int j = 0; j < KW / 8; ++j) {
                x[j][0] = ex2_approx(fmaf(x[j][0], c, z0));
                x[j][1] = ex2_approx(fmaf(x[j][1], c, z0));
                x[j][2] = ex2_approx(fmaf(x[j][2], c, z1));
                x[j][3] = ex2_approx(fmaf(x[j][3], c, z1));
                l0 += x[j][0] + x[j][1];
                l1 += x[j][2] + x[j][3];
            }
            ok = mbar_wait_warp(full0 + 8 * slot, par, abort_flag, a.status, 663);
            if (!ok) break;
            if (k0 + KW > least) {
                // V rows that some row does not see: what is not finite there is set to 0 (0 times it would be NaN), and given at the end to the
                // rows that do see it
                for (int e = lane; e < KW * (D / 8); e += 32) {
                    const int row = wk * KW + e / (D / 8), ch = e % (D / 8);
                    uint4* p = reinterpret_cast<uint4*>(smem + C::RING + slot * C::TILE + (ch >> 3) * C::HALF + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                    const uint4 w = *p;
                    if (u.k0 + row >= least && (not_finite<T>(w.x) || not_finite<T>(w.y) || not_finite<T>(w.z) || not_finite<T>(w.w))) {
                        if (u.k0 + row < u.n) *reinterpret_cast<volatile int*>(&ctl->not_finite) = 1;
                        *p = make_uint4(finite_only<T>(w.x), finite_only<T>(w.y), finite_only<T>(w.z), finite_only<T>(w.w));
                    }
                }
                __syncwarp();
                fence_proxy_async_smem();
            }
            // (P in 16 bits, the sum of what was not rounded: see es_packed_fwd.cu)
            const uint32_t vb = base + C::RING + slot * C::TILE;
#pragma unroll
            for (int j = 0; j < KW / 16; ++j) {
                const uint32_t p[4] = {pack2<T>(x[2 * j][0], x[2 * j][1]), pack2<T>(x[2 * j][2], x[2 * j][3]), pack2<T>(x[2 * j + 1][0], x[2 * j + 1][1]),
                                       pack2<T>(x[2 * j + 1][2], x[2 * j + 1][3])};
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    // 16 keys x 16 d, transposed: lanes 0-15 keys 0-15 of d 0-7, lanes 16-31 of d 8-15
                    const int row = wk * KW + 16 * j + (lane & 15), ch = 2 * (d & 3) + (lane >> 4);
                    uint32_t f0, f1, f2, f3;
                    ldsm4_trans(vb + (d >> 2) * C::HALF + row * 128 + ((ch ^ (row & 7)) << 4), f0, f1, f2, f3);
                    E::mma(o[2 * d], p, f0, f1);
                    E::mma(o[2 * d + 1], p, f2, f3);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * slot);
            if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
            if (!(u.flags & LAST)) continue;
            // ---- the share is done: join the warps that have its rows, and store it
            l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
            if (least < u.n) {
                if (!together()) break;                       // (another warp with the same keys may have found it)
                if (*reinterpret_cast<volatile int*>(&ctl->not_finite)) {
                    const int* list = u.b < 0 ? a.prefix_pages : a.table + (size_t)u.b * a.width;
                    const int kh = u.head0 / (a.H / a.Hk);
                    for (int k = max(least, from); k < min(u.n, u.k0 + UNIT); ++k) {
                        const int p = __ldg(list + (k >> a.log_page));
                        if ((k % UNIT) / KW != wk || p < 0 || p >= a.pages) continue;
                        const T* vr = static_cast<const T*>(a.v) + p * a.rv.page + (int64_t)(k & ((1 << a.log_page) - 1)) * a.rv.token + (int64_t)kh * a.rv.head + 2 * (lane & 3);
#pragma unroll
                        for (int j = 0; j < D / 8; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float f = to_float(vr[8 * j + e]);
                                if (fabsf(f) < INFINITY) continue;
                                if (k < v0) o[j][e] += f;
                                if (k < v1) o[j][2 + e] += f;
                            }
                    }
                }
            }
            float f0 = 1.f, f1 = 1.f;                         // factors of this warp's own sums (MT = 4: the only ones)
            float lt0 = l0, lt1 = l1, mt0 = m0, mt1 = m1;
            float* sum = reinterpret_cast<float*>(smem + C::SUM);
            if constexpr (WK > 1) {
                if (!together()) break;                       // the share before has been read
                if ((lane & 3) == 0) {
                    ctl->ml[warp][lane >> 2] = m0; ctl->ml[warp][8 + (lane >> 2)] = m1;
                    ctl->ml[warp][16 + (lane >> 2)] = l0; ctl->ml[warp][24 + (lane >> 2)] = l1;
                }
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
                    *reinterpret_cast<float4*>(sum + (warp * 16 * D) + (j * 32 + lane) * 4) = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
                if (!together()) break;
                mt0 = mt1 = -INFINITY;
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    mt0 = fmaxf(mt0, ctl->ml[mt * WK + w][lane >> 2]);
                    mt1 = fmaxf(mt1, ctl->ml[mt * WK + w][8 + (lane >> 2)]);
                }
                lt0 = lt1 = 0.f;
            }
            constexpr int JN = D / 8 / WK;                    // every warp stores a share of the columns
            float acc[JN][4];
            if constexpr (WK > 1) {
#pragma unroll
                for (int j = 0; j < JN; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    const int src = mt * WK + w;
                    f0 = mt0 == -INFINITY ? 0.f : ex2_approx(ctl->ml[src][lane >> 2] - mt0);
                    f1 = mt1 == -INFINITY ? 0.f : ex2_approx(ctl->ml[src][8 + (lane >> 2)] - mt1);
                    lt0 += ctl->ml[src][16 + (lane >> 2)] * f0;
                    lt1 += ctl->ml[src][24 + (lane >> 2)] * f1;
#pragma unroll
                    for (int j = 0; j < JN; ++j) {
                        const float4 v = *reinterpret_cast<const float4*>(sum + src * 16 * D + ((wk * JN + j) * 32 + lane) * 4);
                        acc[j][0] += v.x * f0; acc[j][1] += v.y * f0; acc[j][2] += v.z * f1; acc[j][3] += v.w * f1;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < JN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] = o[j][e];
            }
            auto store = [&](int row, float m, float l, int e) {
                if (row >= u.rows) return;
                const float inv = l != 0.f ? 1.f / l : 0.f;
                const int64_t at = (int64_t)(u.t0 + row / a.pack) * a.H + u.head0 + row % a.pack;
                const bool starts = u.flags & STARTS;
                float* dst = (starts ? (u.b < 0 ? a.p_o : a.a_o) + at * D : a.b_o + ((int64_t)blockIdx.x * ROWS + row) * D) + 8 * JN * wk + 2 * (lane & 3);
                float* z = starts ? (u.b < 0 ? a.p_lse : a.a_lse) + at : a.b_lse + (int64_t)blockIdx.x * ROWS + row;
#pragma unroll
                for (int j = 0; j < JN; ++j)
                    *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(acc[j][e] * inv, acc[j][e + 1] * inv);
                if (wk == 0 && (lane & 3) == 0) *z = l != 0.f ? m + log2f(l) : -INFINITY;
            };
            store(r0, mt0, lt0, 0);
            store(r1, mt1, lt1, 2);
        }
    }
    // the join waits for this kernel, this kernel for the one of the prefix
    wait_prerequisites();
    __syncthreads();
}

// A warp per row: the parts of the prefix, part A of the row's own item, and the part B's of the CTAs that went on with it. A lane looks
// up a part's LSE, so that a row costs two round trips to memory and not two per part (256 requests of 2 tokens, 40 heads: 24 us).
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(T* o, float* lse, const __grid_constant__ PrefixArgs a) {
    constexpr int C = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)a.B * a.N * a.H, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    wait_prerequisites();
    if (row >= rows) return;
    const int h = (int)(row % a.H), t = (int)(row / a.H), b = t / a.N, i = t % a.N, vh = h / a.pack;
    const long long W = a.first ? a.first[a.B] : 0, ctas = min((long long)a.ctas, W);
    // parts of an item: A, and B of the CTAs after the one with its first unit up to the one with its last
    struct Item { int n, c0; };
    auto item_at = [&](long long start, int units) {
        Item it{0, 0};
        if (units > 0) {
            it.c0 = (int)(((start + ITEM + 1) * ctas - 1) / W);
            it.n = 1 + (int)(((start + ITEM + units) * ctas - 1) / W) - it.c0;
        }
        return it;
    };
    const int pu = a.prefix_item ? units_of(a.prefix_len) : 0, own = a.first ? units_of(own_length(a, b)) : 0, blk = i / a.per_block;
    const Item pi = a.prefix_item ? item_at((long long)vh * (pu + ITEM), pu) : Item{a.p_parts, 0};
    const Item oi = own ? item_at(a.first[b] + (long long)(blk * a.vheads + vh) * (own + ITEM), own) : Item{0, 0};
    const int parts = pi.n + oi.n, pr = t * a.pack + h % a.pack, orow = (i - blk * a.per_block) * a.pack + h % a.pack;
    // where part p lies: its row of D floats; its LSE
    auto find = [&](int p, const float*& src, const float*& z) {
        if (p < pi.n && !a.prefix_item) { src = a.p_o + (p * rows + row) * D; z = a.p_lse + p * rows + row; return; }
        const bool pre = p < pi.n;
        const int q = pre ? p : p - pi.n, r = pre ? pr : orow;
        const int64_t slot = (int64_t)((pre ? pi.c0 : oi.c0) + q) * ROWS + r;
        src = q ? a.b_o + slot * D : (pre ? a.p_o : a.a_o) + row * D;
        z = q ? a.b_lse + slot : (pre ? a.p_lse : a.a_lse) + row;
    };
    float acc[C] = {}, sum = 0.f, top = -INFINITY;
    for (int p0 = 0; p0 < parts; p0 += 32) {
        const float *src = nullptr, *zp = nullptr;
        float z = -INFINITY;
        if (p0 + lane < parts) {
            find(p0 + lane, src, zp);
            z = *zp;
        }
        float next = fmaxf(top, z);
        for (int d = 16; d; d >>= 1) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, d));
        if (next > top) {
            const float f = ex2_approx(top - next);           // (0 at first)
            sum *= f;
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] *= f;
            top = next;
        }
        // NaN, or +infinity, makes the row NaN; -infinity is a part without a key: what it holds is not read
        const float w = z == -INFINITY ? 0.f : z != z ? z : ex2_approx(z - top);
        float all = w;
        for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
        sum += all;
        const int n = min(32, parts - p0);
#pragma unroll 4
        for (int p = 0; p < n; ++p) {
            const float wp = __shfl_sync(0xffffffffu, w, p);
            const float* sp = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), p));
            float v[C];
            load_floats<C>(sp + C * lane, v);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] += wp == 0.f ? 0.f : v[c] * wp;
        }
    }
    // a wait gave up, here or earlier: parts are missing
    if (*reinterpret_cast<volatile int*>(a.status) != 0) sum = __uint_as_float(kNaN32);
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int c = 0; c < C / 2; ++c)
        reinterpret_cast<uint32_t*>(o + row * D + C * lane)[c] = pack2<T>(sum != 0.f ? acc[2 * c] * inv : 0.f, sum != 0.f ? acc[2 * c + 1] * inv : 0.f);
    if (lane == 0) lse[((int64_t)b * a.H + h) * a.N + i] = sum != 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

// How a call is cut up, from its sizes alone: the workspace and the kernels go by the same plan.
struct Plan {
    bool prefix_item, prefix_tiles, own;
    int pack, per_block, blocks, parts, ctas, row_tiles;
    int64_t rows;
    int64_t bytes_parts, bytes_a, bytes_b, bytes_first;
    long long bytes() const { return bytes_parts + bytes_a + bytes_b + bytes_first; }
};

// Heads of a row group here: the most of a group that 64 rows can hold.
int own_pack(int G) {
    for (int d = G < ROWS ? G : ROWS; d > 1; --d)
        if (G % d == 0) return d;
    return 1;
}

Plan make_plan(int B, int N, int H, int Hk, int D, int prefix_len, int width) {
    Plan p{};
    const int G = H / Hk;
    p.rows = (int64_t)B * N * H;
    p.pack = own_pack(G);
    p.per_block = std::min(N, std::max(1, ROWS / p.pack));
    p.blocks = (N + p.per_block - 1) / p.per_block;
    const int64_t prefix_rows = (int64_t)B * N * p.pack;
    p.prefix_item = prefix_len > 0 && prefix_rows <= ROWS;
    p.prefix_tiles = prefix_len > 0 && !p.prefix_item;
    p.own = width > 0 || p.prefix_item;
    const int most = std::max(width > 0 ? p.per_block * p.pack : 1, p.prefix_item ? (int)prefix_rows : 1);
    p.row_tiles = most <= 16 ? 1 : most <= 32 ? 2 : 4;
    const int sms = sm_count();
    p.ctas = 2 * sms;
    if (p.prefix_tiles) {
        // the keys of a tile pair shared out over as many CTAs as make the waves shortest; START: a CTA's start and end, and its share of the
        // joining, in key tiles
        constexpr int START = 4;
        const int pack = rows_pack(G), span = 2 * (TM / pack);
        const int64_t tiles = (int64_t)(H / pack) * (((int64_t)B * N + span - 1) / span), keys = (prefix_len + TN - 1) / TN;
        int64_t best = INT64_MAX;
        for (int n = 1; n <= std::min<int64_t>(keys, 64); ++n) {
            const int64_t cost = ((tiles * n + sms - 1) / sms) * ((keys + n - 1) / n + START);
            if (cost < best) { best = cost; p.parts = n; }
        }
    }
    const int64_t row = (int64_t)D * 4 + 4;
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    p.bytes_parts = up((p.prefix_tiles ? p.parts : p.prefix_item ? 1 : 0) * p.rows * row);
    p.bytes_a = width > 0 ? up(p.rows * row) : 0;
    p.bytes_b = p.own ? up((int64_t)p.ctas * ROWS * row) : 0;
    p.bytes_first = p.own ? up((int64_t)(B + 1) * 8) : 0;
    return p;
}

template <typename T, int D, int MT>
int launch_own(const CUtensorMap& tk, const CUtensorMap& tv, const PrefixArgs& a, bool behind_prefix, cudaStream_t st) {
    auto kern = own_kernel<T, D, MT>;
    constexpr int bytes = (int)Own<D, MT>::BYTES;
    if (int rc = opt_in_shared_memory((const void*)kern, bytes)) return rc;
    // behind the kernel of the prefix it may start as that one's CTAs end: they have nothing to do with one another
    if (behind_prefix) {
        const cudaError_t e = launch_dependent(kern, dim3(a.ctas), dim3(OWN_THREADS), bytes, st, tk, tv, a);
        if (e != cudaSuccess) return set_error(-2, cudaGetErrorString(e));
    } else {
        kern<<<a.ctas, OWN_THREADS, bytes, st>>>(tk, tv, a);
    }
    ES_CHECK_LAUNCH("own_kernel");
    return 0;
}

template <typename T, int D>
int launch_own(const void* k, CacheRows rk, const void* v, CacheRows rv, const PrefixArgs& a, int row_tiles, bool behind_prefix, cudaStream_t st) {
    CUtensorMap tk, tv;
    if (int rc = make_pages_map<T>(&tk, k, D, a.Hk, 1 << a.log_page, a.pages, rk, UNIT)) return rc;
    if (int rc = make_pages_map<T>(&tv, v, D, a.Hk, 1 << a.log_page, a.pages, rv, UNIT)) return rc;
    return row_tiles == 1 ? launch_own<T, D, 1>(tk, tv, a, behind_prefix, st) : row_tiles == 2 ? launch_own<T, D, 2>(tk, tv, a, behind_prefix, st)
                                                                                              : launch_own<T, D, 4>(tk, tv, a, behind_prefix, st);
}

}  // namespace
}  // namespace packed
}  // namespace es

using namespace es;
using namespace es::packed;

extern "C" long long es_prefix_workspace_bytes(int32_t batch, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t D, int32_t prefix_len, int32_t table_width,
                                               int32_t page_size) {
    (void)page_size;
    if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || prefix_len < 0 || table_width < 0) return 0;
    return make_plan(batch, tokens, heads, kv_heads, D, prefix_len, table_width).bytes();
}

extern "C" int es_prefix_attn(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse, const int32_t* prefix_pages,
                              int32_t n_prefix_pages, int32_t prefix_len, const int32_t* table, int32_t table_width, const int32_t* lengths,
                              int32_t batch, int32_t tokens, int32_t heads, int32_t kv_heads, int32_t D, int32_t pages, int32_t page_size,
                              int64_t k_page, int64_t k_token, int64_t k_head, int64_t v_page, int64_t v_token, int64_t v_head, float scale,
                              int32_t dtype, void* workspace, void* stream) {
    if (int rc = check_sizes("es_prefix_attn", batch, tokens, prefix_len, heads, kv_heads, D, dtype)) return rc;
    if (int rc = check_scale("es_prefix_attn", scale)) return rc;
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        return set_error(-1, "es_prefix_attn: page_size must be 16, 32, 64, 128 or 256");
    if (pages < 0 || table_width < 0 || n_prefix_pages < 0 || (int64_t)table_width * page_size > 0x7FFFFF00 || (int64_t)pages * page_size > 0x7FFFFFFF ||
        (int64_t)n_prefix_pages * page_size < prefix_len || (int64_t)batch * tokens * heads > 0x7FFFFFFF)
        return set_error(-1, "es_prefix_attn: sizes out of range");
    if (batch > MOST_REQUESTS) return set_error(-1, "es_prefix_attn: at most 2^23 requests");
    if (batch == 0 || tokens == 0) return 0;
    if (!q || !o || !lse || !lengths || (prefix_len && !prefix_pages) || (table_width && !table) || (pages && (!k_cache || !v_cache)))
        return set_error(-1, "es_prefix_attn: null pointer");
    if (!aligned(16, q, k_cache, v_cache, o) || !aligned(32, workspace) || !aligned(4, lse, prefix_pages, table, lengths))
        return set_error(-1, "es_prefix_attn: q, k_cache, v_cache, o must be 16-byte, the workspace 32-byte, lse and the int32 arrays 4-byte aligned");
    if (!whole_chunks(k_page, k_token, k_head, v_page, v_token, v_head)) return set_error(-1, "es_prefix_attn: strides must be multiples of 8 elements");
    if (pages == 0) prefix_len = table_width = 0;             // no key can be attended to
    const Plan p = make_plan(batch, tokens, heads, kv_heads, D, prefix_len, table_width);
    if (p.bytes() && !workspace) return set_error(-1, "es_prefix_attn: null pointer (workspace)");
    const CacheRows rk{k_page, k_token, k_head}, rv{v_page, v_token, v_head};
    const cudaStream_t st = (cudaStream_t)stream;
    PrefixArgs a{};
    a.prefix_pages = prefix_pages; a.table = table; a.lengths = lengths;
    a.prefix_len = prefix_len; a.width = table_width; a.B = batch; a.N = tokens; a.H = heads; a.Hk = kv_heads; a.pages = pages;
    while ((1 << a.log_page) < page_size) ++a.log_page;
    a.scale = scale;
    a.pack = p.pack; a.per_block = p.per_block; a.blocks = p.blocks; a.vheads = heads / p.pack;
    a.prefix_item = p.prefix_item; a.ctas = p.ctas; a.q = q; a.v = v_cache; a.rv = rv;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int n_parts = p.prefix_tiles ? p.parts : p.prefix_item ? 1 : 0;
    a.p_o = reinterpret_cast<float*>(ws); a.p_lse = a.p_o + n_parts * p.rows * D; a.p_parts = p.prefix_tiles ? p.parts : 0;
    a.a_o = reinterpret_cast<float*>(ws + p.bytes_parts); a.a_lse = a.a_o + p.rows * D;
    a.b_o = reinterpret_cast<float*>(ws + p.bytes_parts + p.bytes_a); a.b_lse = a.b_o + (int64_t)p.ctas * ROWS * D;
    a.first = p.own ? reinterpret_cast<long long*>(ws + p.bytes_parts + p.bytes_a + p.bytes_b) : nullptr;
    a.status = device_status_ptr();
    if (!a.status) return set_error(-2, "es_prefix_attn: the device status word is not available on this device");
    if (p.prefix_tiles)
        if (int rc = prefix_fwd_tc(q, k_cache, rk, v_cache, rv, a.p_o, a.p_lse, p.parts, prefix_pages, prefix_len, batch * tokens, heads, kv_heads, pages, a.log_page,
                                   scale, D, dtype, st))
            return rc;
    auto go = [&](auto t, auto d) {
        using T = decltype(t);
        if (p.own)
            if (int rc = launch_own<T, d>(k_cache, rk, v_cache, rv, a, p.row_tiles, p.prefix_tiles, st)) return rc;
        const cudaError_t e = launch_dependent(join_kernel<T, d>, dim3((unsigned)((p.rows + 7) / 8)), dim3(256), 0, st, (T*)o, lse, a);
        if (e != cudaSuccess) return set_error(-2, cudaGetErrorString(e));
        ES_CHECK_LAUNCH("join_kernel");
        return 0;
    };
    if (dtype == 0) return D == 64 ? go(__nv_bfloat16{}, std::integral_constant<int, 64>{}) : go(__nv_bfloat16{}, std::integral_constant<int, 128>{});
    return D == 64 ? go(__half{}, std::integral_constant<int, 64>{}) : go(__half{}, std::integral_constant<int, 128>{});
}
