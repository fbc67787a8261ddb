// Attention of a batch's newest tokens to a shared prefix and to each request's own tokens, both in pages of a cache.
//
// The keys of a row are two sets, the prefix and its request's own; each gives a partial result O_p = softmax(S_p) V_p with its LSE z_p (log2),
// and they are joined by O = sum_p 2^(z_p - M) O_p / sum_p 2^(z_p - M).
//   prefix       all rows of the batch that read a key head see the same keys. More than ROWS of them: the tcgen05 kernel of es_packed_fwd.cu,
//                128 rows to a tile, the keys shared out over the SMs. Fewer: as one more item of the kernel below.
//   own tokens   `own_kernel`: tokens x heads of a group rows against each request's pages. Every key is read once and multiplied with a few
//                rows: bound by HBM. Warps with m16n8k16 MMAs, 64 keys at a time, scores and P in registers: the tensor cores are idle most of the
//                time at any shape (16 FLOP a byte; tcgen05 with its 128 rows would compute eight times as much for the same bytes).
// Work of own_kernel: the (request, heads, block of new tokens) items, each a run of 64-key units, one behind the other; CTA c of C takes the
// units c W / C .. (c + 1) W / C of W whatever the lengths are. An item's first share is stored by its rows (part A), one that starts inside an
// item by its CTA (part B; a CTA has at most one). The merge finds them by the same arithmetic.
#include "es_packed_tc.cuh"
#include "es_vsa_mma.cuh"

namespace es {
namespace packed {

int prefix_fwd_tc(const void* q, const void* k, CacheRows rk, const void* v, CacheRows rv, float* part_o, float* part_lse, int parts, const int* list, int prefix_len,
                  int tokens, int H, int Hk, int pages, int log_page, float scale, int D, int dtype, cudaStream_t st);

namespace {
constexpr int UNIT = 64, WARPS = 4, OWN_THREADS = 32 * (WARPS + 1), ROWS = 64;
constexpr int GROUPS = 1024;                                  // requests (or groups of them) whose running sums a CTA keeps

__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

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
    long long* first;                // [B + 1] first unit of each request: written by CTA 0
    int* status;
};

__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) { return min(max(__ldg(a.lengths + b), 0), a.width << a.log_page); }
__device__ __forceinline__ long long prefix_units(const PrefixArgs& a) {
    return a.prefix_item ? (long long)(a.prefix_len + UNIT - 1) / UNIT * a.vheads : 0;
}

template <int D> struct Own {
    static constexpr uint32_t HALF = UNIT * 128, TILE = UNIT * D * 2;
    static constexpr int NSLOT = D == 128 ? 5 : 8;             // two CTAs per SM
    static constexpr uint32_t RING = 0, SUM = NSLOT * TILE, CTL = SUM + 2 * 16 * D * 4, SCAN = CTL + 512, BYTES = SCAN + (GROUPS + 1) * 8;
};
struct OwnCtl {
    uint64_t full[8], empty[8];
    int abort, not_finite;
    float ml[2][32];                 // maxima and sums of the warps that are joined with others
    long long warp_sum[WARPS + 1];
};
static_assert(sizeof(OwnCtl) <= 512, "control block");

// One share of an item: rows of one request (or of the batch, for the prefix) against its units from .. to.
struct Share {
    int b;               // request, -1: the prefix
    int head0, t0, rows; // first head, first new token of the item (in the batch), rows
    int u0, u1;          // units of the item
    bool starts;         // from the item's first unit
    int n;               // keys of the item
};

// Finds the item of unit u: which request, heads and block of tokens, and the unit's number in it.
struct Finder {
    const PrefixArgs& a;
    const long long* sums;           // units before group g of requests
    int group;                       // requests in a group
    __device__ __forceinline__ Share at(long long u, long long end) const {
        Share s;
        const long long pu = prefix_units(a);
        long long per;
        long long x;
        if (u < pu) {
            s.b = -1;
            s.n = a.prefix_len;
            x = u;
        } else {
            int lo = 0, hi = (a.B + group - 1) / group;
            while (lo + 1 < hi) {
                const int m = (lo + hi) >> 1;
                if (sums[m] <= u) lo = m; else hi = m;
            }
            int b = lo * group;
            long long f = sums[lo], w;
            while (f + (w = units(b)) <= u) { f += w; ++b; }
            s.b = b;
            s.n = own_length(a, b);
            x = u - f;
        }
        per = (s.n + UNIT - 1) / UNIT;
        const int item = (int)(x / per);
        s.u0 = (int)(x - item * per);
        s.u1 = (int)min(per, s.u0 + (end - u));
        s.starts = s.u0 == 0;
        s.head0 = item % a.vheads * a.pack;
        const int blk = s.b < 0 ? 0 : item / a.vheads, tokens = s.b < 0 ? a.B * a.N : min(a.per_block, a.N - blk * a.per_block);
        s.t0 = s.b < 0 ? 0 : s.b * a.N + blk * a.per_block;
        s.rows = tokens * a.pack;
        return s;
    }
    __device__ __forceinline__ long long units(int b) const { return (long long)((own_length(a, b) + UNIT - 1) / UNIT) * a.vheads * a.blocks; }
};

// MT: 16-row tiles of an item. One: every warp has them and a quarter of a unit's keys; two: two warps each and half; four: all keys.
template <typename T, int D, int MT>
__global__ void __launch_bounds__(OWN_THREADS, 2)
own_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PrefixArgs a) {
    using C = Own<D>;
    using E = vsa::Elt<T>;
    constexpr int WK = WARPS / MT, KW = UNIT / WK;            // warps that share a row tile, keys of a warp in a unit
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(smem);
    OwnCtl* ctl = reinterpret_cast<OwnCtl*>(smem + C::CTL);
    long long* sums = reinterpret_cast<long long*>(smem + C::SCAN);
    volatile int* abort_flag = &ctl->abort;
    if (tid == 0) {
        const int earlier = *reinterpret_cast<volatile int*>(a.status);
        for (int i = 0; i < C::NSLOT; ++i) {
            mbar_init(smem_u32(&ctl->full[i]), 1);
            mbar_init(smem_u32(&ctl->empty[i]), WARPS);
        }
        ctl->not_finite = 0;
        ctl->abort = (base & 1023u) || earlier ? 1 : 0;      // the swizzled tiles need a 1024-byte aligned base
        if (base & 1023u) atomicCAS(a.status, 0, 913);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    // running sums of the units over groups of requests
    const Finder find{a, sums, max(1, (a.B + GROUPS - 1) / GROUPS)};
    const int groups = (a.B + find.group - 1) / find.group, per = (groups + OWN_THREADS - 1) / OWN_THREADS;
    long long mine = 0;
    for (int g = tid * per; g < min(groups, (tid + 1) * per); ++g)
        for (int b = g * find.group; b < min(a.B, (g + 1) * find.group); ++b) mine += find.units(b);
    long long run = mine;
    for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += y;
    }
    if (lane == 31) ctl->warp_sum[warp] = run;
    __syncthreads();
    long long W = prefix_units(a);
    run += W - mine;
    for (int w = 0; w <= WARPS; ++w) {
        if (w < warp) run += ctl->warp_sum[w];
        W += ctl->warp_sum[w];
    }
    for (int g = tid * per; g < min(groups, (tid + 1) * per); ++g) {
        sums[g] = run;
        for (int b = g * find.group; b < min(a.B, (g + 1) * find.group); ++b) {
            if (blockIdx.x == 0) a.first[b] = run;
            run += find.units(b);
        }
    }
    if (blockIdx.x == 0 && tid == 0) a.first[a.B] = W;
    __syncthreads();
    // (no more CTAs than units: each has one at least)
    const long long ctas = min((long long)a.ctas, W);
    const long long beg = blockIdx.x < ctas ? W * blockIdx.x / ctas : 0, end = blockIdx.x < ctas ? W * (blockIdx.x + 1) / ctas : 0;
    const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
    bool ok = *abort_flag == 0;

    if (warp == WARPS) {
        // ------------------------------------------------------------ loads: K and V of every unit, a lane per box
        const int box = min(UNIT, 1 << a.log_page), boxes = UNIT / box;
        uint32_t slot = 0, par = 1, issued = 0;
        if (lane == 0) {
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
        }
        for (long long u = beg; u < end && ok;) {
            const Share s = find.at(u, end);
            const int* list = s.b < 0 ? a.prefix_pages : a.table + (size_t)s.b * a.width;
            const int kh = s.head0 / (a.H / a.Hk);
            for (int i = s.u0; i < s.u1 && ok; ++i) {
                const int k = i * UNIT + lane * box;
                int page = a.pages;                           // a page that is not of the cache, or behind the keys, is loaded as zeros
                if (lane < boxes && k < s.n) {
                    const int p = __ldg(list + (k >> a.log_page));
                    if (p >= 0 && p < a.pages) page = p;
                }
                for (int x = 0; x < 2 && ok; ++x) {
                    ok = mbar_wait_warp(empty0 + 8 * slot, par, abort_flag, a.status, 661);
                    if (!ok) break;
                    const uint32_t bar = full0 + 8 * slot, dst = base + C::RING + slot * C::TILE;
                    if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE);
                    __syncwarp();
                    if (lane < boxes)
                        for (int d = 0; d < D / 64; ++d)
                            tma_load_4d(dst + d * C::HALF + lane * box * 128, x ? &tmV : &tmK, bar, 64 * d, kh, (i * UNIT) & ((1 << a.log_page) - 1), page);
                    __syncwarp();
                    ++issued;
                    if (++slot == C::NSLOT) { slot = 0; par ^= 1; }
                }
            }
            u += s.u1 - s.u0;
        }
        __syncwarp();
        if (lane == 0 && *abort_flag) {
            // a wait gave up: give the loads a moment (100 us in all) to land before shared memory goes away
            const uint64_t t_end = global_timer_ns() + 100000ull;
            for (uint32_t back = 1; back <= (uint32_t)C::NSLOT && back <= issued; ++back) {
                const uint32_t sq = issued - back;
                while (!mbar_try_wait(full0 + 8 * (sq % C::NSLOT), (sq / C::NSLOT) & 1) && global_timer_ns() < t_end) {}
            }
        }
    } else {
        const int mt = warp / WK, wk = warp % WK;             // row tile, share of the keys
        const int r0 = 16 * mt + (lane >> 2), r1 = r0 + 8;
        const float c = a.scale * kLog2e;
        uint32_t seq = 0;
        for (long long u = beg; u < end;) {
            const Share s = find.at(u, end);
            const int* list = s.b < 0 ? a.prefix_pages : a.table + (size_t)s.b * a.width;
            // keys that the thread's two rows see, and the fewest and most that any row of the item sees
            auto seen = [&](int row) {
                if (s.b < 0) return s.n;
                const int t = s.t0 - s.b * a.N + row / a.pack;
                return max(s.n - a.N + t + 1, 0);
            };
            const int v0 = r0 < s.rows ? seen(r0) : 0, v1 = r1 < s.rows ? seen(r1) : 0, least = seen(0), most = seen(s.rows - 1);
            uint32_t qf[D / 16][4];
            const T* q = static_cast<const T*>(a.q);
            auto q_at = [&](int row) { return q + ((int64_t)(s.t0 + row / a.pack) * a.H + s.head0 + row % a.pack) * D + 2 * (lane & 3); };
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                qf[ks][0] = r0 < s.rows ? *reinterpret_cast<const uint32_t*>(q_at(r0) + 16 * ks) : 0u;
                qf[ks][1] = r1 < s.rows ? *reinterpret_cast<const uint32_t*>(q_at(r1) + 16 * ks) : 0u;
                qf[ks][2] = r0 < s.rows ? *reinterpret_cast<const uint32_t*>(q_at(r0) + 16 * ks + 8) : 0u;
                qf[ks][3] = r1 < s.rows ? *reinterpret_cast<const uint32_t*>(q_at(r1) + 16 * ks + 8) : 0u;
            }
            float o[D / 8][4];
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
            for (int i = s.u0; i < s.u1; ++i) {
                const int k0 = i * UNIT + wk * KW;            // this warp's keys k0 .. k0 + KW - 1
                uint32_t slot = seq % C::NSLOT;
                ok = ok && mbar_wait_warp(full0 + 8 * slot, (seq / C::NSLOT) & 1, abort_flag, a.status, 662);
                ++seq;
                float x[KW / 8][4];
                if (ok) {
                    const uint32_t kb = base + C::RING + slot * C::TILE;
#pragma unroll
                    for (int j = 0; j < KW / 8; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                        for (int j = 0; j < KW / 16; ++j) {
                            // 16 keys x 16 d: lanes 0-7, 8-15 rows 0-7 (d 0-7, 8-15), lanes 16-31 rows 8-15
                            const int row = wk * KW + 16 * j + (lane & 7) + ((lane >> 4) << 3), ch = 2 * (ks & 3) + ((lane >> 3) & 1);
                            uint32_t b0, b1, b2, b3;
                            vsa::ldsm4(kb + (ks >> 2) * C::HALF + row * 128 + ((ch ^ (row & 7)) << 4), b0, b1, b2, b3);
                            E::mma(x[2 * j], qf[ks], b0, b1);
                            E::mma(x[2 * j + 1], qf[ks], b2, b3);
                        }
                    // a page that is not of the cache: its keys are not attended to
                    if (i * UNIT + UNIT > least) {
#pragma unroll
                        for (int j = 0; j < KW / 8; ++j) {
                            const int k = k0 + 8 * j + 2 * (lane & 3);
                            if (k >= v0) x[j][0] = -INFINITY;
                            if (k + 1 >= v0) x[j][1] = -INFINITY;
                            if (k >= v1) x[j][2] = -INFINITY;
                            if (k + 1 >= v1) x[j][3] = -INFINITY;
                        }
                    }
                    const int kp = k0 + 16 * lane;             // (pages hold 16 keys at least)
                    const int pg = 16 * lane < KW && kp < s.n ? __ldg(list + (kp >> a.log_page)) : 0;
                    const uint32_t bad = __ballot_sync(0xffffffffu, pg < 0 || pg >= a.pages);
                    if (bad)
#pragma unroll
                        for (int j = 0; j < KW / 8; ++j)
                            if ((bad >> (j / 2)) & 1) x[j][0] = x[j][1] = x[j][2] = x[j][3] = -INFINITY;
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
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty0 + 8 * slot);
                slot = seq % C::NSLOT;
                ok = ok && mbar_wait_warp(full0 + 8 * slot, (seq / C::NSLOT) & 1, abort_flag, a.status, 663);
                ++seq;
                if (ok) {
                    const uint32_t vb = base + C::RING + slot * C::TILE;
                    if (k0 + KW > least) {
                        // V rows that some row does not see: what is not finite there is set to 0 (0 times it would be NaN), and given at the end to
                        // the rows that do see it
                        for (int e = lane; e < KW * (D / 8); e += 32) {
                            const int row = wk * KW + e / (D / 8), ch = e % (D / 8);
                            uint4* p = reinterpret_cast<uint4*>(smem + C::RING + slot * C::TILE + (ch >> 3) * C::HALF + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                            const uint4 w = *p;
                            if (i * UNIT + row >= least && (not_finite<T>(w.x) || not_finite<T>(w.y) || not_finite<T>(w.z) || not_finite<T>(w.w))) {
                                if (i * UNIT + row < most) *reinterpret_cast<volatile int*>(&ctl->not_finite) = 1;
                                *p = make_uint4(finite_only<T>(w.x), finite_only<T>(w.y), finite_only<T>(w.z), finite_only<T>(w.w));
                            }
                        }
                        __syncwarp();
                        fence_proxy_async_smem();
                    }
#pragma unroll
                    for (int j = 0; j < KW / 16; ++j) {
                        const uint32_t p[4] = {pack2<T>(x[2 * j][0], x[2 * j][1]), pack2<T>(x[2 * j][2], x[2 * j][3]), pack2<T>(x[2 * j + 1][0], x[2 * j + 1][1]),
                                               pack2<T>(x[2 * j + 1][2], x[2 * j + 1][3])};
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
                            // 16 keys x 16 d, transposed: lanes 0-15 keys 0-15 of d 0-7, lanes 16-31 of d 8-15
                            const int row = wk * KW + 16 * j + (lane & 15), ch = 2 * (d & 3) + (lane >> 4);
                            uint32_t b0, b1, b2, b3;
                            ldsm4_trans(vb + (d >> 2) * C::HALF + row * 128 + ((ch ^ (row & 7)) << 4), b0, b1, b2, b3);
                            E::mma(o[2 * d], p, b0, b1);
                            E::mma(o[2 * d + 1], p, b2, b3);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty0 + 8 * slot);
            }
            l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
            // (another warp with the same keys may have found it)
            if (least < most) named_sync(1, 32 * WARPS);
            if (least < most && *reinterpret_cast<volatile int*>(&ctl->not_finite)) {
                const int kh = s.head0 / (a.H / a.Hk);
                for (int k = max(least, s.u0 * UNIT); k < min(most, s.u1 * UNIT); ++k) {
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
            // join the warps that share the rows, halving their number
            float* sum = reinterpret_cast<float*>(smem + C::SUM);
#pragma unroll
            for (int half = WK / 2; half; half >>= 1) {
                const int pair = mt * half + (wk % half);
                float* dst = sum + (size_t)pair * 16 * D;
                if (wk >= half && wk < 2 * half) {
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        *reinterpret_cast<float4*>(dst + (j * 32 + lane) * 4) = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
                    }
                    if ((lane & 3) == 0) {
                        ctl->ml[pair][lane >> 2] = m0; ctl->ml[pair][8 + (lane >> 2)] = m1;
                        ctl->ml[pair][16 + (lane >> 2)] = l0; ctl->ml[pair][24 + (lane >> 2)] = l1;
                    }
                }
                named_sync(1, 32 * WARPS);
                if (wk < half) {
                    const float n0 = ctl->ml[pair][lane >> 2], n1 = ctl->ml[pair][8 + (lane >> 2)], t0 = fmaxf(m0, n0), t1 = fmaxf(m1, n1);
                    const float f0 = t0 == -INFINITY ? 0.f : ex2_approx(m0 - t0), f1 = t1 == -INFINITY ? 0.f : ex2_approx(m1 - t1);
                    const float g0 = t0 == -INFINITY ? 0.f : ex2_approx(n0 - t0), g1 = t1 == -INFINITY ? 0.f : ex2_approx(n1 - t1);
                    l0 = l0 * f0 + ctl->ml[pair][16 + (lane >> 2)] * g0;
                    l1 = l1 * f1 + ctl->ml[pair][24 + (lane >> 2)] * g1;
                    m0 = t0; m1 = t1;
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        const float4 w = *reinterpret_cast<const float4*>(dst + (j * 32 + lane) * 4);
                        o[j][0] = o[j][0] * f0 + w.x * g0; o[j][1] = o[j][1] * f0 + w.y * g0;
                        o[j][2] = o[j][2] * f1 + w.z * g1; o[j][3] = o[j][3] * f1 + w.w * g1;
                    }
                }
                named_sync(1, 32 * WARPS);
            }
            if (wk == 0) {
                const float i0 = l0 != 0.f ? 1.f / l0 : 0.f, i1 = l1 != 0.f ? 1.f / l1 : 0.f;
                auto store = [&](int row, float m, float l, float inv, int e) {
                    if (row >= s.rows) return;
                    const int64_t at = (int64_t)(s.t0 + row / a.pack) * a.H + s.head0 + row % a.pack;
                    float* dst = s.starts ? (s.b < 0 ? a.p_o : a.a_o) + at * D : a.b_o + ((int64_t)blockIdx.x * ROWS + row) * D;
                    float* z = s.starts ? (s.b < 0 ? a.p_lse : a.a_lse) + at : a.b_lse + (int64_t)blockIdx.x * ROWS + row;
                    const bool lost = *abort_flag != 0;       // a wait gave up: NaN
#pragma unroll
                    for (int j = 0; j < D / 8; ++j)
                        *reinterpret_cast<float2*>(dst + 8 * j + 2 * (lane & 3)) =
                            lost ? make_float2(__uint_as_float(kNaN32), __uint_as_float(kNaN32)) : make_float2(o[j][e] * inv, o[j][e + 1] * inv);
                    if ((lane & 3) == 0) *z = lost ? __uint_as_float(kNaN32) : l != 0.f ? m + log2f(l) : -INFINITY;
                };
                store(r0, m0, l0, i0, 0);
                store(r1, m1, l1, i1, 2);
            }
            u += s.u1 - s.u0;
        }
    }
    __syncthreads();
}

// A warp per row: the parts of the prefix, part A of the row's own item, and the part B's of the CTAs that went on with it.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(T* o, float* lse, const __grid_constant__ PrefixArgs a) {
    constexpr int C = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)a.B * a.N * a.H, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int h = (int)(row % a.H), t = (int)(row / a.H), b = t / a.N, i = t % a.N, vh = h / a.pack;
    float acc[C] = {}, sum = 0.f, top = -INFINITY;
    auto add = [&](const float* src, float z) {
        if (z == -INFINITY) return;
        const float next = fmaxf(top, z), f = ex2_approx(top - next), g = z != z ? z : ex2_approx(z - next);
        top = next;
        sum = sum * f + g;
        if constexpr (C == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + C * lane);
            acc[0] = acc[0] * f + v.x * g; acc[1] = acc[1] * f + v.y * g; acc[2] = acc[2] * f + v.z * g; acc[3] = acc[3] * f + v.w * g;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(src + C * lane);
            acc[0] = acc[0] * f + v.x * g; acc[1] = acc[1] * f + v.y * g;
        }
    };
    const long long W = a.first ? a.first[a.B] : 0, ctas = min((long long)a.ctas, W);
    // an item's parts: A, and B of the CTAs after the one with its first unit up to the one with its last
    auto item = [&](long long u, long long units, const float* po, const float* pl, int r) {
        if (units <= 0) return;
        add(po + row * D, pl[row]);
        const int c0 = (int)(((u + 1) * ctas - 1) / W), c1 = (int)(((u + units) * ctas - 1) / W);
        for (int c = c0 + 1; c <= c1; ++c) add(a.b_o + ((int64_t)c * ROWS + r) * D, a.b_lse[(int64_t)c * ROWS + r]);
    };
    if (a.prefix_item) {
        const long long n = (a.prefix_len + UNIT - 1) / UNIT;
        item(vh * n, n, a.p_o, a.p_lse, t * a.pack + h % a.pack);
    } else {
        for (int p = 0; p < a.p_parts; ++p) add(a.p_o + (p * rows + row) * D, a.p_lse[p * rows + row]);
    }
    if (a.first) {
        const long long n = (own_length(a, b) + UNIT - 1) / UNIT;
        const int blk = i / a.per_block;
        item(a.first[b] + (blk * a.vheads + vh) * n, n, a.a_o, a.a_lse, (i - blk * a.per_block) * a.pack + h % a.pack);
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int c = 0; c < C / 2; ++c)
        reinterpret_cast<uint32_t*>(o + row * D + C * lane)[c] = pack2<T>(sum != 0.f ? acc[2 * c] * inv : 0.f, sum != 0.f ? acc[2 * c + 1] * inv : 0.f);
    if (lane == 0) lse[((int64_t)b * a.H + h) * a.N + i] = sum != 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
    return n;
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

template <typename T, int D> int launch_own(const void* k, CacheRows rk, const void* v, CacheRows rv, const PrefixArgs& a, int row_tiles, cudaStream_t st) {
    CUtensorMap tk, tv;
    if (int rc = make_pages_map<T>(&tk, k, D, a.Hk, 1 << a.log_page, a.pages, rk, UNIT)) return rc;
    if (int rc = make_pages_map<T>(&tv, v, D, a.Hk, 1 << a.log_page, a.pages, rv, UNIT)) return rc;
    auto kern = row_tiles == 1 ? own_kernel<T, D, 1> : row_tiles == 2 ? own_kernel<T, D, 2> : own_kernel<T, D, 4>;
    if (int rc = opt_in_shared_memory((const void*)kern, (int)Own<D>::BYTES)) return rc;
    kern<<<a.ctas, OWN_THREADS, Own<D>::BYTES, st>>>(tk, tv, a);
    ES_CHECK_LAUNCH("own_kernel");
    return 0;
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
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        return set_error(-1, "es_prefix_attn: page_size must be 16, 32, 64, 128 or 256");
    if (pages < 0 || table_width < 0 || n_prefix_pages < 0 || (int64_t)table_width * page_size > 0x7FFFFFFF || (int64_t)pages * page_size > 0x7FFFFFFF ||
        (int64_t)n_prefix_pages * page_size < prefix_len || (int64_t)batch * tokens * heads > 0x7FFFFFFF)
        return set_error(-1, "es_prefix_attn: sizes out of range");
    if (batch == 0 || tokens == 0) return 0;
    if (!q || !o || !lse || !lengths || (prefix_len && !prefix_pages) || (table_width && !table) || (pages && (!k_cache || !v_cache)))
        return set_error(-1, "es_prefix_attn: null pointer");
    if (!aligned(16, q, k_cache, v_cache, o, workspace)) return set_error(-1, "es_prefix_attn: q, k_cache, v_cache, o, workspace must be 16-byte aligned");
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
            if (int rc = launch_own<T, d>(k_cache, rk, v_cache, rv, a, p.row_tiles, st)) return rc;
        join_kernel<T, d><<<(unsigned)((p.rows + 7) / 8), 256, 0, st>>>((T*)o, lse, a);
        ES_CHECK_LAUNCH("join_kernel");
        return 0;
    };
    if (dtype == 0) return D == 64 ? go(__nv_bfloat16{}, std::integral_constant<int, 64>{}) : go(__nv_bfloat16{}, std::integral_constant<int, 128>{});
    return D == 64 ? go(__half{}, std::integral_constant<int, 64>{}) : go(__half{}, std::integral_constant<int, 128>{});
}
