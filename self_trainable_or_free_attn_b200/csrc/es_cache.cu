// A paged cache of keys and values: pages and slots of new tokens, and storing them. (Attention to it: es_prefix.cu.)
#include "es_packed.cuh"

namespace es {
namespace packed {
namespace {

// ---------------------------------------------------------------------------------------------- pages and slots
constexpr int PLAN_THREADS = 256, PLAN_CHUNK = 1024;          // requests that a CTA scans at a time
constexpr int PLAN_TOKENS = 256;                              // tokens of a CTA: one to a thread

struct PlanArgs {
    const int *lengths, *new_tokens, *free_pages;
    int *table, *slots, *positions, *cu_new, *lengths_out, *taken;
    int n_free, B, width, page, total;
};

// Pages of x tokens (x below 2^32, which the sum of two lengths is).
__device__ __forceinline__ unsigned pages_of(unsigned x, unsigned page) { return x ? (x - 1) / page + 1 : 0; }

// With len = lengths[b], n = new_tokens[b]: the request has have = ceil(len / page) pages and wants ceil((len + n) / page), at most the row's
// width; its missing pages are free_pages[first ...], first the exclusive sum of need = wanted - held over the requests before it. Every CTA
// makes both running sums itself (a few KB of L2 per thousand requests; a second kernel would cost a launch) and then places its own
// share of the requests and of the tokens. Bound by latency: lengths, the free list or the table, stores (calls behind one another: 3.9 us for 256
// requests of one token, 4.5 for 48 of 341 each in pages of 64). A request's new entries are written by its one thread, 50 ns each: 16,384
// tokens of a single request take 16 us in pages of 64 and 51 in pages of 16.
__global__ void __launch_bounds__(PLAN_THREADS) extend_tables_kernel(PlanArgs a) {
    __shared__ int s_cu[PLAN_CHUNK + 1], s_first[PLAN_CHUNK], s_len[PLAN_CHUNK];
    __shared__ long long s_warp[2][PLAN_THREADS / 32];
    constexpr int PER = PLAN_CHUNK / PLAN_THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long cap = 0x7FFFFFFF;
    const unsigned page = (unsigned)a.page, width = (unsigned)a.width;
    long long tokens = 0, pages = 0, missing = 0;             // of the chunks before (the sums may pass 32 bits; what is stored saturates)
    const long long t0 = (long long)blockIdx.x * PLAN_TOKENS, t1 = min(t0 + PLAN_TOKENS, (long long)a.total);
    for (int b0 = 0; b0 < a.B; b0 += PLAN_CHUNK) {
        const int nb = min(PLAN_CHUNK, a.B - b0);
        unsigned len[PER], n[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = tid * PER + i;
            len[i] = r < nb ? max(a.lengths[b0 + r], 0) : 0;
            n[i] = r < nb ? max(a.new_tokens[b0 + r], 0) : 0;
        }
        long long need[PER], sn = 0, sp = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            need[i] = (long long)min(pages_of(len[i] + n[i], page), width) - (long long)min(pages_of(len[i], page), width);
            sn += n[i]; sp += need[i];
        }
        long long xn = sn, xp = sp;
        for (int d = 1; d < 32; d <<= 1) {
            const long long yn = __shfl_up_sync(0xffffffffu, xn, d), yp = __shfl_up_sync(0xffffffffu, xp, d);
            if (lane >= d) { xn += yn; xp += yp; }
        }
        if (lane == 31) { s_warp[0][warp] = xn; s_warp[1][warp] = xp; }
        __syncthreads();
        long long bn = tokens, bp = pages, an = tokens, ap = pages;
#pragma unroll
        for (int w = 0; w < PLAN_THREADS / 32; ++w) {
            if (w < warp) { bn += s_warp[0][w]; bp += s_warp[1][w]; }
            an += s_warp[0][w]; ap += s_warp[1][w];
        }
        bn += xn - sn; bp += xp - sp;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s_cu[tid * PER + i] = (int)min(bn, cap);
            s_first[tid * PER + i] = (int)min(bp, cap);
            s_len[tid * PER + i] = (int)len[i];
            bn += n[i]; bp += need[i];
        }
        if (tid == 0) s_cu[PLAN_CHUNK] = (int)min(an, cap);
        __syncthreads();
        // requests: their lengths, table entries and shares of the outputs, spread over the CTAs
        for (int r = blockIdx.x * PLAN_THREADS + tid; r < nb; r += gridDim.x * PLAN_THREADS) {
            const int b = b0 + r;
            const unsigned l = (unsigned)s_len[r], after = l + max(a.new_tokens[b], 0);
            const int have = (int)min(pages_of(l, page), width), want = (int)min(pages_of(after, page), width);
            const int first = s_first[r], got = min(max(a.n_free - first, 0), want - have);
            for (int j = have; j < want; ++j) a.table[(size_t)b * a.width + j] = j - have < got ? a.free_pages[first + j - have] : -1;
            a.lengths_out[b] = max((int)l, (int)min(min((long long)after, cap), (long long)(have + got) * a.page));
            a.cu_new[b] = s_cu[r];
        }
        // tokens of this CTA that belong to the chunk
        const int lo = (int)max(t0, (long long)s_cu[0]), hi = (int)min(t1, (long long)s_cu[nb == PLAN_CHUNK ? PLAN_CHUNK : nb]);
        for (int t = lo + tid; t < hi; t += PLAN_THREADS) {
            int x = 0, y = nb;                                // the last request of the chunk that starts at or before t
            while (x + 1 < y) {
                const int m = (x + y) >> 1;
                if (s_cu[m] <= t) x = m; else y = m;
            }
            const unsigned l = (unsigned)s_len[x], pos = l + (unsigned)(t - s_cu[x]), col = pos / page, have = min(pages_of(l, page), width);
            int p = -1;
            if (col < have) p = a.table[(size_t)(b0 + x) * a.width + col];        // (held before the call: nobody writes it)
            else if (col < width && s_first[x] + (long long)(col - have) < a.n_free) p = a.free_pages[s_first[x] + (col - have)];
            const long long slot = (long long)p * a.page + (pos - col * page);
            a.slots[t] = p >= 0 && slot <= cap ? (int)slot : -1;
            a.positions[t] = (int)min((long long)pos, cap);
        }
        if (blockIdx.x == 0)
            for (int r = tid; r < nb; r += PLAN_THREADS) {    // pages needed and not there
                const unsigned l = (unsigned)s_len[r];
                const long long held = pages_of(l, page), wanted = pages_of(l + max(a.new_tokens[b0 + r], 0), page);
                const long long have = min(held, (long long)a.width), want = min(wanted, (long long)a.width);
                missing += (wanted - held) - min(max((long long)a.n_free - s_first[r], 0ll), want - have);
            }
        tokens = an; pages = ap;
        __syncthreads();
    }
    for (long long t = max(t0, tokens) + tid; t < t1; t += PLAN_THREADS) a.slots[t] = a.positions[t] = -1;
    if (blockIdx.x == 0) {
        for (int d = 16; d; d >>= 1) missing += __shfl_xor_sync(0xffffffffu, missing, d);
        if (lane == 0) s_warp[0][warp] = missing;
        __syncthreads();
        if (tid == 0) {
            missing = 0;
            for (int w = 0; w < PLAN_THREADS / 32; ++w) missing += s_warp[0][w];
            a.cu_new[a.B] = (int)min(tokens, cap);
            a.taken[0] = (int)min(pages, (long long)a.n_free);
            a.taken[1] = (int)min(missing, cap);
        }
    }
}

// ---------------------------------------------------------------------------------------------- storing
constexpr int STORE_TOKENS = 4;                               // of a CTA: as many copies of a thread on their way

struct StoreArgs {
    const uint4 *k, *v;
    uint4 *kc, *vc;
    const int* slots;
    Rows rk, rv;                     // strides here in 16-byte chunks
    CacheRows rkc, rvc;
    int total, Hk, pages, page;
};

// A token's chunks of 16 bytes, K's rows and then V's, to consecutive threads; a thread has the same chunk of all tokens of its CTA. Bound by HBM,
// where there is enough: 16,384 tokens, 8 heads of 128: 134 MB in 18.3 us = 7.3 TB/s (what is written stays in L2 in part); 256 tokens: 4.3 us.
template <int D> __global__ void __launch_bounds__(256) store_kv_kernel(StoreArgs a) {
    constexpr int CH = D / 8;
    const int64_t t0 = (int64_t)blockIdx.x * STORE_TOKENS;
    int slot[STORE_TOKENS];
#pragma unroll
    for (int j = 0; j < STORE_TOKENS; ++j) slot[j] = t0 + j < a.total ? __ldg(a.slots + t0 + j) : -1;
    int64_t to_k[STORE_TOKENS], to_v[STORE_TOKENS];
#pragma unroll
    for (int j = 0; j < STORE_TOKENS; ++j) {
        const int page = slot[j] / a.page, at = slot[j] - page * a.page;
        if (slot[j] < 0 || page >= a.pages) slot[j] = -1;
        to_k[j] = page * a.rkc.page + at * a.rkc.token;
        to_v[j] = page * a.rvc.page + at * a.rvc.token;
    }
    for (int i = threadIdx.x; i < 2 * a.Hk * CH; i += 256) {
        const bool is_v = i >= a.Hk * CH;
        const int x = is_v ? i - a.Hk * CH : i, h = x / CH, c = x % CH;
        const uint4* src = (is_v ? a.v + h * a.rv.head : a.k + h * a.rk.head) + c;
        uint4* dst = (is_v ? a.vc + h * a.rvc.head : a.kc + h * a.rkc.head) + c;
        const int64_t step = is_v ? a.rv.token : a.rk.token;
        uint4 w[STORE_TOKENS];
#pragma unroll
        for (int j = 0; j < STORE_TOKENS; ++j)
            if (slot[j] >= 0) w[j] = __ldcs(src + (t0 + j) * step);
#pragma unroll
        for (int j = 0; j < STORE_TOKENS; ++j)
            if (slot[j] >= 0) dst[is_v ? to_v[j] : to_k[j]] = w[j];
    }
}

}  // namespace
}  // namespace packed
}  // namespace es

using namespace es;
using namespace es::packed;

extern "C" int es_extend_tables(const int32_t* lengths, const int32_t* new_tokens, int32_t* table, const int32_t* free_pages, int32_t n_free,
                                int32_t batch, int32_t table_width, int32_t page_size, int32_t total, int32_t* slots, int32_t* positions,
                                int32_t* cu_new, int32_t* lengths_out, int32_t* taken, void* stream) {
    if (n_free < 0 || batch < 0 || table_width < 0 || page_size < 1 || total < 0) return set_error(-1, "es_extend_tables: sizes out of range");
    if (!cu_new || !taken || (batch && (!lengths || !new_tokens || !lengths_out)) || (batch && table_width && !table) || (n_free && !free_pages) ||
        (total && (!slots || !positions)))
        return set_error(-1, "es_extend_tables: null pointer");
    if (!aligned(4, lengths, new_tokens, table, free_pages, slots, positions, cu_new, lengths_out, taken))
        return set_error(-1, "es_extend_tables: the int32 arrays must be 4-byte aligned");
    const PlanArgs a{lengths, new_tokens, free_pages, table, slots, positions, cu_new, lengths_out, taken, n_free, batch, table_width, page_size, total};
    const unsigned grid = (unsigned)std::max<int64_t>(1, ((int64_t)total + PLAN_TOKENS - 1) / PLAN_TOKENS);
    extend_tables_kernel<<<grid, PLAN_THREADS, 0, (cudaStream_t)stream>>>(a);
    ES_CHECK_LAUNCH("extend_tables_kernel");
    return 0;
}

extern "C" int es_store_kv(const void* k, const void* v, void* k_cache, void* v_cache, const int32_t* slots, int32_t total, int32_t kv_heads,
                           int32_t D, int32_t pages, int32_t page_size, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                           int64_t kc_page, int64_t kc_token, int64_t kc_head, int64_t vc_page, int64_t vc_token, int64_t vc_head, void* stream) {
    if (int rc = check_sizes("es_store_kv", 0, total, 0, kv_heads, kv_heads, D, 0)) return rc;
    if (pages < 0 || page_size < 1 || (int64_t)pages * page_size > 0x7FFFFFFF) return set_error(-1, "es_store_kv: sizes out of range");
    if (total == 0 || pages == 0) return 0;
    if (!k || !v || !k_cache || !v_cache || !slots) return set_error(-1, "es_store_kv: null pointer");
    if (!aligned(16, k, v, k_cache, v_cache) || !aligned(4, slots)) return set_error(-1, "es_store_kv: k, v, k_cache, v_cache must be 16-byte, slots 4-byte aligned");
    if (!whole_chunks(k_token, k_head, v_token, v_head, kc_page, kc_token, kc_head, vc_page, vc_token, vc_head))
        return set_error(-1, "es_store_kv: strides must be multiples of 8 elements");
    const StoreArgs a{(const uint4*)k, (const uint4*)v, (uint4*)k_cache, (uint4*)v_cache, slots, {k_token / 8, k_head / 8}, {v_token / 8, v_head / 8},
                      {kc_page / 8, kc_token / 8, kc_head / 8}, {vc_page / 8, vc_token / 8, vc_head / 8}, total, kv_heads, pages, page_size};
    const unsigned grid = (unsigned)(((int64_t)total + STORE_TOKENS - 1) / STORE_TOKENS);
    if (D == 64) store_kv_kernel<64><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
    else store_kv_kernel<128><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
    ES_CHECK_LAUNCH("store_kv_kernel");
    return 0;
}
