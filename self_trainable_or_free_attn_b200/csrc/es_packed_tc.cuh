// Pieces shared by the tcgen05 kernels for packed sequences (es_packed_fwd.cu, es_packed_bwd.cu): the tiles of a packed batch, rows
// of (token, head) pairs, tensor maps, values that are not finite.
#pragma once
#include "es_packed.cuh"
#include "es_vsa_tc.cuh"

namespace es {
namespace packed {

using vsa::pack2;
using vsa::umma_idesc;
using vsa::kNaN16x2;
using vsa::kNaN32;

constexpr int TM = 128, TN = 128, THREADS = 384;
// Registers per thread: 168 at launch (three warps to a quarter of the SM), shared out anew: 224 + 224 + 56 = 3 * 168.
constexpr int REGS_MATH = 224, REGS_REST = 56;
constexpr int FEW = 32;                                      // keys of a row (see is_fine, es_packed_fwd.cu)
constexpr uint32_t HALF = TM * 128;                          // 128 rows x 64 d, one swizzled box

// A value that all lanes have, said so: what is computed from it stays in the registers of the whole warp, where the MMA instructions want their
// operands. (From values of the lanes' registers an MMA takes 55 to 70 clocks to issue, as long as it runs.)
template <typename V> __device__ __forceinline__ V uniform(V x) { return __shfl_sync(0xffffffffu, x, 0); }

// A span of consecutive tokens of one sequence (or of the tokens before the first or behind the last: seq = -1).
struct Piece {
    int seq, length;     // the sequence and its tokens
    int offset;          // of the span in it
    int first, n;        // first token of the batch, tokens (none where n <= 0)
};

// The span of grid slot x. The pieces of a batch are what lies before the first sequence, the sequences, and what lies behind the last. Up to 32 of
// them, a lane each, are taken longest first, so that the last slots are short ones, each from its last span to its first (LAST_FIRST) or from its
// first. (24 ragged prompts x 40 heads: the slowest SM 14 % over the mean in the order of the batch.) More of them stay in their order: piece i
// starts at slot floor(start / span) + i, which leaves each piece at least ceil(length / span) slots without a sum over the lengths, and a
// warp searches 32 pieces at a time. The slots are 0 .. floor(tokens / span) + B + 1.
template <bool LAST_FIRST> __device__ __forceinline__ Piece find_piece(const int* cu, int B, int tokens, int64_t slots, int64_t x, int span, int lane) {
    auto start = [&](int i) { return i == 0 ? 0 : i > B + 1 ? tokens : min(max(__ldg(cu + i - 1), 0), tokens); };
    Piece p;
    if (B + 2 <= 32) {
        const int s = lane < B + 2 ? start(lane) : tokens, e = lane < B + 2 ? start(lane + 1) : tokens;
        const int length = max(e - s, 0), mine = (length + span - 1) / span;
        int before = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int l = __shfl_sync(0xffffffffu, length, i), n = __shfl_sync(0xffffffffu, mine, i);
            if (l > length || (l == length && i < lane)) before += n;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, x >= before && x < before + mine);
        if (found == 0) return Piece{-1, 0, 0, 0, 0};
        const int i = __ffs(found) - 1, at = (int)x - __shfl_sync(0xffffffffu, before, i), n = __shfl_sync(0xffffffffu, mine, i);
        p.seq = i >= 1 && i <= B ? i - 1 : -1;
        p.length = __shfl_sync(0xffffffffu, length, i);
        p.offset = (LAST_FIRST ? n - 1 - at : at) * span;
        p.first = __shfl_sync(0xffffffffu, s, i) + p.offset;
        p.n = min(span, p.length - p.offset);
        return p;
    }
    const int y = (int)(LAST_FIRST ? slots - 1 - x : x);
    int lo = 0, n = B + 2;
    while (n > 1) {
        const int step = (n + 31) >> 5, i = lo + lane * step;
        const bool before = lane * step < n && start(i) / span + i <= y;
        const int c = max(__popc(__ballot_sync(0xffffffffu, before)), 1) - 1;
        n = min(step, n - c * step);
        lo += c * step;
    }
    const int s = start(lo), e = start(lo + 1);
    p.seq = lo >= 1 && lo <= B ? lo - 1 : -1;
    p.length = e - s;
    p.offset = (y - (s / span + lo)) * span;
    p.first = s + p.offset;
    p.n = min(span, e - s - p.offset);
    return p;
}
inline int64_t piece_slots(int tokens, int span, int B) { return tokens / span + B + 2; }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// 2^x for x <= 64 on the FMA pipes: 2^n times a polynomial of the rest f in [-1/2, 1/2], the degree-4 one whose largest relative error is
// smallest (2.6e-6, by the exchange of its extrema). Below -126 the result is 2^-126 instead of less; NaN stays NaN.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    constexpr float ROUND = 12582912.f;                      // 1.5 * 2^23: adding it leaves n in the low bits
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-126.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-126.f));
    const float2 t = __fadd2_rn(x, make_float2(ROUND, ROUND)), n = __fadd2_rn(t, make_float2(-ROUND, -ROUND));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 p = make_float2(0.009570102207362652f, 0.009570102207362652f);
    p = __ffma2_rn(p, f, make_float2(0.05591785907745361f, 0.05591785907745361f));
    p = __ffma2_rn(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
    p = __ffma2_rn(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
    p = __ffma2_rn(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
    return __fmul2_rn(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3F800000u), __uint_as_float((__float_as_uint(t.y) << 23) + 0x3F800000u)));
}

template <typename T> __device__ __forceinline__ bool not_finite(uint32_t w) {       // either of two packed values
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    return (w & E) == E || ((w >> 16) & E) == E;
}
template <typename T> __device__ __forceinline__ uint32_t finite_only(uint32_t w) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if (((w >> 16) & E) == E) w &= 0xFFFFu;
    return w;
}

// Row r of the tile at `tile` in shared memory, its values that are not finite set to 0; whether there were any. (0 times a value, summed: NaN
// if one of them is not finite, in one instruction for two values.)
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <> struct Pair<__half> { typedef __half2 type; };
template <typename T, int D> __device__ __forceinline__ bool clean_row(uint8_t* tile, int r) {
    typedef typename Pair<T>::type P;
    uint8_t* row = tile + r * 128;
    const uint32_t zero = 0;
    P acc[4] = {*reinterpret_cast<const P*>(&zero), *reinterpret_cast<const P*>(&zero), *reinterpret_cast<const P*>(&zero), *reinterpret_cast<const P*>(&zero)};
    const P z = acc[0];
#pragma unroll
    for (int d = 0; d < D / 64; ++d)
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
            const uint4 v = *reinterpret_cast<const uint4*>(row + d * HALF + 16 * (ch ^ (r & 7)));
            const uint32_t* w = &v.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = __hfma2(*reinterpret_cast<const P*>(w + j), z, acc[j]);
        }
    acc[0] = __hadd2(__hadd2(acc[0], acc[1]), __hadd2(acc[2], acc[3]));
    const float2 sum = unpack2<T>(*reinterpret_cast<const uint32_t*>(&acc[0]));
    if (sum.x == 0.f && sum.y == 0.f) return false;
    for (int d = 0; d < D / 64; ++d)
        for (int ch = 0; ch < 8; ++ch) {
            uint4* v = reinterpret_cast<uint4*>(row + d * HALF + 16 * ch);
            *v = make_uint4(finite_only<T>(v->x), finite_only<T>(v->y), finite_only<T>(v->z), finite_only<T>(v->w));
        }
    return true;
}

// 32 bytes at once: a row's sectors are written whole. dst is 32-byte aligned.
__device__ __forceinline__ void store8(void* dst, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int N> __device__ __forceinline__ void load_floats(const float* src, float* v) {
    if constexpr (N == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        const float2 x = *reinterpret_cast<const float2*>(src);
        v[0] = x.x; v[1] = x.y;
    }
}

// The wait of a warp for what may be a whole walk away (a tile's end, or the next tile of the grid that has work; either grows with the input), where
// those inside a walk are an iteration away. Its limit counts from the last time the CTA got on: moved[0] counts the tiles loaded, moved[1] the
// grid's tiles looked at.
__device__ __forceinline__ bool mbar_wait_moving(uint32_t bar, uint32_t parity, volatile uint32_t* moved, volatile int* abort_flag, int* status, int code) {
    bool there = mbar_test_wait(bar, parity) || mbar_try_wait(bar, parity);
    if (!there) {
        uint32_t polls = 0, late = 0, seen = moved[0] + moved[1];
        int64_t t0 = (int64_t)global_timer_ns();
        while (!(there = mbar_try_wait(bar, parity))) {
            if ((++polls & 63u) != 0) continue;
            if (*abort_flag) break;
            if (*reinterpret_cast<volatile int*>(status) != 0) {
                *abort_flag = 1;
                break;
            }
            const uint32_t now = moved[0] + moved[1];
            if (now != seen) {
                seen = now;
                t0 = (int64_t)global_timer_ns();
                late = 0;
                continue;
            }
            late = (int64_t)global_timer_ns() - t0 > (int64_t)kWaitLimitNs ? late + 1 : 0;       // (two in a row: see mbar_wait)
            if (late >= 2) {
                *abort_flag = 1;
                atomicCAS(status, 0, code + 1000 * (int)(blockIdx.x % 100000));
                break;
            }
        }
    }
    return __all_sync(0xffffffffu, there) != 0;
}

// After a wait has given up, whether an answer on its way to shared memory has come (100 us at most).
__device__ __forceinline__ bool mbar_wait_answer(uint32_t bar, uint32_t parity) {
    const uint64_t t_end = global_timer_ns() + 100000ull;
    bool there = mbar_try_wait(bar, parity);
    while (!there && global_timer_ns() < t_end) there = mbar_try_wait(bar, parity);
    return __all_sync(0xffffffffu, there) != 0;
}

// What rounding x and y to the type left of them, itself rounded: together 16 bits of mantissa in bf16.
template <typename T> __device__ __forceinline__ uint32_t rest2(float x, float y, uint32_t rounded) {
    const float2 r = unpack2<T>(rounded);
    return pack2<T>(x - r.x, y - r.y);
}

// Query heads that share a tile's rows: the most heads of a group (a divisor of it) that still fill 15 of 16 rows. More heads make the tile
// shorter in tokens; the rows lost are computed for nothing.
inline int rows_pack(int G) {
    for (int d = G < TM ? G : TM; d > 1; --d)
        if (G % d == 0 && TM / d * d >= TM - TM / 16) return d;
    return 1;
}

template <typename T> int make_rows_map(CUtensorMap* m, const void* ptr, int D, int heads, long long tokens, Rows r, int box_heads, int box_tokens) {
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
    cuuint64_t str[2] = {(cuuint64_t)r.head * 2, (cuuint64_t)r.token * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    cuuint32_t estr[3] = {1, 1, 1};
    return encode_tensor_map(m, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                             const_cast<void*>(ptr), dims, str, box, estr, CU_TENSOR_MAP_SWIZZLE_128B);
}

// A cache in pages [pages][page][heads][D] in boxes of up to `rows` tokens of one page.
template <typename T> int make_pages_map(CUtensorMap* m, const void* ptr, int D, int heads, int page, int pages, CacheRows r, int rows) {
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)page, (cuuint64_t)pages};
    cuuint64_t str[3] = {(cuuint64_t)r.head * 2, (cuuint64_t)r.token * 2, (cuuint64_t)r.page * 2};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)(page < rows ? page : rows), 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return encode_tensor_map(m, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                             const_cast<void*>(ptr), dims, str, box, estr, CU_TENSOR_MAP_SWIZZLE_128B);
}

// A running CTA takes the place of one of its grid that has not started (its index, or -1 where there is none left): CTAs are as many as
// fit, and what one sets up serves all the tiles it takes. One thread asks; after a refusal it must not ask again.
__device__ __forceinline__ void ask_next(uint32_t answer, uint32_t bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ int next_of(uint32_t answer) {
    uint32_t x, got;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t.reg .b32 y, z, w;\n\t"
        "ld.shared.b128 h, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "mov.b32 %0, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, h;\n\t"
        "selp.u32 %1, 1, 0, p;\n\t}"
        : "=r"(x), "=r"(got)
        : "r"(answer)
        : "memory");
    return got ? (int)x : -1;
}

// The loop of the warp that hands out tiles. What it hands out are `Work`s of a control block C, found by work_of(tile): n_tok <= 0 is nothing to do,
// or nothing more. DEALT: tiles blockIdx.x, + gridDim.x, ... of `tiles`. Else as ask_next gives them, each asked for when the last loads of the
// one before have been issued (`want`): its own follow before the ring of the loads is empty, and no CTA holds a tile that another could begin.
template <bool DEALT, typename C, typename F>
__device__ __forceinline__ void hand_out(C* ctl, F&& work_of, int64_t tiles, bool ok, int lane, volatile int* abort_flag, int* status, int code) {
    int64_t t = blockIdx.x;
    uint32_t asked = 0, looked = 0;
    for (int n = 0;;) {
        auto w = work_of(t);                                 // (t < 0: none)
        if (lane == 0) {
            ctl->held = w;
            ctl->moved[1] = ++looked;
        }
        if (t < 0 || w.n_tok > 0) {
            ok = ok && mbar_wait_moving(smem_u32(&ctl->wempty[n & 1]), ((n >> 1) & 1) ^ 1, ctl->moved, abort_flag, status, code);
            if (ok && lane == 0) {
                ctl->work[n & 1] = w;
                ctl->not_finite[n & 1] = 0;
                mbar_arrive(smem_u32(&ctl->wfull[n & 1]));
            }
            __syncwarp();
            if (t < 0) break;
            if (!DEALT) ok = ok && mbar_wait_moving(smem_u32(&ctl->want), n & 1, ctl->moved, abort_flag, status, code + 1);
            ++n;
        }
        if (!ok) break;
        if (DEALT) {
            t = t + gridDim.x < tiles ? t + gridDim.x : -1;
            continue;
        }
        if (lane == 0) ask_next(smem_u32(ctl->answer), smem_u32(&ctl->next));
        // (also where a wait gave up: what the answer takes from the grid nobody else will do)
        ok = mbar_wait_warp(smem_u32(&ctl->next), asked & 1, abort_flag, status, code + 2);
        t = ok || mbar_wait_answer(smem_u32(&ctl->next), asked & 1) ? next_of(smem_u32(ctl->answer)) : -1;
        ++asked;
        fence_proxy_async_smem();
        __syncwarp();
    }
}

}  // namespace packed
}  // namespace es
