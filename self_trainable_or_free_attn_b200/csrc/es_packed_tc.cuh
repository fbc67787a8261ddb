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
constexpr uint32_t HALF = TM * 128;                          // 128 rows x 64 d, one swizzled box

// A span of consecutive tokens of one sequence (or of the tokens before the first or behind the last: seq = -1).
struct Piece {
    int seq, length;     // the sequence and its tokens
    int offset;          // of the span in it
    int first, n;        // first token of the batch, tokens (none where n <= 0)
};

// The span of grid slot x: pieces of the batch are what lies before the first sequence, the sequences, and what lies behind the last; piece
// i starts at slot floor(start / span) + i, which leaves each piece at least ceil(length / span) slots without a sum over the lengths.
// The slots are 0 .. floor(tokens / span) + B + 1. A warp searches 32 pieces at a time.
__device__ __forceinline__ Piece find_piece(const int* cu, int B, int tokens, int x, int span, int lane) {
    auto start = [&](int i) { return i == 0 ? 0 : min(max(__ldg(cu + i - 1), 0), tokens); };
    int lo = 0, n = B + 2;
    while (n > 1) {
        const int step = (n + 31) >> 5, i = lo + lane * step;
        const bool before = lane * step < n && start(i) / span + i <= x;
        const int c = max(__popc(__ballot_sync(0xffffffffu, before)), 1) - 1;
        n = min(step, n - c * step);
        lo += c * step;
    }
    const int s = start(lo), e = lo + 1 < B + 2 ? start(lo + 1) : tokens;
    Piece p;
    p.seq = lo >= 1 && lo <= B ? lo - 1 : -1;
    p.length = e - s;
    p.offset = (x - (s / span + lo)) * span;
    p.first = s + p.offset;
    p.n = min(span, e - s - p.offset);
    return p;
}
inline int64_t piece_slots(int tokens, int span, int B) { return tokens / span + B + 2; }

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

}  // namespace packed
}  // namespace es
