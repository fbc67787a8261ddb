// Attention over packed sequences: the C entry points (kernels: es_packed_fwd.cu, es_packed_bwd.cu), and the row sums of the backward.
//
//   S = scale Q K^T (visible keys: j <= i + nk - nq in causal attention), P = softmax(S), O = P V, LSE = log sum exp S
//   delta = rowsum(dO o O), dS = P o (dO V^T - delta), dQ = scale dS K, dK = scale sum over the group's heads of dS^T Q, dV = ... P^T dO
//
// delta is a difference's second half: with O rounded to bf16 it would be off by 2^-9 of |dO| |O|, which in short sequences is as much as all
// other roundings of dQ and dK together. The forward therefore also keeps what rounding O left (o_rest), and delta is summed from both.
#include "es_packed.cuh"

namespace es {
namespace packed {

int packed_fwd_tc(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, void* o, void* o_rest,
                  float* lse, const Batch& b, int D, int dtype, void* ws, cudaStream_t st);
long long packed_fwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D);
int packed_bwd_tc(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, const void* dout, Rows rdo, const float* lse, const float* delta, void* dq,
                  void* dk, void* dv, const Batch& b, int D, int dtype, void* ws, cudaStream_t st);
long long packed_bwd_workspace(int B, int Tq, int Tk, int H, int Hk, int D);

namespace {

// A thread per 16 bytes: bound by HBM, three reads of a row (32,768 tokens, 12 heads of 128: 44 us = 6.9 TB/s).
template <typename T, int D>
__global__ void __launch_bounds__(256) delta_kernel(const uint4* o, const uint4* o_rest, const T* dout, Rows rdo, float* delta, int Tq, int H) {
    constexpr int L = D / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / L;
    float s = 0.f;
    int t = 0, h = 0;
    launch_dependents();                                     // (the next kernel waits for all of this)
    if (row < (int64_t)Tq * H) {
        t = (int)(row / H);
        h = (int)(row % H);
        const uint4 x = o[i], y = *reinterpret_cast<const uint4*>(dout + t * rdo.token + h * rdo.head + 8 * (i % L));
        const uint4 r = o_rest ? o_rest[i] : make_uint4(0, 0, 0, 0);
        const uint32_t *xp = &x.x, *yp = &y.x, *rp = &r.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 a = unpack2<T>(xp[j]), b = unpack2<T>(yp[j]), c = unpack2<T>(rp[j]);
            s += (a.x + c.x) * b.x + (a.y + c.y) * b.y;
        }
    }
#pragma unroll
    for (int d = L / 2; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (row < (int64_t)Tq * H && i % L == 0) delta[(int64_t)h * Tq + t] = s;
}

// Calls f with a value of the element type and the head dim as a compile-time constant.
template <typename F> int with_type(int dtype, int D, F f) {
    if (dtype == 0) return D == 64 ? f(__nv_bfloat16{}, std::integral_constant<int, 64>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 128>{});
    return D == 64 ? f(__half{}, std::integral_constant<int, 64>{}) : f(__half{}, std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace packed
}  // namespace es

using namespace es;
using namespace es::packed;

extern "C" long long es_packed_fwd_workspace_bytes(int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D) {
    if (check_sizes("es_packed_fwd_workspace_bytes", batch, total_q, total_k, heads, kv_heads, D, 0)) return 0;
    return packed_fwd_workspace(batch, total_q, total_k, heads, kv_heads, D);
}

extern "C" int es_packed_attn_fwd(const void* q, const void* k, const void* v, void* o, void* o_rest, float* lse, const int32_t* cu_q, const int32_t* cu_k,
                                  int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D,
                                  int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                  float scale, int32_t causal, int32_t dtype, void* workspace, void* stream) {
    if (int rc = check_sizes("es_packed_attn_fwd", batch, total_q, total_k, heads, kv_heads, D, dtype)) return rc;
    if (int rc = check_scale("es_packed_attn_fwd", scale)) return rc;
    if (total_q == 0) return 0;
    if (!q || !o || !lse || !cu_q || !cu_k || (total_k && (!k || !v)) || (!workspace && packed_fwd_workspace(batch, total_q, total_k, heads, kv_heads, D)))
        return set_error(-1, "es_packed_attn_fwd: null pointer");
    if (!aligned(16, q, k, v) || !aligned(32, o, o_rest, workspace) || !aligned(4, lse, cu_q, cu_k))
        return set_error(-1, "es_packed_attn_fwd: q, k, v must be 16-byte, o, o_rest and the workspace 32-byte, lse, cu_q, cu_k 4-byte aligned");
    if (!whole_chunks(q_token, q_head, k_token, k_head, v_token, v_head)) return set_error(-1, "es_packed_attn_fwd: strides must be multiples of 8 elements");
    const Batch b{cu_q, cu_k, batch, total_q, total_k, heads, kv_heads, heads / kv_heads, scale, causal};
    return packed_fwd_tc(q, {q_token, q_head}, k, {k_token, k_head}, v, {v_token, v_head}, o, o_rest, lse, b, D, dtype, workspace, (cudaStream_t)stream);
}

// The workspace of the backward: delta, then what dK / dV shared out over several CTAs needs.
static long long delta_bytes(int total_q, int heads) { return ((long long)total_q * heads * 4 + 255) / 256 * 256; }

extern "C" long long es_packed_bwd_workspace_bytes(int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D) {
    if (check_sizes("es_packed_bwd_workspace_bytes", batch, total_q, total_k, heads, kv_heads, D, 0)) return 0;
    return delta_bytes(total_q, heads) + packed_bwd_workspace(batch, total_q, total_k, heads, kv_heads, D);
}

extern "C" int es_packed_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_rest, const void* dout, const float* lse, void* dq,
                                  void* dk, void* dv, const int32_t* cu_q, const int32_t* cu_k, int32_t batch, int32_t total_q, int32_t total_k,
                                  int32_t heads, int32_t kv_heads, int32_t D, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                                  int64_t v_token, int64_t v_head, int64_t do_token, int64_t do_head, float scale, int32_t causal, int32_t dtype,
                                  void* workspace, void* stream) {
    if (int rc = check_sizes("es_packed_attn_bwd", batch, total_q, total_k, heads, kv_heads, D, dtype)) return rc;
    if (int rc = check_scale("es_packed_attn_bwd", scale)) return rc;
    if (!total_q) dq = nullptr;
    if (!total_k) dk = dv = nullptr;
    if (!dq && !dk && !dv) return 0;
    if ((dk == nullptr) != (dv == nullptr)) return set_error(-1, "es_packed_attn_bwd: null pointer (dk and dv go together)");
    if (!cu_q || !cu_k || (total_q && (!q || !o || !dout || !lse || !workspace)) || (total_k && (!k || !v)) ||
        (!workspace && packed_bwd_workspace(batch, total_q, total_k, heads, kv_heads, D)))
        return set_error(-1, "es_packed_attn_bwd: null pointer");
    if (!aligned(16, q, k, v, o, o_rest, dout) || !aligned(32, dq, dk, dv, workspace) || !aligned(4, lse, cu_q, cu_k))
        return set_error(-1, "es_packed_attn_bwd: q, k, v, o, o_rest, dout must be 16-byte, dq, dk, dv and the workspace 32-byte, lse, cu_q, cu_k 4-byte aligned");
    if (!whole_chunks(q_token, q_head, k_token, k_head, v_token, v_head, do_token, do_head))
        return set_error(-1, "es_packed_attn_bwd: strides must be multiples of 8 elements");
    const cudaStream_t st = (cudaStream_t)stream;
    float* delta = static_cast<float*>(workspace);
    if (total_q) {
        const int rc = with_type(dtype, D, [&](auto t, auto d) {
            using T = decltype(t);
            const int64_t grid = ((int64_t)total_q * heads * (d / 8) + 255) / 256;
            if (grid > 0x7FFFFFFF) return set_error(-1, "es_packed_attn_bwd: too many rows");
            delta_kernel<T, d><<<(unsigned)grid, 256, 0, st>>>((const uint4*)o, (const uint4*)o_rest, (const T*)dout, {do_token, do_head}, delta, total_q, heads);
            ES_CHECK_LAUNCH("delta_kernel");
            return 0;
        });
        if (rc) return rc;
    }
    const Batch b{cu_q, cu_k, batch, total_q, total_k, heads, kv_heads, heads / kv_heads, scale, causal};
    return packed_bwd_tc(q, {q_token, q_head}, k, {k_token, k_head}, v, {v_token, v_head}, dout, {do_token, do_head}, lse, delta, dq, dk, dv, b, D, dtype,
                         static_cast<uint8_t*>(workspace) + delta_bytes(total_q, heads), st);
}
