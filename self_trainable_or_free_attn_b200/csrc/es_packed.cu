// Attention over packed sequences: the C entry points, and the kernels.
//
//   S = scale Q K^T (visible keys: j <= i + nk - nq in causal attention), P = softmax(S), O = P V, LSE = log sum exp S
//   delta = rowsum(dO o O), dS = P o (dO V^T - delta), dQ = scale dS K, dK = scale sum over the group's heads of dS^T Q, dV = ... P^T dO
//
// A warp per row: 32 keys at a time, a lane per key for the scores, then a lane per D / 32 columns for the products with P.
#include "es_packed.cuh"

namespace es {
namespace packed {

int packed_fwd_tc(const void* q, Rows rq, const void* k, Rows rk, const void* v, Rows rv, void* o, float* lse, const Batch& b, int D, int dtype, void* ws,
                  cudaStream_t st);

namespace {

template <typename T, int D> __device__ __forceinline__ float dot_row(const float* a, const T* b) {
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; c += 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(b + c);
        const float2 x0 = unpack2<T>(w.x), x1 = unpack2<T>(w.y), x2 = unpack2<T>(w.z), x3 = unpack2<T>(w.w);
        s += a[c] * x0.x + a[c + 1] * x0.y + a[c + 2] * x1.x + a[c + 3] * x1.y + a[c + 4] * x2.x + a[c + 5] * x2.y + a[c + 6] * x3.x + a[c + 7] * x3.y;
    }
    return s;
}

__device__ __forceinline__ float warp_sum(float x) {
    for (int i = 16; i; i >>= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
    return x;
}

constexpr int WARPS = 8;

template <typename T, int D> __global__ void __launch_bounds__(256) delta_kernel(const T* o, const T* dout, Rows rdo, float* delta, int Tq, int H) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * WARPS + warp;
    if (row >= (int64_t)Tq * H) return;
    const int t = (int)(row / H), h = (int)(row % H);
    float s = 0.f;
    for (int c = lane; c < D; c += 32) s += to_float(o[row * D + c]) * to_float(dout[t * rdo.token + h * rdo.head + c]);
    s = warp_sum(s);
    if (lane == 0) delta[(int64_t)h * Tq + t] = s;
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * WARPS) bwd_q_rows_kernel(const T* q, Rows rq, const T* k, Rows rk, const T* v, Rows rv, const T* dout, Rows rdo,
                                                                const float* lse, const float* delta, T* dq, Batch b) {
    constexpr int C = D / 32;
    __shared__ float rows[WARPS][2][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * WARPS + warp;
    if (row >= (int64_t)b.Tq * b.H) return;
    const int t = (int)(row / b.H), h = (int)(row % b.H), hk = h / b.G;
    const int s = sequence_of(b.cu_q, b.B, t);
    int n = 0, k0 = 0;
    if (s >= 0) {
        const int q0 = b.q_at(s), nq = b.q_at(s + 1) - q0, nk = max(b.k_at(s + 1) - b.k_at(s), 0);
        k0 = b.k_at(s);
        n = b.causal ? min(max(t - q0 + 1 + nk - nq, 0), nk) : nk;
    }
    for (int c = lane; c < D; c += 32) {
        rows[warp][0][c] = to_float(q[t * rq.token + h * rq.head + c]);
        rows[warp][1][c] = to_float(dout[t * rdo.token + h * rdo.head + c]);
    }
    __syncwarp();
    const float z = lse[(int64_t)h * b.Tq + t] * kLog2e, d = delta[(int64_t)h * b.Tq + t];
    float acc[C] = {};
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        float ds = 0.f;
        if (j < n) {
            const float x = dot_row<T, D>(rows[warp][0], k + (int64_t)(k0 + j) * rk.token + hk * rk.head) * (b.scale * kLog2e);
            ds = exp2f(x - z) * (dot_row<T, D>(rows[warp][1], v + (int64_t)(k0 + j) * rv.token + hk * rv.head) - d);
        }
        for (int jj = 0; jj < min(32, n - j0); ++jj) {
            const float w = __shfl_sync(0xffffffffu, ds, jj);
            const T* kr = k + (int64_t)(k0 + j0 + jj) * rk.token + hk * rk.head;
            for (int i = 0; i < C; ++i) acc[i] += w * to_float(kr[lane + 32 * i]);
        }
    }
    for (int i = 0; i < C; ++i) dq[((int64_t)t * b.H + h) * D + lane + 32 * i] = from_float<T>(acc[i] * b.scale);
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * WARPS) bwd_kv_rows_kernel(const T* q, Rows rq, const T* k, Rows rk, const T* v, Rows rv, const T* dout, Rows rdo,
                                                                 const float* lse, const float* delta, T* dk, T* dv, Batch b) {
    constexpr int C = D / 32;
    __shared__ float rows[WARPS][2][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * WARPS + warp;
    if (row >= (int64_t)b.Tk * b.Hk) return;
    const int t = (int)(row / b.Hk), hk = (int)(row % b.Hk);
    const int s = sequence_of(b.cu_k, b.B, t);
    int q0 = 0, nq = 0, first = 0;
    if (s >= 0) {
        const int k0 = b.k_at(s), nk = b.k_at(s + 1) - k0;
        q0 = b.q_at(s);
        nq = max(b.q_at(s + 1) - q0, 0);
        first = b.causal ? max(t - k0 - (nk - nq), 0) : 0;   // the first query that sees this key
    }
    for (int c = lane; c < D; c += 32) {
        rows[warp][0][c] = to_float(k[t * rk.token + hk * rk.head + c]);
        rows[warp][1][c] = to_float(v[t * rv.token + hk * rv.head + c]);
    }
    __syncwarp();
    float ak[C] = {}, av[C] = {};
    for (int h = hk * b.G; h < (hk + 1) * b.G; ++h)
        for (int i0 = first; i0 < nq; i0 += 32) {
            const int i = i0 + lane;
            float p = 0.f, ds = 0.f;
            if (i < nq) {
                const int64_t tq = q0 + i;
                const float x = dot_row<T, D>(rows[warp][0], q + tq * rq.token + h * rq.head) * (b.scale * kLog2e);
                p = exp2f(x - lse[(int64_t)h * b.Tq + tq] * kLog2e);
                ds = p * (dot_row<T, D>(rows[warp][1], dout + tq * rdo.token + h * rdo.head) - delta[(int64_t)h * b.Tq + tq]);
            }
            for (int ii = 0; ii < min(32, nq - i0); ++ii) {
                const float wp = __shfl_sync(0xffffffffu, p, ii), wd = __shfl_sync(0xffffffffu, ds, ii);
                const int64_t tq = q0 + i0 + ii;
                for (int c = 0; c < C; ++c) {
                    ak[c] += wd * to_float(q[tq * rq.token + h * rq.head + lane + 32 * c]);
                    av[c] += wp * to_float(dout[tq * rdo.token + h * rdo.head + lane + 32 * c]);
                }
            }
        }
    for (int c = 0; c < C; ++c) {
        dk[row * D + lane + 32 * c] = from_float<T>(ak[c] * b.scale);
        dv[row * D + lane + 32 * c] = from_float<T>(av[c]);
    }
}

// Calls f with a value of the element type and the head dim as a compile-time constant.
template <typename F> int with_type(int dtype, int D, F f) {
    if (dtype == 0) return D == 64 ? f(__nv_bfloat16{}, std::integral_constant<int, 64>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 128>{});
    return D == 64 ? f(__half{}, std::integral_constant<int, 64>{}) : f(__half{}, std::integral_constant<int, 128>{});
}
unsigned blocks(int64_t rows) { return (unsigned)((rows + WARPS - 1) / WARPS); }

}  // namespace
}  // namespace packed
}  // namespace es

using namespace es;
using namespace es::packed;

extern "C" long long es_packed_workspace_bytes(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

extern "C" int es_packed_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* cu_q, const int32_t* cu_k,
                                  int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t kv_heads, int32_t D,
                                  int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                  float scale, int32_t causal, int32_t dtype, void* workspace, void* stream) {
    if (int rc = check_sizes("es_packed_attn_fwd", batch, total_q, total_k, heads, kv_heads, D, dtype)) return rc;
    if (total_q == 0) return 0;
    if (!q || !o || !lse || !cu_q || !cu_k || (total_k && (!k || !v))) return set_error(-1, "es_packed_attn_fwd: null pointer");
    if (!aligned(16, q, k, v, o)) return set_error(-1, "es_packed_attn_fwd: q, k, v, o must be 16-byte aligned");
    if (!whole_chunks(q_token, q_head, k_token, k_head, v_token, v_head)) return set_error(-1, "es_packed_attn_fwd: strides must be multiples of 8 elements");
    const Batch b{cu_q, cu_k, batch, total_q, total_k, heads, kv_heads, heads / kv_heads, scale, causal};
    return packed_fwd_tc(q, {q_token, q_head}, k, {k_token, k_head}, v, {v_token, v_head}, o, lse, b, D, dtype, workspace, (cudaStream_t)stream);
}

extern "C" int es_packed_delta(const void* o, const void* dout, float* delta, int32_t total_q, int32_t heads, int32_t D, int64_t do_token,
                               int64_t do_head, int32_t dtype, void* stream) {
    if (int rc = check_sizes("es_packed_delta", 0, total_q, 0, heads, heads, D, dtype)) return rc;
    if (total_q == 0) return 0;
    if (!o || !dout || !delta) return set_error(-1, "es_packed_delta: null pointer");
    if (!aligned(16, o, dout)) return set_error(-1, "es_packed_delta: o and dout must be 16-byte aligned");
    if (!whole_chunks(do_token, do_head)) return set_error(-1, "es_packed_delta: strides must be multiples of 8 elements");
    return with_type(dtype, D, [&](auto t, auto d) {
        using T = decltype(t);
        delta_kernel<T, d><<<blocks((int64_t)total_q * heads), 32 * WARPS, 0, (cudaStream_t)stream>>>((const T*)o, (const T*)dout, {do_token, do_head}, delta,
                                                                                                      total_q, heads);
        ES_CHECK_LAUNCH("delta_kernel");
        return 0;
    });
}

extern "C" int es_packed_attn_bwd_q(const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* delta, void* dq,
                                    const int32_t* cu_q, const int32_t* cu_k, int32_t batch, int32_t total_q, int32_t total_k, int32_t heads,
                                    int32_t kv_heads, int32_t D, int64_t q_token, int64_t q_head, int64_t k_token, int64_t k_head,
                                    int64_t v_token, int64_t v_head, int64_t do_token, int64_t do_head, float scale, int32_t causal,
                                    int32_t dtype, void* stream) {
    if (int rc = check_sizes("es_packed_attn_bwd_q", batch, total_q, total_k, heads, kv_heads, D, dtype)) return rc;
    if (total_q == 0) return 0;
    if (!q || !dout || !lse || !delta || !dq || !cu_q || !cu_k || (total_k && (!k || !v))) return set_error(-1, "es_packed_attn_bwd_q: null pointer");
    if (!aligned(16, q, k, v, dout, dq)) return set_error(-1, "es_packed_attn_bwd_q: q, k, v, dout, dq must be 16-byte aligned");
    if (!whole_chunks(q_token, q_head, k_token, k_head, v_token, v_head, do_token, do_head))
        return set_error(-1, "es_packed_attn_bwd_q: strides must be multiples of 8 elements");
    const Batch b{cu_q, cu_k, batch, total_q, total_k, heads, kv_heads, heads / kv_heads, scale, causal};
    return with_type(dtype, D, [&](auto t, auto d) {
        using T = decltype(t);
        bwd_q_rows_kernel<T, d><<<blocks((int64_t)total_q * heads), 32 * WARPS, 0, (cudaStream_t)stream>>>(
            (const T*)q, {q_token, q_head}, (const T*)k, {k_token, k_head}, (const T*)v, {v_token, v_head}, (const T*)dout, {do_token, do_head}, lse, delta,
            (T*)dq, b);
        ES_CHECK_LAUNCH("bwd_q_rows_kernel");
        return 0;
    });
}

extern "C" int es_packed_attn_bwd_kv(const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* delta, void* dk,
                                     void* dv, const int32_t* cu_q, const int32_t* cu_k, int32_t batch, int32_t total_q, int32_t total_k,
                                     int32_t heads, int32_t kv_heads, int32_t D, int64_t q_token, int64_t q_head, int64_t k_token,
                                     int64_t k_head, int64_t v_token, int64_t v_head, int64_t do_token, int64_t do_head, float scale,
                                     int32_t causal, int32_t dtype, void* stream) {
    if (int rc = check_sizes("es_packed_attn_bwd_kv", batch, total_q, total_k, heads, kv_heads, D, dtype)) return rc;
    if (total_k == 0) return 0;
    if (!k || !v || !dk || !dv || !cu_q || !cu_k || (total_q && (!q || !dout || !lse || !delta))) return set_error(-1, "es_packed_attn_bwd_kv: null pointer");
    if (!aligned(16, q, k, v, dout, dk, dv)) return set_error(-1, "es_packed_attn_bwd_kv: q, k, v, dout, dk, dv must be 16-byte aligned");
    if (!whole_chunks(q_token, q_head, k_token, k_head, v_token, v_head, do_token, do_head))
        return set_error(-1, "es_packed_attn_bwd_kv: strides must be multiples of 8 elements");
    const Batch b{cu_q, cu_k, batch, total_q, total_k, heads, kv_heads, heads / kv_heads, scale, causal};
    return with_type(dtype, D, [&](auto t, auto d) {
        using T = decltype(t);
        bwd_kv_rows_kernel<T, d><<<blocks((int64_t)total_k * kv_heads), 32 * WARPS, 0, (cudaStream_t)stream>>>(
            (const T*)q, {q_token, q_head}, (const T*)k, {k_token, k_head}, (const T*)v, {v_token, v_head}, (const T*)dout, {do_token, do_head}, lse, delta,
            (T*)dk, (T*)dv, b);
        ES_CHECK_LAUNCH("bwd_kv_rows_kernel");
        return 0;
    });
}
