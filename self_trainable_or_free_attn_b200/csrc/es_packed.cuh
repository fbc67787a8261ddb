// Pieces shared by the kernels for packed sequences and for a paged cache (es_packed.cu, es_cache.cu): sizes and strides of a
// packed batch, the sequence of a token, element conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "es_api_internal.h"
#include "es_ptx.cuh"

namespace es {
namespace packed {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A token and a head stride, in elements.
struct Rows {
    int64_t token, head;
};

// A page, a token and a head stride, in elements.
struct CacheRows {
    int64_t page, token, head;
};

// What the kernels of a packed batch have in common.
struct Batch {
    const int *cu_q, *cu_k;
    int B, Tq, Tk, H, Hk, G;         // G = H / Hk query heads to a key head
    float scale;
    int causal;
    // first token of sequence b, clamped: the values lie in device memory, and no wrong one may lead out of the tensors
    __device__ __forceinline__ int q_at(int b) const { return min(max(__ldg(cu_q + b), 0), Tq); }
    __device__ __forceinline__ int k_at(int b) const { return min(max(__ldg(cu_k + b), 0), Tk); }
};

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

inline int check_sizes(const char* name, int B, int Tq, int Tk, int H, int Hk, int D, int dtype) {
    const char* what = nullptr;
    if (B < 0 || Tq < 0 || Tk < 0 || Tq >= 0x7FFFFF00 || Tk >= 0x7FFFFF00) what = ": sizes out of range";
    else if (H < 1 || Hk < 1 || H % Hk) what = ": heads must be a multiple of kv_heads";
    else if (D != 64 && D != 128) what = ": D must be 64 or 128";
    else if (dtype != 0 && dtype != 1) what = ": dtype must be 0 (bf16) or 1 (fp16)";
    return what ? set_error(-1, (std::string(name) + what).c_str()) : 0;
}

// A factor of the logits: a normal number, as is its product with log2(e). (0 times the -inf of a masked logit is NaN, and so is infinity times 0.)
inline int check_scale(const char* name, float scale) {
    return scale >= 0x1p-126f && scale <= 0x1p126f ? 0 : set_error(-1, (std::string(name) + ": scale must be from 2^-126 to 2^126").c_str());
}

inline int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
    return n;
}

// Rounds of CTAs, from tiles per SM: whole ones where they are few, later ones fill up as the lengths differ.
inline double rounds(double x) { return x < 4 ? std::ceil(x) : x; }

template <typename... S> inline bool whole_chunks(S... s) { return (((uint64_t)s | ... | 0ull) & 7) == 0; }

}  // namespace packed
}  // namespace es
