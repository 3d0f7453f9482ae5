// nl_frag.h -- MFMA fragments of the two element types, single-precision functions, wavefront sums, LDS-DMA and waits: what every kernel file
// of libnanollama_stack.so builds on (device functions only).
#pragma once
#include <hip/hip_runtime.h>

namespace nl {

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int OPT = 512;          // elements of one operand tile (16 rows x 32 columns)

template <typename T> struct Frag;
template <> struct Frag<bf16> { bf16x8 v; };
template <> struct Frag<float> { f32x4 a, b; };

__device__ __forceinline__ void frag_zero(Frag<bf16> &f) { f.v = bf16x8{}; }
__device__ __forceinline__ void frag_zero(Frag<float> &f) { f.a = f32x4{}; f.b = f32x4{}; }
__device__ __forceinline__ float frag_get(const Frag<bf16> &f, int j) { return (float)f.v[j]; }
__device__ __forceinline__ float frag_get(const Frag<float> &f, int j) { return j < 4 ? f.a[j & 3] : f.b[j & 3]; }
__device__ __forceinline__ void frag_set(Frag<bf16> &f, int j, float x) { f.v[j] = (bf16)x; }
__device__ __forceinline__ void frag_set(Frag<float> &f, int j, float x) { if (j < 4) f.a[j & 3] = x; else f.b[j & 3] = x; }

__device__ __forceinline__ f32x4 mma(const Frag<bf16> &A, const Frag<bf16> &B, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(A.v, B.v, c, 0, 0, 0);
}
// the K order inside a fragment is the same permutation on both sides: step j multiplies element j of every lane's run
__device__ __forceinline__ f32x4 mma(const Frag<float> &A, const Frag<float> &B, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(A.a[j], B.a[j], c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(A.b[j], B.b[j], c, 0, 0, 0);
    return c;
}

// index of element (row, k) of an operand with nks tiles per row group
__host__ __device__ inline long long op_index(int row, int k, int nks) {
    return (((long long)(row >> 4) * nks + (k >> 5)) * 64 + ((k & 31) >> 3) * 16 + (row & 15)) * 8 + (k & 7);
}
__device__ __forceinline__ void put(bf16 *p, float v) { *p = (bf16)v; }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put4(bf16 *p, f32x4 v) {
    bf16x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (bf16)v[i];
    *reinterpret_cast<bf16x4 *>(p) = o;
}
__device__ __forceinline__ void put4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }

// Single-precision functions on the hardware's v_exp_f32 / v_rcp_f32 / v_rsq_f32 (1 ulp each).  exp: the rounding of x log2(e) is
// carried as a correction, so the result stays within a few ulp for large |x| too; x finite.
__device__ __forceinline__ float exp_f32(float x) {
    constexpr float L = 1.44269504f, LLO = 1.92596299e-8f, LN2 = 0.693147181f;      // log2(e) = L + LLO
    const float t = x * L, r = fmaf(x, LLO, fmaf(x, L, -t)), e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * LN2, e);
}
__device__ __forceinline__ float rcp_f32(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float rsqrt_f32(float x) { return __builtin_amdgcn_rsqf(x); }
// (past 88.72 the exponential is no float32; v_rcp_f32 leaves 0 below 2^-126, from 87.3 on)
__device__ __forceinline__ float sigmoid_f32(float z) { return rcp_f32(1.f + exp_f32(__builtin_amdgcn_fmed3f(-z, -88.72f, 88.72f))); }
__device__ __forceinline__ float silu_f32(float z) { return z * sigmoid_f32(z); }
__device__ __forceinline__ float gelu_arg(float z) { return z * fmaf(0.071354816f, z * z, 1.5957691216057308f); }
__device__ __forceinline__ float gelu_tanh_f32(float z) {
    // 0.5 (1 + tanh u) = sigmoid(2 u)
    return z * sigmoid_f32(gelu_arg(z));
}
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
// sum over the wavefront, in every lane: rows of 16 lanes by DPP (neighbours, pairs, mirrored halves, mirrored row), then the four rows
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add<0x140>(dpp_add<0x141>(dpp_add<0x4E>(dpp_add<0xB1>(v))));
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}

// 16 bytes per lane straight into LDS: lane i lands at lds_base + 16 i (lds_base wave-uniform)
__device__ __forceinline__ void lds_dma16(const void *src_lane, void *lds_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src_lane,
                                     (__attribute__((address_space(3))) void *)lds_base, 16, 0, 0);
}
// 4 bytes per lane
__device__ __forceinline__ void lds_dma4(const void *src_lane, void *lds_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src_lane,
                                     (__attribute__((address_space(3))) void *)lds_base, 4, 0, 0);
}
// until at most N of this wavefront's vector memory operations are in flight (they complete in order)
template <int N> __device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Workgroup barrier for data that passes through LDS only.  __syncthreads() also waits for every global load and store the wavefront
// has in flight, i.e. for exactly the prefetches that are meant to run past it.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace nl
