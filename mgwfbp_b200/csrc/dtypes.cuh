// Element types of the language-model operators and vector accesses to them: values are held in fp32 inside the kernels
// and rounded (to nearest even) once when they are stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"
#include "lm_api.h"

#ifdef __CUDACC__

__device__ __forceinline__ float mgw_to_float(float x) { return x; }
__device__ __forceinline__ float mgw_to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float mgw_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T mgw_from_float(float x);
template <> __device__ __forceinline__ float mgw_from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half mgw_from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 mgw_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N values of type T that move as one access of N * sizeof(T) bytes (2, 4, 8 or 16)
template <int BYTES> struct MgwRaw;
template <> struct MgwRaw<16> { typedef uint4 type; };
template <> struct MgwRaw<8> { typedef uint2 type; };
template <> struct MgwRaw<4> { typedef uint32_t type; };
template <> struct MgwRaw<2> { typedef uint16_t type; };

template <typename T, int N>
union MgwVec {
    typename MgwRaw<N * sizeof(T)>::type raw;
    T v[N];
    __device__ __forceinline__ MgwVec() {}
};

// Two values at a time: one instruction converts a pair, single values take the slow conversion pipe.
__device__ __forceinline__ float2 mgw_to_float2(const __half* p) { return __half22float2(__halves2half2(p[0], p[1])); }
__device__ __forceinline__ float2 mgw_to_float2(const __nv_bfloat16* p) { return __bfloat1622float2(__halves2bfloat162(p[0], p[1])); }
__device__ __forceinline__ float2 mgw_to_float2(const float* p) { return make_float2(p[0], p[1]); }
__device__ __forceinline__ void mgw_from_float2(__half* p, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    p[0] = __low2half(h);
    p[1] = __high2half(h);
}
__device__ __forceinline__ void mgw_from_float2(__nv_bfloat16* p, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    p[0] = __low2bfloat16(h);
    p[1] = __high2bfloat16(h);
}
__device__ __forceinline__ void mgw_from_float2(float* p, float a, float b) { p[0] = a; p[1] = b; }

template <typename T, int N>
__device__ __forceinline__ void mgw_unpack(const typename MgwRaw<N * sizeof(T)>::type& raw, float (&f)[N]) {
    MgwVec<T, N> u;
    u.raw = raw;
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) {
        const float2 x = mgw_to_float2(u.v + i);
        f[i] = x.x;
        f[i + 1] = x.y;
    }
    if (N & 1) f[N - 1] = mgw_to_float(u.v[N - 1]);
}

template <typename T, int N>
__device__ __forceinline__ typename MgwRaw<N * sizeof(T)>::type mgw_pack(const float (&f)[N]) {
    MgwVec<T, N> u;
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) mgw_from_float2(u.v + i, f[i], f[i + 1]);
    if (N & 1) u.v[N - 1] = mgw_from_float<T>(f[N - 1]);
    return u.raw;
}

// Programmatic dependent launch: a kernel may be launched while the one before it still runs, and waits here for that
// one's end and results.  Without the launch attribute both do nothing.
__device__ __forceinline__ void mgw_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void mgw_let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float mgw_nan() { return __int_as_float(0x7fc00000); }

// The token with index i of an int32 (wide = 0) or int64 (wide = 1) list.
__device__ __forceinline__ long long mgw_token(const void* tokens, int wide, long long i) {
    return wide ? static_cast<const long long*>(tokens)[i] : (long long)static_cast<const int*>(tokens)[i];
}

// Record a token outside the vocabulary: {MGW_STATUS_BOUNDS, operator, position, token, cta}, the first one wins.
#define MGW_OP_EMBEDDING 1
#define MGW_OP_EMBEDDING_GRAD 2
#define MGW_OP_LOGPROB 3
__device__ __forceinline__ void mgw_report_token(int* status, int op, long long position, long long token) {
    const long long lo = -2147483647LL - 1, hi = 2147483647LL;
    mgw_report(status, MGW_STATUS_BOUNDS, op, (int)(position < hi ? position : hi),
               (int)(token < lo ? lo : token > hi ? hi : token));
}

#endif  // __CUDACC__
