// Device side of the 8-bit activations: a block of 128 elements in the registers of one warp, its codes and its scale.
//
// A warp holds a block as four elements per lane, either neighbours (VEC: lane l has elements 4 l .. 4 l + 3, one wide load) or
// 32 apart (l, l + 32, l + 64, l + 96: four coalesced loads of single elements, for rows that do not start on the boundary a
// wide load needs). The largest magnitude of a block is a maximum over bit patterns: those of non-negative floats are ordered
// like the numbers, infinities and NaN are above every finite one, so that one integer reduction over the warp finds both the
// scale and whether the block needs the codes of the non-finite values.
//
// Why whole numbers with one scale and not an 8-bit floating type: dilation and erosion pick a winner among sums x + w, so what
// matters is the absolute error within a neighbourhood. Half a step is m / 252 here; e4m3 with the same scale has a half step of
// m / 16 next to m, and no infinities, which is what a geodesic border or a dropped weight leaves in a feature map.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mc
{

constexpr int CODE_BLOCK = MC_CODE_BLOCK;

/// The type that elements of T are computed in, and that the scales of their blocks have.
template <typename T> struct WideOf { using type = float; };
template <> struct WideOf<double> { using type = double; };
template <typename T> using Wide = typename WideOf<T>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

/// Rounded to T, to nearest even.
template <typename T> __device__ __forceinline__ T narrow(Wide<T> v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ double narrow<double>(double v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

/// Four elements of a lane, as they lie in memory. The widest loads are of 16 bytes.
template <typename T> struct alignas(sizeof(T) == 8 ? 16 : 4 * sizeof(T)) Quad
{
    T e[4];
};

/// Position within the block of a lane's element k.
template <bool VEC> __device__ __forceinline__ int quad_at(int lane, int k) { return VEC ? 4 * lane + k : lane + 32 * k; }

/// A lane's elements of the block at `src`, of which `valid` exist (a multiple of four if VEC); zeros past them.
template <bool VEC, typename T> __device__ __forceinline__ Quad<T> load_quad(const T* src, int lane, int valid)
{
    Quad<T> q;
    if constexpr (VEC)
    {
        if (4 * lane < valid) q = *reinterpret_cast<const Quad<T>*>(src + 4 * lane);
        else
#pragma unroll
            for (int k = 0; k < 4; k++) q.e[k] = T(0.0f);
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++) q.e[k] = lane + 32 * k < valid ? src[lane + 32 * k] : T(0.0f);
    return q;
}

template <bool VEC, typename T> __device__ __forceinline__ void store_quad(T* dst, const Quad<T>& q, int lane, int valid)
{
    if constexpr (VEC)
    {
        if (4 * lane < valid) *reinterpret_cast<Quad<T>*>(dst + 4 * lane) = q;
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (lane + 32 * k < valid) dst[lane + 32 * k] = q.e[k];
}

/// A lane's four codes, element k in byte k.
template <bool VEC> __device__ __forceinline__ uint32_t load_codes(const int8_t* src, int lane, int valid)
{
    uint32_t q = 0;
    if constexpr (VEC)
    {
        if (4 * lane < valid) q = *reinterpret_cast<const uint32_t*>(src + 4 * lane);
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (lane + 32 * k < valid) q |= static_cast<uint32_t>(static_cast<uint8_t>(src[lane + 32 * k])) << (8 * k);
    return q;
}

template <bool VEC> __device__ __forceinline__ void store_codes(int8_t* dst, uint32_t codes, int lane, int valid)
{
    if constexpr (VEC)
    {
        if (4 * lane < valid) *reinterpret_cast<uint32_t*>(dst + 4 * lane) = codes;
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (lane + 32 * k < valid) dst[lane + 32 * k] = static_cast<int8_t>(codes >> (8 * k));
}

__device__ __forceinline__ uint32_t pack_bytes(const uint32_t (&q)[4])
{
    return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}

/// Code of a value without a number: -128 for NaN, -127 and 127 for the infinities.
template <typename W> __device__ __forceinline__ uint32_t code_of_nonfinite(W v) { return v != v ? 0x80u : (v > W(0) ? 0x7fu : 0x81u); }

/// Codes of the block that the warp holds (absent elements are zeros), and its scale, the same in every lane. Called by whole
/// warps. The rounding is that of one fused multiply-add: x * (126 / m) + 1.5 * 2^23 has the whole number in its low bits.
__device__ __forceinline__ uint32_t encode_quad(const float (&v)[4], float& scale)
{
    constexpr uint32_t INF = 0x7f800000u;
    uint32_t bits[4];
#pragma unroll
    for (int k = 0; k < 4; k++) bits[k] = __float_as_uint(v[k]) & 0x7fffffffu;
    uint32_t top = __reduce_max_sync(0xffffffffu, max(max(bits[0], bits[1]), max(bits[2], bits[3])));
    const bool all_finite = top < INF;
    if (!all_finite)
    {
        top = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) top = bits[k] < INF ? max(top, bits[k]) : top;
        top = __reduce_max_sync(0xffffffffu, top);
    }
    const float m = __uint_as_float(top);
    const bool none = m < 0x1p-100f;
    const float inverse = none ? 0.0f : __fdiv_rn(126.0f, m);
    scale = none ? 0.0f : m * (1.0f / 126.0f);
    uint32_t q[4];
#pragma unroll
    for (int k = 0; k < 4; k++) q[k] = __float_as_uint(fmaf(v[k], inverse, 12582912.0f));
    if (!all_finite)
#pragma unroll
        for (int k = 0; k < 4; k++) q[k] = bits[k] < INF ? q[k] : code_of_nonfinite(v[k]);
    return pack_bytes(q);
}

__device__ __forceinline__ uint32_t encode_quad(const double (&v)[4], double& scale)
{
    double m = 0.0;
#pragma unroll
    for (int k = 0; k < 4; k++) m = isfinite(v[k]) ? fmax(m, fabs(v[k])) : m;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, d));
    const bool none = m < 0x1p-900;
    const double inverse = none ? 0.0 : 126.0 / m;
    scale = none ? 0.0 : m * (1.0 / 126.0);
    uint32_t q[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
        q[k] = isfinite(v[k]) ? static_cast<uint32_t>(__double2loint(fma(v[k], inverse, 6755399441055744.0))) : code_of_nonfinite(v[k]);
    return pack_bytes(q);
}

/// Code k of four as a number: its byte becomes the low mantissa byte of 2^23 + 128 + code.
__device__ __forceinline__ float code_value(uint32_t codes, int k)
{
    return __uint_as_float(__byte_perm(codes ^ 0x80808080u, 0x4B000000u, 0x7540u | static_cast<uint32_t>(k))) - 8388736.0f;
}

/// What code k of a block with this scale stands for.
__device__ __forceinline__ float decode_code(uint32_t codes, int k, float scale)
{
    const float q = code_value(codes, k);
    if (fabsf(q) > 126.0f) return q < -127.0f ? __uint_as_float(0x7fc00000u) : copysignf(__uint_as_float(0x7f800000u), q);
    return q * scale;
}
__device__ __forceinline__ double decode_code(uint32_t codes, int k, double scale)
{
    const double q = code_value(codes, k);
    if (fabs(q) > 126.0) return q < -127.0 ? __longlong_as_double(0x7ff8000000000000ll) : copysign(__longlong_as_double(0x7ff0000000000000ll), q);
    return q * scale;
}

/// Calls f(T{}) for the type an mc_dtype names.
template <typename F> inline int dispatch_dtype(int32_t dtype, F f)
{
    switch (dtype)
    {
        case MC_F32: return f(float{});
        case MC_F64: return f(double{});
        case MC_F16: return f(__half{});
        default: return f(__nv_bfloat16{});
    }
}

/// Whether every pointer (NULL ones aside) may be read or written as whole quads of T, and every row of `length` too.
template <typename T> inline bool quads_fit(int64_t length, std::initializer_list<const void*> tensors, std::initializer_list<const void*> codes)
{
    if (length % 4 != 0) return false;
    for (const void* p : tensors)
        if (reinterpret_cast<uintptr_t>(p) % alignof(Quad<T>) != 0) return false;
    for (const void* p : codes)
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return false;
    return true;
}

inline int64_t code_blocks(int64_t length) { return (length + CODE_BLOCK - 1) / CODE_BLOCK; }

}  // namespace mc
