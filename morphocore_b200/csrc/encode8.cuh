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

#include <type_traits>

#include "common.cuh"

namespace mc
{

constexpr int CODE_BLOCK = MC_CODE_BLOCK;

/// The type that elements of T are computed in, and that the scales of their blocks have.
template <typename T> struct WideOf { using type = float; };
template <> struct WideOf<double> { using type = double; };
template <typename T> using Wide = typename WideOf<T>::type;

/// One element of a parameter.
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(Wide<T> v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ double narrow<double>(double v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

/// Four elements of a lane, as they lie in memory; the widest loads are of 16 bytes. Half precision stays packed until it is widened: taking
/// the halves apart where they are loaded would make every conditional load wait for its data (encoding bfloat16 took 132 us where
/// float takes 84 on the same number of elements).
template <typename T> struct alignas(16) Quad
{
    T e[4];
};
struct alignas(8) PackedQuad
{
    uint32_t word[2];
};
template <> struct alignas(8) Quad<__half> : PackedQuad
{
};
template <> struct alignas(8) Quad<__nv_bfloat16> : PackedQuad
{
};

template <typename T> __device__ __forceinline__ void widen_quad(const Quad<T>& q, Wide<T> (&v)[4])
{
    if constexpr (std::is_same<T, __half>::value)
    {
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q.word[h]));
            v[2 * h] = f.x;
            v[2 * h + 1] = f.y;
        }
    }
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    {
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            v[2 * h] = __uint_as_float(q.word[h] << 16);
            v[2 * h + 1] = __uint_as_float(q.word[h] & 0xffff0000u);
        }
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = q.e[k];
}

/// Rounded to T, to nearest even.
template <typename T> __device__ __forceinline__ Quad<T> narrow_quad(const Wide<T> (&v)[4])
{
    Quad<T> q;
    if constexpr (std::is_same<T, __half>::value)
    {
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            const __half2 pair = __floats2half2_rn(v[2 * h], v[2 * h + 1]);
            q.word[h] = *reinterpret_cast<const uint32_t*>(&pair);
        }
    }
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    {
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            const __nv_bfloat162 pair = __floats2bfloat162_rn(v[2 * h], v[2 * h + 1]);
            q.word[h] = *reinterpret_cast<const uint32_t*>(&pair);
        }
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++) q.e[k] = v[k];
    return q;
}

/// Position within the block of a lane's first element; and of element k.
template <bool VEC> __device__ __forceinline__ int lane_at(int lane) { return VEC ? 4 * lane : lane; }
template <bool VEC, int LANES = 32> __device__ __forceinline__ int quad_at(int lane, int k) { return lane_at<VEC>(lane) + (VEC ? k : LANES * k); }

// The four functions below take the address of the lane's first element and how many elements of the block lie from there on: with
// VEC all four of a lane exist (left > 0) or none, otherwise element k does where 32 k < left. Where LANES lanes share a shorter block, they stand
// for the 32.

/// A lane's elements; zeros where there are none.
template <bool VEC, int LANES = 32, typename T> __device__ __forceinline__ Quad<T> load_quad(const T* src, int left)
{
    Quad<T> q{};
    if constexpr (VEC)
    {
        if (left > 0) q = *reinterpret_cast<const Quad<T>*>(src);
    }
    else if constexpr (sizeof(T) == 2)
    {
        uint32_t half[4];
#pragma unroll
        for (int k = 0; k < 4; k++) half[k] = LANES * k < left ? reinterpret_cast<const uint16_t*>(src)[LANES * k] : 0u;
#pragma unroll
        for (int h = 0; h < 2; h++) q.word[h] = half[2 * h] | half[2 * h + 1] << 16;
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++) q.e[k] = LANES * k < left ? src[LANES * k] : T(0);
    return q;
}

template <bool VEC, int LANES = 32, typename T> __device__ __forceinline__ void store_quad(T* dst, const Quad<T>& q, int left)
{
    if constexpr (VEC)
    {
        if (left > 0) *reinterpret_cast<Quad<T>*>(dst) = q;
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (LANES * k < left)
            {
                if constexpr (sizeof(T) == 2) reinterpret_cast<uint16_t*>(dst)[LANES * k] = static_cast<uint16_t>(q.word[k / 2] >> (16 * (k % 2)));
                else dst[LANES * k] = q.e[k];
            }
}

/// A lane's four codes, element k in byte k.
template <bool VEC, int LANES = 32> __device__ __forceinline__ uint32_t load_codes(const int8_t* src, int left)
{
    uint32_t q = 0;
    if constexpr (VEC)
    {
        if (left > 0) q = *reinterpret_cast<const uint32_t*>(src);
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (LANES * k < left) q |= static_cast<uint32_t>(static_cast<uint8_t>(src[LANES * k])) << (8 * k);
    return q;
}

template <bool VEC, int LANES = 32> __device__ __forceinline__ void store_codes(int8_t* dst, uint32_t codes, int left)
{
    if constexpr (VEC)
    {
        if (left > 0) *reinterpret_cast<uint32_t*>(dst) = codes;
    }
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (LANES * k < left) dst[LANES * k] = static_cast<int8_t>(codes >> (8 * k));
}

__device__ __forceinline__ uint32_t pack_bytes(const uint32_t (&q)[4])
{
    return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}

/// First statement of a branch that is hardly ever taken: keeps the compiler from computing both sides and selecting, which would cost
/// every element the instructions of the exception (encoding bfloat16 issued 19 instructions an element instead of 7).
__device__ __forceinline__ void rarely() { asm volatile(""); }

/// Code of a value without a number: -128 for NaN, -127 and 127 for the infinities.
template <typename W> __device__ __forceinline__ uint32_t code_of_nonfinite(W v) { return v != v ? 0x80u : (v > W(0) ? 0x7fu : 0x81u); }

/// Scale and 126 / m of a block whose largest finite magnitude is m.
__device__ __forceinline__ void block_scale(float m, float& scale, float& inverse)
{
    const bool none = m < 0x1p-100f;
    inverse = none ? 0.0f : __fdiv_rn(126.0f, m);
    scale = none ? 0.0f : m * (1.0f / 126.0f);
}

/// Codes of N blocks that the warp holds, four elements of each a lane (absent elements are zeros). Lane i < N returns the scale of
/// block i. Called by whole warps. The rounding is that of one fused multiply-add: x * (126 / m) + 1.5 * 2^23 has the whole number in
/// its low bits. The division, a dozen instructions that a warp would repeat for every block, is done once: lane i does that of
/// block i.
template <int N> __device__ __forceinline__ float encode_blocks(const float (&v)[N][4], uint32_t (&codes)[N], int lane)
{
    constexpr uint32_t INF = 0x7f800000u;
    uint32_t top[N], largest = 0, mine = 0;
#pragma unroll
    for (int i = 0; i < N; i++)
    {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) m = max(m, __float_as_uint(v[i][k]) & 0x7fffffffu);
        top[i] = __reduce_max_sync(0xffffffffu, m);
        largest = max(largest, top[i]);
    }
    const bool all_finite = largest < INF;
    if (!all_finite)
    {
        rarely();
#pragma unroll
        for (int i = 0; i < N; i++)
        {
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < 4; k++)
            {
                const uint32_t bits = __float_as_uint(v[i][k]) & 0x7fffffffu;
                m = bits < INF ? max(m, bits) : m;
            }
            top[i] = __reduce_max_sync(0xffffffffu, m);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) mine = lane == i ? top[i] : mine;
    float scale, inverse;
    block_scale(__uint_as_float(mine), scale, inverse);
#pragma unroll
    for (int i = 0; i < N; i++)
    {
        const float of_block = __shfl_sync(0xffffffffu, inverse, i);
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < 4; k++) q[k] = __float_as_uint(fmaf(v[i][k], of_block, 12582912.0f));
        if (!all_finite)
        {
            rarely();
#pragma unroll
            for (int k = 0; k < 4; k++) q[k] = (__float_as_uint(v[i][k]) & 0x7fffffffu) < INF ? q[k] : code_of_nonfinite(v[i][k]);
        }
        codes[i] = pack_bytes(q);
    }
    return scale;
}

template <int N> __device__ __forceinline__ double encode_blocks(const double (&v)[N][4], uint32_t (&codes)[N], int lane)
{
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < N; i++)
    {
        double m = 0.0;
#pragma unroll
        for (int k = 0; k < 4; k++) m = isfinite(v[i][k]) ? fmax(m, fabs(v[i][k])) : m;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, d));
        mine = lane == i ? m : mine;
    }
    const bool none = mine < 0x1p-900;
    const double inverse = none ? 0.0 : 126.0 / mine, scale = none ? 0.0 : mine * (1.0 / 126.0);
#pragma unroll
    for (int i = 0; i < N; i++)
    {
        const double of_block = __shfl_sync(0xffffffffu, inverse, i);
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            q[k] = isfinite(v[i][k]) ? static_cast<uint32_t>(__double2loint(fma(v[i][k], of_block, 6755399441055744.0))) : code_of_nonfinite(v[i][k]);
        codes[i] = pack_bytes(q);
    }
    return scale;
}

/// Code k of four as a number: its byte becomes the low mantissa byte of 2^23 + 128 + code.
__device__ __forceinline__ float code_value(uint32_t codes, int k)
{
    return __uint_as_float(__byte_perm(codes ^ 0x80808080u, 0x4B000000u, 0x7540u | static_cast<uint32_t>(k))) - 8388736.0f;
}

/// What a lane's four codes of a block with this scale stand for.
__device__ __forceinline__ void decode_quad(uint32_t codes, float scale, float (&v)[4])
{
    float q[4];
#pragma unroll
    for (int k = 0; k < 4; k++) q[k] = code_value(codes, k);
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = q[k] * scale;
    if (fmaxf(fmaxf(fabsf(q[0]), fabsf(q[1])), fmaxf(fabsf(q[2]), fabsf(q[3]))) > 126.0f)
    {
        rarely();
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (fabsf(q[k]) > 126.0f) v[k] = q[k] < -127.0f ? __uint_as_float(0x7fc00000u) : copysignf(__uint_as_float(0x7f800000u), q[k]);
    }
}
__device__ __forceinline__ void decode_quad(uint32_t codes, double scale, double (&v)[4])
{
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        const float q = code_value(codes, k);
        v[k] = static_cast<double>(q) * scale;
        if (fabsf(q) > 126.0f)
            v[k] = q < -127.0f ? __longlong_as_double(0x7ff8000000000000ll) : copysign(__longlong_as_double(0x7ff0000000000000ll), static_cast<double>(q));
    }
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
