// Root-mean-square norm over the channels, forward and backward, with the residual's addition and the 8-bit forms of its result
// and of its input.
//
//     s = T(x + residual),  r = 1 / sqrt(mean_c s^2 + eps),  y = T(s r weight_c)
//     gx = r (u - s r^2 mean_c(u s)) + gsum,  u = gy weight_c;   gweight_c = sum over the pixels of gy s r
//
// Every kernel reads its inputs once: the tile of a thread block, all channels of 128 neighbouring pixels (columns) or whole
// rows of channels (rows), stays in registers between the sums over the channels and what is computed from them. Bytes bound
// them: a forward pass with residual moves 16 bytes an element in float (13 with the result in 8 bits), a backward pass 16 (13).
//
// The sums over the channels are taken in double and y is rounded once, from an unevaluated sum of two floats that carries about
// 46 bits: y, and with it every code of its 8-bit form, is then what 64-bit arithmetic gives, whichever kernel computed it and in
// whatever order (a float that is one unit off moves one code in 10^5 to its neighbour). A conversion to double and a fused
// multiply-add an element are a third of what their units do while the bytes of the element pass.
#pragma once
#include "encode8.cuh"

namespace mc
{

struct NormArgs
{
    const void *x, *residual, *weight;
    void *sum, *y, *y_scales, *sum_scales;
    int8_t *y_codes, *sum_codes;
    int64_t outer, channels, inner;
    int64_t tiles_per_row, tiles;   // blocks of 128 pixels in an image and in all (columns), of 128 channels in a row (rows)
    double eps;
};

struct NormGradArgs
{
    const void *sum, *sum_scales, *weight, *gy, *gsum;
    const int8_t* sum_codes;
    void *gx, *gweight;
    void* partial;                  // [grid, channels], Wide<T>
    int64_t outer, channels, inner;
    int64_t tiles_per_row, tiles;
    double eps;
};

/// s r g in the type that T is computed in, rounded once (see above). `fast`: every r of the warp lies within 2^-60 .. 2^60, so that
/// its two halves are ordinary floats and an infinite s cannot meet them (its r is 0).
__device__ __forceinline__ float scaled_value(float s, double r, float g, bool fast)
{
    if (!fast) return static_cast<float>(static_cast<double>(s) * r * static_cast<double>(g));
    const float high = static_cast<float>(r), low = static_cast<float>(r - static_cast<double>(high));
    const float p = s * high, p_low = fmaf(s, low, fmaf(s, high, -p));
    const float y = p * g;
    return fabsf(y) <= Limits<float>::max() ? y + fmaf(p_low, g, fmaf(p, g, -y)) : y;   // an infinite product has no remainder
}
__device__ __forceinline__ double scaled_value(double s, double r, double g, bool) { return s * r * g; }

__device__ __forceinline__ bool ordinary(double r) { return r > 0x1p-60 && r < 0x1p60; }

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

/// x + residual, rounded to T.
template <typename T> __device__ __forceinline__ Quad<T> add_quads(const Quad<T>& a, const Quad<T>& b)
{
    Quad<T> s;
#pragma unroll
    for (int k = 0; k < 4; k++) s.e[k] = narrow<T>(widen(a.e[k]) + widen(b.e[k]));
    return s;
}

template <typename T> __device__ __forceinline__ void widen_quad(const Quad<T>& q, Wide<T> (&v)[4])
{
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = widen(q.e[k]);
}

/// Writes the codes and the scale of a block held as a quad.
template <bool VEC, typename T>
__device__ __forceinline__ void put_codes(int8_t* codes, void* scales, int64_t at, int64_t block, const Quad<T>& q, int lane, int valid)
{
    Wide<T> v[4], scale;
    widen_quad(q, v);
    const uint32_t c = encode_quad(v, scale);
    store_codes<VEC>(codes + at, c, lane, valid);
    if (lane == 0) static_cast<Wide<T>*>(scales)[block] = scale;
}

/// Writes y, and its codes, of a block of s. `r` holds the factor of each of the lane's elements, `g` their weights.
template <bool VEC, typename T>
__device__ __forceinline__ void put_result(const NormArgs& a, const Quad<T>& s, const double (&r)[4], const Wide<T> (&g)[4], bool fast, int64_t at,
                                           int64_t block, int lane, int valid)
{
    Quad<T> y;
#pragma unroll
    for (int k = 0; k < 4; k++) y.e[k] = narrow<T>(scaled_value(widen(s.e[k]), r[k], g[k], fast));
    if (a.y != nullptr) store_quad<VEC>(static_cast<T*>(a.y) + at, y, lane, valid);
    if (a.y_codes != nullptr) put_codes<VEC>(a.y_codes, a.y_scales, at, block, y, lane, valid);
}

/// s of a block: x, or x + residual, which is stored.
template <bool VEC, typename T> __device__ __forceinline__ Quad<T> take_sum(const NormArgs& a, int64_t at, int lane, int valid)
{
    const Quad<T> x = load_quad<VEC>(static_cast<const T*>(a.x) + at, lane, valid);
    if (a.residual == nullptr) return x;
    return add_quads(x, load_quad<VEC>(static_cast<const T*>(a.residual) + at, lane, valid));
}

/// Elements of block j of a row of C (negative or zero past its end; the loads take that as none).
__device__ __forceinline__ int present(int j, int C) { return min(CODE_BLOCK, C - j * CODE_BLOCK); }

/// Forward, feature maps. A block of WARPS warps takes 128 pixels of an image; warp w has the channels w, w + WARPS, ... and keeps
/// up to HELD of them. Where there are more, the second pass reads s again, from `sum` or x: the tiles that are at work then
/// lie in L2 (128 pixels of 512 channels in float are 256 KiB, of 296 thread blocks 76 MiB).
template <typename T, bool VEC, int HELD, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) rms_norm_columns_kernel(const NormArgs a)
{
    static_assert(WARPS >= 4, "a thread for every pixel of the tile");
    __shared__ double part[WARPS][CODE_BLOCK];
    __shared__ double factor[CODE_BLOCK];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t C = a.channels;
    const bool held = C <= HELD * WARPS;
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const int64_t image = tile / a.tiles_per_row, piece = tile - image * a.tiles_per_row;
        const int valid = static_cast<int>(min(static_cast<int64_t>(CODE_BLOCK), a.inner - piece * CODE_BLOCK));
        const int64_t first = image * C * a.inner + piece * CODE_BLOCK, first_block = image * C * a.tiles_per_row + piece;
        Quad<T> s[HELD];
        double sums[4] = {};
        for (int64_t c0 = warp; c0 < C; c0 += HELD * WARPS)
        {
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                const int64_t c = c0 + i * WARPS;
                s[i] = take_sum<VEC, T>(a, first + c * a.inner, lane, c < C ? valid : 0);
            }
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                const int64_t c = c0 + i * WARPS;
#pragma unroll
                for (int k = 0; k < 4; k++) sums[k] = fma(static_cast<double>(widen(s[i].e[k])), static_cast<double>(widen(s[i].e[k])), sums[k]);
                if (c >= C) continue;
                const int64_t at = first + c * a.inner;
                if (a.residual != nullptr) store_quad<VEC>(static_cast<T*>(a.sum) + at, s[i], lane, valid);
                if (a.sum_codes != nullptr) put_codes<VEC>(a.sum_codes, a.sum_scales, at, first_block + c * a.tiles_per_row, s[i], lane, valid);
            }
        }
        if (a.y == nullptr && a.y_codes == nullptr) continue;
#pragma unroll
        for (int k = 0; k < 4; k++) part[warp][quad_at<VEC>(lane, k)] = sums[k];
        __syncthreads();
        if (threadIdx.x < CODE_BLOCK)
        {
            double total = 0.0;
#pragma unroll
            for (int w = 0; w < WARPS; w++) total += part[w][threadIdx.x];
            factor[threadIdx.x] = 1.0 / sqrt(total / static_cast<double>(C) + a.eps);
        }
        __syncthreads();
        double r[4];
        bool fast = true;
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            r[k] = factor[quad_at<VEC>(lane, k)];
            fast = fast && ordinary(r[k]);
        }
        fast = __all_sync(0xffffffffu, fast);
        const T* again = static_cast<const T*>(a.residual != nullptr ? a.sum : a.x);
        for (int64_t c0 = warp; c0 < C; c0 += HELD * WARPS)
        {
            if (!held)
#pragma unroll
                for (int i = 0; i < HELD; i++)
                {
                    const int64_t c = c0 + i * WARPS;
                    s[i] = load_quad<VEC>(again + first + c * a.inner, lane, c < C ? valid : 0);
                }
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                const int64_t c = c0 + i * WARPS;
                if (c >= C) continue;
                const Wide<T> weight = a.weight == nullptr ? Wide<T>(1) : widen(static_cast<const T*>(a.weight)[c]);
                const Wide<T> g[4] = {weight, weight, weight, weight};
                put_result<VEC>(a, s[i], r, g, fast, first + c * a.inner, first_block + c * a.tiles_per_row, lane, valid);
            }
        }
    }
}

/// Sum over the `per_row` warps of a group, which share a row; every warp of the thread block calls it.
template <int WARPS> __device__ __forceinline__ double group_sum(double v, double (&part)[WARPS], int per_row)
{
    v = warp_sum(v);
    if (per_row == 1) return v;
    const int warp = threadIdx.x >> 5, leader = warp / per_row * per_row;
    __syncthreads();   // the sums of the row before have been read
    if ((threadIdx.x & 31) == 0) part[warp] = v;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < per_row; w++) total += part[leader + w];
    return total;
}

/// Forward, rows of channels: `per_row` warps (a power of two) take a row, warp w of them the blocks w, w + per_row, ... of 128
/// channels, at most HELD of them.
template <typename T, bool VEC, int HELD, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) rms_norm_rows_kernel(const NormArgs a, int per_row)
{
    __shared__ double part[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % per_row, groups = WARPS / per_row;
    const int C = static_cast<int>(a.channels), blocks = static_cast<int>(a.tiles_per_row);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups; row0 < a.outer; row0 += static_cast<int64_t>(gridDim.x) * groups)
    {
        const int64_t row = row0 + warp / per_row, first = row * C;
        const bool live = row < a.outer;   // a warp without a row still takes part in the sums
        Quad<T> s[HELD];
        double sums = 0.0;
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            const int j = sub + i * per_row;
            s[i] = take_sum<VEC, T>(a, first + j * CODE_BLOCK, lane, live ? present(j, C) : 0);
        }
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            const int j = sub + i * per_row, valid = live ? present(j, C) : 0;
#pragma unroll
            for (int k = 0; k < 4; k++) sums = fma(static_cast<double>(widen(s[i].e[k])), static_cast<double>(widen(s[i].e[k])), sums);
            if (valid <= 0) continue;
            const int64_t at = first + j * CODE_BLOCK;
            if (a.residual != nullptr) store_quad<VEC>(static_cast<T*>(a.sum) + at, s[i], lane, valid);
            if (a.sum_codes != nullptr) put_codes<VEC>(a.sum_codes, a.sum_scales, at, row * blocks + j, s[i], lane, valid);
        }
        if (a.y == nullptr && a.y_codes == nullptr) continue;
        const double factor = 1.0 / sqrt(group_sum<WARPS>(sums, part, per_row) / static_cast<double>(C) + a.eps);
        const bool fast = ordinary(factor);
        const double r[4] = {factor, factor, factor, factor};
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            const int j = sub + i * per_row, valid = live ? present(j, C) : 0;
            if (valid <= 0) continue;
            Wide<T> g[4] = {1, 1, 1, 1};
            if (a.weight != nullptr) widen_quad(load_quad<VEC>(static_cast<const T*>(a.weight) + j * CODE_BLOCK, lane, valid), g);
            put_result<VEC>(a, s[i], r, g, fast, first + j * CODE_BLOCK, row * blocks + j, lane, valid);
        }
    }
}

/// What the backward kernels hold of a block of s: the elements, or four codes a lane and their scale.
template <typename T, bool CODES> struct HeldSum
{
    Quad<T> q;
    template <bool VEC> __device__ __forceinline__ void load(const NormGradArgs& a, int64_t at, int64_t, int lane, int valid)
    {
        q = load_quad<VEC>(static_cast<const T*>(a.sum) + at, lane, valid);
    }
    __device__ __forceinline__ Wide<T> value(int k) const { return widen(q.e[k]); }
};
template <typename T> struct HeldSum<T, true>
{
    uint32_t codes;
    Wide<T> scale;
    template <bool VEC> __device__ __forceinline__ void load(const NormGradArgs& a, int64_t at, int64_t block, int lane, int valid)
    {
        codes = load_codes<VEC>(a.sum_codes + at, lane, valid);
        scale = valid > 0 ? __ldg(static_cast<const Wide<T>*>(a.sum_scales) + block) : Wide<T>(0);
    }
    __device__ __forceinline__ Wide<T> value(int k) const { return widen(narrow<T>(decode_code(codes, k, scale))); }
};

/// The two numbers that a pixel's gradients need from its sums over the channels.
template <typename W> __device__ __forceinline__ void gradient_factors(double squares, double products, double channels, double eps, W& r, W& pull)
{
    const double factor = 1.0 / sqrt(squares / channels + eps);
    r = static_cast<W>(factor);
    pull = static_cast<W>(factor * factor * (products / channels));
}

/// gx of a lane's quad.
template <bool VEC, typename T>
__device__ __forceinline__ void put_gradient(const NormGradArgs& a, const Wide<T> (&gx)[4], int64_t at, int lane, int valid)
{
    Quad<T> q;
    Wide<T> more[4] = {0, 0, 0, 0};
    if (a.gsum != nullptr) widen_quad(load_quad<VEC>(static_cast<const T*>(a.gsum) + at, lane, valid), more);
#pragma unroll
    for (int k = 0; k < 4; k++) q.e[k] = narrow<T>(gx[k] + more[k]);
    store_quad<VEC>(static_cast<T*>(a.gx) + at, q, lane, valid);
}

/// Backward, feature maps: tiles as in the forward kernel. The thread blocks stay and walk over the tiles, so that gweight is
/// summed in registers over all of a block's tiles and leaves as one row of partial sums, which norm_weight_kernel adds up in a fixed
/// order. With more channels than are held, the tile is read twice (from L2) and gweight's sums live in shared memory.
template <typename T, bool VEC, bool CODES, int HELD, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) rms_norm_columns_backward_kernel(const NormGradArgs a)
{
    using W = Wide<T>;
    static_assert(WARPS >= 4, "a thread for every pixel of the tile");
    __shared__ double part[2][WARPS][CODE_BLOCK];
    __shared__ W factors[2][CODE_BLOCK];
    extern __shared__ __align__(16) unsigned char more_shared[];
    W* const weight_sums = reinterpret_cast<W*>(more_shared);   // [channels], only where the channels are not held
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t C = a.channels;
    const bool held = C <= HELD * WARPS;
    W weight_sum[HELD] = {};
    if (!held && a.gweight != nullptr)
        for (int64_t c = threadIdx.x; c < C; c += WARPS * 32) weight_sums[c] = W(0);
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const int64_t image = tile / a.tiles_per_row, piece = tile - image * a.tiles_per_row;
        const int valid = static_cast<int>(min(static_cast<int64_t>(CODE_BLOCK), a.inner - piece * CODE_BLOCK));
        const int64_t first = image * C * a.inner + piece * CODE_BLOCK, first_block = image * C * a.tiles_per_row + piece;
        HeldSum<T, CODES> s[HELD];
        Quad<T> gy[HELD];
        const auto load = [&](int64_t c0) {
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                const int64_t c = c0 + i * WARPS, at = first + c * a.inner;
                const int present = c < C ? valid : 0;
                s[i].template load<VEC>(a, at, first_block + c * a.tiles_per_row, lane, present);
                gy[i] = load_quad<VEC>(static_cast<const T*>(a.gy) + at, lane, present);
            }
        };
        const auto weight_of = [&](int64_t c) { return a.weight == nullptr || c >= C ? W(1) : widen(static_cast<const T*>(a.weight)[c]); };
        double squares[4] = {}, products[4] = {};
        for (int64_t c0 = warp; c0 < C; c0 += HELD * WARPS)
        {
            load(c0);
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                const W g = weight_of(c0 + i * WARPS);
#pragma unroll
                for (int k = 0; k < 4; k++)
                {
                    const double v = static_cast<double>(s[i].value(k));
                    squares[k] = fma(v, v, squares[k]);
                    products[k] = fma(v, static_cast<double>(widen(gy[i].e[k]) * g), products[k]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            part[0][warp][quad_at<VEC>(lane, k)] = squares[k];
            part[1][warp][quad_at<VEC>(lane, k)] = products[k];
        }
        __syncthreads();
        if (threadIdx.x < CODE_BLOCK)
        {
            double total[2] = {};
#pragma unroll
            for (int w = 0; w < WARPS; w++)
            {
                total[0] += part[0][w][threadIdx.x];
                total[1] += part[1][w][threadIdx.x];
            }
            gradient_factors(total[0], total[1], static_cast<double>(C), a.eps, factors[0][threadIdx.x], factors[1][threadIdx.x]);
        }
        __syncthreads();
        W r[4], pull[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            r[k] = factors[0][quad_at<VEC>(lane, k)];
            pull[k] = factors[1][quad_at<VEC>(lane, k)];
        }
        for (int64_t c0 = warp; c0 < C; c0 += HELD * WARPS)
        {
            if (!held) load(c0);
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                const int64_t c = c0 + i * WARPS;
                if (c >= C) continue;
                const W g = weight_of(c);
                W gx[4], through = 0;
#pragma unroll
                for (int k = 0; k < 4; k++)
                {
                    const W v = s[i].value(k), up = widen(gy[i].e[k]);
                    gx[k] = r[k] * (up * g - v * pull[k]);
                    through += up * (v * r[k]);
                }
                if (held) weight_sum[i] += through;
                else if (a.gweight != nullptr)
                {
                    through = warp_sum(through);
                    if (lane == 0) weight_sums[c] += through;   // channel c belongs to this warp alone
                }
                put_gradient<VEC, T>(a, gx, first + c * a.inner, lane, valid);
            }
        }
    }
    if (a.gweight == nullptr) return;
    W* const partial = static_cast<W*>(a.partial) + static_cast<int64_t>(blockIdx.x) * C;
    if (held)
    {
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            const int64_t c = warp + i * WARPS;
            const W total = warp_sum(weight_sum[i]);
            if (lane == 0 && c < C) partial[c] = total;
        }
    }
    else
    {
        __syncwarp();
        for (int64_t c = warp; c < C; c += WARPS)
            if (lane == 0) partial[c] = weight_sums[c];
    }
}

/// Backward, rows of channels. gweight's sums stay in the lanes that have the channels; the groups of a thread block add theirs
/// up in shared memory, one after the other, at the end.
template <typename T, bool VEC, bool CODES, int HELD, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) rms_norm_rows_backward_kernel(const NormGradArgs a, int per_row)
{
    using W = Wide<T>;
    __shared__ double part[WARPS];
    extern __shared__ __align__(16) unsigned char more_shared[];
    W* const weight_sums = reinterpret_cast<W*>(more_shared);   // [channels]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % per_row, groups = WARPS / per_row;
    const int C = static_cast<int>(a.channels), blocks = static_cast<int>(a.tiles_per_row);
    W weight_sum[HELD][4] = {};
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups; row0 < a.outer; row0 += static_cast<int64_t>(gridDim.x) * groups)
    {
        const int64_t row = row0 + warp / per_row, first = row * C;
        const bool live = row < a.outer;
        HeldSum<T, CODES> s[HELD];
        Quad<T> gy[HELD];
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            const int j = sub + i * per_row, valid = live ? present(j, C) : 0;
            s[i].template load<VEC>(a, first + j * CODE_BLOCK, row * blocks + j, lane, valid);
            gy[i] = load_quad<VEC>(static_cast<const T*>(a.gy) + first + j * CODE_BLOCK, lane, valid);
        }
        const auto weights_of = [&](int j, W (&g)[4]) {
            if (a.weight != nullptr) widen_quad(load_quad<VEC>(static_cast<const T*>(a.weight) + j * CODE_BLOCK, lane, present(j, C)), g);
            else
#pragma unroll
                for (int k = 0; k < 4; k++) g[k] = W(1);
        };
        double squares = 0.0, products = 0.0;
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            W g[4];
            weights_of(sub + i * per_row, g);
#pragma unroll
            for (int k = 0; k < 4; k++)
            {
                const double v = static_cast<double>(s[i].value(k));
                squares = fma(v, v, squares);
                products = fma(v, static_cast<double>(widen(gy[i].e[k]) * g[k]), products);
            }
        }
        squares = group_sum<WARPS>(squares, part, per_row);
        products = group_sum<WARPS>(products, part, per_row);
        W r, pull;
        gradient_factors(squares, products, static_cast<double>(C), a.eps, r, pull);
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            const int j = sub + i * per_row, valid = live ? present(j, C) : 0;
            if (valid <= 0) continue;
            W g[4], gx[4];
            weights_of(j, g);
#pragma unroll
            for (int k = 0; k < 4; k++)
            {
                const W v = s[i].value(k), up = widen(gy[i].e[k]);
                gx[k] = r * (up * g[k] - v * pull);
                weight_sum[i][k] += up * (v * r);
            }
            put_gradient<VEC, T>(a, gx, first + j * CODE_BLOCK, lane, valid);
        }
    }
    if (a.gweight == nullptr) return;
    for (int turn = 0; turn < groups; turn++)
    {
        if (warp / per_row == turn)
#pragma unroll
            for (int i = 0; i < HELD; i++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                {
                    const int c = (sub + i * per_row) * CODE_BLOCK + quad_at<VEC>(lane, k);
                    if (c < C) weight_sums[c] = (turn == 0 ? W(0) : weight_sums[c]) + weight_sum[i][k];
                }
        __syncthreads();
    }
    W* const partial = static_cast<W*>(a.partial) + static_cast<int64_t>(blockIdx.x) * C;
    for (int c = threadIdx.x; c < C; c += WARPS * 32) partial[c] = weight_sums[c];
}

/// gweight from the rows of partial sums: a thread block takes 32 channels, its warps every eighth row, in double and in a fixed order.
template <typename T>
__global__ void __launch_bounds__(THREADS) norm_weight_kernel(const Wide<T>* __restrict__ partial, T* __restrict__ gweight, int64_t channels, int rows)
{
    __shared__ double part[THREADS / 32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    double sum = 0.0;
    if (c < channels)
#pragma unroll 8
        for (int row = warp; row < rows; row += THREADS / 32) sum += static_cast<double>(__ldg(partial + row * channels + c));
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < channels)
    {
        for (int w = 1; w < THREADS / 32; w++) sum += part[w][lane];
        gweight[c] = narrow<T>(static_cast<Wide<T>>(sum));
    }
}

}  // namespace mc
