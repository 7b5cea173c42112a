// Root-mean-square norm over the channels, forward and backward, with the residual's addition and the 8-bit forms of its result
// and of its input.
//
//     s = T(x + residual),  r = 1 / sqrt(mean_c s^2 + eps),  y = T(s r weight_c)
//     gx = r (u - s r^2 mean_c(u s)) + gsum,  u = gy weight_c;   gweight_c = sum over the pixels of gy s r
//
// Every kernel reads its inputs from memory once: the tile of a thread block, all channels of 32 to 128 neighbouring pixels (columns) or whole
// rows of channels (rows), stays in registers, or in L2 where it has too many channels, between the sums over the channels and what is computed
// from them. Bytes bound them: a forward pass with residual moves 16 bytes an element in float (13 with the result in 8 bits), a backward pass 16 (13).
//
// The forward pass takes the sums over the channels in double and rounds y once, from an unevaluated sum of two floats that carries
// about 46 bits (to float, and from there, in half precision; in double after each product): y, and with it every code of its 8-bit form, is then what 64-bit arithmetic gives, whichever kernel computed it and
// in whatever order. A float that is one unit off moves one code in 10^5 to its neighbour; plain float arithmetic behind a result of 11 bits
// moves one result in 2^10, and with the largest of a block its scale ((32, 64, 224, 224) in bfloat16 98 us so, 111 as it is).
#pragma once
#include <type_traits>

#include "encode8.cuh"

namespace mc
{

// T is the tensors' type throughout, G the weight's: T, or float beside half precision, as programs with float master weights have it.

struct NormArgs
{
    const void *x, *residual, *weight;
    void *sum, *y, *y_scales, *sum_scales;
    int8_t *y_codes, *sum_codes;
    int64_t outer, channels, inner;
    int64_t tiles_per_row, tiles;   // blocks of 128 pixels in an image and in all (columns), of 128 channels in a row (rows)
    double eps, per_channel;        // per_channel: 1 / channels
};

struct NormGradArgs
{
    const void *sum, *sum_scales, *weight, *gy, *gsum;
    const int8_t* sum_codes;
    void *gx, *gweight;
    void* partial;                  // [grid, channels], Wide<T>
    int64_t outer, channels, inner;
    int64_t tiles_per_row, tiles;
    double eps, per_channel;
};

/// The factor r of a lane's elements as the products with it are taken, for an ordinary r: the halves are normal floats, and an
/// infinite s cannot meet them (its r is 0). `times` rounds s r g once to float where that is the wide type (r as two floats with about 48 bits of it,
/// pairs of elements by packed instructions) and after each product in double.
template <typename W> struct Factor
{
    W r;
    __device__ __forceinline__ void set(double v) { r = v; }
    __device__ __forceinline__ Factor of_lane(int i) const { return {__shfl_sync(0xffffffffu, r, i)}; }
};
template <> struct Factor<float>
{
    float r, low;
    __device__ __forceinline__ void set(double v)
    {
        r = static_cast<float>(v);
        low = static_cast<float>(v - static_cast<double>(r));
    }
    __device__ __forceinline__ Factor of_lane(int i) const { return {__shfl_sync(0xffffffffu, r, i), __shfl_sync(0xffffffffu, low, i)}; }
};

template <typename W>
__device__ __forceinline__ void times(const W (&s)[4], const Factor<W>& r0, const Factor<W>& r1, const Factor<W>& r2, const Factor<W>& r3, const W (&g)[4], W (&y)[4])
{
    if constexpr (std::is_same<W, float>::value)
    {
        const auto pair = [](float s0, float s1, const Factor<float>& a, const Factor<float>& b, float g0, float g1, float& y0, float& y1) {
            const float2 v = make_float2(s0, s1), g = make_float2(g0, g1);
            const float2 p = __fmul2_rn(v, make_float2(a.r, b.r));
            const float2 p_low = __ffma2_rn(v, make_float2(a.low, b.low), __ffma2_rn(v, make_float2(a.r, b.r), make_float2(-p.x, -p.y)));
            const float2 y = __fmul2_rn(p, g);
            const float2 sum = __fadd2_rn(y, __ffma2_rn(p_low, g, __ffma2_rn(p, g, make_float2(-y.x, -y.y))));
            y0 = sum.x;
            y1 = sum.y;
        };
        pair(s[0], s[1], r0, r1, g[0], g[1], y[0], y[1]);
        pair(s[2], s[3], r2, r3, g[2], g[3], y[2], y[3]);
    }
    else
    {
        y[0] = s[0] * r0.r * g[0];
        y[1] = s[1] * r1.r * g[1];
        y[2] = s[2] * r2.r * g[2];
        y[3] = s[3] * r3.r * g[3];
    }
}

/// Whether the products above hold with weights of this size: an infinite product has no remainder.
__device__ __forceinline__ bool ordinary_weight(float g) { return fabsf(g) < 0x1p100f; }
__device__ __forceinline__ bool ordinary_weight(double) { return true; }

__device__ __forceinline__ bool ordinary(double r) { return r > 0x1p-60 && r < 0x1p60; }

/// r from the sum of the squares.
__device__ __forceinline__ double norm_factor(double squares, double per_channel, double eps) { return rsqrt(squares * per_channel + eps); }

/// Sums in float are taken once more in double where they left its range: squares near its largest value, or, for an eps that does not
/// cover them, near its smallest; infinities and NaN. Products too small for float's normal numbers (upstream gradients below some 1e-33) are not: they
/// lose digits as in any float arithmetic, and a test for them could not tell them from the zeros of a masked pixel.
__device__ __forceinline__ bool out_of_range(double squares, double products, double eps)
{
    return !(squares < 0x1p120) || (squares < 0x1p-60 && eps < 0x1p-60) || !(fabs(products) < 0x1p120);
}

/// Sum over LANES neighbouring lanes, the same in each of them.
template <int LANES, typename V> __device__ __forceinline__ V lanes_sum(V v)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
template <typename V> __device__ __forceinline__ V warp_sum(V v) { return lanes_sum<32>(v); }

/// Keeps the compiler from holding the widened elements of a quad of half precision from one use to the next: they are cheaper to make again
/// than the registers that they fill.
template <typename T> __device__ __forceinline__ void forget_widened(Quad<T>& q)
{
    if constexpr (sizeof(T) == 2) asm("" : "+r"(q.word[0]), "+r"(q.word[1]));
}

/// x + residual, rounded to T.
template <typename T> __device__ __forceinline__ Quad<T> add_quads(const Quad<T>& a, const Quad<T>& b)
{
    Wide<T> u[4], v[4];
    widen_quad(a, u);
    widen_quad(b, v);
#pragma unroll
    for (int k = 0; k < 4; k++) u[k] += v[k];
    return narrow_quad<T>(u);
}

/// Sums of squares of N quads, one or four for a lane's four elements, added to `sums`.
template <int N, int SUMS, typename T> __device__ __forceinline__ void add_squares(const Quad<T> (&s)[N], double (&sums)[SUMS])
{
#pragma unroll
    for (int i = 0; i < N; i++)
    {
        Wide<T> v[4];
        widen_quad(s[i], v);
#pragma unroll
        for (int k = 0; k < 4; k++) sums[k % SUMS] = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), sums[k % SUMS]);
    }
}

/// Codes and scales of N blocks: block i lies `offset(i)` elements and i `block_step` blocks behind the first, whose codes and scale go to `codes`
/// and `scales`; `count` exist from it on, of which the N here are stored: lanes beyond them have no scale, and one place is not to be written by two lanes.
template <bool VEC, int N, typename T, typename Offset>
__device__ __forceinline__ void put_codes(int8_t* codes, void* scales, Offset offset, int64_t block_step, const Quad<T> (&q)[N], int count, int lane, const int (&left)[N])
{
    Wide<T> v[N][4];
    uint32_t c[N];
#pragma unroll
    for (int i = 0; i < N; i++) widen_quad(q[i], v[i]);
    const Wide<T> scale = encode_blocks(v, c, lane);
#pragma unroll
    for (int i = 0; i < N; i++) store_codes<VEC>(codes + offset(i), c[i], left[i]);
    if (lane < min(count, N)) static_cast<Wide<T>*>(scales)[lane * block_step] = scale;
}

// The kernels that keep a tile in registers fetch the next one meanwhile, by asynchronous copies into slots of shared memory that only
// the thread that issued the copy reads: no barrier and no register is spent on it, and the loads of one tile travel while the sums,
// barriers and stores of another take their time. A slot may be fetched into again once its reader has passed a __syncwarp.
// What it gave, when thread blocks had 8 warps and whole tiles: float, (32, 64, 224, 224) 11 % of the time; bfloat16, rows of 512 channels, 27 %. Rows that need copies of single
// elements lose a little ((40, 20, 75, 101): 40 us against 33 then, 35 now). The forward kernels do not
// fetch ahead: with a residual it made 292 us of 247, because thread blocks that stay drift apart, and neighbouring tiles, which share
// pages of memory, are then no longer read together.

/// Bytes of `src` into shared memory, zeros where it does not exist. 4, 8 or 16 bytes.
template <int BYTES> __device__ __forceinline__ void fetch_bytes(void* slot, const void* src, bool exists)
{
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(slot));
    const int bytes = exists ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
/// Waits until all but the newest PENDING groups of the thread's copies have landed.
template <int PENDING> __device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

/// A quad of `base + at` on its way into a slot. Single elements of half precision have no asynchronous copy: they are loaded there and then.
template <bool VEC, int LANES = 32, typename T> __device__ __forceinline__ void fetch_quad(Quad<T>* slot, const T* base, int64_t at, int left)
{
    if constexpr (VEC)
    {
        const T* src = left > 0 ? base + at : base;
        constexpr int BYTES = sizeof(T) == 2 ? 8 : 16;
#pragma unroll
        for (int b = 0; b < static_cast<int>(4 * sizeof(T)); b += BYTES)
            fetch_bytes<BYTES>(reinterpret_cast<unsigned char*>(slot) + b, reinterpret_cast<const unsigned char*>(src) + b, left > 0);
    }
    else if constexpr (sizeof(T) >= 4)
    {
#pragma unroll
        for (int k = 0; k < 4; k++) fetch_bytes<sizeof(T)>(&slot->e[k], LANES * k < left ? base + at + LANES * k : base, LANES * k < left);
    }
    else *slot = load_quad<VEC, LANES>(base + at, left);
}
template <bool VEC, int LANES = 32> __device__ __forceinline__ void fetch_codes(uint32_t* slot, const int8_t* base, int64_t at, int left)
{
    if constexpr (VEC) fetch_bytes<4>(slot, left > 0 ? base + at : base, left > 0);
    else *slot = load_codes<VEC, LANES>(base + at, left);
}

/// Blocks are finished and encoded this many at a time.
constexpr int GROUP = 4;

/// Where a tile of 128 pixels lies, as the lane sees it: its first element and block in the warp's first channel.
struct Place
{
    int64_t first, block;
    int left;
};
template <bool VEC, typename Args> __device__ __forceinline__ Place place_of(const Args& a, int64_t tile, int lane, int warp)
{
    const int64_t image = tile / a.tiles_per_row, piece = tile - image * a.tiles_per_row, row = image * a.channels + warp;
    return {row * a.inner + piece * CODE_BLOCK + lane_at<VEC>(lane), row * a.tiles_per_row + piece,
            static_cast<int>(min(static_cast<int64_t>(CODE_BLOCK), a.inner - piece * CODE_BLOCK)) - lane_at<VEC>(lane)};
}

/// Forward, feature maps. A block of WARPS warps takes 128 pixels of an image; warp w has the channels w, w + WARPS, ... and keeps
/// up to eight of them. Where there are more, the second pass reads s again, from `sum` or x: the tiles that are at work then
/// lie in L2 (128 pixels of 64 channels in float are 32 KiB, of 592 thread blocks 19 MiB; of 512 channels, of 148 thread blocks, 38 MiB).
template <typename T, typename G, bool VEC, int WARPS, int CTAS> __global__ void __launch_bounds__(WARPS * 32, CTAS) rms_norm_columns_kernel(const NormArgs a)
{
    constexpr int HELD = 8;
    static_assert(WARPS >= 4 && HELD % GROUP == 0, "a thread for every pixel of the tile");
    using W = Wide<T>;
    __shared__ double part[WARPS][CODE_BLOCK];
    __shared__ double factor[CODE_BLOCK];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, C = static_cast<int>(a.channels);
    const int own = (C - warp + WARPS - 1) / WARPS;   // channels of this warp
    const bool held = C <= HELD * WARPS;
    const int64_t step = WARPS * a.inner, block_step = WARPS * a.tiles_per_row;
    const auto offset = [&](int i) { return i * step; };
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const int64_t image = tile / a.tiles_per_row, piece = tile - image * a.tiles_per_row;
        const int left = static_cast<int>(min(static_cast<int64_t>(CODE_BLOCK), a.inner - piece * CODE_BLOCK)) - lane_at<VEC>(lane);
        const int64_t first = (image * C + warp) * a.inner + piece * CODE_BLOCK + lane_at<VEC>(lane);
        const int64_t first_block = (image * C + warp) * a.tiles_per_row + piece;
        Quad<T> s[HELD];
        const auto load = [&](const void* from, int i0, Quad<T> (&q)[HELD]) {
            const T* p = static_cast<const T*>(from) + first + i0 * step;
#pragma unroll
            for (int i = 0; i < HELD; i++, p += step) q[i] = load_quad<VEC>(p, i0 + i < own ? left : 0);
        };
        double sums[4] = {};
        for (int i0 = 0; i0 < own; i0 += HELD)
        {
            load(a.x, i0, s);
            if (a.residual != nullptr)
            {
                Quad<T> more[HELD];
                load(a.residual, i0, more);
#pragma unroll
                for (int i = 0; i < HELD; i++) s[i] = add_quads(s[i], more[i]);
                T* p = static_cast<T*>(a.sum) + first + i0 * step;
#pragma unroll
                for (int i = 0; i < HELD; i++, p += step) store_quad<VEC>(p, s[i], i0 + i < own ? left : 0);
            }
            add_squares(s, sums);
            if (a.sum_codes != nullptr)
#pragma unroll
                for (int g0 = 0; g0 < HELD; g0 += GROUP)
                {
                    const int at = i0 + g0;
                    if (at >= own) break;
                    const Quad<T> q[GROUP] = {s[g0], s[g0 + 1], s[g0 + 2], s[g0 + 3]};
                    const int lefts[GROUP] = {left, at + 1 < own ? left : 0, at + 2 < own ? left : 0, at + 3 < own ? left : 0};
                    put_codes<VEC>(a.sum_codes + first + at * step, static_cast<W*>(a.sum_scales) + first_block + at * block_step, offset, block_step, q,
                                   own - at, lane, lefts);
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
            factor[threadIdx.x] = norm_factor(total, a.per_channel, a.eps);
        }
        __syncthreads();
        Factor<W> r[4];
        bool all_ordinary = true;
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            const double v = factor[quad_at<VEC>(lane, k)];
            r[k].set(v);
            all_ordinary = all_ordinary && ordinary(v);
        }
        all_ordinary = __all_sync(0xffffffffu, all_ordinary);
        for (int i0 = 0; i0 < own; i0 += HELD)
        {
            if (!held) load(a.residual != nullptr ? a.sum : a.x, i0, s);
#pragma unroll
            for (int g0 = 0; g0 < HELD; g0 += GROUP)
            {
                const int at = i0 + g0;
                if (at >= own) break;
                const int lefts[GROUP] = {left, at + 1 < own ? left : 0, at + 2 < own ? left : 0, at + 3 < own ? left : 0};
                W g[GROUP];
                bool usual = all_ordinary;
#pragma unroll
                for (int i = 0; i < GROUP; i++)
                {
                    g[i] = a.weight == nullptr || at + i >= own ? W(1) : widen(static_cast<const G*>(a.weight)[warp + (at + i) * WARPS]);
                    usual = usual && ordinary_weight(g[i]);
                }
                Quad<T> y[GROUP];
#pragma unroll
                for (int i = 0; i < GROUP; i++)
                {
                    W v[4], result[4];
                    widen_quad(s[g0 + i], v);
                    const W weights[4] = {g[i], g[i], g[i], g[i]};
                    if (usual) times(v, r[0], r[1], r[2], r[3], weights, result);
                    else
                    {
                        rarely();
                        times(v, r[0], r[1], r[2], r[3], weights, result);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                        {
                            const double exact = factor[quad_at<VEC>(lane, k)];
                            if (!ordinary(exact) || !ordinary_weight(g[i])) result[k] = static_cast<W>(static_cast<double>(v[k]) * exact * static_cast<double>(g[i]));
                        }
                    }
                    y[i] = narrow_quad<T>(result);
                }
                if (a.y != nullptr)
                {
                    T* p = static_cast<T*>(a.y) + first + at * step;
#pragma unroll
                    for (int i = 0; i < GROUP; i++, p += step) store_quad<VEC>(p, y[i], lefts[i]);
                }
                if (a.y_codes != nullptr)
                    put_codes<VEC>(a.y_codes + first + at * step, static_cast<W*>(a.y_scales) + first_block + at * block_step, offset, block_step, y, own - at, lane,
                                   lefts);
            }
        }
    }
}

/// Sums over the warp of R values (1, 2 or 4): lane l returns that of value l % R. A lane gives away the values that others will hold.
template <int R, typename V> __device__ __forceinline__ V spread_sums(const V (&v)[R], int lane)
{
    static_assert(R == 1 || R == 2 || R == 4, "a power of two");
    const auto halve = [&](V even, V odd, int d) {
        const bool upper = (lane & d) != 0;
        return (upper ? odd : even) + __shfl_xor_sync(0xffffffffu, upper ? even : odd, d);
    };
    V sum;
    if constexpr (R == 1) sum = v[0];
    else if constexpr (R == 2) sum = halve(v[0], v[1], 1);
    else sum = halve(halve(v[0], v[1], 1), halve(v[2], v[3], 1), 2);
#pragma unroll
    for (int d = R; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}

/// Adds up K numbers of each of the 2^shift warps that share a row; every lane gets the sums. The warps of a row meet at a barrier of their own:
/// `part` is written in turns, so that one is enough.
template <int K, int WARPS> __device__ __forceinline__ void share_sums(double (&v)[K], double (&part)[2][WARPS][K], int& turn, int shift)
{
    if (shift == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp >> shift, per_row = 1 << shift;
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; k++) part[turn][warp][k] = v[k];
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 << shift) : "memory");
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = part[turn][(group << shift) + (lane & (per_row - 1))][k];
    turn ^= 1;
    for (int d = per_row >> 1; d > 0; d >>= 1)
#pragma unroll
        for (int k = 0; k < K; k++) v[k] += __shfl_xor_sync(0xffffffffu, v[k], d);
}

/// How a warp of the kernels for rows of channels holds ROWS neighbouring rows of BLOCKS blocks of 128 channels each; 2^shift warps share a row, warp
/// `sub` of them has the blocks sub, sub + 2^shift, ... More than one row is for rows of exactly BLOCKS blocks that no warps share. Without that a row
/// of few channels leaves most of what a warp is unrolled for empty: (65536, 64) in float took 45 us forward and 56 backward, 11 and 23 so.
template <bool VEC, int ROWS, int BLOCKS> struct RowTile
{
    int C, c0, own, step, at;   // channels; the lane's first; blocks of this warp; channels from one to the next; the lane's place in a block

    __device__ __forceinline__ RowTile(int64_t channels, int64_t blocks, int shift, int lane, int warp)
        : C(static_cast<int>(channels)), step(CODE_BLOCK << shift), at(lane_at<VEC>(lane))
    {
        const int sub = warp & ((1 << shift) - 1);
        c0 = sub * CODE_BLOCK + at;
        own = (static_cast<int>(blocks) - sub + (1 << shift) - 1) >> shift;
    }
    /// Channels from the lane's of block j to the end of the block.
    __device__ __forceinline__ int left_in(int j) const { return j < own ? min(CODE_BLOCK - at, C - c0 - j * step) : 0; }
    /// The same for quad q, of `rows` rows that exist; where it lies; and how many blocks there are.
    __device__ __forceinline__ int left(int q, int rows) const { return q / BLOCKS < rows ? left_in(q % BLOCKS) : 0; }
    __device__ __forceinline__ int offset(int q) const { return q / BLOCKS * C + q % BLOCKS * step; }
    __device__ __forceinline__ int count(int rows) const { return ROWS == 1 ? own : rows * BLOCKS; }
};

/// Forward, rows of channels. Bytes bound it in float: (32768, 1024) 84 us with the residual, 97 % of the copy rate, 70 with codes. In half precision
/// instructions do, some 20 an element: (65536, 512) in bfloat16 44 us, with residual 53 (77 %). Four thread blocks an SM: three take 48 and 58, five
/// spill (48 and 64).
template <typename T, typename G, bool VEC, int ROWS, int BLOCKS, int WARPS, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS) rms_norm_rows_kernel(const NormArgs a, int shift)
{
    constexpr int N = ROWS * BLOCKS;
    static_assert(N % GROUP == 0, "whole groups");
    using W = Wide<T>;
    __shared__ double part[2][WARPS][1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = WARPS >> shift;
    const RowTile<VEC, ROWS, BLOCKS> t(a.channels, a.tiles_per_row, shift, lane, warp);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * groups * ROWS;
    int turn = 0;
    for (int64_t row = (static_cast<int64_t>(blockIdx.x) * groups + (warp >> shift)) * ROWS; row < a.outer; row += stride)
    {
        const int rows = static_cast<int>(min(static_cast<int64_t>(ROWS), a.outer - row)), count = t.count(rows);
        const int64_t first = row * t.C + t.c0, first_block = row * a.tiles_per_row + (t.c0 - t.at) / CODE_BLOCK;
        Quad<T> s[N];
        const auto load = [&](const void* from, Quad<T> (&q)[N]) {
#pragma unroll
            for (int i = 0; i < N; i++) q[i] = load_quad<VEC>(static_cast<const T*>(from) + first + t.offset(i), t.left(i, rows));
        };
        load(a.x, s);
        if (a.residual != nullptr)
        {
            Quad<T> more[N];
            load(a.residual, more);
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                s[i] = add_quads(s[i], more[i]);
                store_quad<VEC>(static_cast<T*>(a.sum) + first + t.offset(i), s[i], t.left(i, rows));
            }
        }
        const auto put = [&](int8_t* codes, void* scales, const Quad<T> (&q)[GROUP], int g0) {
            const int lefts[GROUP] = {t.left(g0, rows), t.left(g0 + 1, rows), t.left(g0 + 2, rows), t.left(g0 + 3, rows)};
            put_codes<VEC>(codes + first, static_cast<W*>(scales) + first_block + (static_cast<int64_t>(g0) << shift), [&](int i) { return t.offset(g0 + i); },
                           int64_t(1) << shift, q, count - g0, lane, lefts);
        };
        if (a.sum_codes != nullptr)
#pragma unroll
            for (int g0 = 0; g0 < N; g0 += GROUP)
            {
                if (g0 >= count) break;
                const Quad<T> q[GROUP] = {s[g0], s[g0 + 1], s[g0 + 2], s[g0 + 3]};
                put(a.sum_codes, a.sum_scales, q, g0);
            }
        if (a.y == nullptr && a.y_codes == nullptr) continue;
        double squares[ROWS][1] = {}, own[ROWS];
#pragma unroll
        for (int i = 0; i < N; i++)
        {
            const Quad<T> one[1] = {s[i]};
            add_squares(one, squares[i / BLOCKS]);
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++) own[i] = squares[i][0];
        double total[1] = {spread_sums(own, lane)};   // of row lane % ROWS
        share_sums(total, part, turn, shift);
        const double factor = norm_factor(total[0], a.per_channel, a.eps);
        // Bit i: row i. One row as a yes or no of the whole warp, which the compiler turns into a branch around the loop below (50 us against 56 for
        // (65536, 512) bfloat16 with residual).
        const unsigned ordinary_rows = ROWS == 1 ? __all_sync(0xffffffffu, ordinary(factor)) : __ballot_sync(0xffffffffu, ordinary(factor));
        const bool some_ordinary = ordinary_rows != 0;
        Factor<W> mine, r[ROWS];
        mine.set(factor);
#pragma unroll
        for (int i = 0; i < ROWS; i++) r[i] = ROWS == 1 ? mine : mine.of_lane(i);
        W g[4] = {1, 1, 1, 1};
        bool usual = some_ordinary;
#pragma unroll
        for (int g0 = 0; g0 < N; g0 += GROUP)
        {
            if (g0 >= count) break;
            Quad<T> y[GROUP];
#pragma unroll
            for (int i = 0; i < GROUP; i++)
            {
                const int q = g0 + i;
                W v[4], result[4];
                widen_quad(s[q], v);
                if (a.weight != nullptr && (BLOCKS > 1 || q == 0))
                {
                    widen_quad(load_quad<VEC>(static_cast<const G*>(a.weight) + t.c0 + q % BLOCKS * t.step, t.left_in(q % BLOCKS)), g);
                    usual = some_ordinary && __all_sync(0xffffffffu, ordinary_weight(g[0]) && ordinary_weight(g[1]) && ordinary_weight(g[2]) && ordinary_weight(g[3]));
                }
                const Factor<W>& f = r[q / BLOCKS];
                if (usual && (ROWS == 1 || (ordinary_rows >> (q / BLOCKS) & 1u) != 0)) times(v, f, f, f, f, g, result);
                else   // the whole warp
                {
                    rarely();
                    const double exact = __shfl_sync(0xffffffffu, factor, q / BLOCKS);
#pragma unroll
                    for (int k = 0; k < 4; k++) result[k] = static_cast<W>(static_cast<double>(v[k]) * exact * static_cast<double>(g[k]));
                }
                y[i] = narrow_quad<T>(result);
                if (a.y != nullptr) store_quad<VEC>(static_cast<T*>(a.y) + first + t.offset(q), y[i], t.left(q, rows));
            }
            if (a.y_codes != nullptr) put(a.y_codes, a.y_scales, y, g0);
        }
    }
}

/// What the backward kernels hold of a block of s: the elements, or four codes a lane and their scale, which in float and double are fewer registers than
/// the elements; in half precision they are as many, and the elements are made once.
template <typename T, bool CODES> struct HeldSum
{
    Quad<T> q;
    template <bool VEC> __device__ __forceinline__ void load(const NormGradArgs& a, int64_t at, int64_t, int left, bool)
    {
        q = load_quad<VEC>(static_cast<const T*>(a.sum) + at, left);
    }
    using Slot = Quad<T>;
    template <bool VEC, int LANES = 32> static __device__ __forceinline__ void fetch(const NormGradArgs& a, Slot* slot, int64_t at, int left)
    {
        fetch_quad<VEC, LANES>(slot, static_cast<const T*>(a.sum), at, left);
    }
    __device__ __forceinline__ void take(const Slot& slot, Wide<T>) { q = slot; }
    __device__ __forceinline__ void forget_values() { forget_widened(q); }
    __device__ __forceinline__ void values(Wide<T> (&v)[4]) const { widen_quad(q, v); }
};
template <typename T> struct HeldSum<T, true>
{
    static constexpr bool DECODED = sizeof(T) == 2;
    struct Codes
    {
        uint32_t codes;
        Wide<T> scale;
    };
    typename std::conditional<DECODED, Quad<T>, Codes>::type held;
    using Slot = uint32_t;
    template <bool VEC> __device__ __forceinline__ void load(const NormGradArgs& a, int64_t at, int64_t block, int left, bool exists)
    {
        take(load_codes<VEC>(a.sum_codes + at, left), exists ? __ldg(static_cast<const Wide<T>*>(a.sum_scales) + block) : Wide<T>(0));
    }
    template <bool VEC, int LANES = 32> static __device__ __forceinline__ void fetch(const NormGradArgs& a, Slot* slot, int64_t at, int left)
    {
        fetch_codes<VEC, LANES>(slot, a.sum_codes, at, left);
    }
    __device__ __forceinline__ void take(uint32_t codes, Wide<T> scale)
    {
        if constexpr (DECODED)
        {
            Wide<T> v[4];
            decode_quad(codes, scale, v);
            held = narrow_quad<T>(v);
        }
        else held = {codes, scale};
    }
    __device__ __forceinline__ void forget_values()
    {
        if constexpr (DECODED) forget_widened(held);
        else asm("" : "+r"(held.codes));
    }
    __device__ __forceinline__ void values(Wide<T> (&v)[4]) const
    {
        if constexpr (DECODED) widen_quad(held, v);
        else decode_quad(held.codes, held.scale, v);
    }
};

/// The two numbers that a pixel's gradients need from its sums over the channels. The square of a factor that only double holds may leave even its range.
template <typename W> __device__ __forceinline__ void gradient_factors(double squares, double products, double per_channel, double eps, W& r, W& pull)
{
    const double factor = norm_factor(squares, per_channel, eps), mean = products * per_channel;
    r = static_cast<W>(factor);
    if (sizeof(W) == 4 || ordinary(factor)) pull = static_cast<W>(factor * factor * mean);
    else pull = static_cast<W>(factor * (factor * mean));
}

// The kernels of the backward pass compute gradients in W from these factors. In float that needs an eps of 2^-120 or more (TINY_EPS): r is 2^60 at most
// then, also for the pixels of zeros whose r is that of eps alone, the places of a tile that lie outside the image among them. For a smaller
// eps in float and half precision there are variants (EXACT) that take the pixels whose factors float does not hold by way of double: an
// infinite factor times a zero would be NaN, and one such pixel the end of all of gweight. As one kernel for every eps the rare branch cost the usual
// ones their registers: 5 to 10 % of most shapes, (64, 256, 56, 56) from codes 113 to 146 us.
constexpr double TINY_EPS = 0x1p-120;

/// Whether a pixel's gradients may be computed from these factors in float.
__device__ __forceinline__ bool gradients_fit(float r, float pull) { return r > 0x1p-60f && r < 0x1p60f && fabsf(pull) < 0x1p100f; }

/// gx of an element and what it gives to gweight, added to `through`; the same by way of double, which holds what float does not.
template <typename W> __device__ __forceinline__ void element_gradient(W v, W up, W g, W r, W pull, W& gx, W& through)
{
    gx = r * (up * g - v * pull);
    through += up * (v * r);
}
template <typename W> __device__ __forceinline__ void element_gradient_in_double(W v, W up, W g, double r, double pull, W& gx, W& through)
{
    gx = static_cast<W>(r * (static_cast<double>(up) * static_cast<double>(g) - static_cast<double>(v) * pull));
    through += static_cast<W>(static_cast<double>(up) * (static_cast<double>(v) * r));
}

/// gx of a lane's quad, `more` pointing to the gradient that comes past the norm.
template <bool VEC, int LANES, typename T> __device__ __forceinline__ void put_gradient(const NormGradArgs& a, Wide<T> (&gx)[4], const Quad<T>* more, int64_t at, int left)
{
    if (a.gsum != nullptr)
    {
        Wide<T> v[4];
        widen_quad(*more, v);
#pragma unroll
        for (int k = 0; k < 4; k++) gx[k] += v[k];
    }
    store_quad<VEC, LANES>(static_cast<T*>(a.gx) + at, narrow_quad<T>(gx), left);
}

/// The factors of a tile's pixels in the backward kernels, r and the pull of the sum, in shared memory for all threads. `add_up` adds squares and
/// products of the warp's channels up in the type that it is given, and again in double where float's range was left: squares and products in
/// turn then, because the room is that of both in float. EXACT: false where some factors do not fit float, and `exact` has all of them in double
/// then. Ends with a barrier.
template <bool VEC, int LANES, bool EXACT, typename W, int GROUPS, int PIXELS, int PLACES, typename AddUp>
__device__ __forceinline__ bool tile_gradient_factors(W (&part)[2][GROUPS][PIXELS], W (&factors)[2][PIXELS], double (&exact)[2][PLACES], double per_channel, double eps, int lane,
                                                      int group, AddUp add_up)
{
    W sums[2][4] = {};
    add_up(sums);
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        part[0][group][quad_at<VEC, LANES>(lane, k)] = sums[0][k];
        part[1][group][quad_at<VEC, LANES>(lane, k)] = sums[1][k];
    }
    __syncthreads();
    bool again = false, fits = true;
    double total[2];
    if (threadIdx.x < PIXELS)
    {
        total[0] = total[1] = 0.0;
#pragma unroll
        for (int g = 0; g < GROUPS; g++)
        {
            total[0] += static_cast<double>(part[0][g][threadIdx.x]);
            total[1] += static_cast<double>(part[1][g][threadIdx.x]);
        }
        gradient_factors(total[0], total[1], per_channel, eps, factors[0][threadIdx.x], factors[1][threadIdx.x]);
        again = out_of_range(total[0], total[1], eps);
        if constexpr (EXACT) fits = gradients_fit(factors[0][threadIdx.x], factors[1][threadIdx.x]);
    }
    if constexpr (sizeof(W) == 8) __syncthreads();
    else if (__syncthreads_or(again || !fits))   // for the pixels that need it: no result depends on what its neighbours hold
    {
        rarely();
        double sums_again[2][4] = {}, total_again[2] = {};
        add_up(sums_again);
        double(*const wide)[PIXELS] = reinterpret_cast<double(*)[PIXELS]>(&part[0][0][0]);   // [GROUPS][PIXELS]
        for (int q = 0; q < 2; q++)
        {
#pragma unroll
            for (int k = 0; k < 4; k++) wide[group][quad_at<VEC, LANES>(lane, k)] = q == 0 ? sums_again[0][k] : sums_again[1][k];
            __syncthreads();
            if (again)
                for (int g = 0; g < GROUPS; g++) total_again[q] += wide[g][threadIdx.x];
            __syncthreads();
        }
        if (again) gradient_factors(total_again[0], total_again[1], per_channel, eps, factors[0][threadIdx.x], factors[1][threadIdx.x]);
        if constexpr (EXACT)
            if (threadIdx.x < PIXELS)
                gradient_factors(again ? total_again[0] : total[0], again ? total_again[1] : total[1], per_channel, eps, exact[0][threadIdx.x], exact[1][threadIdx.x]);
        __syncthreads();
        return false;
    }
    return true;
}

/// Adds squares and products of a quad to sums of type A.
template <typename A, typename W> __device__ __forceinline__ void add_products(A (&sums)[2][4], const W (&v)[4], const W (&up)[4], W g)
{
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        sums[0][k] = fma(static_cast<A>(v[k]), static_cast<A>(v[k]), sums[0][k]);
        sums[1][k] = fma(static_cast<A>(v[k]), static_cast<A>(up[k]) * static_cast<A>(g), sums[1][k]);
    }
}

/// gx of a quad, and the sum over its elements of what they give to gweight; `fit` and `exact` as tile_gradient_factors left them.
template <bool VEC, int LANES, bool EXACT, typename W, int PLACES>
__device__ __forceinline__ W quad_gradient(const W (&v)[4], const W (&up)[4], W g, const W (&r)[4], const W (&pull)[4], bool fit, const double (&exact)[2][PLACES], int lane, W (&gx)[4])
{
    W through = 0;
#pragma unroll
    for (int k = 0; k < 4; k++)
    {
        if constexpr (EXACT)
            if (!fit && !gradients_fit(r[k], pull[k]))
            {
                const int pixel = quad_at<VEC, LANES>(lane, k);
                element_gradient_in_double(v[k], up[k], g, exact[0][pixel], exact[1][pixel], gx[k], through);
                continue;
            }
        element_gradient(v[k], up[k], g, r[k], pull[k], gx[k], through);
    }
    return through;
}

/// Shared memory of the slots of the kernel below.
template <typename T, bool CODES> constexpr size_t gradient_slot_bytes(int held, int threads)
{
    return (2 * sizeof(Quad<T>) + sizeof(typename HeldSum<T, CODES>::Slot)) * static_cast<size_t>(held) * threads;
}

/// Backward, feature maps of up to HELD * WARPS * SPLIT channels. A tile is 128 / SPLIT pixels of an image; SPLIT groups of lanes of a warp have
/// channels of their own, so that a thread block of few warps holds many channels and several of them, which hide each other's barriers, stay
/// resident. Tiles of 32 pixels, read once, against whole ones read twice: (64, 256, 56, 56) 144 us against 170, (64, 512, 28, 28) 97 against
/// 118. Three thread blocks of 4 warps with tiles of 64 pixels against two of 8 with whole ones: (32, 64, 224, 224) 257 us against 268, from codes 219
/// against 245; in half precision, four against two: (64, 32, 112, 112) 48 against 50, from codes 50 against 57. The thread blocks walk over the tiles with
/// gweight's sums in registers; what they have at the end leaves as one row of partial sums, which norm_weight_kernel adds up in a fixed order.
template <typename T, typename G, bool VEC, bool CODES, bool EXACT, int HELD, int WARPS, int SPLIT, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS) rms_norm_columns_backward_kernel(const NormGradArgs a)
{
    using W = Wide<T>;
    using Held = HeldSum<T, CODES>;
    constexpr int COUNT = WARPS * 32, LANES = 32 / SPLIT, PIXELS = CODE_BLOCK / SPLIT, STEP = WARPS * SPLIT;
    static_assert(WARPS * 32 >= PIXELS && HELD <= LANES, "a thread for every pixel of the tile, a lane for every scale");
    __shared__ __align__(8) W part[2][STEP][PIXELS];   // tile_gradient_factors reads it as double as well
    __shared__ W factors[2][PIXELS];
    __shared__ double exact[2][EXACT ? PIXELS : 1];
    extern __shared__ __align__(16) unsigned char slots[];
    Quad<T>* const gy_slot = reinterpret_cast<Quad<T>*>(slots) + threadIdx.x;   // [HELD][threads] each
    Quad<T>* const more_slot = gy_slot + HELD * COUNT;
    typename Held::Slot* const sum_slot = reinterpret_cast<typename Held::Slot*>(slots + 2 * HELD * COUNT * sizeof(Quad<T>)) + threadIdx.x;
    const int C = static_cast<int>(a.channels);
    const int lane = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;   // the group has the channels group, group + STEP, ...
    const int own = (C - group + STEP - 1) / STEP;
    const int64_t step = STEP * a.inner, block_step = STEP * a.tiles_per_row, pieces = (a.inner + PIXELS - 1) / PIXELS, tiles = a.outer * pieces;
    W next_scale = 0;   // lane i: of the group's channel i
    const auto place = [&](int64_t tile) {
        const int64_t image = tile / pieces, pixel = (tile - image * pieces) * PIXELS, row = image * C + group;
        return Place{row * a.inner + pixel + lane_at<VEC>(lane), row * a.tiles_per_row + pixel / CODE_BLOCK,
                     static_cast<int>(min(static_cast<int64_t>(PIXELS), a.inner - pixel)) - lane_at<VEC>(lane)};
    };
    const auto fetch = [&](const Place& p) {
        int64_t at = p.first;
#pragma unroll
        for (int i = 0; i < HELD; i++, at += step)
        {
            Held::template fetch<VEC, LANES>(a, sum_slot + i * COUNT, at, i < own ? p.left : 0);
            fetch_quad<VEC, LANES>(gy_slot + i * COUNT, static_cast<const T*>(a.gy), at, i < own ? p.left : 0);
        }
        if (CODES && lane < min(own, HELD)) next_scale = __ldg(static_cast<const W*>(a.sum_scales) + p.block + lane * block_step);
    };
    const auto fetch_more = [&](const Place& p) {
        if (a.gsum == nullptr) return;
        int64_t at = p.first;
#pragma unroll
        for (int i = 0; i < HELD; i++, at += step) fetch_quad<VEC, LANES>(more_slot + i * COUNT, static_cast<const T*>(a.gsum), at, i < own ? p.left : 0);
    };
    const auto weight_of = [&](int i) { return a.weight == nullptr || i >= own ? W(1) : widen(static_cast<const G*>(a.weight)[group + i * STEP]); };
    W weight_sum[HELD] = {};
    int64_t tile = blockIdx.x;
    Place p = place(tile);
    if (tile < tiles) fetch(p);
    fetch_commit();
    if (tile < tiles) fetch_more(p);
    fetch_commit();
    for (; tile < tiles; tile += gridDim.x)
    {
        fetch_wait<1>();   // gsum may still travel
        Held s[HELD];
        Quad<T> gy[HELD];
#pragma unroll
        for (int i = 0; i < HELD; i++)
        {
            s[i].take(sum_slot[i * COUNT], CODES ? __shfl_sync(0xffffffffu, next_scale, i, LANES) : W(0));
            gy[i] = gy_slot[i * COUNT];
        }
        __syncwarp();
        const Place here = p;
        const bool last = tile + gridDim.x >= tiles;
        if (!last)
        {
            p = place(tile + gridDim.x);
            fetch(p);
        }
        fetch_commit();
        const bool fit = tile_gradient_factors<VEC, LANES, EXACT>(part, factors, exact, a.per_channel, a.eps, lane, group, [&](auto& sums) {
#pragma unroll
            for (int i = 0; i < HELD; i++)
            {
                W v[4], up[4];
                s[i].values(v);
                widen_quad(gy[i], up);
                add_products(sums, v, up, weight_of(i));
            }
        });
        W r[4], pull[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            r[k] = factors[0][quad_at<VEC, LANES>(lane, k)];
            pull[k] = factors[1][quad_at<VEC, LANES>(lane, k)];
        }
        fetch_wait<1>();   // gsum is here, the next tile may travel
        int64_t at = here.first;
#pragma unroll
        for (int i = 0; i < HELD; i++, at += step)
        {
            W v[4], up[4], gx[4];
            s[i].forget_values();
            forget_widened(gy[i]);
            s[i].values(v);
            widen_quad(gy[i], up);
            weight_sum[i] += quad_gradient<VEC, LANES, EXACT>(v, up, weight_of(i), r, pull, fit, exact, lane, gx);
            put_gradient<VEC, LANES, T>(a, gx, more_slot + i * COUNT, at, i < own ? here.left : 0);
        }
        __syncwarp();
        if (!last) fetch_more(p);
        fetch_commit();
    }
    if (a.gweight == nullptr) return;
    W* const partial = static_cast<W*>(a.partial) + static_cast<int64_t>(blockIdx.x) * C;
#pragma unroll
    for (int i = 0; i < HELD; i++)
    {
        const W total = lanes_sum<LANES>(weight_sum[i]);
        if (lane == 0 && i < own) partial[group + i * STEP] = total;
    }
}

/// Backward, feature maps of more channels: the tile is read twice, the second time from L2, HELD of a warp's channels at a time, and gweight's
/// sums live in shared memory.
template <typename T, typename G, bool VEC, bool CODES, bool EXACT, int HELD, int WARPS, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS) rms_norm_columns_twice_backward_kernel(const NormGradArgs a)
{
    using W = Wide<T>;
    static_assert(WARPS >= 4, "a thread for every pixel of the tile");
    __shared__ __align__(8) W part[2][WARPS][CODE_BLOCK];   // tile_gradient_factors reads it as double as well
    __shared__ W factors[2][CODE_BLOCK];
    __shared__ double exact[2][EXACT ? CODE_BLOCK : 1];
    extern __shared__ __align__(16) unsigned char more_shared[];
    W* const weight_sums = reinterpret_cast<W*>(more_shared);   // [channels]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, C = static_cast<int>(a.channels);
    const int own = (C - warp + WARPS - 1) / WARPS;   // channels of this warp
    const int64_t step = WARPS * a.inner, block_step = WARPS * a.tiles_per_row;
    if (a.gweight != nullptr)
        for (int c = threadIdx.x; c < C; c += WARPS * 32) weight_sums[c] = W(0);
    const auto weight_of = [&](int i) { return a.weight == nullptr || i >= own ? W(1) : widen(static_cast<const G*>(a.weight)[warp + i * WARPS]); };
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const Place p = place_of<VEC>(a, tile, lane, warp);
        HeldSum<T, CODES> s[HELD];
        Quad<T> gy[HELD];
        const auto load = [&](int i0) {
            int64_t at = p.first + i0 * step, block = p.block + i0 * block_step;
#pragma unroll
            for (int i = 0; i < HELD; i++, at += step, block += block_step)
            {
                s[i].template load<VEC>(a, at, block, i0 + i < own ? p.left : 0, i0 + i < own);
                gy[i] = load_quad<VEC>(static_cast<const T*>(a.gy) + at, i0 + i < own ? p.left : 0);
            }
        };
        const bool fit = tile_gradient_factors<VEC, 32, EXACT>(part, factors, exact, a.per_channel, a.eps, lane, warp, [&](auto& sums) {
            for (int i0 = 0; i0 < own; i0 += HELD)
            {
                load(i0);
#pragma unroll
                for (int i = 0; i < HELD; i++)
                {
                    W v[4], up[4];
                    s[i].values(v);
                    widen_quad(gy[i], up);
                    add_products(sums, v, up, weight_of(i0 + i));
                }
            }
        });
        W r[4], pull[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
        {
            r[k] = factors[0][quad_at<VEC>(lane, k)];
            pull[k] = factors[1][quad_at<VEC>(lane, k)];
        }
        for (int i0 = 0; i0 < own; i0 += HELD)
        {
            load(i0);
            Quad<T> more[HELD];
            int64_t at = p.first + i0 * step;
            if (a.gsum != nullptr)
            {
                const T* src = static_cast<const T*>(a.gsum) + at;
#pragma unroll
                for (int i = 0; i < HELD; i++, src += step) more[i] = load_quad<VEC>(src, i0 + i < own ? p.left : 0);
            }
#pragma unroll
            for (int i = 0; i < HELD; i++, at += step)
            {
                W v[4], up[4], gx[4];
                s[i].values(v);
                widen_quad(gy[i], up);
                const W through = quad_gradient<VEC, 32, EXACT>(v, up, weight_of(i0 + i), r, pull, fit, exact, lane, gx);
                if (a.gweight != nullptr)
                {
                    const W total = warp_sum(through);
                    if (lane == 0 && i0 + i < own) weight_sums[warp + (i0 + i) * WARPS] += total;   // the channel belongs to this warp alone
                }
                put_gradient<VEC, 32, T>(a, gx, more + i, at, i0 + i < own ? p.left : 0);
            }
        }
    }
    if (a.gweight == nullptr) return;
    W* const partial = static_cast<W*>(a.partial) + static_cast<int64_t>(blockIdx.x) * C;
    __syncwarp();
    for (int c = warp; c < C; c += WARPS)
        if (lane == 0) partial[c] = weight_sums[c];
}

/// Backward, rows of channels; what a warp takes next is fetched while this is computed (AHEAD: where the slots fit shared memory). gweight's
/// sums stay in the lanes that have the channels; the groups of a thread block add theirs up in shared memory, one after the other, at the end.
template <typename T, typename G, bool VEC, bool CODES, bool EXACT, bool AHEAD, int ROWS, int BLOCKS, int WARPS, int CTAS>
__global__ void __launch_bounds__(WARPS * 32, CTAS) rms_norm_rows_backward_kernel(const NormGradArgs a, int shift)
{
    using W = Wide<T>;
    using Held = HeldSum<T, CODES>;
    constexpr int COUNT = WARPS * 32, N = ROWS * BLOCKS;
    __shared__ double part[2][WARPS][2];
    __shared__ double exact[EXACT ? WARPS : 1][ROWS][2];   // r and the pull of a warp's rows, where float does not hold them
    extern __shared__ __align__(16) unsigned char slots[];
    Quad<T>* const gy_slot = reinterpret_cast<Quad<T>*>(slots) + threadIdx.x;   // [N][threads] each
    Quad<T>* const more_slot = gy_slot + N * COUNT;
    typename Held::Slot* const sum_slot = reinterpret_cast<typename Held::Slot*>(slots + 2 * N * COUNT * sizeof(Quad<T>)) + threadIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = WARPS >> shift;
    const RowTile<VEC, ROWS, BLOCKS> t(a.channels, a.tiles_per_row, shift, lane, warp);
    const auto rows_from = [&](int64_t row) { return static_cast<int>(max(int64_t(0), min(static_cast<int64_t>(ROWS), a.outer - row))); };
    const auto block_of = [&](int64_t row, int q) { return row * a.tiles_per_row + (t.c0 - t.at) / CODE_BLOCK + (static_cast<int64_t>(q) << shift); };
    W next_scale = 0;   // lane q: of quad q
    const auto fetch = [&](int64_t row) {
        const int rows = rows_from(row);
        const int64_t first = row * t.C + t.c0;
#pragma unroll
        for (int q = 0; q < N; q++)
        {
            Held::template fetch<VEC>(a, sum_slot + q * COUNT, first + t.offset(q), t.left(q, rows));
            fetch_quad<VEC>(gy_slot + q * COUNT, static_cast<const T*>(a.gy), first + t.offset(q), t.left(q, rows));
        }
        if (CODES && rows > 0 && lane < min(t.count(rows), N)) next_scale = __ldg(static_cast<const W*>(a.sum_scales) + block_of(row, lane));
    };
    const auto fetch_more = [&](int64_t row) {
        if (a.gsum == nullptr) return;
        const int rows = rows_from(row);
#pragma unroll
        for (int q = 0; q < N; q++) fetch_quad<VEC>(more_slot + q * COUNT, static_cast<const T*>(a.gsum), row * t.C + t.c0 + t.offset(q), t.left(q, rows));
    };
    const auto weights_of = [&](int j, W (&g)[4]) {
        if (a.weight != nullptr) widen_quad(load_quad<VEC>(static_cast<const G*>(a.weight) + t.c0 + j * t.step, t.left_in(j)), g);
        else
#pragma unroll
            for (int k = 0; k < 4; k++) g[k] = W(1);
    };
    const int64_t stride = static_cast<int64_t>(gridDim.x) * groups * ROWS;
    int64_t row = (static_cast<int64_t>(blockIdx.x) * groups + (warp >> shift)) * ROWS;
    int turn = 0;
    if (AHEAD)
    {
        fetch(row);
        fetch_commit();
        fetch_more(row);
        fetch_commit();
    }
    W weight_sum[BLOCKS][4] = {};
    for (; row < a.outer; row += stride)
    {
        const int rows = rows_from(row), count = t.count(rows);
        const int64_t first = row * t.C + t.c0;
        Held s[N];
        Quad<T> gy[N];
        if (AHEAD)
        {
            fetch_wait<1>();   // gsum may still travel
#pragma unroll
            for (int q = 0; q < N; q++)
            {
                s[q].take(sum_slot[q * COUNT], CODES ? __shfl_sync(0xffffffffu, next_scale, q) : W(0));
                gy[q] = gy_slot[q * COUNT];
            }
            __syncwarp();
            fetch(row + stride);
            fetch_commit();
        }
        else
#pragma unroll
            for (int q = 0; q < N; q++)
            {
                s[q].template load<VEC>(a, first + t.offset(q), block_of(row, q), t.left(q, rows), q < count);
                gy[q] = load_quad<VEC>(static_cast<const T*>(a.gy) + first + t.offset(q), t.left(q, rows));
            }
        const auto add_up = [&](auto zero, double (&total)[2]) {   // squares and products of row lane % ROWS
            using A = decltype(zero);
            A squares[ROWS] = {}, products[ROWS] = {};
            W g[4];
#pragma unroll
            for (int q = 0; q < N; q++)
            {
                W v[4], up[4];
                s[q].values(v);
                widen_quad(gy[q], up);
                if (BLOCKS > 1 || q == 0) weights_of(q % BLOCKS, g);
#pragma unroll
                for (int k = 0; k < 4; k++)
                {
                    squares[q / BLOCKS] = fma(static_cast<A>(v[k]), static_cast<A>(v[k]), squares[q / BLOCKS]);
                    products[q / BLOCKS] = fma(static_cast<A>(v[k]), static_cast<A>(up[k]) * static_cast<A>(g[k]), products[q / BLOCKS]);
                }
            }
            total[0] = static_cast<double>(spread_sums(squares, lane));
            total[1] = static_cast<double>(spread_sums(products, lane));
            share_sums(total, part, turn, shift);
        };
        double total[2];
        add_up(W(0), total);
        W r, pull;
        bool fit = true;
        const bool again = sizeof(W) == 4 && out_of_range(total[0], total[1], a.eps);   // the warps that share a row agree
        if constexpr (EXACT)
        {
            gradient_factors(total[0], total[1], a.per_channel, a.eps, r, pull);
            fit = __all_sync(0xffffffffu, gradients_fit(r, pull));
        }
        if (__any_sync(0xffffffffu, again))
        {
            rarely();
            double sums_again[2];
            add_up(0.0, sums_again);
            if (again)
            {
                total[0] = sums_again[0];
                total[1] = sums_again[1];
            }
        }
        gradient_factors(total[0], total[1], a.per_channel, a.eps, r, pull);
        if constexpr (EXACT)
            if (!fit)
            {
                __syncwarp();   // the previous rows' have been read
                if (lane < ROWS) gradient_factors(total[0], total[1], a.per_channel, a.eps, exact[warp][lane][0], exact[warp][lane][1]);
                __syncwarp();
            }
        if (AHEAD) fetch_wait<1>();   // gsum is here, the next rows may travel
        W g[4];
#pragma unroll
        for (int q = 0; q < N; q++)
        {
            if (q >= count) break;
            Quad<T> more;
            if (a.gsum != nullptr) more = AHEAD ? more_slot[q * COUNT] : load_quad<VEC>(static_cast<const T*>(a.gsum) + first + t.offset(q), t.left(q, rows));
            W v[4], up[4], gx[4];
            s[q].forget_values();
            forget_widened(gy[q]);
            s[q].values(v);
            widen_quad(gy[q], up);
            if (BLOCKS > 1 || q == 0) weights_of(q % BLOCKS, g);
            const W r_row = ROWS == 1 ? r : __shfl_sync(0xffffffffu, r, q / BLOCKS), pull_row = ROWS == 1 ? pull : __shfl_sync(0xffffffffu, pull, q / BLOCKS);
#pragma unroll
            for (int k = 0; k < 4; k++)
            {
                if constexpr (EXACT)
                    if (!fit && !gradients_fit(r_row, pull_row))
                    {
                        element_gradient_in_double(v[k], up[k], g[k], exact[warp][q / BLOCKS][0], exact[warp][q / BLOCKS][1], gx[k], weight_sum[q % BLOCKS][k]);
                        continue;
                    }
                element_gradient(v[k], up[k], g[k], r_row, pull_row, gx[k], weight_sum[q % BLOCKS][k]);
            }
            put_gradient<VEC, 32, T>(a, gx, &more, first + t.offset(q), t.left(q, rows));
        }
        if (AHEAD)
        {
            __syncwarp();
            fetch_more(row + stride);
            fetch_commit();
        }
    }
    if (a.gweight == nullptr) return;
    if (AHEAD) fetch_wait<0>();   // nothing lands in what follows
    __syncthreads();
    W* const weight_sums = reinterpret_cast<W*>(slots);   // [channels]
    for (int n = 0; n < groups; n++)
    {
        if (warp >> shift == n)
#pragma unroll
            for (int j = 0; j < BLOCKS; j++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                {
                    const int c = t.c0 - t.at + j * t.step + quad_at<VEC>(lane, k);
                    if (j < t.own && c < t.C) weight_sums[c] = (n == 0 ? W(0) : weight_sums[c]) + weight_sum[j][k];
                }
        __syncthreads();
    }
    W* const partial = static_cast<W*>(a.partial) + static_cast<int64_t>(blockIdx.x) * t.C;
    for (int c = threadIdx.x; c < t.C; c += WARPS * 32) partial[c] = weight_sums[c];
}

/// gweight from the rows of partial sums, in double and in a fixed order: a thread block takes 32 channels and its 32 warps every 32nd row, many
/// of which (592 rows at most) are in flight at once. 7.1 us with 8 warps on 444 rows of 512 channels, 4.3 us so.
constexpr int WEIGHT_WARPS = 32;
template <typename G>
__global__ void __launch_bounds__(WEIGHT_WARPS * 32) norm_weight_kernel(const Wide<G>* __restrict__ partial, G* __restrict__ gweight, int64_t channels, int rows)
{
    __shared__ double part[WEIGHT_WARPS][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    double sum = 0.0;
    if (c < channels)
#pragma unroll 10
        for (int row = warp; row < rows; row += WEIGHT_WARPS) sum += static_cast<double>(__ldg(partial + row * channels + c));
    part[warp][lane] = sum;
    __syncthreads();
    const int64_t mine = static_cast<int64_t>(blockIdx.x) * 32 + warp;   // warp w adds up channel w of the thread block
    const double total = warp_sum(part[lane][warp]);
    if (lane == 0 && mine < channels) gweight[mine] = narrow<G>(static_cast<Wide<G>>(total));
}

}  // namespace mc
