// Per-channel dilation / erosion (identity merge) with its input kept in 8 bits: the forward pass that also writes the input's codes, and the
// backward pass that reads them. Float, square 3 x 3 and 5 x 5 structuring elements, rows of whole quads (W a multiple of four).
//
//     forward   y[h, w] = ext_k ( x[h + R - kh, w + R - kw] + w_k ),  codes and scales of x (mc_encode8)
//     backward  win[h, w] = first k that attains the extremum at the values of the codes;
//               gx[q] = sum of gy over the outputs whose winner reads q,  gw[k] = sum of gy over the outputs with winner k
//
// Nine or twenty-five taps a pixel are little arithmetic for the nine bytes that a pixel moves each way, so both passes are laid out to touch
// memory once: the forward pass takes runs of 2048 consecutive pixels of a plane, which are also whole blocks of codes, and stages them
// with the rows above and below; the backward pass walks down strips of rows with the codes' values, and the gradients under construction,
// in registers. No atomics: every sum is taken in one order.
// MEASURED
#pragma once
#include "encode8.cuh"
#include "tma.cuh"

namespace mc
{

struct Identity8Args
{
    const float* x;        // forward
    const float* w;        // [C, K, K], or one such per image
    const float* gy;       // backward
    float* y;              // forward: output; backward: gx
    int8_t* codes;
    float* scales;
    float* partial;        // backward: [C, taps, parts]
    int64_t weight_batch_stride;
    int64_t plane_blocks;  // blocks of codes of a plane
    int C, H, W;
    int chunks;            // forward: runs of a plane
    int strip_rows, strips, column_tiles, parts;   // backward
    int64_t units;         // backward: strips of all planes
    float fill;
    bool replicate, flipped;
};

constexpr int RUN = 2048;   // pixels a thread block of the forward kernel computes

/// Floats of shared memory of the forward kernel: the run with the rows that its taps reach and a quad on either side.
constexpr size_t identity8_shared(int K, int W) { return sizeof(float) * (RUN + 2 * (static_cast<size_t>(K / 2) * W + 4)); }

template <bool IS_MIN, int K>
__device__ __forceinline__ void load_element(const Identity8Args& a, int image, int channel, float (&w)[K * K])
{
    const float* from = a.w + image * a.weight_batch_stride + static_cast<int64_t>(channel) * (K * K);
#pragma unroll
    for (int k = 0; k < K * K; k++)
    {
        const float v = __ldg(from + (a.flipped ? K * K - 1 - k : k));
        w[k] = IS_MIN ? -v : v;
    }
}

template <bool IS_MIN, int K> __global__ void __launch_bounds__(THREADS) identity_forward8_kernel(const Identity8Args a)
{
    constexpr int R = K / 2;
    extern __shared__ __align__(16) float staged[];
    const int plane = blockIdx.x / a.chunks, chunk = blockIdx.x - plane * a.chunks, image = plane / a.C, channel = plane - image * a.C;
    const int pixels = a.H * a.W, first = chunk * RUN, last = min(first + RUN, pixels);
    const int64_t base = static_cast<int64_t>(plane) * pixels;
    const int low = first - R * a.W - 4;   // what staged[0] is
    for (int e = low + 4 * static_cast<int>(threadIdx.x); e < last + R * a.W + 4; e += 4 * THREADS)
        if (e >= 0 && e < pixels) cp_async_16(staged + (e - low), a.x + base + e);
    float w[K * K];
    load_element<IS_MIN, K>(a, image, channel, w);
    cp_async_wait_all();
    __syncthreads();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int QUADS = RUN / (4 * THREADS);
    float center[QUADS][4];
    int left[QUADS];
#pragma unroll
    for (int q = 0; q < QUADS; q++)
    {
        const int p = first + (q * (THREADS / 32) + warp) * CODE_BLOCK + 4 * lane;   // the warp's quads are a block of codes
        left[q] = pixels - p;
#pragma unroll
        for (int k = 0; k < 4; k++) center[q][k] = 0.0f;
        if (left[q] <= 0) continue;
        const int row = p / a.W, col = p - row * a.W;
        float best[4];
#pragma unroll
        for (int j = 0; j < 4; j++) best[j] = IS_MIN ? Limits<float>::inf() : -Limits<float>::inf();
#pragma unroll
        for (int dy = -R; dy <= R; dy++)
        {
            const int r = row + dy, inside = min(max(r, 0), a.H - 1);
            const float* from = staged + (inside * a.W + col - low);
            float seg[4 + 2 * R];   // columns col - R .. col + 3 + R
            if (a.replicate || r == inside)
            {
                const float4 mid = *reinterpret_cast<const float4*>(from);
                seg[R] = mid.x; seg[R + 1] = mid.y; seg[R + 2] = mid.z; seg[R + 3] = mid.w;
#pragma unroll
                for (int i = 0; i < R; i++)
                {
                    seg[i] = col > 0 ? from[i - R] : (a.replicate ? mid.x : a.fill);
                    seg[R + 4 + i] = col + 4 < a.W ? from[4 + i] : (a.replicate ? mid.w : a.fill);
                }
                if (dy == 0)
                {
                    center[q][0] = mid.x; center[q][1] = mid.y; center[q][2] = mid.z; center[q][3] = mid.w;
                }
            }
            else
#pragma unroll
                for (int i = 0; i < 4 + 2 * R; i++) seg[i] = a.fill;
            // Tap kh reads row + R - kh, tap kw column + R - kw.
            const int kh = R - dy;
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
#pragma unroll
                for (int kw = 0; kw + 1 < K; kw += 2)
                    best[j] = ext3<IS_MIN>(best[j], seg[j + K - 1 - kw] + w[kh * K + kw], seg[j + K - 2 - kw] + w[kh * K + kw + 1]);
                best[j] = ext2<IS_MIN>(best[j], seg[j] + w[kh * K + K - 1]);
            }
        }
        *reinterpret_cast<float4*>(a.y + base + p) = make_float4(best[0], best[1], best[2], best[3]);
    }
    if (a.codes == nullptr) return;
    uint32_t codes[QUADS];
    const float scale = encode_blocks(center, codes, lane);
#pragma unroll
    for (int q = 0; q < QUADS; q++)
    {
        const int block = q * (THREADS / 32) + warp;
        store_codes<true>(a.codes + base + first + block * CODE_BLOCK + 4 * lane, codes[q], left[q]);
        if (lane == q && first + block * CODE_BLOCK < pixels) a.scales[plane * a.plane_blocks + first / CODE_BLOCK + block] = scale;
    }
}

/// Columns of a strip: up to 128 if that is the whole width, else 120 of the strip's own between a quad on either side whose outputs are computed
/// for what they give to their neighbours.
__host__ __device__ constexpr int strip_columns(int W) { return W <= 128 ? 128 : 120; }

/// Lanes that share a row of a strip: narrow images put several strips into a warp.
__host__ __device__ constexpr int strip_lanes(int W) { return W <= 32 ? 8 : W <= 64 ? 16 : 32; }

/// A lane has four neighbouring columns and walks down the rows; a row of outputs needs the 2 R + 1 rows around it and gives to them. The columns on
/// either side come from, and go to, the neighbouring lanes. Of the K * K candidates of a pixel the first that equals their extremum wins, as
/// in the reference's scan (csrc/cpp/morpho_op_cpu_kernels.hxx:212-252): NaN never does, and where nothing beats the initial infinity tap 0 does.
template <bool IS_MIN, int K, int CTAS> __global__ void __launch_bounds__(128, CTAS) identity_backward8_kernel(const Identity8Args a)
{
    constexpr int R = K / 2, COLS = 4 + 2 * R;
    const int lanes = strip_lanes(a.W), lane = threadIdx.x & 31, sub = lane & (lanes - 1);
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5)) * (32 / lanes) + lane / lanes;
    const bool live = unit < a.units;   // the lanes of a strip without work go along, with zeros
    const int64_t u = live ? unit : 0;
    const int strip = static_cast<int>(u % a.strips), tile = static_cast<int>(u / a.strips % a.column_tiles);
    const int plane = static_cast<int>(u / a.strips / a.column_tiles), image = plane / a.C, channel = plane - image * a.C;
    const int row0 = strip * a.strip_rows, row1 = min(row0 + a.strip_rows, a.H);   // input rows, and outputs for gw, of this strip
    const bool whole = a.W <= 128;
    const int col = (whole ? 0 : tile * strip_columns(a.W) - 4) + 4 * sub;         // the lane's first column; -4 in a first halo
    const bool own = live && col >= 0 && col < a.W && (whole || (sub > 0 && sub < 31));
    const bool exists = live && col >= 0 && col < a.W;
    const int64_t pixels = static_cast<int64_t>(a.H) * a.W, base = plane * pixels;
    const int from_col = min(max(col, 0), a.W - 4);

    float w[K * K], through[K * K];
    load_element<IS_MIN, K>(a, image, channel, w);
#pragma unroll
    for (int k = 0; k < K * K; k++) through[k] = 0.0f;

    // A row of the input as it is read: four codes and the scale of their block; the edge pixel, or the fill, outside the image.
    struct Row
    {
        uint32_t codes;
        float scale;
    };
    const auto fetch = [&](int r) {
        const int64_t at = static_cast<int64_t>(min(max(r, 0), a.H - 1)) * a.W + from_col;
        return Row{__ldg(reinterpret_cast<const unsigned int*>(a.codes + base + at)), __ldg(a.scales + plane * a.plane_blocks + at / CODE_BLOCK)};
    };
    const auto fetch_grad = [&](int h) {
        return exists && h >= 0 && h < a.H ? __ldg(reinterpret_cast<const float4*>(a.gy + base + static_cast<int64_t>(h) * a.W + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    const auto open_row = [&](const Row& row, int r, float (&seg)[COLS]) {
        float v[4];
        decode_quad(row.codes, row.scale, v);
        const bool in_row = r >= 0 && r < a.H;
        // Beyond either end of the row: its edge pixel, or the fill.
#pragma unroll
        for (int j = 0; j < 4; j++)
        {
            float value = col < 0 ? v[0] : col > a.W - 4 ? v[3] : v[j];
            if (!a.replicate && (!in_row || col < 0 || col > a.W - 4)) value = a.fill;
            seg[R + j] = value;
        }
        // A whole width has no lanes beyond its ends where it fills its lanes: the edge pixel is the lane's own.
        const float before = a.replicate ? seg[R] : a.fill, after = a.replicate ? seg[R + 3] : a.fill;
#pragma unroll
        for (int i = 0; i < R; i++)
        {
            const float l = __shfl_up_sync(0xffffffffu, seg[R + 4 - R + i], 1, lanes), n = __shfl_down_sync(0xffffffffu, seg[R + i], 1, lanes);
            seg[i] = sub > 0 && !(whole && col == 0) ? l : before;
            seg[R + 4 + i] = sub < lanes - 1 ? n : after;
        }
    };

    float X[K][COLS], acc[K][COLS];   // input rows h - R .. h + R; gradients of the same rows
#pragma unroll
    for (int i = 0; i < K; i++)
#pragma unroll
        for (int c = 0; c < COLS; c++) acc[i][c] = 0.0f;
    // Outputs row0 - R .. row1 - 1 + R: those beyond the strip only for the rows of gx that they give to.
    const int h_first = row0 - R, h_last = row1 - 1 + R;
#pragma unroll
    for (int i = 1; i < K; i++) open_row(fetch(h_first - R + i - 1), h_first - R + i - 1, X[i]);
    Row next = fetch(h_first + R);
    float4 grad = fetch_grad(h_first);
    // The strips of a warp are of one length but for the last of a plane; all lanes go as far as the longest.
    const int steps = a.strip_rows + 2 * R;
    for (int step = 0; step < steps; step++)
    {
        const int h = h_first + step;
#pragma unroll
        for (int i = 0; i + 1 < K; i++)
#pragma unroll
            for (int c = 0; c < COLS; c++)
            {
                X[i][c] = X[i + 1][c];
                acc[i][c] = acc[i + 1][c];
            }
        open_row(next, h + R, X[K - 1]);
#pragma unroll
        for (int c = 0; c < COLS; c++) acc[K - 1][c] = 0.0f;
        const float4 here = grad;
        next = fetch(h + R + 1);
        grad = step + 1 < steps ? fetch_grad(h + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float g4[4] = {here.x, here.y, here.z, here.w};
        const bool counts = own && h >= row0 && h < row1;   // for gw: every output once
        if (h <= h_last)
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                float v[K * K];
                float m = IS_MIN ? Limits<float>::inf() : -Limits<float>::inf();
#pragma unroll
                for (int k = 0; k < K * K; k++) v[k] = X[K - 1 - k / K][j + K - 1 - k % K] + w[k];   // row h + R - kh, column col + j + R - kw
#pragma unroll
                for (int k = 0; k + 1 < K * K; k += 2) m = ext3<IS_MIN>(m, v[k], v[k + 1]);
                m = ext2<IS_MIN>(m, v[K * K - 1]);
                const float g = g4[j], gc = counts ? g : 0.0f;
                bool open = true;
#pragma unroll
                for (int k = 0; k < K * K; k++)
                {
                    const bool wins = open && (v[k] == m || (k == 0 && m == (IS_MIN ? Limits<float>::inf() : -Limits<float>::inf())));
                    if (wins)
                    {
                        acc[K - 1 - k / K][j + K - 1 - k % K] += g;
                        through[k] += gc;
                    }
                    open = open && !wins;
                }
            }
        // Row h - R has all that it will get from this strip's outputs.
        const int r = h - R;
        float sum[4];
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] = acc[0][R + j];
#pragma unroll
        for (int i = 0; i < R; i++)
        {
            const float l = __shfl_up_sync(0xffffffffu, acc[0][R + 4 + i], 1, lanes), n = __shfl_down_sync(0xffffffffu, acc[0][i], 1, lanes);
            if (sub > 0) sum[i] += l;
            if (sub < lanes - 1) sum[4 - R + i] += n;
        }
        if (own && r >= row0 && r < row1)
            *reinterpret_cast<float4*>(a.y + base + static_cast<int64_t>(r) * a.W + col) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }

    // gw: the strip's lanes, in one order; strips are added up by identity_weight8_kernel.
#pragma unroll
    for (int k = 0; k < K * K; k++)
    {
        float total = through[k];
        for (int d = lanes / 2; d > 0; d /= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
        if (live && sub == 0) a.partial[(static_cast<int64_t>(channel) * (K * K) + k) * a.parts + (image * a.column_tiles + tile) * a.strips + strip] = total;
    }
}

/// gw of a channel's tap from its parts, one warp each, in double and in a fixed order.
static __global__ void __launch_bounds__(THREADS) identity_weight8_kernel(const float* __restrict__ partial, float* __restrict__ gw, int count, int taps, int parts, float sign,
                                                                         bool flipped)
{
    const int lane = threadIdx.x & 31, at = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    if (at >= count) return;
    double sum = 0.0;
    for (int p = lane; p < parts; p += 32) sum += static_cast<double>(__ldg(partial + static_cast<int64_t>(at) * parts + p));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const int channel = at / taps, k = at - channel * taps;
    if (lane == 0) gw[channel * taps + (flipped ? taps - 1 - k : k)] = sign * static_cast<float>(sum);
}

}  // namespace mc
