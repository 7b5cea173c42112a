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
// Measured, (16, 64, 112, 112): forward 34 us at 3 x 3 and 53 at 5 x 5, backward 63 and 137; the bytes alone are 18 us each way. The forward pass is
// bound by its staging (a wave of loads, a barrier, then arithmetic), the backward pass by the half-rate pipe of comparisons, selects and
// extrema (64 % busy at 96 instructions a pixel). The separate kernels took 75 + 13 us and 257 + 12 + 11 at 3 x 3.
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
    int chunks, run_step;  // forward: runs of a plane; 4 * THREADS modulo W
    int strip_rows, strips, column_tiles, parts;   // backward
    int64_t units;         // backward: strips of all planes
    float fill;
    bool replicate, flipped;
};

/// Warps, each a thread block, of the backward kernel that are resident on an SM.
constexpr int BACKWARD_WARPS_3 = 20, BACKWARD_WARPS_5 = 8;

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

/// The rows beyond the image are resolved where they are staged, so that a pixel's taps are K runs of the staged pixels, W apart; the columns
/// beyond a row's ends where they are used.
template <bool IS_MIN, int K> __global__ void __launch_bounds__(THREADS) identity_forward8_kernel(const Identity8Args a)
{
    constexpr int R = K / 2;
    extern __shared__ __align__(16) float staged[];
    const int plane = blockIdx.x / a.chunks, chunk = blockIdx.x - plane * a.chunks, image = plane / a.C, channel = plane - image * a.C;
    const int pixels = a.H * a.W, first = chunk * RUN, last = min(first + RUN, pixels);
    const int64_t base = static_cast<int64_t>(plane) * pixels;
    const int low = first - R * a.W - 4;   // what staged[0] is
    for (int e = low + 4 * static_cast<int>(threadIdx.x); e < last + R * a.W + 4; e += 4 * THREADS)
    {
        int from = e;
        if (e < 0 || e >= pixels)
        {
            if (!a.replicate)
            {
                *reinterpret_cast<float4*>(staged + (e - low)) = make_float4(a.fill, a.fill, a.fill, a.fill);
                continue;
            }
            while (from < 0) from += a.W;
            while (from >= pixels) from -= a.W;
        }
        cp_async_16(staged + (e - low), a.x + base + from);
    }
    float w[K * K];
    load_element<IS_MIN, K>(a, image, channel, w);
    cp_async_wait_all();
    __syncthreads();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int QUADS = RUN / (4 * THREADS);
    float center[QUADS][4];
    int left[QUADS], p = first + warp * CODE_BLOCK + 4 * lane, col = p % a.W;   // the warp's quads are a block of codes
#pragma unroll
    for (int q = 0; q < QUADS; q++, p += 4 * THREADS)
    {
        left[q] = pixels - p;
#pragma unroll
        for (int k = 0; k < 4; k++) center[q][k] = 0.0f;
        if (left[q] > 0)
        {
            const bool at_start = col == 0, at_end = col + 4 >= a.W;
            const float* from = staged + (p - low - R * a.W);
            float best[4];
#pragma unroll
            for (int j = 0; j < 4; j++) best[j] = IS_MIN ? Limits<float>::inf() : -Limits<float>::inf();
#pragma unroll
            for (int r = 0; r < K; r++, from += a.W)
            {
                float seg[4 + 2 * R];   // columns col - R .. col + 3 + R of row h - R + r
                const float4 mid = *reinterpret_cast<const float4*>(from);
                seg[R] = mid.x; seg[R + 1] = mid.y; seg[R + 2] = mid.z; seg[R + 3] = mid.w;
                const float before = a.replicate ? mid.x : a.fill, after = a.replicate ? mid.w : a.fill;
#pragma unroll
                for (int i = 0; i < R; i++)
                {
                    const float l = from[i - R], n = from[4 + i];   // of another row at a row's ends
                    seg[i] = at_start ? before : l;
                    seg[R + 4 + i] = at_end ? after : n;
                }
                if (r == R)
#pragma unroll
                    for (int k = 0; k < 4; k++) center[q][k] = seg[R + k];
                // Tap (kh, kw) reads row h + R - kh, column col + j + R - kw.
                const float* taps = w + (K - 1 - r) * K;
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
#pragma unroll
                    for (int kw = 0; kw + 1 < K; kw += 2)
                        best[j] = ext3<IS_MIN>(best[j], seg[j + K - 1 - kw] + taps[kw], seg[j + K - 2 - kw] + taps[kw + 1]);
                    best[j] = ext2<IS_MIN>(best[j], seg[j] + taps[K - 1]);
                }
            }
            *reinterpret_cast<float4*>(a.y + base + p) = make_float4(best[0], best[1], best[2], best[3]);
        }
        col += a.run_step;   // 4 * THREADS pixels on, less whole rows
        if (col >= a.W) col -= a.W;
    }
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

/// Shared memory by address, without barriers: every lane has words of its own, and its accesses stay in order.
__device__ __forceinline__ float shared_word(uint32_t address)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(address));
    return v;
}
__device__ __forceinline__ void set_shared_word(uint32_t address, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(address), "f"(v) : "memory"); }

/// A lane has four neighbouring columns and walks down the rows; a row of outputs needs the 2 R + 1 rows around it, which stay in registers, and
/// gives to them. The columns on either side come from, and go to, the neighbouring lanes. Of the K * K candidates of a pixel the first
/// that equals their extremum wins, as in the reference's scan (csrc/cpp/morpho_op_cpu_kernels.hxx:212-252): NaN never does, and where
/// nothing beats the initial infinity tap 0 does. What the selects pick is the byte offset (kh * COLS + kw) * 128 of the winner, which leads both
/// to its word among the rows of gx under construction, a ring of K rows, and to its bin of gw: [slot][lane], so that no bank is hit twice
/// and no atomic is needed. (Adding to registers under a predicate a tap instead took 78 us where this takes 70; the selects and comparisons,
/// which issue at half rate, are what bounds it.)
template <bool IS_MIN, int K, int WARPS> __global__ void __launch_bounds__(32, WARPS) identity_backward8_kernel(const Identity8Args a)
{
    constexpr int R = K / 2, COLS = 4 + 2 * R, TAPS = K * K;
    __shared__ float sums[K * COLS + K * COLS][32];   // [rows of gx under construction][columns][lane]; [bins: kh * COLS + kw][lane]
    const int lanes = strip_lanes(a.W), lane = threadIdx.x & 31, sub = lane & (lanes - 1);
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (32 / lanes) + lane / lanes;
    const bool live = unit < a.units;   // the lanes of a strip without work go along, with zeros
    const int64_t u = live ? unit : 0;
    const int strip = static_cast<int>(u % a.strips), tile = static_cast<int>(u / a.strips % a.column_tiles);
    const int plane = static_cast<int>(u / a.strips / a.column_tiles), image = plane / a.C, channel = plane - image * a.C;
    const int row0 = strip * a.strip_rows, row1 = min(row0 + a.strip_rows, a.H);   // input rows, and outputs for gw, of this strip
    const bool whole = a.W <= 128;
    const int col = (whole ? 0 : tile * strip_columns(a.W) - 4) + 4 * sub;         // the lane's first column; -4 in a first halo
    const bool exists = live && col >= 0 && col < a.W, own = exists && (whole || (sub > 0 && sub < 31));
    const int64_t pixels = static_cast<int64_t>(a.H) * a.W, base = plane * pixels;
    const int from_col = min(max(col, 0), a.W - 4);
    const int8_t* const codes = a.codes + base + from_col;
    const float* const scales = a.scales + plane * a.plane_blocks;
    const float* const gy = a.gy + base + from_col;
    float w[TAPS];
    load_element<IS_MIN, K>(a, image, channel, w);
    for (int i = 0; i < 2 * K * COLS; i++) sums[i][lane] = 0.0f;
    const uint32_t acc_base = smem_addr(&sums[0][lane]), bin_base = smem_addr(&sums[K * COLS][lane]);
    // A row of the input as it is read: four codes and the scale of their block; the edge pixel, or the fill, outside the image.
    struct Row
    {
        uint32_t codes;
        float scale;
    };
    const auto fetch = [&](int r) {
        const int at = min(max(r, 0), a.H - 1) * a.W;
        return Row{__ldg(reinterpret_cast<const unsigned int*>(codes + at)), __ldg(scales + static_cast<unsigned>(at + from_col) / CODE_BLOCK)};
    };
    const auto fetch_grad = [&](int h) {
        return exists && h >= 0 && h < a.H ? __ldg(reinterpret_cast<const float4*>(gy + h * a.W)) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    const bool before_row = col < 0, after_row = col > a.W - 4;
    const auto open_row = [&](const Row& row, int r, float (&seg)[COLS]) {
        float v[4];
        decode_quad(row.codes, row.scale, v);
        // Beyond either end of the row: its edge pixel, or the fill.
        const bool filled = !a.replicate && (r < 0 || r >= a.H || before_row || after_row);
#pragma unroll
        for (int j = 0; j < 4; j++) seg[R + j] = filled ? a.fill : before_row ? v[0] : after_row ? v[3] : v[j];
        const float before = a.replicate ? seg[R] : a.fill, after = a.replicate ? seg[R + 3] : a.fill;
#pragma unroll
        for (int i = 0; i < R; i++)
        {
            const float l = __shfl_up_sync(0xffffffffu, seg[4 + i], 1, lanes), n = __shfl_down_sync(0xffffffffu, seg[R + i], 1, lanes);
            seg[i] = sub > 0 ? l : before;
            seg[R + 4 + i] = sub < lanes - 1 ? n : after;
        }
    };
    float X[K][COLS];   // input rows h - R .. h + R
    // Outputs row0 - R .. row1 - 1 + R: those beyond the strip only for the rows of gx that they give to, nothing for gw.
    const int h_first = row0 - R, h_last = row1 - 1 + R;
#pragma unroll
    for (int i = 1; i < K; i++) open_row(fetch(h_first - R + i - 1), h_first - R + i - 1, X[i]);
    Row next = fetch(h_first + R);
    float4 grad = fetch_grad(h_first);
    // The strips of a warp are of one length but for the last of a plane; all lanes go as far as the longest.
    const int steps = a.strip_rows + 2 * R;
    int top = (K - 1) * COLS * 128;
    for (int step = 0; step < steps; step++)
    {
        const int h = h_first + step;
#pragma unroll
        for (int i = 0; i + 1 < K; i++)
#pragma unroll
            for (int c = 0; c < COLS; c++) X[i][c] = X[i + 1][c];
        open_row(next, h + R, X[K - 1]);
        const float4 here = grad;
        next = fetch(h + R + 1);
        grad = fetch_grad(h + 1);
        const bool inside = h <= h_last, counts = own && h >= row0 && h < row1;
        const float g4[4] = {inside ? here.x : 0.f, inside ? here.y : 0.f, inside ? here.z : 0.f, inside ? here.w : 0.f};
        uint32_t off[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
        {
            constexpr float INITIAL = IS_MIN ? Limits<float>::inf() : -Limits<float>::inf();
            float v[TAPS], m = INITIAL;
#pragma unroll
            for (int k = 0; k < TAPS; k++) v[k] = X[K - 1 - k / K][j + K - 1 - k % K] + w[k];
#pragma unroll
            for (int k = 0; k + 1 < TAPS; k += 2) m = ext3<IS_MIN>(m, v[k], v[k + 1]);
            m = ext2<IS_MIN>(m, v[TAPS - 1]);
            uint32_t at = ((K - 1) * COLS + K - 1) * 128u;
#pragma unroll
            for (int k = TAPS - 2; k >= 0; k--) at = v[k] == m ? ((k / K) * COLS + k % K) * 128u : at;
            off[j] = m == INITIAL ? 0u : at;
        }
        // `top` is where row h + R lies in the ring of rows of gx; the row that tap (kh, kw) reads lies kh places before it, its column K - 1 - kw
        // after the output's.
#pragma unroll
        for (int j = 0; j < 4; j++)
        {
            int at = top + (j + K - 1) * 128 - static_cast<int>(off[j]);
            const uint32_t bin = bin_base + off[j];
            if (at < 0) at += K * COLS * 128;
            const float x0 = shared_word(acc_base + at), b0 = shared_word(bin);
            set_shared_word(acc_base + at, x0 + g4[j]);
            set_shared_word(bin, b0 + (counts ? g4[j] : 0.0f));
        }
        // Row h - R has all that it will get from this strip's outputs; its place is that of the next row to begin.
        float done[COLS];
        top = top + COLS * 128 == K * COLS * 128 ? 0 : top + COLS * 128;
#pragma unroll
        for (int c = 0; c < COLS; c++)
        {
            done[c] = shared_word(acc_base + top + c * 128);
            set_shared_word(acc_base + top + c * 128, 0.0f);
        }
        const int r = h - R;
        float sum[4];
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] = done[R + j];
#pragma unroll
        for (int i = 0; i < R; i++)
        {
            const float l = __shfl_up_sync(0xffffffffu, done[R + 4 + i], 1, lanes), n = __shfl_down_sync(0xffffffffu, done[i], 1, lanes);
            if (sub > 0) sum[i] += l;
            if (sub < lanes - 1) sum[4 - R + i] += n;
        }
        if (own && r >= row0 && r < row1)
            *reinterpret_cast<float4*>(a.y + base + static_cast<int64_t>(r) * a.W + col) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
#pragma unroll
    for (int k = 0; k < TAPS; k++)
    {
        float total = sums[K * COLS + (k / K) * COLS + k % K][lane];
        for (int d = lanes / 2; d > 0; d /= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
        if (live && sub == 0) a.partial[(static_cast<int64_t>(channel) * TAPS + k) * a.parts + (image * a.column_tiles + tile) * a.strips + strip] = total;
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
