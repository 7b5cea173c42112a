// What the entry points of the root-mean-square norm share with its per-type translation units.
#pragma once
#include "encode8.cuh"

namespace mc
{

struct NormArgs;
struct NormGradArgs;

/// T: the tensors' type, G: the weight's and its gradient's.
template <typename T, typename G> int rms_norm_forward(const NormArgs& a, cudaStream_t stream);
template <typename T, typename G> int rms_norm_backward(const NormGradArgs& a, cudaStream_t stream);

/// How rows of channels are dealt out: a thread block of `warps` warps takes `rows` rows at once, 2^shift warps a row, and a warp holds `blocks` blocks
/// of 128 channels of each of its rows. Rows of one and two blocks go four and two to a warp.
struct RowSplit
{
    int rows, warps, shift, blocks;
};
inline RowSplit split_rows(int64_t blocks)
{
    if (blocks <= 2) return {blocks == 1 ? 32 : 16, 8, 0, static_cast<int>(blocks)};
    if (blocks > 64) return {1, 16, 4, 8};
    if (blocks > 32) return {1, 16, 4, 4};
    int shift = 0;
    while (blocks > (4 << shift)) shift++;
    return {8 >> shift, 8, shift, 4};
}

/// Thread blocks an SM of the backward kernels for rows of channels.
constexpr int row_gradient_blocks_per_sm(int warps) { return warps == 8 ? 2 : 1; }

/// A variant of the backward kernel for feature maps that holds its tile: up to `channels` of 128 / `split` pixels, `held` by each of split * warps groups of
/// lanes, in thread blocks of which an SM has `blocks_per_sm`. The kernel's launch and the number of its thread blocks both go by gradient_tile.
struct GradientTile
{
    int channels, held, warps, split, blocks_per_sm;
};
/// How many variants there are for elements of so many bytes, for more and more channels; what has more channels than the last reads its tile twice. Eight quads of
/// doubles do not fit the registers.
constexpr int gradient_tiles(int element) { return element == 8 ? 3 : 5; }
constexpr GradientTile gradient_tile(int element, int i)
{
    const int held = element == 8 ? 4 : 8, blocks_per_sm = element == 8 ? 2 : element == 4 ? 3 : 4;
    return i < 3 ? GradientTile{32 << i, held, 32 / held, 1 << i, blocks_per_sm} : i == 3 ? GradientTile{256, held, 8, 4, 2} : GradientTile{512, held, 16, 4, 1};
}

/// Thread blocks of the backward kernels, each of which leaves one row of partial sums of gweight. They walk over the tiles (or
/// rows): more of them than are resident would only add rows. `element`: bytes of one.
inline int64_t norm_backward_grid(int64_t outer, int64_t channels, int64_t inner, int element)
{
    constexpr int64_t SMS = 148;
    if (inner == 1)
    {
        const RowSplit split = split_rows(code_blocks(channels));
        return std::min((outer + split.rows - 1) / split.rows, SMS * row_gradient_blocks_per_sm(split.warps));
    }
    int64_t pixels = CODE_BLOCK, resident = 1;   // of the kernel that reads its tile twice
    for (int i = gradient_tiles(element) - 1; i >= 0; i--)
    {
        const GradientTile tile = gradient_tile(element, i);
        if (channels > tile.channels) break;
        pixels = CODE_BLOCK / tile.split;
        resident = tile.blocks_per_sm;
    }
    return std::min(outer * ((inner + pixels - 1) / pixels), SMS * resident);
}

}  // namespace mc
