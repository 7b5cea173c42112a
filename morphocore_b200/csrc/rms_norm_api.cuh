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

/// Thread blocks an SM of the backward kernel for feature maps of up to 128 channels, whose elements have this many bytes: as many as its registers let in
/// without spilling them.
constexpr int gradient_blocks_per_sm(int element) { return element == 8 ? 2 : element == 4 ? 3 : 4; }

/// Thread blocks of the backward kernels, each of which leaves one row of partial sums of gweight. They walk over the tiles (or
/// rows): more of them than are resident would only add rows. `element`: bytes of one.
inline int64_t norm_backward_grid(int64_t outer, int64_t channels, int64_t inner, int element)
{
    constexpr int64_t SMS = 148;
    if (inner != 1)
    {
        // As the launches choose: the pixels of a tile, and the thread blocks an SM.
        const int64_t held = element == 8 ? 128 : 512;
        const int64_t pixels = channels <= 32 ? 128 : channels <= 64 ? 64 : channels <= held ? 32 : 128;
        const int64_t resident = channels <= 128 ? gradient_blocks_per_sm(element) : channels <= 256 && element < 8 ? 2 : 1;
        return std::min(outer * ((inner + pixels - 1) / pixels), SMS * resident);
    }
    const RowSplit split = split_rows(code_blocks(channels));
    return std::min((outer + split.rows - 1) / split.rows, SMS * (split.warps == 8 ? 2 : 1));
}

}  // namespace mc
