// What the entry points of the root-mean-square norm share with its per-type translation units.
#pragma once
#include "encode8.cuh"

namespace mc
{

struct NormArgs;
struct NormGradArgs;

template <typename T> int rms_norm_forward(const NormArgs& a, cudaStream_t stream);
template <typename T> int rms_norm_backward(const NormGradArgs& a, cudaStream_t stream);

/// Thread blocks of the backward kernels, each of which leaves one row of partial sums of gweight. They walk over the tiles (or
/// rows): more of them than are resident would only add rows.
inline int64_t norm_backward_grid(int64_t outer, int64_t channels, int64_t inner, bool wide)
{
    constexpr int64_t SMS = 148;
    if (inner != 1)
    {
        // As the launches choose: the pixels of a tile, and one or two thread blocks an SM.
        const int64_t whole = wide ? 32 : 64, held = wide ? 128 : 512;
        const int64_t pixels = channels <= whole ? 128 : channels <= 2 * whole ? 64 : channels <= held ? 32 : 128;
        return std::min(outer * ((inner + pixels - 1) / pixels), SMS * (channels <= 4 * whole ? 2 : 1));
    }
    const int64_t blocks = code_blocks(channels);
    int64_t groups = 8;   // rows that a thread block has at work
    while (groups > 1 && blocks * groups > 32) groups /= 2;
    return std::min((outer + groups - 1) / groups, SMS * (blocks > 32 ? 1 : 2));
}

}  // namespace mc
