// Instantiates mc::rms_norm_forward<MC_T> and mc::rms_norm_backward<MC_T>; included by rms_norm_f32.cu, _f64, _f16 and _bf16.
#include "rms_norm.cuh"
#include "rms_norm_api.cuh"

namespace mc
{

namespace
{

constexpr int LARGEST_GRID = 0x7fffffff;

template <typename Kernel, typename Args, typename... More>
int launch_norm(Kernel kernel, int64_t grid, int warps, size_t shared, cudaStream_t stream, const char* what, const Args& a, More... more)
{
    if (shared > 30 * 1024)   // with what a kernel declares itself, the 48 KiB that need no opt-in
    {
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
        if (err != cudaSuccess)
        {
            set_last_error("%s: %s", what, cudaGetErrorString(err));
            return MC_ERR_CUDA;
        }
    }
    kernel<<<static_cast<unsigned>(std::min<int64_t>(grid, LARGEST_GRID)), warps * 32, shared, stream>>>(a, more...);
    return check_launch(what);
}

/// Warps that share a row of `blocks` blocks when each keeps up to `held`: a power of two, at most `most`.
int warps_per_row(int64_t blocks, int held, int most)
{
    int n = 1;
    while (n < most && blocks > static_cast<int64_t>(n) * held) n *= 2;
    return n;
}

template <typename T, bool VEC> int forward(const NormArgs& a, bool rows, cudaStream_t stream)
{
    if (rows)
    {
        if (a.tiles_per_row > 32)
            return launch_norm(rms_norm_rows_kernel<T, VEC, 8, 16, 1>, a.outer, 16, 0, stream, "rms_norm_rows_kernel", a, 16);
        const int per_row = warps_per_row(a.tiles_per_row, 4, 8), groups = 8 / per_row;
        return launch_norm(rms_norm_rows_kernel<T, VEC, 4, 8, sizeof(T) == 8 ? 2 : 3>, (a.outer + groups - 1) / groups, 8, 0, stream, "rms_norm_rows_kernel", a, per_row);
    }
    const auto columns = [&](auto kernel, int warps) { return launch_norm(kernel, a.tiles, warps, 0, stream, "rms_norm_columns_kernel", a); };
    if (a.channels <= 32) return columns(rms_norm_columns_kernel<T, VEC, 4, 8, 2>, 8);
    if constexpr (sizeof(T) == 8) return columns(rms_norm_columns_kernel<T, VEC, 4, 16, 1>, 16);   // eight quads of doubles do not fit the registers
    else
    {
        if (a.channels <= 64) return columns(rms_norm_columns_kernel<T, VEC, 8, 8, sizeof(T) == 2 ? 3 : 2>, 8);
        return columns(rms_norm_columns_kernel<T, VEC, 8, 16, sizeof(T) == 2 ? 2 : 1>, 16);
    }
}

template <typename T, bool VEC, bool CODES> int backward(const NormGradArgs& a, bool rows, cudaStream_t stream)
{
    const int64_t grid = norm_backward_grid(a.outer, a.channels, a.inner);
    const size_t sums = a.gweight == nullptr ? 0 : sizeof(Wide<T>) * static_cast<size_t>(a.channels);
    int rc;
    if (rows)
    {
        // Slots, or nothing, for the rows to come; gweight's sums take their place at the end.
        const auto run = [&](auto kernel, size_t slots, int warps, int per_row) {
            return launch_norm(kernel, grid, warps, std::max(slots, sums), stream, "rms_norm_rows_backward_kernel", a, per_row);
        };
        constexpr size_t FEW = gradient_slot_bytes<T, CODES>(4, 256), MANY = gradient_slot_bytes<T, CODES>(8, 512);
        constexpr bool FITS = MANY <= 200 * 1024;
        rc = a.tiles_per_row > 32 ? run(rms_norm_rows_backward_kernel<T, VEC, CODES, FITS, 8, 16, 1>, FITS ? MANY : 0, 16, 16)
                                  : run(rms_norm_rows_backward_kernel<T, VEC, CODES, true, 4, 8, 2>, FEW, 8, warps_per_row(a.tiles_per_row, 4, 8));
    }
    else
    {
        const auto columns = [&](auto kernel, int held, int warps) {
            return launch_norm(kernel, grid, warps, gradient_slot_bytes<T, CODES>(held, warps * 32), stream, "rms_norm_columns_backward_kernel", a);
        };
        const auto twice = [&](auto kernel) { return launch_norm(kernel, grid, 16, sums, stream, "rms_norm_columns_twice_backward_kernel", a); };
        if (a.channels <= 32) rc = columns(rms_norm_columns_backward_kernel<T, VEC, CODES, 4, 8, 2>, 4, 8);
        else if constexpr (sizeof(T) == 8)
            rc = a.channels <= 64 ? columns(rms_norm_columns_backward_kernel<T, VEC, CODES, 4, 16, 1>, 4, 16)
                                  : twice(rms_norm_columns_twice_backward_kernel<T, VEC, CODES, 4, 16, 1>);
        else if (a.channels <= 64) rc = columns(rms_norm_columns_backward_kernel<T, VEC, CODES, 8, 8, 2>, 8, 8);
        else if (a.channels <= 128) rc = columns(rms_norm_columns_backward_kernel<T, VEC, CODES, 8, 16, 1>, 8, 16);
        else rc = twice(rms_norm_columns_twice_backward_kernel<T, VEC, CODES, 4, 16, 1>);
    }
    if (rc != MC_OK || a.gweight == nullptr) return rc;
    norm_weight_kernel<T><<<static_cast<unsigned>((a.channels + 31) / 32), WEIGHT_WARPS * 32, 0, stream>>>(static_cast<const Wide<T>*>(a.partial),
                                                                                                static_cast<T*>(a.gweight), a.channels, static_cast<int>(grid));
    return check_launch("norm_weight_kernel");
}

}  // namespace

template <> int rms_norm_forward<MC_T>(const NormArgs& a, cudaStream_t stream)
{
    using T = MC_T;
    const bool rows = a.inner == 1;
    const bool quads = quads_fit<T>(rows ? a.channels : a.inner, {a.x, a.residual, rows ? a.weight : nullptr, a.sum, a.y}, {a.y_codes, a.sum_codes});
    return quads ? forward<T, true>(a, rows, stream) : forward<T, false>(a, rows, stream);
}

template <> int rms_norm_backward<MC_T>(const NormGradArgs& a, cudaStream_t stream)
{
    using T = MC_T;
    const bool rows = a.inner == 1, codes = a.sum == nullptr;
    const bool quads = quads_fit<T>(rows ? a.channels : a.inner, {a.sum, rows ? a.weight : nullptr, a.gy, a.gsum, a.gx}, {a.sum_codes});
    if (codes) return quads ? backward<T, true, true>(a, rows, stream) : backward<T, false, true>(a, rows, stream);
    return quads ? backward<T, true, false>(a, rows, stream) : backward<T, false, false>(a, rows, stream);
}

}  // namespace mc
