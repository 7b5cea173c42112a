// Instantiates mc::rms_norm_forward<MC_T, MC_G> and mc::rms_norm_backward<MC_T, MC_G>; included by rms_norm_f32.cu, _f64, _f16, _bf16 and, with float
// weights, _f16_f32 and _bf16_f32.
#include <atomic>

#include "rms_norm.cuh"
#include "rms_norm_api.cuh"

namespace mc
{

namespace
{

constexpr int LARGEST_GRID = 0x7fffffff;
template <int N> using Int = std::integral_constant<int, N>;

/// Launches KERNEL, whose shared memory needs an opt-in where it leaves the first 48 KiB together with what the kernel declares itself: up to 34 KiB, so
/// that the dynamic part alone says nothing. The opt-in is to all that the kernel can have, asked for once a device (it is 1 us of host time): threads with
/// launches of different sizes agree on it.
template <auto KERNEL, typename Args, typename... More>
int launch_norm(int64_t grid, int warps, size_t shared, cudaStream_t stream, const char* what, const Args& a, More... more)
{
    if (shared > 0)
    {
        constexpr int MAX_DEVICES = 64;
        static std::atomic<bool> allowed[MAX_DEVICES];
        int device = 0;
        cudaError_t err = cudaGetDevice(&device);
        const bool known = err == cudaSuccess && device >= 0 && device < MAX_DEVICES;
        if (err == cudaSuccess && !(known && allowed[device].load(std::memory_order_relaxed)))
        {
            cudaFuncAttributes declared;
            err = cudaFuncGetAttributes(&declared, KERNEL);
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(MAX_SHARED_BYTES - declared.sharedSizeBytes));
            if (err == cudaSuccess && known) allowed[device].store(true, std::memory_order_relaxed);
        }
        if (err != cudaSuccess)
        {
            set_last_error("%s: %s", what, cudaGetErrorString(err));
            return MC_ERR_CUDA;
        }
    }
    KERNEL<<<static_cast<unsigned>(std::min<int64_t>(grid, LARGEST_GRID)), warps * 32, shared, stream>>>(a, more...);
    return check_launch(what);
}

template <typename T, typename G, bool VEC> int forward(const NormArgs& a, bool rows, cudaStream_t stream)
{
    constexpr bool WIDE = sizeof(T) == 8, HALF = sizeof(T) == 2;
    constexpr const char* ROWS = "rms_norm_rows_kernel";
    constexpr const char* COLUMNS = "rms_norm_columns_kernel";
    if (rows)
    {
        const RowSplit split = split_rows(a.tiles_per_row);
        const auto launch = [&](auto rows, auto blocks, auto warps, auto ctas) {
            return launch_norm<rms_norm_rows_kernel<T, G, VEC, rows, blocks, warps, ctas>>((a.outer + split.rows - 1) / split.rows, warps, 0, stream, ROWS, a, split.shift);
        };
        constexpr Int<WIDE ? 2 : 4> CTAS;
        if (split.blocks == 1) return launch(Int<4>(), Int<1>(), Int<8>(), CTAS);
        if (split.blocks == 2) return launch(Int<2>(), Int<2>(), Int<8>(), CTAS);
        if (split.blocks == 8) return launch(Int<1>(), Int<8>(), Int<16>(), Int<1>());
        if (split.warps == 8) return launch(Int<1>(), Int<4>(), Int<8>(), CTAS);
        return launch(Int<1>(), Int<4>(), Int<16>(), Int<WIDE ? 1 : 2>());
    }
    // Few warps a thread block: four thread blocks of 4 warps that hide each other's barriers take 66 us for (64, 32, 112, 112) in float with residual where
    // two of 8 took 80, and hold 64 channels well enough although they read half of them again from L2 (154 to 250 us for (32, 64, 224, 224) against
    // 176 to 247); with 128 channels that is so of 8 warps (49 to 71 against 56 to 71 in 16), beyond no longer (140 against 135 for (64, 256, 56, 56)).
    // In half precision, 4 and 8 warps for 64 channels: 111 and 114 us for (32, 64, 224, 224), 60 and 58 for rows of 75 * 101 pixels. In double,
    // (16, 64, 112, 112): 50 to 81 us with 4 warps, 62 to 91 with 16 that hold all.
    const auto launch = [&](auto warps, auto ctas) { return launch_norm<rms_norm_columns_kernel<T, G, VEC, warps, ctas>>(a.tiles, warps, 0, stream, COLUMNS, a); };
    if constexpr (WIDE) return launch(Int<4>(), Int<3>());
    else if constexpr (HALF) return a.channels <= (VEC ? 64 : 32) ? launch(Int<4>(), Int<6>()) : launch(Int<8>(), Int<3>());
    else return a.channels <= 64 ? launch(Int<4>(), Int<4>()) : a.channels <= 128 ? launch(Int<8>(), Int<2>()) : launch(Int<16>(), Int<1>());
}

/// Feature maps: the first variant from the Ith on that holds all channels.
template <typename T, typename G, bool VEC, bool CODES, bool EXACT, int I = 0> int backward_columns(const NormGradArgs& a, int64_t grid, cudaStream_t stream)
{
    if constexpr (I < gradient_tiles(sizeof(T)))
    {
        constexpr GradientTile TILE = gradient_tile(sizeof(T), I);
        static_assert(TILE.held * TILE.warps * TILE.split == TILE.channels, "a place for every channel");
        if (a.channels > TILE.channels) return backward_columns<T, G, VEC, CODES, EXACT, I + 1>(a, grid, stream);
        return launch_norm<rms_norm_columns_backward_kernel<T, G, VEC, CODES, EXACT, TILE.held, TILE.warps, TILE.split, TILE.blocks_per_sm>>(
            grid, TILE.warps, gradient_slot_bytes<T, CODES>(TILE.held, TILE.warps * 32), stream, "rms_norm_columns_backward_kernel", a);
    }
    else
    {
        const size_t sums = a.gweight == nullptr ? 0 : sizeof(Wide<T>) * static_cast<size_t>(a.channels);
        return launch_norm<rms_norm_columns_twice_backward_kernel<T, G, VEC, CODES, EXACT, 4, 16, 1>>(grid, 16, sums, stream, "rms_norm_columns_twice_backward_kernel", a);
    }
}

template <typename T, typename G, bool VEC, bool CODES, bool EXACT> int backward_rows(const NormGradArgs& a, int64_t grid, cudaStream_t stream)
{
    // Slots, or nothing, for the rows to come; gweight's sums take their place at the end.
    constexpr bool FITS = gradient_slot_bytes<T, CODES>(8, 512) <= 200 * 1024;
    const size_t sums = a.gweight == nullptr ? 0 : sizeof(Wide<T>) * static_cast<size_t>(a.channels);
    const RowSplit split = split_rows(a.tiles_per_row);
    const auto launch = [&](auto ahead, auto rows, auto blocks, auto warps) {
        const size_t slots = ahead ? gradient_slot_bytes<T, CODES>(rows * blocks, warps * 32) : 0;
        return launch_norm<rms_norm_rows_backward_kernel<T, G, VEC, CODES, EXACT, ahead, rows, blocks, warps, row_gradient_blocks_per_sm(warps)>>(
            grid, warps, std::max(slots, sums), stream, "rms_norm_rows_backward_kernel", a, split.shift);
    };
    constexpr std::true_type AHEAD;
    if (split.blocks == 1) return launch(AHEAD, Int<4>(), Int<1>(), Int<8>());
    if (split.blocks == 2) return launch(AHEAD, Int<2>(), Int<2>(), Int<8>());
    if (split.blocks == 8) return launch(std::bool_constant<FITS>(), Int<1>(), Int<8>(), Int<16>());
    return split.warps == 8 ? launch(AHEAD, Int<1>(), Int<4>(), Int<8>()) : launch(AHEAD, Int<1>(), Int<4>(), Int<16>());
}

template <typename T, typename G, bool VEC, bool CODES, bool EXACT = false> int backward(const NormGradArgs& a, bool rows, cudaStream_t stream)
{
    const int64_t grid = norm_backward_grid(a.outer, a.channels, a.inner, sizeof(T));
    const int rc = rows ? backward_rows<T, G, VEC, CODES, EXACT>(a, grid, stream) : backward_columns<T, G, VEC, CODES, EXACT>(a, grid, stream);
    if (rc != MC_OK || a.gweight == nullptr) return rc;
    norm_weight_kernel<G><<<static_cast<unsigned>((a.channels + 31) / 32), WEIGHT_WARPS * 32, 0, stream>>>(
        static_cast<const Wide<G>*>(a.partial), static_cast<G*>(a.gweight), a.channels, static_cast<int>(grid));
    return check_launch("norm_weight_kernel");
}

/// Whether a weight that is read as quads (rows of channels) may be.
template <typename G> bool weight_fits(const void* weight, bool rows) { return !rows || reinterpret_cast<uintptr_t>(weight) % alignof(Quad<G>) == 0; }

}  // namespace

template <> int rms_norm_forward<MC_T, MC_G>(const NormArgs& a, cudaStream_t stream)
{
    using T = MC_T;
    using G = MC_G;
    const bool rows = a.inner == 1;
    const bool quads = quads_fit<T>(rows ? a.channels : a.inner, {a.x, a.residual, a.sum, a.y}, {a.y_codes, a.sum_codes}) && weight_fits<G>(a.weight, rows);
    return quads ? forward<T, G, true>(a, rows, stream) : forward<T, G, false>(a, rows, stream);
}

template <> int rms_norm_backward<MC_T, MC_G>(const NormGradArgs& a, cudaStream_t stream)
{
    using T = MC_T;
    using G = MC_G;
    const bool rows = a.inner == 1, codes = a.sum == nullptr;
    const bool quads = quads_fit<T>(rows ? a.channels : a.inner, {a.sum, a.gy, a.gsum, a.gx}, {a.sum_codes}) && weight_fits<G>(a.weight, rows);
    if constexpr (sizeof(T) < 8)
        if (a.eps < TINY_EPS) return codes ? backward<T, G, false, true, true>(a, rows, stream) : backward<T, G, false, false, true>(a, rows, stream);
    if (codes) return quads ? backward<T, G, true, true>(a, rows, stream) : backward<T, G, false, true>(a, rows, stream);
    return quads ? backward<T, G, true, false>(a, rows, stream) : backward<T, G, false, false>(a, rows, stream);
}

}  // namespace mc
