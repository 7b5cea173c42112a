// Entry points of the root-mean-square norm: argument checks and the type's dispatch.
#include "rms_norm.cuh"
#include "rms_norm_api.cuh"

namespace mc
{

namespace
{

/// Rows of partial sums and the lanes' sums of gweight are laid out for this many channels.
constexpr int64_t MAX_CHANNELS = 16384;

int checked_norm(const mc_norm_desc* d)
{
    if (d == nullptr) { set_last_error("descriptor is NULL"); return MC_ERR_INVALID_ARGUMENT; }
    if (d->outer < 0 || d->channels <= 0 || d->inner < 0)
    {
        set_last_error("sizes must be positive (outer=%lld channels=%lld inner=%lld)", static_cast<long long>(d->outer),
                       static_cast<long long>(d->channels), static_cast<long long>(d->inner));
        return MC_ERR_INVALID_ARGUMENT;
    }
    const unsigned __int128 limit = static_cast<unsigned __int128>(1) << 40;
    const unsigned __int128 pixels = static_cast<unsigned __int128>(d->outer) * static_cast<unsigned __int128>(d->inner);
    if (pixels > limit || pixels * static_cast<unsigned __int128>(d->channels) > limit)
    {
        set_last_error("tensor of more than 2^40 elements (outer=%lld channels=%lld inner=%lld)", static_cast<long long>(d->outer),
                       static_cast<long long>(d->channels), static_cast<long long>(d->inner));
        return MC_ERR_INVALID_ARGUMENT;
    }
    if (d->dtype < MC_F32 || d->dtype > MC_BF16) { set_last_error("unknown dtype %d", d->dtype); return MC_ERR_INVALID_ARGUMENT; }
    if ((d->flags & ~MC_NORM_FLOAT_WEIGHT) != 0) { set_last_error("unknown flags 0x%x", static_cast<unsigned>(d->flags)); return MC_ERR_INVALID_ARGUMENT; }
    if ((d->flags & MC_NORM_FLOAT_WEIGHT) != 0 && d->dtype != MC_F16 && d->dtype != MC_BF16)
    {
        set_last_error("MC_NORM_FLOAT_WEIGHT is for tensors in half precision, not for dtype %d", d->dtype);
        return MC_ERR_INVALID_ARGUMENT;
    }
    if (!(d->eps > 0.0) || d->eps > std::numeric_limits<double>::max()) { set_last_error("eps must be positive and finite, got %g", d->eps); return MC_ERR_INVALID_ARGUMENT; }
    if (d->channels > MAX_CHANNELS)
    {
        set_last_error("a norm over %lld channels; at most %lld are supported", static_cast<long long>(d->channels), static_cast<long long>(MAX_CHANNELS));
        return MC_ERR_UNSUPPORTED;
    }
    return MC_OK;
}

template <typename Args> void set_sizes(Args& a, const mc_norm_desc& d)
{
    a.outer = d.outer;
    a.channels = d.channels;
    a.inner = d.inner;
    a.tiles_per_row = code_blocks(d.inner == 1 ? d.channels : d.inner);
    a.tiles = d.outer * a.tiles_per_row;
    a.eps = d.eps;
    a.per_channel = 1.0 / static_cast<double>(d.channels);
}

int refuse(const char* why)
{
    set_last_error("%s", why);
    return MC_ERR_INVALID_ARGUMENT;
}

/// Calls f(T{}, G{}) for the types of the tensors and of the weight.
template <typename F> int dispatch_norm(const mc_norm_desc& d, F f)
{
    const bool float_weight = (d.flags & MC_NORM_FLOAT_WEIGHT) != 0;
    return dispatch_dtype(d.dtype, [&](auto t) {
        if constexpr (sizeof(t) == 2)
            if (float_weight) return f(t, float{});
        return f(t, t);
    });
}

int weight_bytes(const mc_norm_desc& d) { return d.dtype == MC_F64 ? 8 : d.dtype == MC_F32 || (d.flags & MC_NORM_FLOAT_WEIGHT) != 0 ? 4 : 2; }

int element_bytes(const mc_norm_desc& d) { return d.dtype == MC_F64 ? 8 : d.dtype == MC_F32 ? 4 : 2; }

}  // namespace

}  // namespace mc

using namespace mc;

extern "C" {

int mc_rms_norm_forward(const mc_norm_desc* desc, const void* x, const void* residual, const void* weight, void* sum, void* y, int8_t* y_codes,
                        void* y_scales, int8_t* sum_codes, void* sum_scales, void* stream)
{
    const int rc = checked_norm(desc);
    if (rc != MC_OK) return rc;
    if (desc->outer * desc->inner == 0) return MC_OK;
    if (x == nullptr) return refuse("x is NULL");
    if ((residual == nullptr) != (sum == nullptr)) return refuse("sum is written where there is a residual, and NULL where there is none");
    if ((y_codes == nullptr) != (y_scales == nullptr)) return refuse("y_codes and y_scales are NULL together or not");
    if ((sum_codes == nullptr) != (sum_scales == nullptr)) return refuse("sum_codes and sum_scales are NULL together or not");
    if (y == nullptr && y_codes == nullptr && sum == nullptr && sum_codes == nullptr) return refuse("nothing to compute: every output is NULL");
    NormArgs a{};
    set_sizes(a, *desc);
    a.x = x; a.residual = residual; a.weight = weight; a.sum = sum; a.y = y;
    a.y_codes = y_codes; a.y_scales = y_scales; a.sum_codes = sum_codes; a.sum_scales = sum_scales;
    return dispatch_norm(*desc, [&](auto t, auto g) { return rms_norm_forward<decltype(t), decltype(g)>(a, static_cast<cudaStream_t>(stream)); });
}

size_t mc_rms_norm_backward_workspace_bytes(const mc_norm_desc* desc, int have_gweight)
{
    if (!have_gweight || checked_norm(desc) != MC_OK || desc->outer * desc->inner == 0) return 0;
    return (desc->dtype == MC_F64 ? 8 : 4) * static_cast<size_t>(norm_backward_grid(desc->outer, desc->channels, desc->inner, element_bytes(*desc))) * static_cast<size_t>(desc->channels);
}

int mc_rms_norm_backward(const mc_norm_desc* desc, const void* sum, const int8_t* sum_codes, const void* sum_scales, const void* weight, const void* gy,
                         const void* gsum, void* gx, void* gweight, void* workspace, size_t workspace_bytes, void* stream)
{
    const int rc = checked_norm(desc);
    if (rc != MC_OK) return rc;
    if ((weight == nullptr) != (gweight == nullptr)) return refuse("weight and gweight are NULL together or not");
    if (desc->outer * desc->inner == 0)
    {
        if (gweight == nullptr) return MC_OK;
        const cudaError_t err = cudaMemsetAsync(gweight, 0, static_cast<size_t>(weight_bytes(*desc)) * static_cast<size_t>(desc->channels), static_cast<cudaStream_t>(stream));
        if (err == cudaSuccess) return MC_OK;
        set_last_error("cudaMemsetAsync: %s", cudaGetErrorString(err));
        return MC_ERR_CUDA;
    }
    if ((sum == nullptr) == (sum_codes == nullptr) || (sum_codes == nullptr) != (sum_scales == nullptr))
        return refuse("either sum, or sum_codes and sum_scales, are given");
    if (gy == nullptr || gx == nullptr) return refuse("gy or gx is NULL");
    const size_t need = mc_rms_norm_backward_workspace_bytes(desc, gweight != nullptr);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    {
        set_last_error("workspace of %zu bytes needed, %zu given", need, workspace_bytes);
        return MC_ERR_WORKSPACE;
    }
    NormGradArgs a{};
    set_sizes(a, *desc);
    a.sum = sum; a.sum_codes = sum_codes; a.sum_scales = sum_scales; a.weight = weight; a.gy = gy; a.gsum = gsum;
    a.gx = gx; a.gweight = gweight; a.partial = workspace;
    return dispatch_norm(*desc, [&](auto t, auto g) { return rms_norm_backward<decltype(t), decltype(g)>(a, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
