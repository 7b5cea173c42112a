// Entry points of the per-channel layers whose input is kept in 8 bits.
#include "morpho_identity8.cuh"

namespace mc
{

namespace
{

/// Whether the kernels cover a call. Not covered, and left to mc_morpho_forward / mc_morpho_backward with mc_encode8 / mc_decode8: what
/// mixes channels, double, other structuring elements (7 x 7 needs more registers than a thread has), rows that are not whole quads, rows too long to stage.
bool covered(const mc_desc& d)
{
    return d.merge == MC_MERGE_IDENTITY && d.dtype == MC_F32 && d.kH == d.kW && (d.kH == 3 || d.kH == 5) && d.W % 4 == 0 && d.W <= 4096
           && static_cast<int64_t>(d.B) * d.Ci <= 0x7fffffff && static_cast<int64_t>(d.H) * d.W < (1 << 30) && static_cast<int64_t>(d.H) * d.W > 1 && (d.flags & MC_FLAG_ACCUMULATE) == 0;
}

bool aligned16(std::initializer_list<const void*> pointers)
{
    for (const void* p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    return true;
}

Identity8Args common(const mc_desc& d)
{
    Identity8Args a{};
    a.weight_batch_stride = d.weight_batch_stride;
    a.plane_blocks = code_blocks(static_cast<int64_t>(d.H) * d.W);
    a.C = d.Ci;
    a.H = d.H;
    a.W = d.W;
    a.fill = static_cast<float>(d.fill);
    a.replicate = d.pad_kind == MC_PAD_REPLICATE;
    a.flipped = (d.flags & MC_FLAG_FLIPPED_WEIGHT) != 0;
    return a;
}

/// Strips of the backward kernel. A strip of r rows takes r + K - 1 steps, and the warps of all strips come in waves of what is resident: the strips
/// of at least 8 rows with the fewest steps in all. ((16, 64, 112, 112) at 3 x 3: three strips a plane, a few more than are resident at once,
/// took 125 us where two take 78.) False where there are more of them than can be counted.
bool set_strips(Identity8Args& a, const mc_desc& d)
{
    const int64_t planes = static_cast<int64_t>(d.B) * d.Ci;
    a.column_tiles = d.W <= 128 ? 1 : (d.W + strip_columns(d.W) - 1) / strip_columns(d.W);
    const int64_t columns = planes * a.column_tiles, resident = 148 * (d.kH == 3 ? BACKWARD_WARPS_3 : BACKWARD_WARPS_5) * (32 / strip_lanes(d.W));
    const int extra = d.kH - 1;
    int64_t best = 0;
    for (int strips = 1; strips <= std::max(1, d.H / 8); strips += 1 + strips / 64)   // not every number of them in a tall image: this is host time
    {
        const int rows = (d.H + strips - 1) / strips, count = (d.H + rows - 1) / rows;
        const int64_t cost = (columns * count + resident - 1) / resident * (rows + extra);
        if (best != 0 && cost >= best) continue;
        best = cost;
        a.strip_rows = rows;
        a.strips = count;
    }
    a.units = columns * a.strips;
    a.parts = static_cast<int>(std::min<int64_t>(a.units / d.Ci, std::numeric_limits<int>::max()));
    return a.units / d.Ci < std::numeric_limits<int>::max();
}

/// Validation of what both entry points take.
int checked(const mc_desc* d)
{
    const int rc = validate(d, true);
    if (rc != MC_OK) return rc;
    return covered(*d) ? MC_OK : MC_ERR_UNSUPPORTED;
}

template <bool IS_MIN> int forward8(const Identity8Args& a, int K, int64_t blocks, cudaStream_t stream)
{
    const auto kernel = K == 3 ? identity_forward8_kernel<IS_MIN, 3> : identity_forward8_kernel<IS_MIN, 5>;
    const size_t shared = identity8_shared(K, a.W);
    if (!allow_shared(kernel, shared)) { set_last_error("identity_forward8_kernel: %zu bytes of shared memory refused", shared); return MC_ERR_CUDA; }
    kernel<<<static_cast<unsigned>(blocks), THREADS, shared, stream>>>(a);
    return check_launch("identity_forward8_kernel");
}

template <bool IS_MIN> int backward8(const Identity8Args& a, int K, int64_t blocks, cudaStream_t stream)
{
    const auto kernel = K == 3 ? identity_backward8_kernel<IS_MIN, 3, BACKWARD_WARPS_3> : identity_backward8_kernel<IS_MIN, 5, BACKWARD_WARPS_5>;
    kernel<<<static_cast<unsigned>(blocks), 32, 0, stream>>>(a);
    return check_launch("identity_backward8_kernel");
}

}  // namespace

}  // namespace mc

using namespace mc;

extern "C" {

int mc_morpho_forward8(const mc_desc* desc, const void* x, const void* w, void* y, int8_t* codes, void* scales, void* stream)
{
    const int rc = checked(desc);
    if (rc != MC_OK) return rc;
    const int64_t planes = static_cast<int64_t>(desc->B) * desc->Ci;
    if (planes == 0) return MC_OK;
    if (x == nullptr || w == nullptr || y == nullptr || codes == nullptr || scales == nullptr)
    {
        set_last_error("x, w, y, codes or scales is NULL");
        return MC_ERR_INVALID_ARGUMENT;
    }
    if (!aligned16({x, y, codes})) return MC_ERR_UNSUPPORTED;
    Identity8Args a = common(*desc);
    a.x = static_cast<const float*>(x);
    a.w = static_cast<const float*>(w);
    a.y = static_cast<float*>(y);
    a.codes = codes;
    a.scales = static_cast<float*>(scales);
    a.chunks = (desc->H * desc->W + RUN - 1) / RUN;
    a.run_step = 4 * THREADS % desc->W;
    const int64_t blocks = planes * a.chunks;
    if (blocks > 0x7fffffff) return MC_ERR_UNSUPPORTED;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return desc->op == MC_OP_EROSION ? forward8<true>(a, desc->kH, blocks, s) : forward8<false>(a, desc->kH, blocks, s);
}

size_t mc_morpho_backward8_workspace_bytes(const mc_desc* desc)
{
    if (checked(desc) != MC_OK || desc->B == 0) return 0;
    Identity8Args a = common(*desc);
    if (!set_strips(a, *desc)) return 0;
    return sizeof(float) * static_cast<size_t>(desc->Ci) * desc->kH * desc->kW * static_cast<size_t>(a.parts);
}

int mc_morpho_backward8(const mc_desc* desc, const int8_t* codes, const void* scales, const void* w, const void* gy, void* gx, void* gw, void* workspace,
                        size_t workspace_bytes, void* stream)
{
    const int rc = checked(desc);
    if (rc != MC_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (gw == nullptr) { set_last_error("gw is NULL"); return MC_ERR_INVALID_ARGUMENT; }
    const int taps = desc->kH * desc->kW, count = desc->Ci * taps;
    if (desc->B == 0)
    {
        if (cudaMemsetAsync(gw, 0, sizeof(float) * count, s) == cudaSuccess) return MC_OK;
        set_last_error("cudaMemsetAsync failed");
        return MC_ERR_CUDA;
    }
    if (codes == nullptr || scales == nullptr || w == nullptr || gy == nullptr || gx == nullptr)
    {
        set_last_error("codes, scales, w, gy or gx is NULL");
        return MC_ERR_INVALID_ARGUMENT;
    }
    if (!aligned16({gy, gx}) || reinterpret_cast<uintptr_t>(codes) % 4 != 0) return MC_ERR_UNSUPPORTED;
    const size_t need = mc_morpho_backward8_workspace_bytes(desc);
    if (need == 0) return MC_ERR_UNSUPPORTED;
    if (workspace == nullptr || workspace_bytes < need)
    {
        set_last_error("workspace of %zu bytes needed, %zu given", need, workspace_bytes);
        return MC_ERR_WORKSPACE;
    }
    Identity8Args a = common(*desc);
    (void)set_strips(a, *desc);
    a.w = static_cast<const float*>(w);
    a.gy = static_cast<const float*>(gy);
    a.y = static_cast<float*>(gx);
    a.codes = const_cast<int8_t*>(codes);
    a.scales = const_cast<float*>(static_cast<const float*>(scales));
    a.partial = static_cast<float*>(workspace);
    const int64_t units_per_block = 32 / strip_lanes(desc->W), blocks = (a.units + units_per_block - 1) / units_per_block;
    if (blocks > 0x7fffffff) return MC_ERR_UNSUPPORTED;
    const bool erosion = desc->op == MC_OP_EROSION;
    const int launched = erosion ? backward8<true>(a, desc->kH, blocks, s) : backward8<false>(a, desc->kH, blocks, s);
    if (launched != MC_OK) return launched;
    identity_weight8_kernel<<<static_cast<unsigned>((count + THREADS / 32 - 1) / (THREADS / 32)), THREADS, 0, s>>>(
        a.partial, static_cast<float*>(gw), count, taps, a.parts, erosion ? -1.0f : 1.0f, a.flipped);
    return check_launch("identity_weight8_kernel");
}

}  // extern "C"
