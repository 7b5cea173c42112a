// Activations in 8 bits: mc_encode8 and mc_decode8. Both are one pass over memory; a warp takes whole blocks of 128.
#include "encode8.cuh"

namespace mc
{

namespace
{

constexpr int BATCH = 4;   // blocks that a warp has in flight

struct RowBlocks
{
    int64_t length, per_row, blocks;   // elements of a row, its blocks, blocks in all
    bool whole;                        // rows are made of full blocks: block b starts at element 128 b
};

/// First element of block b and how many it has.
__device__ __forceinline__ int64_t block_start(const RowBlocks& r, int64_t b, int& valid)
{
    valid = CODE_BLOCK;
    if (r.whole) return b * CODE_BLOCK;
    const int64_t row = r.blocks <= 0xffffffffll ? static_cast<uint32_t>(b) / static_cast<uint32_t>(r.per_row) : b / r.per_row;
    const int64_t first = (b - row * r.per_row) * CODE_BLOCK;
    valid = static_cast<int>(min(static_cast<int64_t>(CODE_BLOCK), r.length - first));
    return row * r.length + first;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) encode8_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, Wide<T>* __restrict__ scales, const RowBlocks r)
{
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
    for (int64_t b0 = (static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5)) * BATCH; b0 < r.blocks; b0 += warps * BATCH)
    {
        Quad<T> q[BATCH];
        int64_t start[BATCH];
        int valid[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++)
        {
            valid[i] = 0;
            start[i] = 0;
            if (b0 + i < r.blocks) start[i] = block_start(r, b0 + i, valid[i]);
            q[i] = load_quad<VEC>(x + start[i], lane, valid[i]);
        }
#pragma unroll
        for (int i = 0; i < BATCH; i++)
        {
            Wide<T> v[4], scale;
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = widen(q[i].e[k]);
            const uint32_t c = encode_quad(v, scale);
            store_codes<VEC>(codes + start[i], c, lane, valid[i]);
            if (lane == 0 && b0 + i < r.blocks) scales[b0 + i] = scale;
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) decode8_kernel(const int8_t* __restrict__ codes, const Wide<T>* __restrict__ scales, T* __restrict__ x, const RowBlocks r)
{
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
    for (int64_t b0 = (static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5)) * BATCH; b0 < r.blocks; b0 += warps * BATCH)
    {
        uint32_t c[BATCH];
        Wide<T> scale[BATCH];
        int64_t start[BATCH];
        int valid[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++)
        {
            valid[i] = 0;
            start[i] = 0;
            scale[i] = 0;
            if (b0 + i < r.blocks)
            {
                start[i] = block_start(r, b0 + i, valid[i]);
                scale[i] = __ldg(scales + b0 + i);
            }
            c[i] = load_codes<VEC>(codes + start[i], lane, valid[i]);
        }
#pragma unroll
        for (int i = 0; i < BATCH; i++)
        {
            Quad<T> q;
#pragma unroll
            for (int k = 0; k < 4; k++) q.e[k] = narrow<T>(decode_code(c[i], k, scale[i]));
            store_quad<VEC>(x + start[i], q, lane, valid[i]);
        }
    }
}

int checked_rows(const mc_rows_desc* d)
{
    if (d == nullptr) { set_last_error("descriptor is NULL"); return MC_ERR_INVALID_ARGUMENT; }
    if (d->rows < 0 || d->length < 0)
    {
        set_last_error("sizes must not be negative (rows=%lld length=%lld)", static_cast<long long>(d->rows), static_cast<long long>(d->length));
        return MC_ERR_INVALID_ARGUMENT;
    }
    if (static_cast<unsigned __int128>(d->rows) * static_cast<unsigned __int128>(d->length) > static_cast<unsigned __int128>(1) << 40)
    {
        set_last_error("tensor of more than 2^40 elements (rows=%lld length=%lld)", static_cast<long long>(d->rows), static_cast<long long>(d->length));
        return MC_ERR_INVALID_ARGUMENT;
    }
    if (d->dtype < MC_F32 || d->dtype > MC_BF16) { set_last_error("unknown dtype %d", d->dtype); return MC_ERR_INVALID_ARGUMENT; }
    if (d->reserved != 0) { set_last_error("reserved must be 0"); return MC_ERR_INVALID_ARGUMENT; }
    return MC_OK;
}

RowBlocks row_blocks(const mc_rows_desc& d)
{
    const int64_t per_row = code_blocks(d.length);
    return {d.length, per_row, d.rows * per_row, d.length % CODE_BLOCK == 0};
}

unsigned grid_of(const RowBlocks& r)
{
    const int64_t warps = (r.blocks + BATCH - 1) / BATCH, ctas = (warps + THREADS / 32 - 1) / (THREADS / 32);
    return static_cast<unsigned>(std::min<int64_t>(ctas, 148 * 64));
}

}  // namespace

}  // namespace mc

using namespace mc;

extern "C" {

int mc_encode8(const mc_rows_desc* desc, const void* x, int8_t* codes, void* scales, void* stream)
{
    const int rc = checked_rows(desc);
    if (rc != MC_OK) return rc;
    if (desc->rows * desc->length == 0) return MC_OK;
    if (x == nullptr || codes == nullptr || scales == nullptr) { set_last_error("x, codes or scales is NULL"); return MC_ERR_INVALID_ARGUMENT; }
    const RowBlocks r = row_blocks(*desc);
    return dispatch_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        const auto kernel = quads_fit<T>(desc->length, {x}, {codes}) ? encode8_kernel<T, true> : encode8_kernel<T, false>;
        kernel<<<grid_of(r), THREADS, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const T*>(x), codes, static_cast<Wide<T>*>(scales), r);
        return check_launch("encode8_kernel");
    });
}

int mc_decode8(const mc_rows_desc* desc, const int8_t* codes, const void* scales, void* x, void* stream)
{
    const int rc = checked_rows(desc);
    if (rc != MC_OK) return rc;
    if (desc->rows * desc->length == 0) return MC_OK;
    if (x == nullptr || codes == nullptr || scales == nullptr) { set_last_error("codes, scales or x is NULL"); return MC_ERR_INVALID_ARGUMENT; }
    const RowBlocks r = row_blocks(*desc);
    return dispatch_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        const auto kernel = quads_fit<T>(desc->length, {x}, {codes}) ? decode8_kernel<T, true> : decode8_kernel<T, false>;
        kernel<<<grid_of(r), THREADS, 0, static_cast<cudaStream_t>(stream)>>>(codes, static_cast<const Wide<T>*>(scales), static_cast<T*>(x), r);
        return check_launch("decode8_kernel");
    });
}

}  // extern "C"
