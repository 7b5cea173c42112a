// Activations in 8 bits: mc_encode8 and mc_decode8. Both are one pass over memory; a warp takes whole blocks of 128.
#include "encode8.cuh"

namespace mc
{

namespace
{

/// Blocks that a warp has in flight: enough of its loads to cover their latency. Encoding holds their elements, decoding their codes.
constexpr int ENCODE_BATCH = 4, DECODE_BATCH = 8, ENCODE_HALF_BATCH = 8, DECODE_HALF_BATCH = 8;

/// How the blocks are dealt out: a unit is up to `batch` of them, a fixed distance apart, either neighbours in a row or the same block of
/// neighbouring rows. Rows of whole blocks are one long row.
struct RowBlocks
{
    int64_t length, per_row, rows;   // elements of a row, its blocks, rows
    int64_t units, units_per_row;    // units in all, and of a row (neighbours) or of a set of `batch` rows (per_row)
    int64_t step, block_step;        // elements and blocks between the blocks of a unit
    bool across;                     // a unit holds the same block of several rows
};

struct Unit
{
    int64_t start, block;   // first element, first block
    int count, valid;       // blocks; elements of the last one (neighbours) or of each (across)
};

template <int BATCH> __device__ __forceinline__ Unit unit_of(const RowBlocks& r, int64_t u)
{
    int64_t q = 0, rest = u;   // one division a unit, in 32 bits where they suffice
    if (r.units_per_row != r.units)
    {
        q = r.units <= 0xffffffffll ? static_cast<uint32_t>(u) / static_cast<uint32_t>(r.units_per_row) : u / r.units_per_row;
        rest = u - q * r.units_per_row;
    }
    const int64_t row = r.across ? q * BATCH : q, j = r.across ? rest : rest * BATCH;
    const int64_t there = r.across ? r.rows - row : r.per_row - j;   // blocks from here on
    const int count = static_cast<int>(min(static_cast<int64_t>(BATCH), there));
    const int64_t last = r.across ? j : j + count - 1;
    return {row * r.length + j * CODE_BLOCK, row * r.per_row + j, count, static_cast<int>(min(static_cast<int64_t>(CODE_BLOCK), r.length - last * CODE_BLOCK))};
}

/// Elements of block i of a unit from the lane's first on.
template <bool VEC> __device__ __forceinline__ int left_in(const RowBlocks& r, const Unit& u, int i, int lane)
{
    const int all = i >= u.count ? 0 : r.across || i == u.count - 1 ? u.valid : CODE_BLOCK;
    return all - lane_at<VEC>(lane);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) encode8_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, Wide<T>* __restrict__ scales, const RowBlocks r)
{
    constexpr int BATCH = ENCODE_BATCH;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); n < r.units; n += warps)
    {
        const Unit u = unit_of<BATCH>(r, n);
        Quad<T> q[BATCH];
        const T* from = x + u.start + lane_at<VEC>(lane);
#pragma unroll
        for (int i = 0; i < BATCH; i++, from += r.step) q[i] = load_quad<VEC>(from, left_in<VEC>(r, u, i, lane));
        Wide<T> v[BATCH][4];
        uint32_t c[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++) widen_quad(q[i], v[i]);
        const Wide<T> scale = encode_blocks(v, c, lane);
        int8_t* to = codes + u.start + lane_at<VEC>(lane);
#pragma unroll
        for (int i = 0; i < BATCH; i++, to += r.step) store_codes<VEC>(to, c[i], left_in<VEC>(r, u, i, lane));
        if (lane < u.count) scales[u.block + lane * r.block_step] = scale;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) decode8_kernel(const int8_t* __restrict__ codes, const Wide<T>* __restrict__ scales, T* __restrict__ x, const RowBlocks r)
{
    constexpr int BATCH = DECODE_BATCH;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); n < r.units; n += warps)
    {
        const Unit u = unit_of<BATCH>(r, n);
        uint32_t c[BATCH];
        const int8_t* from = codes + u.start + lane_at<VEC>(lane);
        const Wide<T> scale = lane < u.count ? __ldg(scales + u.block + lane * r.block_step) : Wide<T>(0);   // lane i has that of block i
#pragma unroll
        for (int i = 0; i < BATCH; i++, from += r.step) c[i] = load_codes<VEC>(from, left_in<VEC>(r, u, i, lane));
        T* to = x + u.start + lane_at<VEC>(lane);
#pragma unroll
        for (int i = 0; i < BATCH; i++, to += r.step)
        {
            Wide<T> v[4];
            decode_quad(c[i], __shfl_sync(0xffffffffu, scale, i), v);
            store_quad<VEC>(to, narrow_quad<T>(v), left_in<VEC>(r, u, i, lane));
        }
    }
}

/// Half precision, rows that fit loads of 16 bytes: half a warp takes a block, eight elements a lane, so that what is done once a lane
/// (addresses, conditions, the shuffle of the scale) serves twice as many elements. (32, 64, 224, 224) in bfloat16: encode 56 us
/// against 78 with four elements a lane, decode 52 against 66.
template <typename T> __device__ __forceinline__ void widen_eight(const uint4& w, float (&v)[2][4])
{
    Quad<T> q;
    q.word[0] = w.x;
    q.word[1] = w.y;
    widen_quad(q, v[0]);
    q.word[0] = w.z;
    q.word[1] = w.w;
    widen_quad(q, v[1]);
}

/// The larger magnitudes of the low and of the high halves of four words; a NaN among them stays one.
template <typename T> __device__ __forceinline__ uint32_t largest_of_pairs(const uint4& w)
{
    using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    Pair p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = __habs2(*reinterpret_cast<const Pair*>(&words[i]));
    const Pair m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
    return *reinterpret_cast<const uint32_t*>(&m);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) encode8_half_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scales, const RowBlocks r)
{
    constexpr int BATCH = ENCODE_HALF_BATCH;
    constexpr uint32_t LARGEST = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;   // infinity; NaN lies above
    const int lane = threadIdx.x & 31, half = lane >> 4, offset = 8 * (lane & 15);
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); n < r.units; n += warps)
    {
        const Unit u = unit_of<BATCH>(r, n);
        uint4 w[BATCH / 2];
        const T* from = x + u.start + half * r.step + offset;
        const auto left_of = [&](int p) {
            const int i = 2 * p + half;
            return (i >= u.count ? 0 : r.across || i == u.count - 1 ? u.valid : CODE_BLOCK) - offset;
        };
#pragma unroll
        for (int p = 0; p < BATCH / 2; p++, from += 2 * r.step)
        {
            w[p] = make_uint4(0u, 0u, 0u, 0u);
            if (left_of(p) > 0) w[p] = *reinterpret_cast<const uint4*>(from);
        }
        uint32_t mine = 0, largest = 0;
        const auto reduce = [&](int p, uint32_t m) {
            const uint32_t low = __reduce_max_sync(0xffffffffu, half == 0 ? m : 0u), high = __reduce_max_sync(0xffffffffu, half == 1 ? m : 0u);
            largest = max(largest, max(low, high));
            mine = lane == 2 * p ? low : lane == 2 * p + 1 ? high : mine;
        };
#pragma unroll
        for (int p = 0; p < BATCH / 2; p++)
        {
            const uint32_t m = largest_of_pairs<T>(w[p]);
            reduce(p, max(m >> 16, m & 0xffffu));
        }
        const bool all_finite = largest < LARGEST;
        if (!all_finite)
        {
            rarely();
#pragma unroll
            for (int p = 0; p < BATCH / 2; p++)
            {
                uint32_t m = 0;
                const uint32_t words[4] = {w[p].x, w[p].y, w[p].z, w[p].w};
#pragma unroll
                for (int k = 0; k < 8; k++)
                {
                    const uint32_t bits = (words[k / 2] >> (16 * (k % 2))) & 0x7fffu;
                    m = bits < LARGEST ? max(m, bits) : m;
                }
                reduce(p, m);
            }
        }
        float scale, inverse;
        const uint16_t top = static_cast<uint16_t>(mine);
        block_scale(widen(*reinterpret_cast<const T*>(&top)), scale, inverse);
        int8_t* to = codes + u.start + half * r.step + offset;
#pragma unroll
        for (int p = 0; p < BATCH / 2; p++, to += 2 * r.step)
        {
            const float of_block = __shfl_sync(0xffffffffu, inverse, 2 * p + half);
            float v[2][4];
            widen_eight<T>(w[p], v);
            uint2 packed;
#pragma unroll
            for (int h = 0; h < 2; h++)
            {
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; k++) q[k] = __float_as_uint(fmaf(v[h][k], of_block, 12582912.0f));
                if (!all_finite)
                {
                    rarely();
#pragma unroll
                    for (int k = 0; k < 4; k++) q[k] = isfinite(v[h][k]) ? q[k] : code_of_nonfinite(v[h][k]);
                }
                (h == 0 ? packed.x : packed.y) = pack_bytes(q);
            }
            if (left_of(p) > 0) *reinterpret_cast<uint2*>(to) = packed;
        }
        if (lane < u.count) scales[u.block + lane * r.block_step] = scale;
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) decode8_half_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ x, const RowBlocks r)
{
    constexpr int BATCH = DECODE_HALF_BATCH;
    const int lane = threadIdx.x & 31, half = lane >> 4, offset = 8 * (lane & 15);
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (THREADS / 32);
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5); n < r.units; n += warps)
    {
        const Unit u = unit_of<BATCH>(r, n);
        uint2 c[BATCH / 2];
        const int8_t* from = codes + u.start + half * r.step + offset;
        const float scale = lane < u.count ? __ldg(scales + u.block + lane * r.block_step) : 0.0f;   // lane i has that of block i
        const auto left_of = [&](int p) {
            const int i = 2 * p + half;
            return (i >= u.count ? 0 : r.across || i == u.count - 1 ? u.valid : CODE_BLOCK) - offset;
        };
#pragma unroll
        for (int p = 0; p < BATCH / 2; p++, from += 2 * r.step)
        {
            c[p] = make_uint2(0u, 0u);
            if (left_of(p) > 0) c[p] = *reinterpret_cast<const uint2*>(from);
        }
        T* to = x + u.start + half * r.step + offset;
#pragma unroll
        for (int p = 0; p < BATCH / 2; p++, to += 2 * r.step)
        {
            const float of_block = __shfl_sync(0xffffffffu, scale, 2 * p + half);
            float v[2][4];
            decode_quad(c[p].x, of_block, v[0]);
            decode_quad(c[p].y, of_block, v[1]);
            const Quad<T> low = narrow_quad<T>(v[0]), high = narrow_quad<T>(v[1]);
            if (left_of(p) > 0) *reinterpret_cast<uint4*>(to) = make_uint4(low.word[0], low.word[1], high.word[0], high.word[1]);
        }
    }
}

/// Whether rows of `length` in half precision can be read and written 16 bytes, their codes 8 bytes, at a time.
bool eights_fit(int64_t length, const void* x, const void* codes)
{
    return length % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
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

/// Rows of at least `batch` whole units go as neighbours; shorter ones, a last unit of which would be mostly empty, across rows.
RowBlocks row_blocks(const mc_rows_desc& d, int batch)
{
    RowBlocks r{};
    r.length = d.length;
    r.rows = d.rows;
    if (d.length % CODE_BLOCK == 0)
    {
        r.length *= r.rows;
        r.rows = 1;
    }
    r.per_row = code_blocks(r.length);
    const int64_t within = (r.per_row + batch - 1) / batch * r.rows, across = (r.rows + batch - 1) / batch * r.per_row;
    r.across = across < within;
    r.units = std::min(within, across);
    r.units_per_row = r.across ? r.per_row : r.units / r.rows;
    r.step = r.across ? r.length : CODE_BLOCK;
    r.block_step = r.across ? r.per_row : 1;
    return r;
}

unsigned grid_of(const RowBlocks& r)
{
    return static_cast<unsigned>(std::min<int64_t>((r.units + THREADS / 32 - 1) / (THREADS / 32), 148 * 64));
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
    return dispatch_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2)
        {
            if (eights_fit(desc->length, x, codes))
            {
                const RowBlocks r = row_blocks(*desc, ENCODE_HALF_BATCH);
                encode8_half_kernel<T><<<grid_of(r), THREADS, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const T*>(x), codes, static_cast<float*>(scales), r);
                return check_launch("encode8_half_kernel");
            }
        }
        const RowBlocks r = row_blocks(*desc, ENCODE_BATCH);
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
    return dispatch_dtype(desc->dtype, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2)
        {
            if (eights_fit(desc->length, x, codes))
            {
                const RowBlocks r = row_blocks(*desc, DECODE_HALF_BATCH);
                decode8_half_kernel<T><<<grid_of(r), THREADS, 0, static_cast<cudaStream_t>(stream)>>>(codes, static_cast<const float*>(scales), static_cast<T*>(x), r);
                return check_launch("decode8_half_kernel");
            }
        }
        const RowBlocks r = row_blocks(*desc, DECODE_BATCH);
        const auto kernel = quads_fit<T>(desc->length, {x}, {codes}) ? decode8_kernel<T, true> : decode8_kernel<T, false>;
        kernel<<<grid_of(r), THREADS, 0, static_cast<cudaStream_t>(stream)>>>(codes, static_cast<const Wide<T>*>(scales), static_cast<T*>(x), r);
        return check_launch("decode8_kernel");
    });
}

}  // extern "C"
