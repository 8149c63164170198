// Entries of a table by index, the order of points by their index, and the table's gradient summed in that order (gfx950).
//
// All are bound by memory: the lookup and the gradient by scattered requests (of 4 bytes a channel in the columns layout,
// of whole rows in the rows layout), the order by the passes of its sort.
#include <algorithm>

#include "abi_common.h"

#include "../../include/trips_lookup.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int64_t kMostEntries = 0x7ffffffell;  // texels or points: positions and T + 1 starts in 32 bits
constexpr int kMostChannels    = 1 << 20;  // a grid's y holds 65535 groups of 16

template <bool I32>
__device__ __forceinline__ long long load_index(const void* index, long long i)
{
    if constexpr (I32)
        return reinterpret_cast<const int32_t*>(index)[i];
    else
        return reinterpret_cast<const int64_t*>(index)[i];
}
__device__ __forceinline__ long long load_index(bool i32, const void* index, long long i)
{
    return i32 ? load_index<true>(index, i) : load_index<false>(index, i);
}

struct LookupParams
{
    const void* table;   // or d_values
    const void* index;   // or NULL
    void* values;        // or d_table
    const int32_t* order;
    const int32_t* starts;
    long long texels, points, table_stride, values_stride;
    int channels, i32, accumulate;
    float scale;
};

// ---- lookup ----

// One point a lane; channels in groups of kColumnGroup along grid.y.
constexpr int kColumnGroup = 16;
template <int D>
__global__ __launch_bounds__(256) void lookup_columns_kernel(const LookupParams p)
{
    using E = Element<D>;
    using T = typename E::type;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.points) return;
    const long long t = load_index(p.i32 != 0, p.index, i);
    const bool in     = t >= 0 && t < p.texels;
    const int c0 = blockIdx.y * kColumnGroup, c1 = min(c0 + kColumnGroup, p.channels);
    for (int c = c0; c < c1; ++c)
    {
        const float x = in ? E::to_float(reinterpret_cast<const T*>(p.table)[c * p.table_stride + t]) : 0.f;
        reinterpret_cast<T*>(p.values)[c * p.values_stride + i] = E::from_float(in ? x * p.scale : 0.f);
    }
}

// LANES lanes a point, 16 bytes a lane and step.
template <int D>
__global__ __launch_bounds__(256) void lookup_rows_kernel(const LookupParams p, int lanes_log2)
{
    using E         = Element<D>;
    using T         = typename E::type;
    constexpr int V = 16 / sizeof(T);
    const int lanes = 1 << lanes_log2, j = threadIdx.x & (lanes - 1);
    const long long step = (long long)gridDim.x * (256 >> lanes_log2);
    for (long long i = (long long)blockIdx.x * (256 >> lanes_log2) + (threadIdx.x >> lanes_log2); i < p.points; i += step)
    {
        const long long t = load_index(p.i32 != 0, p.index, i);
        const bool in     = t >= 0 && t < p.texels;
        const T* from     = reinterpret_cast<const T*>(p.table) + (in ? t : 0) * p.table_stride;
        T* to             = reinterpret_cast<T*>(p.values) + i * p.values_stride;
        for (int c = j * V; c < p.channels; c += lanes * V)
        {
            if (c + V <= p.channels)
            {
                typename Pack<T, V>::type x = {};
                if (in) x = *reinterpret_cast<const typename Pack<T, V>::type*>(from + c);
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = in ? E::from_float(E::to_float(x[e]) * p.scale) : T(0);
                *reinterpret_cast<typename Pack<T, V>::type*>(to + c) = x;
            }
            else
                for (int e = c; e < p.channels; ++e) to[e] = in ? E::from_float(E::to_float(from[e]) * p.scale) : T(0);
        }
    }
}

// ---- the order of the points: a stable radix sort, least significant digit first ----

constexpr int kSortThreads = 256, kSortItems = 16, kSortTile = kSortThreads * kSortItems;
constexpr int kDigits = 256;

struct SortParams
{
    const void* index;        // first pass
    const uint32_t* keys_in;  // later passes
    const int32_t* points_in;
    uint32_t* keys_out;
    int32_t* points_out;
    uint32_t* hist;    // [kDigits][tiles]: of each digit, its keys in each tile; then those in the tiles before
    uint32_t* totals;  // [kDigits]
    uint32_t n, texels, tiles;
    int first, i32, shift, bits;
};

// A point's key: its texel, or T outside the table.
__device__ __forceinline__ uint32_t sort_key(const SortParams& p, uint32_t i)
{
    if (!p.first) return p.keys_in[i];
    const long long t = load_index(p.i32 != 0, p.index, i);
    return t >= 0 && t < (long long)p.texels ? (uint32_t)t : p.texels;
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const SortParams p)
{
    __shared__ uint32_t s[kDigits];
    s[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t mask = (1u << p.bits) - 1u;
    for (int k = 0; k < kSortItems; ++k)
    {
        const uint32_t i = blockIdx.x * (uint32_t)kSortTile + k * kSortThreads + threadIdx.x;
        if (i < p.n) atomicAdd(&s[(sort_key(p, i) >> p.shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x <= mask) p.hist[(size_t)threadIdx.x * p.tiles + blockIdx.x] = s[threadIdx.x];
}

// Sum over the threads of the workgroup up to this one, itself included; s: 4 words.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* s)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
    {
        const uint32_t y = (uint32_t)__shfl_up((int)x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) s[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x += s[w];
    __syncthreads();
    return x;
}

// One workgroup a digit: its counts become the sums of the tiles before.
__global__ __launch_bounds__(kSortThreads) void sort_scan_kernel(const SortParams p)
{
    __shared__ uint32_t s[4], s_sum;
    uint32_t* row  = p.hist + (size_t)blockIdx.x * p.tiles;
    uint32_t before = 0;
    for (uint32_t base = 0; base < p.tiles; base += kSortThreads)
    {
        const uint32_t i = base + threadIdx.x;
        const uint32_t x = i < p.tiles ? row[i] : 0u;
        const uint32_t y = block_scan(x, s);
        if (i < p.tiles) row[i] = before + y - x;
        if (threadIdx.x == kSortThreads - 1) s_sum = y;
        __syncthreads();
        before += s_sum;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.totals[blockIdx.x] = before;
}

// A tile's keys go to their places. A wavefront takes 64 keys after the other, the keys of equal digit found by ballots; the
// tile is put in order in LDS first, so that each digit's keys leave side by side.
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(const SortParams p)
{
    __shared__ uint32_t s_count[4][kDigits];  // keys of a digit in each wavefront, then those of the tile before them
    __shared__ uint32_t s_place[kDigits];     // of the tile's first key of a digit: its place, less its place in the tile
    __shared__ uint32_t s_key[kSortTile];
    __shared__ int32_t s_point[kSortTile];
    __shared__ uint32_t s_scan[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t mask  = (1u << p.bits) - 1u;
    const uint32_t begin = blockIdx.x * (uint32_t)kSortTile;
    const uint32_t count = min((uint32_t)kSortTile, p.n - begin);
    for (int w = 0; w < 4; ++w) s_count[w][threadIdx.x] = 0;
    __syncthreads();
    uint32_t key[kSortItems], rank[kSortItems];
    int32_t point[kSortItems];
    const uint32_t mine = wave * (uint32_t)(kSortTile / 4) + lane;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
    {
        const uint32_t i = mine + k * 64;
        key[k]   = i < count ? sort_key(p, begin + i) : ~0u;
        point[k] = i < count ? (p.first ? (int32_t)(begin + i) : p.points_in[begin + i]) : 0;
    }
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
    {
        const bool in        = mine + k * 64 < count;
        const uint32_t digit = (key[k] >> p.shift) & mask;
        unsigned long long same = __ballot(in);
        for (int b = 0; b < p.bits; ++b)
        {
            const bool set = (digit >> b) & 1u;
            const unsigned long long v = __ballot(set);
            same &= set ? v : ~v;
        }
        const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        uint32_t base = 0;
        if (in) base = s_count[wave][digit];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in && before == 0) s_count[wave][digit] = base + (uint32_t)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[k] = base + before;
    }
    __syncthreads();
    {
        const int d = threadIdx.x;
        uint32_t c[4], sum = 0;
        for (int w = 0; w < 4; ++w) c[w] = s_count[w][d], sum += c[w];
        const uint32_t in_tile = block_scan(sum, s_scan) - sum;  // the tile's keys of lower digits
        for (uint32_t w = 0, x = in_tile; w < 4; ++w) s_count[w][d] = x, x += c[w];
        const uint32_t total = d <= (int)mask ? p.totals[d] : 0u;
        const uint32_t below = block_scan(total, s_scan) - total;  // all keys of lower digits
        if (d <= (int)mask) s_place[d] = below + p.hist[(size_t)d * p.tiles + blockIdx.x] - in_tile;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
    {
        if (mine + k * 64 >= count) continue;
        const uint32_t at = s_count[wave][(key[k] >> p.shift) & mask] + rank[k];
        s_key[at]   = key[k];
        s_point[at] = point[k];
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < count; at += kSortThreads)
    {
        const uint32_t k  = s_key[at];
        const uint32_t to = s_place[(k >> p.shift) & mask] + at;
        p.keys_out[to]    = k;
        p.points_out[to]  = s_point[at];
    }
}

// starts[t] = the first of the sorted keys that is t or more
__global__ __launch_bounds__(256) void starts_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t texels, int32_t* starts)
{
    const uint32_t t = blockIdx.x * 256u + threadIdx.x;
    if (t > texels) return;
    uint32_t lo = 0, hi = n;
    while (lo < hi)
    {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] < t)
            lo = mid + 1;
        else
            hi = mid;
    }
    starts[t] = (int32_t)lo;
}

// ---- the gradient ----

__device__ __forceinline__ void segment(const LookupParams& p, long long t, uint32_t& from, uint32_t& to)
{
    // (a plan of another scene must not lead outside)
    from = min((uint32_t)p.starts[t], (uint32_t)p.points);
    to   = max(from, min((uint32_t)p.starts[t + 1], (uint32_t)p.points));
}

template <int D>
__global__ __launch_bounds__(256) void lookup_backward_columns_kernel(const LookupParams p)
{
    using E = Element<D>;
    using T = typename E::type;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t >= p.texels) return;
    uint32_t from, to;
    segment(p, t, from, to);
    const int c0 = blockIdx.y * kColumnGroup;
    float sum[kColumnGroup];
#pragma unroll
    for (int c = 0; c < kColumnGroup; ++c) sum[c] = 0.f;
    for (uint32_t k = from; k < to; ++k)
    {
        const uint32_t i = (uint32_t)p.order[k];
        if (i >= (uint32_t)p.points) continue;
#pragma unroll
        for (int c = 0; c < kColumnGroup; ++c)
            if (c0 + c < p.channels) sum[c] += E::to_float(reinterpret_cast<const T*>(p.table)[(c0 + c) * p.values_stride + i]);
    }
#pragma unroll
    for (int c = 0; c < kColumnGroup; ++c)
    {
        if (c0 + c >= p.channels) break;
        T* to_ = reinterpret_cast<T*>(p.values) + (c0 + c) * p.table_stride + t;
        if (p.accumulate)
        {
            if (from < to) *to_ = E::from_float(E::to_float(*to_) + p.scale * sum[c]);
        }
        else
            *to_ = E::from_float(p.scale * sum[c]);
    }
}

template <int D>
__global__ __launch_bounds__(256) void lookup_backward_rows_kernel(const LookupParams p, int lanes_log2)
{
    using E         = Element<D>;
    using T         = typename E::type;
    constexpr int V = 16 / sizeof(T);
    const int lanes = 1 << lanes_log2, j = threadIdx.x & (lanes - 1);
    const long long step = (long long)gridDim.x * (256 >> lanes_log2);
    for (long long t = (long long)blockIdx.x * (256 >> lanes_log2) + (threadIdx.x >> lanes_log2); t < p.texels; t += step)
    {
        uint32_t from, to;
        segment(p, t, from, to);
        if (p.accumulate && from == to) continue;
        T* out = reinterpret_cast<T*>(p.values) + t * p.table_stride;
        for (int c = j * V; c < p.channels; c += lanes * V)
        {
            const int count = min(V, p.channels - c);
            float sum[V];
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] = 0.f;
            for (uint32_t k = from; k < to; ++k)
            {
                const uint32_t i = (uint32_t)p.order[k];
                if (i >= (uint32_t)p.points) continue;
                const T* row = reinterpret_cast<const T*>(p.table) + (long long)i * p.values_stride + c;
                if (count == V)
                {
                    const auto x = *reinterpret_cast<const typename Pack<T, V>::type*>(row);
#pragma unroll
                    for (int e = 0; e < V; ++e) sum[e] += E::to_float(x[e]);
                }
                else
                {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e < count) sum[e] += E::to_float(row[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < count) out[c + e] = E::from_float(p.accumulate ? E::to_float(out[c + e]) + p.scale * sum[e] : p.scale * sum[e]);
        }
    }
}

// ---- host ----

constexpr long long kMostRowGroups = 1 << 20;  // a launch has less than 2^32 threads

int lanes_log2_of(int channels, int dtype)
{
    const int v = 16 / dtype_bytes(dtype), chunks = (channels + v - 1) / v;
    int l = 0;
    while ((1 << l) < chunks && l < 6) ++l;
    return l;
}

int key_bits(int64_t texels)
{
    int bits = 1;  // of T itself, the key of what is outside
    while ((int64_t)1 << bits <= texels) ++bits;
    return bits;
}

struct PlanLayout
{
    size_t keys[2], points, hist, totals, bytes;
};
PlanLayout plan_layout(int64_t points)
{
    auto up            = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t tiles = (size_t)((points + kSortTile - 1) / kSortTile);
    PlanLayout l;
    size_t o  = 0;
    l.keys[0] = o, o += up((size_t)points * 4);
    l.keys[1] = o, o += up((size_t)points * 4);
    l.points = o, o += up((size_t)points * 4);
    l.hist = o, o += up(tiles * kDigits * 4);
    l.totals = o, o += up(kDigits * 4);
    l.bytes = o;
    return l;
}

hipError_t launch_plan(int64_t texels, int64_t points, const void* index, int index_dtype, int32_t* order, int32_t* starts, char* ws,
                       hipStream_t stream, Profiler* prof)
{
    const PlanLayout l = plan_layout(points);
    const int bits     = key_bits(texels), passes = (bits + 7) / 8;
    SortParams p;
    p.index = index, p.i32 = index_dtype == TRIPS_INDEX_I32, p.n = (uint32_t)points, p.texels = (uint32_t)texels;
    p.tiles = (uint32_t)((points + kSortTile - 1) / kSortTile);
    p.hist = reinterpret_cast<uint32_t*>(ws + l.hist), p.totals = reinterpret_cast<uint32_t*>(ws + l.totals);
    p.keys_out = nullptr, p.points_out = nullptr;
    ProfScope ps(prof, "lookup_plan", stream);
    int shift = 0;
    for (int pass = 0; pass < passes && points > 0; ++pass)
    {
        p.first = pass == 0, p.shift = shift, p.bits = (bits - shift + passes - pass - 1) / (passes - pass);
        p.keys_in    = p.keys_out;
        p.points_in  = p.points_out;
        p.keys_out   = reinterpret_cast<uint32_t*>(ws + l.keys[pass & 1]);
        p.points_out = (passes - 1 - pass) % 2 == 0 ? order : reinterpret_cast<int32_t*>(ws + l.points);
        hipLaunchKernelGGL(sort_count_kernel, dim3(p.tiles), dim3(kSortThreads), 0, stream, p);
        hipLaunchKernelGGL(sort_scan_kernel, dim3(1 << p.bits), dim3(kSortThreads), 0, stream, p);
        hipLaunchKernelGGL(sort_scatter_kernel, dim3(p.tiles), dim3(kSortThreads), 0, stream, p);
        shift += p.bits;
    }
    hipLaunchKernelGGL(starts_kernel, dim3((unsigned)(texels / 256 + 1)), dim3(256), 0, stream, p.keys_out, (uint32_t)points,
                       (uint32_t)texels, starts);
    return hipGetLastError();
}

int check_lookup(const TripsLookupDesc* d)
{
    if (!d) return set_error(TRIPS_ERR_INVALID_ARG, "desc is NULL");
    if (d->abi_version != TRIPS_ABI_VERSION) return set_error(TRIPS_ERR_INVALID_ARG, "abi_version %d, library has %d", d->abi_version, TRIPS_ABI_VERSION);
    if (d->layout != TRIPS_TABLE_COLUMNS && d->layout != TRIPS_TABLE_ROWS) return set_error(TRIPS_ERR_INVALID_ARG, "layout %d", d->layout);
    if (!dtype_ok(d->dtype)) return set_error(TRIPS_ERR_UNSUPPORTED, "dtype %d (float32, bfloat16 and float16 are supported)", d->dtype);
    if (d->index_dtype != TRIPS_INDEX_I64 && d->index_dtype != TRIPS_INDEX_I32) return set_error(TRIPS_ERR_UNSUPPORTED, "index_dtype %d", d->index_dtype);
    if (d->num_texels < 0 || d->num_texels > kMostEntries) return set_error(TRIPS_ERR_INVALID_ARG, "num_texels = %lld", (long long)d->num_texels);
    if (d->num_points < 0 || d->num_points > kMostEntries) return set_error(TRIPS_ERR_INVALID_ARG, "num_points = %lld", (long long)d->num_points);
    if (d->num_channels < 1 || d->num_channels >= kMostChannels) return set_error(TRIPS_ERR_INVALID_ARG, "num_channels = %d", d->num_channels);
    return TRIPS_OK;
}

// Strides of what is written must keep its rows apart; what is read may repeat a row.
int check_stride(const char* name, int64_t stride, int64_t row, int64_t rows, bool written)
{
    if (stride < 0 || stride > ((int64_t)1 << 48) || (written && rows > 1 && stride < row))
        return set_error(TRIPS_ERR_INVALID_ARG, "%s %lld (rows have %lld elements)", name, (long long)stride, (long long)row);
    return TRIPS_OK;
}

hipError_t launch_lookup(const TripsLookupDesc& d, const LookupParams& p, hipStream_t stream, Profiler* prof)
{
    ProfScope ps(prof, "lookup", stream);
    if (d.layout == TRIPS_TABLE_COLUMNS)
    {
        const dim3 grid((unsigned)((d.num_points + 255) / 256), (unsigned)((d.num_channels + kColumnGroup - 1) / kColumnGroup));
        if (d.dtype == TRIPS_DTYPE_F32)
            hipLaunchKernelGGL(lookup_columns_kernel<TRIPS_DTYPE_F32>, grid, dim3(256), 0, stream, p);
        else if (d.dtype == TRIPS_DTYPE_BF16)
            hipLaunchKernelGGL(lookup_columns_kernel<TRIPS_DTYPE_BF16>, grid, dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL(lookup_columns_kernel<TRIPS_DTYPE_F16>, grid, dim3(256), 0, stream, p);
    }
    else
    {
        const int l = lanes_log2_of(d.num_channels, d.dtype);
        const dim3 grid((unsigned)std::min<long long>(((d.num_points << l) + 255) / 256, kMostRowGroups));
        if (d.dtype == TRIPS_DTYPE_F32)
            hipLaunchKernelGGL(lookup_rows_kernel<TRIPS_DTYPE_F32>, grid, dim3(256), 0, stream, p, l);
        else if (d.dtype == TRIPS_DTYPE_BF16)
            hipLaunchKernelGGL(lookup_rows_kernel<TRIPS_DTYPE_BF16>, grid, dim3(256), 0, stream, p, l);
        else
            hipLaunchKernelGGL(lookup_rows_kernel<TRIPS_DTYPE_F16>, grid, dim3(256), 0, stream, p, l);
    }
    return hipGetLastError();
}

hipError_t launch_lookup_backward(const TripsLookupDesc& d, const LookupParams& p, hipStream_t stream, Profiler* prof)
{
    ProfScope ps(prof, "lookup_backward", stream);
    if (d.layout == TRIPS_TABLE_COLUMNS)
    {
        const dim3 grid((unsigned)((d.num_texels + 255) / 256), (unsigned)((d.num_channels + kColumnGroup - 1) / kColumnGroup));
        if (d.dtype == TRIPS_DTYPE_F32)
            hipLaunchKernelGGL(lookup_backward_columns_kernel<TRIPS_DTYPE_F32>, grid, dim3(256), 0, stream, p);
        else if (d.dtype == TRIPS_DTYPE_BF16)
            hipLaunchKernelGGL(lookup_backward_columns_kernel<TRIPS_DTYPE_BF16>, grid, dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL(lookup_backward_columns_kernel<TRIPS_DTYPE_F16>, grid, dim3(256), 0, stream, p);
    }
    else
    {
        const int l = lanes_log2_of(d.num_channels, d.dtype);
        const dim3 grid((unsigned)std::min<long long>(((d.num_texels << l) + 255) / 256, kMostRowGroups));
        if (d.dtype == TRIPS_DTYPE_F32)
            hipLaunchKernelGGL(lookup_backward_rows_kernel<TRIPS_DTYPE_F32>, grid, dim3(256), 0, stream, p, l);
        else if (d.dtype == TRIPS_DTYPE_BF16)
            hipLaunchKernelGGL(lookup_backward_rows_kernel<TRIPS_DTYPE_BF16>, grid, dim3(256), 0, stream, p, l);
        else
            hipLaunchKernelGGL(lookup_backward_rows_kernel<TRIPS_DTYPE_F16>, grid, dim3(256), 0, stream, p, l);
    }
    return hipGetLastError();
}

LookupParams params_of(const TripsLookupDesc& d)
{
    LookupParams p;
    p.table = p.index = nullptr, p.values = nullptr, p.order = p.starts = nullptr;
    p.texels = d.num_texels, p.points = d.num_points, p.table_stride = d.table_stride, p.values_stride = d.values_stride;
    p.channels = d.num_channels, p.i32 = d.index_dtype == TRIPS_INDEX_I32, p.accumulate = d.accumulate != 0, p.scale = d.scale;
    return p;
}
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" {

int trips_lookup_forward(TripsCtx* ctx, const TripsLookupDesc* desc, const void* table, const void* index, void* values, void* stream)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (int e = check_lookup(desc)) return e;
    const TripsLookupDesc& d = *desc;
    const bool columns       = d.layout == TRIPS_TABLE_COLUMNS;
    if (int e = check_stride("table_stride", d.table_stride, columns ? d.num_texels : d.num_channels, columns ? d.num_channels : d.num_texels, false)) return e;
    if (int e = check_stride("values_stride", d.values_stride, columns ? d.num_points : d.num_channels, columns ? d.num_channels : d.num_points, true)) return e;
    if (d.num_points == 0) return TRIPS_OK;
    const size_t size = dtype_bytes(d.dtype);
    if (!index || !aligned(index, d.index_dtype == TRIPS_INDEX_I32 ? 4 : 8)) return set_error(TRIPS_ERR_INVALID_ARG, "index is NULL or not aligned");
    if ((!table && d.num_texels > 0) || !aligned(table, size)) return set_error(TRIPS_ERR_INVALID_ARG, "table is NULL or not aligned");
    if (!values || !aligned(values, size)) return set_error(TRIPS_ERR_INVALID_ARG, "values is NULL or not aligned");
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    LookupParams p = params_of(d);
    p.table = table, p.index = index, p.values = values;
    hipError_t e = launch_lookup(d, p, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "lookup launch");
}

int trips_lookup_plan_workspace_size(int64_t num_texels, int64_t num_points, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (num_texels < 0 || num_texels > kMostEntries) return set_error(TRIPS_ERR_INVALID_ARG, "num_texels = %lld", (long long)num_texels);
    if (num_points < 0 || num_points > kMostEntries) return set_error(TRIPS_ERR_INVALID_ARG, "num_points = %lld", (long long)num_points);
    *bytes = plan_layout(num_points).bytes;
    return TRIPS_OK;
}

int trips_lookup_plan(TripsCtx* ctx, int64_t num_texels, int64_t num_points, const void* index, int index_dtype, int32_t* order,
                      int32_t* starts, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    size_t need = 0;
    if (int e = trips_lookup_plan_workspace_size(num_texels, num_points, &need)) return e;
    if (index_dtype != TRIPS_INDEX_I64 && index_dtype != TRIPS_INDEX_I32) return set_error(TRIPS_ERR_UNSUPPORTED, "index_dtype %d", index_dtype);
    if (!starts || !aligned(starts, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "starts is NULL or not aligned");
    if (num_points > 0)
    {
        if (!index || !aligned(index, index_dtype == TRIPS_INDEX_I32 ? 4 : 8)) return set_error(TRIPS_ERR_INVALID_ARG, "index is NULL or not aligned");
        if (!order || !aligned(order, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "order is NULL or not aligned");
        if (!workspace || !aligned(workspace, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
        if (workspace_bytes < need) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %zu needed", workspace_bytes, need);
    }
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    hipError_t e = launch_plan(num_texels, num_points, index, index_dtype, order, starts, reinterpret_cast<char*>(workspace),
                               reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "plan launch");
}

int trips_lookup_backward_workspace_size(const TripsLookupDesc* desc, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (int e = check_lookup(desc)) return e;
    *bytes = 0;
    return TRIPS_OK;
}

int trips_lookup_backward(TripsCtx* ctx, const TripsLookupDesc* desc, const void* d_values, const int32_t* order,
                          const int32_t* starts, void* d_table, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (int e = check_lookup(desc)) return e;
    const TripsLookupDesc& d = *desc;
    const bool columns       = d.layout == TRIPS_TABLE_COLUMNS;
    if (int e = check_stride("table_stride", d.table_stride, columns ? d.num_texels : d.num_channels, columns ? d.num_channels : d.num_texels, true)) return e;
    if (int e = check_stride("values_stride", d.values_stride, columns ? d.num_points : d.num_channels, columns ? d.num_channels : d.num_points, false)) return e;
    if (d.num_texels == 0) return TRIPS_OK;
    const size_t size = dtype_bytes(d.dtype);
    if (!starts || !aligned(starts, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "starts is NULL or not aligned");
    if (!d_table || !aligned(d_table, size)) return set_error(TRIPS_ERR_INVALID_ARG, "d_table is NULL or not aligned");
    if (d.num_points > 0 && (!order || !aligned(order, 4) || !d_values || !aligned(d_values, size)))
        return set_error(TRIPS_ERR_INVALID_ARG, "order or d_values is NULL or not aligned");
    size_t need = 0;
    if (int e = trips_lookup_backward_workspace_size(desc, &need)) return e;
    if (need > 0 && (!workspace || !aligned(workspace, 256))) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
    if (workspace_bytes < need) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %zu needed", workspace_bytes, need);
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    LookupParams p = params_of(d);
    p.table = d_values, p.values = d_table, p.order = order, p.starts = starts;
    hipError_t e = launch_lookup_backward(d, p, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "lookup backward launch");
}

}  // extern "C"
