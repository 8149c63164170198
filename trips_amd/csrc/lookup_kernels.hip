// Entries of a table by index, the order of points by their index, and the table's gradient summed in that order (gfx950).
//
//   values[i] = scale table[index[i]]          d_table[t] (+)= scale sum of d_values[i] over the i with index[i] = t, in their order
//
// Large calls are bound by memory: lookup and gradient in no order by the lines of 128 bytes that each scattered request moves
// (7 TB/s of lines), short ones and those of whole rows by latency or by the table's bytes; the order of the points by the three
// passes of its sort. us a call: 6M points of 1.5M texels in four channels 117, their gradient 157, their order 132; 8191 tokens of
// a table of 50,000 rows of 1024 bfloat16 numbers 7.5, order and gradient 42 to 47. Below each kernel its own share.
#include <algorithm>
#include <type_traits>

#include "abi_common.h"

#include "../../include/trips_lookup.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int64_t kMostEntries = 0x7ffffffell;  // texels or points: positions and T + 1 starts in 32 bits
constexpr int kMostChannels    = 1 << 17;  // lanes of 16 bytes that a grid's y holds

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
    const void* table;
    const void* index;
    void* values;
    long long texels, points, table_stride, values_stride;
    int channels, i32, lanes_log2;
    float scale;
};

// ---- columns to rows ----

// [channels, n] to [n, row] with 16 bytes (8 where two or four channels of 16 bits make no more) a lane: what the kernels below
// gather is then one request of a point, not one per channel. Bound by memory, read and written once (6M points in four channels
// of 32 bits 30 us, 6.4 TB/s).
// (row: channels rounded up to whole lanes; the elements added are zeros.)
template <int D, int V>
__global__ __launch_bounds__(256) void rows_kernel(const void* columns, void* rows, long long n, long long stride, int channels, int row)
{
    using T           = typename Element<D>::type;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int c0   = blockIdx.y * V;
    const T* from  = reinterpret_cast<const T*>(columns) + i;
    typename Pack<T, V>::type x;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = c0 + e < channels ? from[(c0 + e) * stride] : T(0);
    *reinterpret_cast<typename Pack<T, V>::type*>(reinterpret_cast<T*>(rows) + i * row + c0) = x;
}

// ---- lookup ----

// One point a lane; channels in groups of kColumnGroup along grid.y. For one channel, and for so few points that turning the
// table's columns to rows would cost more than it saves.
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

// V elements a lane, 1 << lanes_log2 lanes a point. OUT_COLUMNS: the values are columns (and the table's rows whole lanes wide).
// 6M points of 24 MB of rows in no order: 107 us, 6.0M lines of 128 bytes that no L2 holds (7.1 TB/s of them; an XCD's L2 has 4 MB).
// 8191 rows of 1024 bfloat16 numbers: 7.9 us where it starts alone, 5.4 for the bytes: an index, then its row, in one wave of workgroups.
template <int D, int V, bool OUT_COLUMNS>
__global__ __launch_bounds__(256) void lookup_rows_kernel(const LookupParams p)
{
    using E = Element<D>;
    using T = typename E::type;
    const int lanes = 1 << p.lanes_log2, j = threadIdx.x & (lanes - 1), at_once = 256 >> p.lanes_log2;
    const T* table       = reinterpret_cast<const T*>(p.table);
    T* values            = reinterpret_cast<T*>(p.values);
    // whose rows a lane has on the way at a time (of eight columns the addresses of four points took 188 registers: 2M points of 500,000
    // texels in 16 bfloat16 channels 62 us, with two 57)
    constexpr int POINTS = OUT_COLUMNS && V == 8 ? 2 : 4;
    for (long long base = (long long)blockIdx.x * at_once * POINTS; base < p.points; base += (long long)gridDim.x * at_once * POINTS)
    {
        long long t[POINTS];
        auto load = [&](auto i32)
        {
#pragma unroll
            for (int q = 0; q < POINTS; ++q)
                t[q] = load_index<decltype(i32)::value>(p.index, min(base + q * at_once + (threadIdx.x >> p.lanes_log2), p.points - 1));
        };
        if (p.i32)  // (not at each load: they would wait for one another)
            load(std::true_type{});
        else
            load(std::false_type{});
#pragma unroll
        for (int q = 0; q < POINTS; ++q)
            if (t[q] >= p.texels) t[q] = -1;
        for (int c = j * V; c < p.channels; c += lanes * V)
        {
            const int count = OUT_COLUMNS ? V : min(V, p.channels - c);
            typename Pack<T, V>::type x[POINTS];
#pragma unroll
            for (int q = 0; q < POINTS; ++q)
            {
                x[q] = typename Pack<T, V>::type{};
                if (t[q] < 0) continue;
                const T* from = table + t[q] * p.table_stride + c;
                if (count == V)
                    x[q] = *reinterpret_cast<const typename Pack<T, V>::type*>(from);
                else
                {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e < count) x[q][e] = from[e];
                }
            }
#pragma unroll
            for (int q = 0; q < POINTS; ++q)
            {
                const long long i = base + q * at_once + (threadIdx.x >> p.lanes_log2);
                if (i >= p.points) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) x[q][e] = t[q] >= 0 ? E::from_float(E::to_float(x[q][e]) * p.scale) : T(0);
                if constexpr (OUT_COLUMNS)
                {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (c + e < p.channels) __builtin_nontemporal_store(x[q][e], values + (c + e) * p.values_stride + i);
                }
                else if (count == V)
                    *reinterpret_cast<typename Pack<T, V>::type*>(values + i * p.values_stride + c) = x[q];
                else
                {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e < count) values[i * p.values_stride + c + e] = x[q][e];
                }
            }
        }
    }
}

// ---- the order of the points: a stable radix sort, least significant digit first ----

// A tile: 1024 threads with 2 points each below 2^20 points, with 4 below 2^22, with 6 above (two tiles a CU at a time in any case;
// us: 20k points, by passes, 22 with 2 and 31 with 8 of 512 threads, 1M 56 and with 6 59, 2M 68 with 4 and 74 with 6, 6M 147 with 4 and 132 with 6).
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int sort_items(int64_t points) { return points < (1 << 20) ? 2 : points < (1 << 22) ? 4 : 6; }
constexpr int kDigits = 256;
constexpr uint32_t kFewTiles = 32;  // so few that each tile's workgroup sums the counts of the others itself: a launch less a pass

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
    int shift, bits;
};

// Where keys come from: the pass before, or the index, of 32 or 64 bits. (A constant of the kernels: with a branch at each load the
// loads waited for one another: a pass over 6M points 34 us and 32, the count before it 9 and 8.)
enum { kFromKeys = 0, kFromI32 = 1, kFromI64 = 2 };

// A point's key: its texel, or T outside the table.
template <int FROM>
__device__ __forceinline__ uint32_t sort_key(const SortParams& p, uint32_t i)
{
    if constexpr (FROM == kFromKeys) return p.keys_in[i];
    const long long t = load_index<FROM == kFromI32>(p.index, i);
    return t >= 0 && t < (long long)p.texels ? (uint32_t)t : p.texels;
}

// Bound by memory and by launching: 6M keys 7 us.
template <int ITEMS, int FROM>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const SortParams p)
{
    constexpr int kSortItems = ITEMS, kSortTile = kSortThreads * ITEMS;
    __shared__ uint32_t s[kDigits];
    const uint32_t first = blockIdx.x * (uint32_t)kSortTile + threadIdx.x;
    uint32_t key[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) key[k] = sort_key<FROM>(p, min(first + k * kSortThreads, p.n - 1u));
    if (threadIdx.x < kDigits) s[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t mask = (1u << p.bits) - 1u;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
        if (first + k * kSortThreads < p.n) atomicAdd(&s[(key[k] >> p.shift) & mask], 1u);
    __syncthreads();
    if (threadIdx.x <= mask) p.hist[(size_t)threadIdx.x * p.tiles + blockIdx.x] = s[threadIdx.x];
}

// Sum over the threads of the workgroup up to this one, itself included; s: a word a wavefront.
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

constexpr int kScanThreads = 1024;
// One workgroup a digit: its counts become the sums of the tiles before. (977 tiles 4.8 us, nearly all of it latency.)
__global__ __launch_bounds__(kScanThreads) void sort_scan_kernel(const SortParams p)
{
    __shared__ uint32_t s[kScanThreads / 64], s_sum;
    uint32_t* row   = p.hist + (size_t)blockIdx.x * p.tiles;
    uint32_t before = 0;
    for (uint32_t base = 0; base < p.tiles; base += kScanThreads)
    {
        const uint32_t i = base + threadIdx.x;
        const uint32_t x = i < p.tiles ? row[i] : 0u;
        const uint32_t y = block_scan(x, s);
        if (i < p.tiles) row[i] = before + y - x;
        if (threadIdx.x == kScanThreads - 1) s_sum = y;
        __syncthreads();
        before += s_sum;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.totals[blockIdx.x] = before;
}

// Ranks of a wavefront's keys among its keys of the same digit: ITEMS rounds of 64 keys, the keys of a round that share a digit
// found by ballots. The first of them adds their number to the digit's count in LDS; LDS serves a wavefront in order, so no round
// waits for the one before. `count`: the wavefront's counts, zeros before, its keys of each digit behind a barrier.
template <int ITEMS>
__device__ __forceinline__ void rank_keys(const uint32_t (&key)[ITEMS], uint32_t valid, int shift, int bits, uint32_t* count, uint32_t (&rank)[ITEMS])
{
    const int lane      = threadIdx.x & 63;
    const uint32_t mask = (1u << bits) - 1u;
    uint32_t base[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
    {
        const bool in        = k * 64u + lane < valid;
        const uint32_t digit = (key[k] >> shift) & mask;
        const unsigned long long all = __ballot(in);
        uint32_t low = (uint32_t)all, high = (uint32_t)(all >> 32);
#pragma unroll 1
        for (int b = 0; b < bits; ++b)
        {
            const uint32_t set         = (uint32_t)__builtin_amdgcn_sbfe((int)digit, (uint32_t)b, 1u);  // all ones or zeros
            const unsigned long long v = __ballot(set != 0u);
            low &= ~((uint32_t)v ^ set);
            high &= ~((uint32_t)(v >> 32) ^ set);
        }
        const unsigned long long same = (unsigned long long)high << 32 | low;
        const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        rank[k] = before | (((uint32_t)__ffsll((long long)same) - 1u) & 63u) << 8;  // and the lane of the first of them
        base[k] = 0;
        if (in && before == 0)
            base[k] = __hip_atomic_fetch_add(count + digit, (uint32_t)__popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) rank[k] = (rank[k] & 255u) + (uint32_t)__shfl((int)base[k], (int)(rank[k] >> 8));
}

// A tile's keys go to their places; the tile is put in order in LDS first, so that each digit's keys leave side by side.
// 6M pairs 28 us: vector instructions of the ranks 15 of it, the bytes of pairs 15, both beside barriers and LDS.
template <int ITEMS, int FROM>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(const SortParams p)
{
    constexpr int kSortItems = ITEMS, kSortTile = kSortThreads * ITEMS;
    __shared__ uint32_t s_count[kSortWaves][kDigits];  // keys of a digit in each wavefront, then those of the tile before them
    __shared__ uint32_t s_place[kDigits];              // of the tile's first key of a digit: its place, less its place in the tile
    __shared__ uint32_t s_key[kSortTile];
    __shared__ int32_t s_point[kSortTile];
    __shared__ uint32_t s_scan[kSortWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t mask  = (1u << p.bits) - 1u;
    const uint32_t begin = blockIdx.x * (uint32_t)kSortTile;
    const uint32_t count = min((uint32_t)kSortTile, p.n - begin);
    uint32_t key[kSortItems], rank[kSortItems];
    int32_t point[kSortItems];
    const uint32_t mine = wave * 64u * kSortItems, valid = count > mine ? count - mine : 0u;
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
    {
        const uint32_t i = begin + min(mine + k * 64 + lane, count - 1u);  // (the last lanes' copies of the last key count for nothing)
        key[k]   = sort_key<FROM>(p, i);
        point[k] = FROM == kFromKeys ? p.points_in[i] : (int32_t)i;
    }
    for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) s_count[0][i] = 0;
    __syncthreads();
    rank_keys(key, valid, p.shift, p.bits, s_count[wave], rank);
    __syncthreads();
    {
        const int d    = threadIdx.x;
        const bool has = d <= (int)mask;
        uint32_t sum   = 0;
        if (has)
            for (int w = 0; w < kSortWaves; ++w) sum += s_count[w][d];
        const uint32_t in_tile = block_scan(sum, s_scan) - sum;  // the tile's keys of lower digits
        // of all keys, those of the digit, and of the tiles before this one
        uint32_t total = 0, before = 0;
        if (has && p.tiles > kFewTiles)
            total = p.totals[d], before = p.hist[(size_t)d * p.tiles + blockIdx.x];
        else if (has)
            for (uint32_t t = 0; t < p.tiles; ++t)
            {
                const uint32_t c = p.hist[(size_t)d * p.tiles + t];
                total += c;
                before += t < blockIdx.x ? c : 0u;
            }
        const uint32_t below = block_scan(total, s_scan) - total;  // all keys of lower digits
        if (has)
        {
            s_place[d] = below + before - in_tile;
            for (uint32_t w = 0, x = in_tile; w < kSortWaves; ++w)
            {
                const uint32_t c = s_count[w][d];
                s_count[w][d]    = x;
                x += c;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k)
    {
        if (k * 64u + lane >= valid) continue;
        const uint32_t at = s_count[wave][(key[k] >> p.shift) & mask] + rank[k];
        s_key[at]   = key[k];
        s_point[at] = point[k];
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < count; at += kSortThreads)
    {
        const uint32_t k  = s_key[at];
        const uint32_t to = s_place[(k >> p.shift) & mask] + at;
        if (to >= p.n) continue;  // (an index that was written to since it was counted must not lead outside)
        p.keys_out[to]   = k;
        p.points_out[to] = s_point[at];
    }
}

// Few points of a large table: a point's place is the number of keys below its own and of equal ones before it, counted outright. All
// keys in LDS, 32 points a workgroup, each by 32 threads with a 32nd of the keys. One launch, on all of the card, where the sort's
// passes are launches in a row. Bound by the LDS that every key of every workgroup is read from (3.4 us of 11 at 8191 points) and
// the pairs' two instructions (as much).
// Behind the points' places, if `starts`: the keys below each t, 1 << starts_log2 of them a workgroup, each by as many threads as that
// leaves: as many as it takes for about two workgroups a CU (16 points of 643k texels: 32 a workgroup 66 us, 1024 6).
constexpr int kCountThreads = 1024, kCountItems = 32;
constexpr int kStartsGroups = 480;
constexpr int64_t kSmallPoints = 8192;             // a workgroup a CU (8192 of 500,000 texels 12.4 us; 20,000 by passes 29)
constexpr int64_t kSmallPairs  = (int64_t)1 << 25; // keys and starts (16 points of 980,000 texels 7.5 us, by a launch of its own 9.8;
                                                   // 500 of 260,000 12.5, 9.5)
constexpr uint32_t small_part(uint32_t n) { return ((n + 31u) / 32u + 31u) & ~31u; }  // keys of a thread, whole words of signs
template <int FROM>
__global__ __launch_bounds__(kCountThreads) void sort_small_kernel(const SortParams p, int32_t* starts, int starts_log2)
{
    extern __shared__ uint4 s_keys[];
    __shared__ uint32_t s_rank[kCountThreads];
    uint32_t* s_key     = reinterpret_cast<uint32_t*>(s_keys);
    const uint32_t part = small_part(p.n);
    // (four words between the parts: a wavefront reads two of them at a time, from other banks)
    const uint32_t first = (threadIdx.x >> 5) * part, shift = (threadIdx.x >> 5) * 4u;
    for (uint32_t j = first + (threadIdx.x & 31u); j < first + part; j += 32)
        s_key[j + shift] = j < p.n ? sort_key<FROM>(p, j) : 0x7fffffffu;  // (no key is that)
    s_rank[threadIdx.x] = 0u;
    __syncthreads();
    // (the points' workgroups first, then those of the starts)
    const uint32_t point_groups = (p.n + kCountItems - 1) / kCountItems;
    const bool of_points        = blockIdx.x < point_groups;
    const uint32_t items_log2   = of_points ? 5u : (uint32_t)starts_log2, at_item = threadIdx.x & ((1u << items_log2) - 1u);
    const uint32_t i0 = (of_points ? blockIdx.x : blockIdx.x - point_groups) << items_log2, i = i0 + at_item;
    const uint32_t mine = of_points ? (i < p.n ? sort_key<FROM>(p, i) : 0u) : i;
    // The signs of 32 differences in a word: a subtraction and a shift a pair, where the carry of a comparison must be waited for.
    auto less = [&](uint32_t at, uint32_t limit)
    {
        uint32_t signs = 0;
#pragma unroll
        for (uint32_t q = 0; q < 32; q += 4)
        {
            const uint4 k = s_keys[(at + q) / 4];
            signs = __builtin_amdgcn_alignbit(signs, k.x - limit, 31u);
            signs = __builtin_amdgcn_alignbit(signs, k.y - limit, 31u);
            signs = __builtin_amdgcn_alignbit(signs, k.z - limit, 31u);
            signs = __builtin_amdgcn_alignbit(signs, k.w - limit, 31u);
        }
        return signs;
    };
    uint32_t below = 0;
    const uint32_t parts = 1u << (items_log2 - 5u);  // of a thread
    for (uint32_t k = (threadIdx.x >> items_log2) * parts, last = k + parts; k < last && k * part < p.n; ++k)
        for (uint32_t j = k * part; j < (k + 1) * part; j += 32)
        {
            // equal keys count where they lie before the point
            const uint32_t signs = less(j + k * 4u, mine + (of_points && j < i0 ? 1u : 0u));
            below += (uint32_t)__popc(signs);
            if (of_points && __ballot(j == i0))
            {
                const uint32_t equal = less(j + k * 4u, mine + 1u) & ~signs & ~(~0u >> (i & 31u));  // (the word's first keys are its highest bits)
                below += j == i0 ? (uint32_t)__popc(equal) : 0u;
            }
        }
    atomicAdd(&s_rank[at_item], below);
    __syncthreads();
    if (threadIdx.x >> items_log2) return;
    const uint32_t at = s_rank[threadIdx.x];
    if (!of_points)
    {
        if (i <= p.texels) starts[i] = (int32_t)at;
    }
    else if (i < p.n && at < p.n)  // (an index that is written to meanwhile must not lead outside)
    {
        p.points_out[at] = (int32_t)i;
        if (p.keys_out) p.keys_out[at] = mine;
    }
}

// A medium number of points, in one launch: each workgroup takes a range of the texels and reads all keys for it. What lies below the
// range counts for where its points begin; its own keys are counted by wavefront and texel, each wavefront having a piece of the
// points, and then put to their places in order. The starts come out of it for nothing. Every workgroup reads every key (from L2),
// on its way while the counts are cleared, and compares it twice: latency and vector instructions bound it. us: 20,000 points of
// 5000 texels 10.3 (by passes 22), 8191 of 60,000 8.5 (counted outright and by a launch for the starts 12.5), 32,768 13 (23.5) or, all
// of one texel, 17.7 (14.5); 65,536, with 64 rounds, no better than the passes.
constexpr int kRangeThreads = 1024, kRangeWaves = kRangeThreads / 64;
constexpr int64_t kRangePoints = 1 << 15;
constexpr int64_t kRangeGroups = 256;  // a workgroup a CU
constexpr int64_t kMostRange   = 960;  // texels of a workgroup: 60 KB of counts
template <int ROUNDS, int FROM>
__global__ __launch_bounds__(kRangeThreads) void sort_range_kernel(const SortParams p, int32_t* starts, uint32_t range, int bits)
{
    extern __shared__ uint32_t s_counts[];  // [wavefronts][range]
    __shared__ uint32_t s_scan[kRangeWaves], s_below;
    const int lane       = threadIdx.x & 63;
    const uint32_t lo    = blockIdx.x * range, rounds = (p.n + kRangeThreads - 1) / kRangeThreads;
    const uint32_t first = (threadIdx.x >> 6) * rounds * 64u + lane;
    uint32_t* count      = s_counts + (threadIdx.x >> 6) * range;
    uint32_t key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) key[r] = sort_key<FROM>(p, min(first + r * 64u, p.n - 1u));
    for (uint32_t i = threadIdx.x; i < kRangeWaves * range; i += kRangeThreads) s_counts[i] = 0u;
    if (threadIdx.x == 0) s_below = 0u;
    __syncthreads();
    uint32_t below = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
    {
        if ((uint32_t)r >= rounds || first + r * 64u >= p.n) key[r] = ~0u;
        below += key[r] < lo ? 1u : 0u;
        const uint32_t d = key[r] - lo;
        const unsigned long long mine = __ballot(d < range);
        if (!mine) continue;
        // (one addition where they are all of one texel: 64 to one word would be 64 in a row)
        const uint32_t d0 = (uint32_t)__builtin_amdgcn_readlane((int)d, __ffsll((long long)mine) - 1);
        if (__ballot(d == d0) == mine)
        {
            if (lane == 0) atomicAdd(&count[d0], (uint32_t)__popcll(mine));
        }
        else if (d < range)
            atomicAdd(&count[d], 1u);
    }
    for (int o = 32; o > 0; o >>= 1) below += (uint32_t)__shfl_xor((int)below, o);
    if (lane == 0) atomicAdd(&s_below, below);
    __syncthreads();
    uint32_t total = 0;
    if (threadIdx.x < range)
        for (int w = 0; w < kRangeWaves; ++w)
        {
            const uint32_t k = s_counts[w * range + threadIdx.x];
            s_counts[w * range + threadIdx.x] = total;
            total += k;
        }
    const uint32_t start = s_below + block_scan(total, s_scan) - total;
    if (threadIdx.x < range)
    {
        if (lo + threadIdx.x <= p.texels) starts[lo + threadIdx.x] = (int32_t)start;
        for (int w = 0; w < kRangeWaves; ++w) s_counts[w * range + threadIdx.x] += start;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
    {
        const uint32_t d = key[r] - lo;
        const bool mine  = d < range;
        unsigned long long same = __ballot(mine);
        if (!same) continue;
        // the wavefront's keys of the same texel
        const uint32_t d0 = (uint32_t)__builtin_amdgcn_readlane((int)d, __ffsll((long long)same) - 1);
        if (__ballot(d == d0) != same)
        {
#pragma unroll 1
            for (int b = 0; b < bits; ++b)
            {
                const unsigned long long set = __ballot((d >> b) & 1u);
                same &= (d >> b) & 1u ? set : ~set;
            }
        }
        const uint32_t before = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        uint32_t at = 0;
        if (mine && before == 0) at = atomicAdd(&count[d], (uint32_t)__popcll(same));
        at = (uint32_t)__shfl((int)at, mine ? __ffsll((long long)same) - 1 : 0) + before;
        if (mine && at < p.n) p.points_out[at] = (int32_t)(first + r * 64u);
    }
}

// The first of n ascending numbers that is `x` or more, by the whole wavefront: 64 probes a round.
template <typename T>
__device__ __forceinline__ uint32_t lower_bound(const T* a, uint32_t n, uint32_t x, int lane)
{
    uint32_t lo = 0, len = n;  // in [lo, lo + len]
    while (len > 0)
    {
        const uint32_t step = len / 64 + 1, at = (uint32_t)lane * step;
        const bool less     = at < len && (uint32_t)a[lo + at] < x;
        const uint32_t k    = (uint32_t)__popcll(__ballot(less));  // probes below x, the first ones
        if (k == 0) return lo;
        const uint32_t from = (k - 1) * step + 1;
        len = min(k * step, len) - from;
        lo += from;
    }
    return lo;
}

// starts[t] = the first of the sorted keys that is t or more, for kStartsTexels texels a workgroup. Two wavefronts find the keys
// that belong to them; where these are about as many as the texels, each key that differs from the one before is noted in LDS
// and the texels in between take the next one's; where they are many more, each texel is searched for. ITEMS texels a thread: 8,
// or 1 where there are more than two points a texel or few texels. 6M keys of 1.5M texels 18 us with 1, of 6M texels 20 with 8. (The whole
// order with 1 and with 8, us: 50,000 points of 100,000 texels 32.8, 34.7; 40,000 of 250,000 and of 300,000 32.2, 32.1; 500,000 of 500,000
// 42.8, 44.6, 40,000 of 1.5M 37.3, 33.1; 500,000 of 6M 73.2, 50.5.)
constexpr int64_t kFewTexels = 1 << 18;
template <int ITEMS>
__global__ __launch_bounds__(256) void starts_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t texels, int32_t* starts)
{
    constexpr int kStartsItems = ITEMS, kStartsTexels = 256 * ITEMS;
    __shared__ uint32_t s_range[2], s_first[kStartsTexels], s_next[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t first = blockIdx.x * (uint32_t)kStartsTexels, count = min((uint32_t)kStartsTexels, texels + 1u - first);
    if (wave < 2)
    {
        const uint32_t at = lower_bound(keys, n, wave == 0 ? first : first + count, lane);
        if (lane == 0) s_range[wave] = at;
    }
#pragma unroll
    for (int q = 0; q < kStartsItems; ++q) s_first[q * 256 + threadIdx.x] = ~0u;
    __syncthreads();
    const uint32_t from = s_range[0], to = s_range[1];
    if (to - from > 8u * kStartsTexels)
    {
        for (uint32_t t = threadIdx.x; t < count; t += 256)
        {
            uint32_t lo = from, hi = to;
            while (lo < hi)
            {
                const uint32_t mid = lo + (hi - lo) / 2;
                if (keys[mid] < first + t)
                    lo = mid + 1;
                else
                    hi = mid;
            }
            starts[first + t] = (int32_t)lo;
        }
        return;
    }
#pragma unroll 4
    for (uint32_t k = from + threadIdx.x; k < to; k += 256)
    {
        const uint32_t key = keys[k], before = keys[max(k, 1u) - 1u];
        if (k == from || before != key) s_first[key - first] = k;
    }
    __syncthreads();
    // the least of a thread's texels' and all that follow
    uint32_t at[kStartsItems], least = ~0u;
#pragma unroll
    for (int q = kStartsItems - 1; q >= 0; --q) at[q] = least = min(least, s_first[threadIdx.x * kStartsItems + q]);
    uint32_t behind = least;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
    {
        const uint32_t y = (uint32_t)__shfl_down((int)behind, o);
        if (lane + o < 64) behind = min(behind, y);
    }
    if (lane == 0) s_next[wave] = behind;
    behind = (uint32_t)__shfl_down((int)behind, 1);
    if (lane == 63) behind = ~0u;
    __syncthreads();
    for (int w = wave + 1; w < 4; ++w) behind = min(behind, s_next[w]);
    behind = min(behind, to);
#pragma unroll
    for (int q = 0; q < kStartsItems; ++q) s_first[threadIdx.x * kStartsItems + q] = min(at[q], behind);
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < count; t += 256) starts[first + t] = (int32_t)s_first[t];
}

// ---- the gradient ----
//
// The rows of a texel's points are gathered in the order of the plan and added up by the lanes that hold the texel's row. Texels
// with more than kShort points are listed and left to a second kernel, a workgroup each, and what lies in between is summed
// beforehand in tiles of the plan's positions that one texel fills, so that no entry of a table, however many points refer to
// it, is left to one wavefront. Which points are added to which sum first goes by the plan and the sizes alone.

constexpr int kShort      = 32;
constexpr int kShortOfFew = 64;
constexpr int kLongGroups = 2048;  // workgroups for the listed texels
constexpr int kWideThreads = 1024; // of a workgroup that adds up rows of more than eight lanes; 256 for others

struct GradParams
{
    const void* rows;  // gradients [points, row], or columns [channels, row]
    void* d_table;
    const int32_t* order;
    const int32_t* starts;
    float* tiles;     // [points / tile, padded] sums of the tiles that one texel fills (zeros for the others)
    uint32_t* listed;  // texels for the second kernel: how many, then 63 words on, which
    long long texels, table_stride, row;
    uint32_t points, tile, capacity;
    int channels, padded, lanes_log2, accumulate;
    float scale;
};
constexpr int kListHead = 64;

__device__ __forceinline__ void segment(const GradParams& p, long long t, uint32_t& from, uint32_t& to)
{
    // (a plan of another scene must not lead outside)
    from = min((uint32_t)p.starts[t], p.points);
    to   = max(from, min((uint32_t)p.starts[t + 1], p.points));
}

// sum += the rows of the points order[k], k = from, from + step .. below to; V channels from c on. AHEAD rows are on their way at a
// time: 8 short ones of columns (6M points of 1.5M texels 157 us, with 4 160), 4 of longer rows (8191 tokens with 8 1 to 3 us more).
// FROM_COLUMNS: they are columns still (those of the channels behind the last one are the last one's, and go nowhere).
template <int D, int V, int AHEAD, bool FROM_COLUMNS = false>
__device__ __forceinline__ void add_rows(const GradParams& p, uint32_t from, uint32_t to, uint32_t step, int c, int count, float (&sum)[V])
{
    using E       = Element<D>;
    using T       = typename E::type;
    const T* rows = reinterpret_cast<const T*>(p.rows) + (FROM_COLUMNS ? 0 : c);
    for (uint32_t k = from; k < to; k += AHEAD * step)
    {
        uint32_t i[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) i[q] = k + q * step < to ? (uint32_t)p.order[k + q * step] : ~0u;
        typename Pack<T, V>::type x[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
        {
            x[q] = typename Pack<T, V>::type{};
            if (i[q] >= p.points) continue;
            if (FROM_COLUMNS)
            {
#pragma unroll
                for (int e = 0; e < V; ++e) x[q][e] = rows[min(c + e, p.channels - 1) * p.row + i[q]];
                continue;
            }
            const T* row = rows + (long long)i[q] * p.row;
            if (count == V)
                x[q] = *reinterpret_cast<const typename Pack<T, V>::type*>(row);
            else
            {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < count) x[q][e] = row[e];
            }
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] += E::to_float(x[q][e]);
    }
}

template <int D, int V, bool OUT_COLUMNS>
__device__ __forceinline__ void store_sum(const GradParams& p, long long t, int c, int count, const float (&sum)[V])
{
    using E = Element<D>;
    using T = typename E::type;
    T* to             = reinterpret_cast<T*>(p.d_table) + (OUT_COLUMNS ? c * p.table_stride + t : t * p.table_stride + c);
    const long long s = OUT_COLUMNS ? p.table_stride : 1;
    if (!OUT_COLUMNS && count == V && !p.accumulate)
    {
        typename Pack<T, V>::type x;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = E::from_float(p.scale * sum[e]);
        *reinterpret_cast<typename Pack<T, V>::type*>(to) = x;
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (c + e < p.channels) to[e * s] = E::from_float(p.accumulate ? E::to_float(to[e * s]) + p.scale * sum[e] : p.scale * sum[e]);
}

// The sums of the threads of one column (threadIdx.x >> lanes_log2 counts them), in their order; valid in the first `lanes` threads.
template <int V>
__device__ __forceinline__ void add_threads(float (&sum)[V], float* s, int lanes_log2)
{
    const int lanes = 1 << lanes_log2;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) s[e * blockDim.x + threadIdx.x] = sum[e];
    __syncthreads();
    for (int half = (int)blockDim.x / 2; half >= lanes; half >>= 1)
    {
        if ((int)threadIdx.x < half)
        {
#pragma unroll
            for (int e = 0; e < V; ++e) s[e * blockDim.x + threadIdx.x] += s[e * blockDim.x + threadIdx.x + half];
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = s[e * blockDim.x + threadIdx.x];
}

// OUT_COLUMNS: the table's gradient is columns, and the rows were made of columns (whole lanes wide; not if FEW). 6M points of 1.5M texels in
// no order: 118 us, 6.3M lines of 128 bytes (6.8 TB/s of them). 8191 tokens: 20 us, the 102 MB of 50,000 rows, mostly zeros, 5.2 TB/s.
// Groups of lanes' channels go along grid.y where there are few texels, and one behind the other. FEW: so few points that no texel is listed: those with more than
// kShortOfFew are added up by all of the workgroup that they belong to, one behind the other (at most seven, 1.4 us each).
template <int D, int V, bool OUT_COLUMNS, bool FEW>
__global__ __launch_bounds__(256) void lookup_backward_kernel(const GradParams p)
{
    extern __shared__ float s[];  // [V][threads] if FEW
    __shared__ uint32_t s_later[FEW ? 256 : 1], s_count;
    const int lanes = 1 << p.lanes_log2, j = threadIdx.x & (lanes - 1), at_once = 256 >> p.lanes_log2, lane = threadIdx.x & 63;
    const int c0 = (int)blockIdx.y * lanes * V, c_step = (int)gridDim.y * lanes * V;
    if (FEW)
    {
        if (threadIdx.x == 0) s_count = 0u;
        __syncthreads();
    }
    for (long long base = (long long)blockIdx.x * at_once; base < p.texels; base += (long long)gridDim.x * at_once)
    {
        const long long t = base + (threadIdx.x >> p.lanes_log2);
        uint32_t from = 0, to = 0;
        if (t < p.texels) segment(p, t, from, to);
        const bool later = to - from > (FEW ? kShortOfFew : kShort);
        if (FEW)
        {
            if (later && j == 0) s_later[atomicAdd(&s_count, 1u)] = (uint32_t)t;
        }
        else if (const unsigned long long mask = __ballot(later && j == 0 && blockIdx.y == 0))
        {
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(p.listed, (uint32_t)__popcll(mask));
            at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + (uint32_t)__popcll(mask & ((1ull << lane) - 1ull));
            if (later && j == 0 && at < p.capacity) p.listed[kListHead + at] = (uint32_t)t;
        }
        float sum[V];
        if (t < p.texels && !later && !(p.accumulate && from == to))
        {
            for (int c = c0 + j * V; c < p.channels; c += c_step)
            {
                const int count = OUT_COLUMNS ? V : min(V, p.channels - c);
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] = 0.f;
                add_rows<D, V, OUT_COLUMNS && !FEW ? 8 : 4, OUT_COLUMNS && FEW>(p, from, to, 1, c, count, sum);
                store_sum<D, V, OUT_COLUMNS>(p, t, c, count, sum);
            }
        }
        if (!FEW) continue;
        __syncthreads();
        const uint32_t n = s_count;
        for (uint32_t k = 0; k < n; ++k)
        {
            const long long tk = s_later[k];
            segment(p, tk, from, to);
            for (int first = c0; first < p.channels; first += c_step)
            {
                const int c = first + j * V, count = OUT_COLUMNS ? V : min(V, p.channels - c);
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] = 0.f;
                if (c < p.channels) add_rows<D, V, OUT_COLUMNS && !FEW ? 8 : 4, OUT_COLUMNS && FEW>(p, from + (threadIdx.x >> p.lanes_log2), to, at_once, c, count, sum);
                add_threads(sum, s, p.lanes_log2);
                if ((int)threadIdx.x < lanes && c < p.channels) store_sum<D, V, OUT_COLUMNS>(p, tk, c, count, sum);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) s_count = 0u;
        __syncthreads();
    }
}

// One workgroup a tile of the plan's positions (and a group of lanes' channels). Clears the list's length as well. Where no texel
// fills a tile it reads the tile's ends and stores zeros: 3 to 7 us.
template <int D, int V, bool OUT_COLUMNS>
__global__ __launch_bounds__(kWideThreads) void lookup_tiles_kernel(const GradParams p)
{
    extern __shared__ float s[];  // [V][threads]
    __shared__ uint32_t s_in;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.listed = 0u;
    const uint32_t from = blockIdx.x * p.tile, to = from + p.tile;
    if (to > p.points) return;  // (the last positions, and the workgroup of a plan with no whole tile)
    if (threadIdx.x < 64)
    {
        // the last texel that begins at `from` or before, and whether it ends behind the tile
        const uint32_t t = lower_bound(reinterpret_cast<const uint32_t*>(p.starts), (uint32_t)p.texels + 1u, from + 1u, threadIdx.x);
        if (threadIdx.x == 0) s_in = t > 0 && t <= (uint32_t)p.texels && (uint32_t)p.starts[t] >= to ? 1u : 0u;
    }
    __syncthreads();
    const int lanes = 1 << p.lanes_log2, j = threadIdx.x & (lanes - 1), r = threadIdx.x >> p.lanes_log2;
    const int c     = (blockIdx.y * lanes + j) * V;
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    if (s_in)
    {
        if (c < p.channels) add_rows<D, V, OUT_COLUMNS ? 8 : 4>(p, from + r, to, blockDim.x >> p.lanes_log2, c, OUT_COLUMNS ? V : min(V, p.channels - c), sum);
        add_threads(sum, s, p.lanes_log2);
    }
    if ((int)threadIdx.x < lanes && c < p.padded)
    {
#pragma unroll
        for (int e = 0; e < V; ++e) p.tiles[(long long)blockIdx.x * p.padded + c + e] = sum[e];
    }
}

// One workgroup a listed texel (and a group of lanes' channels): the points before its first whole tile, those behind its last
// one, and the tiles. 4 us with nothing listed; 8191 tokens, most frequent ones a few hundred times, 8: a texel's sum is one
// workgroup's chain.
template <int D, int V, bool OUT_COLUMNS>
__global__ __launch_bounds__(kWideThreads) void lookup_backward_long_kernel(const GradParams p)
{
    extern __shared__ float s[];  // [V][threads]
    const int lanes = 1 << p.lanes_log2, j = threadIdx.x & (lanes - 1), r = threadIdx.x >> p.lanes_log2;
    const uint32_t rows = blockDim.x >> p.lanes_log2;
    const int c         = (blockIdx.y * lanes + j) * V;
    const int count     = OUT_COLUMNS ? V : min(V, p.channels - c);
    const uint32_t n    = min(*p.listed, p.capacity);
    for (uint32_t at = blockIdx.x; at < n; at += gridDim.x)
    {
        const long long t = p.listed[kListHead + at];
        uint32_t from, to;
        segment(p, t, from, to);
        const uint32_t first = (from + p.tile - 1) / p.tile, last = to / p.tile;
        float sum[V];
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] = 0.f;
        if (c < p.channels)
        {
            if (first < last)
            {
                add_rows<D, V, OUT_COLUMNS ? 8 : 4>(p, from + r, first * p.tile, rows, c, count, sum);
                for (uint32_t k = first + r; k < last; k += rows)
                {
#pragma unroll
                    for (int e = 0; e < V; ++e) sum[e] += p.tiles[(long long)k * p.padded + c + e];
                }
                add_rows<D, V, OUT_COLUMNS ? 8 : 4>(p, last * p.tile + r, to, rows, c, count, sum);
            }
            else
                add_rows<D, V, OUT_COLUMNS ? 8 : 4>(p, from + r, to, rows, c, count, sum);
        }
        add_threads(sum, s, p.lanes_log2);
        if ((int)threadIdx.x < lanes && c < p.channels) store_sum<D, V, OUT_COLUMNS>(p, t, c, count, sum);
    }
}

// ---- host ----

constexpr long long kMostRowGroups = 1 << 20;  // a launch has less than 2^32 threads
constexpr long long kFewRowGroups  = 4096;     // (8191 points of 50,000 texels in 1024 bfloat16 channels 31 us, with twice as many groups 34)
constexpr size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a row of channels is spread over lanes: 16 bytes a lane, 8 where all of a row in columns fits them, or the one channel that
// a column has.
struct RowShape
{
    int lane_bytes, lanes_log2, groups, padded;  // groups of lanes a row; padded: channels in whole lanes
};
RowShape row_shape(const TripsLookupDesc& d)
{
    const int size = dtype_bytes(d.dtype);
    RowShape r;
    r.lane_bytes    = d.layout == TRIPS_TABLE_ROWS || d.num_channels * size > 8 ? 16 : d.num_channels > 1 ? 8 : size;
    const int v     = r.lane_bytes / size, chunks = (d.num_channels + v - 1) / v;
    r.lanes_log2    = 0;
    while ((1 << r.lanes_log2) < chunks && r.lanes_log2 < 6) ++r.lanes_log2;
    r.groups = (chunks + (1 << r.lanes_log2) - 1) >> r.lanes_log2;
    r.padded = chunks * v;
    return r;
}

// f(type, elements of a lane, whether columns) with all three as constants; SINGLE: with the one channel of a lane, too
template <bool SINGLE, typename F>
void with_types(int dtype, int lane_bytes, bool columns, const F& f)
{
    auto with_columns = [&](auto d, auto v)
    {
        if (columns)
            f(d, v, std::true_type{});
        else
            f(d, v, std::false_type{});
    };
    auto with_lane = [&](auto d)
    {
        constexpr int size = decltype(d)::value == TRIPS_DTYPE_F32 ? 4 : 2;
        if constexpr (SINGLE)
            if (lane_bytes == size) return f(d, std::integral_constant<int, 1>{}, std::true_type{});  // (columns alone)
        if (lane_bytes == 8)
            f(d, std::integral_constant<int, 8 / size>{}, std::true_type{});  // (columns alone)
        else
            with_columns(d, std::integral_constant<int, 16 / size>{});
    };
    if (dtype == TRIPS_DTYPE_F32)
        with_lane(std::integral_constant<int, TRIPS_DTYPE_F32>{});
    else if (dtype == TRIPS_DTYPE_BF16)
        with_lane(std::integral_constant<int, TRIPS_DTYPE_BF16>{});
    else
        with_lane(std::integral_constant<int, TRIPS_DTYPE_F16>{});
}

// Columns [channels, n] to rows [n, padded].
void launch_rows(const TripsLookupDesc& d, const RowShape& r, const void* columns, void* rows, int64_t n, int64_t stride, hipStream_t stream)
{
    const int v = r.lane_bytes / dtype_bytes(d.dtype);
    const dim3 grid((unsigned)((n + 255) / 256), (unsigned)(r.padded / v));
    with_types<false>(d.dtype, r.lane_bytes, true, [&](auto D, auto V, auto) {
        hipLaunchKernelGGL((rows_kernel<decltype(D)::value, decltype(V)::value>), grid, dim3(256), 0, stream, columns, rows, n, stride,
                           d.num_channels, r.padded);
    });
}

// Whether a lookup in columns turns the table to rows first. Scattered requests are what a lookup costs, one a point and channel
// in columns, one a point in rows (6M points and four channels of 1.5M texels in no order: 350 us and 107); turning the table
// costs its bytes twice (9), as much as about an eighth of a request a texel.
bool turns_table(const TripsLookupDesc& d)
{
    return d.layout == TRIPS_TABLE_COLUMNS && d.num_channels > 1 && d.num_points >= d.num_texels / 8;
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
    auto up            = up256;
    const int tile     = kSortThreads * sort_items(points);
    const size_t tiles = (size_t)((points + tile - 1) / tile);
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
    const bool i32 = index_dtype == TRIPS_INDEX_I32;
    p.index = index, p.n = (uint32_t)points, p.texels = (uint32_t)texels;
    const int tile = kSortThreads * sort_items(points);
    p.tiles        = (uint32_t)((points + tile - 1) / tile);
    p.hist = reinterpret_cast<uint32_t*>(ws + l.hist), p.totals = reinterpret_cast<uint32_t*>(ws + l.totals);
    p.keys_out = nullptr, p.points_out = nullptr;
    ProfScope ps(prof, "lookup_plan", stream);
    if (points > 0 && points <= kRangePoints && texels + 1 <= kRangeGroups * kMostRange)
    {
        const uint32_t range = (uint32_t)((texels + kRangeGroups) / kRangeGroups), groups = (uint32_t)(texels / range) + 1u;
        const size_t lds     = sizeof(uint32_t) * kRangeWaves * range;
        const int range_bits = range > 1 ? key_bits(range - 1) : 0;
        p.points_out         = order;
        auto launch = [&](auto rounds, auto from)
        {
            hipLaunchKernelGGL((sort_range_kernel<decltype(rounds)::value, decltype(from)::value>), dim3(groups), dim3(kRangeThreads), lds, stream, p, starts,
                               range, range_bits);
        };
        auto launch_from = [&](auto rounds)
        {
            if (i32)
                launch(rounds, std::integral_constant<int, kFromI32>{});
            else
                launch(rounds, std::integral_constant<int, kFromI64>{});
        };
        if (points <= 8 * kRangeThreads)
            launch_from(std::integral_constant<int, 8>{});
        else if (points <= 16 * kRangeThreads)
            launch_from(std::integral_constant<int, 16>{});
        else if (points <= 24 * kRangeThreads)
            launch_from(std::integral_constant<int, 24>{});
        else
            launch_from(std::integral_constant<int, 32>{});
        return hipGetLastError();
    }
    if (points > 0 && points <= kSmallPoints)
    {
        const bool whole = (texels + 1) * std::max<int64_t>(points, 32) <= kSmallPairs;
        p.shift = 0, p.bits = 0, p.keys_in = nullptr, p.points_in = nullptr;
        p.keys_out   = whole ? nullptr : reinterpret_cast<uint32_t*>(ws + l.keys[0]);
        p.points_out = order;
        const size_t lds      = 32 * sizeof(uint32_t) * (small_part(p.n) + 4);
        int log2 = 5;
        while (log2 < 10 && (texels >> log2) >= kStartsGroups) ++log2;
        const unsigned groups = (p.n + kCountItems - 1) / kCountItems, more = whole ? (unsigned)(texels >> log2) + 1u : 0u;
        if (i32)
            hipLaunchKernelGGL(sort_small_kernel<kFromI32>, dim3(groups + more), dim3(kCountThreads), lds, stream, p, starts, log2);
        else
            hipLaunchKernelGGL(sort_small_kernel<kFromI64>, dim3(groups + more), dim3(kCountThreads), lds, stream, p, starts, log2);
        if (whole) return hipGetLastError();
    }
    int shift = 0;
    for (int pass = 0; pass < passes && points > kSmallPoints; ++pass)
    {
        p.shift      = shift, p.bits = (bits - shift + passes - pass - 1) / (passes - pass);
        p.keys_in    = p.keys_out;
        p.points_in  = p.points_out;
        p.keys_out   = reinterpret_cast<uint32_t*>(ws + l.keys[pass & 1]);
        p.points_out = (passes - 1 - pass) % 2 == 0 ? order : reinterpret_cast<int32_t*>(ws + l.points);
        auto launch = [&](auto items, auto from)
        {
            hipLaunchKernelGGL((sort_count_kernel<decltype(items)::value, decltype(from)::value>), dim3(p.tiles), dim3(kSortThreads), 0, stream, p);
            if (p.tiles > kFewTiles) hipLaunchKernelGGL(sort_scan_kernel, dim3(1 << p.bits), dim3(kScanThreads), 0, stream, p);
            hipLaunchKernelGGL((sort_scatter_kernel<decltype(items)::value, decltype(from)::value>), dim3(p.tiles), dim3(kSortThreads), 0, stream, p);
        };
        auto launch_from = [&](auto items)
        {
            if (pass > 0)
                launch(items, std::integral_constant<int, kFromKeys>{});
            else if (i32)
                launch(items, std::integral_constant<int, kFromI32>{});
            else
                launch(items, std::integral_constant<int, kFromI64>{});
        };
        if (sort_items(points) == 2)
            launch_from(std::integral_constant<int, 2>{});
        else if (sort_items(points) == 4)
            launch_from(std::integral_constant<int, 4>{});
        else
            launch_from(std::integral_constant<int, 6>{});
        shift += p.bits;
    }
    if (points > 2 * texels || texels < kFewTexels)
        hipLaunchKernelGGL(starts_kernel<1>, dim3((unsigned)(texels / 256 + 1)), dim3(256), 0, stream, p.keys_out, (uint32_t)points, (uint32_t)texels, starts);
    else
        hipLaunchKernelGGL(starts_kernel<8>, dim3((unsigned)(texels / 2048 + 1)), dim3(256), 0, stream, p.keys_out, (uint32_t)points, (uint32_t)texels, starts);
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

int check_workspace(const void* workspace, size_t bytes, size_t need)
{
    if (need == 0) return TRIPS_OK;
    if (!workspace || !aligned(workspace, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
    if (bytes < need) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %zu needed", bytes, need);
    return TRIPS_OK;
}

// Strides of what is written must keep its rows apart; what is read may repeat a row.
int check_stride(const char* name, int64_t stride, int64_t row, int64_t rows, bool written)
{
    if (stride < 0 || stride > ((int64_t)1 << 48) || (written && rows > 1 && stride < row))
        return set_error(TRIPS_ERR_INVALID_ARG, "%s %lld (rows have %lld elements)", name, (long long)stride, (long long)row);
    return TRIPS_OK;
}

// Rows of one channel, one behind the other, are a column. (It needs no more workspace than they do.)
TripsLookupDesc as_columns(TripsLookupDesc d)
{
    if (d.num_channels == 1 && d.table_stride == 1 && d.values_stride == 1) d.layout = TRIPS_TABLE_COLUMNS;
    return d;
}

size_t lookup_bytes(const TripsLookupDesc& d)
{
    return turns_table(d) ? up256((size_t)d.num_texels * (size_t)row_shape(d).padded * dtype_bytes(d.dtype)) : 0;
}

hipError_t launch_lookup(const TripsLookupDesc& d, const void* table, const void* index, void* values, void* workspace, hipStream_t stream,
                         Profiler* prof)
{
    ProfScope ps(prof, "lookup", stream);
    const RowShape r = row_shape(d);
    LookupParams p;
    p.table = table, p.index = index, p.values = values, p.texels = d.num_texels, p.points = d.num_points;
    p.table_stride = d.table_stride, p.values_stride = d.values_stride, p.channels = d.num_channels;
    p.i32 = d.index_dtype == TRIPS_INDEX_I32, p.lanes_log2 = r.lanes_log2, p.scale = d.scale;
    const bool columns = d.layout == TRIPS_TABLE_COLUMNS;
    if (columns && !turns_table(d))
    {
        const dim3 grid((unsigned)((d.num_points + 255) / 256), (unsigned)((d.num_channels + kColumnGroup - 1) / kColumnGroup));
        with_types<false>(d.dtype, 16, true, [&](auto D, auto, auto) {
            hipLaunchKernelGGL(lookup_columns_kernel<decltype(D)::value>, grid, dim3(256), 0, stream, p);
        });
        return hipGetLastError();
    }
    if (columns)
    {
        if (d.num_texels > 0) launch_rows(d, r, table, workspace, d.num_texels, d.table_stride, stream);
        p.table = workspace, p.table_stride = r.padded;
    }
    const long long at_once = 4ll * (256 >> r.lanes_log2);
    const dim3 grid((unsigned)std::min<long long>((d.num_points + at_once - 1) / at_once, kMostRowGroups));
    with_types<false>(d.dtype, r.lane_bytes, columns, [&](auto D, auto V, auto C) {
        hipLaunchKernelGGL((lookup_rows_kernel<decltype(D)::value, decltype(V)::value, decltype(C)::value>), grid, dim3(256), 0, stream, p);
    });
    return hipGetLastError();
}

// Points that are few: those of one texel are 16 rounds of loads of its workgroup, at most. (500 points of 300,000 texels in four
// channels 9.4 us, with the two launches for listed texels 14; 8192 points of 100 texels by the texels' workgroups 141, listed 18.)
constexpr int64_t few_points(int lanes_log2) { return lanes_log2 < 6 ? 512 : 256; }
struct GradLayout
{
    size_t rows, tiles, listed, bytes;
    uint32_t tile, count, capacity;  // positions of a tile, tiles, texels of the list
};
GradLayout grad_layout(const TripsLookupDesc& d)
{
    const RowShape r = row_shape(d);
    GradLayout l;
    l.tile = 256;
    while ((int64_t)l.tile * 4096 < d.num_points) l.tile *= 2;
    l.count    = (uint32_t)(d.num_points / l.tile);
    l.capacity = d.num_points <= few_points(r.lanes_log2) ? 0u : (uint32_t)(d.num_points / (kShort + 1));
    size_t o   = 0;
    l.rows     = o;
    if (d.layout == TRIPS_TABLE_COLUMNS && d.num_channels > 1 && l.capacity > 0) o += up256((size_t)d.num_points * (size_t)r.padded * dtype_bytes(d.dtype));
    l.tiles = o, o += up256((size_t)l.count * (size_t)r.padded * sizeof(float));
    l.listed = o, o += up256((kListHead + (size_t)l.capacity) * sizeof(uint32_t));
    l.bytes = o;
    return l;
}

hipError_t launch_lookup_backward(const TripsLookupDesc& d, const void* d_values, const int32_t* order, const int32_t* starts, void* d_table,
                                  char* ws, hipStream_t stream, Profiler* prof)
{
    ProfScope ps(prof, "lookup_backward", stream);
    const RowShape r   = row_shape(d);
    const GradLayout l = grad_layout(d);
    const bool columns = d.layout == TRIPS_TABLE_COLUMNS;
    GradParams p;
    p.rows = d_values, p.row = d.values_stride, p.d_table = d_table, p.order = order, p.starts = starts;
    p.tiles = reinterpret_cast<float*>(ws + l.tiles), p.listed = reinterpret_cast<uint32_t*>(ws + l.listed);
    p.texels = d.num_texels, p.table_stride = d.table_stride, p.points = (uint32_t)d.num_points, p.tile = l.tile, p.capacity = l.capacity;
    p.channels = d.num_channels, p.padded = r.padded, p.lanes_log2 = r.lanes_log2, p.accumulate = d.accumulate != 0, p.scale = d.scale;
    if (columns && d.num_channels == 1)
        p.row = 1;
    else if (columns && l.capacity > 0)
    {
        launch_rows(d, r, d_values, ws + l.rows, d.num_points, d.values_stride, stream);
        p.rows = ws + l.rows, p.row = r.padded;
    }
    const long long at_once = 256 >> r.lanes_log2;
    const long long across  = std::min((d.num_texels + at_once - 1) / at_once, kMostRowGroups);
    const dim3 grid((unsigned)across, (unsigned)std::max(1ll, std::min<long long>(r.groups, kFewRowGroups / across)));
    const dim3 tiles(l.count > 0 ? l.count : 1, r.groups), longs(std::min<uint32_t>(l.capacity, kLongGroups), r.groups);
    with_types<true>(d.dtype, r.lane_bytes, columns, [&](auto D, auto V, auto C) {
        constexpr int kD = decltype(D)::value, kV = decltype(V)::value;
        constexpr bool kC = decltype(C)::value;
        const int threads = r.lanes_log2 > 3 ? kWideThreads : 256;
        const size_t lds  = (size_t)kV * threads * sizeof(float);
        if (l.capacity > 0) hipLaunchKernelGGL((lookup_tiles_kernel<kD, kV, kC>), tiles, dim3(threads), lds, stream, p);
        if (l.capacity > 0)
            hipLaunchKernelGGL((lookup_backward_kernel<kD, kV, kC, false>), grid, dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL((lookup_backward_kernel<kD, kV, kC, true>), grid, dim3(256), kV * 256 * sizeof(float), stream, p);
        if (l.capacity > 0) hipLaunchKernelGGL((lookup_backward_long_kernel<kD, kV, kC>), longs, dim3(threads), lds, stream, p);
    });
    return hipGetLastError();
}
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" {

int trips_lookup_workspace_size(const TripsLookupDesc* desc, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (int e = check_lookup(desc)) return e;
    *bytes = lookup_bytes(*desc);
    return TRIPS_OK;
}

int trips_lookup_forward(TripsCtx* ctx, const TripsLookupDesc* desc, const void* table, const void* index, void* values,
                         void* workspace, size_t workspace_bytes, void* stream)
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
    if (int e = check_workspace(workspace, workspace_bytes, lookup_bytes(d))) return e;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    hipError_t e = launch_lookup(as_columns(d), table, index, values, workspace, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
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
        if (int e = check_workspace(workspace, workspace_bytes, need)) return e;
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
    *bytes = grad_layout(*desc).bytes;
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
    if (int e = check_workspace(workspace, workspace_bytes, grad_layout(d).bytes)) return e;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    hipError_t e = launch_lookup_backward(as_columns(d), d_values, order, starts, d_table, reinterpret_cast<char*>(workspace),
                                          reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "lookup backward launch");
}

}  // extern "C"
