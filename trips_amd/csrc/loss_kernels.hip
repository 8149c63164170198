// Softmax cross entropy of rows against all entries of a table, and its gradients, without keeping the logits (gfx950).
//
//   l_ij = scale <x_i, w_j>;  lse_i = log sum_j exp l_ij;  loss_i = lse_i - l_i,target_i
//   d_ij = g_i (exp(l_ij - lse_i) - [j = target_i]);  d_x = scale d w;  d_w = scale d^T x
//
// Rows that do not count are left out at the start: gather_kernel lays the others one behind the other. What is kept of a row's
// logits is the largest product <x_i, w_j>, not scaled, and the sum of exponentials of the others' distance from it, whose logarithm
// is kept apart: where all entries are masked with the type's lowest value their probabilities are still equal.
#include <algorithm>
#include <cmath>

#include "abi_common.h"

#include "../../include/trips_loss.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int64_t kMostRows    = 1ll << 28;  // threads of a launch
constexpr int64_t kMostEntries = 0x7fffffffll - 256;
constexpr int kMostChannels    = 1 << 17;
constexpr double kLog2e = 1.4426950408889634;
constexpr double kLog2  = 0.6931471805599453;

// ---- rows that count ----

constexpr int kGatherRows = 16;     // rows of a workgroup
constexpr int kChunk      = 1024;   // targets of a chunk that count_kernel counts
constexpr int kCountedBy  = 8192;   // rows from which the chunks are counted beforehand

struct GatherParams
{
    const void* rows;
    const void* target;
    const float* d_loss;     // backward: [n] or [1]
    const float2* state;     // backward: [n]
    const int* chunk_count;  // valid targets of each chunk, or NULL: every workgroup looks at all targets
    const float* chunk_top;  // largest |d_loss| among them
    void* packed;            // [count][kp], zeros from C on; negated where scale is, so that the products behind need only |scale|
    int* place;              // [n]: where a row went, -1 if it does not count
    int* packed_target;
    float2* packed_state;
    float* packed_factor;    // backward: what its gradients are multiplied by in d_ij
    int* count;              // [1]
    float* unscale;          // [2]: what undoes the scaling of d_ij, times scale and times |scale|
    unsigned* ticket;        // cleared for the kernels behind
    long long n, entries, stride;
    int channels, kp, i32, reduction, backward;
    float scale;
};

template <bool I32>
__device__ __forceinline__ bool counts(const void* target, long long i, long long entries)
{
    const long long t = I32 ? (long long)reinterpret_cast<const int32_t*>(target)[i] : (long long)reinterpret_cast<const int64_t*>(target)[i];
    return t >= 0 && t < entries;
}

__device__ __forceinline__ int wave_sum(int x)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ float wave_max(float x)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// |g|, 0 where it is not finite: such a row's factor is g itself, the others' go by the largest that is.
__device__ __forceinline__ float size_of(float g)
{
    const float a = fabsf(g);
    return a <= 3.4028234663852886e38f ? a : 0.f;
}

template <bool I32>
__global__ __launch_bounds__(256) void count_kernel(const void* target, const float* d_loss, long long n, long long entries, int* chunk_count, float* chunk_top)
{
    __shared__ int sums[4];
    __shared__ float tops[4];
    int own     = 0;
    float top   = 0.f;
    for (int e = 0; e < kChunk / 256; ++e)
    {
        const long long i = (long long)blockIdx.x * kChunk + e * 256 + threadIdx.x;
        if (i < n && counts<I32>(target, i, entries))
        {
            ++own;
            if (d_loss) top = fmaxf(top, size_of(d_loss[i]));
        }
    }
    own = wave_sum(own), top = wave_max(top);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = own, tops[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        chunk_count[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
        chunk_top[blockIdx.x]   = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    }
}

__device__ __forceinline__ float negative(float x) { return -x; }
__device__ __forceinline__ unsigned short negative(unsigned short x) { return x ^ 0x8000u; }

// A workgroup takes kGatherRows rows; it counts the rows that count before its own (and all of them) by itself, from the targets or
// from the chunks' counts: one launch, no order left to chance.
template <int D, bool I32>
__global__ __launch_bounds__(256) void gather_kernel(const GatherParams p)
{
    using T = typename Element<D>::type;
    __shared__ int before_w[4], all_w[4];
    __shared__ float top_w[4];
    __shared__ int own_place[kGatherRows];
    const long long first = (long long)blockIdx.x * kGatherRows;
    int before = 0, all = 0;
    float top = 0.f;
    const bool tops = p.backward && p.reduction == TRIPS_REDUCE_NONE;
    if (p.chunk_count)
    {
        const long long chunks = (p.n + kChunk - 1) / kChunk, own_chunk = first / kChunk;
        for (long long c = threadIdx.x; c < chunks; c += 256)
        {
            const int k = p.chunk_count[c];
            all += k;
            if (c < own_chunk) before += k;
            if (tops) top = fmaxf(top, p.chunk_top[c]);
        }
        for (long long i = own_chunk * kChunk + threadIdx.x; i < first; i += 256) before += counts<I32>(p.target, i, p.entries);
    }
    else
        for (long long i = threadIdx.x; i < p.n; i += 256)
            if (counts<I32>(p.target, i, p.entries))
            {
                ++all;
                if (i < first) ++before;
                if (tops) top = fmaxf(top, size_of(p.d_loss[i]));
            }
    before = wave_sum(before), all = wave_sum(all), top = wave_max(top);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0) before_w[wave] = before, all_w[wave] = all, top_w[wave] = top;
    __syncthreads();
    before = before_w[0] + before_w[1] + before_w[2] + before_w[3];
    all    = all_w[0] + all_w[1] + all_w[2] + all_w[3];
    top    = fmaxf(fmaxf(top_w[0], top_w[1]), fmaxf(top_w[2], top_w[3]));
    if (wave == 0)
    {
        const long long i   = first + lane;
        const bool in       = lane < kGatherRows && i < p.n && counts<I32>(p.target, i, p.entries);
        const uint64_t mask = __ballot(in);
        if (lane < kGatherRows)
        {
            const int at    = in ? before + __popcll(mask & ((1ull << lane) - 1)) : -1;
            own_place[lane] = at;
            if (i < p.n) p.place[i] = at;
            if (in)
            {
                p.packed_target[at] = I32 ? reinterpret_cast<const int32_t*>(p.target)[i] : (int)reinterpret_cast<const int64_t*>(p.target)[i];
                if (p.backward)
                {
                    p.packed_state[at] = p.state[i];
                    // Largest factor: 1 in 32 bits and bfloat16, 2^15 in float16, whose range is short (probabilities from 2^-29 on then
                    // are normal numbers); d_ij has those for bounds.
                    const float one = D == TRIPS_DTYPE_F16 ? 32768.f : 1.f;
                    float f         = one;
                    if (p.reduction == TRIPS_REDUCE_NONE) f = top > 0.f ? p.d_loss[i] / top * one : p.d_loss[i];
                    p.packed_factor[at] = f;
                }
            }
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0)
    {
        *p.count  = all;
        *p.ticket = 0u;
        if (p.backward)
        {
            const float one = D == TRIPS_DTYPE_F16 ? 1.f / 32768.f : 1.f;
            const float g   = p.reduction == TRIPS_REDUCE_NONE ? (top > 0.f ? top : 1.f) : p.reduction == TRIPS_REDUCE_SUM ? p.d_loss[0] : p.d_loss[0] / (float)max(all, 1);
            p.unscale[0]    = g * one * p.scale;
            p.unscale[1]    = g * one * fabsf(p.scale);
        }
    }
    __syncthreads();
    for (int r = wave; r < kGatherRows; r += 4)
    {
        const int at = own_place[r];
        if (at < 0) continue;
        const T* from = reinterpret_cast<const T*>(p.rows) + (first + r) * p.stride;
        T* to         = reinterpret_cast<T*>(p.packed) + (long long)at * p.kp;
        for (int c = lane * 8; c < p.kp; c += 512)
        {
            typename Pack<T, 8>::type x;
            if (c + 8 <= p.channels)
                x = *reinterpret_cast<const typename Pack<T, 8>::type*>(from + c);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = c + e < p.channels ? from[c + e] : T(0);
            if (p.scale < 0.f)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = negative(x[e]);
            *reinterpret_cast<typename Pack<T, 8>::type*>(to + c) = x;
        }
    }
}

// ---- products ----

// What a product's tiles are of: rows of the first operand run along a lane's registers, those of the second along the lanes.
//   LOGITS  entries x rows, over the channels: the largest product and the sum of exponentials of each row and stripe of tiles
//   PROBS   the same again: d_ij, [rows][piece]
//   D_ROWS  channels x rows, over the piece's entries
//   D_TABLE channels x entries, over the rows
enum { LOGITS, PROBS, D_ROWS, D_TABLE };

constexpr int kTile = 128, kStep = 16, kRow = kTile + 4;

struct ProductParams
{
    const void* table;     // of entry 0
    const void* packed;    // [count][kp]
    const int* count;
    const int* packed_target;
    const float2* packed_state;  // {largest product, log2 of the sum}
    const float* packed_factor;
    const float* unscale;
    float2* partial;       // LOGITS: [stripes][rows_pad] {largest product, sum of exponentials}
    float* own_product;    // [rows_pad]
    float* probs;          // [rows_pad][piece]
    float* slabs;          // D_ROWS: [splits][rows_pad][kp]
    void* d_table;
    long long table_stride, d_table_stride, entries, first_entry, rows_pad;
    int channels, kp, piece, stripes, splits, add;
    unsigned tiles_x, tiles_y;
    float scale_log2;
};

typedef float Acc __attribute__((ext_vector_type(16)));

// exp(scale (x - base)); 0 for an x of minus infinity.
__device__ __forceinline__ float part_of(float x, float base, float scale_log2) { return __builtin_amdgcn_exp2f((x - base) * scale_log2); }

template <int D, int MODE>
__global__ __launch_bounds__(256) void product_kernel(const ProductParams p)
{
    using E = Element<D>;
    using T = typename E::type;
    __shared__ float first[2][kStep][kRow], second[2][kStep][kRow];
    __shared__ float2 joined[2][kTile];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int count = *p.count;
    constexpr bool FIRST_ALONG_K  = MODE == LOGITS || MODE == PROBS;
    constexpr bool SECOND_ALONG_K = MODE != D_TABLE;

    // the tile
    const unsigned block_x = blockIdx.x % p.tiles_x, block_y = blockIdx.x / p.tiles_x % p.tiles_y, block_z = blockIdx.x / p.tiles_x / p.tiles_y;
    const long long n0     = (long long)block_y * kTile;
    const int in_piece = (int)min((long long)p.piece, p.entries - p.first_entry);
    if ((MODE == D_TABLE ? (long long)in_piece : (long long)count) <= n0) return;
    const int rows_up = (count + kStep - 1) / kStep * kStep;
    int k_begin = 0, k_end = MODE == D_TABLE ? rows_up : p.kp;
    if (MODE == D_ROWS)
    {
        const int steps = (in_piece + kStep - 1) / kStep, each = (steps + p.splits - 1) / p.splits;
        k_begin = min(in_piece, (int)block_z * each * kStep), k_end = min(in_piece, k_begin + each * kStep);
    }

    float2 best[2];  // LOGITS: of the wave's rows (a lane: one of 32), in this stripe
    best[0] = best[1] = make_float2(-__builtin_inff(), 0.f);
    const long long tiles = MODE == LOGITS ? (p.entries + kTile - 1) / kTile : 0;
    for (long long tile = block_x; tile < (MODE == LOGITS ? tiles : (long long)block_x + 1); tile += MODE == LOGITS ? p.stripes : 1)
    {
        const long long m0 = tile * kTile;
        Acc acc[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

        // eight elements a thread of each operand: along k, or along the tile
        float a[8], b[8];
        auto fetch = [&](int k0)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.f;
            if constexpr (FIRST_ALONG_K)
            {
                const long long j = (MODE == PROBS ? p.first_entry : 0) + m0 + (threadIdx.x >> 1);
                const int k       = k0 + (threadIdx.x & 1) * 8;
                const T* at       = reinterpret_cast<const T*>(p.table) + j * p.table_stride + k;
                if (j < p.entries)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (k + e < p.channels) a[e] = E::to_float(at[e]);
            }
            else
            {
                const int k = k0 + (threadIdx.x >> 4), c = (int)m0 + (threadIdx.x & 15) * 8;
                const T* at = MODE == D_ROWS ? reinterpret_cast<const T*>(p.table) + (p.first_entry + k) * p.table_stride + c
                                             : reinterpret_cast<const T*>(p.packed) + (long long)k * p.kp + c;
                if (k < (MODE == D_ROWS ? in_piece : count))
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c + e < p.channels) a[e] = E::to_float(at[e]);
            }
            if constexpr (MODE == LOGITS || MODE == PROBS)
            {
                const long long r = n0 + (threadIdx.x >> 1);
                const T* at       = reinterpret_cast<const T*>(p.packed) + r * p.kp + k0 + (threadIdx.x & 1) * 8;
                if (r < count)
#pragma unroll
                    for (int e = 0; e < 8; ++e) b[e] = E::to_float(at[e]);
            }
            else if constexpr (MODE == D_ROWS)
            {
                const long long r = n0 + (threadIdx.x >> 1);
                const int k       = k0 + (threadIdx.x & 1) * 8;
                if (r < count)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (k + e < in_piece) b[e] = p.probs[r * p.piece + k + e];
            }
            else
            {
                const int k = k0 + (threadIdx.x >> 4);
                if (k < count)
#pragma unroll
                    for (int e = 0; e < 8; ++e) b[e] = p.probs[(long long)k * p.piece + n0 + (threadIdx.x & 15) * 8 + e];
            }
        };
        auto put = [&](int buffer)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                if constexpr (FIRST_ALONG_K)
                    first[buffer][(threadIdx.x & 1) * 8 + e][threadIdx.x >> 1] = a[e];
                else
                    first[buffer][threadIdx.x >> 4][(threadIdx.x & 15) * 8 + e] = a[e];
                if constexpr (SECOND_ALONG_K)
                    second[buffer][(threadIdx.x & 1) * 8 + e][threadIdx.x >> 1] = b[e];
                else
                    second[buffer][threadIdx.x >> 4][(threadIdx.x & 15) * 8 + e] = b[e];
            }
        };
        int buffer = 0;
        if (k_begin < k_end)
        {
            fetch(k_begin);
            __syncthreads();
            put(0);
        }
        for (int k0 = k_begin; k0 < k_end; k0 += kStep)
        {
            __syncthreads();
            if (k0 + kStep < k_end) fetch(k0 + kStep);
#pragma unroll
            for (int k = 0; k < kStep; k += 2)
            {
                float x[2], y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    x[i] = first[buffer][k + (lane >> 5)][wm + i * 32 + (lane & 31)];
                    y[i] = second[buffer][k + (lane >> 5)][wn + i * 32 + (lane & 31)];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[j], acc[i][j], 0, 0, 0);
            }
            buffer ^= 1;
            if (k0 + kStep < k_end) put(buffer);
        }

        // a lane's elements: of row n0 + wn + 32 j + lane % 32, of the first operand's rows m0 + wm + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            const long long n = n0 + wn + j * 32 + (lane & 31);
            if constexpr (MODE == LOGITS)
            {
                const int own = n < count ? p.packed_target[n] : -1;
                float top     = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                    {
                        const long long m = m0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                        const float l     = m < p.entries ? acc[i][j][e] : -__builtin_inff();
                        if (m == own) p.own_product[n] = l;
                        acc[i][j][e] = l;
                        top          = fmaxf(top, l);
                    }
                top              = fmaxf(top, __shfl_xor(top, 32));
                const float now  = fmaxf(best[j].x, top);
                const float base = now == -__builtin_inff() ? 0.f : now;
                float sum        = 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum += part_of(acc[i][j][e], base, p.scale_log2);
                sum += __shfl_xor(sum, 32);
                best[j] = make_float2(now, best[j].y * part_of(best[j].x, base, p.scale_log2) + sum);
            }
            else if constexpr (MODE == PROBS)
            {
                const bool in   = n < count;
                const int own   = in ? p.packed_target[n] : -1;
                const float2 state = in ? p.packed_state[n] : make_float2(0.f, 0.f);
                const float factor = in ? p.packed_factor[n] : 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                    {
                        const int in_tile = (int)m0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                        const long long m = p.first_entry + in_tile;
                        float q           = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e] - state.x, p.scale_log2, -state.y));
                        if (m == own) q -= 1.f;
                        if (in && in_tile < p.piece) p.probs[n * p.piece + in_tile] = in_tile < in_piece ? q * factor : 0.f;
                    }
            }
            else
            {
                const float unscale = MODE == D_TABLE ? p.unscale[1] : 1.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                    {
                        const int c = (int)m0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                        if constexpr (MODE == D_ROWS)
                        {
                            float* at = p.slabs + ((long long)block_z * p.rows_pad + n) * p.kp + c;
                            if (n < count && c < p.channels) *at = p.add ? *at + acc[i][j][e] : acc[i][j][e];
                        }
                        else
                        {
                            if (n < in_piece && c < p.channels)
                                reinterpret_cast<T*>(p.d_table)[(p.first_entry + n) * p.d_table_stride + c] = E::from_float(acc[i][j][e] * unscale);
                        }
                    }
            }
        }
    }
    if constexpr (MODE == LOGITS)
    {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (lane < 32) joined[wave & 1][wn + j * 32 + lane] = best[j];
        __syncthreads();
        if (threadIdx.x < kTile)
        {
            const float2 a = joined[0][threadIdx.x], b = joined[1][threadIdx.x];
            const float top = fmaxf(a.x, b.x), base = top == -__builtin_inff() ? 0.f : top;
            p.partial[block_x * p.rows_pad + n0 + threadIdx.x] = make_float2(top, a.y * part_of(a.x, base, p.scale_log2) + b.y * part_of(b.x, base, p.scale_log2));
        }
    }
}

// ---- joins ----

// 16 rows a workgroup, 16 lanes a row over the stripes: state and loss; the last workgroup adds the workgroups' sums up, in their order.
struct JoinParams
{
    const float2* partial;
    const float* own_product;
    const int* place;
    const int* count;
    float* loss;
    float2* state;
    double* sums;
    unsigned* ticket;
    long long n, rows_pad;
    int stripes, reduction;
    float scale, scale_log2;
};
__global__ __launch_bounds__(256) void join_kernel(const JoinParams p)
{
    __shared__ float2 part[16][17];
    __shared__ float losses[16];
    __shared__ bool last;
    __shared__ double sums[256];
    const int lane = threadIdx.x & 15, share = threadIdx.x >> 4;
    const long long i = (long long)blockIdx.x * 16 + lane;
    const int at      = i < p.n ? p.place[i] : -1;
    float2 own        = make_float2(-__builtin_inff(), 0.f);
    if (at >= 0)
        for (int s = share; s < p.stripes; s += 16)
        {
            const float2 x  = p.partial[s * p.rows_pad + at];
            const float top = fmaxf(own.x, x.x), base = top == -__builtin_inff() ? 0.f : top;
            own = make_float2(top, own.y * part_of(own.x, base, p.scale_log2) + x.y * part_of(x.x, base, p.scale_log2));
        }
    part[share][lane] = own;
    __syncthreads();
    if (threadIdx.x < 16)
    {
        float top = -__builtin_inff(), sum = 0.f;
        for (int s = 0; s < 16; ++s) top = fmaxf(top, part[s][lane].x);
        const float base = top == -__builtin_inff() ? 0.f : top;
        for (int s = 0; s < 16; ++s) sum += part[s][lane].y * part_of(part[s][lane].x, base, p.scale_log2);
        float loss = 0.f, log_sum = 0.f;
        if (at >= 0)
        {
            const double log = log2((double)sum);
            loss    = (float)(((double)top - (double)p.own_product[at]) * (double)p.scale + log * kLog2);
            log_sum = (float)log;
        }
        losses[lane] = loss;
        if (i < p.n)
        {
            p.state[i] = make_float2(at >= 0 ? top : 0.f, log_sum);
            if (p.reduction == TRIPS_REDUCE_NONE) p.loss[i] = loss;
        }
    }
    if (p.reduction == TRIPS_REDUCE_NONE) return;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        double sum = 0.0;
        for (int l = 0; l < 16; ++l) sum += (double)losses[l];
        __hip_atomic_store(&p.sums[blockIdx.x], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    double sum = 0.0;
    for (unsigned b = threadIdx.x; b < gridDim.x; b += 256) sum += __hip_atomic_load(&p.sums[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sums[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1)
    {
        if ((int)threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *p.loss = (float)(p.reduction == TRIPS_REDUCE_MEAN ? sums[0] / (double)max(*p.count, 1) : sums[0]);
}

// d_rows: the splits' sums, in their order, at their rows' own places.
template <int D>
__global__ __launch_bounds__(256) void rows_out_kernel(const float* slabs, const int* place, const float* unscale, void* d_rows, long long n, long long rows_pad,
                                                       long long stride, int channels, int kp, int splits)
{
    using E       = Element<D>;
    const float f = *unscale;
    for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (long long)gridDim.x * 4)
    {
    const int at = place[i];
    for (int c = threadIdx.x & 63; c < channels; c += 64)
    {
        float sum = 0.f;
        if (at >= 0)
            for (int s = 0; s < splits; ++s) sum += slabs[((long long)s * rows_pad + at) * kp + c];
        reinterpret_cast<typename E::type*>(d_rows)[i * stride + c] = E::from_float(at >= 0 ? sum * f : 0.f);
    }
    }
}

// ---- host ----

constexpr int64_t kPieceBytes = 256ll << 20;

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

struct Layout
{
    int64_t rows_pad, chunks, piece, pieces;
    int kp, stripes, splits;
    size_t packed, place, target, state, factor, count, chunk_count, chunk_top, partial, own_product, sums, probs, slabs, bytes;
};

Layout layout_of(const TripsTableLossDesc& d, bool backward)
{
    Layout l{};
    l.rows_pad = up(d.num_rows, 256), l.chunks = d.num_rows > kCountedBy ? up(d.num_rows, kChunk) / kChunk : 0;
    l.kp       = (int)up(d.num_channels, 64);
    size_t at  = 0;
    auto take  = [&](size_t bytes)
    {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    l.count  = take(256);
    l.packed = take((size_t)d.num_rows * l.kp * dtype_bytes(d.dtype));
    l.place = take(d.num_rows * 4), l.target = take(d.num_rows * 4);
    l.chunk_count = take(l.chunks * 4), l.chunk_top = take(l.chunks * 4);
    const int64_t row_tiles = up(d.num_rows, kTile) / kTile, tiles = up(d.num_entries, kTile) / kTile;
    if (!backward)
    {
        l.stripes   = (int)std::max<int64_t>(1, std::min(tiles, std::max<int64_t>(1, 4096 / std::max<int64_t>(row_tiles, 1))));
        l.partial   = take((size_t)l.stripes * l.rows_pad * sizeof(float2));
        l.own_product = take(l.rows_pad * 4);
        l.sums      = take((d.num_rows / 16 + 1) * 8);
    }
    else
    {
        l.state = take(d.num_rows * 8), l.factor = take(d.num_rows * 4);
        const int64_t most = std::max<int64_t>(kPieceBytes / (std::max<int64_t>(l.rows_pad, 1) * 4) / 256, 1) * 256;
        l.pieces = std::max<int64_t>(1, (d.num_entries + most - 1) / most);
        l.piece  = up((d.num_entries + l.pieces - 1) / l.pieces, 256);
        l.probs  = take((size_t)l.rows_pad * l.piece * 4);
        const int64_t out_tiles = std::max<int64_t>(1, row_tiles * (up(d.num_channels, kTile) / kTile));
        l.splits = (int)std::max<int64_t>(1, std::min<int64_t>({1024 / out_tiles, l.piece / 256, 64}));
        l.slabs  = take((size_t)l.splits * l.rows_pad * l.kp * 4);
    }
    l.bytes = at;
    return l;
}

// (not 0: 0 times minus infinity, which stands for entries that are not there, is no number)
float scale_log2(const TripsTableLossDesc& d) { return std::max((float)(std::fabs((double)d.scale) * kLog2e), 1.2e-38f); }

template <int D>
hipError_t gather(const TripsTableLossDesc& d, const Layout& l, const void* rows, const void* target, bool backward, const float* d_loss, const float* state, char* w, hipStream_t stream, Profiler* prof)
{
    GatherParams p{};
    p.rows = rows, p.target = target, p.d_loss = d_loss, p.state = (const float2*)state;
    p.packed = w + l.packed, p.place = (int*)(w + l.place), p.packed_target = (int*)(w + l.target);
    p.packed_state = (float2*)(w + l.state), p.packed_factor = (float*)(w + l.factor);
    p.count = (int*)(w + l.count), p.unscale = (float*)(w + l.count) + 2, p.ticket = (unsigned*)(w + l.count) + 1;
    p.n = d.num_rows, p.entries = d.num_entries, p.stride = d.rows_stride;
    p.channels = d.num_channels, p.kp = l.kp, p.i32 = d.index_dtype == TRIPS_INDEX_I32, p.reduction = d.reduction, p.backward = backward, p.scale = d.scale;
    if (l.chunks)
    {
        p.chunk_count = (int*)(w + l.chunk_count), p.chunk_top = (float*)(w + l.chunk_top);
        ProfScope scope(prof, "loss_count", stream);
        (p.i32 ? count_kernel<true> : count_kernel<false>)<<<(unsigned)l.chunks, 256, 0, stream>>>(target, d.reduction == TRIPS_REDUCE_NONE ? d_loss : nullptr, d.num_rows, d.num_entries,
                                                                                                  (int*)(w + l.chunk_count), (float*)(w + l.chunk_top));
        if (hipError_t e = hipGetLastError()) return e;
    }
    ProfScope scope(prof, "loss_gather", stream);
    (p.i32 ? gather_kernel<D, true> : gather_kernel<D, false>)<<<std::max(1u, (unsigned)((d.num_rows + kGatherRows - 1) / kGatherRows)), 256, 0, stream>>>(p);
    return hipGetLastError();
}

ProductParams product_params(const TripsTableLossDesc& d, const Layout& l, const void* table, char* w)
{
    ProductParams p{};
    p.table = table, p.packed = w + l.packed, p.count = (int*)(w + l.count), p.packed_target = (int*)(w + l.target);
    p.packed_state = (float2*)(w + l.state), p.packed_factor = (float*)(w + l.factor), p.unscale = (float*)(w + l.count) + 2;
    p.partial = (float2*)(w + l.partial), p.own_product = (float*)(w + l.own_product), p.probs = (float*)(w + l.probs), p.slabs = (float*)(w + l.slabs);
    p.table_stride = d.table_stride, p.d_table_stride = d.d_table_stride, p.entries = d.num_entries, p.rows_pad = l.rows_pad;
    p.channels = d.num_channels, p.kp = l.kp, p.piece = (int)l.piece, p.stripes = l.stripes, p.splits = l.splits;
    p.scale_log2 = scale_log2(d);
    return p;
}

unsigned tiles_of(int64_t n) { return (unsigned)((n + kTile - 1) / kTile); }

template <int D, int MODE>
hipError_t launch_product(const char* name, ProductParams p, unsigned x, unsigned y, unsigned z, hipStream_t stream, Profiler* prof)
{
    if (x == 0 || y == 0) return hipSuccess;
    p.tiles_x = x, p.tiles_y = y;
    ProfScope scope(prof, name, stream);
    product_kernel<D, MODE><<<x * y * z, 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <int D>
hipError_t forward(const TripsTableLossDesc& d, const void* rows, const void* table, const void* target, float* loss, float* state, char* w, hipStream_t stream, Profiler* prof)
{
    const Layout l = layout_of(d, false);
    if (hipError_t e = gather<D>(d, l, rows, target, false, nullptr, nullptr, w, stream, prof)) return e;
    if (hipError_t e = launch_product<D, LOGITS>("loss_logits", product_params(d, l, table, w), l.stripes, tiles_of(d.num_rows), 1, stream, prof)) return e;
    JoinParams j{};
    j.partial = (float2*)(w + l.partial), j.own_product = (float*)(w + l.own_product), j.place = (int*)(w + l.place), j.count = (int*)(w + l.count);
    j.loss = loss, j.state = (float2*)state, j.scale = std::fabs(d.scale), j.scale_log2 = scale_log2(d), j.sums = (double*)(w + l.sums), j.ticket = (unsigned*)(w + l.count) + 1;
    j.n = d.num_rows, j.rows_pad = l.rows_pad, j.stripes = l.stripes, j.reduction = d.reduction;
    ProfScope scope(prof, "loss_join", stream);
    join_kernel<<<std::max(1u, (unsigned)((d.num_rows + 15) / 16)), 256, 0, stream>>>(j);
    return hipGetLastError();
}

template <int D>
hipError_t backward(const TripsTableLossDesc& d, const void* rows, const void* table, const void* target, const float* state, const float* d_loss, void* d_rows, void* d_table, char* w,
                    hipStream_t stream, Profiler* prof)
{
    const Layout l = layout_of(d, true);
    if (hipError_t e = gather<D>(d, l, rows, target, true, d_loss, state, w, stream, prof)) return e;
    ProductParams p = product_params(d, l, table, w);
    p.d_table       = d_table;
    for (int64_t piece = 0; piece < l.pieces; ++piece)
    {
        p.first_entry = piece * l.piece, p.add = piece > 0;
        if (p.first_entry >= d.num_entries) break;
        const unsigned row_tiles = tiles_of(d.num_rows), channel_tiles = tiles_of(d.num_channels), entry_tiles = (unsigned)(l.piece / kTile);
        if (hipError_t e = launch_product<D, PROBS>("loss_probs", p, entry_tiles, row_tiles, 1, stream, prof)) return e;
        if (d_rows)
            if (hipError_t e = launch_product<D, D_ROWS>("loss_d_rows", p, channel_tiles, row_tiles, l.splits, stream, prof)) return e;
        if (d_table)
            if (hipError_t e = launch_product<D, D_TABLE>("loss_d_table", p, channel_tiles, entry_tiles, 1, stream, prof)) return e;
    }
    if (!d_rows || d.num_rows == 0) return hipSuccess;
    ProfScope scope(prof, "loss_rows_out", stream);
    rows_out_kernel<D><<<(unsigned)std::min<int64_t>((d.num_rows + 3) / 4, 1 << 20), 256, 0, stream>>>((float*)(w + l.slabs), (int*)(w + l.place), p.unscale, d_rows, d.num_rows, l.rows_pad, d.d_rows_stride,
                                                                           d.num_channels, l.kp, l.splits);
    return hipGetLastError();
}

int check_stride(const char* name, int64_t stride, int64_t row, int64_t rows, bool written)
{
    if (stride < 0 || stride > ((int64_t)1 << 40) || (written && rows > 1 && stride < row))
        return set_error(TRIPS_ERR_INVALID_ARG, "%s %lld (rows have %lld elements)", name, (long long)stride, (long long)row);
    return TRIPS_OK;
}

int check_desc(const TripsTableLossDesc* d)
{
    if (!d) return set_error(TRIPS_ERR_INVALID_ARG, "desc is NULL");
    if (d->abi_version != TRIPS_ABI_VERSION) return set_error(TRIPS_ERR_INVALID_ARG, "abi_version %d, library is %d", d->abi_version, TRIPS_ABI_VERSION);
    if (!dtype_ok(d->dtype)) return set_error(TRIPS_ERR_UNSUPPORTED, "dtype %d", d->dtype);
    if (d->index_dtype != TRIPS_INDEX_I64 && d->index_dtype != TRIPS_INDEX_I32) return set_error(TRIPS_ERR_UNSUPPORTED, "index_dtype %d", d->index_dtype);
    if (d->reduction != TRIPS_REDUCE_NONE && d->reduction != TRIPS_REDUCE_SUM && d->reduction != TRIPS_REDUCE_MEAN) return set_error(TRIPS_ERR_INVALID_ARG, "reduction %d", d->reduction);
    if (d->num_rows < 0 || d->num_rows >= kMostRows) return set_error(TRIPS_ERR_INVALID_ARG, "num_rows = %lld", (long long)d->num_rows);
    if (d->num_entries < 0 || d->num_entries >= kMostEntries) return set_error(TRIPS_ERR_INVALID_ARG, "num_entries = %lld", (long long)d->num_entries);
    if (d->num_channels < 1 || d->num_channels >= kMostChannels) return set_error(TRIPS_ERR_INVALID_ARG, "num_channels = %d", d->num_channels);
    if (!(d->scale - d->scale == 0.f)) return set_error(TRIPS_ERR_INVALID_ARG, "scale is not finite");
    if (int e = check_stride("rows_stride", d->rows_stride, d->num_channels, d->num_rows, false)) return e;
    return check_stride("table_stride", d->table_stride, d->num_channels, d->num_entries, false);
}

int check_pointer(const char* name, const void* p, size_t align, bool needed)
{
    if ((!p && needed) || !aligned(p, align)) return set_error(TRIPS_ERR_INVALID_ARG, "%s is NULL or not aligned", name);
    return TRIPS_OK;
}

int check_call(TripsCtx* ctx, const TripsTableLossDesc* d, bool backward, const void* rows, const void* table, const void* target, const void* workspace, size_t bytes)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (int e = check_desc(d)) return e;
    const size_t size = dtype_bytes(d->dtype);
    if (int e = check_pointer("rows", rows, size, d->num_rows > 0)) return e;
    if (int e = check_pointer("table", table, size, d->num_entries > 0)) return e;
    if (int e = check_pointer("target", target, d->index_dtype == TRIPS_INDEX_I32 ? 4 : 8, d->num_rows > 0)) return e;
    if (!workspace || !aligned(workspace, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
    const size_t need = layout_of(*d, backward).bytes;
    if (bytes < need) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %zu needed", bytes, need);
    return TRIPS_OK;
}
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" {

int trips_table_loss_workspace_size(const TripsTableLossDesc* desc, int backward, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (int e = check_desc(desc)) return e;
    *bytes = layout_of(*desc, backward != 0).bytes;
    return TRIPS_OK;
}

int trips_table_loss_forward(TripsCtx* ctx, const TripsTableLossDesc* desc, const void* rows, const void* table, const void* target,
                             float* loss, float* state, void* workspace, size_t workspace_bytes, void* stream)
{
    if (int e = check_call(ctx, desc, false, rows, table, target, workspace, workspace_bytes)) return e;
    if (int e = check_pointer("loss", loss, 4, desc->num_rows > 0 || desc->reduction != TRIPS_REDUCE_NONE)) return e;
    if (int e = check_pointer("state", state, 8, desc->num_rows > 0)) return e;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    const auto call    = desc->dtype == TRIPS_DTYPE_F32 ? forward<TRIPS_DTYPE_F32> : desc->dtype == TRIPS_DTYPE_BF16 ? forward<TRIPS_DTYPE_BF16> : forward<TRIPS_DTYPE_F16>;
    const hipError_t e = call(*desc, rows, table, target, loss, state, (char*)workspace, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "table loss launch");
}

int trips_table_loss_backward(TripsCtx* ctx, const TripsTableLossDesc* desc, const void* rows, const void* table, const void* target,
                              const float* state, const float* d_loss, void* d_rows, void* d_table, void* workspace, size_t workspace_bytes,
                              void* stream)
{
    if (int e = check_call(ctx, desc, true, rows, table, target, workspace, workspace_bytes)) return e;
    const size_t size = dtype_bytes(desc->dtype);
    if (int e = check_pointer("state", state, 8, desc->num_rows > 0)) return e;
    if (int e = check_pointer("d_loss", d_loss, 4, desc->num_rows > 0 || desc->reduction != TRIPS_REDUCE_NONE)) return e;
    if (int e = check_pointer("d_rows", d_rows, size, false)) return e;
    if (int e = check_pointer("d_table", d_table, size, false)) return e;
    if (d_rows)
        if (int e = check_stride("d_rows_stride", desc->d_rows_stride, desc->num_channels, desc->num_rows, true)) return e;
    if (d_table)
        if (int e = check_stride("d_table_stride", desc->d_table_stride, desc->num_channels, desc->num_entries, true)) return e;
    if (!d_rows && !d_table) return TRIPS_OK;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    const auto call    = desc->dtype == TRIPS_DTYPE_F32 ? backward<TRIPS_DTYPE_F32> : desc->dtype == TRIPS_DTYPE_BF16 ? backward<TRIPS_DTYPE_BF16> : backward<TRIPS_DTYPE_F16>;
    const hipError_t e = call(*desc, rows, table, target, state, d_loss, d_rows, d_table, (char*)workspace, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "table loss launch");
}

}  // extern "C"
