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
#include <limits>
#include <type_traits>

#include "abi_common.h"

#include "../../include/trips_loss.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int64_t kMostRows    = (1ll << 28) - 16;  // gather_kernel's threads, 16 a row, stay below 2^32
constexpr int64_t kMostEntries = 0x7fffffffll - 256;
constexpr int kMostChannels    = 1 << 17;
constexpr double kLog2e = 1.4426950408889634;
constexpr double kLog2  = 0.6931471805599453;

// ---- rows that count ----

constexpr int kGatherRows = 16;     // rows of a workgroup
constexpr int kChunk      = 1024;   // targets of a chunk that count_kernel counts
constexpr int kAhead      = 4;      // pieces of 16 bytes that a thread asks for before it stores the first (8000 rows of 4000 floats 68 us one by one, 52 so)
constexpr int kCountedBy  = 8192;   // rows from which the chunks are counted beforehand (losses of 8191 rows of 16 floats 15.7 us without, 16.8 with; of 12,000 19.5 and 18.2)
constexpr int64_t kScannedBy = 1 << 19;  // rows from which the chunks' counts are summed beforehand, once for all workgroups, whose work would grow with the square of the rows (gathering 16 floats:
                                         // 262,144 rows 30 us without, 34 with; a million 119 and 110; 6M 1438 and 794)

// What the forward call leaves for the backward call; "packed" is an index among the rows that count.
struct Kept
{
    int* count;            // [1]
    int* place;            // [n]: where a row went, -1 if it does not count
    int* row;              // [packed]: where it comes from
    int* target;           // [packed]
    float2* state;         // [packed]: {largest product, log2 of the sum of exponentials over its own}
    void* packed;          // [packed][kp], zeros from the channels on; negated where scale is, so that the products need only |scale|
};

struct GatherParams
{
    const void* rows;
    const void* target;
    const int* chunk_count;  // targets that count of each chunk, or NULL: every workgroup looks at all targets
    int scanned;             // whether they are those of the chunks before instead, and of all chunks behind the last one
    Kept kept;
    long long n, entries, stride;
    int channels, kp, negate;
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

template <bool I32>
__global__ __launch_bounds__(256) void count_kernel(const void* target, long long n, long long entries, int* chunk_count)
{
    __shared__ int sums[4];
    int own = 0;
#pragma unroll
    for (int e = 0; e < kChunk / 256; ++e)
    {
        const long long i = (long long)blockIdx.x * kChunk + e * 256 + threadIdx.x;
        own += i < n && counts<I32>(target, i, entries);
    }
    own = wave_sum(own);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = own;
    __syncthreads();
    if (threadIdx.x == 0) chunk_count[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// Each chunk's count becomes that of the chunks before it; all of them behind the last. One workgroup: bound by latency, 1.5 us for each 4096 chunks.
__global__ __launch_bounds__(1024) void scan_kernel(int* count, long long chunks)
{
    __shared__ int sums[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int carry = 0;
    for (long long first = 0; first < chunks; first += 4096)
    {
        const long long i = first + threadIdx.x * 4;
        int own[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) own[e] = i + e < chunks ? count[i + e] : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += own[e];
        int up_to = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
        {
            const int x = __shfl_up(up_to, o);
            if (lane >= o) up_to += x;
        }
        if (lane == 63) sums[wave] = up_to;
        __syncthreads();
        int before = carry + up_to - sum;
        for (int w = 0; w < 16; ++w)
        {
            if (w < wave) before += sums[w];
            carry += sums[w];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            if (i + e < chunks) count[i + e] = before;
            before += own[e];
        }
        __syncthreads();  // (the sums are written again)
    }
    if (threadIdx.x == 0) count[chunks] = carry;
}

__device__ __forceinline__ float negative(float x) { return -x; }
__device__ __forceinline__ unsigned short negative(unsigned short x) { return x ^ 0x8000u; }

// A workgroup takes kGatherRows rows, or of few wide ones some of their pieces; it counts the rows that count before its own (and all of them) by itself, from the targets or
// from the chunks' counts: one launch, no order left to chance. Bound by latency, the targets and then the rows, and by memory for wide rows: 8191 rows of
// 1024 bfloat16 numbers 13 us, 8000 of 4000 floats 52 (4.9 TB/s).
template <int D, bool I32>
__global__ __launch_bounds__(256) void gather_kernel(const GatherParams p)
{
    using T         = typename Element<D>::type;
    constexpr int V = 16 / sizeof(T);
    __shared__ int before_w[4], all_w[4];
    __shared__ int own_place[kGatherRows];
    const long long first = (long long)blockIdx.x * kGatherRows;
    int before = 0, all = 0;
    if (p.chunk_count)
    {
        const long long chunks = (p.n + kChunk - 1) / kChunk, own_chunk = first / kChunk;
        if (p.scanned)
        {
            if (threadIdx.x == 0) before = p.chunk_count[own_chunk], all = p.chunk_count[chunks];
        }
        else
            for (long long c = threadIdx.x; c < chunks; c += 256)
            {
                const int k = p.chunk_count[c];
                all += k;
                if (c < own_chunk) before += k;
            }
        for (long long i = own_chunk * kChunk + threadIdx.x; i < first; i += 256) before += counts<I32>(p.target, i, p.entries);
    }
    else
        // (eight targets of a thread on their way at a time)
        for (long long i0 = threadIdx.x; i0 < p.n; i0 += 2048)
        {
            bool in[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) in[e] = counts<I32>(p.target, min(i0 + e * 256, p.n - 1), p.entries) && i0 + e * 256 < p.n;
#pragma unroll
            for (int e = 0; e < 8; ++e) all += in[e], before += in[e] && i0 + e * 256 < first;
        }
    before = wave_sum(before), all = wave_sum(all);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0) before_w[wave] = before, all_w[wave] = all;
    __syncthreads();
    if (wave == 0)
    {
        before              = before_w[0] + before_w[1] + before_w[2] + before_w[3];
        const long long i   = first + lane;
        const bool in       = lane < kGatherRows && i < p.n && counts<I32>(p.target, i, p.entries);
        const uint64_t mask = __ballot(in);
        if (lane < kGatherRows)
        {
            const int at    = in ? before + __popcll(mask & ((1ull << lane) - 1)) : -1;
            own_place[lane] = at;
            if (i < p.n && blockIdx.y == 0) p.kept.place[i] = at;
            if (in && blockIdx.y == 0)
            {
                p.kept.row[at]    = (int)i;
                p.kept.target[at] = I32 ? reinterpret_cast<const int32_t*>(p.target)[i] : (int)reinterpret_cast<const int64_t*>(p.target)[i];
            }
        }
        if (blockIdx.x == 0 && blockIdx.y == 0 && lane == 0) *p.kept.count = all_w[0] + all_w[1] + all_w[2] + all_w[3];
    }
    __syncthreads();
    using Wide       = typename Pack<T, V>::type;
    const int pieces = p.kp / V;
    for (int q0 = blockIdx.y * kAhead * 256 + threadIdx.x; q0 < kGatherRows * pieces; q0 += gridDim.y * kAhead * 256)
    {
        Wide x[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
        {
            const int q = q0 + k * 256, r = q / pieces, c = (q - r * pieces) * V;
            if (r >= kGatherRows || own_place[r] < 0) continue;
            const T* from = reinterpret_cast<const T*>(p.rows) + (first + r) * p.stride + c;
            if (c + V <= p.channels)
                x[k] = *reinterpret_cast<const Wide*>(from);
            else
#pragma unroll
                for (int e = 0; e < V; ++e) x[k][e] = c + e < p.channels ? from[e] : T(0);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
        {
            const int q = q0 + k * 256, r = q / pieces, c = (q - r * pieces) * V;
            if (r >= kGatherRows || own_place[r] < 0) continue;
            if (p.negate)
#pragma unroll
                for (int e = 0; e < V; ++e) x[k][e] = negative(x[k][e]);
            *reinterpret_cast<Wide*>(reinterpret_cast<T*>(p.kept.packed) + (long long)own_place[r] * p.kp + c) = x[k];
        }
    }
}

// ---- the loss's gradient ----

// d_ij is held for float16, whose range is short, 2^15 times as large and divided by the largest gradient of a row's loss: probabilities from
// 2^-29 on are normal numbers then. In the other types it is what it is, or without the gradient where that is the same of all rows.
template <int D>
constexpr float kHeld = D == TRIPS_DTYPE_F16 ? 32768.f : 1.f;

// In 16 bits d_ij is off by up to 2^-8 (bfloat16) or 2^-11 (float16) of itself, and so is what it adds to the gradients, which are rounded as far once more: their
// error against the exact ones is 1.1 to 1.8 times that of this last rounding alone, the more the fewer entries share a row's probability. Holding the
// rest of d_ij as well, as a second part of the same type, takes that away and doubles the gradients' products: done where those are few (see
// parts_of()).

constexpr int64_t kTopBy = 65536;  // rows from which several workgroups look for the largest gradient (with one 40,000 rows 6.5 us, with several 5.1 in two launches; 70,000 10 and 5.5, 6M 831 and 14)
constexpr int kTops      = 256;

// The largest |gradient| of the rows that count (not PLACED: of all), finite ones only: the others are left as they are. Of several workgroups each its own, which a second
// launch takes together.
template <bool PLACED>
__global__ __launch_bounds__(1024) void top_kernel(const float* d_loss, const int* place, long long n, float* top)
{
    __shared__ float tops[16];
    float own = 0.f;
    for (long long i0 = blockIdx.x * 8192ll + threadIdx.x; i0 < n; i0 += gridDim.x * 8192ll)
    {
        float g[8];
        int at[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = d_loss[min(i0 + e * 1024, n - 1)], at[e] = PLACED ? place[min(i0 + e * 1024, n - 1)] : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            const float size = fabsf(g[e]);
            if (at[e] >= 0 && size <= 3.4028234663852886e38f) own = fmaxf(own, size);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) own = fmaxf(own, __shfl_xor(own, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = own;
    __syncthreads();
    if (threadIdx.x > 0) return;
    for (int w = 0; w < 16; ++w) own = fmaxf(own, tops[w]);
    top[blockIdx.x] = gridDim.x > 1 || own > 0.f ? own : 1.f;
}

struct Upstream
{
    const float* d_loss;  // [n] or [1]
    const float* top;     // float16 and a gradient of each row
    int reduction;
    float scale;
};
// What a row's probabilities are multiplied by to be held, and what undoes that.
template <int D>
__device__ __forceinline__ float held_factor(const Upstream& u, int row)
{
    if (u.reduction != TRIPS_REDUCE_NONE) return kHeld<D>;
    return D == TRIPS_DTYPE_F16 ? u.d_loss[row] / *u.top * kHeld<D> : u.d_loss[row];
}
template <int D>
__device__ __forceinline__ float unheld(const Upstream& u, const int* count)
{
    float g = 1.f;
    if (u.reduction != TRIPS_REDUCE_NONE)
    {
        const int rows = *count;
        g              = rows == 0 ? 0.f : u.reduction == TRIPS_REDUCE_MEAN ? u.d_loss[0] / (float)rows : u.d_loss[0];  // (no row, no gradient, whatever the loss's is)
    }
    if (D == TRIPS_DTYPE_F16 && u.reduction == TRIPS_REDUCE_NONE) g = *u.top;
    return g / kHeld<D>;
}

// ---- products ----

// What a product's tiles are of: rows of the first operand run along a lane's registers, those of the second along the lanes.
//   LOGITS  entries x rows, over the channels: the largest product and the sum of exponentials of each row and stripe of tiles
//   PROBS   the same again: d_ij, [rows][piece]
//   D_ROWS  channels x rows, over the piece's entries
//   D_TABLE channels x entries, over the rows
//   GRADS   both of those
enum { LOGITS, PROBS, D_ROWS, D_TABLE, GRADS };

struct ProductParams
{
    const void* table;  // the piece's entries
    Kept kept;
    Upstream upstream;
    float2* partial;     // LOGITS: [tiles of entries][partial_pad] {largest product, sum of exponentials}
    float* own_product;  // [rows_pad]
    void* probs;         // [parts][rows_pad][piece], in the tensors' type
    float* slabs;        // D_ROWS: [splits][rows_pad][kp]
    float* table_slabs;  // D_TABLE, where in_table_slabs: [table_splits][piece][kp]
    const void* d_rows;  // whether they are wanted
    void* d_table;
    long long table_stride, d_table_stride, rows_pad, partial_pad;
    int held;  // channels that a row of the table has: those, or of a copy with zeros behind them to 16 bytes
    int first_entry, in_piece, channels, kp, piece, first_tile, splits, table_splits, parts, add;
    int first_row, most_rows;         // of the rows that count, those of the launch: kept is theirs (but for the count)
    int in_table_slabs, add_to_table;  // D_TABLE: whether its results are parts of sums, of the rows' (table_splits) or of the blocks of rows, and whether those have begun
    float scale_log2;
};

typedef float Acc __attribute__((ext_vector_type(16)));

// exp(scale (x - base)); 0 for an x of minus infinity.
__device__ __forceinline__ float part_of(float x, float base, float scale_log2) { return __builtin_amdgcn_exp2f((x - base) * scale_log2); }

// What -scale_log2 base - minus is beyond less - minus, for less = -scale_log2 base as rounded.
__device__ __forceinline__ float rest_of(float base, float scale_log2, float less, float minus)
{
    const float sum = less - minus, back = sum - less;
    return __builtin_fmaf(-base, scale_log2, -less) + ((less - (sum - back)) + (-minus - back));
}

// Entries one behind the other in rows of kp elements, zeros from the channels on: for tables whose rows the direct loads cannot take.
template <typename T>
__global__ __launch_bounds__(256) void copy_entries_kernel(const T* table, long long stride, T* to, long long entries, int channels, int kp)
{
    constexpr int V     = 16 / sizeof(T);
    using Wide          = typename Pack<T, V>::type;
    const int pieces    = kp / V;
    const long long all = entries * pieces;
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < all; q += (long long)gridDim.x * 256)
    {
        const long long j = q / pieces;
        const int c       = (int)(q % pieces) * V;
        const T* from     = table + j * stride + c;
        Wide x;
        if (c + V <= channels)
            x = *reinterpret_cast<const Wide*>(from);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = c + e < channels ? from[e] : T(0);
        *reinterpret_cast<Wide*>(to + q * V) = x;
    }
}

constexpr int kStepBytes = 128, kRounds = 4;  // of a row along k in a step; a round of the matrix instructions takes a quarter of them

// Tiles of BM x BN in steps along k, both operands by direct loads to LDS, STAGES steps of them at a time; WM x WN wavefronts, WK of them along a step's
// rounds, whose sums are joined behind the last step; PER_CU such workgroups.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int PER_CU_, int WK_ = 1>
struct Shape
{
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, PER_CU = PER_CU_, WK = WK_;
    static constexpr int WAVES = WM * WN * WK, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    static constexpr int FIRST_BYTES = BM * kStepBytes, SECOND_BYTES = BN * kStepBytes, STAGE_BYTES = FIRST_BYTES + SECOND_BYTES;
    static constexpr int FIRST_LOADS = FIRST_BYTES / 1024 / WAVES, SECOND_LOADS = SECOND_BYTES / 1024 / WAVES;
    static_assert(WK == 1 || (WK == kRounds && WM * WN == 1), "a round of each step for each wavefront");
    static_assert(FIRST_LOADS * WAVES * 1024 == FIRST_BYTES && SECOND_LOADS * WAVES * 1024 == SECOND_BYTES, "whole loads of a wavefront");
};

using Big   = Shape<256, 256, 2, 4, 2, 1>;
using Small = Shape<128, 128, 2, 2, 2, 2>;
using Tiny  = Shape<64, 64, 2, 2, 4, 2>;
// Of the gradients, whose units are many and may be of a few steps: a wavefront's waits for loads wait for the results stored before them too, which more
// workgroups hide and deeper loads do not (8000 rows of 90 entries of 4000 bfloat16 channels 168 us with Tiny, 108 so; 130 with three of each).
using Tight = Shape<64, 64, 2, 2, 2, 4>;
// Of the logits where tiles of 64 leave CUs without one, or rows are few: the wavefronts share each step's products, not the tile (4000 rows of 10 entries
// of 4000 floats 41 us, 89 with Tiny; 644 of 487 of 1596 28 and 40).
using Deep = Shape<32, 32, 1, 1, 4, 3, 4>;

typedef int Words4 __attribute__((ext_vector_type(4)));
typedef short Half4 __attribute__((ext_vector_type(4)));
typedef short Half8 __attribute__((ext_vector_type(8)));
typedef __bf16 Bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 F8 __attribute__((ext_vector_type(8)));
typedef float Float4 __attribute__((ext_vector_type(4)));

// 16 bytes a lane of either operand: 32 rows, the lane's element of it and those that follow along k, 16 (of 16 bits) or 8 in two halves of the
// wavefront. Which elements a half has does not matter, as long as it has the same ones of both operands.
template <int D>
__device__ __forceinline__ Acc product(Half8 a, Half8 b, Acc c)
{
    if constexpr (D == TRIPS_DTYPE_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf8, a), __builtin_bit_cast(Bf8, b), c, 0, 0, 0);
    else if constexpr (D == TRIPS_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(F8, a), __builtin_bit_cast(F8, b), c, 0, 0, 0);
    else
    {
        const Float4 x = __builtin_bit_cast(Float4, a), y = __builtin_bit_cast(Float4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
}

// 64 lanes' 16 bytes from a buffer, each at its own offset, to LDS one behind the other; zeros from beyond the buffer's end.
// (By itself: of a builtin the compiler would wait for the last load before any read of LDS.)
__device__ __forceinline__ void load_to_lds(const Words4& buffer, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory", "m0");
}
__device__ __forceinline__ Words4 buffer_of(const void* base, long long bytes)
{
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    const int n      = (int)min(max(bytes, 0ll), 0x7fffffffll);
    return Words4{__builtin_amdgcn_readfirstlane((int)a), __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xFFFF)), __builtin_amdgcn_readfirstlane(n), 0x00020000};
}
template <int LOADS>
__device__ __forceinline__ void wait_and_meet()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
}

// (of LDS; the loads under way stay so)
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Up to which |base| scale_log2 the distance from the largest product is taken behind the scaling, scale x + less in one operation with less = -scale base, in
// types of 16 bits. Products masked with the lowest value lie beyond it. The rounding of `less` is the same for all of a row's products and known
// (rest_of()): the sums are corrected by it, without which a row whose target is far ahead lost less than nothing (-3e-4 at logits of 10^4). Of d_ij only
// the target's, a difference of two numbers near 1, is corrected; for the others it stays below 2^-16 of them, less than d_ij in 16 bits shows.
constexpr float kFar = 65536.f, kFarOfOne = 256.f;

constexpr unsigned kBeyond = 0x80000000u;  // an offset beyond any buffer

// Where a wavefront's loads of an operand's steps come from: each lane's offsets, the same for all tiles, and the operand's elements from the
// next step on.
template <int LOADS>
struct Source
{
    unsigned offset[LOADS];
    const char* base;
    long long bytes, step;
    __device__ __forceinline__ void at(const void* from, long long size) { base = reinterpret_cast<const char*>(from), bytes = size; }
    __device__ __forceinline__ void next() { base += step, bytes -= step; }
    __device__ __forceinline__ void load(int i, unsigned lds, int wave) const { load_to_lds(buffer_of(base, bytes), offset[i], lds + (wave * LOADS + i) * 1024); }
    // of rows along k, of which `left` elements are left: zeros behind them
    __device__ __forceinline__ void load(int i, unsigned lds, int wave, int k, int left) const
    {
        load_to_lds(buffer_of(base, bytes), k < left ? offset[i] : kBeyond, lds + (wave * LOADS + i) * 1024);
    }
};

// An operand whose rows run along k: LDS rows of 128 bytes, their pieces of 16 in an order that depends on the row, so that 16 lanes that
// read the same piece of 16 rows meet 16 different places of the 256 bytes that the banks of LDS are wide.
template <int ROWS, int LOADS>
struct AlongK
{
    static constexpr int PIECES = kStepBytes / 16;
    static __device__ __forceinline__ int turn(int row) { return (row >> 1) & 7; }
    static __device__ __forceinline__ int row_of(int i, int wave, int lane) { return (wave * LOADS + i) * (64 / PIECES) + lane / PIECES; }
    static __device__ __forceinline__ int piece_of(int i, int wave, int lane) { return (lane % PIECES) ^ turn(row_of(i, wave, lane)); }
    static __device__ __forceinline__ void begin(Source<LOADS>& s, long long stride_bytes, int wave, int lane)
    {
        s.step = kStepBytes;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) s.offset[i] = (unsigned)(row_of(i, wave, lane) * stride_bytes) + piece_of(i, wave, lane) * 16;
    }
    // fragment f of the wavefront's rows from `row` on, round kk
    static __device__ __forceinline__ Half8 read(const char* lds, int row, int f, int kk, int lane)
    {
        const int r = row + (lane & 31);
        return *reinterpret_cast<const Half8*>(lds + (r + f * 32) * kStepBytes + (((kk * 2 + (lane >> 5)) ^ turn(r)) * 16));
    }
};

// An operand whose rows run along the tile: LDS rows of ROWS elements, one of each k. Of 16 bits they are read through the transposing loads (of
// 16 lanes' four elements: lane i gets element i % 4 of lanes i / 4, i / 4 + 4, ...). A row's pieces of 64 bytes (32 bits: 128) are in an order
// that depends on k, so that the four (two) rows that are read at once lie apart.
template <int SIZE, int ROWS, int LOADS>
struct AcrossK
{
    static constexpr int PIECES = ROWS * SIZE / 16, GROUP = SIZE == 2 ? 4 : 8, TURNS = PIECES / GROUP;
    static __device__ __forceinline__ int turn(int k) { return (SIZE == 2 ? (k & 3) | ((k >> 3) & 1) << 2 : (k >> 2) & 1) & (TURNS - 1); }
    static __device__ __forceinline__ void begin(Source<LOADS>& s, long long stride_bytes, int wave, int lane)
    {
        s.step = kStepBytes / SIZE * stride_bytes;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
        {
            const int at = (wave * LOADS + i) * 64 + lane, k = at / PIECES, piece = at % PIECES;
            s.offset[i]  = (unsigned)(k * stride_bytes) + (((piece / GROUP) ^ turn(k)) * GROUP + piece % GROUP) * 16;
        }
    }
    static __device__ __forceinline__ Half8 read(const char* lds, int row, int f, int kk, int lane)
    {
        if constexpr (SIZE == 2)
        {
            const int k    = kk * 16 + (lane >> 5) * 8 + ((lane >> 2) & 3);
            const char* at = lds + k * (ROWS * 2) + (((row >> 5) + f) ^ turn(k)) * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
            using P        = __attribute__((address_space(3))) Half4*;
            const Half4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)at), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 4 * ROWS * 2));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        else
        {
            const int k     = kk * 8 + (lane >> 5) * 4;
            const float* at = reinterpret_cast<const float*>(lds + k * (ROWS * 4) + (((row >> 5) + f) ^ turn(k)) * 128) + (lane & 31);
            return __builtin_bit_cast(Half8, Float4{at[0], at[ROWS], at[2 * ROWS], at[3 * ROWS]});
        }
    }
};

// f(fragment, element of it, row of a lane's first fragment) for each of a lane's elements of one column of fragments
template <int FM, typename F>
__device__ __forceinline__ void each_element(F f)
{
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) f(i, e, i * 32 + 8 * (e >> 2) + (e & 3));
}

// Two numbers rounded to 16 bits, side by side.
template <int D>
__device__ __forceinline__ unsigned pair_of(float a, float b)
{
    using Type = std::conditional_t<D == TRIPS_DTYPE_BF16, __bf16, _Float16>;
    typedef Type Two __attribute__((ext_vector_type(2)));
    typedef float Floats __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector(Floats{a, b}, Two));
}

// A workgroup's share of a launch: its tiles, one after the other.
struct Unit
{
    int mode;  // of the tile, -1: there is no further one
    int x, y, z, steps;
};

// Eight tiles along y share one along x at a time: consecutive tiles go to one XCD, whose L2 holds what they share.
__device__ __forceinline__ void place(Unit& u, int id, int across, int down)
{
    u.z         = id / (across * down);
    id          = id % (across * down);
    const int g = id / (across * 8), in = id % (across * 8), high = min(8, down - g * 8);
    u.x = in / high, u.y = g * 8 + in % high;
}

// Where part z of `steps` in `parts` begins (steps are below 2^26, parts at most 64). Units of one step are made faster than they are worked out: no
// division where there is one part.
__device__ __forceinline__ int part_begin(int z, int steps, int parts) { return parts == 1 ? z * steps : (int)((unsigned)z * (unsigned)steps / (unsigned)parts); }

// The units of worker w of `all`: unit w, w + all, ... of the larger kind (a of them, size_a steps each), then those of the smaller kind: workers
// that have one of the larger kind less take so many smaller ones first.
struct Share
{
    int a, size_a, b, size_b;
};
__device__ __forceinline__ int share_of(const Share& s, int ordinal, int w, int all, bool& second)
{
    const int own = w < s.a ? (s.a - w + all - 1) / all : 0;
    second        = ordinal >= own;
    if (!second) return w + ordinal * all;
    const int rest = s.a % all, early = rest == 0 ? 0 : all - rest, more = early && s.size_b > 0 ? s.size_a / s.size_b : 0;
    int j = ordinal - own;
    if (early && w >= rest)
    {
        if (j < more) return w - rest + j * early;
        j -= more;
    }
    return early * more + (w >= rest ? w - rest : w + early) + j * all;
}

// Large problems of 16 bits are bound by the card's power and by the tiles' results: the matrix instructions fill 52 to 66 % of a busy CU's cycles at 1.6 to 1.9 GHz of 2.4, no bank
// of LDS conflicts, and fewer waits lower the clock. What is left of the cycles goes to the results: of 772 and 830 us for the logits of 7782 rows and 50,000 entries of
// 1024 bfloat16 channels and their gradient 637 and 633 are without them. There: logits 731 to 774 us (1.06 PFLOP/s), their gradient 813 to 837 (0.97), both gradients 1395 to 1408
// (1.14; a library's product of 16384 a side reaches 1.58, of these sizes 1.20). In 32 bits the matrix instructions fill 80 to 87 % at 2.2 GHz (1023 rows, 20,000 entries
// of 384: 144, 152 and 289 us, 108 TFLOP/s of 154). Few rows are bound by the table's way in: one row and 50,000 entries of 1024 bfloat16 channels 21.3 us, 4.8 TB/s.
//
// LOGITS, PROBS, or GRADS: D_ROWS and D_TABLE in one launch. S::PER_CU workgroups a CU, each goes through its units; the loads run STAGES steps
// ahead of the products and go on into the next unit, so that they are under way while a unit's results are written.
template <int D, int KIND, typename S>
__global__ __launch_bounds__(S::WAVES * 64, S::PER_CU * S::WAVES / 4) void product_kernel(const ProductParams p)
{
    using E = Element<D>;
    using T = typename E::type;
    constexpr int SIZE = sizeof(T), BK = kStepBytes / SIZE, LOADS = S::FIRST_LOADS + S::SECOND_LOADS, LATE = LOADS / 2;
    using FirstAlong   = AlongK<S::BM, S::FIRST_LOADS>;
    using FirstAcross  = AcrossK<SIZE, S::BM, S::FIRST_LOADS>;
    using SecondAlong  = AlongK<S::BN, S::SECOND_LOADS>;
    using SecondAcross = AcrossK<SIZE, S::BN, S::SECOND_LOADS>;
    __shared__ __attribute__((aligned(1024))) char lds[S::STAGES * S::STAGE_BYTES];
    __shared__ float2 joined[KIND == LOGITS ? S::WM * S::BN : 1];
    __shared__ Acc others[S::WK > 1 ? S::WK - 1 : 1][S::WK > 1 ? 64 : 1];
    const unsigned lds_at = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool writes = S::WK == 1 || wave == 0;
    const int wm = wave % S::WM * S::TM, wn = wave / S::WM % S::WN * S::TN;
    const int count = min(max(*p.kept.count - p.first_row, 0), p.most_rows);

    // Workgroups as they start go around the eight XCDs: of each 256, which take a CU each, workers by XCD.
    const int all = gridDim.x, run = (int)blockIdx.x & ~255, runs = min(256, all - run), in_run = (int)blockIdx.x & 255;
    const int worker = run + (runs % 8 ? in_run : in_run % 8 * (runs / 8) + in_run / 8);
    const int row_tiles = (count + S::BN - 1) / S::BN, entry_tiles = (p.in_piece + (KIND == GRADS ? S::BN : S::BM) - 1) / (KIND == GRADS ? S::BN : S::BM);
    const int channel_tiles = (p.channels + S::BM - 1) / S::BM;
    const int piece_steps = (p.in_piece + BK - 1) / BK, row_steps = (count + BK - 1) / BK;
    constexpr bool TABLE_SPLITS = KIND == GRADS && S::BM < Big::BM;  // (tiles of 256 make units enough by themselves)
    const int table_splits      = TABLE_SPLITS ? p.table_splits : 1;
    Share share{};
    bool rows_first = true;
    if constexpr (KIND == GRADS)
    {
        const int rows = p.d_rows ? channel_tiles * row_tiles * p.splits : 0, table = p.d_table ? channel_tiles * entry_tiles * table_splits : 0;
        const int rows_size = piece_steps / p.splits, table_size = row_steps / table_splits;
        rows_first = rows_size >= table_size;
        share      = rows_first ? Share{rows, rows_size, table, table_size} : Share{table, table_size, rows, rows_size};
    }
    else
        share = Share{entry_tiles * row_tiles, 1, 0, 1};
    auto unit_of = [&](int ordinal)
    {
        Unit u{};
        bool second;
        const int id = share_of(share, ordinal, worker, all, second);
        if (id >= (second ? share.b : share.a))
        {
            u.mode = -1;
            return u;
        }
        if constexpr (KIND == GRADS)
        {
            u.mode = second == rows_first ? D_TABLE : D_ROWS;
            if (u.mode == D_ROWS)
            {
                place(u, id, channel_tiles, row_tiles);
                u.steps = part_begin(u.z + 1, piece_steps, p.splits) - part_begin(u.z, piece_steps, p.splits);
            }
            else
            {
                place(u, id, channel_tiles, entry_tiles);
                u.steps = part_begin(u.z + 1, row_steps, table_splits) - part_begin(u.z, row_steps, table_splits);
            }
        }
        else
        {
            u.mode = KIND, u.steps = (p.held + BK - 1) / BK;
            place(u, id, entry_tiles, row_tiles);
        }
        return u;
    };

    // ---- the loads, ahead ----
    const char* table  = reinterpret_cast<const char*>(p.table);
    const char* packed = reinterpret_cast<const char*>(p.kept.packed);
    const char* probs  = reinterpret_cast<const char*>(p.probs);
    Source<S::FIRST_LOADS> first;
    Source<S::SECOND_LOADS> second;
    int ahead_ordinal = 0, ahead_part = 0, ahead_mode = -1, ahead_steps = 0, left = 0;
    auto open = [&]()
    {
        Unit u = unit_of(ahead_ordinal);
        while (u.mode >= 0 && u.steps == 0) u = unit_of(++ahead_ordinal);
        ahead_steps = u.mode < 0 ? 0x7fffffff : u.steps;
        if (u.mode < 0)
        {
            first.at(table, 0), second.at(table, 0);  // (zeros, so that the waits count alike)
            first.step = second.step = 0;
            return;
        }
        const char* part       = probs + ahead_part * p.rows_pad * p.piece * SIZE;
        const long long stride = p.table_stride * SIZE, wide = (long long)p.kp * SIZE, piece = (long long)p.piece * SIZE, held = ((long long)p.held * SIZE + 3) / 4 * 4;
        if constexpr (KIND != GRADS)
        {
            if (ahead_mode != u.mode) FirstAlong::begin(first, stride, wave, lane), SecondAlong::begin(second, wide, wave, lane);
            const long long m0 = (long long)u.x * S::BM, n0 = (long long)u.y * S::BN;
            first.at(table + m0 * stride, (min(p.in_piece - m0, (long long)S::BM) - 1) * stride + held);
            second.at(packed + n0 * wide, (count - n0) * wide);
            left = p.held;
        }
        else if (u.mode == D_ROWS)
        {
            if (ahead_mode != u.mode) FirstAcross::begin(first, stride, wave, lane), SecondAlong::begin(second, piece, wave, lane);
            const long long k = (long long)part_begin(u.z, piece_steps, p.splits) * BK, m0 = (long long)u.x * S::BM * SIZE, n0 = (long long)u.y * S::BN;
            first.at(table + k * stride + m0, (p.in_piece - 1 - k) * stride + held - m0);
            second.at(part + n0 * piece + k * SIZE, (p.rows_pad - n0) * piece - k * SIZE);
        }
        else
        {
            if (ahead_mode != u.mode) FirstAcross::begin(first, wide, wave, lane), SecondAcross::begin(second, piece, wave, lane);
            const long long k = (long long)part_begin(u.z, row_steps, table_splits) * BK, m0 = (long long)u.x * S::BM * SIZE, n0 = (long long)u.y * S::BN * SIZE;
            first.at(packed + k * wide + m0, (count - k) * wide - m0);
            second.at(part + k * piece + n0, (count - k) * piece - n0);
        }
        ahead_mode = u.mode;
    };
    auto load = [&](int i, int stage)
    {
        const unsigned to = lds_at + stage * S::STAGE_BYTES;
        if (i < S::FIRST_LOADS)
        {
            if (KIND != GRADS)
                first.load(i, to, wave, FirstAlong::piece_of(i, wave, lane) * (16 / SIZE), left);
            else
                first.load(i, to, wave);
        }
        else
        {
            const int q = i - S::FIRST_LOADS;
            if (KIND != GRADS)
                second.load(q, to + S::FIRST_BYTES, wave, SecondAlong::piece_of(q, wave, lane) * (16 / SIZE), left);
            else
                second.load(q, to + S::FIRST_BYTES, wave);
        }
    };
    auto loaded_step = [&]()
    {
        first.next(), second.next();
        left -= BK;
        if (--ahead_steps > 0) return;
        if (KIND != GRADS || ++ahead_part == p.parts) ++ahead_ordinal, ahead_part = 0;
        open();
    };
    open();
#pragma unroll
    for (int s = 0; s < S::STAGES; ++s)
    {
#pragma unroll
        for (int i = 0; i < (s + 1 < S::STAGES ? LOADS : LOADS - LATE); ++i) load(i, s);
        if (s + 1 < S::STAGES || LATE == 0) loaded_step();
    }
    wait_and_meet<(S::STAGES - 1) * LOADS - LATE>();
    int stage = 0;

    // ---- a unit's products ----
    Acc acc[S::FM][S::FN];
    // Of the lane's rows of the second operand (LOGITS, PROBS): asked for before a unit's first step and there behind its first meeting. (A wait for
    // a load waits for all that went before it, and as the compiler counts them for those behind it too: when the results are written, the next unit's.)
    int target[S::FN];
    float2 state[S::FN];
    auto ask = [&](const Unit& u)
    {
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
        {
            const long long n = min((long long)u.y * S::BN + wn + j * 32 + (lane & 31), count - 1ll);
            target[j]         = p.kept.target[n];
            if (KIND == PROBS) state[j] = p.kept.state[n];
        }
    };
    auto receive = [&]()
    {
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
        {
            asm volatile("" : "+v"(target[j]));
            if (KIND == PROBS) asm volatile("" : "+v"(state[j].x), "+v"(state[j].y));
        }
    };
    auto products = [&](auto along, int steps)
    {
        using First  = std::conditional_t<KIND == GRADS, FirstAcross, FirstAlong>;
        using Second = std::conditional_t<decltype(along)::value, SecondAlong, SecondAcross>;
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
        // Fragments are read a round of the matrix instructions ahead of their use, those of the next step's first round behind the one
        // meeting of a step, which says that every wavefront has read what the next loads replace, and that the next step is there. The
        // loads go out between the last round's instructions.
        Half8 x[2][S::FM], y[2][S::FN];
        auto read = [&](int set, int from, int kk)
        {
            const char* a = lds + from * S::STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < S::FM; ++i) x[set][i] = First::read(a, wm, i, kk, lane);
#pragma unroll
            for (int j = 0; j < S::FN; ++j) y[set][j] = Second::read(a + S::FIRST_BYTES, wn, j, kk, lane);
        };
        // Of a table whose rows are no whole pieces of 16 bytes, the last one that a row has brings elements of what lies behind the row: they meet
        // zeros of the second operand, but might be no numbers.
        constexpr int V = 16 / SIZE;
        const bool ragged = KIND != GRADS && p.held % V;
        auto clear_ends = [&](int of)
        {
            for (int row = threadIdx.x; row < S::BM; row += S::WAVES * 64)
            {
                T* piece = reinterpret_cast<T*>(lds + of * S::STAGE_BYTES + row * kStepBytes + ((p.held % BK / V) ^ FirstAlong::turn(row)) * 16);
                for (int e = p.held % V; e < V; ++e) piece[e] = 0;
            }
            meet();
        };
        if (ragged && steps == 1) clear_ends(stage);
        if (steps > 0) read(0, stage, S::WK > 1 ? wave : 0);
        for (int step = 0; step < steps; ++step)
        {
            const int next = stage + 1 == S::STAGES ? 0 : stage + 1, free = stage == 0 ? S::STAGES - 1 : stage - 1;
            if constexpr (S::WK > 1)
            {
                // (each wavefront its own round of every step)
#pragma unroll
                for (int i = LOADS - LATE; i < LOADS; ++i) load(i, free);
                if (LATE > 0) loaded_step();
                acc[0][0] = product<D>(x[0][0], y[0][0], acc[0][0]);
                wait_and_meet<(S::STAGES - 2) * LOADS>();
                if (KIND != GRADS && step == 0) receive();
                if (ragged && step + 2 == steps) clear_ends(next);
                read(0, next, wave);
#pragma unroll
                for (int i = 0; i < LOADS - LATE; ++i) load(i, stage);
            }
            else
#pragma unroll
            for (int kk = 0; kk < kRounds; ++kk)
            {
                if (kk + 1 < kRounds)
                    read((kk + 1) & 1, stage, kk + 1);
                else
                {
                    wait_and_meet<(S::STAGES - 2) * LOADS>();
                    if (KIND != GRADS && step == 0) receive();
                    if (ragged && step + 2 == steps) clear_ends(next);
                    read(0, next, 0);  // (behind the last step: of the next unit, which reads it again)
                }
                __builtin_amdgcn_sched_barrier(0);
                // of `of` loads from `from` on, the share behind product q of the round
                auto loads = [&](int q, int from, int of, int to)
                {
                    constexpr int PAIRS = S::FM * S::FN;
#pragma unroll
                    for (int i = from + q * of / PAIRS; i < from + (q + 1) * of / PAIRS; ++i) load(i, to);
                };
#pragma unroll
                for (int i = 0; i < S::FM; ++i)
#pragma unroll
                    for (int j = 0; j < S::FN; ++j)
                    {
                        acc[i][j] = product<D>(x[kk & 1][i], y[kk & 1][j], acc[i][j]);
                        if (kk == 0 && LATE > 0) loads(i * S::FN + j, LOADS - LATE, LATE, free);
                        if (kk + 1 == kRounds) loads(i * S::FN + j, 0, LOADS - LATE, stage);
                        if (kk == 0 || kk + 1 == kRounds) __builtin_amdgcn_sched_barrier(0);
                    }
                __builtin_amdgcn_sched_barrier(0);
                if (LATE > 0 && kk == 0) loaded_step();
            }
            if (LATE == 0) loaded_step();
            stage = next;
        }
        if constexpr (S::WK > 1)
        {
            if (wave > 0) others[wave - 1][lane] = acc[0][0];
            meet();
            if (wave == 0)
#pragma unroll
                for (int w = 0; w < S::WK - 1; ++w) acc[0][0] += others[w][lane];
        }
    };

    // ---- a unit's results ----
    // a lane's elements: of row n0 + wn + 32 j + lane % 32, of the first operand's rows m0 + wm + 32 i + 8 (e / 4) + 4 (lane / 32) + e % 4
    auto sums = [&](const Unit& u)
    {
        const long long n0 = (long long)u.y * S::BN;
        const int m0 = u.x * S::BM, m_lane = m0 + wm + 4 * (lane >> 5);
        float2 best[S::FN];
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
        {
            if (!writes) break;
            const long long n = n0 + wn + j * 32 + (lane & 31);
            const int own     = n < count ? target[j] - p.first_entry - m_lane : -1;  // (of the lane's own elements)
            float top         = -__builtin_inff();
            if (m0 + S::BM > p.in_piece)
                each_element<S::FM>([&](int i, int e, int m)
                {
                    if (m_lane + m >= p.in_piece) acc[i][j][e] = -__builtin_inff();
                });
            if (__any(own >= 0 && own < S::TM))
            {
                float product = 0.f;
                bool here     = false;
                each_element<S::FM>([&](int i, int e, int m)
                {
                    if (m == own) product = acc[i][j][e], here = m_lane + m < p.in_piece;
                });
                if (here) p.own_product[n] = product;
            }
            // (the larger: fmaxf would first quiet each product's NaN by an operation of its own)
            each_element<S::FM>([&](int i, int e, int) { top = __builtin_amdgcn_fmed3f(top, acc[i][j][e], __builtin_inff()); });
            top              = fmaxf(top, __shfl_xor(top, 32));
            const float base = top == -__builtin_inff() ? 0.f : top, less = -base * p.scale_log2;
            float sum        = 0.f;
            const bool near  = D != TRIPS_DTYPE_F32 && fabsf(less) < kFar;  // (each lane by itself: a row's bits do not depend on other rows)
            if (near)
                each_element<S::FM>([&](int i, int e, int) { sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], p.scale_log2, less)); });
            else
                each_element<S::FM>([&](int i, int e, int) { sum += part_of(acc[i][j][e], base, p.scale_log2); });
            sum += __shfl_xor(sum, 32);
            if (near)
            {
                sum *= __builtin_amdgcn_exp2f(rest_of(base, p.scale_log2, less, 0.f));
                if (top > -__builtin_inff() && sum < 1.f) sum = 1.f;  // (the largest one's own)
            }
            best[j] = make_float2(top, sum);
        }
        meet();  // (the last unit's have been read)
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
            if (lane < 32 && writes) joined[wave % S::WM * S::BN + wn + j * 32 + lane] = best[j];
        meet();
        for (int n = threadIdx.x; n < S::BN; n += S::WAVES * 64)
        {
            float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
            for (int w = 0; w < S::WM; ++w) top = fmaxf(top, joined[w * S::BN + n].x);
            const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
            for (int w = 0; w < S::WM; ++w) sum += joined[w * S::BN + n].y * part_of(joined[w * S::BN + n].x, base, p.scale_log2);
            p.partial[(p.first_tile + u.x) * p.partial_pad + n0 + n] = make_float2(top, sum);
        }
    };
    auto written = [&](auto mode, const Unit& u)
    {
        constexpr int MODE = decltype(mode)::value;
        const long long n0 = (long long)u.y * S::BN;
        const int m0 = u.x * S::BM, m_lane = m0 + wm + 4 * (lane >> 5);
        const bool in_slabs = TABLE_SPLITS && MODE == D_TABLE && p.in_table_slabs;
        const float unscale = MODE == D_TABLE && !in_slabs ? unheld<D>(p.upstream, p.kept.count) * fabsf(p.upstream.scale) : 1.f;
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
        {
            const long long n = n0 + wn + j * 32 + (lane & 31);
            if constexpr (MODE == PROBS)
            {
                const float2 of = state[j];
                const int own      = n < count ? target[j] - p.first_entry - m_lane : -1;
                const float factor = held_factor<D>(p.upstream, p.upstream.reduction == TRIPS_REDUCE_NONE ? p.kept.row[min(n, count - 1ll)] : 0);
                const float less   = -of.x * p.scale_log2, held = D == TRIPS_DTYPE_F16 ? factor : 1.f;
                const bool near = D != TRIPS_DTYPE_F32 && fabsf(less) < kFarOfOne;
                if (near)
                    each_element<S::FM>([&](int i, int e, int) { acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], p.scale_log2, less - of.y)) * held; });
                else
                    each_element<S::FM>([&](int i, int e, int) { acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e] - of.x, p.scale_log2, -of.y)) * held; });
                if (D != TRIPS_DTYPE_F16 && p.upstream.reduction == TRIPS_REDUCE_NONE) each_element<S::FM>([&](int i, int e, int) { acc[i][j][e] *= factor; });
                if (__any(own >= 0 && own < S::TM))
                {
                    const float rest = near ? __builtin_amdgcn_exp2f(rest_of(of.x, p.scale_log2, less, of.y)) : 1.f;
                    each_element<S::FM>([&](int i, int e, int m)
                    {
                        if (m == own) acc[i][j][e] = acc[i][j][e] * rest - factor;
                    });
                }
                if (m0 + S::BM > p.in_piece)
                    each_element<S::FM>([&](int i, int e, int m)
                    {
                        if (m_lane + m >= p.in_piece) acc[i][j][e] = 0.f;
                    });
            }
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
            {
                if (MODE == D_ROWS || in_slabs)
                {
                    float* slab = MODE == D_ROWS ? p.slabs + ((long long)u.z * p.rows_pad + n) * p.kp : p.table_slabs + ((long long)u.z * p.piece + n) * p.kp;
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                    {
                        const int c = m_lane + i * 32 + 8 * g;
                        using F4    = Pack<float, 4>::type;
                        if (n < (MODE == D_ROWS ? count : p.in_piece) && c < p.kp)
                        {
                            F4* at = reinterpret_cast<F4*>(slab + c);
                            F4 v   = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                            if (MODE == D_ROWS ? p.add : p.add_to_table) v += *at;
                            *at = v;
                        }
                    }
                    continue;
                }
                if constexpr (MODE != D_ROWS && D == TRIPS_DTYPE_F32)
                {
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                    {
                        const int m = m_lane + i * 32 + 8 * g;
                        using F4    = Pack<float, 4>::type;
                        const F4 v  = {acc[i][j][4 * g] * unscale, acc[i][j][4 * g + 1] * unscale, acc[i][j][4 * g + 2] * unscale, acc[i][j][4 * g + 3] * unscale};
                        if constexpr (MODE == PROBS)
                        {
                            if (n < count) *reinterpret_cast<F4*>(reinterpret_cast<float*>(p.probs) + n * p.piece + m) = v;
                        }
                        else if (n < p.in_piece && m < p.channels)
                        {
                            float* at = reinterpret_cast<float*>(p.d_table) + n * p.d_table_stride + m;
                            if (m + 4 <= p.channels)
                                *reinterpret_cast<F4*>(at) = v;
                            else
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (m + e < p.channels) at[e] = v[e];
                        }
                    }
                }
            }
            if constexpr (D != TRIPS_DTYPE_F32 && MODE != D_ROWS)
            {
                if (in_slabs) continue;
                // Two lanes' fours to eight of one lane: 16 bytes, 32 of each of 32 rows at a time. (Turned in LDS to runs of 128 bytes before they were stored,
                // the logits' gradient took 999 us where it takes 857 so: its wavefronts have nothing to do while they wait for LDS.)
                using T8 = Pack<unsigned short, 8>::type;
                auto out = [&](auto value, T* to, long long stride, long long rows, int columns)
                {
#pragma unroll
                    for (int i = 0; i < S::FM; ++i)
#pragma unroll
                        for (int g = 0; g < 4; g += 2)
                        {
                            unsigned w[4];
#pragma unroll
                            for (int h = 0; h < 4; ++h) w[h] = pair_of<D>(value(acc[i][j][4 * g + 2 * h]), value(acc[i][j][4 * g + 2 * h + 1]));
                            const auto low = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), high = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                            const T8 v  = __builtin_bit_cast(T8, Words4{(int)low[0], (int)high[0], (int)low[1], (int)high[1]});
                            const int m = m0 + wm + i * 32 + 8 * (g + (lane >> 5));
                            T* x        = to + n * stride + m;
                            if (n >= rows || m >= columns) continue;
                            if (m + 8 <= columns)
                                *reinterpret_cast<T8*>(x) = v;
                            else
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    if (m + e < columns) x[e] = v[e];
                        }
                };
                if constexpr (MODE == PROBS)
                {
                    T* to = reinterpret_cast<T*>(p.probs);
                    out([](float x) { return x; }, to, p.piece, count, 0x7fffffff);
                    if (p.parts > 1) out([](float x) { return x - E::to_float(E::from_float(x)); }, to + p.rows_pad * p.piece, p.piece, count, 0x7fffffff);
                }
                else
                    out([&](float x) { return x * unscale; }, reinterpret_cast<T*>(p.d_table), p.d_table_stride, p.in_piece, p.channels);
            }
        }
    };

    for (int ordinal = 0;; ++ordinal)
    {
        const Unit u = unit_of(ordinal);
        if (u.mode < 0) break;
        if constexpr (KIND == LOGITS)
        {
            ask(u);
            products(std::true_type{}, u.steps);
            sums(u);
        }
        else if constexpr (KIND == PROBS)
        {
            ask(u);
            products(std::true_type{}, u.steps);
            if (writes) written(std::integral_constant<int, PROBS>{}, u);
            // (zeros behind the piece's last entry to a whole step of the gradients)
            if (S::BM < BK && wave == 1 && u.x + 1 == entry_tiles && entry_tiles % (BK / S::BM) != 0)
            {
                const long long n = (long long)u.y * S::BN + (lane & 31);
                if (n < count)
                    for (int part = 0; part < p.parts; ++part)
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            *reinterpret_cast<Words4*>(reinterpret_cast<T*>(p.probs) + (part * p.rows_pad + n) * p.piece + (u.x + 1) * S::BM + ((lane >> 5) * 2 + q) * 8) = Words4{};
            }
        }
        else if (u.mode == D_ROWS)
        {
            products(std::true_type{}, u.steps * p.parts);
            written(std::integral_constant<int, D_ROWS>{}, u);
        }
        else
        {
            products(std::false_type{}, u.steps * p.parts);
            written(std::integral_constant<int, D_TABLE>{}, u);
        }
    }
    wait_and_meet<0>();  // (nothing is on its way to LDS when the workgroup ends)
}

// ---- joins ----

// 1 << lanes_log2 lanes a row over the tiles: state and loss, and the workgroup's sum of losses; of tiles that are not all, the sum of exponentials in the place of its logarithm. Bound by latency: 4 us for few tiles and rows, 10 for 7782 rows and
// 196 tiles (12 MB).
struct JoinParams
{
    const float2* partial;
    const float* own_product;
    Kept kept;
    float* loss;
    double* sums;
    long long n, partial_pad;
    int tiles, reduction, lanes_log2;
    int more, last;  // whether earlier tiles are in the state; whether there are no further ones
    float scale, scale_log2;
};
__global__ __launch_bounds__(256) void join_kernel(const JoinParams p)
{
    __shared__ float2 part[256];
    __shared__ double sums[4];
    const int rows_log2 = 8 - p.lanes_log2, row = threadIdx.x & ((1 << rows_log2) - 1), lanes = 1 << p.lanes_log2;
    const long long i = ((long long)blockIdx.x << rows_log2) + row;
    const int at      = i < p.n ? p.kept.place[i] : -1;
    float2 own        = make_float2(-__builtin_inff(), 0.f);
    if (at >= 0)
    {
        const float product = p.own_product[at];
        if (p.more && threadIdx.x >> rows_log2 == 0) own = p.kept.state[at];
#pragma unroll 4
        for (int s = threadIdx.x >> rows_log2; s < p.tiles; s += lanes)
        {
            const float2 x  = p.partial[s * p.partial_pad + at];
            const float top = fmaxf(own.x, x.x), base = top == -__builtin_inff() ? 0.f : top;
            own = make_float2(top, own.y * part_of(own.x, base, p.scale_log2) + x.y * part_of(x.x, base, p.scale_log2));
        }
        part[threadIdx.x] = own;
        own.y             = product;
    }
    for (int o = lanes >> 1; o > 0; o >>= 1)
    {
        __syncthreads();
        if (threadIdx.x >> rows_log2 < o && at >= 0)
        {
            const float2 x = part[threadIdx.x], y = part[threadIdx.x + (o << rows_log2)];
            const float top = fmaxf(x.x, y.x), base = top == -__builtin_inff() ? 0.f : top;
            part[threadIdx.x] = make_float2(top, x.y * part_of(x.x, base, p.scale_log2) + y.y * part_of(y.x, base, p.scale_log2));
        }
    }
    if (!p.last)
    {
        if (threadIdx.x >> rows_log2 == 0 && at >= 0) p.kept.state[at] = part[threadIdx.x];
        return;
    }
    float loss = 0.f;
    if (threadIdx.x >> rows_log2 == 0 && at >= 0)  // (what a thread reads it wrote itself)
    {
        const float2 all = part[threadIdx.x];
        const double log = log2((double)all.y);
        loss             = (float)(((double)all.x - (double)own.y) * (double)p.scale + log * kLog2);
        p.kept.state[at] = make_float2(all.x, (float)log);
    }
    if (threadIdx.x >> rows_log2 == 0 && i < p.n && p.reduction == TRIPS_REDUCE_NONE) p.loss[i] = loss;
    if (p.reduction == TRIPS_REDUCE_NONE) return;
    double sum = (double)loss;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (gridDim.x == 1)
            *p.loss = (float)(p.reduction == TRIPS_REDUCE_MEAN ? sum / (double)max(*p.kept.count, 1) : sum);
        else
            p.sums[blockIdx.x] = sum;
    }
}

// The workgroups' sums, in an order that their number alone determines (a launch of its own, 4 to 5 us: the last of join_kernel's workgroups to do it
// would need fences and a counter that is cleared).
__global__ __launch_bounds__(1024) void sum_kernel(const double* from, int n, const int* count, int reduction, float* loss)
{
    __shared__ double sums[16];
    double sum = 0.0;
    for (int b = threadIdx.x; b < n; b += 1024) sum += from[b];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x > 0) return;
    sum = 0.0;
    for (int w = 0; w < 16; ++w) sum += sums[w];
    *loss = (float)(reduction == TRIPS_REDUCE_MEAN ? sum / (double)max(*count, 1) : sum);
}

// What a slab's rows are of: entries (d_table's splits and blocks, which are where they belong), all rows (whose places say which of the slab's they are; zeros
// for those that do not count), or a block of the rows that count, which `row` says the places of; the others are written by a launch of their own then.
enum { ENTRIES, ALL_ROWS, BLOCK_ROWS, OTHER_ROWS };
struct SlabsOut
{
    const float* slabs;
    Kept kept;  // BLOCK_ROWS: the block's
    Upstream upstream;
    void* out;
    long long n, rows_pad, stride;
    int what, first_row, channels, kp, splits;
    float scale;
};
// The splits' sums, in their order; four channels a lane. Bound by memory: 7 parts of 7782 rows of 1024 channels 43 us, 5.4 TB/s.
template <int D>
__global__ __launch_bounds__(256) void slabs_out_kernel(const SlabsOut p)
{
    using E  = Element<D>;
    using T  = typename E::type;
    using F4 = Pack<float, 4>::type;
    using T4 = typename Pack<T, 4>::type;
    const float f       = unheld<D>(p.upstream, p.kept.count) * p.scale;
    const int quads     = (p.channels + 3) >> 2;
    const long long n   = p.what == BLOCK_ROWS ? min(p.n, *p.kept.count - (long long)p.first_row) : p.n;
    const long long all = n * quads, slab = p.rows_pad * p.kp;
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < all; q += (long long)gridDim.x * 256)
    {
        const long long i = q / quads;
        const int c = (int)(q - i * quads) * 4, at = p.what == ALL_ROWS || p.what == OTHER_ROWS ? p.kept.place[i] : (int)i;
        if (p.what == OTHER_ROWS && at >= 0) continue;
        F4 sum = {0.f, 0.f, 0.f, 0.f};
        if (at >= 0)
        {
            const float* from = p.slabs + (long long)at * p.kp + c;
#pragma unroll 4
            for (int s = 0; s < p.splits; ++s) sum += *reinterpret_cast<const F4*>(from + s * slab);
        }
        T* to = reinterpret_cast<T*>(p.out) + (p.what == BLOCK_ROWS ? (long long)p.kept.row[i] : i) * p.stride + c;
        T4 out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = E::from_float(at >= 0 ? sum[e] * f : 0.f);
        if (c + 4 <= p.channels)
            *reinterpret_cast<T4*>(to) = out;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < p.channels) to[e] = out[e];
    }
}

// ---- host ----

constexpr int64_t kPieceBytes = 1ll << 30;  // of d_ij
constexpr int64_t kBlockRows  = 1ll << 20;  // rows that d_ij is held of at once: 256 entries of them are kPieceBytes (in 32 bits, or in two parts)
constexpr int64_t kPartialBytes = 1ll << 30;  // of the maxima and sums of the rows' tiles that are joined at once
constexpr int64_t kSlabBytes  = 256ll << 20;  // of the parts of the rows' gradients
constexpr int kCus            = 256;
constexpr int kMostSplits     = 64;
constexpr int64_t kFewRows    = 64;
constexpr int64_t kCopyBytes = 64ll << 20, kLeastCopyBytes = 16ll << 20;  // of copied entries

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
unsigned tiles_of(int64_t n, int tile) { return (unsigned)((n + tile - 1) / tile); }

// Whether the direct loads take the table's rows as they are: whole words, 256 rows within 31 bits.
bool rows_in_place(const TripsTableLossDesc& d) { return d.table_stride * dtype_bytes(d.dtype) % 4 == 0 && d.table_stride < 1 << 20; }

int packed_channels(const TripsTableLossDesc& d)
{
    const int v = 16 / dtype_bytes(d.dtype);
    return (d.num_channels + v - 1) / v * v;
}

struct Taker
{
    size_t at = 0;
    size_t operator()(size_t bytes)
    {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    }
};

// Where what is kept lies; its size where kept is NULL.
size_t kept_of(const TripsTableLossDesc& d, void* kept, Kept* k)
{
    Taker take;
    char* at = reinterpret_cast<char*>(kept);
    Kept got;
    got.count  = (int*)(at + take(4));
    got.place  = (int*)(at + take(d.num_rows * 4));
    got.row    = (int*)(at + take(d.num_rows * 4));
    got.target = (int*)(at + take(d.num_rows * 4));
    got.state  = (float2*)(at + take(d.num_rows * 8));
    got.packed = at + take((size_t)d.num_rows * packed_channels(d) * dtype_bytes(d.dtype));
    if (k) *k = got;
    return take.at;
}

// Steps of a call over the table; what each takes of the workspace.
struct Layout
{
    int64_t rows_pad, partial_pad, chunks, piece, pieces;
    int kp, tiles, splits, table_splits, parts;
    int at_once;            // pieces whose tiles are joined at once
    int64_t block, blocks;  // backward: rows taken at a time
    bool copies;
    size_t chunk_count, top, partial, own_product, sums, probs, slabs, table_slabs, copy, bytes;
};

// f(a shape): the largest tiles of which a product of `down` x `across` makes one for each CU at least; never the largest in 32 bits, whose
// products take so long that the loads do not count, nor for rows that half of one holds (32 rows of 50,000 entries of 1024 channels:
// gradients with d_ij in two parts 122 us, 98 with Small). Few rows take smaller ones where a tile's products would be of rows that are not there: in
// 32 bits (3 rows of 200,000 entries of 2000 floats, logits 848 us with Small, 388 with Deep, gradients 1451 and 1157 with Tight; 40 of 200,000 of 100,
// gradients 238 and 101), in 16 the logits of up to 32 wide rows (one of 100,000 entries of 4000 channels 165 and 141, of 50,000 of 1024 21.0 and 21.8; 33 rows of
// 60,000 entries of 2000 53 and 73). (With four wavefronts of 128 x 128 the logits of 8191 rows and 50,000 entries of 1024 bfloat16 channels took 1084 us where eight
// take 870, the gradients 1475 and 1434.)
template <typename F>
auto with_shape(const TripsTableLossDesc& d, bool grads, F f)
{
    auto units = [&](int64_t tile)
    {
        const int64_t rows = up(d.num_rows, tile) / tile, entries = up(d.num_entries, tile) / tile, channels = up(d.num_channels, tile) / tile;
        return grads ? channels * entries : rows * entries;
    };
    // (the largest leave no parts of the table's gradient, which blocks of rows are)
    if (d.dtype != TRIPS_DTYPE_F32 && d.num_rows > 128 && units(256) >= kCus && !(grads && d.num_rows > kBlockRows)) return f(Big{});
    const bool wide = d.dtype == TRIPS_DTYPE_F32;
    const bool few  = !grads && d.num_rows <= 32 && (wide || d.num_channels >= 2048);
    if (units(128) >= kCus && !few && (!wide || d.num_rows > 64)) return f(Small{});
    if (grads) return f(Tight{});
    if (few || units(64) < kCus) return f(Deep{});
    return f(Tiny{});
}
// Entries, and rows, of a tile of the logits.
int tile_of_logits(const TripsTableLossDesc& d)
{
    return with_shape(d, false, [](auto shape) { return decltype(shape)::BM; });
}

// Parts that d_ij is held in: two where the tiles are the smallest, or the rows and the table, so that launches and latency take most of the time
// (7 rows of 19 entries of 2696 bfloat16 channels 70 us a pass either way; 3 of 221,303 of 2122 would take 1.24 ms for the gradients and not 0.71).
int parts_of(const TripsTableLossDesc& d)
{
    if (d.dtype == TRIPS_DTYPE_F32) return 1;
    const bool little = d.num_rows <= 128 && d.num_entries * d.num_channels <= 1 << 22;
    return little || with_shape(d, true, [](auto shape) { return decltype(shape)::BM == Tiny::BM; }) ? 2 : 1;
}

// Into how many parts the rows' gradients are cut along the entries, and the table's along the rows where its tiles are few, so that they keep all
// CUs busy to the end, by what a step and a unit's results take, and the parts' way to memory and back. (rows: of a block; in_slabs: entries whose
// gradients' parts are held at once.)
struct Splits
{
    int rows, table;
};
Splits splits_of(const TripsTableLossDesc& d, int64_t rows, int64_t rows_pad, int64_t piece, int64_t in_slabs, int kp)
{
    return with_shape(d, true, [&](auto shape)
    {
        using S = decltype(shape);
        const bool wide       = d.dtype == TRIPS_DTYPE_F32;
        const int step_k      = kStepBytes / dtype_bytes(d.dtype), workers = kCus * S::PER_CU;
        const double step     = (wide ? 4.0 : S::BM == 256 ? 1.6 : 0.8) * (S::BM == 64 ? 0.5 : 1.0);  // microseconds
        const double results  = S::BM == 256 ? 10.0 : S::BM == 128 ? 4.0 : 2.0, slab = (double)rows_pad * kp * 4, table_slab = (double)in_slabs * kp * 4;
        const int64_t channel_tiles = up(d.num_channels, S::BM) / S::BM, units = up(rows, S::BN) / S::BN * channel_tiles, steps = piece / step_k;
        const int64_t table_tiles = up(std::min(piece, d.num_entries), S::BN) / S::BN * channel_tiles, table_steps = up(rows, step_k) / step_k;
        int table    = 1;
        double least = 1e300;
        for (int s = 1; s <= kMostSplits && (s == 1 || (S::BM < Big::BM && table_tiles * (s - 1) < workers && table_steps / s >= 4 && table_slab * s <= (double)kSlabBytes)); ++s)
        {
            // a unit's time, no less than a share of everything; the parts' way to memory and back
            const double unit = (double)((table_steps + s - 1) / s) * step + results;
            const double all  = ((double)(units * steps + table_tiles * table_steps) * step + (double)table_tiles * s * results) / workers;
            const double end  = std::max(unit, all) + (s > 1 ? 3.0 + s * table_slab / 3.5e6 : 0.0);
            if (end < least) table = s, least = end;
        }
        const int64_t table_units = table_tiles * table;
        int best = 1;
        least    = 1e300;
        for (int s = 1; s <= kMostSplits && (s == 1 || (steps / s >= 4 && slab * s <= (double)kSlabBytes)); ++s)
        {
            // the larger units first, each to the first workgroup that is free
            int64_t a = units * s, b = table_units;
            double size_a = (double)((steps + s - 1) / s) * step + results, size_b = (double)((table_steps + table - 1) / table) * step + results;
            if (size_a < size_b) std::swap(a, b), std::swap(size_a, size_b);
            const int64_t rest = a % workers;
            const double full  = (double)(a / workers) * size_a;
            double end         = full + (rest ? size_a : 0.0);
            // (the least number of rounds of b by whose end all of it is done, which is found by doubling and halving: what is done grows with the rounds)
            auto enough = [&](int64_t k)
            {
                const double late = (double)k * size_b - size_a;
                return (workers - rest) * k + (rest && late > 0 ? rest * (int64_t)(late / size_b) : 0) >= b;
            };
            int64_t low = b / workers, high = low;
            for (int64_t by = 1; !enough(high); by *= 2) low = high + 1, high += by;
            while (low < high)
            {
                const int64_t k = (low + high) / 2;
                if (enough(k)) high = k; else low = k + 1;
            }
            end = std::max(end, full + (double)low * size_b);
            end += s * slab / 3.5e6;
            if (end < least) best = s, least = end;
        }
        return Splits{best, table};
    });
}

// copies: the table's entries are copied, a piece at a time, before the products read them.
Layout layout_of(const TripsTableLossDesc& d, bool backward, bool copies)
{
    Layout l{};
    const int size = dtype_bytes(d.dtype);
    l.rows_pad = up(d.num_rows, 256), l.chunks = d.num_rows > kCountedBy ? up(d.num_rows, kChunk) / kChunk : 0;
    l.kp     = packed_channels(d);
    l.copies = copies;
    l.parts  = parts_of(d);
    if (backward)
    {
        l.blocks   = std::max<int64_t>(1, (d.num_rows + kBlockRows - 1) / kBlockRows);
        l.block    = l.blocks > 1 ? up((d.num_rows + l.blocks - 1) / l.blocks, 256) : d.num_rows;
        l.rows_pad = up(l.block, 256);
    }
    Taker take;
    const int64_t grain = d.num_entries < 256 ? std::max(tile_of_logits(d), 64) : 256;  // (whole tiles of the logits, whole steps of the gradients; few entries are not padded to more)
    int64_t most        = up(std::max<int64_t>(d.num_entries, 1), grain);
    if (copies)
    {
        most   = std::min(most, std::max<int64_t>((rows_in_place(d) ? kLeastCopyBytes : kCopyBytes) / (l.kp * size) / 256, 1) * 256);
        l.copy = take((size_t)most * l.kp * size);
    }
    if (!backward)
    {
        const int64_t tile = tile_of_logits(d), tiles = kPartialBytes / (std::max<int64_t>(up(d.num_rows, tile), 1) * (int64_t)sizeof(float2));
        most               = std::min(most, std::max<int64_t>(tiles * tile / 256, 1) * 256);
    }
    if (backward) most = std::min(most, std::max<int64_t>(kPieceBytes / (std::max<int64_t>(l.rows_pad, 1) * size * l.parts) / 256, 1) * 256);
    l.pieces = std::max<int64_t>(1, (d.num_entries + most - 1) / most);
    l.piece  = up((d.num_entries + l.pieces - 1) / l.pieces, grain);
    if (!backward)
    {
        l.chunk_count = take((l.chunks + 1) * 4);
        l.tiles       = (int)(l.piece / tile_of_logits(d));
        l.partial_pad = up(d.num_rows, tile_of_logits(d));
        l.at_once     = (int)std::min(l.pieces, std::max<int64_t>(1, kPartialBytes / (std::max<int64_t>(l.partial_pad * l.tiles, 1) * (int64_t)sizeof(float2))));
        l.partial     = take((size_t)l.tiles * l.at_once * l.partial_pad * sizeof(float2));
        l.own_product = take(l.rows_pad * 4);
        l.sums        = take((std::max(d.num_rows / 4, kFewRows) + 1) * 8);
    }
    else
    {
        l.top   = take((1 + kTops) * 4);
        l.probs = take((size_t)l.parts * l.rows_pad * l.piece * size);
        const int64_t in_slabs = l.blocks > 1 ? l.pieces * l.piece : l.piece;  // (of several blocks the whole table's)
        const Splits s         = splits_of(d, l.block, l.rows_pad, l.piece, in_slabs, l.kp);
        l.splits = s.rows, l.table_splits = s.table;
        l.slabs = take((size_t)l.splits * l.rows_pad * l.kp * 4);
        if (l.table_splits > 1 || l.blocks > 1) l.table_slabs = take((size_t)l.table_splits * in_slabs * l.kp * 4);
    }
    l.bytes = take.at;
    return l;
}

bool copies_of(const TripsTableLossDesc& d, const void* table) { return !(rows_in_place(d) && aligned(table, 4)); }

// For any address of the table.
size_t workspace_of(const TripsTableLossDesc& d, bool backward)
{
    const size_t copied = layout_of(d, backward, true).bytes;
    return copies_of(d, nullptr) ? copied : std::max(copied, layout_of(d, backward, false).bytes);
}

// (not 0: 0 times minus infinity, which stands for entries that are not there, is no number. The smallest number there is: times the distance of two of the
// largest, where entries are masked with the lowest value, it is 2^-20.)
float scale_log2(const TripsTableLossDesc& d) { return std::max((float)(std::fabs((double)d.scale) * kLog2e), std::numeric_limits<float>::denorm_min()); }

template <int D>
hipError_t gather(const TripsTableLossDesc& d, const Layout& l, const void* rows, const void* target, const Kept& kept, char* w, hipStream_t stream, Profiler* prof)
{
    GatherParams p{};
    p.rows = rows, p.target = target, p.kept = kept;
    p.n = d.num_rows, p.entries = d.num_entries, p.stride = d.rows_stride;
    p.channels = d.num_channels, p.kp = l.kp, p.negate = d.scale < 0.f;
    const bool i32 = d.index_dtype == TRIPS_INDEX_I32;
    if (l.chunks)
    {
        int* chunk_count = (int*)(w + l.chunk_count);
        p.chunk_count    = chunk_count;
        ProfScope scope(prof, "loss_count", stream);
        (i32 ? count_kernel<true> : count_kernel<false>)<<<(unsigned)l.chunks, 256, 0, stream>>>(target, d.num_rows, d.num_entries, chunk_count);
        if (hipError_t e = hipGetLastError()) return e;
        p.scanned = d.num_rows > kScannedBy;
        if (p.scanned)
        {
            ProfScope scope(prof, "loss_scan", stream);
            scan_kernel<<<1, 1024, 0, stream>>>(chunk_count, l.chunks);
            if (hipError_t e = hipGetLastError()) return e;
        }
    }
    ProfScope scope(prof, "loss_gather", stream);
    const unsigned groups = std::max(1u, (unsigned)((d.num_rows + kGatherRows - 1) / kGatherRows));
    const int64_t rounds  = ((int64_t)kGatherRows * l.kp * dtype_bytes(d.dtype) / 16 + kAhead * 256 - 1) / (kAhead * 256);
    const unsigned along  = (unsigned)std::max<int64_t>(1, std::min<int64_t>(rounds, 2 * kCus / groups));  // (1000 rows of 4000 floats 26 us with one workgroup a group of rows, 9 so)
    (i32 ? gather_kernel<D, true> : gather_kernel<D, false>)<<<dim3(groups, along), 256, 0, stream>>>(p);
    return hipGetLastError();
}

ProductParams product_params(const TripsTableLossDesc& d, const Layout& l, const Kept& kept, char* w)
{
    ProductParams p{};
    p.kept = kept;
    p.partial = (float2*)(w + l.partial), p.own_product = (float*)(w + l.own_product), p.probs = w + l.probs, p.slabs = (float*)(w + l.slabs), p.table_slabs = (float*)(w + l.table_slabs);
    p.d_table_stride = d.d_table_stride, p.rows_pad = l.rows_pad, p.partial_pad = l.partial_pad;
    p.channels = d.num_channels, p.kp = l.kp, p.piece = (int)l.piece, p.splits = l.splits, p.table_splits = l.table_splits, p.parts = l.parts;
    p.most_rows = 0x7fffffff, p.in_table_slabs = l.table_splits > 1 || l.blocks > 1;
    p.scale_log2 = scale_log2(d);
    return p;
}

// The entries of piece `piece` as the products read them.
template <int D>
hipError_t take_piece(const TripsTableLossDesc& d, const Layout& l, int64_t piece, const void* table, void* d_table, char* w, ProductParams& p, hipStream_t stream, Profiler* prof)
{
    using T          = typename Element<D>::type;
    const T* entries = reinterpret_cast<const T*>(table) + piece * l.piece * d.table_stride;
    p.first_entry = (int)(piece * l.piece), p.in_piece = (int)std::min(l.piece, d.num_entries - piece * l.piece);
    p.first_tile = l.at_once ? (int)(piece % l.at_once * l.tiles) : 0, p.add = piece > 0;
    p.table = entries, p.table_stride = d.table_stride, p.held = d.num_channels;
    p.d_table = d_table ? reinterpret_cast<T*>(d_table) + piece * l.piece * d.d_table_stride : nullptr;
    if (!l.copies) return hipSuccess;
    p.table = w + l.copy, p.table_stride = p.held = l.kp;
    ProfScope scope(prof, "loss_copy", stream);
    const int64_t pieces = (int64_t)p.in_piece * l.kp * (int64_t)sizeof(T) / 16;
    copy_entries_kernel<T><<<(unsigned)std::min<int64_t>((pieces + 255) / 256, 1 << 16), 256, 0, stream>>>(entries, d.table_stride, reinterpret_cast<T*>(w + l.copy), p.in_piece,
                                                                                                          d.num_channels, l.kp);
    return hipGetLastError();
}

template <int D, int KIND>
hipError_t launch_product(const TripsTableLossDesc& d, const ProductParams& p, hipStream_t stream, Profiler* prof)
{
    return with_shape(d, KIND == GRADS, [&](auto shape)
    {
        using Given = decltype(shape);
        // (no code for what with_shape() does not give)
        using S = std::conditional_t<D == TRIPS_DTYPE_F32 && Given::BM == 256, Small, std::conditional_t<KIND == GRADS && Given::BM <= Tiny::BM, Tight, std::conditional_t<KIND != GRADS && std::is_same<Given, Tight>::value, Tiny, Given>>>;
        const int64_t row_tiles = tiles_of(d.num_rows, S::BN), channel_tiles = tiles_of(d.num_channels, S::BM);
        const int64_t units = KIND == GRADS ? channel_tiles * ((p.d_rows ? row_tiles * p.splits : 0) + (p.d_table ? tiles_of(p.in_piece, S::BN) * p.table_splits : 0)) : tiles_of(p.in_piece, S::BM) * row_tiles;
        if (units == 0) return hipSuccess;
        ProfScope scope(prof, KIND == LOGITS ? "loss_logits" : KIND == PROBS ? "loss_probs" : "loss_grads", stream);
        product_kernel<D, KIND, S><<<(unsigned)std::min<int64_t>(units, S::PER_CU * kCus), S::WAVES * 64, 0, stream>>>(p);
        return hipGetLastError();
    });
}

template <int D>
hipError_t forward(const TripsTableLossDesc& d, const void* rows, const void* table, const void* target, float* loss, const Kept& kept, char* w, hipStream_t stream, Profiler* prof)
{
    const Layout l = layout_of(d, false, copies_of(d, table));
    if (hipError_t e = gather<D>(d, l, rows, target, kept, w, stream, prof)) return e;
    ProductParams p = product_params(d, l, kept, w);
    JoinParams j{};
    j.partial = p.partial, j.own_product = p.own_product, j.kept = kept;
    j.loss = loss, j.scale = std::fabs(d.scale), j.scale_log2 = p.scale_log2, j.sums = (double*)(w + l.sums);
    j.n = d.num_rows, j.partial_pad = l.partial_pad, j.reduction = d.reduction;
    int64_t groups = 1;
    for (int64_t piece = 0; !j.last;)
    {
        const int64_t first = piece * l.piece;
        for (int k = 0; k < l.at_once && piece * l.piece < d.num_entries; ++k, ++piece)
        {
            if (hipError_t e = take_piece<D>(d, l, piece, table, nullptr, w, p, stream, prof)) return e;
            if (hipError_t e = launch_product<D, LOGITS>(d, p, stream, prof)) return e;
        }
        j.tiles = (int)tiles_of(std::min(piece * l.piece, d.num_entries) - first, tile_of_logits(d));
        j.more = first > 0, j.last = piece * l.piece >= d.num_entries;
        j.lanes_log2 = 0;
        while (j.lanes_log2 < 6 && 8 << j.lanes_log2 < j.tiles) ++j.lanes_log2;
        // (the rows of few in one workgroup, whose sum is the loss then, or of very many tiles in one each)
        if (d.num_rows <= kFewRows && j.tiles > 2048)
            while (j.lanes_log2 < 8 && 16 << j.lanes_log2 < j.tiles) ++j.lanes_log2;
        else
            while (j.lanes_log2 > 2 && d.num_rows > 256 >> j.lanes_log2 && d.num_rows <= kFewRows) --j.lanes_log2;
        const int64_t rows_each = 256 >> j.lanes_log2;  // (a launch's threads stay below 2^32: rows of many tiles are few, see kPartialBytes)
        groups                  = std::max<int64_t>(1, (d.num_rows + rows_each - 1) / rows_each);
        ProfScope scope(prof, "loss_join", stream);
        join_kernel<<<(unsigned)groups, 256, 0, stream>>>(j);
        if (hipError_t e = hipGetLastError()) return e;
    }
    if (d.reduction == TRIPS_REDUCE_NONE || groups == 1) return hipSuccess;
    ProfScope scope(prof, "loss_sum", stream);
    sum_kernel<<<1, 1024, 0, stream>>>(j.sums, (int)groups, kept.count, d.reduction, loss);
    return hipGetLastError();
}

template <int D>
hipError_t slabs_out(const char* name, const SlabsOut& p, hipStream_t stream, Profiler* prof)
{
    ProfScope scope(prof, name, stream);
    slabs_out_kernel<D><<<(unsigned)std::min<int64_t>((p.n * ((p.channels + 3) / 4) + 255) / 256, 1 << 16), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <int D>
hipError_t backward(const TripsTableLossDesc& d, const void* table, const Kept& kept, const float* d_loss, void* d_rows, void* d_table, char* w, hipStream_t stream, Profiler* prof)
{
    const Layout l  = layout_of(d, true, copies_of(d, table));
    ProductParams p = product_params(d, l, kept, w);
    p.d_rows        = d_rows;
    p.upstream      = Upstream{d_loss, (float*)(w + l.top), d.reduction, d.scale};
    if (D == TRIPS_DTYPE_F16 && d.reduction == TRIPS_REDUCE_NONE && d.num_rows > 0)
    {
        ProfScope scope(prof, "loss_top", stream);
        float* top       = (float*)(w + l.top);
        const int groups = d.num_rows > kTopBy ? (int)std::min<int64_t>((d.num_rows + 8191) / 8192, kTops) : 1;
        top_kernel<true><<<groups, 1024, 0, stream>>>(d_loss, kept.place, d.num_rows, groups > 1 ? top + 1 : top);
        if (hipError_t e = hipGetLastError()) return e;
        if (groups > 1)
        {
            top_kernel<false><<<1, 1024, 0, stream>>>(top + 1, nullptr, groups, top);
            if (hipError_t e = hipGetLastError()) return e;
        }
    }
    SlabsOut entries{}, out{};
    entries.kept = kept, entries.upstream = p.upstream, entries.rows_pad = l.piece, entries.stride = d.d_table_stride, entries.what = ENTRIES;
    entries.channels = d.num_channels, entries.kp = l.kp, entries.splits = l.table_splits, entries.scale = std::fabs(d.scale);
    out          = entries;
    out.slabs = p.slabs, out.out = d_rows, out.n = d.num_rows, out.rows_pad = l.rows_pad, out.stride = d.d_rows_stride, out.splits = l.splits, out.scale = d.scale;
    const bool rows_out = d_rows && d.num_rows > 0;
    if (l.blocks > 1 && rows_out)
    {
        out.what = OTHER_ROWS;
        if (hipError_t e = slabs_out<D>("loss_rows_out", out, stream, prof)) return e;
    }
    for (int64_t block = 0; block < l.blocks; ++block)
    {
        const int64_t first = block * l.block;
        p.first_row = (int)first, p.most_rows = (int)l.block, p.add_to_table = block > 0;
        p.kept.row = kept.row + first, p.kept.target = kept.target + first, p.kept.state = kept.state + first;
        p.kept.packed = reinterpret_cast<char*>(kept.packed) + first * l.kp * dtype_bytes(d.dtype);
        for (int64_t piece = 0; piece * l.piece < d.num_entries; ++piece)
        {
            if (hipError_t e = take_piece<D>(d, l, piece, table, d_table, w, p, stream, prof)) return e;
            p.table_slabs = (float*)(w + l.table_slabs) + (l.blocks > 1 ? piece * l.table_splits * l.piece * l.kp : 0);
            if (hipError_t e = launch_product<D, PROBS>(d, p, stream, prof)) return e;
            if (hipError_t e = launch_product<D, GRADS>(d, p, stream, prof)) return e;
            if (!d_table || !p.in_table_slabs || block + 1 < l.blocks) continue;
            entries.slabs = p.table_slabs, entries.out = p.d_table, entries.n = p.in_piece;
            if (hipError_t e = slabs_out<D>("loss_table_out", entries, stream, prof)) return e;
        }
        if (!rows_out) continue;
        if (l.blocks > 1) out.what = BLOCK_ROWS, out.kept = p.kept, out.first_row = p.first_row, out.n = l.block;
        else out.what = ALL_ROWS;
        if (hipError_t e = slabs_out<D>("loss_rows_out", out, stream, prof)) return e;
    }
    return hipSuccess;
}

int check_stride(const char* name, int64_t stride, int64_t row, int64_t rows, bool written)
{
    if (stride < 0 || stride > ((int64_t)1 << 40) || (written && rows > 1 && stride < row))
        return set_error(TRIPS_ERR_INVALID_ARG, "%s %lld (rows have %lld elements)", name, (long long)stride, (long long)row);
    return TRIPS_OK;
}

// A launch's units are numbered in 31 bits.
int check_units(const TripsTableLossDesc& d)
{
    for (int grads = 0; grads < 2; ++grads)
    {
        const double units = with_shape(d, grads, [&](auto shape)
        {
            using S = decltype(shape);
            const double rows = (double)(up(grads ? std::min(d.num_rows, kBlockRows) : d.num_rows, S::BN) / S::BN), entries = (double)(up(d.num_entries, S::BN) / S::BN), channels = (double)(up(d.num_channels, S::BM) / S::BM);
            return grads ? channels * (rows * kMostSplits + entries) + kCus * S::PER_CU : rows * entries;  // (see splits_of())
        });
        if (units >= 2147000000.0) return set_error(TRIPS_ERR_UNSUPPORTED, "%lld rows and %lld entries are too many for one call", (long long)d.num_rows, (long long)d.num_entries);
    }
    return TRIPS_OK;
}

int check_desc(const TripsTableLossDesc* d)
{
    if (!d) return set_error(TRIPS_ERR_INVALID_ARG, "desc is NULL");
    if (d->abi_version != TRIPS_ABI_VERSION) return set_error(TRIPS_ERR_INVALID_ARG, "abi_version %d, library is %d", d->abi_version, TRIPS_ABI_VERSION);
    if (!dtype_ok(d->dtype)) return set_error(TRIPS_ERR_UNSUPPORTED, "dtype %d", d->dtype);
    if (d->index_dtype != TRIPS_INDEX_I64 && d->index_dtype != TRIPS_INDEX_I32) return set_error(TRIPS_ERR_UNSUPPORTED, "index_dtype %d", d->index_dtype);
    if (d->reduction != TRIPS_REDUCE_NONE && d->reduction != TRIPS_REDUCE_SUM && d->reduction != TRIPS_REDUCE_MEAN) return set_error(TRIPS_ERR_INVALID_ARG, "reduction %d", d->reduction);
    if (d->num_rows < 0 || d->num_rows > kMostRows) return set_error(TRIPS_ERR_INVALID_ARG, "num_rows = %lld", (long long)d->num_rows);
    if (d->num_entries < 0 || d->num_entries >= kMostEntries) return set_error(TRIPS_ERR_INVALID_ARG, "num_entries = %lld", (long long)d->num_entries);
    if (d->num_channels < 1 || d->num_channels >= kMostChannels) return set_error(TRIPS_ERR_INVALID_ARG, "num_channels = %d", d->num_channels);
    if (!(std::fabs((double)d->scale) * kLog2e <= (double)std::numeric_limits<float>::max())) return set_error(TRIPS_ERR_INVALID_ARG, "scale = %g", (double)d->scale);
    if (int e = check_stride("rows_stride", d->rows_stride, d->num_channels, d->num_rows, false)) return e;
    if (int e = check_stride("table_stride", d->table_stride, d->num_channels, d->num_entries, false)) return e;
    return check_units(*d);
}

int check_pointer(const char* name, const void* p, size_t align, bool needed)
{
    if ((!p && needed) || !aligned(p, align)) return set_error(TRIPS_ERR_INVALID_ARG, "%s is NULL or not aligned", name);
    return TRIPS_OK;
}

int check_call(TripsCtx* ctx, const TripsTableLossDesc* d, bool backward, const void* table, const void* kept, size_t kept_bytes, const void* workspace, size_t bytes)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (int e = check_desc(d)) return e;
    if (int e = check_pointer("table", table, dtype_bytes(d->dtype), d->num_entries > 0)) return e;
    if (!kept || !aligned(kept, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "kept must be a 256-byte aligned device pointer");
    if (kept_bytes < kept_of(*d, nullptr, nullptr)) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "kept has %zu bytes, %zu needed", kept_bytes, kept_of(*d, nullptr, nullptr));
    if (!workspace || !aligned(workspace, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
    const size_t need = workspace_of(*d, backward);
    if (bytes < need) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %zu needed", bytes, need);
    return TRIPS_OK;
}

template <typename F>
int with_dtype(int dtype, F f)
{
    if (dtype == TRIPS_DTYPE_F32) return f(std::integral_constant<int, TRIPS_DTYPE_F32>{});
    return dtype == TRIPS_DTYPE_BF16 ? f(std::integral_constant<int, TRIPS_DTYPE_BF16>{}) : f(std::integral_constant<int, TRIPS_DTYPE_F16>{});
}
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" {

int trips_table_loss_kept_size(const TripsTableLossDesc* desc, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (int e = check_desc(desc)) return e;
    *bytes = kept_of(*desc, nullptr, nullptr);
    return TRIPS_OK;
}

int trips_table_loss_workspace_size(const TripsTableLossDesc* desc, int backward, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (int e = check_desc(desc)) return e;
    *bytes = workspace_of(*desc, backward != 0);
    return TRIPS_OK;
}

int trips_table_loss_forward(TripsCtx* ctx, const TripsTableLossDesc* desc, const void* rows, const void* table, const void* target, float* loss,
                             void* kept, size_t kept_bytes, void* workspace, size_t workspace_bytes, void* stream)
{
    if (int e = check_call(ctx, desc, false, table, kept, kept_bytes, workspace, workspace_bytes)) return e;
    if (int e = check_pointer("rows", rows, dtype_bytes(desc->dtype), desc->num_rows > 0)) return e;
    if (int e = check_pointer("target", target, desc->index_dtype == TRIPS_INDEX_I32 ? 4 : 8, desc->num_rows > 0)) return e;
    if (int e = check_pointer("loss", loss, 4, desc->num_rows > 0 || desc->reduction != TRIPS_REDUCE_NONE)) return e;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    Kept k;
    kept_of(*desc, kept, &k);
    return with_dtype(desc->dtype, [&](auto dtype)
    {
        const hipError_t e = forward<decltype(dtype)::value>(*desc, rows, table, target, loss, k, (char*)workspace, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
        return e == hipSuccess ? (int)TRIPS_OK : hip_error(e, "table loss launch");
    });
}

int trips_table_loss_backward(TripsCtx* ctx, const TripsTableLossDesc* desc, const void* table, const void* kept, size_t kept_bytes, const float* d_loss,
                              void* d_rows, void* d_table, void* workspace, size_t workspace_bytes, void* stream)
{
    if (int e = check_call(ctx, desc, true, table, kept, kept_bytes, workspace, workspace_bytes)) return e;
    const size_t size = dtype_bytes(desc->dtype);
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
    Kept k;
    kept_of(*desc, const_cast<void*>(kept), &k);  // (only read here)
    return with_dtype(desc->dtype, [&](auto dtype)
    {
        const hipError_t e = backward<decltype(dtype)::value>(*desc, table, k, d_loss, d_rows, d_table, (char*)workspace, reinterpret_cast<hipStream_t>(stream), profiler(ctx));
        return e == hipSuccess ? (int)TRIPS_OK : hip_error(e, "table loss launch");
    });
}

}  // extern "C"
