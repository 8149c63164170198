// AdamW over many tensors in one launch, moments in 32 or 8 bits, and the global norm of their gradients (gfx950).
//
// Both are bound by memory: a step reads and writes each element of weights and moments once and reads each gradient once
// (28 bytes an element in 32 bits, 16 with moments in 8), the norm reads the gradients. 60M elements: 300 us in 32 bits (5.6 TB/s;
// a large copy 5.2 to 6.2), 166 in 8 (5.8), the norm 38 (6.3). A step is two launches: one workgroup counts the steps, takes the
// tensors' rates in double and lays out the table that the step's workgroups search; the norm is one more, its sums being joined in
// that workgroup. Small calls are those launches, 4 to 5 us each.
#include <float.h>

#include <algorithm>
#include <cmath>

#include "abi_common.h"
#include "row16.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int kTensors     = 40;   // tensors of a table in the kernel's arguments (4 KB)
constexpr int kGroups      = 8;    // different sets of options among them
constexpr int kStepTensors = 4096; // tensors of a step's launch
constexpr int kTileOptim   = 1024; // elements of a tile: four wavefronts with a block of 256 each
constexpr int kStepGroups  = 2048; // workgroups of a step with a tile each
constexpr int kStepRun     = 2;    // tiles of a workgroup, one behind the other, where there are more tiles: moments in 8 bits gain by it
                                   // (us a step with 1 and 2: 3000 tiles 16.0, 15.4; 8000 29.4, 28.3; 24,000 75.5, 73.7; 60M elements 181,
                                   // 169, with 4 178, 8 188, 2048 workgroups in turn 194), in 32 bits only the largest steps do (8000 tiles
                                   // 41.7, 46.1; 24,000 124, 130; 40,000 203, 199; 60M elements 297 to 305, in turn 331)
constexpr int kNormTensors = 140; // of a launch: 4 KB of arguments
constexpr int kNormTile    = 2048; // elements of a tile of the norm
constexpr int kNormGroups  = 1024; // workgroups of the norm = partial sums
static_assert(TRIPS_MOMENT_BLOCK == 256, "a block is four elements a lane");
static_assert(kNormGroups * sizeof(double) <= TRIPS_GRAD_NORM_WORKSPACE_BYTES, "workspace");

// A tensor as the step's kernel reads it, made by the kernel before it from what the host knows (StepTensor) and the step count
// on the device. (In the step's own arguments, searched by every workgroup entry by entry, the table cost more than the work
// of a small call: the benchmark's net 10 us, 40 tensors 39.)
struct StepEntry
{
    void* w;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    void* copy;
    long long n;
    double b1, c1, b2, c2;        // beta and 1 - beta
    float fb1, fc1, fb2, fc2;     // the same in float
    float keep, rate, root, eps;  // 1 - lr decay, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
    uint32_t key;                 // of the rounding
    uint32_t first_block;         // of the call, in blocks of 256 elements
    uint32_t copy_dtype, unused;
};

struct StepTensor
{
    void* w;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    void* copy;
    int32_t* step;
    long long n;
    uint32_t first_tile;  // of the step's launch
    uint32_t first_block;
    uint8_t group, copy_dtype;
};
struct StepOptions
{
    double lr, beta1, beta2, eps, decay;
};
struct StepTable
{
    StepTensor t[kTensors];
    StepOptions o[kGroups];
    uint32_t n, seed;
    float* norm;           // {norm, factor} or NULL
    const double* sums;    // squares to make the norm of first, or NULL
    uint32_t groups;       // how many
    float max_norm, loss_scale;
    StepEntry* entries;
    uint32_t* first_tiles;
};
static_assert(sizeof(StepTable) <= 4096, "kernel arguments");

struct StepParams
{
    const StepEntry* entries;
    const uint32_t* first_tiles;
    uint32_t n, tiles, run;  // run: tiles of a workgroup, one behind the other
    const float* norm;
    float factor;  // where there is no `norm`
};

// beta^t by squaring, in double
__device__ __forceinline__ double power(double beta, uint32_t t)
{
    double r = 1.0;
    while (t)
    {
        if (t & 1u) r *= beta;
        beta *= beta;
        t >>= 1;
    }
    return r;
}

// 32 well-mixed bits of 32
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x9E3779B9u;
    x ^= x >> 15;
    x *= 0xB504F333u;
    x ^= x >> 16;
    return x;
}

// Of all lanes, the same for all.
__device__ __forceinline__ uint32_t wave_max(uint32_t x)
{
    x = max(x, (uint32_t)dpp_i<kDppXor1>((int)x));
    x = max(x, (uint32_t)dpp_i<kDppXor2>((int)x));
    x = max(x, (uint32_t)dpp_i<kDppHalfMirror>((int)x));
    x = max(x, (uint32_t)dpp_i<kDppMirror>((int)x));
    auto of = [&](int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); };
    return max(max(of(0), of(16)), max(of(32), of(48)));
}

// The high word of |x|, one more where the low word holds something: compares like |x| against numbers of 20 mantissa bits.
__device__ __forceinline__ uint32_t high_word_up(double x)
{
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return ((uint32_t)(u >> 32) & 0x7fffffffu) + ((uint32_t)u != 0u ? 1u : 0u);
}

// Smallest k in [-118, 111] with top <= 0.875 2^(9 + k) (448 and 57344 are 0.875 times a power of two); `top` as high_word_up
// gives it, LARGEST_EXPONENT = 9 or 16.
template <int LARGEST_EXPONENT>
__device__ __forceinline__ int scale_exponent(uint32_t top)
{
    const int e = (int)(top >> 20) - 1022;  // top = f 2^e, f in [0.5, 1)
    const int k = e - LARGEST_EXPONENT + ((top & 0xfffffu) > 0xc0000u ? 1 : 0);
    return min(max(k, -118), 111);
}

// |x| 2^-k as a code of an 8-bit float with MANTISSA bits and exponent bias BIAS: floor(y / q + (r + 0.5) / 65536) steps q,
// at most MOST; `hi`: the high word of |x|, finite. The bits of a double are such a code, followed by 52 - MANTISSA more and with
// another bias; the steps are added to those of the high word, whose carry is the rounding (what the low word holds can make no
// carry: the addend is a multiple of the high word's last place). Below the lowest normal number steps stay as they are: the
// significand shifts right instead.
template <int MANTISSA, int BIAS, int MOST>
__device__ __forceinline__ uint32_t encode(uint32_t hi, int k, uint32_t r)
{
    const int t        = (int)hi - (k + 1023 - BIAS) * (1 << 20);
    const int e        = t >> 20;
    const uint32_t sig = 0x100000u | (hi & 0xfffffu);
    const uint32_t y   = e >= 1 ? (uint32_t)t : sig >> min(1 - e, 31);
    constexpr int DROP = 20 - MANTISSA;
    return min((y + ((2u * r + 1u) << (DROP - 17))) >> DROP, (uint32_t)MOST);
}

// The new weight. Root and reciprocal are the instructions' own (off by one place each); a root of v below the normal numbers
// counts as 0, which is nothing beside an eps of 2^-40 or more. Below that they are taken exactly.
constexpr float kLeastEps = 0x1p-40f;
template <bool EXACT>
__device__ __forceinline__ float stepped(Constant<StepEntry> r, float w, float m, float v)
{
    if constexpr (EXACT) return fmaf(-r->rate, m / fmaf(sqrtf(v), r->root, r->eps), r->keep * w);
    const float down = __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(v), r->root, r->eps));
    return fmaf(-r->rate * m, down, r->keep * w);
}

typedef uint32_t Codes __attribute__((aligned(1)));  // four codes of 8 bits

template <typename T>
__device__ __forceinline__ void load4(Global<const T> from, bool whole, int count, T (&x)[4])
{
    if (whole)
    {
        const auto q = __builtin_nontemporal_load((Global<const typename Pack<T, 4>::type>)from);
        x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < count ? from[i] : T(0);
    }
}
template <typename T>
__device__ __forceinline__ void store4(Global<T> to, bool whole, int count, const T (&x)[4])
{
    if (whole)
    {
        typename Pack<T, 4>::type q = {x[0], x[1], x[2], x[3]};
        __builtin_nontemporal_store(q, (Global<typename Pack<T, 4>::type>)to);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) to[i] = x[i];
    }
}

template <int WD>
__device__ __forceinline__ void store_weights(Constant<StepEntry> T, long long i0, bool whole, int count, const float (&nw)[4])
{
    using W = typename Element<WD>::type;
    W w4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w4[i] = Element<WD>::from_float(nw[i]);
    store4(global(reinterpret_cast<W*>(T->w)) + i0, whole, count, w4);
    if (!T->copy) return;
    if (T->copy_dtype == TRIPS_DTYPE_F32)
        store4(global(reinterpret_cast<float*>(T->copy)) + i0, whole, count, nw);
    else
    {
        const bool bf = T->copy_dtype == TRIPS_DTYPE_BF16;
        unsigned short c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = bf ? Element<TRIPS_DTYPE_BF16>::from_float(nw[i]) : Element<TRIPS_DTYPE_F16>::from_float(nw[i]);
        store4(global(reinterpret_cast<unsigned short*>(T->copy)) + i0, whole, count, c);
    }
}

// Four elements a lane, a block of 256 a wavefront. Returns whether it was done: not where the block is one for step_any.
template <int WD, int GD, int BITS>
__device__ __forceinline__ bool step_whole(Constant<StepEntry> T, float factor, long long block, int lane)
{
    using W = typename Element<WD>::type;
    using G = typename Element<GD>::type;
    const long long i0 = block * TRIPS_MOMENT_BLOCK + lane * 4;
    W w4[4];
    G g4[4];
    load4(global(reinterpret_cast<const G*>(T->g)) + i0, true, 4, g4);
    load4(global(reinterpret_cast<const W*>(T->w)) + i0, true, 4, w4);
    float nw[4];
    if constexpr (BITS == 32)
    {
        float m[4], v[4];
        const auto mo = global(reinterpret_cast<float*>(T->m)) + i0;
        const auto vo = global(reinterpret_cast<float*>(T->v)) + i0;
        load4(mo, true, 4, m);
        load4(vo, true, 4, v);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float g = Element<GD>::to_float(g4[i]) * factor;
            m[i]  = fmaf(T->fc1, g, T->fb1 * m[i]);
            v[i]  = fmaf(T->fc2 * g, g, T->fb2 * v[i]);
            nw[i] = stepped<false>(T, Element<WD>::to_float(w4[i]), m[i], v[i]);
        }
        store4(mo, true, 4, m);
        store4(vo, true, 4, v);
    }
    else
    {
        // The new moments in double: which code they get must not depend on roundings on the way.
        const auto mo = (Global<Codes>)(global(reinterpret_cast<unsigned char*>(T->m)) + i0);
        const auto vo = (Global<Codes>)(global(reinterpret_cast<unsigned char*>(T->v)) + i0);
        const int mw = (int)__builtin_nontemporal_load(mo), vw = (int)__builtin_nontemporal_load(vo);
        const double bm = T->b1 * (double)((Constant<float>)T->ms)[block], bv = T->b2 * (double)((Constant<float>)T->vs)[block];
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(mw, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(mw, true);
        const auto v01 = __builtin_amdgcn_cvt_pk_f32_bf8(vw, false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8(vw, true);
        const float mf[4] = {m01[0], m01[1], m23[0], m23[1]}, vf[4] = {v01[0], v01[1], v23[0], v23[1]};
        uint32_t mh[4], vh[4], mtop = 0, vtop = 0;  // the high words of the moments
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const double g = (double)Element<GD>::to_float(g4[i]) * (double)factor;
            const double m = fma(T->c1, g, bm * (double)mf[i]);
            const double v = fma(T->c2 * g, g, bv * (double)vf[i]);
            nw[i] = stepped<false>(T, Element<WD>::to_float(w4[i]), (float)m, (float)v);
            mh[i] = (uint32_t)((unsigned long long)__double_as_longlong(m) >> 32);
            vh[i] = (uint32_t)((unsigned long long)__double_as_longlong(v) >> 32);
            mtop  = max(mtop, mh[i] & 0x7fffffffu);
            vtop  = max(vtop, vh[i]);
        }
        mtop = wave_max(mtop), vtop = wave_max(vtop);
        // not finite (or a negative v), or a largest number so near the border of two scales that the low words decide
        if (mtop >= 0x7ff00000u || vtop >= 0x7ff00000u || (mtop & 0xfffffu) == 0xc0000u || (vtop & 0xfffffu) == 0xc0000u) return false;
        const int km = scale_exponent<9>(mtop), kv = scale_exponent<16>(vtop);
        const uint32_t at = (T->first_block + (uint32_t)block) * TRIPS_MOMENT_BLOCK + (uint32_t)lane * 4u;
        uint32_t mc = 0, vc = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const uint32_t bits = mix((at + i) ^ T->key);
            mc |= (encode<3, 7, 0x7e>(mh[i] & 0x7fffffffu, km, bits & 0xffffu) | (mh[i] >> 24 & 0x80u)) << (8 * i);
            vc |= max(encode<2, 15, 0x7b>(vh[i], kv, bits >> 16), vh[i] ? 1u : 0u) << (8 * i);
        }
        __builtin_nontemporal_store(mc, mo);
        __builtin_nontemporal_store(vc, vo);
        if (lane == 0)
        {
            global(T->ms)[block] = __uint_as_float((uint32_t)(km + 127) << 23);
            global(T->vs)[block] = __uint_as_float((uint32_t)(kv + 127) << 23);
        }
    }
    store_weights<WD>(T, i0, true, 4, nw);
    return true;
}

__device__ __forceinline__ float stepped_any(Constant<StepEntry> T, float w, float m, float v)
{
    return T->eps < kLeastEps ? stepped<true>(T, w, m, v) : stepped<false>(T, w, m, v);
}

// The same for any block: a tensor's last, numbers that are not finite, an eps near zero.
template <int WD, int GD, int BITS>
__device__ __forceinline__ void step_any(Constant<StepEntry> T, float factor, long long block, int lane)
{
    using W = typename Element<WD>::type;
    using G = typename Element<GD>::type;
    const long long i0 = block * TRIPS_MOMENT_BLOCK + lane * 4;
    const long long left = T->n - i0;
    const int count      = left >= 4 ? 4 : left > 0 ? (int)left : 0;
    const bool whole     = count == 4;
    W w4[4];
    G g4[4];
    load4(global(reinterpret_cast<const G*>(T->g)) + i0, whole, count, g4);
    load4(global(reinterpret_cast<const W*>(T->w)) + i0, whole, count, w4);
    float nw[4];
    if constexpr (BITS == 32)
    {
        float m[4], v[4];
        const auto mo = global(reinterpret_cast<float*>(T->m)) + i0;
        const auto vo = global(reinterpret_cast<float*>(T->v)) + i0;
        load4(mo, whole, count, m);
        load4(vo, whole, count, v);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float g = Element<GD>::to_float(g4[i]) * factor;
            m[i]  = fmaf(T->fc1, g, T->fb1 * m[i]);
            v[i]  = fmaf(T->fc2 * g, g, T->fb2 * v[i]);
            nw[i] = stepped_any(T, Element<WD>::to_float(w4[i]), m[i], v[i]);
        }
        store4(mo, whole, count, m);
        store4(vo, whole, count, v);
    }
    else
    {
        unsigned char m4[4], v4[4];
        const auto mo = global(reinterpret_cast<unsigned char*>(T->m)) + i0;
        const auto vo = global(reinterpret_cast<unsigned char*>(T->v)) + i0;
        load4(mo, whole, count, m4);
        load4(vo, whole, count, v4);
        const unsigned mw = m4[0] | m4[1] << 8 | m4[2] << 16 | (unsigned)m4[3] << 24;
        const unsigned vw = v4[0] | v4[1] << 8 | v4[2] << 16 | (unsigned)v4[3] << 24;
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mw, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mw, true);
        const auto v01 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vw, false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vw, true);
        const float mf[4] = {m01[0], m01[1], m23[0], m23[1]}, vf[4] = {v01[0], v01[1], v23[0], v23[1]};
        const double bm = T->b1 * (double)global(T->ms)[block], bv = T->b2 * (double)global(T->vs)[block];
        double m[4], v[4];
        uint32_t mtop = 0, vtop = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const double g = (double)Element<GD>::to_float(g4[i]) * (double)factor;
            m[i]  = fma(T->c1, g, bm * (double)mf[i]);
            v[i]  = fma(T->c2 * g, g, bv * (double)vf[i]);
            nw[i] = stepped_any(T, Element<WD>::to_float(w4[i]), (float)m[i], (float)v[i]);
            const uint32_t mh = high_word_up(m[i]), vh = high_word_up(v[i]);
            mtop = max(mtop, mh < 0x7ff00000u ? mh : 0u);
            vtop = max(vtop, vh < 0x7ff00000u ? vh : 0u);
        }
        const int km = scale_exponent<9>(wave_max(mtop)), kv = scale_exponent<16>(wave_max(vtop));
        const uint32_t at = (T->first_block + (uint32_t)block) * TRIPS_MOMENT_BLOCK + (uint32_t)lane * 4u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const uint32_t bits = mix((at + i) ^ T->key);
            const uint32_t mh = (uint32_t)((unsigned long long)__double_as_longlong(m[i]) >> 32) & 0x7fffffffu;
            const uint32_t vh = (uint32_t)((unsigned long long)__double_as_longlong(v[i]) >> 32) & 0x7fffffffu;
            const uint32_t mc = mh < 0x7ff00000u ? encode<3, 7, 0x7e>(mh, km, bits & 0xffffu) : 0x7fu;  // (no number)
            const uint32_t vc = vh < 0x7ff00000u ? encode<2, 15, 0x7b>(vh, kv, bits >> 16) : 0x7fu;
            m4[i] = (unsigned char)(mc | (__double_as_longlong(m[i]) < 0 ? 0x80u : 0u));
            v4[i] = (unsigned char)(v[i] > 0.0 ? max(vc, 1u) : vc);
        }
        store4(mo, whole, count, m4);
        store4(vo, whole, count, v4);
        if (lane == 0 && count > 0)
        {
            global(T->ms)[block] = __uint_as_float((uint32_t)(km + 127) << 23);
            global(T->vs)[block] = __uint_as_float((uint32_t)(kv + 127) << 23);
        }
    }
    store_weights<WD>(T, i0, whole, count, nw);
}

// The last entry of first_tiles[0..n) that is not behind `tile`, by the whole wavefront; n <= 4096.
__device__ __forceinline__ uint32_t tensor_of_tile(const uint32_t* first_tiles, uint32_t n, uint32_t tile, int lane)
{
    uint32_t base = 0, stride = (n + 63) / 64;
    if (stride > 1)
    {
        const uint32_t i = lane * stride;
        base = ((uint32_t)__popcll(__ballot(i < n && first_tiles[i] <= tile)) - 1u) * stride;
        const uint32_t j = base + lane;
        return base + (uint32_t)__popcll(__ballot(lane < (int)stride && j < n && first_tiles[j] <= tile)) - 1u;
    }
    return (uint32_t)__popcll(__ballot(lane < (int)n && first_tiles[lane] <= tile)) - 1u;
}

// 60M weights of 32 bits: moments in 32 bits 300 us (5.6 TB/s), in 8 bits 164 to 166 (5.8 TB/s; the card's clocks as they settle, in passes 10 to 100 up to 225; 7.5e7 vector instructions of wavefronts,
// 122 us if nothing else were issued: the codes are half of them); the 18 tensors of the benchmark's net 4.7.
template <int WD, int GD, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const StepParams p)
{
    const float factor = p.norm ? p.norm[1] : p.factor;
    if (!(fabsf(factor) <= FLT_MAX)) return;  // the step is skipped
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    uint32_t first = 0, behind = 0;
    Constant<StepEntry> T = (Constant<StepEntry>)p.entries;
    bool any = false;
    const uint32_t end = min(p.tiles, (blockIdx.x + 1u) * p.run);
    for (uint32_t tile = blockIdx.x * p.run; tile < end; ++tile)
    {
        if (tile >= behind)
        {
            const uint32_t i = (uint32_t)__builtin_amdgcn_readfirstlane((int)tensor_of_tile(p.first_tiles, p.n, tile, lane));
            T      = (Constant<StepEntry>)p.entries + i;
            first  = ((Constant<uint32_t>)p.first_tiles)[i];
            behind = i + 1 < p.n ? ((Constant<uint32_t>)p.first_tiles)[i + 1] : p.tiles;
            any    = T->eps < kLeastEps;
        }
        const long long block = (long long)(tile - first) * (kTileOptim / TRIPS_MOMENT_BLOCK) + wave;
        if (block * TRIPS_MOMENT_BLOCK >= T->n) continue;
        if (any || (block + 1) * TRIPS_MOMENT_BLOCK > T->n || !step_whole<WD, GD, BITS>(T, factor, block, lane))
            step_any<WD, GD, BITS>(T, factor, block, lane);
    }
}

// ---- the norm ----

struct NormTensor
{
    const void* g;
    long long n;
    uint32_t dtype;
};
struct NormTable
{
    NormTensor t[kNormTensors];
    uint32_t first_tiles[kNormTensors];
    uint32_t n, tiles, add;  // add: to the sums of an earlier launch of the call
    double* sums;            // [kNormGroups]
};
static_assert(sizeof(NormTable) <= 4096, "kernel arguments");

__device__ __forceinline__ double block_sum(double x, double* s)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    return s[0] + s[1] + s[2] + s[3];
}

template <int GD>
__device__ __forceinline__ double tile_squares(const NormTensor& T, long long tile)
{
    using G = typename Element<GD>::type;
    constexpr int E = 16 / sizeof(G), PASSES = kNormTile / (256 * E);
    const G* g = reinterpret_cast<const G*>(T.g);
    double sum = 0.0;
    const long long i0 = tile * kNormTile + (long long)threadIdx.x * E;
    if (tile * kNormTile + kNormTile <= T.n)
    {
        typename Pack<G, E>::type x[PASSES];
#pragma unroll
        for (int p = 0; p < PASSES; ++p)
            x[p] = __builtin_nontemporal_load(reinterpret_cast<const typename Pack<G, E>::type*>(g + i0 + p * 256 * E));
#pragma unroll
        for (int p = 0; p < PASSES; ++p)
#pragma unroll
            for (int e = 0; e < E; ++e)
            {
                const double y = (double)Element<GD>::to_float(x[p][e]);
                sum            = fma(y, y, sum);
            }
        return sum;
    }
    for (long long i = tile * kNormTile + threadIdx.x; i < T.n; i += 256)
    {
        const double y = (double)Element<GD>::to_float(g[i]);
        sum            = fma(y, y, sum);
    }
    return sum;
}

// 60M elements 38 us (6.3 TB/s), a net of 16,000 elements 4: a launch. At most kNormGroups partial sums, added by one workgroup.
__global__ __launch_bounds__(256) void grad_squares_kernel(const NormTable tab)
{
    __shared__ double s[4];
    double sum = 0.0;
    uint32_t i = 0, first = 0, behind = 0;
    for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x)
    {
        if (tile >= behind)
        {
            i      = (uint32_t)__builtin_amdgcn_readfirstlane((int)tensor_of_tile(tab.first_tiles, tab.n, tile, threadIdx.x & 63));
            first  = tab.first_tiles[i];
            behind = i + 1 < tab.n ? tab.first_tiles[i + 1] : tab.tiles;
        }
        const NormTensor& T    = tab.t[i];
        const long long within = tile - first;
        if (T.dtype == TRIPS_DTYPE_F32)
            sum += tile_squares<TRIPS_DTYPE_F32>(T, within);
        else if (T.dtype == TRIPS_DTYPE_BF16)
            sum += tile_squares<TRIPS_DTYPE_BF16>(T, within);
        else
            sum += tile_squares<TRIPS_DTYPE_F16>(T, within);
    }
    sum = block_sum(sum, s);
    if (threadIdx.x == 0) tab.sums[blockIdx.x] = tab.add ? tab.sums[blockIdx.x] + sum : sum;
}

// `sum`: this thread's share of the squares
__device__ __forceinline__ void write_norm(double sum, float max_norm, float loss_scale, float* out, double* s)
{
    sum = block_sum(sum, s);
    if (threadIdx.x == 0)
    {
        const double norm = sqrt(sum) / (double)loss_scale;
        double factor     = max_norm > 0.f ? fmin(1.0, (double)max_norm / (norm + 1e-6)) : 1.0;
        factor /= (double)loss_scale;
        out[0] = (float)norm;
        out[1] = norm <= DBL_MAX ? (float)factor : __builtin_nanf("");
    }
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* sums, int n, float max_norm, float loss_scale, float* out)
{
    __shared__ double s[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) sum += sums[i];
    write_norm(sum, max_norm, loss_scale, out, s);
}

// Before a step, one workgroup: the norm of the squares, if they were summed for it; the step counts go on; the step's table.
// All of it waits on memory and on double precision's long chains: what the tensors' rates need comes first, beside the sums.
__global__ __launch_bounds__(256) void adamw_begin_kernel(const StepTable tab)
{
    __shared__ double s[4];
    const uint32_t i    = threadIdx.x;
    const bool mine     = i < tab.n;
    const StepTensor& T = tab.t[mine ? i : 0];
    uint32_t t          = 0;
    if (mine) t = (uint32_t)*T.step + 1u;
    double sum = 0.0;
    if (tab.sums)
        for (uint32_t k = i; k < tab.groups; k += 256) sum += tab.sums[k];
    StepEntry e;
    if (mine)
    {
        const StepOptions& o = tab.o[T.group];
        e.w = T.w, e.g = T.g, e.m = T.m, e.v = T.v, e.ms = T.ms, e.vs = T.vs, e.copy = T.copy, e.n = T.n;
        e.b1 = o.beta1, e.c1 = 1.0 - o.beta1, e.b2 = o.beta2, e.c2 = 1.0 - o.beta2;
        e.fb1 = (float)e.b1, e.fc1 = (float)e.c1, e.fb2 = (float)e.b2, e.fc2 = (float)e.c2;
        e.keep = (float)(1.0 - o.lr * o.decay);
        e.rate = (float)(o.lr / (1.0 - power(o.beta1, t)));
        e.root = (float)(1.0 / sqrt(1.0 - power(o.beta2, t)));
        e.eps  = (float)o.eps;
        e.key  = mix(tab.seed + t * 0x9E3779B9u);
        e.first_block = T.first_block, e.copy_dtype = T.copy_dtype, e.unused = 0;
    }
    if (tab.sums)
    {
        write_norm(sum, tab.max_norm, tab.loss_scale, tab.norm, s);
        __syncthreads();
    }
    // (written by this workgroup, or by another launch)
    if (tab.norm && !(fabsf(__hip_atomic_load(tab.norm + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) <= FLT_MAX)) return;
    if (!mine) return;
    *T.step            = (int32_t)t;
    tab.entries[i]     = e;
    tab.first_tiles[i] = T.first_tile;
}

// `get(i)`: the gradients of tensor i of n, as a TripsGradTensor.
template <typename Get>
hipError_t launch_squares(const Get& get, int n, double* sums, int& groups, hipStream_t stream)
{
    auto tiles_of  = [](long long elements) { return (elements + kNormTile - 1) / kNormTile; };
    long long most = 1;  // tiles of the largest launch: all launches of the call have its grid
    for (int i = 0, used = 0, done = 0; done < n; used = 0)
    {
        long long tiles = 0;
        for (; done < n && used < kNormTensors; ++done, ++i)
            if (get(i).n > 0) tiles += tiles_of(get(i).n), ++used;
        most = tiles > most ? tiles : most;
    }
    if (most > 0x7fffffffll) return hipErrorInvalidValue;
    groups   = (int)(most < kNormGroups ? most : kNormGroups);
    int done = 0;
    bool add = false;
    do
    {
        NormTable tab;
        tab.n = 0, tab.tiles = 0, tab.add = add ? 1u : 0u, tab.sums = sums;
        for (; done < n && tab.n < kNormTensors; ++done)
        {
            const TripsGradTensor T = get(done);
            if (T.n <= 0) continue;
            tab.first_tiles[tab.n] = tab.tiles;
            tab.t[tab.n++]         = NormTensor{T.grads, T.n, (uint32_t)T.dtype};
            tab.tiles += (uint32_t)tiles_of(T.n);
        }
        hipLaunchKernelGGL(grad_squares_kernel, dim3(groups), dim3(256), 0, stream, tab);
        add = true;
    } while (done < n);
    return hipGetLastError();
}

template <int WD, int GD>
void launch_step_of(int bits, const StepParams& p, int groups, hipStream_t stream)
{
    if (bits == 32)
        hipLaunchKernelGGL((adamw_kernel<WD, GD, 32>), dim3(groups), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((adamw_kernel<WD, GD, 8>), dim3(groups), dim3(256), 0, stream, p);
}
template <int WD>
void launch_step(int gd, int bits, const StepParams& p, int groups, hipStream_t stream)
{
    if (gd == TRIPS_DTYPE_F32)
        launch_step_of<WD, TRIPS_DTYPE_F32>(bits, p, groups, stream);
    else if (gd == TRIPS_DTYPE_BF16)
        launch_step_of<WD, TRIPS_DTYPE_BF16>(bits, p, groups, stream);
    else
        launch_step_of<WD, TRIPS_DTYPE_F16>(bits, p, groups, stream);
}

struct StepLayout
{
    size_t sums, first_tiles, entries, bytes;
};
StepLayout step_layout(int n_tensors)
{
    auto up        = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t n = (size_t)(n_tensors < kStepTensors ? n_tensors : kStepTensors);
    StepLayout l;
    l.sums        = 0;
    l.first_tiles = TRIPS_GRAD_NORM_WORKSPACE_BYTES;
    l.entries     = l.first_tiles + up(n * sizeof(uint32_t));
    l.bytes       = l.entries + up(n * sizeof(StepEntry));
    return l;
}

int kind_of(const TripsAdamWTensor& t) { return t.weight_dtype * 8 + t.grad_dtype * 2 + (t.state_bits == 8 ? 1 : 0); }

// The tensors of one combination of types in one launch (of at most kStepTensors), their table before it.
hipError_t launch_steps(const TripsAdamWTensor* tensors, int n, const TripsAdamWOptions& opt, char* workspace, const double* sums, int sum_groups,
                        hipStream_t stream, Profiler* prof)
{
    const StepLayout l = step_layout(n);
    uint32_t kinds     = 0;
    for (int i = 0; i < n; ++i) kinds |= 1u << kind_of(tensors[i]);
    ProfScope ps(prof, "adamw", stream);
    for (int kind = 0; kind < 32; ++kind)
    {
        if (!(kinds >> kind & 1u)) continue;
        uint32_t block = 0;  // (mod 2^32)
        int done       = 0;
        while (done < n)
        {
            StepParams p;
            p.entries     = reinterpret_cast<const StepEntry*>(workspace + l.entries);
            p.first_tiles = reinterpret_cast<const uint32_t*>(workspace + l.first_tiles);
            p.n = 0, p.norm = opt.grad_norm, p.factor = (float)(1.0 / (double)opt.loss_scale);
            long long tiles = 0;
            while (done < n && p.n < kStepTensors && tiles < (1ll << 31))
            {
                StepTable tab;
                tab.n = 0, tab.seed = opt.seed, tab.norm = opt.grad_norm, tab.sums = sums, tab.groups = (uint32_t)sum_groups;
                tab.max_norm = opt.max_norm, tab.loss_scale = opt.loss_scale;
                tab.entries     = reinterpret_cast<StepEntry*>(workspace + l.entries) + p.n;
                tab.first_tiles = reinterpret_cast<uint32_t*>(workspace + l.first_tiles) + p.n;
                int groups      = 0;
                for (; done < n && tab.n < kTensors && p.n + tab.n < kStepTensors && tiles < (1ll << 31); ++done)
                {
                    const TripsAdamWTensor& T = tensors[done];
                    const uint32_t blocks     = (uint32_t)((T.n + TRIPS_MOMENT_BLOCK - 1) / TRIPS_MOMENT_BLOCK);
                    if (kind_of(T) == kind)
                    {
                        const StepOptions o = {T.lr, T.beta1, T.beta2, T.eps, T.weight_decay};
                        int g = groups - 1;
                        while (g >= 0 && !(tab.o[g].lr == o.lr && tab.o[g].beta1 == o.beta1 && tab.o[g].beta2 == o.beta2 &&
                                           tab.o[g].eps == o.eps && tab.o[g].decay == o.decay))
                            --g;
                        if (g < 0)
                        {
                            if (groups == kGroups) break;
                            g        = groups++;
                            tab.o[g] = o;
                        }
                        StepTensor& S = tab.t[tab.n++];
                        S.w = T.weights, S.g = T.grads, S.m = T.first_moment, S.v = T.second_moment, S.ms = T.first_scale;
                        S.vs = T.second_scale, S.copy = T.copy, S.step = T.step, S.n = T.n;
                        S.first_tile = (uint32_t)tiles, S.first_block = block;
                        S.group = (uint8_t)g, S.copy_dtype = (uint8_t)T.copy_dtype;
                        tiles += (T.n + kTileOptim - 1) / kTileOptim;
                    }
                    block += blocks;
                }
                if (tab.n == 0) continue;
                hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(256), 0, stream, tab);
                sums = nullptr;  // (the first one has made the norm)
                p.n += tab.n;
            }
            if (tiles == 0) continue;
            p.tiles     = (uint32_t)tiles;
            p.run       = tiles <= kStepGroups ? 1u : (uint32_t)std::max<long long>(kStepRun, (tiles >> 23) + 1);  // (less than 2^32 threads)
            const int g = (int)((tiles + p.run - 1) / p.run);
            const int wd = kind / 8, gd = kind / 2 % 4, bits = kind & 1 ? 8 : 32;
            if (wd == TRIPS_DTYPE_F32)
                launch_step<TRIPS_DTYPE_F32>(gd, bits, p, g, stream);
            else if (wd == TRIPS_DTYPE_BF16)
                launch_step<TRIPS_DTYPE_BF16>(gd, bits, p, g, stream);
            else
                launch_step<TRIPS_DTYPE_F16>(gd, bits, p, g, stream);
        }
    }
    return hipGetLastError();
}

int check_workspace(const void* workspace, size_t bytes, size_t need)
{
    if (!workspace || !aligned(workspace, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
    if (bytes < need) return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %zu needed", bytes, need);
    return TRIPS_OK;
}

int check_norm(float max_norm, float loss_scale)
{
    if (std::isnan(max_norm)) return set_error(TRIPS_ERR_INVALID_ARG, "max_norm is not a number");
    if (!(loss_scale > 0.f) || !std::isfinite(loss_scale)) return set_error(TRIPS_ERR_INVALID_ARG, "loss_scale %g is not positive and finite", (double)loss_scale);
    return TRIPS_OK;
}

constexpr int64_t kMostElements = (int64_t)1 << 38;  // of a tensor: a launch counts less than 2^32 tiles
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" {

int trips_grad_norm(TripsCtx* ctx, const TripsGradTensor* tensors, int n_tensors, float max_norm, float loss_scale,
                    float* grad_norm, void* workspace, size_t workspace_bytes, void* stream_)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return set_error(TRIPS_ERR_INVALID_ARG, "tensors");
    if (!grad_norm || !aligned(grad_norm, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "grad_norm must be a device pointer to two floats");
    if (int e = check_norm(max_norm, loss_scale)) return e;
    if (int e = check_workspace(workspace, workspace_bytes, TRIPS_GRAD_NORM_WORKSPACE_BYTES)) return e;
    for (int i = 0; i < n_tensors; ++i)
    {
        const TripsGradTensor& t = tensors[i];
        if (t.n < 0 || t.n > kMostElements) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: n = %lld", i, (long long)t.n);
        if (!dtype_ok(t.dtype)) return set_error(TRIPS_ERR_UNSUPPORTED, "tensor %d: dtype %d", i, t.dtype);
        if (t.n > 0 && (!t.grads || !aligned(t.grads, dtype_bytes(t.dtype)))) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: grads is NULL or not aligned to its elements", i);
    }
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    ProfScope ps(profiler(ctx), "grad_norm", stream);
    double* sums = reinterpret_cast<double*>(workspace);
    int groups   = 0;
    hipError_t e = launch_squares([&](int i) { return tensors[i]; }, n_tensors, sums, groups, stream);
    if (e == hipSuccess)
    {
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, stream, sums, groups, max_norm, loss_scale, grad_norm);
        e = hipGetLastError();
    }
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "norm launch");
}

int trips_adamw_workspace_size(int n_tensors, size_t* bytes)
{
    if (!bytes) return set_error(TRIPS_ERR_INVALID_ARG, "bytes is NULL");
    if (n_tensors < 0) return set_error(TRIPS_ERR_INVALID_ARG, "n_tensors = %d", n_tensors);
    *bytes = step_layout(n_tensors).bytes;
    return TRIPS_OK;
}

int trips_adamw_step(TripsCtx* ctx, const TripsAdamWTensor* tensors, int n_tensors, const TripsAdamWOptions* options,
                     void* workspace, size_t workspace_bytes, void* stream_)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (!options) return set_error(TRIPS_ERR_INVALID_ARG, "options is NULL");
    if (options->abi_version != TRIPS_ABI_VERSION)
        return set_error(TRIPS_ERR_INVALID_ARG, "abi_version %d, library has %d", options->abi_version, TRIPS_ABI_VERSION);
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return set_error(TRIPS_ERR_INVALID_ARG, "tensors");
    if (options->compute_norm && !options->grad_norm) return set_error(TRIPS_ERR_INVALID_ARG, "compute_norm without grad_norm");
    if (!aligned(options->grad_norm, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "grad_norm is not aligned");
    if (int e = check_norm(options->max_norm, options->loss_scale)) return e;
    if (options->max_norm > 0.f && !options->grad_norm) return set_error(TRIPS_ERR_INVALID_ARG, "max_norm without grad_norm");
    if (int e = check_workspace(workspace, workspace_bytes, step_layout(n_tensors).bytes)) return e;
    for (int i = 0; i < n_tensors; ++i)
    {
        const TripsAdamWTensor& t = tensors[i];
        if (t.n < 0 || t.n > kMostElements) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: n = %lld", i, (long long)t.n);
        if (!dtype_ok(t.weight_dtype) || !dtype_ok(t.grad_dtype) || (t.copy && !dtype_ok(t.copy_dtype)))
            return set_error(TRIPS_ERR_UNSUPPORTED, "tensor %d: dtypes %d, %d, %d (float32, bfloat16 and float16 are supported)", i, t.weight_dtype, t.grad_dtype, t.copy_dtype);
        if (t.state_bits != 32 && t.state_bits != 8) return set_error(TRIPS_ERR_UNSUPPORTED, "tensor %d: state_bits %d is neither 32 nor 8", i, t.state_bits);
        if (!t.step || !aligned(t.step, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: step is NULL or not aligned", i);
        if (t.n > 0)
        {
            if (!t.weights || !t.grads || !t.first_moment || !t.second_moment || (t.state_bits == 8 && (!t.first_scale || !t.second_scale)))
                return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: NULL pointer", i);
            const size_t state = t.state_bits == 8 ? 1 : 4;
            if (!aligned(t.weights, dtype_bytes(t.weight_dtype)) || !aligned(t.grads, dtype_bytes(t.grad_dtype)) || !aligned(t.first_moment, state) ||
                !aligned(t.second_moment, state) || (t.state_bits == 8 && (!aligned(t.first_scale, 4) || !aligned(t.second_scale, 4))) ||
                (t.copy && !aligned(t.copy, dtype_bytes(t.copy_dtype))))
                return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: a pointer is not aligned to its elements", i);
        }
        // (written so that no number fails too)
        if (!(t.beta1 >= 0.0 && t.beta1 < 1.0 && t.beta2 >= 0.0 && t.beta2 < 1.0)) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: betas %g, %g", i, t.beta1, t.beta2);
        if (!(t.lr >= 0.0 && t.eps >= 0.0 && t.weight_decay >= 0.0) || !std::isfinite(t.lr) || !std::isfinite(t.eps) || !std::isfinite(t.weight_decay))
            return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: lr %g, eps %g, weight_decay %g", i, t.lr, t.eps, t.weight_decay);
    }
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (n_tensors == 0) return TRIPS_OK;
    double* sums = nullptr;
    int groups   = 0;
    if (options->compute_norm)
    {
        ProfScope ps(profiler(ctx), "grad_norm", stream);
        sums         = reinterpret_cast<double*>(workspace);
        auto grads   = [&](int i) { return TripsGradTensor{tensors[i].grads, tensors[i].n, tensors[i].grad_dtype}; };
        hipError_t e = launch_squares(grads, n_tensors, sums, groups, stream);
        if (e != hipSuccess) return hip_error(e, "norm launch");
    }
    hipError_t e = launch_steps(tensors, n_tensors, *options, reinterpret_cast<char*>(workspace), sums, groups, stream, profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "adamw launch");
}

}  // extern "C"
