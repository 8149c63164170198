// AdamW over many tensors in one launch, moments in 32 or 8 bits, and the global norm of their gradients (gfx950).
//
// Both are bound by memory: a step reads and writes each element of weights and moments once and reads each gradient once
// (28 bytes an element in 32 bits, 16 with moments in 8), the norm reads the gradients. Tensors come as a table in the
// kernel's arguments; a workgroup finds the tensor of each of its tiles there.
#include <float.h>

#include <cmath>

#include "abi_common.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int kTensors     = 40;   // tensors of a launch: what 4 KB of kernel arguments hold
constexpr int kGroups      = 8;    // different sets of options among them
constexpr int kTileOptim   = 1024; // elements of a tile: four wavefronts with a block of 256 each
constexpr int kStepGroups  = 2048; // workgroups of a step
constexpr int kNormTensors = 120;
constexpr int kNormTile    = 4096; // elements of a tile of the norm
constexpr int kNormGroups  = 1024; // workgroups of the norm = partial sums
static_assert(TRIPS_MOMENT_BLOCK == 256, "a block is four elements a lane");
static_assert(256 + kNormGroups * sizeof(double) <= TRIPS_ADAMW_WORKSPACE_BYTES, "workspace");

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
    uint32_t first_tile;   // of this launch
    uint32_t first_block;  // of the call, in blocks of 256 elements
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
    uint32_t n, tiles;
    uint32_t seed;
    float factor;            // where there is no `norm`
    const float* norm;       // {norm, factor} or NULL
    uint32_t* ticket;        // workgroups that are done, 0 between launches
};
static_assert(sizeof(StepTable) <= 4096, "kernel arguments");

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

__device__ __forceinline__ uint32_t wave_max(uint32_t x)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
    return x;
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
// at most MOST. The bits of a double are such a code, followed by 52 - MANTISSA more and with another bias; the steps are added
// to those of the high word, whose carry is the rounding (what the low word holds can make no carry: the addend is a multiple
// of the high word's last place). Below the lowest normal number steps stay as they are: the significand shifts right instead.
template <int MANTISSA, int BIAS, int MOST>
__device__ __forceinline__ uint32_t encode(double x, int k, uint32_t r)
{
    const uint32_t hi = (uint32_t)((unsigned long long)__double_as_longlong(x) >> 32) & 0x7fffffffu;
    if (hi >= 0x7ff00000u) return 0x7fu;  // infinite or no number: no number
    const int t        = (int)hi - (k + 1023 - BIAS) * (1 << 20);
    const int e        = t >> 20;
    const uint32_t sig = 0x100000u | (hi & 0xfffffu);
    const uint32_t y   = e >= 1 ? (uint32_t)t : sig >> min(1 - e, 31);
    constexpr int DROP = 20 - MANTISSA;
    return min((y + ((2u * r + 1u) << (DROP - 17))) >> DROP, (uint32_t)MOST);
}

// The launch's rates of one tensor at step t.
struct Rates
{
    double b1, c1, b2, c2;       // beta and 1 - beta
    float fb1, fc1, fb2, fc2;    // the same in float
    float keep, rate, root, eps; // 1 - lr decay, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
};
__device__ __forceinline__ Rates rates(const StepOptions& o, uint32_t t)
{
    Rates r;
    r.b1 = o.beta1, r.c1 = 1.0 - o.beta1, r.b2 = o.beta2, r.c2 = 1.0 - o.beta2;
    r.fb1 = (float)r.b1, r.fc1 = (float)r.c1, r.fb2 = (float)r.b2, r.fc2 = (float)r.c2;
    r.keep = (float)(1.0 - o.lr * o.decay);
    r.rate = (float)(o.lr / (1.0 - power(o.beta1, t)));
    r.root = (float)(1.0 / sqrt(1.0 - power(o.beta2, t)));
    r.eps  = (float)o.eps;
    return r;
}

__device__ __forceinline__ float stepped(const Rates& r, float w, float m, float v)
{
    return fmaf(-r.rate, m / fmaf(sqrtf(v), r.root, r.eps), r.keep * w);
}

template <typename T>
__device__ __forceinline__ void load4(const T* from, bool whole, int count, T (&x)[4])
{
    if (whole)
    {
        const auto q = __builtin_nontemporal_load(reinterpret_cast<const typename Pack<T, 4>::type*>(from));
        x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < count ? from[i] : T(0);
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* to, bool whole, int count, const T (&x)[4])
{
    if (whole)
    {
        typename Pack<T, 4>::type q = {x[0], x[1], x[2], x[3]};
        __builtin_nontemporal_store(q, reinterpret_cast<typename Pack<T, 4>::type*>(to));
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < count) to[i] = x[i];
    }
}

// Four elements a lane, a block of 256 a wavefront.
template <int WD, int GD, int BITS>
__device__ __forceinline__ void step_block(const StepTensor& T, const Rates& r, float factor, uint32_t key, long long block, int lane)
{
    using W = typename Element<WD>::type;
    using G = typename Element<GD>::type;
    const long long i0 = block * TRIPS_MOMENT_BLOCK + lane * 4;
    const long long left = T.n - i0;
    const int count      = left >= 4 ? 4 : left > 0 ? (int)left : 0;
    const bool whole     = count == 4;
    W w4[4];
    G g4[4];
    load4(reinterpret_cast<const G*>(T.g) + i0, whole, count, g4);
    load4(reinterpret_cast<const W*>(T.w) + i0, whole, count, w4);
    float nw[4];
    if constexpr (BITS == 32)
    {
        float m[4], v[4];
        float* mo = reinterpret_cast<float*>(T.m) + i0;
        float* vo = reinterpret_cast<float*>(T.v) + i0;
        load4(mo, whole, count, m);
        load4(vo, whole, count, v);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float g = Element<GD>::to_float(g4[i]) * factor;
            m[i]  = fmaf(r.fc1, g, r.fb1 * m[i]);
            v[i]  = fmaf(r.fc2 * g, g, r.fb2 * v[i]);
            nw[i] = stepped(r, Element<WD>::to_float(w4[i]), m[i], v[i]);
        }
        store4(mo, whole, count, m);
        store4(vo, whole, count, v);
    }
    else
    {
        // The new moments in double: which code they get must not depend on roundings on the way.
        unsigned char m4[4], v4[4];
        unsigned char* mo = reinterpret_cast<unsigned char*>(T.m) + i0;
        unsigned char* vo = reinterpret_cast<unsigned char*>(T.v) + i0;
        load4(mo, whole, count, m4);
        load4(vo, whole, count, v4);
        const unsigned mw = m4[0] | m4[1] << 8 | m4[2] << 16 | (unsigned)m4[3] << 24;
        const unsigned vw = v4[0] | v4[1] << 8 | v4[2] << 16 | (unsigned)v4[3] << 24;
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mw, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mw, true);
        const auto v01 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vw, false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vw, true);
        const float mf[4] = {m01[0], m01[1], m23[0], m23[1]}, vf[4] = {v01[0], v01[1], v23[0], v23[1]};
        const double bm = r.b1 * (double)T.ms[block], bv = r.b2 * (double)T.vs[block];
        double m[4], v[4];
        uint32_t mtop = 0, vtop = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const double g = (double)Element<GD>::to_float(g4[i]) * (double)factor;
            m[i]  = fma(r.c1, g, bm * (double)mf[i]);
            v[i]  = fma(r.c2 * g, g, bv * (double)vf[i]);
            nw[i] = stepped(r, Element<WD>::to_float(w4[i]), (float)m[i], (float)v[i]);
            const uint32_t mh = high_word_up(m[i]), vh = high_word_up(v[i]);
            mtop = max(mtop, mh < 0x7ff00000u ? mh : 0u);
            vtop = max(vtop, vh < 0x7ff00000u ? vh : 0u);
        }
        const int km = scale_exponent<9>(wave_max(mtop)), kv = scale_exponent<16>(wave_max(vtop));
        const uint32_t at = (T.first_block + (uint32_t)block) * TRIPS_MOMENT_BLOCK + (uint32_t)lane * 4u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const uint32_t bits = mix((at + i) ^ key);
            const uint32_t mc = encode<3, 7, 0x7e>(m[i], km, bits & 0xffffu);
            const uint32_t vc = encode<2, 15, 0x7b>(v[i], kv, bits >> 16);
            m4[i] = (unsigned char)(mc | (__double_as_longlong(m[i]) < 0 ? 0x80u : 0u));
            v4[i] = (unsigned char)(v[i] > 0.0 ? max(vc, 1u) : vc);
        }
        store4(mo, whole, count, m4);
        store4(vo, whole, count, v4);
        if (lane == 0 && count > 0)
        {
            T.ms[block] = __uint_as_float((uint32_t)(km + 127) << 23);
            T.vs[block] = __uint_as_float((uint32_t)(kv + 127) << 23);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w4[i] = Element<WD>::from_float(nw[i]);
    store4(reinterpret_cast<W*>(T.w) + i0, whole, count, w4);
    if (T.copy)
    {
        if (T.copy_dtype == TRIPS_DTYPE_F32)
            store4(reinterpret_cast<float*>(T.copy) + i0, whole, count, nw);
        else
        {
            const bool bf = T.copy_dtype == TRIPS_DTYPE_BF16;
            unsigned short c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                c[i] = bf ? Element<TRIPS_DTYPE_BF16>::from_float(nw[i]) : Element<TRIPS_DTYPE_F16>::from_float(nw[i]);
            store4(reinterpret_cast<unsigned short*>(T.copy) + i0, whole, count, c);
        }
    }
}

template <int WD, int GD, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const StepTable tab)
{
    const float factor = tab.norm ? tab.norm[1] : tab.factor;
    const bool skip    = !(fabsf(factor) <= FLT_MAX);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (!skip)
    {
        uint32_t ti = 0, known = ~0u, key = 0;
        Rates r;
        for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x)
        {
            while (ti + 1 < tab.n && tile >= tab.t[ti + 1].first_tile) ++ti;
            const StepTensor& T = tab.t[ti];
            if (ti != known)
            {
                const uint32_t t = (uint32_t)*T.step + 1u;
                r     = rates(tab.o[T.group], t);
                key   = mix(tab.seed + t * 0x9E3779B9u);
                known = ti;
            }
            const long long block = (long long)(tile - T.first_tile) * (kTileOptim / TRIPS_MOMENT_BLOCK) + wave;
            if (block * TRIPS_MOMENT_BLOCK < T.n) step_block<WD, GD, BITS>(T, r, factor, key, block, lane);
        }
    }
    // The step counts go on when every workgroup has read them: the last one to get here counts. (All that a workgroup does
    // with the counts ends before its barrier; the ticket orders nothing else.)
    __shared__ uint32_t s_last;
    __syncthreads();
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(tab.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1u ? 1u : 0u;
    __syncthreads();
    if (s_last)
    {
        if (!skip && threadIdx.x < tab.n) *tab.t[threadIdx.x].step += 1;
        if (threadIdx.x == 0) *tab.ticket = 0u;
    }
}

// ---- the norm ----

struct NormTensor
{
    const void* g;
    long long n;
    uint32_t first_tile, dtype;
};
struct NormTable
{
    NormTensor t[kNormTensors];
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

__global__ __launch_bounds__(256) void grad_squares_kernel(const NormTable tab)
{
    __shared__ double s[4];
    double sum  = 0.0;
    uint32_t ti = 0;
    for (uint32_t tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x)
    {
        while (ti + 1 < tab.n && tile >= tab.t[ti + 1].first_tile) ++ti;
        const NormTensor& T    = tab.t[ti];
        const long long within = tile - T.first_tile;
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

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* sums, int n, float max_norm, float loss_scale, float* out)
{
    __shared__ double s[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) sum += sums[i];
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

// `get(i)`: the gradients of tensor i of n, as a TripsGradTensor.
template <typename Get>
hipError_t launch_norm(const Get& get, int n, float max_norm, float loss_scale, float* out, void* workspace, hipStream_t stream,
                       Profiler* prof)
{
    double* sums   = reinterpret_cast<double*>(reinterpret_cast<char*>(workspace) + 256);
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
    const int groups = (int)(most < kNormGroups ? most : kNormGroups);
    ProfScope ps(prof, "grad_norm", stream);
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
            tab.t[tab.n++] = NormTensor{T.grads, T.n, tab.tiles, (uint32_t)T.dtype};
            tab.tiles += (uint32_t)tiles_of(T.n);
        }
        hipLaunchKernelGGL(grad_squares_kernel, dim3(groups), dim3(256), 0, stream, tab);
        add = true;
    } while (done < n);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, stream, sums, groups, max_norm, loss_scale, out);
    return hipGetLastError();
}

template <int WD, int GD>
void launch_step_of(int bits, const StepTable& tab, int groups, hipStream_t stream)
{
    if (bits == 32)
        hipLaunchKernelGGL((adamw_kernel<WD, GD, 32>), dim3(groups), dim3(256), 0, stream, tab);
    else
        hipLaunchKernelGGL((adamw_kernel<WD, GD, 8>), dim3(groups), dim3(256), 0, stream, tab);
}
template <int WD>
void launch_step(int gd, int bits, const StepTable& tab, int groups, hipStream_t stream)
{
    if (gd == TRIPS_DTYPE_F32)
        launch_step_of<WD, TRIPS_DTYPE_F32>(bits, tab, groups, stream);
    else if (gd == TRIPS_DTYPE_BF16)
        launch_step_of<WD, TRIPS_DTYPE_BF16>(bits, tab, groups, stream);
    else
        launch_step_of<WD, TRIPS_DTYPE_F16>(bits, tab, groups, stream);
}

int kind_of(const TripsAdamWTensor& t) { return t.weight_dtype * 8 + t.grad_dtype * 2 + (t.state_bits == 8 ? 1 : 0); }

// The tensors of one combination of types, in launches of at most kTensors.
hipError_t launch_steps(const TripsAdamWTensor* tensors, int n, const TripsAdamWOptions& opt, void* workspace, hipStream_t stream,
                        Profiler* prof)
{
    uint32_t kinds = 0;
    for (int i = 0; i < n; ++i) kinds |= 1u << kind_of(tensors[i]);
    ProfScope ps(prof, "adamw", stream);
    for (int kind = 0; kind < 32; ++kind)
    {
        if (!(kinds >> kind & 1u)) continue;
        uint32_t block = 0;  // (mod 2^32)
        int done       = 0;
        while (done < n)
        {
            StepTable tab;
            tab.n = 0, tab.seed = opt.seed, tab.norm = opt.grad_norm, tab.factor = (float)(1.0 / (double)opt.loss_scale);
            tab.ticket      = reinterpret_cast<uint32_t*>(workspace);
            long long tiles = 0;
            int groups      = 0;
            const TripsAdamWTensor* first = nullptr;
            for (; done < n && tab.n < kTensors; ++done)
            {
                const TripsAdamWTensor& T = tensors[done];
                const uint32_t blocks     = (uint32_t)((T.n + TRIPS_MOMENT_BLOCK - 1) / TRIPS_MOMENT_BLOCK);
                if (kind_of(T) == kind)
                {
                    first = &T;
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
            if (tiles > 0x7fffffffll) return hipErrorInvalidValue;
            tab.tiles   = (uint32_t)tiles;
            const int g = tiles < 1 ? 1 : tiles > kStepGroups ? kStepGroups : (int)tiles;
            if (first->weight_dtype == TRIPS_DTYPE_F32)
                launch_step<TRIPS_DTYPE_F32>(first->grad_dtype, first->state_bits, tab, g, stream);
            else if (first->weight_dtype == TRIPS_DTYPE_BF16)
                launch_step<TRIPS_DTYPE_BF16>(first->grad_dtype, first->state_bits, tab, g, stream);
            else
                launch_step<TRIPS_DTYPE_F16>(first->grad_dtype, first->state_bits, tab, g, stream);
        }
    }
    return hipGetLastError();
}

int check_workspace(const void* workspace, size_t bytes)
{
    if (!workspace || !aligned(workspace, 256)) return set_error(TRIPS_ERR_INVALID_ARG, "workspace must be a 256-byte aligned device pointer");
    if (bytes < TRIPS_ADAMW_WORKSPACE_BYTES)
        return set_error(TRIPS_ERR_WORKSPACE_SMALL, "workspace has %zu bytes, %d needed", bytes, TRIPS_ADAMW_WORKSPACE_BYTES);
    return TRIPS_OK;
}

int check_norm(float max_norm, float loss_scale)
{
    if (std::isnan(max_norm)) return set_error(TRIPS_ERR_INVALID_ARG, "max_norm is not a number");
    if (!(loss_scale > 0.f) || !std::isfinite(loss_scale)) return set_error(TRIPS_ERR_INVALID_ARG, "loss_scale %g is not positive and finite", (double)loss_scale);
    return TRIPS_OK;
}

constexpr int64_t kMostElements = (int64_t)1 << 38;  // of a tensor: tiles are counted in 32 bits
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" {

int trips_grad_norm(TripsCtx* ctx, const TripsGradTensor* tensors, int n_tensors, float max_norm, float loss_scale,
                    float* grad_norm, void* workspace, size_t workspace_bytes, void* stream)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return set_error(TRIPS_ERR_INVALID_ARG, "tensors");
    if (!grad_norm || !aligned(grad_norm, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "grad_norm must be a device pointer to two floats");
    if (int e = check_norm(max_norm, loss_scale)) return e;
    if (int e = check_workspace(workspace, workspace_bytes)) return e;
    for (int i = 0; i < n_tensors; ++i)
    {
        const TripsGradTensor& t = tensors[i];
        if (t.n < 0 || t.n > kMostElements) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: n = %lld", i, (long long)t.n);
        if (!dtype_ok(t.dtype)) return set_error(TRIPS_ERR_UNSUPPORTED, "tensor %d: dtype %d", i, t.dtype);
        if (t.n > 0 && (!t.grads || !aligned(t.grads, dtype_bytes(t.dtype)))) return set_error(TRIPS_ERR_INVALID_ARG, "tensor %d: grads is NULL or not aligned to its elements", i);
    }
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    hipError_t e = launch_norm([&](int i) { return tensors[i]; }, n_tensors, max_norm, loss_scale, grad_norm, workspace,
                               reinterpret_cast<hipStream_t>(stream), profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "norm launch");
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
    if (int e = check_workspace(workspace, workspace_bytes)) return e;
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
    if (options->compute_norm)
    {
        auto grads   = [&](int i) { return TripsGradTensor{tensors[i].grads, tensors[i].n, tensors[i].grad_dtype}; };
        hipError_t e = launch_norm(grads, n_tensors, options->max_norm, options->loss_scale, options->grad_norm, workspace, stream, profiler(ctx));
        if (e != hipSuccess) return hip_error(e, "norm launch");
    }
    hipError_t e = launch_steps(tensors, n_tensors, *options, workspace, stream, profiler(ctx));
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "adamw launch");
}

}  // extern "C"
