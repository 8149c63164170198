// Dropout by a counter-based generator: the mask is made where it is used and never stored (gfx950).
//
//   out_i = (kept_i ? x_i factor : 0) + residual_i
//
// The generator is Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011); a block of its
// 128 bits serves eight elements, 16 bits each, which makes p a multiple of 2^-16.
#include <algorithm>
#include <cmath>

#include "abi_common.h"

#include "../../include/trips_loss.h"

#pragma clang fp contract(off)

namespace trips
{
namespace
{
constexpr int64_t kMostElements = 1ll << 40;
constexpr unsigned kMostBlocks  = 1u << 22;  // of 256 threads

struct DropoutParams
{
    const void* x;
    const void* residual;
    const uint32_t* step_at;
    uint32_t* step_used;
    void* out;
    long long n;
    uint32_t seed_low, seed_high, call, step, border;
    float factor;
};

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1)
{
#pragma unroll
    for (int r = 0; r < 10; ++r)
    {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        const uint32_t x = (uint32_t)(b >> 32) ^ c[1] ^ k0, y = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[0] = x, c[1] = (uint32_t)b, c[2] = y, c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
}

// 16 bytes a thread: one block of the generator, in 32 bits half of one (which two threads make then: with eight elements a thread, whose two
// loads lie 32 bytes apart, 6M x 4 took 37 us, so 30). Stored past the caches' usual order (a residual's sum of 8191 x 4097 bfloat16 numbers
// 40 us, so 32; without a residual no difference). Bound by memory: 6.3 TB/s with a residual, 5.8 without in bfloat16.
template <int D, bool RESIDUAL>
__global__ __launch_bounds__(256) void dropout_kernel(const DropoutParams p)
{
    using E           = Element<D>;
    using T           = typename E::type;
    constexpr int V   = 16 / sizeof(T);
    using Wide        = typename Pack<T, V>::type;
    const uint32_t step = p.step_at ? *p.step_at : p.step;
    if (p.step_used && blockIdx.x == 0 && threadIdx.x == 0) *p.step_used = step;
    const long long pieces = (p.n + V - 1) / V;
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < pieces; q += (long long)gridDim.x * 256)
    {
        const long long i = q * V, block = i >> 3;
        const bool whole  = i + V <= p.n;
        Wide x = {}, residual = {};
        if (whole)
        {
            x = *reinterpret_cast<const Wide*>(reinterpret_cast<const T*>(p.x) + i);
            if (RESIDUAL) residual = *reinterpret_cast<const Wide*>(reinterpret_cast<const T*>(p.residual) + i);
        }
        else
            for (int e = 0; e < (int)(p.n - i); ++e)
            {
                x[e] = reinterpret_cast<const T*>(p.x)[i + e];
                if (RESIDUAL) residual[e] = reinterpret_cast<const T*>(p.residual)[i + e];
            }
        uint32_t c[4] = {(uint32_t)block, (uint32_t)(block >> 32), p.call, step};
        philox(c, p.seed_low, p.seed_high);
        if (V == 4 && (q & 1)) c[0] = c[2], c[1] = c[3];
        Wide out;
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            const uint32_t bits = e & 1 ? c[e >> 1] >> 16 : c[e >> 1] & 0xFFFFu;
            float y             = bits >= p.border ? E::to_float(x[e]) * p.factor : 0.f;
            if (RESIDUAL) y += E::to_float(residual[e]);
            out[e] = E::from_float(y);
        }
        T* to = reinterpret_cast<T*>(p.out) + i;
        if (whole)
            __builtin_nontemporal_store(out, reinterpret_cast<Wide*>(to));
        else
            for (int e = 0; e < (int)(p.n - i); ++e) to[e] = out[e];
    }
}

template <int D>
void launch(const DropoutParams& p, hipStream_t stream)
{
    constexpr int V        = 16 / sizeof(typename Element<D>::type);
    const long long blocks = std::max<long long>(1, ((p.n + V - 1) / V + 255) / 256);
    const unsigned grid    = (unsigned)std::min<long long>(blocks, kMostBlocks);
    (p.residual ? dropout_kernel<D, true> : dropout_kernel<D, false>)<<<grid, 256, 0, stream>>>(p);
}
}  // namespace
}  // namespace trips

using namespace trips;

extern "C" int trips_dropout(TripsCtx* ctx, const TripsDropoutDesc* desc, const void* x, const void* residual, const uint32_t* step_at, uint32_t* step_used,
                             void* out, void* stream)
{
    if (!ctx) return set_error(TRIPS_ERR_INVALID_ARG, "ctx is NULL");
    if (!desc) return set_error(TRIPS_ERR_INVALID_ARG, "desc is NULL");
    const TripsDropoutDesc& d = *desc;
    if (d.abi_version != TRIPS_ABI_VERSION) return set_error(TRIPS_ERR_INVALID_ARG, "abi_version %d, library is %d", d.abi_version, TRIPS_ABI_VERSION);
    if (!dtype_ok(d.dtype)) return set_error(TRIPS_ERR_UNSUPPORTED, "dtype %d", d.dtype);
    if (d.n < 0 || d.n >= kMostElements) return set_error(TRIPS_ERR_INVALID_ARG, "n = %lld", (long long)d.n);
    if (!(d.p >= 0.0 && d.p <= 1.0)) return set_error(TRIPS_ERR_INVALID_ARG, "p = %g", d.p);
    const size_t size = dtype_bytes(d.dtype);
    if ((!x && d.n > 0) || !aligned(x, size)) return set_error(TRIPS_ERR_INVALID_ARG, "x is NULL or not aligned");
    if ((!out && d.n > 0) || !aligned(out, size)) return set_error(TRIPS_ERR_INVALID_ARG, "out is NULL or not aligned");
    if (!aligned(residual, size)) return set_error(TRIPS_ERR_INVALID_ARG, "residual is not aligned");
    if (!aligned(step_at, 4) || !aligned(step_used, 4)) return set_error(TRIPS_ERR_INVALID_ARG, "step_at or step_used is not aligned");
    if (d.n == 0 && !step_used) return TRIPS_OK;
    DropoutParams p{};
    p.x = x, p.residual = residual, p.step_at = step_at, p.step_used = step_used, p.out = out, p.n = d.n;
    p.seed_low = (uint32_t)d.seed, p.seed_high = (uint32_t)(d.seed >> 32), p.call = d.call, p.step = d.step;
    p.border = (uint32_t)std::nearbyint(d.p * 65536.0);
    p.factor = p.border < 65536u ? (float)(65536.0 / (65536.0 - (double)p.border)) : 0.f;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_error(scope.error, "hipSetDevice");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    ProfScope prof(profiler(ctx), "dropout", s);
    if (d.dtype == TRIPS_DTYPE_F32)
        launch<TRIPS_DTYPE_F32>(p, s);
    else if (d.dtype == TRIPS_DTYPE_BF16)
        launch<TRIPS_DTYPE_BF16>(p, s);
    else
        launch<TRIPS_DTYPE_F16>(p, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TRIPS_OK : hip_error(e, "dropout launch");
}
