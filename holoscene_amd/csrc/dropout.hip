// holoscene_amd/csrc/dropout.hip -- dropout whose mask is a function of (seed, call, element) and is never stored (gfx950):
//     y_i = keep_i ? s x_i : 0   (+ r_i),      keep_i = u_i >= t,   t = round(65536 p) = `drop`,   s = 65536 / (65536 - t),
// u_i = 16 bits of Philox-4x32-10 (philox.h): key = seed, counter = (i / 8, call), word (i % 8) / 2, low half first -- one generator call serves the
// eight elements of a thread's 16-byte access.  16 bits per element, not 32: ten rounds are 20 quarter-rate 32x32 multiplies, and at four elements per
// call they, not the memory, would bound the 16-bit types; the probability is p to within 2^-17 and the scale is that of the t actually used, so
// the expectation of y is exactly x.  The backward pass is the same launch on the gradient.  A dropped element is written as 0 (+ r_i) by
// selection, not by a product: what it held -- an infinity, a NaN -- is not read into the result.
// Bound by memory: 16 384 x 4 096 bf16 74 us with a residual (403 MB, 5.4 TB/s), 45 us without (268 MB, 6.0 TB/s; a large copy on the same card 5.0 TB/s).
#include "holoscene_hip.h"
#include "philox.h"
#include "row_types.h"

namespace {

using namespace hs_row;

template <typename T, bool RES>
__global__ __launch_bounds__(256) void k_dropout(const T *__restrict__ x, const T *__restrict__ res, T *__restrict__ y, int64_t n, uint32_t t, float scale,
                                                 const uint64_t *__restrict__ rng) {
    const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x, i0 = g * 8;
    if (i0 >= n) return;
    const uint64_t seed = rng[0], call = rng[1];
    const uint4 w = philox4x32_10(make_uint4((uint32_t)g, (uint32_t)(g >> 32), (uint32_t)call, (uint32_t)(call >> 32)), make_uint2((uint32_t)seed, (uint32_t)(seed >> 32)));
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    auto one = [&](int e, T xv, T rv) -> T {
        const bool keep = ((word[e >> 1] >> (16 * (e & 1))) & 0xffffu) >= t;
        float v = keep ? to_f32(xv) * scale : 0.f;
        if constexpr (RES) v += to_f32(rv);
        return from_f32<T>(v);
    };
    if (i0 + 8 <= n) {
        Loose<T, 8> a = *reinterpret_cast<const Loose<T, 8> *>(x + i0), r = a;
        if constexpr (RES) r = *reinterpret_cast<const Loose<T, 8> *>(res + i0);
#pragma unroll
        for (int e = 0; e < 8; e++) a.v[e] = one(e, a.v[e], r.v[e]);
        *reinterpret_cast<Loose<T, 8> *>(y + i0) = a;
    } else {
        for (int e = 0; i0 + e < n; e++) y[i0 + e] = one(e, x[i0 + e], RES ? res[i0 + e] : x[i0 + e]);
    }
}

}  // namespace

extern "C" int hs_dropout_rows(const void *x, const void *residual, void *y, int64_t n, int32_t dtype, int32_t drop, const uint64_t *rng, void *stream) {
    if (n < 0 || !hs_row::known_dtype(dtype) || drop < 0 || drop > 65536 || n / 2048 >= 0xffffff) return HS_ERR_ARG;
    if (n == 0) return HS_OK;
    if (!x || !y || !rng) return HS_ERR_NULL;
    const float scale = drop < 65536 ? (float)(65536.0 / (65536 - drop)) : 0.f;
    const unsigned blocks = (unsigned)((n + 2047) / 2048);
    HS_BY_DTYPE(dtype, {
        if (residual) k_dropout<T, true><<<blocks, 256, 0, (hipStream_t)stream>>>((const T *)x, (const T *)residual, (T *)y, n, (uint32_t)drop, scale, rng);
        else k_dropout<T, false><<<blocks, 256, 0, (hipStream_t)stream>>>((const T *)x, nullptr, (T *)y, n, (uint32_t)drop, scale, rng);
    });
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}
