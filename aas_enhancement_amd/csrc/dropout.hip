// Dropout from a counter-based generator (philox.h): y = x / (1 - p) where an element is kept, 0 where it is not.  HBM-bound: a thread
// takes the eight elements of one counter (67 M elements: 5.4 TB/s in fp32, 6.5 in bf16 partly from cache; a 1 GiB copy does 5.1).
#include "philox.h"

namespace {

template <class T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t n, unsigned thr, float factor, int64_t seed,
                                                      int64_t offset, const int64_t* __restrict__ d_seed, int64_t* __restrict__ used) {
    const DropKey key = drop_key(seed, offset, d_seed);
    if (used && blockIdx.x == 0 && threadIdx.x == 0) {
        used[0] = (int64_t)(((unsigned long long)key.k1 << 32) | key.k0);
        used[1] = (int64_t)key.off;
    }
    const int64_t groups = (n + 7) / 8;
    for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
        const U4 u = philox(key, (unsigned long long)g);
        const int64_t e = g * 8;
        const T* xp = x + e;
        T* yp = y + e;
        if (VEC && e + 8 <= n) {
            typedef vec_t<T, 16 / sizeof(T)> V;       // 16 bytes
            constexpr int NV = 8 * sizeof(T) / 16, W = 16 / sizeof(T);
            V v[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = reinterpret_cast<const V*>(xp)[i];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float f = half_of(u, i * W + j) >= thr ? (float)v[i][j] * factor : 0.f;
                    v[i][j] = (T)f;
                }
                reinterpret_cast<V*>(yp)[i] = v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e + i < n) yp[i] = (T)(half_of(u, i) >= thr ? (float)xp[i] * factor : 0.f);
        }
    }
}

}  // namespace

extern "C" int aas_dropout(aasStream_t stream, int dtype, int64_t n, const void* x, void* y, int thr, int64_t seed, int64_t offset,
                           const int64_t* d_seed, int64_t* seed_used) {
    AAS_CHECK(aas_dt_ok(dtype), "aas_dropout: dtype %d", dtype);
    AAS_CHECK(n >= 0 && thr >= 0 && thr <= 65536, "aas_dropout: n = %lld, thr = %d", (long long)n, thr);
    if (n == 0 && !seed_used) return 0;
    AAS_CHECK(n == 0 || (x && y), "aas_dropout: null pointer");
    const bool vec = aas_aligned(x, 16) && aas_aligned(y, 16);
    const int64_t blocks = (n + 2047) / 2048;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks < 8192 ? blocks : 8192));
    const float f = drop_factor(thr);
    AAS_DT_SWITCH(dtype, E, {
        if (vec) hipLaunchKernelGGL((dropout_kernel<E, true>), grid, dim3(256), 0, (hipStream_t)stream, (const E*)x, (E*)y, n, (unsigned)thr, f, seed, offset, d_seed, seed_used);
        else hipLaunchKernelGGL((dropout_kernel<E, false>), grid, dim3(256), 0, (hipStream_t)stream, (const E*)x, (E*)y, n, (unsigned)thr, f, seed, offset, d_seed, seed_used);
    });
    AAS_LAUNCH_CHECK("aas_dropout");
    return 0;
}
