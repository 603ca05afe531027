// Residual sum and norm, forward and backward:
//   r = residual + scale drop(x),  v = r - mean,  hat = v rstd,  y = hat weight + bias;
//   g = dy weight,  dv = rstd (g - hat mean(g hat)) (- its mean over the row for the layer norm),  dr = dv + dr_out,
//   dresidual = dr,  dx = scale drop(dr),  dweight = sum dy hat,  dbias = sum dy,  dscale = sum dr drop(x)   (sums over rows).
// HBM-bound: every tensor once.  The norm reads r as it is kept (rounded to r's type), which is also what the backward pass reads: the
// gradient is that of the values that were computed.  The dropout mask is formed again from its counter.  bf16 onto an fp32 residual,
// forward / backward: 16384 x 1024 35 / 66 us (5.8 / 4.6 TB/s), 6000 x 500 with scale and dropout 11.2 / 15.6; above 8192 columns the backward kernel
// spills 120 to 240 registers: 2048 x 16384 87 / 324.
#include "norm_rows.h"
#include "philox.h"

namespace {

struct Drop { unsigned thr; float factor; int64_t seed, offset; const int64_t* d_seed; };

// Rows of 513 to 1024 columns all in 16 bits are held to six waves a SIMD: left alone they take two registers more than those have, and
// 16384 x 1000 takes 27.2 us instead of 26.3.
template <class R, int TPR, int NV, bool VEC> constexpr int residual_fwd_waves() { return sizeof(R) == 2 && NV == 4 && TPR == 64 && VEC ? 6 : 1; }

template <class T, class R, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, (residual_fwd_waves<R, TPR, NV, VEC>())) void residual_fwd_kernel(int64_t rows, int C, const T* __restrict__ x, int64_t x_ld,
                                                                              const R* __restrict__ res, int64_t res_ld, const float* __restrict__ w,
                                                                              const float* __restrict__ b, const float* __restrict__ sc, float eps, int layer,
                                                                              Drop dr, int64_t* __restrict__ used, T* __restrict__ y, R* __restrict__ r_out,
                                                                              float* __restrict__ stat) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float s[TPR / 64][2];
    const int l = threadIdx.x % TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float inv = 1.f / (float)C;
    const f32x4 one = {1.f, 1.f, 1.f, 1.f}, zero = {0.f, 0.f, 0.f, 0.f};
    const DropKey key = drop_key(dr.seed, dr.offset, dr.thr ? dr.d_seed : nullptr);
    if (used && blockIdx.x == 0 && threadIdx.x == 0) {
        used[0] = (int64_t)(((unsigned long long)key.k1 << 32) | key.k0);
        used[1] = (int64_t)key.off;
    }
    int64_t row = (int64_t)blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / TPR : 0);
    RowRaw<T, NV> xn;
    RowRaw<R, NV> rn;
    auto load = [&](int64_t at) {
        xn.template load<TPR, VEC>(x + at * x_ld, C, l);
        if (res) rn.template load<TPR, VEC>(res + at * res_ld, C, l);
    };
    if (row < rows) load(row);
    for (; row < rows; row += step) {                 // (whole waves, and whole workgroups where a row is one's)
        f32x4 v[NV];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = C - c;
            v[i] = xn.get(i);
            if (dr.thr && n > 0) v[i] = drop4<VEC>(v[i], row * C + c, key, dr.thr, dr.factor);
            if (sc) v[i] *= load4n<float, VEC>(sc + c, n);
            if (res) v[i] += rn.get(i);
            if (r_out) {
                store4n<R, VEC>(r_out + row * C + c, v[i], n);
                v[i] = __builtin_convertvector(__builtin_convertvector(v[i], vec_t<R, 4>), f32x4);
            }
            s1 += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        }
        if (row_ahead<TPR, NV>() && row + step < rows) load(row + step);
        float mean = 0.f;
        if (layer) {
            row_sum2<TPR>(s1, s2, s);
            mean = s1 * inv;
        }
        s1 = s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {             // the mean is taken off first: no difference of large squares
                v[i][j] = row_col<TPR, NV>(i, l) + j < C ? v[i][j] - mean : 0.f;
                s1 = fmaf(v[i][j], v[i][j], s1);
            }
        row_sum2<TPR>(s1, s2, s);
        const float rstd = row_rstd<TPR>(v, s1, inv, eps, s);
        if (stat && l == 0) {
            stat[2 * row] = mean;
            stat[2 * row + 1] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = C - c;
            f32x4 o;
            const f32x4 wv = w ? load4n<float, VEC>(w + c, n) : one, bv = b ? load4n<float, VEC>(b + c, n) : zero;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(v[i][j] * rstd, wv[j], bv[j]);
            store4n<T, VEC>(y + row * C + c, o, n);
        }
        if (!row_ahead<TPR, NV>() && row + step < rows) load(row + step);
    }
}

template <class T, class R, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void residual_bwd_kernel(int64_t rows, int C, const T* __restrict__ dy, int64_t dy_ld,
                                                                              const R* __restrict__ dro, int64_t dr_ld, const R* __restrict__ r,
                                                                              int64_t r_ld, const T* __restrict__ x, int64_t x_ld,
                                                                              const float* __restrict__ stat, const float* __restrict__ w,
                                                                              const float* __restrict__ sc, int layer, Drop dr, T* __restrict__ dx,
                                                                              R* __restrict__ dres, float* __restrict__ part, int want_x) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float s[TPR / 64][2];
    __shared__ __align__(16) float cols[TPR == 64 ? 4 * NV * 256 : 4];
    const int l = threadIdx.x % TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const DropKey key = drop_key(dr.seed, dr.offset, dr.thr ? dr.d_seed : nullptr);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, one = {1.f, 1.f, 1.f, 1.f};
    f32x4 aw[NV], ab[NV], as[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) aw[i] = ab[i] = as[i] = zero;
    const float inv = 1.f / (float)C;
    int64_t row = (int64_t)blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / TPR : 0);
    RowRaw<T, NV> gn, xn;
    RowRaw<R, NV> kn, dn;
    float mean = 0.f, rstd = 0.f;
    auto load = [&](int64_t at) {
        if (dy) gn.template load<TPR, VEC>(dy + at * dy_ld, C, l);
        kn.template load<TPR, VEC>(r + at * r_ld, C, l);
        if (dro) dn.template load<TPR, VEC>(dro + at * dr_ld, C, l);
        if (want_x) xn.template load<TPR, VEC>(x + at * x_ld, C, l);
        mean = stat[2 * at];
        rstd = stat[2 * at + 1];
    };
    if (row < rows) load(row);
    for (; row < rows; row += step) {
        f32x4 g[NV], hat[NV];
        float s1 = 0.f, s2 = 0.f;
        const float rs = rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = C - c;
            g[i] = dy ? gn.get(i) : zero;
            hat[i] = kn.get(i);
            const f32x4 wv = w ? load4n<float, VEC>(w + c, n) : one;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hat[i][j] = j < n ? (hat[i][j] - mean) * rs : 0.f;
                aw[i][j] = fmaf(g[i][j], hat[i][j], aw[i][j]);
                ab[i][j] += g[i][j];
                g[i][j] *= wv[j];
                s1 = fmaf(g[i][j], hat[i][j], s1);
                s2 += g[i][j];
            }
        }
        const RowRaw<R, NV> dv = dn;
        const RowRaw<T, NV> xv = xn;
        if (row_ahead<TPR, NV>() && row + step < rows) load(row + step);
        row_sum2<TPR>(s1, s2, s);
        s1 *= inv;
        s2 = layer ? s2 * inv : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = C - c;
            f32x4 d = dro ? dv.get(i) : zero;
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = fmaf(rs, fmaf(-hat[i][j], s1, g[i][j] - s2), d[j]);
            if (dres) store4n<R, VEC>(dres + row * C + c, d, n);
            if (n > 0) {
                // the same bits keep or drop x (for dscale) and the gradient
                f32x4 kept = one;
                if (dr.thr) kept = drop4<VEC>(one, row * C + c, key, dr.thr, dr.factor);
                if (want_x) {
                    const f32x4 xf = xv.get(i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) as[i][j] = j < n && kept[j] != 0.f ? fmaf(d[j], xf[j] * kept[j], as[i][j]) : as[i][j];
                }
                if (dx) {
                    if (sc) d *= load4n<float, VEC>(sc + c, n);
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] = kept[j] != 0.f ? d[j] * kept[j] : 0.f;
                    store4n<T, VEC>(dx + row * C + c, d, n);
                }
            }
        }
        if (!row_ahead<TPR, NV>() && row + step < rows) load(row + step);
    }
    if (part) {
        float* p = part + (int64_t)blockIdx.x * 3 * C;
        put_columns<TPR, NV>(aw, p, C, cols);
        put_columns<TPR, NV>(ab, p + C, C, cols);
        put_columns<TPR, NV>(as, p + 2 * C, C, cols);
    }
}

// workgroups of a backward pass: two a CU (their partial rows are 3 C sums each)
int bwd_blocks(int64_t R, int C) { return norm_blocks(R, C, 512); }

bool norm_args(const char* who, int dtype, int r_dtype, int64_t R, int C, int thr) {
    if (!aas_dt_ok(dtype) || !(r_dtype == dtype || r_dtype == AAS_DT_F32)) { aas_set_error("%s: dtype %d, r_dtype %d", who, dtype, r_dtype); return false; }
    if (R < 0 || C < 1 || C > NORM_MAX_C) { aas_set_error("%s: R = %lld, C = %d (1 to %d)", who, (long long)R, C, NORM_MAX_C); return false; }
    if (R > ((int64_t)1 << 31)) { aas_set_error("%s: R = %lld too large", who, (long long)R); return false; }
    if (thr < 0 || thr > 65536) { aas_set_error("%s: thr = %d", who, thr); return false; }
    return true;
}

#define AAS_NORM_TYPES(dtype, r_dtype, E, Q, ...)                                               \
    do {                                                                                        \
        if ((r_dtype) == AAS_DT_F32) { typedef float Q; AAS_DT_SWITCH(dtype, E, __VA_ARGS__) }   \
        else if ((dtype) == AAS_DT_BF16) { typedef bf16_t E; typedef bf16_t Q; __VA_ARGS__; }    \
        else { typedef f16_t E; typedef f16_t Q; __VA_ARGS__; }                                  \
    } while (0)

}  // namespace

extern "C" int aas_residual_norm_fwd(aasStream_t stream, int dtype, int r_dtype, int64_t R, int C, const void* x, int64_t x_ld, const void* residual,
                                     int64_t res_ld, const float* weight, const float* bias, const float* scale, float eps, int layer, int thr,
                                     int64_t seed, int64_t offset, const int64_t* d_seed, int64_t* seed_used, void* y, void* r, float* stat) {
    const char* who = "aas_residual_norm_fwd";
    if (!norm_args(who, dtype, r_dtype, R, C, thr)) return 1;
    AAS_CHECK(norm_eps_ok(eps), "%s: eps = %g", who, eps);
    if (R == 0) return 0;
    AAS_CHECK(x && y, "%s: null pointer", who);
    AAS_CHECK(r || (!residual && !scale && !thr && r_dtype == dtype), "%s: r is wanted", who);
    const int es = aas_dt_size(dtype), rs = aas_dt_size(r_dtype);
    const bool vec = C % 4 == 0 && x_ld % 4 == 0 && (!residual || res_ld % 4 == 0) && aas_aligned(x, 4 * es) && aas_aligned(y, 4 * es) &&
                     aas_aligned(residual, 4 * rs) && aas_aligned(r, 4 * rs) && aas_aligned(weight, 16) && aas_aligned(bias, 16) && aas_aligned(scale, 16);
    const Drop dr = {(unsigned)thr, drop_factor(thr), seed, offset, d_seed};
    const unsigned grid = (unsigned)norm_blocks(R, C, 2048);
#define GO(TPR, NV, VEC)                                                                                                                       \
    AAS_NORM_TYPES(dtype, r_dtype, E, Q,                                                                                                       \
                   hipLaunchKernelGGL((residual_fwd_kernel<E, Q, TPR, NV, VEC>), dim3(grid), dim3(TPR > 256 ? TPR : 256), 0, (hipStream_t)stream, \
                                      R, C, (const E*)x, x_ld, (const Q*)residual, res_ld, weight, bias, scale, eps, layer, dr, seed_used, (E*)y, \
                                      (Q*)r, stat))
    AAS_ROW_SWITCH(C, vec, GO);
#undef GO
    AAS_LAUNCH_CHECK(who);
    return 0;
}

extern "C" size_t aas_residual_norm_bwd_ws_bytes(int64_t R, int C) {
    if (R <= 0 || C <= 0) return 0;
    return (size_t)bwd_blocks(R, C) * 3 * C * sizeof(float);
}

extern "C" int aas_residual_norm_bwd(aasStream_t stream, int dtype, int r_dtype, int64_t R, int C, const void* dy, int64_t dy_ld, const void* dr_out,
                                     int64_t dr_ld, const void* r, int64_t r_ld, const void* x, int64_t x_ld, const float* stat, const float* weight,
                                     const float* scale, int layer, int thr, int64_t seed, int64_t offset, const int64_t* d_seed, void* dx,
                                     void* dresidual, float* dweight, float* dbias, float* dscale, void* ws) {
    const char* who = "aas_residual_norm_bwd";
    if (!norm_args(who, dtype, r_dtype, R, C, thr)) return 1;
    hipStream_t s = (hipStream_t)stream;
    const bool params = dweight || dbias || dscale;
    int P = 0;
    if (R > 0) {
        AAS_CHECK(r && stat && (x || !dscale) && (ws || !params), "%s: null pointer", who);
        const int es = aas_dt_size(dtype), rs = aas_dt_size(r_dtype);
        const bool vec = C % 4 == 0 && (!dy || dy_ld % 4 == 0) && (!dr_out || dr_ld % 4 == 0) && r_ld % 4 == 0 && (!dscale || x_ld % 4 == 0) &&
                         aas_aligned(dy, 4 * es) && aas_aligned(dr_out, 4 * rs) && aas_aligned(r, 4 * rs) && (!dscale || aas_aligned(x, 4 * es)) &&
                         aas_aligned(dx, 4 * es) && aas_aligned(dresidual, 4 * rs) && aas_aligned(weight, 16) && aas_aligned(scale, 16);
        const Drop dr = {(unsigned)thr, drop_factor(thr), seed, offset, d_seed};
        P = bwd_blocks(R, C);
        float* part = params ? (float*)ws : nullptr;
#define GO(TPR, NV, VEC)                                                                                                                           \
    AAS_NORM_TYPES(dtype, r_dtype, E, Q,                                                                                                           \
                   hipLaunchKernelGGL((residual_bwd_kernel<E, Q, TPR, NV, VEC>), dim3(P), dim3(TPR > 256 ? TPR : 256), 0, s, R, C, (const E*)dy,  \
                                      dy_ld, (const Q*)dr_out, dr_ld, (const Q*)r, r_ld, (const E*)x, x_ld, stat, weight, scale, layer, dr, (E*)dx, \
                                      (Q*)dresidual, part, dscale != nullptr))
        AAS_ROW_SWITCH(C, vec, GO);
#undef GO
        AAS_LAUNCH_CHECK(who);
    }
    if (!params) return 0;
    ColMap map = {{dweight, dbias, dscale, nullptr}, {C, C, C, 0}, 0, 3};
    return aas_sum_partials(s, (const float*)ws, P, 3 * C, map, who);
}
