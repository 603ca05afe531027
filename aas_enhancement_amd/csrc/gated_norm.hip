// Root-mean-square norm with a gate, per group of cg channels, forward and backward.  With G = z sigmoid(z), G' its derivative:
//   norm_first = 0: v = x G, y = hat w;      norm_first = 1: v = x, y = hat w G;      hat = v rstd, rstd = 1 / sqrt(mean(v^2) + eps);
//   g = dy w (G),  dv = rstd (g - hat mean(g hat));   dx = dv G, dz = dv x G', dw = sum dy hat   |   dx = dv, dz = dy hat w G', dw = sum dy hat G.
// HBM-bound: every tensor once; the backward pass forms the statistics again from x and z, which it reads anyway.  16384 x 2048 in bf16,
// forward / backward: 41 / 73 us in 4 groups (4.9 / 4.6 TB/s; without the next row read ahead 52 / 102), 35 / 90 in one; above 8192 channels a group
// the backward kernel spills 27 to 52 registers: 2048 x 16384 38 / 252.
#include "norm_rows.h"

namespace {

// A row whose squares leave fp32's range (norm_rows.h), formed again from memory over what the kernel wrote: held on to, the row would cost the
// ordinary ones a wave a SIMD (16384 x 1024 in bf16: 22.0 us instead of 20.8).
template <class T, int TPR, int NV, bool VEC, bool FIRST>
__device__ __forceinline__ void gated_row_scaled(const T* x, const T* z, const float* w, T* y, int cg, int l, float scale, float inv, float eps, float (*s)[2]) {
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 1
    for (int i = 0; i < NV; ++i) {
        const int c = row_col<TPR, NV>(i, l), n = cg - c;
        f32x4 v = load4n<T, VEC>(x + c, n), gt = load4n<T, VEC>(z + c, n);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!FIRST) v[j] *= gt[j] * sigm(gt[j]);
            v[j] *= scale;
            s1 = fmaf(v[j], v[j], s1);
        }
    }
    row_sum2<TPR>(s1, s2, s);
    const float rstd = __builtin_amdgcn_rsqf(fmaf(s1, inv, eps * scale * scale)) * scale;
#pragma unroll 1
    for (int i = 0; i < NV; ++i) {
        const int c = row_col<TPR, NV>(i, l), n = cg - c;
        f32x4 v = load4n<T, VEC>(x + c, n), gt = load4n<T, VEC>(z + c, n);
        const f32x4 wv = w ? load4n<float, VEC>(w + c, n) : f32x4{1.f, 1.f, 1.f, 1.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            gt[j] *= sigm(gt[j]);
            v[j] = (FIRST ? v[j] : v[j] * gt[j]) * rstd * wv[j];
            if (FIRST) v[j] *= gt[j];
        }
        store4n<T, VEC>(y + c, v, n);
    }
}

// (the gate behind the norm: 75 registers where 72 make seven waves a SIMD, and nothing spills when held to them)
template <class T, int TPR, int NV, bool VEC, bool FIRST> constexpr int gated_fwd_waves() {
    return sizeof(T) == 2 && NV == 4 && TPR == 64 && VEC && FIRST ? 7 : 1;
}

template <class T, int TPR, int NV, bool VEC, bool FIRST>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, (gated_fwd_waves<T, TPR, NV, VEC, FIRST>())) void gated_fwd_kernel(int64_t rows, int C, int cg, const T* __restrict__ x, int64_t x_ld,
                                                                           const T* __restrict__ z, int64_t z_ld, const float* __restrict__ w, float eps,
                                                                           T* __restrict__ y) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float s[TPR / 64][2];
    const int l = threadIdx.x % TPR, base = blockIdx.y * cg;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float inv = 1.f / (float)cg;
    int64_t row = (int64_t)blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / TPR : 0);
    x += base;
    z += base;
    RowRaw<T, NV> xn, zn;
    if (row < rows) {
        xn.template load<TPR, VEC>(x + row * x_ld, cg, l);
        zn.template load<TPR, VEC>(z + row * z_ld, cg, l);
    }
    for (; row < rows; row += step) {                 // (whole waves, and whole workgroups where a row is one's)
        f32x4 v[NV], gt[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = xn.get(i);
            gt[i] = zn.get(i);
        }
        const bool more = row + step < rows;
        if (row_ahead<TPR, NV>() && more) {
            xn.template load<TPR, VEC>(x + (row + step) * x_ld, cg, l);
            zn.template load<TPR, VEC>(z + (row + step) * z_ld, cg, l);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)                  // (beyond the row x and z are zeros, and so is everything made of them)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                gt[i][j] *= sigm(gt[i][j]);
                if (!FIRST) v[i][j] *= gt[i][j];
                s1 = fmaf(v[i][j], v[i][j], s1);
            }
        row_sum2<TPR>(s1, s2, s);
        const float ms = fmaf(s1, inv, eps), rescale = row_rescale(ms), rstd = __builtin_amdgcn_rsqf(ms);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = cg - c;
            const f32x4 wv = w ? load4n<float, VEC>(w + base + c, n) : f32x4{1.f, 1.f, 1.f, 1.f};
            f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = v[i][j] * rstd * wv[j];
                if (FIRST) o[j] *= gt[i][j];
            }
            store4n<T, VEC>(y + row * C + base + c, o, n);
        }
        if (rescale != 0.f) {
            gated_row_scaled<T, TPR, NV, VEC, FIRST>(x + row * x_ld, z + row * z_ld, w ? w + base : nullptr, y + row * C + base, cg, l, rescale, inv, eps, s);
        }
        if (!row_ahead<TPR, NV>() && more) {
            xn.template load<TPR, VEC>(x + (row + step) * x_ld, cg, l);
            zn.template load<TPR, VEC>(z + (row + step) * z_ld, cg, l);
        }
    }
}

// (the same of the backward kernel's element-wise form: 170 registers where 168 make three waves; 6000 x 501 in bf16: 43 us with two, 39.5 with three)
template <class T, int TPR, int NV, bool VEC, bool FIRST> constexpr int gated_bwd_waves() {
    return sizeof(T) == 2 && NV == 4 && TPR == 64 && !VEC && FIRST ? 3 : 1;
}

template <class T, int TPR, int NV, bool VEC, bool FIRST>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, (gated_bwd_waves<T, TPR, NV, VEC, FIRST>())) void gated_bwd_kernel(int64_t rows, int C, int cg, const T* __restrict__ dy, int64_t dy_ld,
                                                                           const T* __restrict__ x, int64_t x_ld, const T* __restrict__ z, int64_t z_ld,
                                                                           const float* __restrict__ w, float eps, T* __restrict__ dx, T* __restrict__ dz,
                                                                           float* __restrict__ part) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    __shared__ float s[TPR / 64][2];
    __shared__ __align__(16) float cols[TPR == 64 ? 4 * NV * 256 : 4];
    const int l = threadIdx.x % TPR, base = blockIdx.y * cg;           // a workgroup stays in one group: its threads own columns
    const int64_t step = (int64_t)gridDim.x * RPB;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, one = {1.f, 1.f, 1.f, 1.f};
    f32x4 aw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) aw[i] = zero;
    const float inv = 1.f / (float)cg;
    int64_t row = (int64_t)blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / TPR : 0);
    x += base;
    z += base;
    dy += base;
    RowRaw<T, NV> xn, zn, gn;
    auto load = [&](int64_t r) {
        xn.template load<TPR, VEC>(x + r * x_ld, cg, l);
        zn.template load<TPR, VEC>(z + r * z_ld, cg, l);
        gn.template load<TPR, VEC>(dy + r * dy_ld, cg, l);
    };
    if (row < rows) load(row);
    for (; row < rows; row += step) {
        const RowRaw<T, NV> xv = xn, zv = zn, gv = gn;
        if (row_ahead<TPR, NV>() && row + step < rows) load(row + step);
        float s1 = 0.f, s2 = 0.f;
        f32x4 sg[NV];                                                  // sigmoid of the gate
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = cg - c;
            const f32x4 wv = w ? load4n<float, VEC>(w + base + c, n) : one, xf = xv.get(i), zf = zv.get(i), gf = gv.get(i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sg[i][j] = sigm(zf[j]);
                const float gt = zf[j] * sg[i][j];
                const float v = FIRST ? xf[j] : xf[j] * gt;
                const float g = FIRST ? gf[j] * wv[j] * gt : gf[j] * wv[j];
                s1 = fmaf(v, v, s1);
                s2 = fmaf(g, v, s2);
            }
        }
        row_sum2<TPR>(s1, s2, s);
        float rstd = fmaf(s1, inv, eps), m = s2 * inv;                                       // mean(v^2) + eps, mean(g v)
        const float c = row_rescale(rstd);
        if (c != 0.f) {                                                                      // (norm_rows.h: both sums again, of v c)
            s1 = s2 = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = row_col<TPR, NV>(i, l);
                const f32x4 wv = w ? load4n<float, VEC>(w + base + col, cg - col) : one, xf = xv.get(i), zf = zv.get(i), gf = gv.get(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float gt = zf[j] * sg[i][j], u = (FIRST ? xf[j] : xf[j] * gt) * c;
                    s1 = fmaf(u, u, s1);
                    s2 = fmaf(FIRST ? gf[j] * wv[j] * gt : gf[j] * wv[j], u, s2);
                }
            }
            row_sum2<TPR>(s1, s2, s);
            rstd = fmaf(s1, inv, eps * c * c);
            m = s2 * inv;
        }
        rstd = __builtin_amdgcn_rsqf(rstd);
        m *= rstd;                                                                           // mean(g hat)
        if (c != 0.f) rstd *= c;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = cg - c;
            const f32x4 wv = w ? load4n<float, VEC>(w + base + c, n) : one, xf = xv.get(i), zf = zv.get(i), gf = gv.get(i);
            f32x4 ox, oz;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float sj = sg[i][j], gt = zf[j] * sj, slope = sj * fmaf(zf[j], 1.f - sj, 1.f);
                const float hat = (FIRST ? xf[j] : xf[j] * gt) * rstd;
                const float g = FIRST ? gf[j] * wv[j] * gt : gf[j] * wv[j];
                const float dv = rstd * fmaf(-hat, m, g);
                ox[j] = FIRST ? dv : dv * gt;
                oz[j] = FIRST ? gf[j] * hat * wv[j] * slope : dv * xf[j] * slope;
                aw[i][j] = fmaf(gf[j], FIRST ? hat * gt : hat, aw[i][j]);
            }
            const int64_t at = row * C + base + c;
            if (dx) store4n<T, VEC>(dx + at, ox, n);
            if (dz) store4n<T, VEC>(dz + at, oz, n);
        }
        if (!row_ahead<TPR, NV>() && row + step < rows) load(row + step);
    }
    if (part) put_columns<TPR, NV>(aw, part + (int64_t)blockIdx.x * C + base, cg, cols);
}

// workgroups a group: about eight a CU in all forward, four backward, where each leaves a partial row of sums (at 8192 x 8192 in bf16: 224 us
// against 257 with eight)
int gated_blocks(int64_t R, int C, int groups, int most) { return norm_blocks(R, C / groups, groups >= most ? 1 : most / groups); }
constexpr int FWD_MOST = 2048, BWD_MOST = 1024;

bool gated_args(const char* who, int dtype, int64_t R, int C, int groups, float eps) {
    if (!norm_eps_ok(eps)) { aas_set_error("%s: eps = %g", who, eps); return false; }
    if (!aas_dt_ok(dtype)) { aas_set_error("%s: dtype %d", who, dtype); return false; }
    if (R < 0 || C < 1 || groups < 1 || C % groups) { aas_set_error("%s: R = %lld, C = %d, groups = %d", who, (long long)R, C, groups); return false; }
    if (C / groups > NORM_MAX_C) { aas_set_error("%s: %d channels a group, at most %d", who, C / groups, NORM_MAX_C); return false; }
    if (groups > 65535 || R > 0x7fffffff / groups) { aas_set_error("%s: R = %lld, groups = %d too large", who, (long long)R, groups); return false; }
    return true;
}

}  // namespace

extern "C" int aas_gated_norm_fwd(aasStream_t stream, int dtype, int64_t R, int C, int groups, const void* x, int64_t x_ld, const void* gate,
                                  int64_t gate_ld, const float* weight, float eps, int norm_first, void* y) {
    const char* who = "aas_gated_norm_fwd";
    if (!gated_args(who, dtype, R, C, groups, eps)) return 1;
    if (R == 0) return 0;
    AAS_CHECK(x && gate && y, "%s: null pointer", who);
    const int es = aas_dt_size(dtype), cg = C / groups;
    const bool vec = cg % 4 == 0 && x_ld % 4 == 0 && gate_ld % 4 == 0 && aas_aligned(x, 4 * es) && aas_aligned(gate, 4 * es) && aas_aligned(y, 4 * es) &&
                     aas_aligned(weight, 16);
    const dim3 grid(gated_blocks(R, C, groups, FWD_MOST), groups);
#define GO1(TPR, NV, VEC, FIRST)                                                                                                                  \
    AAS_DT_SWITCH(dtype, E, hipLaunchKernelGGL((gated_fwd_kernel<E, TPR, NV, VEC, FIRST>), grid, dim3(TPR > 256 ? TPR : 256), 0,                 \
                                               (hipStream_t)stream, R, C, cg, (const E*)x, x_ld, (const E*)gate, gate_ld, weight, eps, (E*)y))
#define GO(TPR, NV, VEC) if (norm_first) { GO1(TPR, NV, VEC, true) } else { GO1(TPR, NV, VEC, false) }
    AAS_ROW_SWITCH(cg, vec, GO);
#undef GO
#undef GO1
    AAS_LAUNCH_CHECK(who);
    return 0;
}

extern "C" size_t aas_gated_norm_bwd_ws_bytes(int64_t R, int C, int groups) {
    if (R <= 0 || C <= 0 || groups <= 0 || C % groups) return 0;
    return (size_t)gated_blocks(R, C, groups, BWD_MOST) * C * sizeof(float);
}

extern "C" int aas_gated_norm_bwd(aasStream_t stream, int dtype, int64_t R, int C, int groups, const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                  const void* gate, int64_t gate_ld, const float* weight, float eps, int norm_first, void* dx, void* dgate,
                                  float* dweight, void* ws) {
    const char* who = "aas_gated_norm_bwd";
    if (!gated_args(who, dtype, R, C, groups, eps)) return 1;
    // (the launch that sums dweight has a workgroup of 256 per 16 columns, and fewer than 2^32 threads)
    AAS_CHECK(!dweight || cdiv(C, 16) < (1 << 24), "%s: C = %d too large for a weight's gradient", who, C);
    hipStream_t s = (hipStream_t)stream;
    int P = 0;
    if (R > 0) {
        AAS_CHECK(dy && x && gate && (ws || !dweight), "%s: null pointer", who);
        const int es = aas_dt_size(dtype), cg = C / groups;
        const bool vec = cg % 4 == 0 && dy_ld % 4 == 0 && x_ld % 4 == 0 && gate_ld % 4 == 0 && aas_aligned(dy, 4 * es) && aas_aligned(x, 4 * es) &&
                         aas_aligned(gate, 4 * es) && aas_aligned(dx, 4 * es) && aas_aligned(dgate, 4 * es) && aas_aligned(weight, 16);
        P = gated_blocks(R, C, groups, BWD_MOST);
        float* part = dweight ? (float*)ws : nullptr;
#define GO1(TPR, NV, VEC, FIRST)                                                                                                                       \
    AAS_DT_SWITCH(dtype, E, hipLaunchKernelGGL((gated_bwd_kernel<E, TPR, NV, VEC, FIRST>), dim3(P, groups), dim3(TPR > 256 ? TPR : 256), 0, s, R, C,  \
                                               cg, (const E*)dy, dy_ld, (const E*)x, x_ld, (const E*)gate, gate_ld, weight, eps, (E*)dx, (E*)dgate, part))
#define GO(TPR, NV, VEC) if (norm_first) { GO1(TPR, NV, VEC, true) } else { GO1(TPR, NV, VEC, false) }
        AAS_ROW_SWITCH(cg, vec, GO);
#undef GO
#undef GO1
        AAS_LAUNCH_CHECK(who);
    }
    if (!dweight) return 0;
    ColMap map = {{dweight, nullptr, nullptr, nullptr}, {C, 0, 0, 0}, 0, 1};
    return aas_sum_partials(s, (const float*)ws, P, C, map, who);
}
