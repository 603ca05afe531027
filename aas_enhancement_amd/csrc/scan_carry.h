// First launch of a scan whose time axis is split (ssm_scan.h): per chunk k and channel the sum of d, and what the chunk leaves behind when
// nothing comes in:
//   forward, all but the last:  h = exp(d A) h + d x B  from zero (chunk 0: from the given state) over the chunk's frames;
//   REV,     all but the first: c = exp(d A) (c + go C), from the last frame to the first: the gradient of the state in front of the chunk.
#pragma once
#include "ssm_scan.h"

namespace {

template <class T, int NG, bool VEC, bool REV>
__global__ __launch_bounds__(256) void scan_carry_kernel(ScanDev a, const float* __restrict__ state, const T* __restrict__ dy, int64_t dy_st, int64_t dy_sn,
                                                         float* __restrict__ ends, float* __restrict__ sums) {
    __shared__ __align__(16) float2 dd[2][SCAN_TT][SCAN_CH];          // d, and d x (REV: go)
    __shared__ __align__(16) float bs[2][SCAN_TT][NG * 16];
    const ScanBlock b = scan_block(a);
    const int k = blockIdx.y + (REV ? a.fine : 0), len = a.tiles_per_chunk / a.fine;
    const int tid = threadIdx.x, q = tid & 3, cw = tid >> 2;
    const int lr = tid >> 4, lc = (tid & 15) * 4, ln = b.cn - lc, ls = tid & 15;
    const int L = row_length(a.len, b.n, a.T);
    const bool on = cw < b.cn, svec = a.svec != 0;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const T* tp = (const T*)a.dt + b.n * a.dt_sn + b.c0;
    const T* vp = REV ? dy + b.n * dy_sn + b.c0 : (const T*)a.x + b.n * a.x_sn + b.c0;
    const T* zp = REV && a.z ? (const T*)a.z + b.n * a.z_sn + b.c0 : nullptr;
    const T* bp = REV ? (const T*)a.C + b.n * a.C_sn + b.grp * a.C_sg : (const T*)a.B + b.n * a.B_sn + b.grp * a.B_sg;
    const int64_t v_st = REV ? dy_st : a.x_st, b_st = REV ? a.C_st : a.B_st;
    const int64_t rows = (int64_t)a.N * a.Ch, ch = (int64_t)b.n * a.Ch + b.c0 + cw;

    f32x4 A2[NG], h[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int s0 = g * 16 + 4 * q;
        A2[g] = on ? scan_rates4(a.A + (int64_t)(b.c0 + cw) * a.S, s0, a.S, svec) : zero;
        h[g] = on && !REV && state && k == 0 ? scan_states4(state + ch * a.S, s0, a.S, svec) : zero;
    }
    const f32x4 bias = a.dt_bias ? load4n<float, false>(a.dt_bias + b.c0 + lc, ln) : zero;
    f32x4 tr, vr, zr = zero, sum = zero;
    float br[NG];
    const int tiles = (L + SCAN_TT - 1) / SCAN_TT, t0 = k * len;
    const int t1 = t0 + len < tiles ? t0 + len : tiles;
    auto tile_of = [&](int i) { return REV ? t1 - 1 - i : t0 + i; };
    const ScanCols<VEC> cols(lc, b.cn);
    auto load = [&](int tile) {                         // (a frame behind the row's end: its last one, dropped again in stage)
        const int f = tile * SCAN_TT + lr;
        const int64_t t = f < L ? f : L - 1;
        tr = cols.get(tp + t * a.dt_st);
        vr = cols.get(vp + t * v_st);
        if (zp) zr = cols.get(zp + t * a.z_st);
#pragma unroll
        for (int g = 0; g < NG; ++g) br[g] = (float)bp[t * b_st + (g * 16 + ls < a.S ? g * 16 + ls : 0)];
    };
    auto stage = [&](int tile, int u) {
        const bool live = tile * SCAN_TT + lr < L;      // behind the end: d = 0 leaves the state as it is
        const f32x4 d = cols.keep(scan_delta4(tr, bias, a.softplus), live);
        f32x4 v = cols.keep(vr, live);
        sum += d;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= REV ? (zp ? zr[i] * sigm(zr[i]) : 1.f) : d[i];
        if (REV) v = cols.keep(v, live);
        scan_stage(&dd[u][lr][lc], d, v);
#pragma unroll
        for (int g = 0; g < NG; ++g) bs[u][lr][g * 16 + ls] = live && g * 16 + ls < a.S ? br[g] : 0.f;
    };
    const int n = t1 - t0;
    if (n > 0) {
        load(tile_of(0));
        stage(tile_of(0), 0);
        if (n > 1) load(tile_of(1));
    }
    for (int i = 0; i < n; ++i) {
        const int u = i & 1;
        __syncthreads();                                // the tile is staged; everybody is through with the one before
#pragma unroll 4
        for (int r = 0; r < SCAN_TT; ++r) {
            const int t = REV ? SCAN_TT - 1 - r : r;
            const float2 d = dd[u][t][cw];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const f32x4 B = reinterpret_cast<const f32x4*>(bs[u][t])[g * 4 + q];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float e = __builtin_amdgcn_exp2f(d.x * A2[g][j]);
                    h[g][j] = REV ? e * fmaf(d.y, B[j], h[g][j]) : fmaf(e, h[g][j], d.y * B[j]);
                }
            }
        }
        if (i + 1 < n) {
            stage(tile_of(i + 1), u ^ 1);
            if (i + 2 < n) load(tile_of(i + 2));
        }
    }
    // (the last place of `ends` is no chunk's: a copy of the given state, which the main launch overwrites, for its first chunk)
    if (!REV && state && on && k == 0)
#pragma unroll
        for (int g = 0; g < NG; ++g)
            scan_put_states4(ends + (((int64_t)a.nchunk * a.fine - 1) * rows + ch) * a.S, g * 16 + 4 * q, a.S, svec, scan_states4(state + ch * a.S, g * 16 + 4 * q, a.S, svec));
    if (on)
#pragma unroll
        for (int g = 0; g < NG; ++g) scan_put_states4(ends + (k * rows + ch) * a.S, g * 16 + 4 * q, a.S, svec, h[g]);
    __syncthreads();
    float(*s)[SCAN_CH] = reinterpret_cast<float(*)[SCAN_CH]>(dd);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[lr][lc + i] = sum[i];
    __syncthreads();
    if (tid < b.cn) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < SCAN_TT; ++i) v += s[i][tid];
        sums[k * rows + (int64_t)b.n * a.Ch + b.c0 + tid] = v;
    }
}

template <class T, bool REV>
void launch_carry(hipStream_t s, const ScanDev& a, bool vec, const float* state, const void* dy, int64_t dy_st, int64_t dy_sn, float* ends, float* sums) {
    const dim3 grid((unsigned)((int64_t)a.N * a.nbg * a.G), (a.nchunk - 1) * a.fine);
#define AAS_GO(NG_)                                                                                                                               \
    do {                                                                                                                                          \
        if (vec) hipLaunchKernelGGL((scan_carry_kernel<T, NG_, true, REV>), grid, dim3(256), 0, s, a, state, (const T*)dy, dy_st, dy_sn, ends, sums);  \
        else hipLaunchKernelGGL((scan_carry_kernel<T, NG_, false, REV>), grid, dim3(256), 0, s, a, state, (const T*)dy, dy_st, dy_sn, ends, sums);     \
    } while (0)
    if (a.S <= 16) AAS_GO(1);
    else if (a.S <= 32) AAS_GO(2);
    else AAS_GO(4);
#undef AAS_GO
}

}  // namespace
