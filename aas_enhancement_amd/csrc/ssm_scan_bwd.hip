// Selective state space scan, backward (ssm_scan.h has the layout).  With go = dy z sigmoid(z) and g_s[t] the gradient of h_s[t]:
//
//   g_s[t] = C_s go + a_s[t+1] g_s[t+1],  a_s = exp(d A_s),     p_s = a_s h_s[t-1],  q_s = g_s p_s,
//   u = sum_s g_s B_s,  w = sum_s q_s A_s:   dx = D go + d u,   dd = w + x u,   ddt = dd softplus',   dz = dy o (z sigmoid(z))',
//   dA_s = sum_{t,n} q_s d,   dB_s = sum_c g_s d x,   dC_s = sum_c go h_s,   dD = sum go x,   ddt_bias = sum ddt.
//
// Tiles of 16 frames from the last to the first, in runs of 8: a lane goes forward from the state that the forward pass kept in front of
// the run, holding a and p of its frames in registers, then back through them.  (States kept every 16 frames and the exponentials
// formed twice was 289 us where this was 275, at 4096 x 4 x 1024 in bf16; now 258 to 273, at 200 x 30 x 1000 in fp32 95.  All 16 frames' a and p
// do not fit the registers.)  Bound by instruction issue (105 a frame and wave, VALU active in 79 % of the busy cycles) at two waves a
// SIMD; held to three by launch bounds it spills: 561 us, and with a thread's own elements parked in LDS, where it nearly fits, three waves
// were no faster (pass 578 us against 507).  Above 16 states there is one wave a SIMD (256 registers and 8 to 100 more of the accumulators'):
// 1000 x 8 x 512 in bf16 takes 108, 244 and 450 us with 16, 32 and 64 states.  dB and dC are sums over channels: eight values a lane (four
// states x {dB, dC}) over the 16 channels of a wave go by exchanges that halve the number of values with the number of lanes still to
// add (lane halves, rows of 16, then within the row), then over the four waves through LDS, then - plain stores, no atomics - over the
// workgroups by a second launch.
#include "scan_carry.h"

namespace {

__device__ __forceinline__ float add_halves(float a, float b) {         // lanes 0-31: a summed over the halves; lanes 32-63: b
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_rows(float a, float b) {           // rows 0, 2 of 16 lanes: a summed over row pairs; rows 1, 3: b
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int ROW_ROR_4 = 0x124, ROW_ROR_8 = 0x128;

// v[0..7] summed over the 16 channels of the wave (lane bits 2 .. 5); the lane is left with the sum of value
// (bit 5) + 2 (bit 4) + 4 (bit 3) of its lane number
__device__ __forceinline__ float sum_channels8(const float v[8], bool bit3) {
    const float a = add_rows(add_halves(v[0], v[1]), add_halves(v[2], v[3]));
    const float b = add_rows(add_halves(v[4], v[5]), add_halves(v[6], v[7]));
    const float a1 = add_dpp<ROW_ROR_4>(add_dpp<ROW_ROR_8>(a)), b1 = add_dpp<ROW_ROR_4>(add_dpp<ROW_ROR_8>(b));
    return bit3 ? b1 : a1;
}

template <class T, int NG, bool VEC>
__global__ __launch_bounds__(256) void scan_bwd_kernel(ScanDev a, const T* __restrict__ dy, int64_t dy_st, int64_t dy_sn, const float* __restrict__ hsave,
                                                       T* __restrict__ dx, T* __restrict__ ddt, T* __restrict__ dz, float* __restrict__ part_bc,
                                                       float* __restrict__ part_a, float* __restrict__ part_d,
                                                       const float* __restrict__ ends, const float* __restrict__ sums) {
    __shared__ __align__(16) float2 dd[SCAN_TT][SCAN_CH];             // d, d x
    __shared__ __align__(16) float go[SCAN_TT][SCAN_CH];
    __shared__ __align__(16) float bs[SCAN_TT][NG * 16], cs[SCAN_TT][NG * 16];
    __shared__ __align__(16) float us[SCAN_TT][SCAN_YP], ws[SCAN_TT][SCAN_YP], os[SCAN_TT][SCAN_YP];
    __shared__ float bc[4][SCAN_TT][NG * 32];           // per wave, frame: dB of the 16 NG states, dC
    const ScanBlock b = scan_block(a);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = tid & 3, cw = tid >> 2;
    const int lr = tid >> 4, lc = (tid & 15) * 4, ln = b.cn - lc, ls = tid & 15;
    const int L = row_length(a.len, b.n, a.T);
    const bool on = cw < b.cn, svec = a.svec != 0;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const T* xp = (const T*)a.x + b.n * a.x_sn + b.c0;
    const T* tp = (const T*)a.dt + b.n * a.dt_sn + b.c0;
    const T* zp = a.z ? (const T*)a.z + b.n * a.z_sn + b.c0 : nullptr;
    const T* gp = dy + b.n * dy_sn + b.c0;
    const T* bp = (const T*)a.B + b.n * a.B_sn + b.grp * a.B_sg;
    const T* cp = (const T*)a.C + b.n * a.C_sn + b.grp * a.C_sg;
    const int64_t srow = ((int64_t)b.n * a.Ch + b.c0 + cw) * a.S;

    f32x4 A2[NG], dA[NG], carry[NG];                                    // carry = a[t+1] g[t+1]
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        A2[g] = on ? scan_rates4(a.A + (int64_t)(b.c0 + cw) * a.S, g * 16 + 4 * q, a.S, svec) : zero;
        dA[g] = carry[g] = zero;
    }
    const int chunk = blockIdx.y;
    if (on && chunk + 1 < a.nchunk)
        scan_fold<NG, true>(carry, A2, ends, sums, chunk * a.fine + a.fine - 1, a.nchunk * a.fine, (int64_t)a.N * a.Ch, (int64_t)b.n * a.Ch + b.c0 + cw, a.S, q, svec, a.softplus != 0);
    const f32x4 bias = a.dt_bias ? load4n<float, false>(a.dt_bias + b.c0 + lc, ln) : zero;
    const f32x4 Dv = a.D ? load4n<float, false>(a.D + b.c0 + lc, ln) : zero;
    f32x4 dD = zero, dbias = zero;

    constexpr int HALVES = SCAN_TT / SCAN_HT;
    f32x4 xr, tr, zr = zero, gr, h0[HALVES][NG];
    float br[NG], cr[NG];
    const ScanCols<VEC> cols(lc, b.cn);
    auto load = [&](int tile) {                                         // (a frame behind the row's end: its last one, dropped again below)
        const int f = tile * SCAN_TT + lr;
        const int64_t t = f < L ? f : L - 1;
        xr = cols.get(xp + t * a.x_st);
        tr = cols.get(tp + t * a.dt_st);
        if (zp) zr = cols.get(zp + t * a.z_st);
        gr = cols.get(gp + t * dy_st);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int s = g * 16 + ls < a.S ? g * 16 + ls : 0;
            br[g] = (float)bp[t * a.B_st + s];
            cr[g] = (float)cp[t * a.C_st + s];
        }
#pragma unroll
        for (int i = 0; i < HALVES; ++i)
#pragma unroll
            for (int g = 0; g < NG; ++g)                                // (kept also where the row ends inside the tile)
                h0[i][g] = on ? scan_states4(hsave + ((int64_t)(tile * HALVES + i) * a.N * a.Ch) * a.S + srow, g * 16 + 4 * q, a.S, svec) : zero;
    };
    const int all = (L + SCAN_TT - 1) / SCAN_TT, k0 = chunk * a.tiles_per_chunk;
    const int k1 = k0 + a.tiles_per_chunk, tiles = k1 < all ? k1 : all;                       // tiles [k0, tiles) have frames, up to k1 are written
    const int64_t orow = (int64_t)a.N * a.Ch, obase = (int64_t)b.n * a.Ch + b.c0 + lc;
    const int nblk = a.nbg;
    const int cb = (b.c0 - b.grp * a.cpg) / SCAN_CH;
    if (tiles > k0) load(tiles - 1);
    for (int k = tiles - 1; k >= k0; --k) {
        const int64_t t = (int64_t)k * SCAN_TT + lr;
        const bool live = t < L;
        // this thread's elements: x, d, softplus', go, and what o is multiplied by for dz; zeros behind the end and beside the channels
        f32x4 slope;
        const f32x4 xe = cols.keep(xr, live), de = cols.keep(scan_delta4(tr, bias, a.softplus, slope), live);
        f32x4 oe = gr, gz = zero;
        if (zp) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float s = sigm(zr[i]);
                oe[i] = gr[i] * (zr[i] * s);
                gz[i] = gr[i] * (s * fmaf(zr[i], 1.f - s, 1.f));
            }
            gz = cols.keep(gz, live);
        }
        oe = cols.keep(oe, live);
        scan_stage(&dd[lr][lc], de, de * xe);
        *reinterpret_cast<f32x4*>(&go[lr][lc]) = oe;
        f32x4 h[HALVES][NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const bool in = live && g * 16 + ls < a.S;
            bs[lr][g * 16 + ls] = in ? br[g] : 0.f;
            cs[lr][g * 16 + ls] = in ? cr[g] : 0.f;
#pragma unroll
            for (int i = 0; i < HALVES; ++i) h[i][g] = h0[i][g];
        }
        if (k > k0) load(k - 1);
        __syncthreads();
#pragma unroll
        for (int half = HALVES - 1; half >= 0; --half) {
            constexpr int HT = SCAN_HT;
            const int t0 = half * HT;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 e[HT], p[HT], hh = h[half][g];                    // a, a h[t-1]
                float keep = 0.f;
#pragma unroll
                for (int i = 0; i < HT; ++i) {
                    const float2 d = dd[t0 + i][cw];
                    const f32x4 B = reinterpret_cast<const f32x4*>(bs[t0 + i])[g * 4 + q];
                    float acc = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        e[i][j] = __builtin_amdgcn_exp2f(d.x * A2[g][j]);
                        p[i][j] = e[i][j] * hh[j];
                        hh[j] = fmaf(d.y, B[j], p[i][j]);
                    }
                    const f32x4 C = reinterpret_cast<const f32x4*>(cs[t0 + i])[g * 4 + q];   // (o, wanted for dz; without z it costs a few per cent)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc = fmaf(hh[j], C[j], acc);
                    acc = quad_sum(acc);
                    keep = q == (i & 3) ? acc : keep;
                    if ((i & 3) == 3) {
                        float* o = &os[t0 + (i & ~3) + q][cw];
                        *o = g == 0 ? keep : *o + keep;
                    }
                    if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);
                }
                // B, C and d are read again (an address the compiler cannot match with the one above): kept from the run forward they would
                // be 80 registers more
                int ch = cw, sq = g * 4 + q;
                asm volatile("" : "+v"(ch), "+v"(sq));
                float ku = 0.f, kw = 0.f;
#pragma unroll
                for (int i = HT - 1; i >= 0; --i) {
                    const float2 d = dd[t0 + i][ch];
                    const float o = go[t0 + i][ch];
                    const f32x4 B = reinterpret_cast<const f32x4*>(bs[t0 + i])[sq];
                    const f32x4 C = reinterpret_cast<const f32x4*>(cs[t0 + i])[sq];
                    float u = 0.f, w = 0.f, v[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float gh = fmaf(C[j], o, carry[g][j]);
                        v[4 + j] = o * fmaf(d.y, B[j], p[i][j]);
                        v[j] = gh * d.y;
                        u = fmaf(gh, B[j], u);
                        const float r = gh * p[i][j];
                        w = fmaf(r, A2[g][j], w);
                        dA[g][j] = fmaf(r, d.x, dA[g][j]);
                        carry[g][j] = gh * e[i][j];
                    }
                    u = quad_sum(u);
                    w = quad_sum(w);
                    ku = q == (i & 3) ? u : ku;
                    kw = q == (i & 3) ? w : kw;
                    if ((i & 3) == 0) {
                        float *pu = &us[t0 + i + q][cw], *pw = &ws[t0 + i + q][cw];
                        *pu = g == 0 ? ku : *pu + ku;
                        *pw = g == 0 ? kw : *pw + kw;
                    }
                    asm volatile("" : "+v"(dA[g][0]), "+v"(dA[g][1]), "+v"(dA[g][2]), "+v"(dA[g][3]));   // added up here, not products kept for later
                    const float s = sum_channels8(v, (lane & 8) != 0);
                    if ((i & 3) == 0) __builtin_amdgcn_sched_barrier(0);           // (reads no further ahead: registers)
                    // value (bit 5) + 2 (bit 4) is the state of the quad, bit 3 says dB or dC; the lanes that differ in bit 2 hold the same
                    bc[wave][t0 + i][((lane & 8) ? NG * 16 : 0) + g * 16 + 4 * q + ((lane >> 5) & 1) + ((lane >> 3) & 2)] = s;
                }
            }
        }
        __syncthreads();
        if (t < a.T) {
            f32x4 vx, vt, vz;
            const f32x4 u = *reinterpret_cast<const f32x4*>(&us[lr][lc]), w = *reinterpret_cast<const f32x4*>(&ws[lr][lc]);
            const f32x4 o = *reinterpret_cast<const f32x4*>(&os[lr][lc]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vx[i] = fmaf(de[i], u[i], Dv[i] * oe[i]);
                vt[i] = fmaf(w[i], SCAN_LN2, xe[i] * u[i]) * slope[i];
                vz[i] = gz[i] * fmaf(Dv[i], xe[i], o[i]);
                dD[i] = fmaf(oe[i], xe[i], dD[i]);
            }
            vt = cols.keep(vt, live);                     // (zeros behind the end also where the row's state has overflowed: 0 inf is none)
            dbias += vt;
            const int64_t at = t * orow + obase;
            store4n<T, VEC>(dx + at, cols.keep(vx, live), ln);
            store4n<T, VEC>(ddt + at, vt, ln);
            if (dz) store4n<T, VEC>(dz + at, cols.keep(vz, live), ln);
        }
        // partial dB, dC of this workgroup: [T][N][G][nblk][2][S]
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) {
            const int e = tid + 256 * i, f = e / (NG * 32), j = e - f * (NG * 32);
            const int which = j >= NG * 16 ? 1 : 0, s = j - which * NG * 16;
            const int64_t tt = (int64_t)k * SCAN_TT + f;
            if (s < a.S && tt < L)
                part_bc[((((tt * a.N + b.n) * a.G + b.grp) * nblk + cb) * 2 + which) * a.S + s] =
                    (bc[0][f][j] + bc[1][f][j]) + (bc[2][f][j] + bc[3][f][j]);
        }
    }
    const int te = chunk + 1 == a.nchunk || (int64_t)k1 * SCAN_TT > a.T ? a.T : k1 * SCAN_TT;
    for (int64_t t = (int64_t)(tiles > k0 ? tiles : k0) * SCAN_TT + lr; t < te; t += SCAN_TT) {
        const int64_t at = t * orow + obase;
        store4n<T, VEC>(dx + at, zero, ln);
        store4n<T, VEC>(ddt + at, zero, ln);
        if (dz) store4n<T, VEC>(dz + at, zero, ln);
    }
    if (on)
#pragma unroll
        for (int g = 0; g < NG; ++g) scan_put_states4(part_a + (int64_t)chunk * a.N * a.Ch * a.S + srow, g * 16 + 4 * q, a.S, svec, dA[g]);
    __syncthreads();                                                    // (the last tile's readers of us, ws)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        us[lr][lc + i] = dD[i];
        ws[lr][lc + i] = dbias[i];
    }
    __syncthreads();
    if (tid < 2 * SCAN_CH) {
        const int c = tid & (SCAN_CH - 1);
        const float(*from)[SCAN_YP] = tid < SCAN_CH ? us : ws;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < SCAN_TT; ++i) v += from[i][c];
        if (c < b.cn) part_d[(((int64_t)chunk * a.N + b.n) * 2 + (tid >= SCAN_CH ? 1 : 0)) * a.Ch + b.c0 + c] = v;
    }
}

// The sums that cross workgroups, in one launch: workgroups [0, nbc) form dB and dC [T,N,G,S] from the partial sums of the group's
// workgroups (frames behind a row's end: zeros), the next `na` form dA, the rest dD and ddt_bias.
template <class T>
__global__ __launch_bounds__(256) void scan_finish_kernel(ScanDev a, const float* __restrict__ bc, const float* __restrict__ pa, const float* __restrict__ pd,
                                                          int P, int nbc, int na, T* __restrict__ dB, T* __restrict__ dC, ColMap ma, ColMap md) {
    if ((int)blockIdx.x >= nbc + na) return sum_columns(pd, P, 2 * a.Ch, md, blockIdx.x - nbc - na);
    if ((int)blockIdx.x >= nbc) return sum_columns(pa, P, a.Ch * a.S, ma, blockIdx.x - nbc);
    const int S2 = 2 * a.S;
    const int64_t total = (int64_t)a.T * a.N * a.G * S2;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)nbc * 256) {
        const int64_t row = e / S2;
        const int j = (int)(e - row * S2);
        const int64_t tn = row / a.G;
        float v = 0.f;
        if (tn / a.N < row_length(a.len, (int)(tn % a.N), a.T)) {
            const float* p = bc + row * a.nbg * S2 + j;
            int i = 0;
            for (; i + 4 <= a.nbg; i += 4) {
                const float p0 = p[(int64_t)i * S2], p1 = p[(int64_t)(i + 1) * S2], p2 = p[(int64_t)(i + 2) * S2], p3 = p[(int64_t)(i + 3) * S2];
                v += (p0 + p1) + (p2 + p3);
            }
            for (; i < a.nbg; ++i) v += p[(int64_t)i * S2];
        }
        if (j < a.S) dB[row * a.S + j] = (T)v;
        else dC[row * a.S + j - a.S] = (T)v;
    }
}

// Two workgroups a CU are resident (220 registers); twice as many even out the rows' lengths.  The carry launch needs a third of the
// registers and takes chunks of half the length (at 4096 x 4 x 1024: 71 us against 88 with the main launch's own).
constexpr int FINE = 2;
ScanChunks bwd_chunks(int T, int N, int Ch, int G) { return scan_chunks(T, N, Ch, G, 1024, FINE); }

struct BwdWs { size_t bc, a, d, ends, sums, total; };   // byte offsets
BwdWs bwd_ws(int T, int N, int Ch, int S, int G) {
    BwdWs w;
    const int n = bwd_chunks(T, N, Ch, G).n;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    w.bc = 0;
    w.a = up((size_t)T * N * G * cdiv(Ch / G, SCAN_CH) * 2 * S * sizeof(float));
    w.d = w.a + up((size_t)n * N * Ch * S * sizeof(float));
    w.ends = w.d + up((size_t)n * N * 2 * Ch * sizeof(float));
    w.sums = w.ends + (n > 1 ? up((size_t)n * FINE * N * Ch * S * sizeof(float)) : 0);
    w.total = w.sums + (n > 1 ? up((size_t)n * FINE * N * Ch * sizeof(float)) : 0);
    return w;
}

template <class T>
void launch_bwd(hipStream_t s, const ScanDev& a, bool vec, const void* dy, int64_t dy_st, int64_t dy_sn, const float* hsave, void* dx, void* ddt, void* dz,
                float* bc, float* pa, float* pd, float* ends, float* sums) {
    if (a.nchunk > 1) launch_carry<T, true>(s, a, vec, nullptr, dy, dy_st, dy_sn, ends, sums);
    const dim3 grid((unsigned)((int64_t)a.N * a.nbg * a.G), a.nchunk);
#define AAS_GO(NG_)                                                                                                                   \
    do {                                                                                                                              \
        if (vec)                                                                                                                      \
            hipLaunchKernelGGL((scan_bwd_kernel<T, NG_, true>), grid, dim3(256), 0, s, a, (const T*)dy, dy_st, dy_sn, hsave, (T*)dx,  \
                               (T*)ddt, (T*)dz, bc, pa, pd, ends, sums);                                                                          \
        else                                                                                                                          \
            hipLaunchKernelGGL((scan_bwd_kernel<T, NG_, false>), grid, dim3(256), 0, s, a, (const T*)dy, dy_st, dy_sn, hsave, (T*)dx, \
                               (T*)ddt, (T*)dz, bc, pa, pd, ends, sums);                                                                          \
    } while (0)
    if (a.S <= 16) AAS_GO(1);
    else if (a.S <= 32) AAS_GO(2);
    else AAS_GO(4);
#undef AAS_GO
}

}  // namespace

extern "C" size_t aas_ssm_scan_bwd_ws_bytes(int T, int N, int Ch, int S, int G) {
    if (T <= 0 || N <= 0 || Ch <= 0 || S <= 0 || G <= 0 || Ch % G) return 0;
    return bwd_ws(T, N, Ch, S, G).total;
}

extern "C" int aas_ssm_scan_bwd(aasStream_t stream, const aasScan* d, const void* dy, int64_t dy_st, int64_t dy_sn, const float* hsave, void* dx,
                                void* ddt, void* dz, void* dB, void* dC, float* dA, float* dD, float* ddt_bias, void* ws) {
    const char* who = "aas_ssm_scan_bwd";
    if (scan_check(who, d)) return 1;
    hipStream_t s = (hipStream_t)stream;
    const bool empty = d->T == 0 || d->N == 0;
    const int64_t want = ((int64_t)d->T * d->N * d->G * 2 * d->S + 255) / 256;
    const int nbc = (int)(want < 8192 ? want : 8192);
    if (d->Ch == 0) {                                     // dB and dC are the sums of no channels
        if (empty) return 0;
        AAS_CHECK(dB && dC, "%s: null pointer", who);
        ScanDev a;
        scan_dev(d, &a);
        const ColMap none = {};
        AAS_DT_SWITCH(d->dtype, E, hipLaunchKernelGGL(scan_finish_kernel<E>, dim3(nbc), dim3(256), 0, s, a, (const float*)nullptr, (const float*)nullptr,
                                                      (const float*)nullptr, 0, nbc, 0, (E*)dB, (E*)dC, none, none));
        AAS_LAUNCH_CHECK(who);
        return 0;
    }
    AAS_CHECK(dA != nullptr, "%s: null pointer", who);
    if (!empty) {
        const BwdWs w = bwd_ws(d->T, d->N, d->Ch, d->S, d->G);
        const ScanChunks ck = bwd_chunks(d->T, d->N, d->Ch, d->G);
        char* base = (char*)ws;
        AAS_CHECK(dy && hsave && dx && ddt && dB && dC && ws && (dz || !d->z), "%s: null pointer", who);
        AAS_CHECK(aas_aligned(hsave, 16) && aas_aligned(ws, 16), "%s: hsave and ws must be 16-byte aligned", who);
        ScanDev a;
        scan_dev(d, &a);
        a.nchunk = ck.n;
        a.tiles_per_chunk = ck.tiles;
        a.fine = FINE;
        const int al = 4 * aas_dt_size(d->dtype);
        const bool vec = scan_vec(a, d->dtype) && dy_st % 4 == 0 && dy_sn % 4 == 0 && aas_aligned(dy, al) && aas_aligned(dx, al) && aas_aligned(ddt, al) &&
                         (!dz || aas_aligned(dz, al));
        AAS_DT_SWITCH(d->dtype, E, launch_bwd<E>(s, a, vec, dy, dy_st, dy_sn, hsave, dx, ddt, d->z ? dz : nullptr, (float*)(base + w.bc),
                                                 (float*)(base + w.a), (float*)(base + w.d), (float*)(base + w.ends),
                                                 (float*)(base + w.sums)));
        AAS_LAUNCH_CHECK(who);
        const ColMap ma = {{dA, nullptr, nullptr, nullptr}, {d->Ch * d->S, 0, 0, 0}, 0, 1};
        const ColMap md = {{dD, ddt_bias, nullptr, nullptr}, {d->Ch, d->Ch, 0, 0}, 0, 2};
        const int na = cdiv((int64_t)d->Ch * d->S, 16), nd = dD || ddt_bias ? cdiv(2 * (int64_t)d->Ch, 16) : 0;
        AAS_DT_SWITCH(d->dtype, E, hipLaunchKernelGGL(scan_finish_kernel<E>, dim3(nbc + na + nd), dim3(256), 0, s, a, (const float*)(base + w.bc),
                                                      (const float*)(base + w.a), (const float*)(base + w.d), d->N * ck.n, nbc, na, (E*)dB, (E*)dC, ma, md));
        AAS_LAUNCH_CHECK(who);
        return 0;
    }
    // no frames: the sums of nothing
    const ColMap ma = {{dA, dD, ddt_bias, nullptr}, {d->Ch * d->S, d->Ch, d->Ch, 0}, 0, 3};
    return aas_sum_partials(s, nullptr, 0, d->Ch * (d->S + 2), ma, who);
}
