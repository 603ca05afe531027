// Selective state space scan, forward (ssm_scan.h has the mathematics and the layout).  Bound by instruction issue (the VALU is active in
// 95 % of the busy cycles at 4096 x 4 x 1024): a frame is 23 instructions a wave for the recurrence of 16 channels x 16 states, four of them exponentials at a
// quarter of the rate, and 14 for staging and the gate.  2001 x 3 x 1000 in bf16: 19 us carry + 31 us; 4096 x 4 x 1024 with the states kept
// for the backward pass: 59 + 97 us; 200 x 30 x 1000 unsplit in fp32: 42.
#include "scan_carry.h"

namespace {

template <class T, int NG, bool VEC>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanDev a, float* __restrict__ state, T* __restrict__ y, float* __restrict__ hsave,
                                                       const float* __restrict__ ends, const float* __restrict__ sums) {
    __shared__ __align__(16) float2 dd[2][SCAN_TT][SCAN_CH];          // d, d x
    __shared__ __align__(16) float bs[2][SCAN_TT][NG * 16], cs[2][SCAN_TT][NG * 16];
    __shared__ __align__(16) float ys[2][SCAN_TT][SCAN_YP];
    const ScanBlock b = scan_block(a);
    const int tid = threadIdx.x, q = tid & 3, cw = tid >> 2;            // scanning: lane q of channel cw
    const int lr = tid >> 4, lc = (tid & 15) * 4, ln = b.cn - lc, ls = tid & 15;   // loading: channels lc .. lc+3 of frame lr of the tile
    const int L = row_length(a.len, b.n, a.T);
    const bool on = cw < b.cn, svec = a.svec != 0;
    const T* xp = (const T*)a.x + b.n * a.x_sn + b.c0;
    const T* tp = (const T*)a.dt + b.n * a.dt_sn + b.c0;
    const T* zp = a.z ? (const T*)a.z + b.n * a.z_sn + b.c0 : nullptr;
    const T* bp = (const T*)a.B + b.n * a.B_sn + b.grp * a.B_sg;
    const T* cp = (const T*)a.C + b.n * a.C_sn + b.grp * a.C_sg;

    f32x4 A2[NG], h[NG];
    const int64_t srow = ((int64_t)b.n * a.Ch + b.c0 + cw) * a.S;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int s0 = g * 16 + 4 * q;
        A2[g] = h[g] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (on) {
            A2[g] = scan_rates4(a.A + (int64_t)(b.c0 + cw) * a.S, s0, a.S, svec);
            // (a split launch: the first chunk's end has the state in it; and the last chunk, which writes the new state, may finish first, so
            // the first one reads the copy that the carry launch left)
            if (state && a.nchunk == 1) h[g] = scan_states4(state + srow, s0, a.S, svec);
            if (state && a.nchunk > 1 && blockIdx.y == 0) h[g] = scan_states4(ends + ((int64_t)(a.nchunk - 1) * a.N * a.Ch) * a.S + srow, s0, a.S, svec);
        }
    }
    if (on && blockIdx.y > 0)
        scan_fold<NG, false>(h, A2, ends, sums, blockIdx.y, a.nchunk, (int64_t)a.N * a.Ch, (int64_t)b.n * a.Ch + b.c0 + cw, a.S, q, svec, a.softplus != 0);
    const f32x4 bias = a.dt_bias ? load4n<float, false>(a.dt_bias + b.c0 + lc, ln) : f32x4{0.f, 0.f, 0.f, 0.f};
    const f32x4 Dv = a.D ? load4n<float, false>(a.D + b.c0 + lc, ln) : f32x4{0.f, 0.f, 0.f, 0.f};

    f32x4 xr, tr, zr, xe, ze;
    float br[NG], cr[NG];
    const ScanCols<VEC> cols(lc, b.cn);
    auto load = [&](int tile) {                                         // (a frame behind the row's end: its last one, dropped again in stage)
        const int f = tile * SCAN_TT + lr;
        const int64_t t = f < L ? f : L - 1;
        xr = cols.get(xp + t * a.x_st);
        tr = cols.get(tp + t * a.dt_st);
        if (zp) zr = cols.get(zp + t * a.z_st);
#pragma unroll
        for (int g = 0; g < NG; ++g) {                                  // one state of one frame per thread and group
            const int s = g * 16 + ls < a.S ? g * 16 + ls : 0;
            br[g] = (float)bp[t * a.B_st + s];
            cr[g] = (float)cp[t * a.C_st + s];
        }
    };
    auto stage = [&](int tile, int u) {
        const bool live = tile * SCAN_TT + lr < L;                      // behind the end: d = 0 leaves the state as it is
        const f32x4 d = cols.keep(scan_delta4(tr, bias, a.softplus), live);
        xr = cols.keep(xr, live);
        scan_stage(&dd[u][lr][lc], d, d * xr);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const bool in = live && g * 16 + ls < a.S;
            bs[u][lr][g * 16 + ls] = in ? br[g] : 0.f;
            cs[u][lr][g * 16 + ls] = in ? cr[g] : 0.f;
        }
    };
    const int all = (L + SCAN_TT - 1) / SCAN_TT, k0 = blockIdx.y * a.tiles_per_chunk;
    const int k1 = k0 + a.tiles_per_chunk, tiles = k1 < all ? k1 : all;                       // tiles [k0, tiles) have frames, up to k1 are written
    T* yp = y + ((int64_t)(k0 * SCAN_TT + lr) * a.N + b.n) * a.Ch + b.c0 + lc;
    const int64_t ytile = (int64_t)SCAN_TT * a.N * a.Ch;
    if (tiles > k0) {
        load(k0);
        stage(k0, k0 & 1);
        xe = xr;
        ze = zr;
        if (tiles > k0 + 1) load(k0 + 1);
        __syncthreads();
    }
    for (int k = k0; k < tiles; ++k, yp += ytile) {
        const int u = k & 1;
#pragma unroll 1
        for (int t = 0; t < SCAN_TT; t += 4) {
            if (hsave && on && t % SCAN_HT == 0) {
                float* hp = hsave + ((int64_t)(k * (SCAN_TT / SCAN_HT) + t / SCAN_HT) * a.N * a.Ch) * a.S + srow;
#pragma unroll
                for (int g = 0; g < NG; ++g) scan_put_states4(hp, g * 16 + 4 * q, a.S, svec, h[g]);
            }
            float keep = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 d = dd[u][t + i][cw];
                float acc = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const f32x4 B = reinterpret_cast<const f32x4*>(bs[u][t + i])[g * 4 + q];
                    const f32x4 C = reinterpret_cast<const f32x4*>(cs[u][t + i])[g * 4 + q];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        h[g][j] = fmaf(__builtin_amdgcn_exp2f(d.x * A2[g][j]), h[g][j], d.y * B[j]);
                        acc = fmaf(h[g][j], C[j], acc);
                    }
                }
                acc = quad_sum(acc);
                keep = q == i ? acc : keep;
            }
            ys[u][t + q][cw] = keep;
        }
        f32x4 xn = xe, zn = ze;
        if (k + 1 < tiles) {
            stage(k + 1, u ^ 1);
            xn = xr;
            zn = zr;
            if (k + 2 < tiles) load(k + 2);
        }
        __syncthreads();
        if (k * SCAN_TT + lr < a.T) {
            f32x4 o = *reinterpret_cast<const f32x4*>(&ys[u][lr][lc]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[i] = fmaf(Dv[i], xe[i], o[i]);
                if (zp) o[i] *= ze[i] * sigm(ze[i]);
            }
            store4n<T, VEC>(yp, cols.keep(o, k * SCAN_TT + lr < L), ln);
        }
        xe = xn;
        ze = zn;
    }
    const int te = blockIdx.y + 1 == gridDim.y || (int64_t)k1 * SCAN_TT > a.T ? a.T : k1 * SCAN_TT;
    for (int t = (tiles > k0 ? tiles : k0) * SCAN_TT + lr; t < te; t += SCAN_TT, yp += ytile) store4n<T, VEC>(yp, f32x4{0.f, 0.f, 0.f, 0.f}, ln);
    if (state && on && blockIdx.y + 1 == gridDim.y)
#pragma unroll
        for (int g = 0; g < NG; ++g) scan_put_states4(state + srow, g * 16 + 4 * q, a.S, svec, h[g]);
}

// One frame: the state once in, once out, nothing staged.  Latency is what counts (30 x 1000 channels x 16 states: 3.8 MB, 4.0 us a launch
// against 6.8 for the tiled kernel, which walks its 16 frames).  Same lanes, same order of sums, as above.
template <class T, int NG>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanDev a, int bvec, float* __restrict__ state, T* __restrict__ y) {
    const ScanBlock b = scan_block(a);
    const int q = threadIdx.x & 3, cw = threadIdx.x >> 2, c = b.c0 + cw;
    if (cw >= b.cn) return;                              // (whole quads)
    const int64_t ch = (int64_t)b.n * a.Ch + c;
    if (row_length(a.len, b.n, 1) == 0) {
        if (q == 0) y[ch] = (T)0.f;
        return;
    }
    const bool svec = a.svec != 0;
    const float x = (float)((const T*)a.x)[b.n * a.x_sn + c], z = a.z ? (float)((const T*)a.z)[b.n * a.z_sn + c] : 0.f;
    float d = (float)((const T*)a.dt)[b.n * a.dt_sn + c] + (a.dt_bias ? a.dt_bias[c] : 0.f);
    if (a.softplus) d = scan_softplus(d, nullptr);
    const T* bp = (const T*)a.B + b.n * a.B_sn + b.grp * a.B_sg;
    const T* cp = (const T*)a.C + b.n * a.C_sn + b.grp * a.C_sg;
    const float dx = d * x;
    float acc = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int s0 = g * 16 + 4 * q;
        const f32x4 A2 = scan_rates4(a.A + (int64_t)c * a.S, s0, a.S, svec);
        f32x4 h = {0.f, 0.f, 0.f, 0.f};
        if (state) h = scan_states4(state + ch * a.S, s0, a.S, svec);
        const f32x4 B = bvec ? load4n<T, true>(bp + s0, a.S - s0) : load4n<T, false>(bp + s0, a.S - s0);
        const f32x4 C = bvec ? load4n<T, true>(cp + s0, a.S - s0) : load4n<T, false>(cp + s0, a.S - s0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(__builtin_amdgcn_exp2f(d * A2[j]), h[j], dx * B[j]);
            acc = fmaf(h[j], C[j], acc);
        }
        if (state) scan_put_states4(state + ch * a.S, s0, a.S, svec, h);
    }
    acc = quad_sum(acc);
    acc = fmaf(a.D ? a.D[c] : 0.f, x, acc);
    if (a.z) acc *= z * sigm(z);
    if (q == 0) y[ch] = (T)acc;
}

template <class T>
void launch_step(hipStream_t s, const ScanDev& a, float* state, void* y) {
    const int al = 4 * (int)sizeof(T);
    const int bvec = a.S % 4 == 0 && a.B_sn % 4 == 0 && a.B_sg % 4 == 0 && a.C_sn % 4 == 0 && a.C_sg % 4 == 0 && aas_aligned(a.B, al) && aas_aligned(a.C, al);
    const dim3 grid((unsigned)((int64_t)a.N * a.nbg * a.G));
    if (a.S <= 16) hipLaunchKernelGGL((scan_step_kernel<T, 1>), grid, dim3(256), 0, s, a, bvec, state, (T*)y);
    else if (a.S <= 32) hipLaunchKernelGGL((scan_step_kernel<T, 2>), grid, dim3(256), 0, s, a, bvec, state, (T*)y);
    else hipLaunchKernelGGL((scan_step_kernel<T, 4>), grid, dim3(256), 0, s, a, bvec, state, (T*)y);
}

template <class T>
void launch_fwd(hipStream_t s, const ScanDev& a, bool vec, float* state, void* y, float* hsave, float* ends, float* sums) {
    if (a.nchunk > 1) launch_carry<T, false>(s, a, vec, state, nullptr, 0, 0, ends, sums);
    const dim3 grid((unsigned)((int64_t)a.N * a.nbg * a.G), a.nchunk);
#define AAS_GO(NG_)                                                                                                                   \
    do {                                                                                                                              \
        if (vec) hipLaunchKernelGGL((scan_fwd_kernel<T, NG_, true>), grid, dim3(256), 0, s, a, state, (T*)y, hsave, ends, sums);                  \
        else hipLaunchKernelGGL((scan_fwd_kernel<T, NG_, false>), grid, dim3(256), 0, s, a, state, (T*)y, hsave, ends, sums);                     \
    } while (0)
    if (a.S <= 16) AAS_GO(1);
    else if (a.S <= 32) AAS_GO(2);
    else AAS_GO(4);
#undef AAS_GO
}

}  // namespace

int scan_check(const char* who, const aasScan* d) {
    AAS_CHECK(d != nullptr, "%s: null descriptor", who);
    AAS_CHECK(d->size == (int)sizeof(aasScan), "%s: aasScan.size = %d, this library's is %d", who, d->size, (int)sizeof(aasScan));
    AAS_CHECK(aas_dt_ok(d->dtype), "%s: dtype %d", who, d->dtype);
    AAS_CHECK(d->T >= 0 && d->N >= 0 && d->Ch >= 0, "%s: T = %d, N = %d, Ch = %d", who, d->T, d->N, d->Ch);
    AAS_CHECK(d->T <= 0x7fffffff - 2 * SCAN_TT, "%s: T = %d too long", who, d->T);
    AAS_CHECK(d->S >= 1 && d->S <= 64, "%s: S = %d, must be 1 to 64", who, d->S);
    AAS_CHECK(d->G >= 1 && d->Ch % d->G == 0, "%s: Ch = %d is no multiple of G = %d", who, d->Ch, d->G);
    // (a launch has fewer than 2^32 threads, 256 a workgroup; the finishing one a workgroup per 16 of Ch (S + 2) sums)
    AAS_CHECK((int64_t)d->N * (cdiv(d->Ch / d->G, SCAN_CH) * (int64_t)d->G) <= (1 << 23) && (int64_t)d->Ch * (d->S + 2) <= (1 << 27), "%s: N = %d, Ch = %d too large", who, d->N, d->Ch);
    if (d->T == 0 || d->N == 0 || d->Ch == 0) return 0;
    AAS_CHECK(d->x && d->dt && d->A && d->B && d->C, "%s: null pointer", who);
    return 0;
}

void scan_dev(const aasScan* d, ScanDev* a) {
    a->T = d->T; a->N = d->N; a->Ch = d->Ch; a->S = d->S; a->G = d->G; a->softplus = d->softplus;
    a->cpg = d->Ch / d->G;
    a->nbg = cdiv(a->cpg, SCAN_CH);
    a->tiles_per_chunk = scan_tiles(d->T);
    a->nchunk = a->fine = 1;                                      // (set by the launcher)
    a->svec = d->S % 4 == 0 && aas_aligned(d->A, 16);
    a->x = d->x; a->dt = d->dt; a->z = d->z; a->B = d->B; a->C = d->C;
    a->A = d->A; a->D = d->D; a->dt_bias = d->dt_bias; a->len = d->len;
    a->x_st = d->x_st; a->x_sn = d->x_sn; a->dt_st = d->dt_st; a->dt_sn = d->dt_sn; a->z_st = d->z_st; a->z_sn = d->z_sn;
    a->B_st = d->B_st; a->B_sn = d->B_sn; a->B_sg = d->B_sg; a->C_st = d->C_st; a->C_sn = d->C_sn; a->C_sg = d->C_sg;
}

// four channels at a time: channels of a group and every stride a multiple of four, bases on four elements (svec says
// the same of A and the states)
bool scan_vec(const ScanDev& a, int dtype) {
    const int al = 4 * aas_dt_size(dtype);
    return a.Ch % 4 == 0 && a.cpg % 4 == 0 && a.x_st % 4 == 0 && a.x_sn % 4 == 0 && a.dt_st % 4 == 0 && a.dt_sn % 4 == 0 && aas_aligned(a.x, al) &&
           aas_aligned(a.dt, al) && (!a.z || (a.z_st % 4 == 0 && a.z_sn % 4 == 0 && aas_aligned(a.z, al)));
}

ScanChunks scan_chunks(int T, int N, int Ch, int G, int want_blocks, int fine) {
    const int tiles = scan_tiles(T);
    const int64_t blocks = (int64_t)N * cdiv(Ch / G, SCAN_CH) * G;
    ScanChunks c = {1, tiles};
    // Unsplit above one workgroup a CU.  Measured, forward / forward and backward, unsplit against split: 800 x 16 x 1000 (256 workgroups) 112
    // / 443 us against 115 / 373; 200 x 30 x 1000 (480 workgroups) 53 / 170 against 64 / 185, 800 x 30 x 1000 164 / 604 against 193 / 625.
    if (blocks == 0 || blocks > 256) return c;
    int n = (int)(want_blocks / blocks);
    if (n > 32) n = 32;
    if (n > tiles / 4) n = tiles / 4;                   // at least four tiles a chunk
    if (n < 3) return c;                                // (two chunks: the carry launch and half of the main one take as long as the whole)
    c.tiles = cdiv(cdiv(tiles, n), fine) * fine;
    c.n = cdiv(tiles, c.tiles);
    return c;
}

// (2001 x 3 x 1000: 54.7 us a call with 1024 workgroups, 50.4 with 1536 and with 2048)
static ScanChunks fwd_chunks(int T, int N, int Ch, int G) { return scan_chunks(T, N, Ch, G, 1536, 1); }

extern "C" size_t aas_ssm_scan_fwd_ws_bytes(int T, int N, int Ch, int S, int G) {
    if (T <= 0 || N <= 0 || Ch <= 0 || S <= 0 || G <= 0 || Ch % G) return 0;
    const int n = fwd_chunks(T, N, Ch, G).n;
    return n == 1 ? 0 : (size_t)n * N * Ch * (S + 1) * sizeof(float);
}

extern "C" int aas_ssm_scan_fwd(aasStream_t stream, const aasScan* d, float* state, void* y, float* hsave, void* ws) {
    if (scan_check("aas_ssm_scan_fwd", d)) return 1;
    if (d->T == 0 || d->N == 0 || d->Ch == 0) return 0;
    AAS_CHECK(y != nullptr, "aas_ssm_scan_fwd: null pointer");
    AAS_CHECK(aas_aligned(hsave, 16) && aas_aligned(ws, 16), "aas_ssm_scan_fwd: hsave and ws must be 16-byte aligned");
    ScanDev a;
    scan_dev(d, &a);
    if (d->T == 1 && !hsave) {
        if (!aas_aligned(state, 16)) a.svec = 0;
        AAS_DT_SWITCH(d->dtype, E, launch_step<E>((hipStream_t)stream, a, state, y));
        AAS_LAUNCH_CHECK("aas_ssm_scan_fwd: one frame");
        return 0;
    }
    const ScanChunks c = fwd_chunks(d->T, d->N, d->Ch, d->G);
    AAS_CHECK(c.n == 1 || ws, "aas_ssm_scan_fwd: ws is wanted");
    a.nchunk = c.n;
    a.tiles_per_chunk = c.tiles;
    if (!aas_aligned(state, 16)) a.svec = 0;
    const bool vec = scan_vec(a, d->dtype) && aas_aligned(y, 4 * aas_dt_size(d->dtype));
    float* ends = (float*)ws;
    float* sums = ends ? ends + (int64_t)c.n * d->N * d->Ch * d->S : nullptr;
    AAS_DT_SWITCH(d->dtype, E, launch_fwd<E>((hipStream_t)stream, a, vec, state, y, hsave, ends, sums));
    AAS_LAUNCH_CHECK("aas_ssm_scan_fwd");
    return 0;
}
