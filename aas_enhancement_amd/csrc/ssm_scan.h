// Shared by the kernels of the selective state space scan (ssm_scan_fwd.hip, ssm_scan_bwd.hip).
//
//   d = softplus(dt + dt_bias),  h_s[t] = exp(d A_s) h_s[t-1] + d x B_s[t],  o = sum_s C_s h_s + D x,  y = o z sigmoid(z).
//
// Layout of a workgroup: 64 channels of one row n x 4 lanes a channel, each lane with NG groups of 4 states (state g*16 + 4*q + j for lane
// q of the quad), so up to 16 NG states; the sum over a channel's states is two quad exchanges.  The time axis goes by in tiles of 16
// frames staged in LDS: each thread loads four neighbouring channels of one frame and forms what depends on (frame, channel) only -
// softplus, gates - ONCE, not once per state; B and C of the tile are read as quads by all channels.
#pragma once
#include "seq_common.h"

constexpr int SCAN_CH = 64;      // channels per workgroup
constexpr int SCAN_TT = 16;      // frames per tile
constexpr int SCAN_HT = 8;       // frames between the states that the forward pass keeps for the backward pass
constexpr int SCAN_YP = 80;      // pitch of a [16 frames][64 channels] tile that the scanning lanes write: 4 frames x 16 channels a wave, no two on one bank
constexpr float SCAN_LOG2E = 1.4426950408889634f;
constexpr float SCAN_LN2 = 0.6931471805599453f;

struct ScanDev {                 // aasScan with the pointers' types left to the kernels, plus what the host derives
    int T, N, Ch, S, G, softplus;
    int cpg, nbg;                // channels per group, workgroups per group
    int tiles_per_chunk, nchunk; // chunks of the time axis (1: none)
    int fine;                    // chunks of the carry launch per chunk of the main one
    int svec;                    // rows of S fp32 states (A, the state) can be read four at a time
    const void *x, *dt, *z, *B, *C;
    const float *A, *D, *dt_bias;
    const int* len;
    int64_t x_st, x_sn, dt_st, dt_sn, z_st, z_sn, B_st, B_sn, B_sg, C_st, C_sn, C_sg;
};

// Splitting the time axis.  With few rows and channels a launch of one workgroup per (row, 64 channels) leaves most of the chip idle while
// each walks the whole sequence.  The axis is then cut into chunks of whole tiles: a first launch (scan_carry.h) forms what each chunk
// adds to the state - its own end, from zero - and the sum of its d; the state in front of chunk k is the ends of the chunks before it,
// each decayed by exp(A sum of d) of the chunks between, which every workgroup of the main launch folds for itself.  The decays are
// formed once more than unsplit, so it pays only where the chip is far from full.
struct ScanChunks { int n, tiles; };
ScanChunks scan_chunks(int T, int N, int Ch, int G, int want_blocks, int fine);

struct ScanBlock {               // where a workgroup stands
    int n, grp, c0, cn;          // row, group of B / C, first channel, channels (<= 64)
};
__device__ __forceinline__ ScanBlock scan_block(const ScanDev& a) {
    ScanBlock b;
    const int per_n = a.nbg * a.G;
    b.n = blockIdx.x / per_n;
    const int cb = blockIdx.x - b.n * per_n;
    b.grp = cb / a.nbg;
    const int i = cb - b.grp * a.nbg;
    b.c0 = b.grp * a.cpg + i * SCAN_CH;
    const int left = a.cpg - i * SCAN_CH;
    b.cn = left < SCAN_CH ? left : SCAN_CH;
    return b;
}

// The four neighbouring channels of the loading thread, brought inside the workgroup's: loads need no branches, what lies outside is
// replaced by zeros behind them.  Frames are brought inside the row in the same way.
template <bool VEC> struct ScanCols {
    int c[VEC ? 1 : 4];
    bool in[VEC ? 1 : 4];
    __device__ __forceinline__ ScanCols(int lc, int cn) {
#pragma unroll
        for (int i = 0; i < (VEC ? 1 : 4); ++i) {
            in[i] = lc + i < cn;
            c[i] = in[i] ? lc + i : (VEC ? cn - 4 : cn - 1);
        }
    }
    template <class T> __device__ __forceinline__ f32x4 get(const T* row) const {
        if (VEC) return load4(row + c[0]);
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)row[c[VEC ? 0 : i]];
        return v;
    }
    __device__ __forceinline__ f32x4 keep(f32x4 v, bool live) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = live && in[VEC ? 0 : i] ? v[i] : 0.f;
        return v;
    }
};

// d = softplus(v) = max(v, 0) + log(1 + e), e = e^-|v|, and its derivative.  log(1 + e) = 2 atanh(e / (2 + e)): the argument s is at most
// 1/3 and atanh(s) / s a polynomial in s^2 (Chebyshev interpolation, off by less than 8e-9), so d keeps full relative accuracy where e is tiny (d
// of 1e-3 and below), which log(1 + e) formed in fp32 has not.  The exponential takes the rounding of v log2(e) along.
__device__ __forceinline__ float scan_softplus(float v, float* slope) {
    const float a = fabsf(v), m = a > 200.f ? 200.f : a, p = m * SCAN_LOG2E;               // (e is 0 from 104 on; an infinite m would make NaN below)
    const float lost = fmaf(m, SCAN_LOG2E, -p) + m * 1.925963033500e-8f;                // m log2(e) - p
    float e = __builtin_amdgcn_exp2f(-p);
    e = fmaf(e, -SCAN_LN2 * lost, e);
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float y = fmaf(0.14078889f, q, 0.13982579f);
    y = fmaf(y, q, 0.20012298f);
    y = fmaf(y, q, 0.33333161f);
    y = fmaf(y, q, 1.f);
    if (slope) {
        const float r = __builtin_amdgcn_rcpf(1.f + e);
        *slope = v >= 0.f ? r : e * r;
    }
    return fmaf(2.f * s, y, fmaxf(v, 0.f));             // (a NaN comes through y)
}
__device__ __forceinline__ f32x4 scan_delta4(f32x4 dt, f32x4 bias, int softplus) {
    f32x4 v = dt + bias;
    if (softplus)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = scan_softplus(v[i], nullptr);
    return v;
}
__device__ __forceinline__ f32x4 scan_delta4(f32x4 dt, f32x4 bias, int softplus, f32x4& slope) {
    f32x4 v = dt + bias;
    slope = f32x4{1.f, 1.f, 1.f, 1.f};
    if (softplus)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float k;
            v[i] = scan_softplus(v[i], &k);
            slope[i] = k;
        }
    return v;
}
// (d, value) of four channels of one frame
__device__ __forceinline__ void scan_stage(float2* at, f32x4 d, f32x4 v) {
    reinterpret_cast<f32x4*>(at)[0] = f32x4{d[0], v[0], d[1], v[1]};
    reinterpret_cast<f32x4*>(at)[1] = f32x4{d[2], v[2], d[3], v[3]};
}

// the 4 states of lane q, group g, of a [S] row (zeros behind the last)
__device__ __forceinline__ f32x4 scan_states4(const float* row, int s0, int S, bool vec) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (vec) { if (s0 < S) v = *reinterpret_cast<const f32x4*>(row + s0); }
    else
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (s0 + j < S) v[j] = row[s0 + j];
    return v;
}
__device__ __forceinline__ void scan_put_states4(float* row, int s0, int S, bool vec, f32x4 v) {
    if (vec) { if (s0 < S) *reinterpret_cast<f32x4*>(row + s0) = v; }
    else
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (s0 + j < S) row[s0 + j] = v[j];
}

// A log2(e) of the same states: exp(d A) is one exp2.  Brought inside the finite numbers (a NaN stays): a rate of -inf, or one that the
// factor takes there, forgets everything in one frame, and d = 0 behind a row's end still leaves the state as it is (0 inf is none).
__device__ __forceinline__ f32x4 scan_rates4(const float* row, int s0, int S, bool vec) {
    f32x4 v = scan_states4(row, s0, S, vec) * SCAN_LOG2E;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = v[j] < -3.4028234e38f ? -3.4028234e38f : v[j];
        v[j] = v[j] > 3.4028234e38f ? 3.4028234e38f : v[j];
    }
    return v;
}

// exp2(p) h where exp2(p) alone may pass fp32's range: zeros stay zeros, and a small state grows to what it is
__device__ __forceinline__ float scan_grow(float p, float h) {
    p = p > 400.f ? 400.f : p < -400.f ? -400.f : p;                                        // (400 takes the smallest number past the largest)
    const float i = __builtin_rintf(p);
    return __builtin_ldexpf(h * __builtin_amdgcn_exp2f(p - i), (int)i);
}
// h in front of carry chunk k (REV: the carry behind it) from the chunks' ends [nchunk][N][Ch][S] and sums of d [nchunk][N][Ch]
template <int NG, bool REV, bool GROW>
__device__ __forceinline__ void scan_fold_by(f32x4 (&h)[NG], const f32x4 (&A2)[NG], const float* ends, const float* sums, int k, int nchunk, int64_t rows,
                                             int64_t ch, int S, int q, bool svec) {
    // forward: chunk j's own end for j = 0 .. k-1, the newest last;  REV: j = nchunk-1 .. k+1
    const int first = REV ? nchunk - 1 : 0, count = REV ? nchunk - 1 - k : k;
#pragma unroll (GROW ? 1 : 4)
    for (int i = 0; i < count; ++i) {
        const int j = REV ? first - i : first + i;
        const int64_t at = j * rows + ch;
        const float d = sums[at];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const f32x4 e = scan_states4(ends + at * S, g * 16 + 4 * q, S, svec);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float p = d * A2[g][m];
                h[g][m] = i == 0 ? e[m] : GROW ? scan_grow(p, h[g][m]) + e[m] : fmaf(__builtin_amdgcn_exp2f(p), h[g][m], e[m]);
            }
        }
    }
}
// A chunk's decay is one exponential of its whole sum.  It shrinks with d >= 0 and A <= 0; a wave with a positive rate, or with steps given as
// they are that go back, takes the exponent apart (doing so wherever softplus is off made a prompt of 2001 x 3 x 1000 62 us instead of 58).
template <int NG, bool REV>
__device__ __forceinline__ void scan_fold(f32x4 (&h)[NG], const f32x4 (&A2)[NG], const float* ends, const float* sums, int k, int nchunk, int64_t rows,
                                          int64_t ch, int S, int q, bool svec, bool softplus) {
    bool grows = false;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int m = 0; m < 4; ++m) grows = grows || A2[g][m] > 0.f;
    if (!softplus) {
        float least = 0.f;
#pragma unroll 8
        for (int j = REV ? k + 1 : 0; j < (REV ? nchunk : k); ++j) least = fminf(least, sums[j * rows + ch]);
        grows = grows || least < 0.f;
    }
    if (__any(grows)) scan_fold_by<NG, REV, true>(h, A2, ends, sums, k, nchunk, rows, ch, S, q, svec);
    else scan_fold_by<NG, REV, false>(h, A2, ends, sums, k, nchunk, rows, ch, S, q, svec);
}

// host side
int scan_check(const char* who, const aasScan* d);             // 0 fine, 1 error (aas_last_error)
void scan_dev(const aasScan* d, ScanDev* a);                   // fills everything but the chunks
bool scan_vec(const ScanDev& a, int dtype);                    // rows of x, dt, z can be read four channels at a time
static inline int scan_tiles(int T) { return cdiv(T, SCAN_TT); }
