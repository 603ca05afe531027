// Depthwise causal convolution over K frames (+ SiLU), forward and backward, and the joining of partial sums that the sequence
// operators share.
//
//   p[t] = bias + sum_k w[k] x[t-K+1+k],  y = p sigmoid(p);   dp = dy sigmoid(p) (1 + p (1 - sigmoid(p))),
//   dx[t] = sum_k w[k] dp[t+K-1-k],  dw[k] = sum_t dp[t] x[t-K+1+k],  dbias = sum_t dp[t].
//
// HBM-bound: x in, y out (backward: x and dy in, dx out).  A thread owns four neighbouring channels and runs over a stretch of the time
// axis with the K frames of its window in registers, so each element is read once plus K - 1 frames of overlap per stretch; lanes
// run along channels, then rows, then stretches.  4096 x 4 x 2048, K = 4, forward / backward: 27 / 81 us in bf16 (4.9 / 2.5
// TB/s of x, dy and dx), 50 / 101 in fp32.  The backward kernel is held to four waves a SIMD (128 registers): with K = 4 its fp32 and its element-wise
// forms spill 3 and 8 of them.  Where C is small and T large the launch that joins the partial rows has few workgroups and decides: 4096 x 32 x 16
// 50 us backward, 2000 x 32 x 80 43.
#include "seq_common.h"

namespace {

// taps of four channels, w[channel][K] -> wk[tap][channel]; whole quads by 16-byte loads where the row is aligned for them
template <int K> __device__ __forceinline__ void load_taps(f32x4 (&wk)[K], const float* w, int cn) {
    if (cn == 4 && ((uintptr_t)w & 15) == 0) {
        f32x4 v[K];
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = reinterpret_cast<const f32x4*>(w)[k];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) wk[k][i] = v[(i * K + k) / 4][(i * K + k) % 4];
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) wk[k][i] = i < cn ? w[i * K + k] : 0.f;
    }
}

// win[1 .. K-1] = the frames t0-K+1 .. t0-1 of a row of L frames: from the state (zeros without one) where a row begins, zeros behind its
// end.  No load waits for another: addresses are chosen and brought inside, what is not wanted is dropped behind the loads.
template <class T, int K, bool VEC>
__device__ __forceinline__ void load_window(f32x4 (&win)[K], const T* xp, int64_t x_st, const T* sp, int64_t C, int t0, int L, int cn) {
    const T* at[K - 1];
    bool keep[K - 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int t = t0 - (K - 1) + k, r = t < L ? t : L - 1;
        at[k] = t >= 0 ? xp + (int64_t)(r > 0 ? r : 0) * x_st : (sp ? sp + (int64_t)(t + K - 1) * C : xp);
        keep[k] = t >= 0 ? t < L : sp != nullptr;
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[k + 1] = load4n<T, VEC>(at[k], cn);
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) win[k + 1][i] = keep[k] ? win[k + 1][i] : 0.f;
}

template <class T, int K, bool VEC>
__global__ __launch_bounds__(256) void conv_fwd_kernel(int TT, int N, int C, int CV, int stretch, int nstretch, const T* __restrict__ x, int64_t x_st,
                                                       int64_t x_sn, const float* __restrict__ w, const float* __restrict__ bias, int silu,
                                                       const int* __restrict__ len, T* __restrict__ state, T* __restrict__ y) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int cv = (int)(id % CV);
    const int64_t rest = id / CV;
    const int n = (int)(rest % N), part = (int)(rest / N);
    if (part >= nstretch) return;
    const int c = cv * 4, cn = C - c < 4 ? C - c : 4;
    const int L = row_length(len, n, TT);
    const int t0 = part * stretch, t1 = t0 + stretch < TT ? t0 + stretch : TT;
    const T* xp = x + n * x_sn + c;
    T* sp = state ? state + (int64_t)n * (K - 1) * C + c : nullptr;

    f32x4 wk[K], b = load4n<float, false>(bias ? bias + c : nullptr, bias ? cn : 0);
    load_taps<K>(wk, w + (int64_t)c * K, cn);

    f32x4 win[K];                                     // win[K-1] is the newest frame
    load_window<T, K, VEC>(win, xp, x_st, sp, C, t0, L, cn);
    const int te = t1 < L ? t1 : L;
    T* yp = y + ((int64_t)t0 * N + n) * C + c;
    const int64_t ys = (int64_t)N * C;
    int t = t0;
#pragma unroll 4
    for (; t < te; ++t, yp += ys) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[k] = win[k + 1];
        win[K - 1] = load4n<T, VEC>(xp + t * x_st, cn);
        f32x4 p = b;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = fmaf(wk[k][i], win[k][i], p[i]);
        if (silu)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] *= sigm(p[i]);
        store4n<T, VEC>(yp, p, cn);
    }
    for (; t < t1; ++t, yp += ys) store4n<T, VEC>(yp, f32x4{0.f, 0.f, 0.f, 0.f}, cn);
    // The new state is the last K-1 of [old state, the row's frames]: the window, where one thread has walked the whole row.  Where
    // several share it, the first one's thread is the only reader of the old state (the others begin behind frame K-1), so it writes.
    if (sp && L > 0 && part == 0) {
        f32x4 next[K - 1];
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            const int src = L - (K - 1) + k;          // frame index; < 0: from the old state
            next[k] = nstretch == 1 ? win[k + 1]
                                    : (src >= 0 ? load4n<T, VEC>(xp + src * x_st, cn) : load4n<T, VEC>(sp + (int64_t)(src + K - 1) * C, cn));
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k) store4n<T, VEC>(sp + (int64_t)k * C, next[k], cn);
    }
}

template <class T, int K, bool VEC>
__global__ __launch_bounds__(256, 4) void conv_bwd_kernel(int TT, int N, int C, int CV, int stretch, int nstretch, int lanes, const T* __restrict__ x, int64_t x_st,
                                                       int64_t x_sn, const float* __restrict__ w, const float* __restrict__ bias, int silu,
                                                       const int* __restrict__ len, const T* __restrict__ dy, int64_t dy_st, int64_t dy_sn,
                                                       T* __restrict__ dx, float* __restrict__ part_out) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int cv = (int)(id % CV);
    const int64_t first = id / CV;
    if (first >= lanes) return;
    const int c = cv * 4, cn = C - c < 4 ? C - c : 4;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    f32x4 wk[K], dw[K], b = load4n<float, false>(bias ? bias + c : nullptr, bias ? cn : 0), db = zero;
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k] = zero;
    load_taps<K>(wk, w + (int64_t)c * K, cn);
    const int64_t ys = (int64_t)N * C;
    // a stretch of one row; where there are more of them than `lanes` (many short rows) a thread takes several, one partial row for all
    for (int64_t rest = first; rest < (int64_t)N * nstretch; rest += lanes) {
        const int n = (int)(rest % N), part = (int)(rest / N);
        const int L = row_length(len, n, TT);
        const int t0 = part * stretch, t1 = t0 + stretch < TT ? t0 + stretch : TT;
        const int te = t1 < L ? t1 : L;
        const T* xp = x + n * x_sn + c;
        const T* gp = dy + n * dy_sn + c;
        f32x4 win[K], dp[K];                              // x[t-K+1 .. t], dp[t-K+1 .. t]
#pragma unroll
        for (int k = 0; k < K; ++k) dp[k] = zero;
        load_window<T, K, VEC>(win, xp, x_st, nullptr, C, t0, L, cn);
        T* op = dx ? dx + ((int64_t)t0 * N + n) * C + c : nullptr;
        // One frame: dp[t], its share of dw and dbias (mine), and dx[t-K+1], which is complete behind dp[t].
        auto frame = [&](int t, f32x4 xv, f32x4 g, bool mine) {
#pragma unroll
            for (int k = 0; k < K - 1; ++k) { win[k] = win[k + 1]; dp[k] = dp[k + 1]; }
            win[K - 1] = xv;
            if (silu) {
                f32x4 p = b;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = fmaf(wk[k][i], win[k][i], p[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s = sigm(p[i]);
                    g[i] *= s * fmaf(p[i], 1.f - s, 1.f);
                }
            }
            dp[K - 1] = g;
            if (mine) {
#pragma unroll
                for (int i = 0; i < 4; ++i) db[i] += g[i];
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) dw[k][i] = fmaf(g[i], win[k][i], dw[k][i]);
            }
            if (op && t >= t0 + K - 1) {
                f32x4 v = zero;                           // dp[0] is frame t-K+1: its own tap is the newest, w[K-1]
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = fmaf(wk[K - 1 - k][i], dp[k][i], v[i]);
                store4n<T, VEC>(op, v, cn);
                op += ys;
            }
        };
        // The stretch's own frames, whose loads nothing holds back; up to K-1 frames of the next stretch, whose dp is formed again; behind the
        // row's end zeros.
        int t = t0;
#pragma unroll 4
        for (; t < te; ++t) frame(t, load4n<T, VEC>(xp + t * x_st, cn), load4n<T, VEC>(gp + t * dy_st, cn), true);
        if (te > t0) {
            const int tl = te + K - 1 < L ? te + K - 1 : L;
            for (; t < tl; ++t) frame(t, load4n<T, VEC>(xp + t * x_st, cn), load4n<T, VEC>(gp + t * dy_st, cn), false);
            for (; t < te + K - 1; ++t) frame(t, zero, zero, false);
        }
        if (op)
            for (t = te > t0 ? te : t0; t < t1; ++t, op += ys) store4n<T, VEC>(op, zero, cn);
    }
    if (part_out) {                                   // one row of [K taps | bias] x C per lane
        float* pp = part_out + first * (int64_t)(K + 1) * C + c;
#pragma unroll
        for (int k = 0; k < K; ++k) store4n<float, false>(pp + (int64_t)k * C, dw[k], cn);
        store4n<float, false>(pp + (int64_t)K * C, db, cn);
    }
}

__global__ __launch_bounds__(256) void sum_partials_kernel(const float* __restrict__ part, int P, int M, ColMap map) {
    sum_columns(part, P, M, map, blockIdx.x);
}

// Stretch of the time axis per thread: short enough that the launch has the 262144 threads that keep the memory system busy (half as many:
// 37 us instead of 28 forward at 4096 x 4 x 2048 in bf16), and at least `least` frames - 8 forward, where an overlap of K - 1 frames
// mostly hits the cache (200 x 30 x 1000 in fp32: 12.7 us, 13.8 with 16), 16 backward, where each stretch leaves a partial row of K + 1 sums.
constexpr int FWD_LEAST = 8, BWD_LEAST = 16;
int conv_stretch(int T, int N, int C, int least) {
    const int64_t rows4 = (int64_t)cdiv(C, 4) * N;
    int64_t per = 262144 / (rows4 > 0 ? rows4 : 1);
    if (per < 1) per = 1;
    const int s = cdiv(T, per);
    return s < least ? least : s;
}

// partial rows of the backward pass: every (stretch, row) its own while there are at most 2048, or as many as make 524288 threads
int conv_lanes(int T, int N, int C) {
    const int64_t all = (int64_t)cdiv(T, conv_stretch(T, N, C, BWD_LEAST)) * N, most = 524288 / cdiv(C, 4);
    return (int)(all < 2048 ? all : (all < most ? all : (most > 2048 ? most : 2048)));
}

template <int K, bool VEC>
void launch_fwd(hipStream_t s, int dtype, int T, int N, int C, const void* x, int64_t x_st, int64_t x_sn, const float* w, const float* b, int silu,
                const int* len, void* state, void* y) {
    const int CV = cdiv(C, 4), st = conv_stretch(T, N, C, FWD_LEAST), ns = cdiv(T, st);
    const int64_t threads = (int64_t)CV * N * ns;
    AAS_DT_SWITCH(dtype, E, hipLaunchKernelGGL((conv_fwd_kernel<E, K, VEC>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, T, N, C, CV, st, ns,
                                               (const E*)x, x_st, x_sn, w, b, silu, len, (E*)state, (E*)y));
}
template <int K, bool VEC>
void launch_bwd(hipStream_t s, int dtype, int T, int N, int C, const void* x, int64_t x_st, int64_t x_sn, const float* w, const float* b, int silu,
                const int* len, const void* dy, int64_t dy_st, int64_t dy_sn, void* dx, float* part) {
    const int CV = cdiv(C, 4), st = conv_stretch(T, N, C, BWD_LEAST), ns = cdiv(T, st), lanes = conv_lanes(T, N, C);
    const int64_t threads = (int64_t)CV * lanes;
    AAS_DT_SWITCH(dtype, E, hipLaunchKernelGGL((conv_bwd_kernel<E, K, VEC>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, T, N, C, CV, st, ns,
                                               lanes, (const E*)x, x_st, x_sn, w, b, silu, len, (const E*)dy, dy_st, dy_sn, (E*)dx, part));
}

bool conv_args_ok(const char* who, int dtype, int T, int N, int C, int K) {
    if (!aas_dt_ok(dtype)) { aas_set_error("%s: dtype %d", who, dtype); return false; }
    if (T < 0 || N < 0 || C < 0 || T > (1 << 30)) { aas_set_error("%s: T = %d, N = %d, C = %d", who, T, N, C); return false; }
    if (K < 2 || K > 4) { aas_set_error("%s: K = %d, must be 2, 3 or 4", who, K); return false; }
    // (a launch has fewer than 2^32 threads)
    if (C > (1 << 24) || (int64_t)N * cdiv(C, 4) > ((int64_t)1 << 30)) { aas_set_error("%s: N = %d, C = %d too large", who, N, C); return false; }
    return true;
}

}  // namespace

int aas_sum_partials(hipStream_t s, const float* part, int P, int M, const ColMap& map, const char* who) {
    if (M == 0) return 0;
    hipLaunchKernelGGL(sum_partials_kernel, dim3(cdiv(M, 16)), dim3(256), 0, s, part, P, M, map);
    AAS_LAUNCH_CHECK(who);
    return 0;
}

extern "C" int aas_causal_conv1d_fwd(aasStream_t stream, int dtype, int T, int N, int C, int K, const void* x, int64_t x_st, int64_t x_sn,
                                     const float* weight, const float* bias, int silu, const int* len, void* state, void* y) {
    if (!conv_args_ok("aas_causal_conv1d_fwd", dtype, T, N, C, K)) return 1;
    if (T == 0 || N == 0 || C == 0) return 0;
    AAS_CHECK(x && weight && y, "aas_causal_conv1d_fwd: null pointer");
    const int es = aas_dt_size(dtype);
    const bool vec = C % 4 == 0 && x_st % 4 == 0 && x_sn % 4 == 0 && aas_aligned(x, 4 * es) && aas_aligned(y, 4 * es) && (!state || aas_aligned(state, 4 * es));
#define AAS_FWD(K_)                                                                                                                    \
    (vec ? launch_fwd<K_, true>((hipStream_t)stream, dtype, T, N, C, x, x_st, x_sn, weight, bias, silu, len, state, y)                 \
         : launch_fwd<K_, false>((hipStream_t)stream, dtype, T, N, C, x, x_st, x_sn, weight, bias, silu, len, state, y))
    if (K == 2) AAS_FWD(2);
    else if (K == 3) AAS_FWD(3);
    else AAS_FWD(4);
#undef AAS_FWD
    AAS_LAUNCH_CHECK("aas_causal_conv1d_fwd");
    return 0;
}

extern "C" size_t aas_causal_conv1d_bwd_ws_bytes(int T, int N, int C, int K) {
    if (T <= 0 || N <= 0 || C <= 0 || K < 2 || K > 4) return 0;
    return (size_t)conv_lanes(T, N, C) * (K + 1) * C * sizeof(float);
}

extern "C" int aas_causal_conv1d_bwd(aasStream_t stream, int dtype, int T, int N, int C, int K, const void* x, int64_t x_st, int64_t x_sn,
                                     const float* weight, const float* bias, int silu, const int* len, const void* dy, int64_t dy_st,
                                     int64_t dy_sn, void* dx, float* dweight, float* dbias, void* ws) {
    if (!conv_args_ok("aas_causal_conv1d_bwd", dtype, T, N, C, K)) return 1;
    if (C == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    const bool empty = T == 0 || N == 0, params = dweight || dbias;
    AAS_CHECK(empty || (x && weight && dy && (ws || !params)), "aas_causal_conv1d_bwd: null pointer");
    const int P = empty ? 0 : conv_lanes(T, N, C);
    if (!empty) {
        const int es = aas_dt_size(dtype);
        const bool vec = C % 4 == 0 && x_st % 4 == 0 && x_sn % 4 == 0 && dy_st % 4 == 0 && dy_sn % 4 == 0 && aas_aligned(x, 4 * es) &&
                         aas_aligned(dy, 4 * es) && (!dx || aas_aligned(dx, 4 * es));
        float* part = params ? (float*)ws : nullptr;
#define AAS_BWD(K_)                                                                                                                          \
    (vec ? launch_bwd<K_, true>(s, dtype, T, N, C, x, x_st, x_sn, weight, bias, silu, len, dy, dy_st, dy_sn, dx, part)                       \
         : launch_bwd<K_, false>(s, dtype, T, N, C, x, x_st, x_sn, weight, bias, silu, len, dy, dy_st, dy_sn, dx, part))
        if (K == 2) AAS_BWD(2);
        else if (K == 3) AAS_BWD(3);
        else AAS_BWD(4);
#undef AAS_BWD
        AAS_LAUNCH_CHECK("aas_causal_conv1d_bwd");
    }
    if (!params) return 0;
    ColMap map = {{dweight, dbias, nullptr, nullptr}, {K * C, C, 0, 0}, K, 2};   // (no rows: the sums of nothing, zeros)
    return aas_sum_partials(s, (const float*)ws, P, (K + 1) * C, map, "aas_causal_conv1d_bwd: sums");
}
