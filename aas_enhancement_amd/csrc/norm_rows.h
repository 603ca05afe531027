// Row norms of the causal block (residual_norm.hip, gated_norm.hip): one pass over the row, which stays in registers.  TPR threads
// hold a row, each NV column quads: two neighbouring ones make one 16-byte access of a 16-bit type.  Rows of up to 1024 columns are a wave each, four rows a workgroup, and
// need no barrier; longer ones are a workgroup's.
#pragma once
#include "seq_common.h"

constexpr int NORM_MAX_C = 16384;

// first column of quad i of thread l
template <int TPR, int NV> __device__ __forceinline__ int row_col(int i, int l) {
    return NV == 1 ? l * 4 : ((i >> 1) * TPR + l) * 8 + (i & 1) * 4;
}

// a row's share of one thread in its own type: what is read ahead for the next row
template <class T, int NV> struct RowRaw {
    vec_t<T, 4> q[NV];
    template <int TPR, bool VEC> __device__ __forceinline__ void load(const T* row, int C, int l) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = row_col<TPR, NV>(i, l), n = C - c;
            q[i] = vec_t<T, 4>{(T)0.f, (T)0.f, (T)0.f, (T)0.f};
            if (VEC) {
                if (n > 0) q[i] = *reinterpret_cast<const vec_t<T, 4>*>(row + c);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < n) q[i][j] = row[c + j];
            }
        }
    }
    __device__ __forceinline__ f32x4 get(int i) const { return __builtin_convertvector(q[i], f32x4); }
};
// Rows go to resident workgroups in turn; with up to four quads a thread the next row is on its way while this one is worked on (more, or
// in a workgroup of 1024, would not fit the registers of the backward passes).  Rows of 8192 columns on 512 threads with the next row
// ahead were no faster than on 256 without: 99 / 225 us forward / backward against 93 / 224 at 8192 x 8192 in bf16.
template <int TPR, int NV> constexpr bool row_ahead() { return NV <= 4 && TPR <= 256; }

// sums of a and b over the row's threads, handed to all of them
template <int TPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float (*s)[2]) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (TPR > 64) {
        constexpr int W = TPR / 64;
        __syncthreads();                              // the last sums have been read
        if ((threadIdx.x & 63) == 0) {
            s[threadIdx.x >> 6][0] = a;
            s[threadIdx.x >> 6][1] = b;
        }
        __syncthreads();
        a = s[0][0];
        b = s[0][1];
#pragma unroll
        for (int i = 1; i < W; ++i) {
            a += s[i][0];
            b += s[i][1];
        }
    }
}

// Rows whose squares leave fp32's range are summed once more, scaled by a power of two (the same answer for all of a row's threads).  Below
// a mean square of 2^-100 (eps = 0: a larger eps holds it up) squares lose bits that count and the hardware root takes a denormal for
// zero; at infinity they have overflowed.  2^76 up brings the former's mean squares to 2^-100 .. 2^52 (normal numbers), 2^76 down those of
// finite numbers (a root mean square of 2^57 or more if the squares overflow over 16384 columns, 2^128 at most) to 2^-38 .. 2^104.  0: an
// ordinary row, or one that holds a NaN.
constexpr float ROW_SMALL = 0x1p-100f, ROW_UP = 0x1p76f, ROW_DOWN = 0x1p-76f;
__device__ __forceinline__ float row_rescale(float ms) { return ms < ROW_SMALL ? ROW_UP : ms > 3.4028234e38f ? ROW_DOWN : 0.f; }

// 1 / sqrt(mean(v^2) + eps) from the sum of the squares
template <int TPR, int NV> __device__ __forceinline__ float row_rstd(const f32x4 (&v)[NV], float sum, float inv, float eps, float (*s)[2]) {
    const float ms = fmaf(sum, inv, eps), c = row_rescale(ms);
    if (c == 0.f) return __builtin_amdgcn_rsqf(ms);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float u = v[i][j] * c;
            s1 = fmaf(u, u, s1);
        }
    row_sum2<TPR>(s1, s2, s);
    return __builtin_amdgcn_rsqf(fmaf(s1, inv, eps * c * c)) * c;
}

// the column sums acc[i] (quad i) of a workgroup's rows -> out[0 .. C); four rows a workgroup are joined through LDS
template <int TPR, int NV> __device__ __forceinline__ void put_columns(const f32x4* acc, float* out, int C, float* lds) {
    const int l = threadIdx.x % TPR, r = threadIdx.x / TPR;
    if (TPR == 64) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) *reinterpret_cast<f32x4*>(lds + r * (NV * 256) + row_col<TPR, NV>(i, l)) = acc[i];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += 256) out[c] = (lds[c] + lds[NV * 256 + c]) + (lds[2 * NV * 256 + c] + lds[3 * NV * 256 + c]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) store4n<float, false>(out + row_col<TPR, NV>(i, l), acc[i], C - row_col<TPR, NV>(i, l));
    }
}

// (threads a row, column quads a thread) by the number of columns.  The element-wise (unaligned) form has the larger of each kind only:
// the quads it has beyond the row add zeros, so a row gives the same bits however it is aligned.
#define AAS_ROW_SWITCH(C, vec, GO)                       \
    do {                                                 \
        if (vec) {                                       \
            if ((C) <= 256) { GO(64, 1, true); }         \
            else if ((C) <= 512) { GO(64, 2, true); }    \
            else if ((C) <= 1024) { GO(64, 4, true); }   \
            else if ((C) <= 2048) { GO(256, 2, true); }  \
            else if ((C) <= 4096) { GO(256, 4, true); }  \
            else if ((C) <= 8192) { GO(256, 8, true); }  \
            else { GO(1024, 4, true); }                  \
        } else {                                         \
            if ((C) <= 256) { GO(64, 1, false); }        \
            else if ((C) <= 1024) { GO(64, 4, false); }  \
            else if ((C) <= 8192) { GO(256, 8, false); } \
            else { GO(1024, 4, false); }                 \
        }                                                \
    } while (0)

// workgroups that share `rows` rows of C columns, at most `most`; in a backward pass each leaves one partial row of the parameters' gradients
static inline int norm_blocks(int64_t rows, int C, int most) {
    const int64_t groups = C <= 1024 ? (rows + 3) / 4 : rows;
    return (int)(groups < most ? (groups < 1 ? 1 : groups) : most);
}
static inline bool norm_eps_ok(float eps) { return eps >= 0.f && eps <= 3.4028234e38f; }
