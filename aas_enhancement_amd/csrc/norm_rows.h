// Row norms of the causal block (residual_norm.hip, gated_norm.hip): one pass over the row, which stays in registers.  TPR threads
// hold a row, thread l the columns 4 (i TPR + l) .. + 3 for i < NV.  Rows of up to 1024 columns are a wave each, four rows a workgroup, and
// need no barrier; longer ones are a workgroup's.
#pragma once
#include "seq_common.h"

constexpr int NORM_MAX_C = 16384;

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

// the column sums acc[i] (columns 4 (i TPR + l)) of a workgroup's rows -> out[0 .. C); four rows a workgroup are joined through LDS
template <int TPR, int NV> __device__ __forceinline__ void put_columns(const f32x4* acc, float* out, int C, float* lds) {
    const int l = threadIdx.x % TPR, r = threadIdx.x / TPR;
    if (TPR == 64) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) *reinterpret_cast<f32x4*>(lds + r * (NV * 256) + (i * 64 + l) * 4) = acc[i];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += 256) out[c] = (lds[c] + lds[NV * 256 + c]) + (lds[2 * NV * 256 + c] + lds[3 * NV * 256 + c]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) store4n<float, false>(out + (i * TPR + l) * 4, acc[i], C - (i * TPR + l) * 4);
    }
}

// (threads a row, column quads a thread) by the number of columns; the element-wise (unaligned) form has the larger of each kind only
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
            if ((C) <= 1024) { GO(64, 4, false); }       \
            else if ((C) <= 4096) { GO(256, 4, false); } \
            else { GO(1024, 4, false); }                 \
        }                                                \
    } while (0)

// workgroups of a backward pass, each of which leaves one partial row of the parameters' gradients
static inline int norm_bwd_blocks(int64_t rows, int C) {
    const int64_t groups = C <= 1024 ? (rows + 3) / 4 : rows;
    return (int)(groups < 512 ? (groups < 1 ? 1 : groups) : 512);
}
