// Shared device helpers of the causal sequence operators (conv_causal.hip, ssm_scan*.hip, residual_norm.hip, gated_norm.hip,
// dropout.hip): activations in fp32, bf16 or fp16 (type code AAS_DT_*), parameters, the scan's states and every sum in fp32.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
template <class T, int V> using vec_t = T __attribute__((ext_vector_type(V)));

// V consecutive elements as fp32; p is aligned to V elements
template <class T> __device__ __forceinline__ f32x4 load4(const T* p) { return __builtin_convertvector(*reinterpret_cast<const vec_t<T, 4>*>(p), f32x4); }
template <> __device__ __forceinline__ f32x4 load4<float>(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
template <class T> __device__ __forceinline__ void store4(T* p, f32x4 v) {      // one rounding to nearest even
    *reinterpret_cast<vec_t<T, 4>*>(p) = __builtin_convertvector(v, vec_t<T, 4>);
}
template <> __device__ __forceinline__ void store4<float>(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }

// four elements p[0 .. 3], of which the first `n` exist (n <= 0: none); VEC: p is aligned to four elements and n is 4 or <= 0
template <class T, bool VEC> __device__ __forceinline__ f32x4 load4n(const T* p, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (n > 0) v = load4(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) v[i] = (float)p[i];
    }
    return v;
}
template <class T, bool VEC> __device__ __forceinline__ void store4n(T* p, f32x4 v, int n) {
    if (VEC) {
        if (n > 0) store4(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// 1 / (1 + e^-x) on the hardware exponential and reciprocal (1 ulp each): relative error below 2e-7 (1 + |x|) down to x = -87, where the
// value is e^x; 0 below that (1 + e^-x passes what the reciprocal of a normal number can hold), 0 and 1 at the infinities, NaN stays
__device__ __forceinline__ float sigm(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }

// sum over the four lanes of a quad (every lane gets it)
__device__ __forceinline__ float quad_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));   // quad_perm 2 3 0 1
    return v;
}

__device__ __forceinline__ int row_length(const int* len, int n, int T) {   // any value of the caller's is brought into [0, T]
    if (len == nullptr) return T;
    const int v = len[n];
    return v < 0 ? 0 : (v > T ? T : v);
}

// Sums over partial rows: out[map(m)] = sum over p of part[p][m], in 16 interleaved chains over p that are joined in order: the same
// bits on every run.  A workgroup takes 16 columns with 16 row lanes: a few hundred partial rows are a few rounds of loads in flight.
struct ColMap {                 // column m of a partial row -> where its sum goes: segment i holds cols[i] columns
    float* out[4];
    int cols[4];
    int inner;                  // > 0: segment 0 is stored [inner][cols / inner] in the partial row and [cols / inner][inner] in out[0]
    int n;
};
__device__ __forceinline__ void sum_columns(const float* __restrict__ part, int P, int M, const ColMap& map, int block) {
    __shared__ float s[16][17];
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int m = block * 16 + cl;
    float v = 0.f;
    if (m < M) {
        const float* p = part + m;
        int r = rl;
        for (; r + 7 * 16 < P; r += 8 * 16) {         // eight loads in flight
            float u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = p[(int64_t)(r + 16 * i) * M];
#pragma unroll
            for (int i = 0; i < 8; ++i) v += u[i];
        }
        for (; r < P; r += 16) v += p[(int64_t)r * M];
    }
    s[rl][cl] = v;
    __syncthreads();
    if (rl == 0 && m < M) {
        float t = s[0][cl];
#pragma unroll
        for (int i = 1; i < 16; ++i) t += s[i][cl];
        int col = m, seg = 0;
        while (seg + 1 < map.n && col >= map.cols[seg]) { col -= map.cols[seg]; ++seg; }
        if (map.out[seg]) {
            if (seg == 0 && map.inner > 0) {
                const int w = map.cols[0] / map.inner;
                col = (col % w) * map.inner + col / w;
            }
            map.out[seg][col] = t;
        }
    }
}
int aas_sum_partials(hipStream_t s, const float* part, int P, int M, const ColMap& map, const char* who);

#define AAS_DT_SWITCH(code, T, ...)                                   \
    switch (code) {                                                   \
        case AAS_DT_F32: { typedef float T; __VA_ARGS__; break; }     \
        case AAS_DT_BF16: { typedef bf16_t T; __VA_ARGS__; break; }   \
        default: { typedef f16_t T; __VA_ARGS__; break; }             \
    }
static inline int aas_dt_size(int code) { return code == AAS_DT_F32 ? 4 : 2; }
static inline bool aas_dt_ok(int code) { return code == AAS_DT_F32 || code == AAS_DT_BF16 || code == AAS_DT_F16; }
static inline bool aas_aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
