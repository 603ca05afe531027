// Philox-4x32 with 10 rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): 128
// random bits as a function of a counter and a key, so a dropout mask is formed again wherever it is needed and never stored.  A
// counter gives 8 elements 16 bits each: p is met to 2^-17, and a 16-bit activation costs ~15 integer instructions an element, which
// hides behind its memory traffic; 32 bits an element would double that.
#pragma once
#include "seq_common.h"

struct DropKey { unsigned k0, k1; unsigned long long off; };

__device__ __forceinline__ DropKey drop_key(int64_t seed, int64_t offset, const int64_t* d_seed) {
    if (d_seed) { seed = d_seed[0]; offset = d_seed[1]; }
    DropKey k;
    k.k0 = (unsigned)seed;
    k.k1 = (unsigned)((unsigned long long)seed >> 32);
    k.off = (unsigned long long)offset;
    return k;
}

struct U4 { unsigned w[4]; };
__device__ __forceinline__ U4 philox(const DropKey& key, unsigned long long ctr) {
    ctr += key.off;
    unsigned c0 = (unsigned)ctr, c1 = (unsigned)(ctr >> 32), c2 = 0, c3 = 0, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return U4{{c0, c1, c2, c3}};
}

// bits i = 0 .. 7 of the counter's elements
__device__ __forceinline__ unsigned half_of(const U4& u, int i) { return (i & 1) ? u.w[i >> 1] >> 16 : u.w[i >> 1] & 0xffffu; }

// v with the dropped ones of elements e .. e+3 at zero and the kept ones times `factor`; EVEN: e is a multiple of 4
template <bool EVEN> __device__ __forceinline__ f32x4 drop4(f32x4 v, int64_t e, const DropKey& key, unsigned thr, float factor) {
    const U4 u = philox(key, (unsigned long long)e >> 3);
    if (EVEN) {
        const bool up = (e & 4) != 0;
        const unsigned a = up ? u.w[2] : u.w[0], b = up ? u.w[3] : u.w[1];
        v[0] = (a & 0xffffu) >= thr ? v[0] * factor : 0.f;
        v[1] = (a >> 16) >= thr ? v[1] * factor : 0.f;
        v[2] = (b & 0xffffu) >= thr ? v[2] * factor : 0.f;
        v[3] = (b >> 16) >= thr ? v[3] * factor : 0.f;
    } else {
        const int at = (int)(e & 7);
        U4 n = u;
        if (at > 4) n = philox(key, ((unsigned long long)e >> 3) + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned bits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {             // (constant indices: the words stay in registers)
                bits = at + i == j ? half_of(u, j) : bits;
                bits = at + i == j + 8 ? half_of(n, j) : bits;
            }
            v[i] = bits >= thr ? v[i] * factor : 0.f;
        }
    }
    return v;
}

static inline float drop_factor(int thr) { return thr >= 65536 ? 0.f : 65536.f / (float)(65536 - thr); }
