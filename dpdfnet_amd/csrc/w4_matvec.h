// w4_matvec.h -- dense layers with 4-bit weights for a few rows:
//     y[m][n] = sum_k x[m][k] (code[n][k] - zero[n][k / group]) scale[n][k / group] + bias[n]
// code: 0 .. 15, two to a byte, the lower half first; zero: 0 .. 15, 8 where there are none; group: a multiple of 32, the last one may be short.
#pragma once
#include "gated_delta.h"

struct W4Args {
    const void* x; long xs;                       // [M][K], row stride in elements
    const unsigned char* codes; long cs;          // [N][(K + 1) / 2], row pitch in bytes
    const void* scales; long ss;                  // [N][groups], row stride in elements
    const unsigned char* zeros; long zs;          // [N][groups], null: 8
    const void* bias;                             // [N], null: none
    void* y; long ys;                             // [M][N], row stride in elements
    int M, K, N, group;
};

// One wave per output, byte by byte: any alignment.  Eight rows of x at a time.
template <typename T, typename G>
__global__ __launch_bounds__(256) void w4_matvec_any_kernel(W4Args a) {
    const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6), m0 = blockIdx.y * 8;
    if (n >= a.N) return;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const unsigned char* cp = a.codes + (long)n * a.cs;
    for (int k = 2 * lane; k < a.K; k += 128) {
        const unsigned c = cp[k >> 1];
        const int g = k / a.group;
        const float s = gd_load<G>(a.scales, (long)n * a.ss + g), z = a.zeros ? (float)a.zeros[(long)n * a.zs + g] : 8.f;
        const float w0 = ((float)(c & 15) - z) * s, w1 = ((float)(c >> 4) - z) * s;
        const bool two = k + 1 < a.K;
#pragma unroll
        for (int m = 0; m < 8; ++m)
            if (m0 + m < a.M) {
                const long xi = (long)(m0 + m) * a.xs + k;
                acc[m] = __builtin_fmaf(gd_load<T>(a.x, xi), w0, acc[m]);
                if (two) acc[m] = __builtin_fmaf(gd_load<T>(a.x, xi + 1), w1, acc[m]);
            }
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) acc[m] += __shfl_xor(acc[m], o);
        if (lane == 0 && m0 + m < a.M) gd_store<T>(a.y, (long)(m0 + m) * a.ys + n, acc[m] + (a.bias ? gd_load<T>(a.bias, n) : 0.f));
    }
}

// Codes, scales and zeros of a weight matrix, one wave per group.  With zeros: the group's range with 0 in it over 15 steps; without: its largest
// magnitude over 7 steps around code 8.  The scale is rounded to its type first, codes are the nearest (ties to even) under the rounded scale.
struct W4QuantArgs {
    const void* w; long ws;                       // [N][K], row stride in elements
    unsigned char* codes; long cs;
    void* scales; long ss;
    unsigned char* zeros; long zs;                // null: symmetric
    int N, K, group, groups;
};

template <typename T>
__global__ __launch_bounds__(256) void w4_quantize_kernel(W4QuantArgs a) {
    const int lane = threadIdx.x & 63;
    const long e = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (e >= (long)a.N * a.groups) return;
    const int n = (int)(e / a.groups), g = (int)(e - (long)n * a.groups);
    const int k0 = g * a.group, k1 = a.K - k0 < a.group ? a.K : k0 + a.group;
    const long wb = (long)n * a.ws;
    float lo = 0.f, hi = 0.f;
    for (int k = k0 + lane; k < k1; k += 64) {
        const float v = gd_load<T>(a.w, wb + k);
        lo = v < lo ? v : lo; hi = v > hi ? v : hi;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { lo = fminf(lo, __shfl_xor(lo, o)); hi = fmaxf(hi, __shfl_xor(hi, o)); }
    float s = a.zeros ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f;
    if (lane == 0) gd_store<T>(a.scales, (long)n * a.ss + g, s);
    if constexpr (sizeof(T) == 2) {               // the value as it is stored
        if constexpr (__is_same(T, __half)) s = __half2float(__float2half(s));
        else s = (float)(__bf16)s;
    }
    const float z = a.zeros ? (s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f) : 8.f;
    if (a.zeros && lane == 0) a.zeros[(long)n * a.zs + g] = (unsigned char)z;
    for (int k = k0 + 2 * lane; k < k1; k += 128) {
        unsigned c = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float v = k + i < k1 ? gd_load<T>(a.w, wb + k + i) : 0.f;
            const float r = s > 0.f ? rintf(v / s) + z : z;
            c |= (unsigned)fminf(fmaxf(r, 0.f), 15.f) << (4 * i);
        }
        a.codes[(long)n * a.cs + (k >> 1)] = (unsigned char)c;
    }
}
