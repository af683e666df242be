// w4_matvec.h -- dense layers with 4-bit weights for a few rows:
//     y[m][n] = sum_k x[m][k] (code[n][k] - zero[n][k / group]) scale[n][k / group] + bias[n]
// code: 0 .. 15, two to a byte, the lower half first; zero: 0 .. 15, 8 where there are none; group: a multiple of 32, the last one may be short.
#pragma once
#include "gated_delta.h"
#include "gru_limb.h"

struct W4Args {
    const void* x; long xs;                       // [M][K], row stride in elements
    const unsigned char* codes; long cs;          // [N][(K + 1) / 2], row pitch in bytes
    const void* scales; long ss;                  // [N][groups], row stride in elements
    const unsigned char* zeros; long zs;          // [N][groups], null: 8
    const void* bias;                             // [N], null: none
    void* y; long ys;                             // [M][N], row stride in elements
    int M, K, N, group;
};

// Sixteen outputs at a time on the matrix units: x is the left operand (its rows the tile's rows, so that one row costs what sixteen do: the
// time is that of reading the codes), the weights are the right one.  A nibble becomes a 16-bit float in two instructions, a shift and an
// and-or, as 16 + code: the four bits are the significand of a number in [16, 32), exactly, in bf16 and in fp16.  The offset goes out with the
// zero, for a group: sum x (code - zero) = sum x (16 + code) - (16 + zero) sum x, sum x from one more product, with ones.  Products are exact;
// sums are fp32 and up to (16 + 15) / |code - zero| (five times on average) the magnitude they end with, which costs about two bits of 24.
// Nibble t and t + 4 of a word come out together, so x is brought into the order 0 4 1 5 2 6 3 7.  fp32 rows go in as three bf16 limbs
// (exact, see gru_limb.h), three products each.
//
// A workgroup is 16 NT outputs; its waves take every NW-th block of 128 inputs, their sums meet in LDS in a fixed order.  Lane (q, n) reads the
// codes of output n: R words at a stretch, 32 R / 8 inputs.. of each run of 32 R inputs, so that a product's 32 inputs lie in one group
// whatever its size: R = 4 where 128 divides the group, 2 where 64 does, else 1.
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ unsigned w4_load4(const unsigned char* p) { unsigned v; __builtin_memcpy(&v, p, 4); return v; }

template <typename T> struct W4X;                 // eight inputs of a row as a left operand: LIMBS fragments
template <> struct W4X<__hip_bfloat16> { enum { LIMBS = 1 }; };
template <> struct W4X<__half> { enum { LIMBS = 1 }; };
template <> struct W4X<float> { enum { LIMBS = 3 }; };

template <typename T> __device__ __forceinline__ uint4 w4_weights(unsigned w) {
    uint4 r;
    if constexpr (__is_same(T, __half)) {
        r.x = ((w << 6) & 0x03c003c0u) | 0x4c004c00u; r.y = ((w << 2) & 0x03c003c0u) | 0x4c004c00u;
        r.z = ((w >> 2) & 0x03c003c0u) | 0x4c004c00u; r.w = ((w >> 6) & 0x03c003c0u) | 0x4c004c00u;
    } else {
        r.x = ((w << 3) & 0x00780078u) | 0x41804180u; r.y = ((w >> 1) & 0x00780078u) | 0x41804180u;
        r.z = ((w >> 5) & 0x00780078u) | 0x41804180u; r.w = ((w >> 9) & 0x00780078u) | 0x41804180u;
    }
    return r;
}
template <typename T> __device__ __forceinline__ unsigned w4_one() { return __is_same(T, __half) ? 0x3c003c00u : 0x3f803f80u; }
template <typename T> __device__ __forceinline__ f32x4 w4_mfma(const uint4& a, const uint4& b, f32x4 c) {
    if constexpr (__is_same(T, __half)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else return mfma_bf16(a, b, c);
}
// eight consecutive inputs from index i of a row that ends at `end`
template <typename T> __device__ __forceinline__ void w4_inputs(const void* x, long i, int left, uint4 (&f)[W4X<T>::LIMBS]) {
    if constexpr (sizeof(T) == 2) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (left >= 8) __builtin_memcpy(&v, (const T*)x + i, 16);
        else if (left > 0) {
            unsigned short h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = e < left ? ((const unsigned short*)x)[i + e] : 0;
            v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
        f[0] = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                          __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
    } else {
        float h[8];
        if (left >= 8) __builtin_memcpy(h, (const float*)x + i, 32);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = e < left ? ((const float*)x)[i + e] : 0.f;
        uint2 a0, a1, a2, b0, b1, b2;
        split3(make_float4(h[0], h[4], h[1], h[5]), a0, a1, a2);
        split3(make_float4(h[2], h[6], h[3], h[7]), b0, b1, b2);
        f[0] = make_uint4(a0.x, a0.y, b0.x, b0.y); f[1] = make_uint4(a1.x, a1.y, b1.x, b1.y); f[2] = make_uint4(a2.x, a2.y, b2.x, b2.y);
    }
}

template <typename T, typename G, int R, int NT>
__global__ __launch_bounds__(512) void w4_matvec_kernel(W4Args a) {
    constexpr int L = W4X<T>::LIMBS, SUB = 4 / R;       // groups that a block of 128 inputs is cut into
    __shared__ float red[8][NT][16][17];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, n = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16;
    const bool row = m0 + n < a.M;                      // lane n of the left operand is row n of the tile
    const long xi = (long)(m0 + n) * a.xs;
    f32x4 y[NT];
    long crow[NT], srow[NT], zrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        y[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
        const int o = n0 + 16 * t + n < a.N ? n0 + 16 * t + n : a.N - 1;      // a tile's surplus outputs are the last one again
        crow[t] = (long)o * a.cs; srow[t] = (long)o * a.ss; zrow[t] = (long)o * a.zs;
    }
    const int bytes = (a.K + 1) >> 1;
    for (int kb = 128 * w; kb < a.K; kb += 128 * nw) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int k0 = kb + 32 * R * s, k = k0 + 8 * R * q;
            if (k0 >= a.K) break;
            unsigned c[NT][R];
            float sc[NT], zr[NT];
            const int g = k0 / a.group;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const unsigned char* p = a.codes + crow[t] + (k >> 1);
                if (k + 8 * R <= a.K) __builtin_memcpy(c[t], p, 4 * R);
                else
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        c[t][r] = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if ((k >> 1) + 4 * r + e < bytes) c[t][r] |= (unsigned)p[4 * r + e] << (8 * e);
                    }
                sc[t] = gd_load<G>(a.scales, srow[t] + g);
                zr[t] = a.zeros ? (float)a.zeros[zrow[t] + g] : 8.f;
            }
            f32x4 acc[NT], one = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = one;
            const unsigned o1 = w4_one<T>();
#pragma unroll
            for (int r = 0; r < R; ++r) {
                uint4 f[L];
                w4_inputs<T>(a.x, xi + k + 8 * r, row ? a.K - (k + 8 * r) : 0, f);
#pragma unroll
                for (int l = L - 1; l >= 0; --l) {
                    one = w4_mfma<T>(f[l], make_uint4(o1, o1, o1, o1), one);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] = w4_mfma<T>(f[l], w4_weights<T>(c[t][r]), acc[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[t][i] = __builtin_fmaf(sc[t], __builtin_fmaf(-16.f - zr[t], one[i], acc[t][i]), y[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[w][t][4 * q + i][n] = y[t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < NT * 256; e += blockDim.x) {
        const int t = e >> 8, m = (e >> 4) & 15, c = e & 15, o = n0 + 16 * t + c;
        if (m0 + m >= a.M || o >= a.N) continue;
        float v = red[0][t][m][c];
        for (int i = 1; i < nw; ++i) v += red[i][t][m][c];
        gd_store<T>(a.y, (long)(m0 + m) * a.ys + o, v + (a.bias ? gd_load<T>(a.bias, o) : 0.f));
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
