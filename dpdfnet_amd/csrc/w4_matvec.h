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
    unsigned tiles;                               // of 16 NT outputs
};

// Sixteen outputs at a time on the matrix units: x is the left operand (its rows the tile's rows, so that one row costs what sixteen do: the
// time is that of reading the codes), the weights are the right one, as code - zero, which both 16-bit types hold exactly: a term whose code is
// the zero is 0, products are exact, and the sums' roundings go by the terms alone.  A group's sum is taken before its scale.
// Four codes to a word of bytes, e = 128 + zero - code: from 128 on that is a sign and |code - zero|, below it 128 - e is, and a byte of a
// sign and 0 .. 15 is that many steps of 2^-9 as an 8-bit float (e4m3, whose steps are even up to there): 17 instructions for eight weights.  A zero
// above 15 has no such bytes; its group's scale counts as NaN.
// Codes 0 2 4 6 and 1 3 5 7 of a word come out together, so x is brought into that order.  fp32 rows go in as three bf16 limbs
// (exact, see gru_limb.h), three products each.
//
// A workgroup is 16 NT outputs; each wave takes a run of blocks of 128 inputs, two blocks in flight, and the waves' sums meet in LDS in a fixed
// order.  Lane (q, n) reads 16 bytes of output n's codes; the words then change places over q (four lane swaps), so that a product's 32 inputs are
// 32 in a row: one group whatever its size, and x is read 64 bytes of a row at a time.  R such products are of one group: 4 where 128
// divides the group, 2 where 64 does, else 1.  Scales and zeros are read for four blocks at once, those of block q by lane (q, n), and go through
// LDS as fp32: read block by block, 2 bytes of 16 rows at a time, they cost more than the codes (8192 x 32768: 25 of 72 us).
//
// Bound: reading the codes; what keeps it from a plain read's rate (24.6 us for the codes of 8192 x 32768, 5.5 TB/s) is the traffic beside them,
// x about 7 us and scales 5, and the instructions for code - zero (16 + code, with (16 + zero) sum x taken off a group's sum, took 8 for eight weights and
// 5 % less time, but its error went by 16 to 31 times |x|).  8192 x 32768, eight rows of bf16: 42.6 us, 3.3 TB/s; 4096 x 16384, one row: 11.5 us, 3.0 TB/s;
// 4096 x 4096, 16 rows of fp16: 8.0 us.
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

template <typename T> struct W4X;                 // eight inputs of a row as a left operand: LIMBS fragments
template <> struct W4X<__hip_bfloat16> { enum { LIMBS = 1 }; };
template <> struct W4X<__half> { enum { LIMBS = 1 }; };
template <> struct W4X<float> { enum { LIMBS = 3 }; };

// code - zero of four codes in bytes, as signs and magnitudes; zero: 128 + the zero in every byte
__device__ __forceinline__ unsigned w4_signed(unsigned codes, unsigned zero) {
    const unsigned e = zero - codes, over = ~e & 0x80808080u, one = over >> 7;      // over: where the code is more than the zero
    return (e ^ (over - one)) + one;
}
template <typename T> __device__ __forceinline__ uint4 w4_weights(unsigned w, unsigned zero) {
    const unsigned a = w4_signed(w & 0x0f0f0f0fu, zero), b = w4_signed(w >> 4 & 0x0f0f0f0fu, zero);
    if constexpr (__is_same(T, __half))
        return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 512.f, false)), __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 512.f, true)),
                          __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 512.f, false)), __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 512.f, true)));
    else
        return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.f, false)), __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.f, true)),
                          __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.f, false)), __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.f, true)));
}
template <typename T> __device__ __forceinline__ f32x4 w4_mfma(const uint4& a, const uint4& b, f32x4 c) {
    if constexpr (__is_same(T, __half)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else return mfma_bf16(a, b, c);
}
// eight inputs in the codes' order, as limbs
template <typename T> struct W4Eight { T v[8]; };
template <typename T> __device__ __forceinline__ void w4_limbs(const W4Eight<T>& x, uint4 (&f)[W4X<T>::LIMBS]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 v = __builtin_bit_cast(uint4, x);
        f[0] = make_uint4(__builtin_amdgcn_perm(v.y, v.x, 0x05040100u), __builtin_amdgcn_perm(v.w, v.z, 0x05040100u),
                          __builtin_amdgcn_perm(v.y, v.x, 0x07060302u), __builtin_amdgcn_perm(v.w, v.z, 0x07060302u));
    } else {
        const float* h = x.v;
        uint2 a0, a1, a2, b0, b1, b2;
        split3(make_float4(h[0], h[2], h[4], h[6]), a0, a1, a2);
        split3(make_float4(h[1], h[3], h[5], h[7]), b0, b1, b2);
        f[0] = make_uint4(a0.x, a0.y, b0.x, b0.y); f[1] = make_uint4(a1.x, a1.y, b1.x, b1.y); f[2] = make_uint4(a2.x, a2.y, b2.x, b2.y);
    }
}
// rows of 16 lanes: the upper two of a with the lower two of b; the odd ones of a with the even ones of b
__device__ __forceinline__ void w4_swap32(unsigned& a, unsigned& b) { const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false); a = r[0]; b = r[1]; }
__device__ __forceinline__ void w4_swap16(unsigned& a, unsigned& b) { const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false); a = r[0]; b = r[1]; }

constexpr int W4_WAVES = 8, W4_AHEAD = 2;        // waves of a workgroup at most; blocks of codes and inputs on their way
// a block of 128 inputs as it is loaded
template <int NT> struct W4Codes { gd_u4 v[NT]; };
template <typename T> struct W4Inputs { W4Eight<T> v[4]; };

template <typename T, typename G, int R, int NT>
__global__ __launch_bounds__(64 * W4_WAVES) void w4_matvec_kernel(W4Args a) {
    constexpr int L = W4X<T>::LIMBS, SUB = 4 / R;       // SUB: groups that a block is cut into
    typedef float2 Scales[4 * SUB][16 * NT];            // of four blocks: scale, 128 + zero in every byte
    typedef float Sums[NT][16][17];
    constexpr int ROOM = sizeof(Scales) > sizeof(Sums) ? sizeof(Scales) : sizeof(Sums);
    __shared__ __attribute__((aligned(16))) unsigned char room[W4_WAVES][ROOM];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6, n = lane & 15, q = lane >> 4;
    // Row tiles of the same outputs follow each other on one XCD, whose L2 then holds the codes: workgroups go to the eight XCDs in turn.
    unsigned tile = blockIdx.x, mt = 0;
    if (a.tiles != gridDim.x) {
        const unsigned rows = gridDim.x / a.tiles, whole = a.tiles & ~7u, width = tile < whole * rows ? 8 : a.tiles & 7, from = tile < whole * rows ? tile / (8 * rows) * 8 : whole;
        const unsigned r = tile - from * rows;
        mt = r / width; tile = from + r % width;
    }
    const long n0 = (long)tile * 16 * NT;
    const int m0 = mt * 16;
    const bool zeros = a.zeros;
    const T* xrow = (const T*)a.x + (long)(m0 + n < a.M ? m0 + n : a.M - 1) * a.xs;      // a tile's surplus rows and outputs are the last one again
    f32x4 y[NT];
    const unsigned char *crow[NT], *zrow[NT];
    const G* srow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const long o = n0 + 16 * t + n < a.N ? n0 + 16 * t + n : a.N - 1;
        crow[t] = a.codes + o * a.cs; srow[t] = (const G*)a.scales + o * a.ss;
        zrow[t] = zeros ? a.zeros + o * a.zs : (const unsigned char*)srow[t];      // where there are none, bytes of the scales: read without a branch, not used
        const float first = a.bias && w == 0 ? gd_load<T>(a.bias, o) : 0.f;      // the bias goes into the first wave's sums
        y[t] = (f32x4){first, first, first, first};
    }
    const unsigned per32 = (unsigned)a.group / 32;
    Scales& sc = *(Scales*)room[w];
    auto put = [&](const G (&s)[NT][SUB], const unsigned char (&z)[NT][SUB]) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < SUB; ++u) sc[SUB * q + u][16 * t + n] = make_float2(zeros && z[t][u] > 15 ? gd_nan() : gd_load<G>(&s[t][u], 0), __builtin_bit_cast(float, zeros ? 0x01010101u * (128u + z[t][u]) : 0x88888888u));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    // one block, the j-th of the four whose scales are in LDS
    auto add = [&](const W4Codes<NT>& codes, const W4Inputs<T>& x, int j) {
        unsigned c[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) c[t][r] = codes.v[t][r];
            w4_swap32(c[t][0], c[t][2]); w4_swap32(c[t][1], c[t][3]); w4_swap16(c[t][0], c[t][1]); w4_swap16(c[t][2], c[t][3]);
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            f32x4 acc[NT];
            float2 s[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) { acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f}; s[t] = sc[SUB * j + u][16 * t + n]; }
#pragma unroll
            for (int r = R * u; r < R * (u + 1); ++r) {
                uint4 f[L];
                w4_limbs<T>(x.v[r], f);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 wt = w4_weights<T>(c[t][r], __builtin_bit_cast(unsigned, s[t].y));
#pragma unroll
                    for (int l = L - 1; l >= 0; --l) acc[t] = w4_mfma<T>(f[l], wt, acc[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[t][i] = __builtin_fmaf(s[t].x, acc[t][i], y[t][i]);
        }
    };
    // the last wave takes what is left of the inputs, and nothing else where the others have no more to do for it
    const int blocks = a.K >> 7, left = a.K & 127, alone = left && nw > 1 && (blocks + nw - 2) / (nw - 1) == (blocks + nw - 1) / nw;
    const int per = (blocks + nw - 1) / nw, first = w * per, end = alone && w == nw - 1 ? 0 : blocks < first + per ? blocks : first + per;
    if (first < end) {
        // this lane's group in the next four blocks: that of the first 32 inputs of block q
        unsigned g = 4 * (unsigned)(first + q) / per32, in = 4 * (unsigned)(first + q) - g * per32;
        const unsigned dg = 16 / per32, din = 16 - dg * per32, top = 4 * (unsigned)(blocks - 1) / per32, most = ((unsigned)a.K - 1) / (unsigned)a.group;
        auto scales = [&](G (&s)[NT][SUB], unsigned char (&z)[NT][SUB]) {
            const unsigned g0 = g < top ? g : top;                 // behind the last block: read, not used
            if (SUB == 1 || per32 == R)
#pragma unroll
                for (int t = 0; t < NT; ++t) { __builtin_memcpy(s[t], srow[t] + g0, SUB * sizeof(G)); __builtin_memcpy(z[t], zrow[t] + g0, SUB); }
            else
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    const unsigned g1 = g0 + (in + R * u >= per32), gu = g1 < most ? g1 : most;        // a group is longer than half a block: one border at most
#pragma unroll
                    for (int t = 0; t < NT; ++t) { s[t][u] = srow[t][gu]; z[t][u] = zrow[t][gu]; }
                }
            g += dg; in += din;
            if (in >= per32) { in -= per32; ++g; }
        };
        auto codes = [&](int i, W4Codes<NT>& c) {
            const int at = i < end ? i : end - 1;                  // behind the last block: read, not used
#pragma unroll
            for (int t = 0; t < NT; ++t) __builtin_memcpy(&c.v[t], crow[t] + 64L * at + 16 * q, 16);
        };
        auto inputs = [&](int i, W4Inputs<T>& x) {
            const int at = i < end ? i : end - 1;
#pragma unroll
            for (int r = 0; r < 4; ++r) __builtin_memcpy(&x.v[r], xrow + 128L * at + 32 * r + 8 * q, sizeof(x.v[r]));
        };
        G s[NT][SUB];
        unsigned char z[NT][SUB];
        W4Codes<NT> c[W4_AHEAD];
        W4Inputs<T> x[W4_AHEAD];
        scales(s, z);
#pragma unroll
        for (int j = 0; j < W4_AHEAD; ++j) {
            codes(first + j, c[j]);
            inputs(first + j, x[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
        int i = first;
        for (; i + 4 < end; i += 4) {
            put(s, z);
            scales(s, z);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                add(c[j % W4_AHEAD], x[j % W4_AHEAD], j);
                __builtin_amdgcn_sched_barrier(0);                 // the compiler would put the loads off to the end, behind all four blocks
                codes(i + j + W4_AHEAD, c[j % W4_AHEAD]);
                inputs(i + j + W4_AHEAD, x[j % W4_AHEAD]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        put(s, z);                                                 // one to four blocks, nothing to load behind them
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j >= end) break;
            add(c[j % W4_AHEAD], x[j % W4_AHEAD], j);
            if (j + W4_AHEAD < 4) {
                codes(i + j + W4_AHEAD, c[j % W4_AHEAD]);
                inputs(i + j + W4_AHEAD, x[j % W4_AHEAD]);
            }
        }
    }
    if (w == nw - 1 && left) {
        const int k0 = a.K - left, last = (a.K - 1) >> 1;
        unsigned char v[NT][16], z[NT][SUB];
        G s[NT][SUB];
        T xv[32];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int p = (k0 >> 1) + 16 * q + e;
                v[t][e] = crow[t][p < last ? p : last];            // behind the end any code will do, x is 0 there
            }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int i = k0 + (e & ~7) * 4 + 8 * q + (e & 7);
            xv[e] = xrow[i < a.K ? i : a.K - 1];
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int k = k0 + 32 * R * u, g = (k < a.K ? k : a.K - 1) / a.group;
#pragma unroll
            for (int t = 0; t < NT; ++t) { s[t][u] = srow[t][g]; z[t][u] = zrow[t][g]; }
        }
        __builtin_amdgcn_sched_barrier(0);                         // all of the loads before the first use of one
        W4Codes<NT> c;
        W4Inputs<T> x;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) c.v[t][r] = v[t][4 * r] | v[t][4 * r + 1] << 8 | v[t][4 * r + 2] << 16 | (unsigned)v[t][4 * r + 3] << 24;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
                if (k0 + 32 * R * u >= a.K) s[t][u] = (G)0.f;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) x.v[e / 8].v[e & 7] = k0 + (e & ~7) * 4 + 8 * q + (e & 7) < a.K ? xv[e] : (T)0.f;
        put(s, z);
        add(c, x, 0);
    }
    __syncthreads();
    Sums& mine = *(Sums*)room[w];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[t][4 * q + i][n] = y[t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < NT * 256; e += blockDim.x) {
        const int t = e >> 8, m = (e >> 4) & 15, c = e & 15;
        const long o = n0 + 16 * t + c;
        if (m0 + m >= a.M || o >= a.N) continue;
        float v[W4_WAVES];
#pragma unroll
        for (int i = 0; i < W4_WAVES; ++i) v[i] = (*(Sums*)room[i])[t][m][c];
#pragma unroll
        for (int i = 1; i < W4_WAVES; ++i) v[0] += i < nw ? v[i] : 0.f;
        gd_store<T>(a.y, (long)(m0 + m) * a.ys + o, v[0]);
    }
}

// Codes, scales and zeros of a weight matrix, one wave per group.  With zeros: the group's range with 0 in it over 15 steps; without: its largest
// magnitude over 7 steps around code 8.  The scale is rounded to its type first, codes are the nearest (ties to even) under the rounded scale.
// A group with a weight that is not finite has NaN for its scale, and its zero for codes.
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
    for (long e = (long)blockIdx.x * 4 + (threadIdx.x >> 6); e < (long)a.N * a.groups; e += (long)gridDim.x * 4) {
        const int n = (int)(e / a.groups), g = (int)(e - (long)n * a.groups);
        const int k0 = g * a.group, k1 = a.K - k0 < a.group ? a.K : k0 + a.group;
        const long wb = (long)n * a.ws;
        float lo = 0.f, hi = 0.f;
        bool bad = false;
        for (int k = k0 + lane; k < k1; k += 64) {
            const float v = gd_load<T>(a.w, wb + k);
            bad |= !gd_finite(v);
            lo = v < lo ? v : lo; hi = v > hi ? v : hi;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { lo = fminf(lo, __shfl_xor(lo, o)); hi = fmaxf(hi, __shfl_xor(hi, o)); }
        float s = a.zeros ? (gd_finite(hi - lo) ? (hi - lo) / 15.f : hi / 15.f - lo / 15.f) : fmaxf(hi, -lo) / 7.f;      // a range may leave fp32, a step does not
        if (__any(bad)) s = gd_nan();                 // no code stands for it: the layer's output shows it
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
}
