// gated_delta.h -- the gated delta rule: a recurrence over frames whose state is a matrix S [Dk][Dv] (fp32) per sequence and value head,
//     S' = exp(g_t) S_{t-1};   e_t = beta_t (v_t - S'^T k_t);   S_t = S' + k_t e_t^T;   o_t = scale S_t^T q_t
// in the two forms that the GRU scans have: hop by hop with the state in HBM (gated_delta_step_kernel) and over whole clips
// (gated_delta_clip_kernel).  Value head h reads key head h / (Hv / Hk).
#pragma once
#include "common.h"
#include "gru_limb.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

struct GatedDeltaArgs {
    const void *q, *k, *v, *g, *beta;
    void* out;
    const float* state_in;            // [B][Hv][Dk][Dv], null: zeros
    float* state_out;                 // the same layout (may be state_in itself), null: not wanted
    const int* lengths;               // [B], null: T each
    const unsigned char* active;      // [B], null: all
    long qs[3], ks[3], vs[3], gs[3], bs[3], os[3];      // strides in elements: batch, frame, head
    int B, T, Hk, Hv, Dk, Dv;
    int strips;                       // workgroups (clip) or waves (step) per head
    int gate;                         // type of g and beta: 0 fp32, 1 fp16, 2 bf16
    int sorted;                       // clips: the longest first (batch: at most GD_RANKED)
    int whole, even;                  // k and q can be read in pieces of eight values (hops: v in pieces of four too), out written in pieces of four
    int segments, seg;                // clips: how many pieces a clip is cut into, and their frames
    float* starts;                    // [segments][B Hv][Dk][Dv]: the states that segments start with (the first: if there is a state_in); before they are joined, what each adds
    float* moves;                     // [segments][B Hv][Dk][Dk]: segment i's effect on the state before it, i = 1 .. segments - 2
    float scale;
};

template <typename T> __device__ __forceinline__ float gd_load(const void* p, long i);
template <> __device__ __forceinline__ float gd_load<float>(const void* p, long i) { return ((const float*)p)[i]; }
template <> __device__ __forceinline__ float gd_load<__half>(const void* p, long i) { return __half2float(((const __half*)p)[i]); }
template <> __device__ __forceinline__ float gd_load<__hip_bfloat16>(const void* p, long i) {
    return __builtin_bit_cast(float, (unsigned)((const unsigned short*)p)[i] << 16);
}
template <typename T> __device__ __forceinline__ void gd_store(void* p, long i, float v);
template <> __device__ __forceinline__ void gd_store<float>(void* p, long i, float v) { ((float*)p)[i] = v; }
template <> __device__ __forceinline__ void gd_store<__half>(void* p, long i, float v) { ((__half*)p)[i] = __float2half(v); }
template <> __device__ __forceinline__ void gd_store<__hip_bfloat16>(void* p, long i, float v) { ((__bf16*)p)[i] = (__bf16)v; }

__device__ __forceinline__ float gd_gate(const void* p, long i, int type) {
    return type == 0 ? gd_load<float>(p, i) : type == 1 ? gd_load<__half>(p, i) : gd_load<__hip_bfloat16>(p, i);
}
__device__ __forceinline__ bool gd_finite(float v) { return (__builtin_bit_cast(unsigned, v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float gd_nan() { return __builtin_bit_cast(float, 0x7fc00000u); }

// What a hop or a chunk reads and writes goes through buffer descriptors that end with it: behind that, and at GD_OUT, loads give 0 and stores do
// nothing, so that there is no branch around a load (behind one the compiler cannot count the loads in flight and waits for them), no clamp
// and 32 bits of address.
constexpr unsigned GD_OUT = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t gd_buffer(const void* base, long first, long count, int elem) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + first * elem), 0, (int)(count * elem), 0x00027000);
}
template <typename T> struct GdRow { T v[8]; };
typedef unsigned gd_u4 __attribute__((ext_vector_type(4)));
// eight values of a row, at `off` (whole: in one piece), the first `left` of them
template <typename T> __device__ __forceinline__ GdRow<T> gd_row(__amdgpu_buffer_rsrc_t r, unsigned off, int left, bool whole) {
    GdRow<T> x;
    if (whole) {
        const unsigned o = left > 0 ? off : GD_OUT;
        gd_u4 v[sizeof(T) / 2];
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e) v[e] = __builtin_amdgcn_raw_buffer_load_b128(r, o + 16 * e, 0, 0);
        __builtin_memcpy(&x, v, sizeof(x));
    } else
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned o = e < left ? off + e * (unsigned)sizeof(T) : GD_OUT;
            if constexpr (sizeof(T) == 2) { const unsigned short v = __builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0); __builtin_memcpy(&x.v[e], &v, 2); }
            else { const unsigned v = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0); __builtin_memcpy(&x.v[e], &v, 4); }
        }
    return x;
}
template <typename T> __device__ __forceinline__ unsigned gd_get(__amdgpu_buffer_rsrc_t r, unsigned off) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
}
template <typename T> __device__ __forceinline__ float gd_value(unsigned raw) {
    if constexpr (__is_same(T, __hip_bfloat16)) return __builtin_bit_cast(float, raw << 16);
    else if constexpr (__is_same(T, __half)) return (float)__builtin_bit_cast(_Float16, (unsigned short)raw);
    else return __builtin_bit_cast(float, raw);
}
// four columns of a row, `left` of them inside (even: in one piece)
template <typename T> __device__ __forceinline__ void gd_put(__amdgpu_buffer_rsrc_t r, unsigned off, const f32x4& v, int left, bool even) {
    if constexpr (sizeof(T) == 4) {
        if (even) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(gd_u4, v), r, left > 0 ? off : GD_OUT, 0, 0);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = v[i];                      // a bit cast of v[i] itself takes element 0
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), r, i < left ? off + 4 * i : GD_OUT, 0, 0);
            }
    } else {
        typedef unsigned u2 __attribute__((ext_vector_type(2)));
        u2 w;
        if constexpr (__is_same(T, __hip_bfloat16)) w = (u2){pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
        else {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            w = (u2){__builtin_bit_cast(unsigned, (h2){(_Float16)v[0], (_Float16)v[1]}), __builtin_bit_cast(unsigned, (h2){(_Float16)v[2], (_Float16)v[3]})};
        }
        if (even) __builtin_amdgcn_raw_buffer_store_b64(w, r, left > 0 ? off : GD_OUT, 0, 0);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_buffer_store_b16((unsigned short)(w[i / 2] >> (16 * (i & 1))), r, i < left ? off + 2 * i : GD_OUT, 0, 0);
    }
}
// N bytes into registers
template <int N> __device__ __forceinline__ void gd_piece(__amdgpu_buffer_rsrc_t r, unsigned off, void* to) {
    if constexpr (N == 2) { const unsigned short v = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0); __builtin_memcpy(to, &v, 2); }
    else if constexpr (N == 4) { const unsigned v = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0); __builtin_memcpy(to, &v, 4); }
    else if constexpr (N == 8) { const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0); __builtin_memcpy(to, &v, 8); }
    else { const gd_u4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0); __builtin_memcpy(to, &v, 16); }
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Hops: one wave = 32 columns of one head's state, all Dk rows of them in registers for the T hops of the call; lane (rg, cl) holds the
// DKP / 8 rows rg * DKP / 8 + j of the columns 4 cl .. 4 cl + 3.  A hop needs S'^T k and S'^T q; with o = scale (S'^T q + (q.k) e) both are
// sums over the OLD state, so that one butterfly over the eight row groups serves them, and no wave waits for another.
// Rows behind Dk are loaded as 0; a column behind Dv holds what comes next in memory, meets no other column and is not stored.
// Bound: HBM, the state read once and written once (192 streams of 32 heads of 128 x 128, two hops: 164 us, 5.0 TB/s; a large copy does 5.1).
// ---------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int R> struct GdHop { T k[R], q[R], v[4]; float g, beta; };      // what a lane reads for a hop

template <typename T, int DKP, bool WHOLE>
__global__ __launch_bounds__(64) void gated_delta_step_kernel(GatedDeltaArgs a) {
    constexpr int R = DKP / 8, E = sizeof(T);
    const int lane = threadIdx.x, cl = lane & 7, rg = lane >> 3;
    const unsigned head = blockIdx.x / (unsigned)a.strips, strip = blockIdx.x - head * a.strips, b = head / (unsigned)a.Hv, h = head - b * a.Hv, hk = h / (unsigned)(a.Hv / a.Hk);
    if (a.active && !a.active[b]) return;
    const int c0 = 32 * (int)strip + 4 * cl, r0 = rg * R;
    const long sbase = (long)head * a.Dk * a.Dv;
    const auto si = gd_buffer(a.state_in, sbase, (long)a.Dk * a.Dv, 4), so = gd_buffer(a.state_out, sbase, (long)a.Dk * a.Dv, 4);
    f32x4 S[R];
#pragma unroll
    for (int j = 0; j < R; ++j)
        S[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(si, r0 + j < a.Dk ? ((unsigned)(r0 + j) * a.Dv + c0) * 4 : GD_OUT, 0, 0));
    const long qb = (long)b * a.qs[0] + (long)hk * a.qs[2], kb = (long)b * a.ks[0] + (long)hk * a.ks[2];
    const long vb = (long)b * a.vs[0] + (long)h * a.vs[2], ob = (long)b * a.os[0] + (long)h * a.os[2];
    const long gb = (long)b * a.gs[0] + (long)h * a.gs[2], bb = (long)b * a.bs[0] + (long)h * a.bs[2];
    auto fetch = [&](int t) {
        GdHop<T, R> x;
        const auto rk = gd_buffer(a.k, kb + t * a.ks[1], a.Dk, E), rq = gd_buffer(a.q, qb + t * a.qs[1], a.Dk, E), rv = gd_buffer(a.v, vb + t * a.vs[1], a.Dv, E);
        if constexpr (WHOLE) {
            // rows in pieces of 4 bytes or more; one that begins inside Dk ends there
            constexpr int P = R * E % 16 == 0 ? 16 : R * E % 8 == 0 ? 8 : 4;
#pragma unroll
            for (int e = 0; e < R * E / P; ++e) {
                const unsigned o = r0 * E + P * e < (unsigned)(a.Dk * E) ? r0 * E + P * e : GD_OUT;
                gd_piece<P>(rk, o, (char*)x.k + P * e); gd_piece<P>(rq, o, (char*)x.q + P * e);
            }
            gd_piece<4 * E>(rv, c0 * E, x.v);
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const unsigned o = r0 + j < a.Dk ? (r0 + j) * E : GD_OUT;
                gd_piece<E>(rk, o, &x.k[j]); gd_piece<E>(rq, o, &x.q[j]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) gd_piece<E>(rv, (c0 + i) * E, &x.v[i]);
        }
        x.g = gd_gate(a.g, gb + t * a.gs[1], a.gate); x.beta = gd_gate(a.beta, bb + t * a.bs[1], a.gate);
        return x;
    };
    GdHop<T, R> next = fetch(0);
    for (int t = 0; t < a.T; ++t) {
        const GdHop<T, R> now = next;
        if (t + 1 < a.T) next = fetch(t + 1);
        const float alpha = __expf(now.g);
        f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sq = sk;
        float qk = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float k = gd_load<T>(&now.k[j], 0), q = gd_load<T>(&now.q[j], 0);
            qk = __builtin_fmaf(q, k, qk);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                S[j][i] *= alpha;
                sk[i] = __builtin_fmaf(k, S[j][i], sk[i]);
                sq[i] = __builtin_fmaf(q, S[j][i], sq[i]);
            }
        }
#pragma unroll
        for (int m = 8; m < 64; m <<= 1) {
            qk += __shfl_xor(qk, m);
#pragma unroll
            for (int i = 0; i < 4; ++i) { sk[i] += __shfl_xor(sk[i], m); sq[i] += __shfl_xor(sq[i], m); }
        }
        f32x4 e, o;
#pragma unroll
        for (int i = 0; i < 4; ++i) { e[i] = now.beta * (gd_load<T>(&now.v[i], 0) - sk[i]); o[i] = a.scale * __builtin_fmaf(qk, e[i], sq[i]); }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float k = gd_load<T>(&now.k[j], 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][i] = __builtin_fmaf(k, e[i], S[j][i]);
        }
        gd_put<T>(gd_buffer(a.out, ob + t * a.os[1], a.Dv, E), c0 * E, o, rg == 0 ? a.Dv - c0 : 0, WHOLE);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) gd_put<float>(so, ((unsigned)(r0 + j) * a.Dv + c0) * 4, S[j], r0 + j < a.Dk ? a.Dv - c0 : 0, WHOLE);
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Clips: chunks of C frames.  With gamma = the running sum of g inside the chunk, d_ij = exp(gamma_i - gamma_j) and S the state before it,
//     A_ij = beta_i d_ij k_i.k_j (j < i),   (I + A) u = beta (v - exp(gamma) (K S)),
//     O = scale (exp(gamma) (Q S) + P u),   P_ij = d_ij q_i.k_j (j <= i),   S <- exp(gamma_C) S + K^T (exp(gamma_C - gamma) u):
// matrix products, and 16 dependent steps for the inverses of the 16 x 16 diagonal blocks of I + A where the definition has C.
//
// A workgroup is one head and 16 NW columns: wave w owns 16 columns of S, u and O in the matrix units' result layout (row 4 q + i, column n),
// in which a result IS the next product's right operand -- K slot 8 q + 4 h + i of two 16-row blocks is row 4 q + i of block h -- so that
// K S -> u -> P u, K^T u chain in registers, and the waves meet only over the chunk's K, Q, A and P in LDS, which are laid out in that order.
//
// Every fp32 operand goes in as bf16 limbs (split3 of gru_limb.h: exact), products of limbs whose indices add up to more than 2 (2^-24 of the
// term) left out; bf16 values of k and q are one limb, fp16 two, fp32 three.  Outputs of 16 bits take as many limbs as the state's path: where a key
// is written again, Q S and P u cancel, and what counts is 2^-24 of the terms, not the rounding of the result.
//
// Where there are fewer heads than the chip holds workgroups, the frames are cut into segments.  A segment's effect on the state before it is
// linear, S -> M S + N: MOVE runs a segment from S = 0 with its v (N; the first one from the clip's state) and from the unit matrix without (M, Dk
// columns more), no outputs;
// gated_delta_join_kernel then walks the segments (N becomes the state that the next one starts with), and the segments run as
// clips of their own.  About two and a half times the work, over `segments` times the workgroups.
//
// Bound: neither bytes nor products but the chain through a chunk, about 14 thousand cycles of which two workgroups on a CU overlap: K and Q into LDS
// 1.4 thousand, the next chunk's loads 1 to 1.8, the blocks of A and P 1.8, inverses and the other blocks 2, K S and Q S 2, u, the outputs
// and S 5 (4 heads of 64, bf16; vector units 42 % busy, matrix units 27 %; counted with outputs of two limbs, 6 % faster).  The first four do not
// depend on S and could be made ahead of it.  256 clips of 334 to 1003 frames, 4 heads of 64, bf16: 176 us, 2.1 TB/s; one recording of 16384 frames,
// 16 heads of 128: 407 us, in 16 segments (2.26 ms in one).  Chunks of 32 frames in 16-bit types took a third longer.
//
// gamma and its differences are 64-bit: they are small differences of long sums.  A non-finite k, g or beta makes its head's outputs from its
// frame on, and the final state, NaN; a non-finite v does that to its column; earlier frames stay as they are (the products run over all
// frames of the chunk, so that such values are taken out of the operands first).
// ---------------------------------------------------------------------------------------------------------------------------------------
template <typename T> struct GdIn;
template <> struct GdIn<__hip_bfloat16> { enum { L = 1 }; };
template <> struct GdIn<__half> { enum { L = 2 }; };
template <> struct GdIn<float> { enum { L = 3 }; };

// the running sum over a wave's lanes
__device__ __forceinline__ double gd_scan(double v) {
#define GD_STEP_(ctrl, rows) { \
        const unsigned long b = __builtin_bit_cast(unsigned long, v); \
        const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)b, ctrl, rows, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), ctrl, rows, 0xf, false); \
        v += __builtin_bit_cast(double, (unsigned long)hi << 32 | lo); }
    GD_STEP_(0x111, 0xf) GD_STEP_(0x112, 0xf) GD_STEP_(0x114, 0xf) GD_STEP_(0x118, 0xf)      // row_shr 1, 2, 4, 8: inside 16 lanes
    GD_STEP_(0x142, 0xa) GD_STEP_(0x143, 0xc)                                                // lane 15's sum to the next row, lane 31's to the upper half
#undef GD_STEP_
    return v;
}
// the row's limbs, 8 x 16 bit each; true where a value is not finite
template <typename T> __device__ __forceinline__ bool gd_limbs(const GdRow<T>& r, uint4 (&f)[GdIn<T>::L]) {
    if constexpr (GdIn<T>::L == 1) {
        f[0] = __builtin_bit_cast(uint4, r);
        // an exponent of all ones carries into the sign's place
        const unsigned t = ((f[0].x & 0x7f807f80u) + 0x00800080u) | ((f[0].y & 0x7f807f80u) + 0x00800080u) | ((f[0].z & 0x7f807f80u) + 0x00800080u) | ((f[0].w & 0x7f807f80u) + 0x00800080u);
        return t & 0x80008000u;
    } else {
        float x[8], t = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = gd_load<T>(r.v, e); t = __builtin_fmaf(x[e], 0.f, t); }
        uint2 l[2][3];
        split3(make_float4(x[0], x[1], x[2], x[3]), l[0][0], l[0][1], l[0][2]);
        split3(make_float4(x[4], x[5], x[6], x[7]), l[1][0], l[1][1], l[1][2]);
#pragma unroll
        for (int e = 0; e < GdIn<T>::L; ++e) f[e] = make_uint4(l[0][e].x, l[0][e].y, l[1][e].x, l[1][e].y);
        return !(t == 0.f);
    }
}
// the limbs of four values into the lower or upper half of a fragment of each
template <int N> __device__ __forceinline__ void gd_split(const f32x4& v, uint4 (&f)[N], int half) {
    float r0 = v[0], r1 = v[1], r2 = v[2], r3 = v[3];
#pragma unroll
    for (int l = 0; l < N; ++l) {
        const unsigned p = pk_bf16(r0, r1), s = pk_bf16(r2, r3);
        if (half) { f[l].z = p; f[l].w = s; } else { f[l].x = p; f[l].y = s; }
        if (l + 1 < N) { r0 -= bf_lo(p); r1 -= bf_hi(p); r2 -= bf_lo(s); r3 -= bf_hi(s); }
    }
}
// acc + a b over 32 slots, NA limbs by NB limbs, pairs up to 2
template <int NA, int NB> __device__ __forceinline__ f32x4 gd_mul(const uint4 (&a)[NA], const uint4 (&b)[NB], f32x4 acc) {
#pragma unroll
    for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int l = 0; l < NA; ++l)
            if (o - l >= 0 && o - l < NB) acc = mfma_bf16(a[l], b[o - l], acc);
    return acc;
}
// the same over 16 slots, those of the lower halves: two limbs of a side share a fragment
__device__ __forceinline__ uint4 gd_two(const uint4& x, const uint4& y) { return make_uint4(x.x, x.y, y.x, y.y); }
__device__ __forceinline__ f32x4 gd_mul16(const uint2 (&a)[3], const uint4* b, f32x4 acc) {
    const uint4 a01 = make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
    acc = mfma_bf16(make_uint4(a[0].x, a[0].y, a[2].x, a[2].y), gd_two(b[2], b[0]), acc);
    acc = mfma_bf16(a01, gd_two(b[1], b[1]), acc);
    return mfma_bf16(a01, gd_two(b[0], b[0]), acc);
}
// The transposes of such products: the two operands' layouts are the same, so the other order gives the transpose, a lane four columns of a row.
template <int NA, int NB> __device__ __forceinline__ f32x4 gd_mul_t(const uint4 (&a)[NA], const uint4 (&b)[NB], f32x4 acc) {
#pragma unroll
    for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int l = 0; l < NA; ++l)
            if (o - l >= 0 && o - l < NB) acc = mfma_bf16(b[o - l], a[l], acc);
    return acc;
}
__device__ __forceinline__ f32x4 gd_mul16_t(const uint2 (&a)[3], const uint4* b, f32x4 acc) {
    const uint4 a01 = make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
    acc = mfma_bf16(gd_two(b[2], b[0]), make_uint4(a[0].x, a[0].y, a[2].x, a[2].y), acc);
    acc = mfma_bf16(gd_two(b[1], b[1]), a01, acc);
    return mfma_bf16(gd_two(b[0], b[0]), a01, acc);
}
// four rows of a column out of rows in LDS: lane p of 16 gives the address of row p / 4, columns 4 (p % 4) .. + 3 and gets column p of all four
typedef short gd_s4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 gd_column(const unsigned short* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gd_s4*)p));
}

// The clip that is `place`-th in a batch from long to short: thread i counts the clips before clip i, by chunks of 16 frames and number.  Workgroups
// start in this order, so that no long clip begins when the others are done; the order has no part in the results.
constexpr int GD_RANKED = 256;                             // clips of a batch that is put in order, at most (and at most a workgroup's threads)
__device__ __forceinline__ int gd_ranked(const GatedDeltaArgs& a, int place) {
    __shared__ __attribute__((aligned(16))) unsigned keys[GD_RANKED];
    __shared__ int found;
    const int i = threadIdx.x;
    unsigned mine = 0;
    if (i < a.B) {
        const int n = a.lengths[i];
        mine = (n < 0 ? 0u : (unsigned)(n > a.T ? a.T : n) >> 4) << 8 | (255u - i);
    }
    for (int j = i; j < GD_RANKED; j += blockDim.x) keys[j] = j == i ? mine : 0;
    __syncthreads();
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < GD_RANKED; j += 4) {
        const uint4 k = *(const uint4*)&keys[j];
        before += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
    }
    if (i < a.B && before == place) found = i;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(found);
}

template <typename T, int DKP, int NW, int C, bool MOVE>
__global__ __launch_bounds__(64 * NW, 2) void gated_delta_clip_kernel(GatedDeltaArgs a) {
    constexpr int L = GdIn<T>::L, NB = DKP / 16, NC = DKP / 32, CB = C / 16, CC = C / 32, LDK = DKP + 8, E = sizeof(T);
    constexpr int BLOCKS = CB * (CB + 1) / 2;
    constexpr int ITEMS = (C / 2 * (DKP / 8) + 64 * NW - 1) / (64 * NW);
    // blocks of A below the diagonal and of P on and below it, two neighbours of a row to a fragment: row bi of A starts at bi^2 / 4, of P at (bi + 1)^2 / 4
    constexpr int ASLOTS = CB * CB / 4, PSLOTS = (CB + 1) * (CB + 1) / 4;
    __shared__ __attribute__((aligned(16))) unsigned short Kr[L][C][LDK], Qr[MOVE ? 1 : L][MOVE ? 1 : C][LDK];
    __shared__ __attribute__((aligned(16))) uint2 Af[ASLOTS][3][64][2], Pf[MOVE ? 1 : PSLOTS][3][64][2];
    __shared__ __attribute__((aligned(16))) float Ad[CB][16][20];
    __shared__ __attribute__((aligned(16))) float2 gam[C];
    __shared__ __attribute__((aligned(16))) float eg[C], ee[C], bt[C];
    __shared__ int kbad[2];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, q = lane >> 4;
    const unsigned unit = blockIdx.x / (unsigned)a.strips, place = unit / (unsigned)a.segments;               // (head, segment)
    const int sg = (int)(unit - place * a.segments);
    const long heads = gridDim.x / (unsigned)a.strips / (unsigned)a.segments;
    int b = (int)(place / (unsigned)a.Hv);
    const int h = (int)(place - (unsigned)b * a.Hv), hk = h / (a.Hv / a.Hk);
    long head = place;
    if (!MOVE && a.sorted) { b = gd_ranked(a, b); head = (long)b * a.Hv + h; }
    int col = 16 * NW * (int)(blockIdx.x - unit * a.strips) + 16 * w + n;
    const int vcols = (a.Dv + 15) & ~15;
    const bool eye = MOVE && col >= vcols;                 // a column of the unit matrix: the same for a wave
    if (MOVE && (sg == a.segments - 1 || (sg == 0 && 16 * NW * (int)(blockIdx.x - unit * a.strips) >= vcols))) return;
    if (eye) col -= vcols;
    const bool cin = col < (eye ? a.Dk : a.Dv);
    int len = a.lengths ? a.lengths[b] : a.T;
    len = len < 0 ? 0 : len > a.T ? a.T : len;
    const int first = sg * a.seg;
    if (len - first > a.seg) len = first + a.seg;          // the segment's end
    const long qb = (long)b * a.qs[0] + (long)hk * a.qs[2], kb = (long)b * a.ks[0] + (long)hk * a.ks[2];
    const long vb = (long)b * a.vs[0] + (long)h * a.vs[2], ob = (long)b * a.os[0] + (long)h * a.os[2];
    const long gb = (long)b * a.gs[0] + (long)h * a.gs[2], bb = (long)b * a.bs[0] + (long)h * a.bs[2];
    const long sb = head * a.Dk * a.Dv + col;
    // the last segment may write the final state over state_in: the first one starts from the copy of it that the join, the launch before, has left
    const float* from = MOVE ? (sg == 0 ? a.state_in : nullptr) : sg > 0 || (a.segments > 1 && a.state_in) ? a.starts + (long)sg * heads * a.Dk * a.Dv : a.state_in;
    const unsigned vstep = (unsigned)a.vs[1] * E, ostep = (unsigned)a.os[1] * E;
    const unsigned voff = cin && !eye ? 4 * q * vstep + col * E : GD_OUT;
    const int ocol = col - n + 4 * q;                      // out: row n of a block, four columns
    const unsigned ooff = n * ostep + ocol * E;
    f32x4 S[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 16 * c + 4 * q + i;
            S[c][i] = eye ? (r == col ? 1.f : 0.f) : from && cin && r < a.Dk ? from[sb + (long)r * a.Dv] : 0.f;
        }

    // a chunk on its way: two rows of eight k and q per item, this lane's v, the gates of frame `lane`
    GdRow<T> nk[ITEMS][2], nq[ITEMS][2];
    unsigned nv[CB][4];
    float ng = 0.f, nbt = 0.f;
    const bool whole = a.whole;
    auto fetch = [&](int t0) {
        const int m = len - t0 < C ? len - t0 : C;
        const auto rk = gd_buffer(a.k, kb + (long)t0 * a.ks[1], (m - 1) * a.ks[1] + a.Dk, E), rq = gd_buffer(a.q, qb + (long)t0 * a.qs[1], (m - 1) * a.qs[1] + a.Dk, E);
        const auto rv = gd_buffer(a.v, vb + (long)t0 * a.vs[1], (m - 1) * a.vs[1] + a.Dv, E);
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int e = tid + 64 * NW * it, j = e % (DKP / 8), p = e / (DKP / 8);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                nk[it][x] = gd_row<T>(rk, (2 * p + x) * (unsigned)a.ks[1] * E + 8 * j * E, a.Dk - 8 * j, whole);
                if constexpr (!MOVE) nq[it][x] = gd_row<T>(rq, (2 * p + x) * (unsigned)a.qs[1] * E + 8 * j * E, a.Dk - 8 * j, whole);
            }
        }
#pragma unroll
        for (int bl = 0; bl < CB; ++bl)
#pragma unroll
            for (int i = 0; i < 4; ++i) nv[bl][i] = gd_get<T>(rv, voff + (16 * bl + i) * vstep);
        if (w == 0) {
            const int r = t0 + (lane < m ? lane : m - 1);
            ng = gd_gate(a.g, gb + (long)r * a.gs[1], a.gate);
            nbt = gd_gate(a.beta, bb + (long)r * a.bs[1], a.gate);
        }
    };
    if (tid < 2) kbad[tid] = C;
    if (len > first) fetch(first);
    for (int t0 = first, par = 0; t0 < len; t0 += C, par ^= 1) {
        const int m = len - t0 < C ? len - t0 : C;
        __syncthreads();
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int e = tid + 64 * NW * it, j = e % (DKP / 8), p = e / (DKP / 8);
            if (p >= C / 2) break;
            uint4 kl[2][L], ql[2][L];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (gd_limbs<T>(nk[it][x], kl[x])) {
                    atomicMin(&kbad[par], 2 * p + x);
#pragma unroll
                    for (int l = 0; l < L; ++l) kl[x][l] = make_uint4(0, 0, 0, 0);
                }
                if constexpr (!MOVE) gd_limbs<T>(nq[it][x], ql[x]);
            }
            const int c0 = 32 * (j >> 2) + 8 * (2 * j & 3) + 4 * (j >> 1 & 1);                    // slots of k 8 j .. 8 j + 3; the next four are 8 on
            const int r0 = 2 * p;
#pragma unroll
            for (int l = 0; l < L; ++l)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    *(uint2*)&Kr[l][r0 + x][c0] = make_uint2(kl[x][l].x, kl[x][l].y); *(uint2*)&Kr[l][r0 + x][c0 + 8] = make_uint2(kl[x][l].z, kl[x][l].w);
                    if constexpr (MOVE) continue;
                    *(uint2*)&Qr[l][r0 + x][c0] = make_uint2(ql[x][l].x, ql[x][l].y); *(uint2*)&Qr[l][r0 + x][c0 + 8] = make_uint2(ql[x][l].z, ql[x][l].w);
                }
        }
        if (w == 0) {
            if (lane >= m) { ng = 0.f; nbt = 0.f; }
            if (!(ng < __builtin_inff()) || !gd_finite(nbt)) { atomicMin(&kbad[par], lane); ng = 0.f; nbt = 0.f; }
            // in powers of two; -inf, a reset, comes as -8192, without inf - inf: far below what growth inside a chunk, which is held to 2^127, brings back
            auto sum = [&] { return gd_scan((ng < -8192.f ? -8192.0 : (double)ng) * 1.4426950408889634); };
            double s = sum();
            if (__any(ng > 0.f)) {
                // growth since the chunk's beginning or a frame of it: from the first frame on that has more than fp32 holds, NaN, and finite operands
                float low = fminf((float)s, 0.f);
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) low = fminf(low, __shfl_up(low, o));         // lanes below o get their own
                const unsigned long over = __ballot((float)s - low > 127.f);
                if (over) {
                    const int at = __builtin_ctzl(over);
                    if (lane == 0) atomicMin(&kbad[par], at);
                    if (lane >= at) { ng = 0.f; nbt = 0.f; }
                    s = sum();
                }
            }
            const double last = __shfl(s, C - 1);
            if (lane < C) {
                const float hi = (float)s;
                gam[lane] = make_float2(hi, (float)(s - (double)hi)); bt[lane] = nbt;
                eg[lane] = __builtin_amdgcn_exp2f(hi);
                ee[lane] = __builtin_amdgcn_exp2f((float)(last - s));
            }
        }
        float v[CB][4], vsum = 0.f;
#pragma unroll
        for (int bl = 0; bl < CB; ++bl)
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[bl][i] = gd_value<T>(nv[bl][i]); vsum = __builtin_fmaf(v[bl][i], 0.f, vsum); }
        __syncthreads();
        if (t0 + C < len) fetch(t0 + C);
        if (tid == 0) kbad[par ^ 1] = C;
        // A and P, the 16 x 16 blocks on and below the diagonal, as their transposes: a lane then holds what it will read, [row n][4 q ..].
        // The diagonal ones first: then one wave inverts those of I + A while the others see to the rest.
        auto blocks = [&](int e) {
            int bi = e, bj = e;
            if (e >= CB) {
                bi = 1; bj = e - CB;
                while (bj >= bi) { bj -= bi; ++bi; }
            }
            f32x4 xa = {0.f, 0.f, 0.f, 0.f}, xp = xa;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint4 kj[L], ki[L], qi[L];
#pragma unroll
                for (int l = 0; l < L; ++l) {
                    kj[l] = *(const uint4*)&Kr[l][16 * bj + n][32 * c + 8 * q];
                    ki[l] = *(const uint4*)&Kr[l][16 * bi + n][32 * c + 8 * q];
                    if constexpr (!MOVE) qi[l] = *(const uint4*)&Qr[l][16 * bi + n][32 * c + 8 * q];
                }
                xa = gd_mul(kj, ki, xa);
                if constexpr (!MOVE) xp = gd_mul(kj, qi, xp);
            }
            const float2 gr = gam[16 * bi + n];
            const float br = -bt[16 * bi + n];
            const float4 g01 = *(const float4*)&gam[16 * bj + 4 * q], g23 = *(const float4*)&gam[16 * bj + 4 * q + 2];
            const float gh[4] = {g01.x, g01.z, g23.x, g23.z}, gl[4] = {g01.y, g01.w, g23.y, g23.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float d = __builtin_amdgcn_exp2f((gr.x - gh[i]) + (gr.y - gl[i]));
                xa[i] *= br * d;
                xp[i] *= d;
            }
            if (bi == bj) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (4 * q + i >= n) xa[i] = 0.f;
                    if (4 * q + i > n) xp[i] = 0.f;
                }
                *(float4*)&Ad[bi][n][4 * q] = make_float4(xa[0], xa[1], xa[2], xa[3]);
            } else {
                uint4 f[3];
                gd_split(xa, f, 0);
#pragma unroll
                for (int l = 0; l < 3; ++l) Af[bi * bi / 4 + bj / 2][l][lane][bj & 1] = make_uint2(f[l].x, f[l].y);
            }
            if constexpr (MOVE) return;
            uint4 f[3];
            gd_split(xp, f, 0);
#pragma unroll
            for (int l = 0; l < 3; ++l) Pf[(bi + 1) * (bi + 1) / 4 + bj / 2][l][lane][bj & 1] = make_uint2(f[l].x, f[l].y);
        };
        constexpr int FIRST = NW > CB ? NW < BLOCKS ? NW : BLOCKS : CB;
        for (int e = w; e < FIRST; e += NW) blocks(e);
        __syncthreads();
        if (w == 0) {
            // lane (q, n): column n of block q, forward substitution, in place
            float t[16];
            float(*D)[20] = Ad[CB == 4 ? q : q & 1];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s = i == n ? 1.f : 0.f;
#pragma unroll
                for (int j = 0; j < i; ++j) s = __builtin_fmaf(D[i][j], t[j], s);
                t[i] = s;
            }
            if (q < CB)
#pragma unroll
                for (int i = 0; i < 16; ++i) D[i][n] = t[i];
        } else
            for (int e = FIRST + w - 1; e < BLOCKS; e += NW - 1) blocks(e);
        // x = K S, o = the transpose of Q S: frame n, columns 4 q ..
        f32x4 x[CB], o[MOVE ? 1 : CB];
        {
            uint4 sl[NC][3];
#pragma unroll
            for (int c = 0; c < NB; ++c) gd_split(S[c], sl[c / 2], c & 1);
#pragma unroll
            for (int bl = 0; bl < CB; ++bl) {
                x[bl] = (f32x4){0.f, 0.f, 0.f, 0.f};
                if constexpr (!MOVE) o[bl] = x[bl];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    uint4 kf[L], qf[L];
#pragma unroll
                    for (int l = 0; l < L; ++l) {
                        kf[l] = *(const uint4*)&Kr[l][16 * bl + n][32 * c + 8 * q];
                        if constexpr (!MOVE) qf[l] = *(const uint4*)&Qr[l][16 * bl + n][32 * c + 8 * q];
                    }
                    x[bl] = gd_mul(kf, sl[c], x[bl]);
                    if constexpr (!MOVE) o[bl] = gd_mul_t(qf, sl[c], o[bl]);
                }
            }
        }
        __syncthreads();
        int bad = kbad[par];
        if (__any(!(vsum == 0.f) || bad < C)) {
#pragma unroll
            for (int bl = 0; bl < CB; ++bl)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!gd_finite(v[bl][i])) { const int r = 16 * bl + 4 * q + i; bad = r < bad ? r : bad; v[bl][i] = 0.f; }
            { const int z = __shfl_xor(bad, 16); bad = z < bad ? z : bad; }
            { const int z = __shfl_xor(bad, 32); bad = z < bad ? z : bad; }
        }
        const bool hurt = __any(bad < C);
        const float end = eg[C - 1];
        const auto ro = gd_buffer(a.out, ob + (long)t0 * a.os[1], (m - 1) * a.os[1] + a.Dv, E);
        uint4 ul[CC][3], wl[3];
#pragma unroll
        for (int c = 0; c < NB; ++c) S[c] *= end;
#pragma unroll
        for (int bl = 0; bl < CB; ++bl) {
            const float4 be = *(const float4*)&bt[16 * bl + 4 * q], e4 = *(const float4*)&eg[16 * bl + 4 * q], f4 = *(const float4*)&ee[16 * bl + 4 * q];
            f32x4 z;
            z[0] = be.x * __builtin_fmaf(-e4.x, x[bl][0], v[bl][0]); z[1] = be.y * __builtin_fmaf(-e4.y, x[bl][1], v[bl][1]);
            z[2] = be.z * __builtin_fmaf(-e4.z, x[bl][2], v[bl][2]); z[3] = be.w * __builtin_fmaf(-e4.w, x[bl][3], v[bl][3]);
#pragma unroll
            for (int c = 0; c < bl / 2; ++c) {
                uint4 f[3];
#pragma unroll
                for (int l = 0; l < 3; ++l) f[l] = *(const uint4*)Af[bl * bl / 4 + c][l][lane];
                z = gd_mul(f, ul[c], z);
            }
            if (bl & 1) {
                uint2 f[3];
#pragma unroll
                for (int l = 0; l < 3; ++l) f[l] = Af[bl * bl / 4 + bl / 2][l][lane][0];
                z = gd_mul16(f, ul[bl / 2], z);
            }
            const float4 t = *(const float4*)&Ad[bl][n][4 * q];
            f32x4 u = {0.f, 0.f, 0.f, 0.f};
            u = mfma16(t.x, z[0], u); u = mfma16(t.y, z[1], u); u = mfma16(t.z, z[2], u); u = mfma16(t.w, z[3], u);
            gd_split(u, ul[bl / 2], bl & 1);
            if constexpr (!MOVE) {
                o[bl] *= eg[16 * bl + n];
#pragma unroll
                for (int c = 0; c < (bl + 1) / 2; ++c) {
                    uint4 f[3];
#pragma unroll
                    for (int l = 0; l < 3; ++l) f[l] = *(const uint4*)Pf[(bl + 1) * (bl + 1) / 4 + c][l][lane];
                    o[bl] = gd_mul_t(f, ul[c], o[bl]);
                }
                if (!(bl & 1)) {
                    uint2 f[3];
#pragma unroll
                    for (int l = 0; l < 3; ++l) f[l] = Pf[(bl + 1) * (bl + 1) / 4 + bl / 2][l][lane][0];
                    o[bl] = gd_mul16_t(f, ul[bl / 2], o[bl]);
                }
                o[bl] *= a.scale;                          // not a factor of P: d alone may be near fp32's end
                if (hurt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * bl + n >= __shfl(bad, 4 * q + i)) o[bl][i] = gd_nan();
                gd_put<T>(ro, ooff + 16 * bl * ostep, o[bl], a.Dv - ocol, a.even);
            }
            u[0] *= f4.x; u[1] *= f4.y; u[2] *= f4.z; u[3] *= f4.w;
            gd_split(u, wl, bl & 1);
            if (bl & 1)
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    uint4 f[L];
#pragma unroll
                    for (int l = 0; l < L; ++l) {
                        const unsigned short* p = &Kr[l][16 * (bl - 1) + 4 * q + (n >> 2)][32 * (c >> 1) + 8 * (n & 3) + 4 * (c & 1)];
                        const uint2 f0 = gd_column(p), f1 = gd_column(p + 16 * LDK);
                        f[l] = make_uint4(f0.x, f0.y, f1.x, f1.y);
                    }
                    S[c] = gd_mul(f, wl, S[c]);
                }
        }
        if (hurt && bad < C) {
            const float z = gd_nan();
#pragma unroll
            for (int c = 0; c < NB; ++c) S[c] = (f32x4){z, z, z, z};
        }
    }
    float* to = MOVE ? (eye ? a.moves + ((long)sg * heads + head) * a.Dk * a.Dk + col : a.starts + (long)(sg + 1) * heads * a.Dk * a.Dv + sb)
                     : sg == a.segments - 1 && a.state_out ? a.state_out + sb : nullptr;
    if (to && cin)
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * c + 4 * q + i;
                if (r < a.Dk) to[(long)r * (eye ? a.Dk : a.Dv)] = S[c][i];
            }
}

// The segments' states one after the other, S <- M S + N on the fp32 matrix instruction: a workgroup is 16 columns of a head, wave c its rows
// 16 c .. 16 c + 15; the state goes round through LDS.  starts[0] becomes a copy of state_in (in this kernel: in MOVE its stores stood in front
// of the first chunk's loads, 16 clips of 1003 frames, 4 heads of 64, fp32, 3 us).
template <int DKP>
__global__ __launch_bounds__(4 * DKP) void gated_delta_join_kernel(GatedDeltaArgs a, long heads) {
    constexpr int NB = DKP / 16;
    __shared__ __attribute__((aligned(16))) float Sx[2][16][DKP + 4];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
    const long head = blockIdx.x / (unsigned)a.strips;
    const int col = 16 * (int)(blockIdx.x - head * a.strips) + n, row = 16 * w + 4 * q;
    const bool cin = col < a.Dv;
    const long step = heads * a.Dk * a.Dv, sb = head * a.Dk * a.Dv + col;
    const int mrow = 16 * w + n < a.Dk ? 16 * w + n : a.Dk - 1;          // what lies behind Dk is 0 on the other side, and not written
    const float* mv = a.moves + (head * a.Dk + mrow) * a.Dk;
    const long mstep = heads * a.Dk * a.Dk;
    auto piece = [&](int s, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = cin && row + i < a.Dk ? a.starts[(long)s * step + sb + (long)(row + i) * a.Dv] : 0.f;
    };
    const bool whole = a.Dk % 4 == 0;
    auto matrix = [&](int s, f32x4 (&x)[NB]) {
        if (whole)
#pragma unroll
            for (int c = 0; c < NB; ++c) x[c] = 16 * c + 4 * q < a.Dk ? *(const f32x4*)&mv[(long)s * mstep + 16 * c + 4 * q] : (f32x4){0.f, 0.f, 0.f, 0.f};
        else
#pragma unroll
            for (int c = 0; c < NB; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[c][i] = 16 * c + 4 * q + i < a.Dk ? mv[(long)s * mstep + 16 * c + 4 * q + i] : 0.f;
    };
    // segment s's matrix and the next one's addition are on their way while segment s - 1 is joined
    float x[4], nx[4], s0[4] = {0.f, 0.f, 0.f, 0.f};
    f32x4 m[NB];
    if (a.state_in)
#pragma unroll
        for (int i = 0; i < 4; ++i) s0[i] = cin && row + i < a.Dk ? a.state_in[sb + (long)(row + i) * a.Dv] : 0.f;
    piece(1, x);
    if (a.segments > 2) { matrix(1, m); piece(2, nx); }
    for (int s = 1; s + 1 < a.segments; ++s) {
        *(float4*)&Sx[s & 1][n][row] = make_float4(x[0], x[1], x[2], x[3]);
        __syncthreads();
        f32x4 y[4] = {{nx[0], nx[1], nx[2], nx[3]}}, cm[NB];      // four sums, so that the products need not wait for each other
#pragma unroll
        for (int c = 1; c < 4; ++c) y[c] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NB; ++c) cm[c] = m[c];
        if (s + 2 < a.segments) { matrix(s + 1, m); piece(s + 2, nx); }
#pragma unroll
        for (int c = 0; c < NB; ++c) {
            const float4 v = *(const float4*)&Sx[s & 1][n][16 * c + 4 * q];
            y[0] = mfma16(cm[c][0], v.x, y[0]); y[1] = mfma16(cm[c][1], v.y, y[1]); y[2] = mfma16(cm[c][2], v.z, y[2]); y[3] = mfma16(cm[c][3], v.w, y[3]);
        }
        y[0] += y[1]; y[2] += y[3]; y[0] += y[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = row + i < a.Dk ? y[0][i] : 0.f;
            if (cin && row + i < a.Dk) a.starts[(long)(s + 1) * step + sb + (long)(row + i) * a.Dv] = y[0][i];
        }
    }
    if (a.state_in)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (cin && row + i < a.Dk) a.starts[sb + (long)(row + i) * a.Dv] = s0[i];
}
