// gated_delta.h -- the gated delta rule: a recurrence over frames whose state is a matrix S [Dk][Dv] (fp32) per sequence and value head,
//     S' = exp(g_t) S_{t-1};   e_t = beta_t (v_t - S'^T k_t);   S_t = S' + k_t e_t^T;   o_t = scale S_t^T q_t
// in the two forms that the GRU scans have: hop by hop with the state in HBM (gated_delta_step_kernel) and over whole clips
// (gated_delta_clip_kernel).  Value head h reads key head h / (Hv / Hk).
#pragma once
#include "common.h"
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
    int T, Hk, Hv, Dk, Dv;
    int strips;                       // workgroups (clip) or waves (step) per head
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

__device__ __forceinline__ bool gd_finite(float v) { return (__builtin_bit_cast(unsigned, v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float gd_nan() { return __builtin_bit_cast(float, 0x7fc00000u); }

// ---------------------------------------------------------------------------------------------------------------------------------------
// Hops: one wave = 32 columns of one head's state, all Dk rows of them in registers for the T hops of the call; lane (rg, cl) holds the
// DKP / 8 rows rg * DKP / 8 + j of the columns 4 cl .. 4 cl + 3.  A hop needs S'^T k and S'^T q; with o = scale (S'^T q + (q.k) e) both are
// sums over the OLD state, so that one butterfly over the eight row groups serves them, and no wave waits for another.
// Bound: HBM, the state read once and written once.
// ---------------------------------------------------------------------------------------------------------------------------------------
template <typename T, typename G, int DKP, bool VEC>
__global__ __launch_bounds__(64) void gated_delta_step_kernel(GatedDeltaArgs a) {
    constexpr int R = DKP / 8;
    const int lane = threadIdx.x, cl = lane & 7, rg = lane >> 3;
    const long head = blockIdx.x / a.strips;
    const int strip = (int)(blockIdx.x - head * a.strips);
    const int b = (int)(head / a.Hv), h = (int)(head - (long)b * a.Hv), hk = h / (a.Hv / a.Hk);
    if (a.active && !a.active[b]) return;
    const int c0 = 32 * strip + 4 * cl, r0 = rg * R;
    const long sbase = head * a.Dk * a.Dv;
    float S[R][4];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int r = r0 + j;
        const float* p = a.state_in + sbase + (long)r * a.Dv + c0;
        if (VEC) {
            const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            const float4 s = a.state_in && r < a.Dk && c0 < a.Dv ? *(const float4*)p : z;
            S[j][0] = s.x; S[j][1] = s.y; S[j][2] = s.z; S[j][3] = s.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][i] = a.state_in && r < a.Dk && c0 + i < a.Dv ? p[i] : 0.f;
        }
    }
    const long qb = (long)b * a.qs[0] + (long)hk * a.qs[2], kb = (long)b * a.ks[0] + (long)hk * a.ks[2];
    const long vb = (long)b * a.vs[0] + (long)h * a.vs[2] + c0, ob = (long)b * a.os[0] + (long)h * a.os[2] + c0;
    const long gb = (long)b * a.gs[0] + (long)h * a.gs[2], bb = (long)b * a.bs[0] + (long)h * a.bs[2];
    for (int t = 0; t < a.T; ++t) {
        float kr[R], qr[R], v[4];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool in = r0 + j < a.Dk;
            kr[j] = in ? gd_load<T>(a.k, kb + t * a.ks[1] + r0 + j) : 0.f;
            qr[j] = in ? gd_load<T>(a.q, qb + t * a.qs[1] + r0 + j) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c0 + i < a.Dv ? gd_load<T>(a.v, vb + t * a.vs[1] + i) : 0.f;
        const float alpha = __expf(gd_load<G>(a.g, gb + t * a.gs[1])), beta = gd_load<G>(a.beta, bb + t * a.bs[1]);
        float sk[4] = {0.f, 0.f, 0.f, 0.f}, sq[4] = {0.f, 0.f, 0.f, 0.f}, qk = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            qk = __builtin_fmaf(qr[j], kr[j], qk);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                S[j][i] *= alpha;
                sk[i] = __builtin_fmaf(kr[j], S[j][i], sk[i]);
                sq[i] = __builtin_fmaf(qr[j], S[j][i], sq[i]);
            }
        }
#pragma unroll
        for (int m = 8; m < 64; m <<= 1) {
            qk += __shfl_xor(qk, m);
#pragma unroll
            for (int i = 0; i < 4; ++i) { sk[i] += __shfl_xor(sk[i], m); sq[i] += __shfl_xor(sq[i], m); }
        }
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = beta * (v[i] - sk[i]);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j][i] = __builtin_fmaf(kr[j], e[i], S[j][i]);
        if (rg == 0)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + i < a.Dv) gd_store<T>(a.out, ob + t * a.os[1] + i, a.scale * __builtin_fmaf(qk, e[i], sq[i]));
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int r = r0 + j;
        float* p = a.state_out + sbase + (long)r * a.Dv + c0;
        if (r >= a.Dk) continue;
        if (VEC) {
            if (c0 < a.Dv) *(float4*)p = make_float4(S[j][0], S[j][1], S[j][2], S[j][3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + i < a.Dv) p[i] = S[j][i];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Clips: chunks of 64 frames.  With gamma = the running sum of g inside the chunk, d_ij = exp(gamma_i - gamma_j) and S the state before it,
//     A_ij = beta_i d_ij k_i.k_j (j < i),   (I + A) u = beta (v - exp(gamma) (K S)),
//     O = scale exp(gamma) (Q S) + P u,   P_ij = scale d_ij q_i.k_j (j <= i),   S <- exp(gamma_63) S + K^T (exp(gamma_63 - gamma) u):
// matrix products, and 16 dependent steps for the inverses of the four 16 x 16 diagonal blocks of I + A where the definition has 64.
// A workgroup is one head and up to 64 columns: wave w owns 16 columns of S, u and O in the matrix units' result layout (row 4 q + i, column
// n), in which a result IS the next product's right operand -- K slot 4 q + i of a block is its row 4 q + i -- so that K S -> u -> P u, K^T u
// chain in registers, and the waves meet only over the chunk's K, Q, A and P in LDS.
// gamma and its differences are 64-bit: they are small differences of long sums.  A non-finite k, g or beta makes its head's outputs from its
// frame on, and the final state, NaN; a non-finite v does that to its column; earlier frames stay as they are (the products run over all 64
// frames of the chunk, so that such values are taken out of the operands first).
// ---------------------------------------------------------------------------------------------------------------------------------------
constexpr int GD_C = 64;

template <typename T, typename G, int DKP>
__global__ __launch_bounds__(256) void gated_delta_clip_kernel(GatedDeltaArgs a) {
    constexpr int NB = DKP / 16, LD = DKP + 4, LA = GD_C + 4;
    __shared__ __attribute__((aligned(16))) float Ks[GD_C][LD], Qs[GD_C][LD], As[GD_C][LA], Ps[GD_C][LA], Ti[4][16][20];
    __shared__ double gam[GD_C];
    __shared__ float eg[GD_C], ee[GD_C], bt[GD_C];
    __shared__ int kbad;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, n = lane & 15, q = lane >> 4;
    const long head = blockIdx.x / a.strips;
    const int b = (int)(head / a.Hv), h = (int)(head - (long)b * a.Hv), hk = h / (a.Hv / a.Hk);
    const int col = 64 * (int)(blockIdx.x - head * a.strips) + 16 * w + n;
    const bool cin = col < a.Dv;
    int len = a.lengths ? a.lengths[b] : a.T;
    len = len < 0 ? 0 : len > a.T ? a.T : len;
    const long qb = (long)b * a.qs[0] + (long)hk * a.qs[2], kb = (long)b * a.ks[0] + (long)hk * a.ks[2];
    const long vb = (long)b * a.vs[0] + (long)h * a.vs[2] + col, ob = (long)b * a.os[0] + (long)h * a.os[2] + col;
    const long gb = (long)b * a.gs[0] + (long)h * a.gs[2], bb = (long)b * a.bs[0] + (long)h * a.bs[2];
    const long sb = head * a.Dk * a.Dv + col;
    f32x4 S[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 16 * c + 4 * q + i;
            S[c][i] = a.state_in && cin && r < a.Dk ? a.state_in[sb + (long)r * a.Dv] : 0.f;
        }
    for (int t0 = 0; t0 < len; t0 += GD_C) {
        const int m = len - t0 < GD_C ? len - t0 : GD_C;
        __syncthreads();
        if (tid == 0) kbad = GD_C;
        __syncthreads();
        for (int e = tid; e < GD_C * DKP; e += 256) {
            const int r = e / DKP, c = e - r * DKP;
            const bool in = r < m && c < a.Dk;
            float kv = in ? gd_load<T>(a.k, kb + (long)(t0 + r) * a.ks[1] + c) : 0.f;
            if (!gd_finite(kv)) { atomicMin(&kbad, r); kv = 0.f; }
            Ks[r][c] = kv;
            Qs[r][c] = in ? gd_load<T>(a.q, qb + (long)(t0 + r) * a.qs[1] + c) : 0.f;
        }
        if (tid < GD_C) {
            float gv = tid < m ? gd_load<G>(a.g, gb + (long)(t0 + tid) * a.gs[1]) : 0.f;
            float bv = tid < m ? gd_load<G>(a.beta, bb + (long)(t0 + tid) * a.bs[1]) : 0.f;
            if (!(gv < __builtin_inff()) || !gd_finite(bv)) { atomicMin(&kbad, tid); gv = 0.f; bv = 0.f; }
            double s = (gv < -128.f ? -128.0 : (double)gv) * 1.4426950408889634;      // in powers of two; exp(-128) is 0 in fp32 already: -inf,
                                                                                      // a reset, comes without inf - inf
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const double u = __shfl_up(s, o); if (tid >= o) s += u; }
            gam[tid] = s; bt[tid] = bv;
            eg[tid] = __builtin_amdgcn_exp2f((float)s);
            ee[tid] = __builtin_amdgcn_exp2f((float)(__shfl(s, 63) - s));
        }
        __syncthreads();
        // A and P, ten 16 x 16 blocks on and below the diagonal of each
        for (int e = w; e < 20; e += 4) {
            const bool isq = e >= 10;
            int f = isq ? e - 10 : e, bi = 0;
            while (f > bi) { f -= bi + 1; ++bi; }
            const int bj = f;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < NB; ++c) {
                const float4 x = *(const float4*)(isq ? &Qs[16 * bi + n][16 * c + 4 * q] : &Ks[16 * bi + n][16 * c + 4 * q]);
                const float4 y = *(const float4*)&Ks[16 * bj + n][16 * c + 4 * q];
                acc = mfma16(x.x, y.x, acc); acc = mfma16(x.y, y.y, acc); acc = mfma16(x.z, y.z, acc); acc = mfma16(x.w, y.w, acc);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * bi + 4 * q + i, s = 16 * bj + n;
                const float d = s <= r ? __builtin_amdgcn_exp2f((float)(gam[r] - gam[s])) : 0.f;
                if (isq) Ps[r][s] = s <= r ? a.scale * d * acc[i] : 0.f;
                else As[r][s] = s < r ? bt[r] * d * acc[i] : 0.f;
            }
        }
        __syncthreads();
        if (lane < 16) {          // inverse of diagonal block w of I + A: lane = column, forward substitution
            float t[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s = i == lane ? 1.f : 0.f;
#pragma unroll
                for (int j = 0; j < i; ++j) s = __builtin_fmaf(-As[16 * w + i][16 * w + j], t[j], s);
                t[i] = s;
                Ti[w][i][lane] = s;
            }
        }
        __syncthreads();
        f32x4 u[4], o[4];
        int bad = kbad;
#pragma unroll
        for (int bl = 0; bl < 4; ++bl) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                const float4 kk = *(const float4*)&Ks[16 * bl + n][16 * c + 4 * q], qq = *(const float4*)&Qs[16 * bl + n][16 * c + 4 * q];
                x = mfma16(kk.x, S[c][0], x); x = mfma16(kk.y, S[c][1], x); x = mfma16(kk.z, S[c][2], x); x = mfma16(kk.w, S[c][3], x);
                y = mfma16(qq.x, S[c][0], y); y = mfma16(qq.y, S[c][1], y); y = mfma16(qq.z, S[c][2], y); y = mfma16(qq.w, S[c][3], y);
            }
            f32x4 z = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < bl; ++c) {
                const float4 aa = *(const float4*)&As[16 * bl + n][16 * c + 4 * q];
                z = mfma16(aa.x, u[c][0], z); z = mfma16(aa.y, u[c][1], z); z = mfma16(aa.z, u[c][2], z); z = mfma16(aa.w, u[c][3], z);
            }
            f32x4 rhs;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * bl + 4 * q + i;
                float v = cin && r < m ? gd_load<T>(a.v, vb + (long)(t0 + r) * a.vs[1]) : 0.f;
                if (!gd_finite(v)) { bad = r < bad ? r : bad; v = 0.f; }
                rhs[i] = __builtin_fmaf(bt[r], __builtin_fmaf(-eg[r], x[i], v), -z[i]);
                o[bl][i] = a.scale * eg[r] * y[i];
            }
            const float4 ti = *(const float4*)&Ti[bl][n][4 * q];
            f32x4 uu = {0.f, 0.f, 0.f, 0.f};
            uu = mfma16(ti.x, rhs[0], uu); uu = mfma16(ti.y, rhs[1], uu); uu = mfma16(ti.z, rhs[2], uu); uu = mfma16(ti.w, rhs[3], uu);
            u[bl] = uu;
            for (int c = 0; c <= bl; ++c) {
                const float4 pp = *(const float4*)&Ps[16 * bl + n][16 * c + 4 * q];
                o[bl] = mfma16(pp.x, u[c][0], o[bl]); o[bl] = mfma16(pp.y, u[c][1], o[bl]); o[bl] = mfma16(pp.z, u[c][2], o[bl]); o[bl] = mfma16(pp.w, u[c][3], o[bl]);
            }
        }
        { const int x = __shfl_xor(bad, 16); bad = x < bad ? x : bad; }
        { const int x = __shfl_xor(bad, 32); bad = x < bad ? x : bad; }
        const float end = eg[GD_C - 1];
#pragma unroll
        for (int bl = 0; bl < 4; ++bl)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * bl + 4 * q + i;
                if (cin && r < m) gd_store<T>(a.out, ob + (long)(t0 + r) * a.os[1], r >= bad ? gd_nan() : o[bl][i]);
                u[bl][i] *= ee[r];
            }
#pragma unroll
        for (int c = 0; c < NB; ++c) {
            S[c] *= end;
#pragma unroll
            for (int bl = 0; bl < 4; ++bl)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[c] = mfma16(Ks[16 * bl + 4 * q + i][16 * c + n], u[bl][i], S[c]);
            if (bad < GD_C) { const float x = gd_nan(); S[c] = (f32x4){x, x, x, x}; }
        }
    }
    if (a.state_out && cin)
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * c + 4 * q + i;
                if (r < a.Dk) a.state_out[sb + (long)r * a.Dv] = S[c][i];
            }
}
