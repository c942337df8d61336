// w4.h -- products with 4-bit weights and group scales (gr_linear_w4, gr_linear_w4_input_grad).
//
//   forward    y[n,m]  = sum_k x[n,k]  * (q[m,k] - z[m,g(k)]) * s[m,g(k)]       g(k) = k / group, group a multiple of 32
//   gradient   gx[n,k] = sum_m gy[n,m] * (q[m,k] - z[m,g(k)]) * s[m,g(k)]
//
// Both run on v_mfma_f32_16x16x32_{bf16,f16}.  q - z is an integer in [-15, 15], exact in bf16 and in f16, so
//   forward   the matrix unit multiplies x by INTEGERS and a group's partial sum is scaled once, in f32:  no weight is ever
//             rounded.  f32 activations are cut into three bf16 pieces (8 + 8 + 8 significand bits: the cut is exact), one
//             matrix instruction each.
//   gradient  the scale changes along the sum (it belongs to m), so it goes to gy: gy * s is formed in f32 and cut into two
//             (16-bit types, 2^-17 relative) or three (f32, exact) bf16 pieces.
// Sums are f32 throughout; only the stored output is rounded to the tensors' type.
//
// Packed layout ("tiles"): 16 rows x 128 contraction steps = 64 lanes x 16 bytes = 1 KB, the operand of four matrix
// instructions.  Lane l holds row l % 16; its dword i holds steps 32*i + 8*(l/16) + e, e = 0..7, with e = 2p in nibble p and
// e = 2p + 1 in nibble p + 4 (one AND then yields the pair (2p, 2p+1) as two 16-bit halves).  A wave reads a tile with ONE
// coalesced 16-byte load per lane.  The gradient reads a second, transposed copy (rows = k, steps = m).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "graphite_hip.h"

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 w4_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 w4_f16x2 __attribute__((ext_vector_type(2)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned w4_u32x4 __attribute__((ext_vector_type(4)));

constexpr int W4_CHUNK = 128;         // contraction steps of a tile

struct W4Params {
    const w4_u32x4* pack;    // [row tiles][chunks][64]
    const void* scales;      // [groups][Mp], type st
    const uint8_t* zeros;    // [groups][Mp], or null: 8 everywhere
    int st;
    int Mp;                  // padded out_features
    int chunks;              // of the contraction
    int C, R;                // contraction length, output columns (true sizes)
    int gsteps;              // group / 32
    const void* x;           // [N][C], row stride ldx
    void* y;                 // [N][R], row stride ldy
    const float* bias;       // [R] or null (forward)
    const void* gate;        // [N][R], row stride ldg, or null (gradient): output 0 where gate <= 0
    int64_t N, ldx, ldy, ldg;
    int relu;
    int xvec;                // x rows are 16-byte aligned
};

template <int DT> struct W4Type;
template <> struct W4Type<GR_DT_F32> { typedef float T; };
template <> struct W4Type<GR_DT_BF16> { typedef __bf16 T; };
template <> struct W4Type<GR_DT_F16> { typedef _Float16 T; };

__device__ __forceinline__ float w4_scale(const void* s, int st, size_t i) {
    if (st == GR_DT_F32) return ((const float*)s)[i];
    if (st == GR_DT_BF16) return (float)((const __bf16*)s)[i];
    return (float)((const _Float16*)s)[i];
}

__device__ __forceinline__ unsigned w4_pack_hi(float a, float b) {       // high halves of a (low) and b (high)
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// eight nibbles - z as bf16 (exact: |v| <= 15)
__device__ __forceinline__ w4_bf16x8 w4_ints_bf16(unsigned w, const float (&z)[8]) {
    union { unsigned u[4]; w4_bf16x8 v; } o;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const float a = (float)((w >> (4 * p)) & 15u) - z[2 * p], b = (float)((w >> (4 * p + 16)) & 15u) - z[2 * p + 1];
        o.u[p] = w4_pack_hi(a, b);
    }
    return o.v;
}
__device__ __forceinline__ w4_bf16x8 w4_ints_bf16(unsigned w, float z) {
    const float zz[8] = {z, z, z, z, z, z, z, z};
    return w4_ints_bf16(w, zz);
}
// the same as f16: 1024 + q has q in its lowest bits, and 1024 + q - (1024 + z) is exact
__device__ __forceinline__ w4_f16x8 w4_ints_f16(unsigned w, float z) {
    union { unsigned u[4]; w4_f16x2 h[4]; w4_f16x8 v; } o;
    const _Float16 zh = (_Float16)(1024.f + z);
    const w4_f16x2 zz = {zh, zh};
#pragma unroll
    for (int p = 0; p < 4; p++) {
        o.u[p] = ((w >> (4 * p)) & 0x000f000fu) | 0x64006400u;
        o.h[p] = o.h[p] - zz;
    }
    return o.v;
}
// v = p0 + p1 (+ p2) with bf16 pieces, each cut from what the ones before leave, the last one rounded: three pieces are
// exact, two leave at most 2^-15 |v|.  An infinity or NaN stays in p0 alone.
template <int P>
__device__ __forceinline__ void w4_pieces(const float (&v)[8], w4_bf16x8 (&out)[P]) {
    union { unsigned u[4]; w4_bf16x8 b; } o[P];
#pragma unroll
    for (int h = 0; h < 4; h++) {
        float r[2] = {v[2 * h], v[2 * h + 1]};
        bool fin[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            fin[i] = __builtin_fabsf(r[i]) < __builtin_inff();
            if (r[i] != r[i]) r[i] = __uint_as_float(0x7fc00000u);
        }
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (p == 1 && P == 2) {
#pragma unroll
                for (int i = 0; i < 2; i++) r[i] = __uint_as_float(__float_as_uint(r[i]) + 0x8000u);
            }
            o[p].u[h] = w4_pack_hi(r[0], r[1]);
            if (p == P - 1) continue;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float t = __uint_as_float(__float_as_uint(r[i]) & 0xffff0000u);
                r[i] = fin[i] ? r[i] - t : 0.f;
            }
        }
    }
#pragma unroll
    for (int p = 0; p < P; p++) out[p] = o[p].b;
}
// eight consecutive values of a row, zero beyond C
template <int DT>
__device__ __forceinline__ void w4_load8(const typename W4Type<DT>::T* row, int k, int C, bool live, bool vec,
                                         typename W4Type<DT>::T (&v)[8]) {
    typedef typename W4Type<DT>::T T;
    if (live && vec && k + 8 <= C) {
        union { w4_u32x4 q[sizeof(T) / 2]; T t[8]; } u;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) u.q[i] = ((const w4_u32x4*)(row + k))[i];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = u.t[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (live && k + e < C) ? row[k + e] : (T)0.f;
    }
}
__device__ __forceinline__ w4_f32x4 w4_mfma(w4_bf16x8 a, w4_bf16x8 b, w4_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ w4_f32x4 w4_mfma(w4_f16x8 a, w4_f16x8 b, w4_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Few rows.  A workgroup owns MT row tiles x NT tiles of 16 batch rows; its waves take the contraction's chunks in turn and
// their sums meet in LDS, in wave order.
template <int DT, int NT, int MT, bool GRAD>
__global__ __launch_bounds__(1024) void k_w4_rows(W4Params p) {
    typedef typename W4Type<DT>::T T;
    extern __shared__ __attribute__((aligned(16))) float w4_red[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nwaves = blockDim.x >> 6;
    const int lr = lane & 15, lh = lane >> 4;
    const int nmt = (p.R + 16 * MT - 1) / (16 * MT);
    const int rt0 = (int)(blockIdx.x % nmt) * MT;
    const int64_t n0 = (int64_t)(blockIdx.x / nmt) * (16 * NT);
    const T* xrow[NT];
    bool live[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int64_t n = n0 + t * 16 + lr;
        live[t] = n < p.N;
        xrow[t] = (const T*)p.x + (live[t] ? n : 0) * p.ldx;
    }
    w4_f32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[a][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};

    for (int c = wave; c < p.chunks; c += nwaves) {
        w4_u32x4 w[MT];
#pragma unroll
        for (int a = 0; a < MT; a++) w[a] = p.pack[((size_t)(rt0 + a) * p.chunks + c) * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int kb = c * W4_CHUNK + i * 32;
            if (kb >= p.C) break;
            T xv[NT][8];
#pragma unroll
            for (int t = 0; t < NT; t++) w4_load8<DT>(xrow[t], kb + lh * 8, p.C, live[t], p.xvec != 0, xv[t]);
            if constexpr (!GRAD) {
                const size_t gb = (size_t)((kb >> 5) / p.gsteps) * p.Mp;
#pragma unroll
                for (int a = 0; a < MT; a++) {
                    const size_t row = gb + (size_t)(rt0 + a) * 16;
                    const float z = p.zeros ? (float)p.zeros[row + lr] : 8.f;
                    float s[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) s[r] = w4_scale(p.scales, p.st, row + lh * 4 + r);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        w4_f32x4 part = {0.f, 0.f, 0.f, 0.f};
                        if constexpr (DT == GR_DT_F32) {
                            w4_bf16x8 pc[3];
                            w4_pieces<3>(xv[t], pc);
                            const w4_bf16x8 wi = w4_ints_bf16(w[a][i], z);
#pragma unroll
                            for (int q = 0; q < 3; q++) part = w4_mfma(wi, pc[q], part);
                        } else {
                            if constexpr (DT == GR_DT_BF16) {
                                union { T t8[8]; w4_bf16x8 v; } u;
#pragma unroll
                                for (int e = 0; e < 8; e++) u.t8[e] = xv[t][e];
                                part = w4_mfma(w4_ints_bf16(w[a][i], z), u.v, part);
                            } else {
                                union { T t8[8]; w4_f16x8 v; } u;
#pragma unroll
                                for (int e = 0; e < 8; e++) u.t8[e] = xv[t][e];
                                part = w4_mfma(w4_ints_f16(w[a][i], z), u.v, part);
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[a][t][r] = __builtin_fmaf(part[r], s[r], acc[a][t][r]);
                    }
                }
            } else {
                constexpr int P = DT == GR_DT_F32 ? 3 : 2;
                const size_t mb = (size_t)(rt0 >> 1) / p.gsteps * p.Mp + kb + lh * 8;      // rt0 * 16 / group: MT is 1 or 2
                float s[8], z[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    s[e] = w4_scale(p.scales, p.st, mb + e);
                    z[e] = p.zeros ? (float)p.zeros[mb + e] : 8.f;
                }
                w4_bf16x8 pc[NT][P];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float g[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) g[e] = (float)xv[t][e] * s[e];
                    w4_pieces<P>(g, pc[t]);
                }
#pragma unroll
                for (int a = 0; a < MT; a++) {
                    const w4_bf16x8 wi = w4_ints_bf16(w[a][i], z);
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int q = 0; q < P; q++) acc[a][t] = w4_mfma(wi, pc[t][q], acc[a][t]);
                }
            }
        }
    }

    // [wave][tile][reg][lane]
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) w4_red[(((wave * MT + a) * NT + t) * 4 + r) * 64 + lane] = acc[a][t][r];
    __syncthreads();
    for (int o = threadIdx.x; o < NT * 16 * MT * 16; o += blockDim.x) {
        const int mm = o % (MT * 16), nn = o / (MT * 16);
        const int64_t n = n0 + nn;
        const int m = rt0 * 16 + mm;
        if (n >= p.N || m >= p.R) continue;
        const int src = (((mm >> 4) * NT + (nn >> 4)) * 4 + (mm & 3)) * 64 + ((mm >> 2) & 3) * 16 + (nn & 15);
        float v = 0.f;
        for (int w = 0; w < nwaves; w++) v += w4_red[w * (MT * NT * 256) + src];
        if constexpr (!GRAD) {
            if (p.bias) v += p.bias[m];
            if (p.relu) v = v < 0.f ? 0.f : v;
        } else if (p.gate) {
            v = (float)((const T*)p.gate)[n * p.ldg + m] > 0.f ? v : 0.f;
        }
        ((T*)p.y)[n * p.ldy + m] = (T)v;
    }
}
