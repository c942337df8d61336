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

// ---------------------------------------------------------------------------------------------
// Many rows: LDS-tiled.  A workgroup of WM x WN waves computes (WM*TM*16) output columns x (WN*TN*16) batch rows; a stage of
// KS * 32 contraction steps is turned into matrix-instruction operands ONCE per workgroup (4-bit weights to integers, f32
// activations to pieces) on its way global -> registers -> LDS.  LDS holds operands in fragment order ([tile][step][64 lanes]
// [16 bytes], the order the packed weights already have), so every LDS access is 64 lanes x 16 consecutive bytes.
// Two LDS buffers, one barrier per stage, global loads one stage ahead.
// ---------------------------------------------------------------------------------------------
template <int DT, bool GRAD> struct W4Pieces {          // pieces of the weights and of the activations
    static constexpr int W = !GRAD ? 1 : DT == GR_DT_F32 ? 3 : 2;
    static constexpr int X = DT == GR_DT_F32 ? 3 : GRAD && DT == GR_DT_F16 ? 2 : 1;
    static constexpr int TOP = W > X ? W : X;           // products i, j with i + j < TOP count
};
template <int DT, bool GRAD, int TM, int TN, int WM, int WN, int KS>
struct W4Gemm {
    using P = W4Pieces<DT, GRAD>;
    static constexpr int NT = WM * WN * 64, BM = WM * TM * 16, BN = WN * TN * 16;
    static constexpr int A_ONE = BM / 16 * KS * 64, X_ONE = BN / 16 * KS * 64;      // 16-byte slots of one piece
    static constexpr int SLOTS = A_ONE * P::W + X_ONE * P::X;
    static constexpr int LDS = 2 * SLOTS * 16;
    static constexpr int AV = BM / 16 * 64 / NT, XV = X_ONE / NT;
    static_assert(BM / 16 * 64 % NT == 0 && X_ONE % NT == 0, "stage loads must divide evenly");
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <int DT, bool GRAD, int TM, int TN, int WM, int WN, int KS>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_w4_gemm(W4Params p) {
    using G = W4Gemm<DT, GRAD, TM, TN, WM, WN, KS>;
    using P = typename G::P;
    typedef typename W4Type<DT>::T T;
    constexpr bool F16OP = !GRAD && DT == GR_DT_F16;     // f16 matrix instructions; bf16 otherwise
    extern __shared__ __attribute__((aligned(16))) w4_u32x4 w4_lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave % WM, wn = wave / WM, lr = lane & 15, lh = lane >> 4;
    // workgroups go round the 8 dies; each die takes a contiguous run of tiles, so that its L2 serves neighbouring ones
    const int nmt = (p.R + G::BM - 1) / G::BM;
    const unsigned nb = gridDim.x, per = nb / 8, die = blockIdx.x % 8, seq = blockIdx.x / 8;
    const unsigned tile = seq < per ? die * per + seq : blockIdx.x;          // the last nb % 8 keep their number
    const int m0 = (int)(tile % nmt) * G::BM;
    const int64_t n0 = (int64_t)(tile / nmt) * G::BN;
    const int nstages = (p.C + KS * 32 - 1) / (KS * 32);

    // ---- staging: thread's share of the weights (AV packed lanes) and of the activations (XV runs of eight)
    unsigned wreg[G::AV][KS];
    T xreg[G::XV][8];
    float zreg[GRAD ? 1 : G::AV][KS];
    const T* xrow[G::XV];
    int xk[G::XV];
    bool xlive[G::XV];
#pragma unroll
    for (int v = 0; v < G::XV; v++) {
        const int f = tid + v * G::NT, l = f & 63, ts = f >> 6;
        const int64_t n = n0 + ts / KS * 16 + (l & 15);
        xlive[v] = n < p.N;
        xrow[v] = (const T*)p.x + (xlive[v] ? n : 0) * p.ldx;
        xk[v] = ts % KS * 32 + (l >> 4) * 8;
    }
    size_t grow[G::AV];                                   // GRAD: scales / zeros of the thread's row
#pragma unroll
    for (int v = 0; v < G::AV; v++) {
        const int row = m0 + (tid + v * G::NT) / 64 * 16 + lr;
        grow[v] = (size_t)((row < p.R ? row : p.R - 1) / (p.gsteps * 32)) * p.Mp;
    }
    int zg = 0, zrem = 0;                                 // group of the next step to load
    auto load = [&](int s) {
#pragma unroll
        for (int v = 0; v < G::AV; v++) {
            const size_t rt = m0 / 16 + (tid + v * G::NT) / 64;
            const unsigned* src = (const unsigned*)(p.pack + (rt * p.chunks + s * KS / 4) * 64 + lane) + s * KS % 4;
            if constexpr (KS == 2) {
                const uint2 d = *(const uint2*)src;
                wreg[v][0] = d.x; wreg[v][1] = d.y;
            } else {
                wreg[v][0] = *src;
            }
        }
        if constexpr (!GRAD) {
#pragma unroll
            for (int i = 0; i < KS; i++) {
#pragma unroll
                for (int v = 0; v < G::AV; v++)
                    zreg[v][i] = p.zeros ? (float)p.zeros[(size_t)zg * p.Mp + m0 + (tid + v * G::NT) / 64 * 16 + lr] : 8.f;
                if (++zrem == p.gsteps) { zrem = 0; if ((s * KS + i + 1) * 32 < p.C) zg++; }
            }
        }
#pragma unroll
        for (int v = 0; v < G::XV; v++) w4_load8<DT>(xrow[v], s * KS * 32 + xk[v], p.C, xlive[v], p.xvec != 0, xreg[v]);
    };
    auto store = [&](int s, w4_u32x4* buf) {
#pragma unroll
        for (int v = 0; v < G::AV; v++) {
            const int rt = (tid + v * G::NT) / 64;
#pragma unroll
            for (int i = 0; i < KS; i++) {
                w4_u32x4* dst = buf + (rt * KS + i) * 64 + lane;
                if constexpr (F16OP) {
                    union { w4_f16x8 h; w4_u32x4 u; } c;
                    c.h = w4_ints_f16(wreg[v][i], zreg[v][i]);
                    dst[0] = c.u;
                } else if constexpr (!GRAD) {
                    union { w4_bf16x8 h; w4_u32x4 u; } c;
                    c.h = w4_ints_bf16(wreg[v][i], zreg[v][i]);
                    dst[0] = c.u;
                } else {
                    const size_t mb = grow[v] + s * KS * 32 + i * 32 + lh * 8;
                    float f[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int q = (int)(wreg[v][i] >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15;
                        f[e] = ((float)q - (p.zeros ? (float)p.zeros[mb + e] : 8.f)) * w4_scale(p.scales, p.st, mb + e);
                    }
                    w4_bf16x8 pc[P::W];
                    w4_pieces<P::W>(f, pc);
#pragma unroll
                    for (int q = 0; q < P::W; q++) {
                        union { w4_bf16x8 h; w4_u32x4 u; } c;
                        c.h = pc[q];
                        dst[q * G::A_ONE] = c.u;
                    }
                }
            }
        }
#pragma unroll
        for (int v = 0; v < G::XV; v++) {
            w4_u32x4* dst = buf + P::W * G::A_ONE + tid + v * G::NT;
            if constexpr (P::X == 1) {
                union { T t[8]; w4_u32x4 u; } c;
#pragma unroll
                for (int e = 0; e < 8; e++) c.t[e] = xreg[v][e];
                dst[0] = c.u;
            } else {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = (float)xreg[v][e];
                w4_bf16x8 pc[P::X];
                w4_pieces<P::X>(f, pc);
#pragma unroll
                for (int q = 0; q < P::X; q++) {
                    union { w4_bf16x8 h; w4_u32x4 u; } c;
                    c.h = pc[q];
                    dst[q * G::X_ONE] = c.u;
                }
            }
        }
    };

    w4_f32x4 acc[TM][TN], part[GRAD ? 1 : TM][GRAD ? 1 : TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
    const w4_f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    union Frag { w4_u32x4 u; w4_bf16x8 b; w4_f16x8 h; };
    int cg = 0, crem = 0;                                 // group of the step being multiplied
    auto step = [&](const w4_u32x4* buf, int i, bool last) {
        Frag a[P::W][TM], x[P::X][TN];
#pragma unroll
        for (int q = 0; q < P::W; q++)
#pragma unroll
            for (int t = 0; t < TM; t++) a[q][t].u = buf[q * G::A_ONE + ((wm * TM + t) * KS + i) * 64 + lane];
#pragma unroll
        for (int q = 0; q < P::X; q++)
#pragma unroll
            for (int t = 0; t < TN; t++) x[q][t].u = buf[P::W * G::A_ONE + q * G::X_ONE + ((wn * TN + t) * KS + i) * 64 + lane];
        auto mul = [&](int qa, int qx, int t, int u, w4_f32x4 c) {
            if constexpr (F16OP) return w4_mfma(a[qa][t].h, x[qx][u].h, c);
            else return w4_mfma(a[qa][t].b, x[qx][u].b, c);
        };
        if constexpr (GRAD) {
#pragma unroll
            for (int qa = 0; qa < P::W; qa++)
#pragma unroll
                for (int qx = 0; qx < P::X; qx++) {
                    if (qa + qx >= P::TOP) continue;
#pragma unroll
                    for (int t = 0; t < TM; t++)
#pragma unroll
                        for (int u = 0; u < TN; u++) acc[t][u] = mul(qa, qx, t, u, acc[t][u]);
                }
        } else {
            const bool flush = crem + 1 == p.gsteps || last;
            float sc[TM][4];
            if (flush) {
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        sc[t][r] = w4_scale(p.scales, p.st, (size_t)cg * p.Mp + m0 + (wm * TM + t) * 16 + lh * 4 + r);
            }
            if (crem == 0) {
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int u = 0; u < TN; u++) part[t][u] = mul(0, 0, t, u, zero4);
            } else {
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int u = 0; u < TN; u++) part[t][u] = mul(0, 0, t, u, part[t][u]);
            }
#pragma unroll
            for (int qx = 1; qx < P::X; qx++)
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int u = 0; u < TN; u++) part[t][u] = mul(0, qx, t, u, part[t][u]);
            crem++;
            if (flush) {
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int u = 0; u < TN; u++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[t][u][r] = __builtin_fmaf(part[t][u][r], sc[t][r], acc[t][u][r]);
                crem = 0;
                cg++;
            }
        }
    };

    load(0);
    store(0, w4_lds);
    if (nstages > 1) load(1);
    __syncthreads();
    for (int s = 0; s < nstages; s++) {
        if (s + 1 < nstages) {
            store(s + 1, w4_lds + ((s + 1) & 1) * G::SLOTS);
            if (s + 2 < nstages) load(s + 2);
        }
        const w4_u32x4* buf = w4_lds + (s & 1) * G::SLOTS;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            if (i > 0 && (s * KS + i) * 32 >= p.C) break;
            step(buf, i, (s * KS + i + 1) * 32 >= p.C);
        }
        __syncthreads();
    }

    const bool vec = ((uintptr_t)p.y % (4 * sizeof(T)) == 0) && p.ldy % 4 == 0;
#pragma unroll
    for (int u = 0; u < TN; u++) {
        const int64_t n = n0 + (wn * TN + u) * 16 + lr;
        if (n >= p.N) continue;
#pragma unroll
        for (int t = 0; t < TM; t++) {
            const int m = m0 + (wm * TM + t) * 16 + lh * 4;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                v[r] = acc[t][u][r];
                if (m + r >= p.R) continue;
                if constexpr (!GRAD) {
                    if (p.bias) v[r] += p.bias[m + r];
                    if (p.relu) v[r] = v[r] < 0.f ? 0.f : v[r];
                } else if (p.gate) {
                    v[r] = (float)((const T*)p.gate)[n * p.ldg + m + r] > 0.f ? v[r] : 0.f;
                }
            }
            T* dst = (T*)p.y + n * p.ldy + m;
            if (vec && m + 4 <= p.R) {
                struct alignas(4 * sizeof(T)) T4 { T t[4]; } o = {{(T)v[0], (T)v[1], (T)v[2], (T)v[3]}};
                *(T4*)dst = o;
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (m + r < p.R) dst[r] = (T)v[r];
            }
        }
    }
}
