// w4.h -- products with 4-bit weights and group scales (gr_linear_w4, gr_linear_w4_input_grad).
//
//   forward    y[n,m]  = sum_k x[n,k]  * (q[m,k] - z[m,g(k)]) * s[m,g(k)]       g(k) = k / group, group a multiple of 32
//   gradient   gx[n,k] = sum_m gy[n,m] * (q[m,k] - z[m,g(k)]) * s[m,g(k)]
//
// Both run on v_mfma_f32_16x16x32_{bf16,f16}.  q - z is an integer in [-15, 15], exact in bf16 and in f16, so
//   forward   the matrix unit multiplies x by INTEGERS and a group's partial sum is scaled once, in f32:  no weight is ever
//             rounded.  f32 activations are cut into three bf16 pieces (8 + 8 + 8 significand bits: the cut is exact), one
//             matrix instruction each.
//   gradient  the scale changes along the sum (it belongs to m), so it goes to a factor: to gy in the few-row kernel (gy * s in
//             f32, its rows sharing one group), to the weights in the tiled one ((q - z) * s in f32, any mix of groups).  That
//             factor is cut into two (16-bit types) or three (f32) bf16 pieces.  A product is off by at most 2^-15 in 16-bit
//             types -- a 128th of bf16's own rounding, a 16th of f16's -- and 1.5 * 2^-23 in f32, a third of it the factor's rounding.
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
    const void* scales;      // [groups][Mp], type ST of the kernel
    const uint8_t* zeros;    // [groups][Mp]; zstride 0: one row of eights for every group
    int Mp, zstride;         // padded out_features, and what zeros advance by per group (Mp or 0)
    int chunks;              // of the contraction
    int C, R;                // contraction length, output columns (true sizes)
    int gsteps;              // group / 32
    const void* x;           // [N][C], row stride ldx
    void* y;                 // [N][R], row stride ldy
    const float* bias;       // [R] or null (forward)
    const void* gate;        // [N][R], row stride ldg, or null (gradient): output 0 where gate <= 0
    int64_t N, ldx, ldy, ldg;
    int relu;
    int waves;               // > 0: few-row kernels of that many waves, whatever N is: one order of summation (W4_MODEL_WAVES)
};

template <int DT> struct W4Type;
template <> struct W4Type<GR_DT_F32> { typedef float T; };
template <> struct W4Type<GR_DT_BF16> { typedef __bf16 T; };
template <> struct W4Type<GR_DT_F16> { typedef _Float16 T; };

__device__ __forceinline__ unsigned w4_pack_hi(float a, float b) {       // high halves of a (low) and b (high)
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// Nibbles p and p + 4 of w as the halves 1024 + q of an f16 pair.  The constants sit in registers of both kinds, so that AND and
// OR are one instruction.
__device__ __forceinline__ unsigned w4_pair(unsigned w, int p) {
    unsigned mask = 0x000f000fu, k = 0x64006400u;
    asm("" : "+s"(mask));
    asm("" : "+v"(k));
    return ((w >> (4 * p)) & mask) | k;
}
// Two nibbles as float, minus z: nibbles p and p + 4 of w become the halves 1024 + q of an f16 pair (q sits in the lowest
// mantissa bits), and one mixed-precision fma per element converts and subtracts.  Exact.
__device__ __forceinline__ void w4_ints_f32(unsigned w, int p, float z0, float z1, float& a, float& b) {
    union { unsigned u; w4_f16x2 h; } c;
    c.u = w4_pair(w, p);
    float one = 1.f;
    asm("" : "+s"(one));                                 // a factor the compiler cannot drop: it would convert and subtract in two steps
    a = __builtin_fmaf((float)c.h[0], one, -z0);
    b = __builtin_fmaf((float)c.h[1], one, -z1);
}
// eight nibbles - z as bf16 (exact: |v| <= 15); zk = 1024 + z
__device__ __forceinline__ w4_bf16x8 w4_ints_bf16(unsigned w, const float (&zk)[8]) {
    union { unsigned u[4]; w4_bf16x8 v; } o;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        float a, b;
        w4_ints_f32(w, p, zk[2 * p], zk[2 * p + 1], a, b);
        o.u[p] = w4_pack_hi(a, b);
    }
    return o.v;
}
__device__ __forceinline__ w4_bf16x8 w4_ints_bf16(unsigned w, float zk) {
    const float zz[8] = {zk, zk, zk, zk, zk, zk, zk, zk};
    return w4_ints_bf16(w, zz);
}
// the same as f16: 1024 + q - (1024 + z), a packed subtraction
__device__ __forceinline__ w4_f16x8 w4_ints_f16(unsigned w, float zk) {
    union { unsigned u[4]; w4_f16x2 h[4]; w4_f16x8 v; } o;
    const _Float16 zh = (_Float16)zk;
    const w4_f16x2 zz = {zh, zh};
#pragma unroll
    for (int p = 0; p < 4; p++) {
        o.u[p] = w4_pair(w, p);
        o.h[p] = o.h[p] - zz;
    }
    return o.v;
}
// v = p0 + p1 (+ p2) with bf16 pieces, each cut from what the ones before leave, the last one of two rounded: three pieces are
// exact, two leave at most 2^-16 |v|.  An infinity stays in p0 alone.
// NEAR, for products of pieces of which the smallest are left out: p0 is rounded to nearest (values next to float32's largest,
// LARGE, to bf16's), so that what it leaves has either sign and is at most 2^-8 |v|, half of what a cut leaves, always with the
// sign of v.  Three pieces are exact still, two leave 2^-17 |v|, of an f16 value (not LARGE) nothing.  Infinities and NaNs leave
// NaN or infinity in p1.
template <int P, bool NEAR = false, bool LARGE = true>
__device__ __forceinline__ void w4_pieces(const float (&v)[8], w4_bf16x8 (&out)[P]) {
    union { unsigned u[4]; w4_bf16x8 b; } o[P];
#pragma unroll
    for (int h = 0; h < 4; h++) {
        float r[2] = {v[2 * h], v[2 * h + 1]};
#pragma unroll
        for (int p = 0; p < P; p++) {
            float t[2] = {r[0], r[1]};
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (p == 1 && P == 2 && !(NEAR && !LARGE)) t[i] = __uint_as_float(__float_as_uint(r[i]) + 0x8000u);
                if (p == 0 && NEAR) {
                    if (LARGE) t[i] = __builtin_amdgcn_fmed3f(r[i], -0x1.fefffep127f, 0x1.fefffep127f);
                    t[i] = __uint_as_float(__float_as_uint(t[i]) + 0x8000u);
                }
            }
            o[p].u[h] = w4_pack_hi(t[0], t[1]);
            if (p == P - 1) continue;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float d = r[i] - __uint_as_float(__float_as_uint(t[i]) & 0xffff0000u);
                r[i] = !NEAR && p == 0 && __builtin_fabsf(r[i]) == __builtin_inff() ? 0.f : d;
            }
        }
    }
#pragma unroll
    for (int p = 0; p < P; p++) out[p] = o[p].b;
}

// Eight consecutive elements of a row, as loaded.  Rows need no alignment beyond their elements' (the hardware takes 16-byte
// loads at any dword).  HALF: rows of 16-bit elements that may begin in the middle of a dword, where a 16-byte load takes
// several times as long.  Whole dwords are loaded instead, a fifth one with the last half, and `settle` moves the elements down
// before they are used; every dword read holds an element of the row.  2048 rows 4095 -> 4096 bf16: 226 us with the long loads,
// 126 so (4096 -> 4096: 100).
typedef unsigned w4_u32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned w4_u32x4_h __attribute__((ext_vector_type(4), aligned(2)));
template <int DT, bool HALF = false> struct W4Raw {
    static constexpr int Q = DT == GR_DT_F32 ? 2 : 1;
    typedef typename W4Type<DT>::T T;
    static_assert(!HALF || sizeof(T) == 2, "only 16-bit elements begin in the middle of a dword");
    w4_u32x4 q[Q];
    unsigned fifth[1];
    __device__ __forceinline__ void load(const T* src) {
        if constexpr (HALF) {
            const bool mid = (uintptr_t)src & 2;
            const unsigned* d = (const unsigned*)(src - (mid ? 1 : 0));
            q[0] = *(const w4_u32x4_u*)d;
            fifth[0] = d[mid ? 4 : 3];
        } else {
#pragma unroll
            for (int i = 0; i < Q; i++) q[i] = *(const w4_u32x4_u*)(src + i * (16 / (int)sizeof(T)));
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < Q; i++) q[i] = w4_u32x4{0u, 0u, 0u, 0u};
        fifth[0] = 0u;
    }
    // HALF: mid = 16 where the row begins in the middle of a dword, 0 elsewhere
    __device__ __forceinline__ void settle(unsigned mid) {
        if constexpr (HALF) {
#pragma unroll
            for (int i = 0; i < 4; i++) q[0][i] = __builtin_amdgcn_alignbit(i < 3 ? q[0][i + 1] : fifth[0], q[0][i], mid);
        }
    }
    __device__ __forceinline__ void unsettle(unsigned mid) {
        if constexpr (HALF) {
            fifth[0] = q[0][3] >> 16;
#pragma unroll
            for (int i = 3; i >= 0; i--) q[0][i] = mid ? __builtin_amdgcn_alignbit(q[0][i], i > 0 ? q[0][i - 1] : 0u, 16) : q[0][i];
        }
    }
    // zero from `count` on (count <= 0: all).  The eight elements that end the row (there are eight: `wide`) take one load, like
    // any others, and move down to their places: one load an element cost a product of 470 rows, 827 -> 3992 f16, 20 us of 52.
    __device__ __forceinline__ void load_part(const T* src, int count, bool wide) {
        union { w4_u32x4 q[Q]; T t[8]; unsigned u[4 * Q]; } u;
        if (wide) {
            const T* from = count < 8 ? src + (count - 8) : src;
            if constexpr (HALF) {
                load(from);
                settle((uintptr_t)from & 2 ? 16 : 0);
#pragma unroll
                for (int i = 0; i < Q; i++) u.q[i] = q[i];
            } else {                                                            // rows of an odd length end inside a dword
#pragma unroll
                for (int i = 0; i < Q; i++) u.q[i] = *(const w4_u32x4_h*)(from + i * (16 / (int)sizeof(T)));
            }
            const int sh = count >= 8 ? 0 : 8 - count;                          // elements to move by; 8 and more leave nothing
            constexpr int W = 4 / (int)sizeof(T);                               // elements of a dword
#pragma unroll
            for (int b = 4; b >= W; b >>= 1) {
#pragma unroll
                for (int i = 0; i < 4 * Q; i++) u.u[i] = sh & b ? (i + b / W < 4 * Q ? u.u[i + b / W] : 0u) : u.u[i];
            }
            if constexpr (W == 2) {
#pragma unroll
                for (int i = 0; i < 4; i++) u.u[i] = sh & 1 ? __builtin_amdgcn_alignbit(i < 3 ? u.u[i + 1] : 0u, u.u[i], 16) : u.u[i];
            }
#pragma unroll
            for (int i = 0; i < 4 * Q; i++) u.u[i] = sh >= 8 ? 0u : u.u[i];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const T v = src[e < count ? e : count - 1];                     // the row's last element
                u.t[e] = e < count ? v : (T)0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < Q; i++) q[i] = u.q[i];
        unsettle((uintptr_t)src & 2 ? 16 : 0);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        if constexpr (DT == GR_DT_F32) {
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = __uint_as_float(q[e / 4][e % 4]);
        } else if constexpr (DT == GR_DT_BF16) {
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = __uint_as_float(e % 2 ? q[0][e / 2] & 0xffff0000u : q[0][e / 2] << 16);
        } else {
            union { w4_u32x4 u; _Float16 h[8]; } c;
            c.u = q[0];
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = (float)c.h[e];
        }
    }
    __device__ __forceinline__ w4_bf16x8 bf16() const { union { w4_u32x4 u; w4_bf16x8 b; } c; c.u = q[0]; return c.b; }
    __device__ __forceinline__ w4_f16x8 f16() const { union { w4_u32x4 u; w4_f16x8 b; } c; c.u = q[0]; return c.b; }
};
// four scales of consecutive rows (16- or 8-byte aligned)
template <int ST> struct W4Scale4 {
    typedef typename W4Type<ST>::T T;
    typedef T V __attribute__((ext_vector_type(4)));
    V v;
    __device__ __forceinline__ void load(const void* s, size_t i) { v = *(const V*)((const T*)s + i); }
    __device__ __forceinline__ float operator[](int r) const { return (float)v[r]; }
};
__device__ __forceinline__ w4_f32x4 w4_mfma(w4_bf16x8 a, w4_bf16x8 b, w4_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ w4_f32x4 w4_mfma(w4_f16x8 a, w4_f16x8 b, w4_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Outputs m .. m + 3 of row n, from their sums through the epilogue to memory.  They lie together in y: one store, which may
// start at any element (four stores each cost a product of 6039 rows, 43 -> 3166 f16, half of 59 us).
template <bool GRAD>
__device__ __forceinline__ void w4_bias(const W4Params& p, int m, float (&bias)[4]) {
#pragma unroll
    for (int r = 0; r < 4; r++) bias[r] = !GRAD && p.bias ? p.bias[m + r < p.R ? m + r : p.R - 1] : 0.f;
}
template <int DT, bool GRAD>
__device__ __forceinline__ void w4_put(const W4Params& p, w4_f32x4 sum, const float (&bias)[4], int64_t n, int m) {
    typedef typename W4Type<DT>::T T;
    typedef unsigned V __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
    union Four { T t[4]; V v; __device__ Four() {} } o;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        float v = sum[r];
        if constexpr (!GRAD) {
            v += bias[r];
            if (p.relu) v = v < 0.f ? 0.f : v;
        } else if (p.gate) {
            v = m + r < p.R && (float)((const T*)p.gate)[n * p.ldg + m + r] > 0.f ? v : 0.f;
        }
        o.t[r] = (T)v;
    }
    T* dst = (T*)p.y + n * p.ldy + m;
    if (m + 4 <= p.R) {
        *(V*)dst = o.v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (m + r < p.R) dst[r] = o.t[r];
    }
}

// ---------------------------------------------------------------------------------------------
// Few rows.  A workgroup owns MT row tiles x NT tiles of 16 batch rows; its waves take the contraction's chunks in turn, D
// chunks at a time (all their loads are issued before the first is used), and their sums meet in LDS, in wave order: the long
// axis is split inside the workgroup, so there is no workspace, no second launch and one order of summation.
// Forward: GS = groups of a chunk (1, 2 or 4; 4 also where a border falls on any step).
// One row is bound by the weights' bytes: the matrix unit pads it to 16 rows for nothing, and what costs is turning nibbles
// into operands, 2.5 VALU instructions a weight.  8192 -> 8192 bf16, g = 128, one row: 10.8 us = 3.2 TB/s of weights (a copy
// reaches 4.7).  2048 -> 1024 f32, 100 rows: 8.2 us a call (its latency: one chunk a wave, then the join, in which a thread
// adds and stores four outputs at once; one output a thread took 9.2).
// ---------------------------------------------------------------------------------------------
constexpr int w4_rows_waves(int nt) { return nt > 1 ? 8 : 16; }            // the most a workgroup may have
template <int DT, int ST, bool HALF, int NT, int MT, int GS, int D, bool GRAD>
__global__ __launch_bounds__(w4_rows_waves(NT) * 64) void k_w4_rows(W4Params p) {
    typedef typename W4Type<DT>::T T;
    extern __shared__ __attribute__((aligned(16))) w4_f32x4 w4_red[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nwaves = blockDim.x >> 6;
    const int lr = lane & 15, lh = lane >> 4;
    const int nmt = (p.R + 16 * MT - 1) / (16 * MT);
    const int rt0 = (int)(blockIdx.x % nmt) * MT;
    const int64_t n0 = (int64_t)(blockIdx.x / nmt) * (16 * NT);
    const T* xrow[NT];
    unsigned mid[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int64_t n = n0 + t * 16 + lr;
        xrow[t] = (const T*)p.x + (n < p.N ? n : p.N - 1) * p.ldx + lh * 8;      // columns beyond the batch: computed, not stored
        mid[t] = (uintptr_t)xrow[t] & 2 ? 16 : 0;
    }
    const size_t grow = GRAD ? (size_t)((rt0 >> 1) / p.gsteps) * p.Mp : 0;        // the rows' one group
    const size_t zrow = GRAD ? (size_t)((rt0 >> 1) / p.gsteps) * p.zstride : 0;
    w4_f32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[a][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};

    struct Chunk {
        w4_u32x4 w[MT];
        W4Raw<DT, HALF> x[4][NT];
        W4Scale4<ST> s[GRAD ? 1 : GS][MT];
        uint8_t z[GRAD ? 1 : GS][MT];
        W4Raw<ST> gs[GRAD ? 4 : 1];
        uint2 gz[GRAD ? 4 : 1];
    };
    auto load = [&](Chunk& h, int c) {
        const int kb = c * W4_CHUNK;
#pragma unroll
        for (int a = 0; a < MT; a++) h.w[a] = p.pack[((size_t)(rt0 + a) * p.chunks + c) * 64 + lane];
        if (kb + W4_CHUNK <= p.C) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int t = 0; t < NT; t++) h.x[i][t].load(xrow[t] + kb + i * 32);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (kb + i * 32 + 32 <= p.C) h.x[i][t].load(xrow[t] + kb + i * 32);
                    else if (kb + i * 32 < p.C) h.x[i][t].load_part(xrow[t] + kb + i * 32, p.C - kb - i * 32 - lh * 8, p.C >= 8);
                    else h.x[i][t].clear();
                }
        }
        if constexpr (!GRAD) {
#pragma unroll
            for (int g = 0; g < GS; g++) {
                int step = c * 4 + g * (4 / GS);
                if (step * 32 >= p.C) step = c * 4;                               // beyond the row: x is 0 there
                const size_t g_ = (size_t)(step / p.gsteps), row = g_ * p.Mp + (size_t)rt0 * 16, zr = g_ * p.zstride + (size_t)rt0 * 16;
#pragma unroll
                for (int a = 0; a < MT; a++) {
                    h.s[g][a].load(p.scales, row + a * 16 + lh * 4);
                    h.z[g][a] = p.zeros[zr + a * 16 + lr];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const size_t mb = grow + kb + i * 32 + lh * 8;
                h.gs[i].load((const typename W4Type<ST>::T*)p.scales + mb);
                h.gz[i] = *(const uint2*)(p.zeros + zrow + kb + i * 32 + lh * 8);
            }
        }
    };
    auto mul = [&](Chunk& h) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < NT; t++) h.x[i][t].settle(mid[t]);
        if constexpr (!GRAD) {
#pragma unroll
            for (int g = 0; g < GS; g++) {
                w4_f32x4 part[MT][NT];
#pragma unroll
                for (int a = 0; a < MT; a++)
#pragma unroll
                    for (int t = 0; t < NT; t++) part[a][t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = g * (4 / GS); i < (g + 1) * (4 / GS); i++) {
                    if constexpr (DT == GR_DT_F16) {
#pragma unroll
                        for (int a = 0; a < MT; a++) {
                            const w4_f16x8 wi = w4_ints_f16(h.w[a][i], 1024.f + (float)h.z[g][a]);
#pragma unroll
                            for (int t = 0; t < NT; t++) part[a][t] = w4_mfma(wi, h.x[i][t].f16(), part[a][t]);
                        }
                    } else {
                        w4_bf16x8 wi[MT];
#pragma unroll
                        for (int a = 0; a < MT; a++) wi[a] = w4_ints_bf16(h.w[a][i], 1024.f + (float)h.z[g][a]);
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            constexpr int P = DT == GR_DT_F32 ? 3 : 1;
                            w4_bf16x8 pc[P];
                            if constexpr (P == 3) {
                                float f[8];
                                h.x[i][t].get(f);
                                w4_pieces<3>(f, pc);
                            } else {
                                pc[0] = h.x[i][t].bf16();
                            }
#pragma unroll
                            for (int q = 0; q < P; q++)
#pragma unroll
                                for (int a = 0; a < MT; a++) part[a][t] = w4_mfma(wi[a], pc[q], part[a][t]);
                        }
                    }
                }
#pragma unroll
                for (int a = 0; a < MT; a++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[a][t][r] = __builtin_fmaf(part[a][t][r], h.s[g][a][r], acc[a][t][r]);
            }
        } else {
            constexpr int P = DT == GR_DT_F32 ? 3 : 2;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float s[8], zk[8];
                h.gs[i].get(s);
#pragma unroll
                for (int e = 0; e < 8; e++) zk[e] = 1024.f + (float)(((e < 4 ? h.gz[i].x : h.gz[i].y) >> (8 * (e & 3))) & 255u);
                w4_bf16x8 wi[MT];
#pragma unroll
                for (int a = 0; a < MT; a++) wi[a] = w4_ints_bf16(h.w[a][i], zk);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float g[8];
                    w4_bf16x8 pc[P];
                    h.x[i][t].get(g);
#pragma unroll
                    for (int e = 0; e < 8; e++) g[e] *= s[e];
                    w4_pieces<P>(g, pc);
#pragma unroll
                    for (int q = 0; q < P; q++)
#pragma unroll
                        for (int a = 0; a < MT; a++) acc[a][t] = w4_mfma(wi[a], pc[q], acc[a][t]);
                }
            }
        }
    };
    int c = wave;
    for (; c + (D - 1) * nwaves < p.chunks; c += D * nwaves) {
        Chunk h[D];
#pragma unroll
        for (int d = 0; d < D; d++) load(h[d], c + d * nwaves);
#pragma unroll
        for (int d = 0; d < D; d++) mul(h[d]);
    }
    if constexpr (D > 1)
        for (; c < p.chunks; c += nwaves) {
            Chunk h;
            load(h, c);
            mul(h);
        }

    // [wave][tile][lane]: four sums; the threads add over the waves, in their order
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int t = 0; t < NT; t++) w4_red[((wave * MT + a) * NT + t) * 64 + lane] = acc[a][t];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * NT * 64; o += blockDim.x) {
        const int64_t n = n0 + (o / 64 % NT) * 16 + lr;
        const int m = (rt0 + o / (64 * NT)) * 16 + lh * 4;
        if (n >= p.N || m >= p.R) continue;
        w4_f32x4 v = w4_red[o];
        for (int w = 1; w < nwaves; w++) v += w4_red[w * (MT * NT * 64) + o];
        float bias[4];
        w4_bias<GRAD>(p, m, bias);
        w4_put<DT, GRAD>(p, v, bias, n, m);
    }
}

// ---------------------------------------------------------------------------------------------
// Many rows: LDS-tiled.  A workgroup of WM x WN waves computes (WM*TM*16) output columns x (WN*TN*16) batch rows; a stage of
// KS * 32 contraction steps is turned into matrix-instruction operands ONCE per workgroup (4-bit weights to integers, f32
// activations to pieces) on its way global -> registers -> LDS.  LDS holds operands in fragment order ([tile][step][64 lanes]
// [16 bytes], the order the packed weights already have), so every LDS access is 64 lanes x 16 consecutive bytes.
// Three LDS buffers, one barrier per stage: while a stage is multiplied, the next one's first operands are already read and
// the one after is written, from registers that global memory filled a stage earlier.
// Measured (4096 -> 4096, 4096 rows, bf16): 159 us = 865 TFLOP/s, a library product of that size 1220; its gradient at 2048 rows
// 131 us = 526 (1050 of matrix work, two pieces); 8192 x 2048 -> 1024 f32 118 us = 292 (875 of matrix work; the f32 matrix
// unit's peak is 157).  Nothing is saturated: the matrix unit is busy 35 % of the cycles (gradient 40), VALU issue takes 46,
// LDS 35; two waves a SIMD, in step through the barrier, overlap them only in part.  Tried and slower, against 192 us at the
// time (the code for groups of 32 still in the same kernel, which spilled for it):  4-wave workgroups of 128 x 128 (251 us),
// halves of the waves taking turns at multiplying and staging (570 us), loads two stages ahead (no gain), partial sums held
// over whole groups (219 us: 64 registers spilled), raised wave priority (+10 %).
// ---------------------------------------------------------------------------------------------
template <int DT, bool GRAD> struct W4Pieces {          // pieces of the weights and of the activations
    static constexpr int W = !GRAD ? 1 : DT == GR_DT_F32 ? 3 : 2;
    static constexpr int X = DT == GR_DT_F32 ? 3 : GRAD && DT == GR_DT_F16 ? 2 : 1;
    // Products of pieces i, j with i + j < TOP count.  What the gradients leave out is at most 2^-23 of |w x| in f32 (1 x 2 and
    // 2 x 1: 2^-8 of one factor, 2^-16 of the other), 2^-16 in f16 (1 x 1; with the weight's rest 1.5 * 2^-16), with either sign.
    static constexpr int TOP = W > X ? W : X;
    static constexpr bool NEAR = W > 1 && X > 1;
    static constexpr int PROD = !GRAD ? X : DT == GR_DT_F32 ? 6 : DT == GR_DT_F16 ? 3 : 2;
};
template <int DT, bool GRAD, int TM, int TN, int WM, int WN, int KS>
struct W4Gemm {
    using P = W4Pieces<DT, GRAD>;
    static constexpr int NT = WM * WN * 64, BM = WM * TM * 16, BN = WN * TN * 16;
    static constexpr int A_ONE = BM / 16 * KS * 64, X_ONE = BN / 16 * KS * 64;      // 16-byte slots of one piece
    static constexpr int SC = GRAD ? 0 : NT;            // forward: f32 scales of the stage's steps, one per row (KS * BM of them, repeated)
    static constexpr int SC0 = A_ONE * P::W + X_ONE * P::X, SLOTS = SC0 + SC / 4;
    static constexpr int LDS = 3 * SLOTS * 16;
    static constexpr int AV = BM / 16 * 64 / NT, XV = X_ONE / NT;
    static_assert(BM / 16 * 64 % NT == 0 && X_ONE % NT == 0, "stage loads must divide evenly");
    static_assert(LDS <= 160 * 1024, "LDS");
    static_assert(GRAD || NT % (KS * BM) == 0, "one scale per thread and stage");
    static_assert(KS == (!GRAD && P::X == 1 ? 2 : 1), "body16 takes two steps a stage, body one");
};

template <int DT, int ST, bool HALF, bool GRAD, int TM, int TN, int WM, int WN, int KS>
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
    W4Raw<DT, HALF> xreg[G::XV];
    uint8_t zreg[GRAD ? 1 : G::AV][KS];
    W4Raw<ST> sreg[GRAD ? G::AV : 1][KS];                 // GRAD: scales and zeros run along the steps
    uint2 szreg[GRAD ? G::AV : 1][KS];
    const T* xrow[G::XV];
    int xk[G::XV];
#pragma unroll
    for (int v = 0; v < G::XV; v++) {
        const int f = tid + v * G::NT, l = f & 63, ts = f >> 6;
        const int64_t n = n0 + ts / KS * 16 + (l & 15);
        xk[v] = ts % KS * 32 + (l >> 4) * 8;
        xrow[v] = (const T*)p.x + (n < p.N ? n : p.N - 1) * p.ldx + xk[v];   // columns beyond the batch: computed, not stored
    }
    size_t grow[G::AV], zrow[G::AV];                      // GRAD: scales / zeros of the thread's row
    const unsigned* wsrc[G::AV];
#pragma unroll
    for (int v = 0; v < G::AV; v++) {
        const int row = m0 + (tid + v * G::NT) / 64 * 16 + lr;
        const size_t g_ = GRAD ? (size_t)((row < p.R ? row : p.R - 1) / (p.gsteps * 32)) : 0;
        grow[v] = g_ * p.Mp + lh * 8;
        zrow[v] = g_ * p.zstride + lh * 8;
        wsrc[v] = (const unsigned*)(p.pack + ((size_t)(m0 / 16 + (tid + v * G::NT) / 64) * p.chunks) * 64 + lane);
    }
    typename W4Type<ST>::T screg;                         // forward: scale of row m0 + tid % BM, step tid / BM % KS of the stage
    const int sstep = __builtin_amdgcn_readfirstlane(tid / G::BM % KS);
    int zg = 0, zrem = 0;                                 // group of the next step to load
    auto load_w = [&](int s) {                            // weights with their scales and zeros
#pragma unroll
        for (int v = 0; v < G::AV; v++) {
            const unsigned* src = wsrc[v] + (size_t)(s * KS / 4) * 256 + s * KS % 4;
            if constexpr (KS == 2) {
                const uint2 d = *(const uint2*)src;
                wreg[v][0] = d.x; wreg[v][1] = d.y;
            } else {
                wreg[v][0] = *src;
            }
        }
        int sg = zg;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            if constexpr (!GRAD) {
#pragma unroll
                for (int v = 0; v < G::AV; v++)
                    zreg[v][i] = p.zeros[(size_t)zg * p.zstride + m0 + (tid + v * G::NT) / 64 * 16 + lr];
                sg = sstep == i ? zg : sg;
                zrem++;
                const bool end = zrem == p.gsteps;        // the next step, if there is one, begins a group
                zg += end && (s * KS + i + 1) * 32 < p.C ? 1 : 0;
                zrem = end ? 0 : zrem;
            } else {
#pragma unroll
                for (int v = 0; v < G::AV; v++) {
                    sreg[v][i].load((const typename W4Type<ST>::T*)p.scales + grow[v] + (s * KS + i) * 32);
                    szreg[v][i] = *(const uint2*)(p.zeros + zrow[v] + (s * KS + i) * 32);
                }
            }
        }
        if constexpr (!GRAD) screg = ((const typename W4Type<ST>::T*)p.scales)[(size_t)sg * p.Mp + m0 + tid % G::BM];
    };
    auto load = [&](int s) {
        load_w(s);
        if ((s + 1) * KS * 32 <= p.C) {
#pragma unroll
            for (int v = 0; v < G::XV; v++) xreg[v].load(xrow[v] + s * KS * 32);
        } else {
#pragma unroll
            for (int v = 0; v < G::XV; v++) xreg[v].load_part(xrow[v] + s * KS * 32, p.C - s * KS * 32 - xk[v], p.C >= 8);
        }
    };
    union Frag { w4_u32x4 u; w4_bf16x8 b; w4_f16x8 h; };
    auto store_w = [&](w4_u32x4* buf, int v, int i) {
        w4_u32x4* dst = buf + ((tid + v * G::NT) / 64 * KS + i) * 64 + lane;
        Frag c;
        if constexpr (F16OP) {
            c.h = w4_ints_f16(wreg[v][i], 1024.f + (float)zreg[v][i]);
            dst[0] = c.u;
        } else if constexpr (!GRAD) {
            c.b = w4_ints_bf16(wreg[v][i], 1024.f + (float)zreg[v][i]);
            dst[0] = c.u;
        } else {
            float f[8], sc[8];
            sreg[v][i].get(sc);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const unsigned zz = (q < 2 ? szreg[v][i].x : szreg[v][i].y) >> (16 * (q & 1));
                w4_ints_f32(wreg[v][i], q, 1024.f + (float)(zz & 255u), 1024.f + (float)(zz >> 8 & 255u), f[2 * q], f[2 * q + 1]);
                f[2 * q] *= sc[2 * q];
                f[2 * q + 1] *= sc[2 * q + 1];
            }
            w4_bf16x8 pc[P::W];
            w4_pieces<P::W, P::NEAR>(f, pc);
#pragma unroll
            for (int q = 0; q < P::W; q++) {
                c.b = pc[q];
                dst[q * G::A_ONE] = c.u;
            }
        }
    };
    auto store_x = [&](w4_u32x4* buf, int v) {
        w4_u32x4* dst = buf + P::W * G::A_ONE + tid + v * G::NT;
        xreg[v].settle((uintptr_t)xrow[v] & 2 ? 16 : 0);
        if constexpr (P::X == 1) {
            dst[0] = xreg[v].q[0];
        } else {
            float f[8];
            xreg[v].get(f);
            w4_bf16x8 pc[P::X];
            w4_pieces<P::X, P::NEAR, DT == GR_DT_F32>(f, pc);
#pragma unroll
            for (int q = 0; q < P::X; q++) {
                Frag c;
                c.b = pc[q];
                dst[q * G::X_ONE] = c.u;
            }
        }
    };
    auto store_sc = [&](w4_u32x4* buf) {
        if constexpr (!GRAD) ((float*)(buf + G::SC0))[tid] = (float)screg;
    };
    auto store = [&](w4_u32x4* buf) {
#pragma unroll
        for (int v = 0; v < G::AV; v++)
#pragma unroll
            for (int i = 0; i < KS; i++) store_w(buf, v, i);
        store_sc(buf);
#pragma unroll
        for (int v = 0; v < G::XV; v++) store_x(buf, v);
    };

    w4_f32x4 acc[TM][TN], part[GRAD ? 1 : TM][GRAD ? 1 : TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
    const w4_f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    int crem = 0;                                         // steps of the group multiplied so far
    bool fresh = true;                                    // none of them is in `part`
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
            // scales come through LDS: a wait on a global load here would wait for the next stage's loads as well
            w4_f32x4 sc[TM];
            if (flush) {
#pragma unroll
                for (int t = 0; t < TM; t++) sc[t] = *(const w4_f32x4*)((const float*)(buf + G::SC0) + i * G::BM + (wm * TM + t) * 16 + lh * 4);
            }
            if (fresh) {
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
            fresh = flush;
            crem = crem + 1 == p.gsteps ? 0 : crem + 1;
            if (flush) {
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int u = 0; u < TN; u++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[t][u][r] = __builtin_fmaf(part[t][u][r], sc[t][r], acc[t][u][r]);
            }
        }
    };

    // Two stages (KS = 1: 64 contraction steps) without borders: straight-line code.  Its matrix instructions are cut into slices
    // of one row tile (TN of them), and the staging is dealt out over the slices, where it runs in the matrix unit's shadow.
    // FIRST: the steps begin a group, FLUSH: they end one.  fa[0], fx[0] hold the first step's operands, then the next pair's.
    Frag fa[2][P::W][TM], fx[2][P::X][TN];
    auto read_a = [&](int f, const w4_u32x4* buf) {
#pragma unroll
        for (int q = 0; q < P::W; q++)
#pragma unroll
            for (int t = 0; t < TM; t++) fa[f][q][t].u = buf[q * G::A_ONE + (wm * TM + t) * 64 + lane];
    };
    auto read_x = [&](int f, const w4_u32x4* buf) {
#pragma unroll
        for (int q = 0; q < P::X; q++)
#pragma unroll
            for (int t = 0; t < TN; t++) fx[f][q][t].u = buf[P::W * G::A_ONE + q * G::X_ONE + (wn * TN + t) * 64 + lane];
    };
    w4_u32x4 *b0 = w4_lds, *b1 = w4_lds + G::SLOTS, *b2 = w4_lds + 2 * G::SLOTS;      // stages s, s + 1, s + 2
    auto body = [&]<bool FIRST, bool FLUSH>(int s) {
        constexpr int NSL = P::PROD * TM, NW = G::AV, ITEMS = NW + 2 + 2 * G::XV;
        auto mul = [&](int f, int qa, int qx, int t, int u, w4_f32x4 c) {
            if constexpr (F16OP) return w4_mfma(fa[f][qa][t].h, fx[f][qx][u].h, c);
            else return w4_mfma(fa[f][qa][t].b, fx[f][qx][u].b, c);
        };
        w4_f32x4 sc[GRAD ? 1 : TM];
        auto flush = [&](int t) {
#pragma unroll
            for (int u = 0; u < TN; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[t][u][r] = __builtin_fmaf(part[t][u][r], sc[t][r], acc[t][u][r]);
        };
#pragma unroll
        for (int f = 0; f < 2; f++) {                     // stage s + f; its operands are fa[f], fx[f]
            int sl = 0;
            auto item = [&](int it) {
                if (it < NW) store_w(b2, it, 0);
                else if (it == NW) store_sc(b2);
                else if (it == NW + 1) load_w(s + f + 3);
                else if ((it - NW) % 2 == 0) store_x(b2, (it - NW - 2) / 2);
                else xreg[(it - NW - 2) / 2].load(xrow[(it - NW - 2) / 2] + (s + f + 3) * 32);
            };
            int pr = 0;
#pragma unroll
            for (int qa = 0; qa < P::W; qa++)
#pragma unroll
                for (int qx = 0; qx < P::X; qx++) {
                    if (qa + qx >= P::TOP) continue;
                    pr++;
#pragma unroll
                    for (int t = 0; t < TM; t++) {
#pragma unroll
                        for (int u = 0; u < TN; u++) {
                            if constexpr (GRAD) acc[t][u] = mul(f, qa, qx, t, u, acc[t][u]);
                            else part[t][u] = mul(f, qa, qx, t, u, FIRST && f == 0 && qx == 0 ? zero4 : part[t][u]);
                        }
                        if (pr == 1 && t == 0) read_a(1 - f, b1);
                        if (pr == 1 && t == 1) read_x(1 - f, b1);
#pragma unroll
                        for (int it = 0; it < ITEMS; it++)
                            if (it * NSL / ITEMS == sl) item(it);
                        if constexpr (!GRAD && FLUSH) {
                            if (f == 1 && pr == P::PROD) {
                                sc[t] = *(const w4_f32x4*)((const float*)(b0 + G::SC0) + (wm * TM + t) * 16 + lh * 4);
                                if (t > 0) flush(t - 1);
                            }
                        }
                        sl++;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            if constexpr (!GRAD && FLUSH) {
                if (f == 1) flush(TM - 1);
            }
            __syncthreads();
            w4_u32x4* t = b0; b0 = b1; b1 = b2; b2 = t;
        }
    };

    // The same for 16-bit activations, forward (KS = 2): a row tile's partial sums live for one slice only -- they are scaled and
    // added after every 64 steps (PERSTEP: 32, for groups that are an odd multiple of that), also inside a group.  Partial sums
    // held over whole groups would need 64 more registers than the 256 there are.
    Frag qa[2][KS], qx[2][KS][TN];
    auto read_qa = [&](const w4_u32x4* buf, int t) {
#pragma unroll
        for (int i = 0; i < KS; i++) qa[t & 1][i].u = buf[((wm * TM + t) * KS + i) * 64 + lane];
    };
    auto read_qx = [&](int set, const w4_u32x4* buf, int t) {
#pragma unroll
        for (int i = 0; i < KS; i++) qx[set][i][t].u = buf[G::A_ONE + ((wn * TN + t) * KS + i) * 64 + lane];
    };
    auto body16 = [&]<bool PERSTEP, int SET>(int s) {
        constexpr int NW = G::AV * KS, ITEMS = NW + 2 + 2 * G::XV;
        auto item = [&](int it) {
            if (it < NW) store_w(b2, it / KS, it % KS);
            else if (it == NW) store_sc(b2);
            else if (it == NW + 1) load_w(s + 3);
            else if ((it - NW) % 2 == 0) store_x(b2, (it - NW - 2) / 2);
            else xreg[(it - NW - 2) / 2].load(xrow[(it - NW - 2) / 2] + (s + 3) * KS * 32);
        };
        constexpr int FS = PERSTEP ? KS : 1;               // partial sums a slice leaves behind, one after the other
        w4_f32x4 ps[2][TN], sc[2];
        auto flush = [&](int j) {
#pragma unroll
            for (int u = 0; u < TN; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[j / FS][u][r] = __builtin_fmaf(ps[j & 1][u][r], sc[j & 1][r], acc[j / FS][u][r]);
        };
#pragma unroll
        for (int t = 0; t < TM; t++) {
            read_qa(t + 1 < TM ? b0 : b1, (t + 1) % TM);
            if (t < TN) read_qx(1 - SET, b1, t);
#pragma unroll
            for (int i = 0; i < KS; i++) {
                const int j = t * FS + (PERSTEP ? i : 0);
                if (PERSTEP || i == 0)
                    sc[j & 1] = *(const w4_f32x4*)((const float*)(b0 + G::SC0) + (PERSTEP ? i : KS - 1) * G::BM + (wm * TM + t) * 16 + lh * 4);
#pragma unroll
                for (int u = 0; u < TN; u++) {
                    const w4_f32x4 c = PERSTEP || i == 0 ? zero4 : ps[j & 1][u];
                    if constexpr (F16OP) ps[j & 1][u] = w4_mfma(qa[t & 1][i].h, qx[SET][i][u].h, c);
                    else ps[j & 1][u] = w4_mfma(qa[t & 1][i].b, qx[SET][i][u].b, c);
                }
                if (j > 0 && (PERSTEP || i == KS - 1)) flush(j - 1);
            }
#pragma unroll
            for (int it = 0; it < ITEMS; it++)
                if (it * TM / ITEMS == t) item(it);
            __builtin_amdgcn_sched_barrier(0);
        }
        flush(TM * FS - 1);
        __syncthreads();
        w4_u32x4* t = b0; b0 = b1; b1 = b2; b2 = t;
    };

    load(0);
    store(b0);
    if (nstages > 1) { load(1); store(b1); }
    if (nstages > 2) load(2);
    __syncthreads();
    int s = 0;
    const int plain = p.C / (KS * 32) - 3;                // stages s < plain: s + 3 is whole
    if constexpr (!GRAD && P::X == 1) {
        if (plain >= 2) {
            read_qa(b0, 0);
#pragma unroll
            for (int t = 0; t < TN; t++) read_qx(0, b0, t);
            bool perstep = false;
            if constexpr (TN == 2) perstep = p.gsteps % 2;             // the whole tile is not used for such groups
            if (perstep) {
                if constexpr (TN == 2)
                    for (; s + 2 <= plain; s += 2) {
                        body16.template operator()<true, 0>(s);
                        body16.template operator()<true, 1>(s + 1);
                    }
            } else {
                for (; s + 2 <= plain; s += 2) {
                    body16.template operator()<false, 0>(s);
                    body16.template operator()<false, 1>(s + 1);
                }
            }
            crem = s * KS % p.gsteps;
        }
    } else if (plain >= 2 && (GRAD || p.gsteps % 2 == 0)) {
        read_a(0, b0);
        read_x(0, b0);
        if constexpr (GRAD) {
            for (; s + 2 <= plain; s += 2) body.template operator()<false, false>(s);
        } else if (p.gsteps == 2) {
            for (; s + 2 <= plain; s += 2) body.template operator()<true, true>(s);
        } else {
            while (s + p.gsteps <= plain) {
                const int e = s + p.gsteps - 2;
                body.template operator()<true, false>(s);
                for (s += 2; s < e; s += 2) body.template operator()<false, false>(s);
                body.template operator()<false, true>(s);
                s += 2;
            }
        }
    }
    for (; s < nstages; s++) {
        if (s + 2 < nstages) {
            store(b2);
            if (s + 3 < nstages) load(s + 3);
        }
#pragma unroll
        for (int i = 0; i < KS; i++) {
            if (i > 0 && (s * KS + i) * 32 >= p.C) break;
            step(b0, i, (s * KS + i + 1) * 32 >= p.C);
        }
        __syncthreads();
        w4_u32x4* t = b0; b0 = b1; b1 = b2; b2 = t;
    }

#pragma unroll
    for (int t = 0; t < TM; t++) {
        const int m = m0 + (wm * TM + t) * 16 + lh * 4;
        float bias[4];
        w4_bias<GRAD>(p, m, bias);
#pragma unroll
        for (int u = 0; u < TN; u++) {
            const int64_t n = n0 + (wn * TN + u) * 16 + lr;
            if (n < p.N && m < p.R) w4_put<DT, GRAD>(p, acc[t][u], bias, n, m);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// launchers (one translation unit per activation type: w4_f32.hip, w4_bf16.hip, w4_f16.hip, and w4_bf16_half.hip, w4_f16_half.hip
// for rows that begin in the middle of a dword)
// ---------------------------------------------------------------------------------------------
hipError_t w4_launch_f32(const W4Params&, int scale_type, bool grad, hipStream_t);
hipError_t w4_launch_bf16(const W4Params&, int scale_type, bool grad, hipStream_t);
hipError_t w4_launch_f16(const W4Params&, int scale_type, bool grad, hipStream_t);
hipError_t w4_launch_bf16_half(const W4Params&, int scale_type, bool grad, hipStream_t);      // rows that begin in the middle of a dword
hipError_t w4_launch_f16_half(const W4Params&, int scale_type, bool grad, hipStream_t);

#ifdef W4_KERNELS
template <int DT, int ST, bool HALF, int NT, int MT, int GS, bool GRAD>
static hipError_t launch_rows(const W4Params& p, hipStream_t st) {
    constexpr int D = DT == GR_DT_F32 || NT > 1 || GRAD || HALF ? 1 : 2;
    const int64_t blocks = (int64_t)((p.R + 16 * MT - 1) / (16 * MT)) * ((p.N + 16 * NT - 1) / (16 * NT));
    int waves = p.waves > 0 ? p.waves : blocks >= 2048 ? 4 : blocks >= 512 ? 8 : w4_rows_waves(NT);
    if (waves > p.chunks) waves = p.chunks;
    const size_t lds = (size_t)waves * MT * NT * 1024;
    auto kern = &k_w4_rows<DT, ST, HALF, NT, MT, GS, D, GRAD>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(waves * 64), lds, st, p);
    return hipGetLastError();
}
template <int DT, int ST, bool HALF, int NT, int MT, bool GRAD>
static hipError_t launch_rows(const W4Params& p, hipStream_t st) {
    if constexpr (GRAD) {
        return launch_rows<DT, ST, HALF, NT, MT, 1, true>(p, st);
    } else {
        if (p.gsteps % 4 == 0) return launch_rows<DT, ST, HALF, NT, MT, 1, false>(p, st);
        if constexpr (!(HALF && NT == 4))                  // that one is not taken for groups of odd multiples of 32
            if (p.gsteps % 2) return launch_rows<DT, ST, HALF, NT, MT, 4, false>(p, st);
        return launch_rows<DT, ST, HALF, NT, MT, 2, false>(p, st);
    }
}
template <int DT, int ST, bool HALF, bool GRAD, int TM, int TN, int WM, int WN, int KS>
static hipError_t launch_gemm(const W4Params& p, hipStream_t st) {
    using G = W4Gemm<DT, GRAD, TM, TN, WM, WN, KS>;
    typedef typename W4Type<DT>::T T;
    auto kern = &k_w4_gemm<DT, ST, HALF, GRAD, TM, TN, WM, WN, KS>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS);
    if (e != hipSuccess) return e;
    const int64_t across = (p.R + G::BM - 1) / G::BM;
    const int64_t most = 0xffffffffu / G::NT / across * G::BN;          // rows of a launch, whose threads are counted in 32 bits
    for (int64_t n0 = 0; n0 < p.N; n0 += most) {
        W4Params q = p;
        q.N = p.N - n0 < most ? p.N - n0 : most;
        q.x = (const T*)p.x + n0 * p.ldx;
        q.y = (T*)p.y + n0 * p.ldy;
        if (p.gate) q.gate = (const T*)p.gate + n0 * p.ldg;
        hipLaunchKernelGGL(kern, dim3((unsigned)(across * ((q.N + G::BN - 1) / G::BN))), dim3(G::NT), G::LDS, st, q);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <int DT, int ST, bool HALF, bool GRAD>
static hipError_t launch_typed(const W4Params& p, hipStream_t st) {
    // A variant's time is about that of a workgroup, which grows with the contraction, times the rounds that its workgroups need,
    // and something for each output.  In microseconds:  out * workgroups / 256 + chunk * chunks * rounds, where rounds is
    //   max(1, workgroups / (256 * more))            for small workgroups, several of which share a CU,
    //   1 + more * (ceil(workgroups / 256) - 1)      for large ones (LDS), one a CU.
    // The numbers are fitted to the variants' times at 900 sizes (17 to 8192 rows, 33 to 8192 on both sides, every group).  At 340
    // others (profiles/lowbit_variant_times.csv) the variant with the least estimate takes 2 to 6 % longer than the fastest one
    // (geometric mean by direction and type; at most 37 %); limits on the number of output tiles took 6 to 13 % and up to 3.3
    // times as long.
    // Small tiles carry short contractions and few rows, the tiled kernel large products (us, in the order of `fwd`):  bf16,
    // 320 rows 96 -> 6528  10.7 8.4 9.3 10.3 14.4 11.5;  f32, 384 rows 7680 -> 2848  -, -, 169 122 217 184;  bf16, 2464 rows
    // 3648 -> 2048  -, -, 159 110 138 81.  The tiled kernel's half tile: 2048 rows 4096 -> 4096 bf16, groups of 128  116 (whole
    // 95), of 32  118 (130: twice the partial sums, and registers spilled).
    struct Cost { float out, chunk, more; };
    constexpr bool F32 = DT == GR_DT_F32, F16 = DT == GR_DT_F16;
    constexpr Cost fwd[7] = {F32 ? Cost{0.05f, 0.16f, 0.67f} : Cost{0.05f, 0.09f, 0.83f},      // row tiles x batch tiles: 1 x 1
                             F32 ? Cost{0.05f, 0.22f, 0.71f} : Cost{0.05f, 0.11f, 0.68f},      // 2 x 1
                             Cost{0.09f, 0.21f, 0.74f},                                        // 2 x 2 (16-bit)
                             F32 ? Cost{0.30f, 0.59f, 0.60f} : Cost{0.18f, 0.31f, 0.57f},      // 4 x 2
                             Cost{2.32f, 0.58f, 1.25f},                                        // 4 x 4 (16-bit)
                             F32 ? Cost{2.88f, 2.80f, 1.32f} : Cost{5.72f, 2.91f, 1.20f},      // tiled
                             Cost{2.67f, 1.39f, 1.50f}};                                       // tiled, half the batch rows (16-bit)
    constexpr Cost grad[4] = {F32 ? Cost{0.05f, 0.28f, 0.72f} : Cost{0.05f, 0.20f, 0.77f},     // 2 x 1
                              F32 ? Cost{0.05f, 0.34f, 0.70f} : Cost{0.05f, 0.28f, 0.72f},     // 4 x 1
                              F32 ? Cost{0.80f, 1.08f, 1.26f} : Cost{1.35f, 0.78f, 1.15f},     // 8 x 2
                              F32 ? Cost{2.19f, 3.97f, 1.72f} : F16 ? Cost{0.69f, 2.76f, 1.82f} : Cost{4.08f, 3.20f, 1.43f}};  // tiled
    auto time = [&](const Cost& c, int rows, int cols, bool large, float slower) {          // of workgroups of rows x cols outputs
        const int64_t blocks = (int64_t)((p.R + rows - 1) / rows) * ((p.N + cols - 1) / cols);
        if (rows * cols < 128 * 128 && blocks > 1 << 23) return 1e30f;      // threads of a launch are counted in 32 bits
        const float share = (float)blocks / 256.f;
        const float rounds = large ? 1.f + c.more * (float)((blocks + 255) / 256 - 1) : share > c.more ? share / c.more : 1.f;
        return c.out * share + c.chunk * slower * (float)p.chunks * rounds;
    };
    const bool odd = p.gsteps % 2;                         // groups end inside 64 steps: the tiled kernels' partial sums end every 32
    constexpr int tiled_cols = F32 || (GRAD && F16) ? 128 : 256;
    int best = 0;
    float least = 3e38f;
    auto consider = [&](int i, float t) {
        if (t < least) { least = t; best = i; }
    };
    if constexpr (!GRAD) {
        consider(0, time(fwd[0], 16, 16, false, 1.f));
        consider(1, time(fwd[1], 32, 16, false, 1.f));
        if (p.N > 16) {
            if (!F32) consider(2, time(fwd[2], 32, 32, false, 1.f));
            consider(3, time(fwd[3], 64, 32, false, 1.f));
            // 4 x 4 spills registers where a chunk has several groups or rows begin inside a dword: measured against the above
            if (!F32 && !(HALF && odd)) consider(4, time(fwd[4], 64, 64, true, (odd ? 1.4f : p.gsteps % 4 ? 1.1f : 1.f) * (HALF ? 1.5f : 1.f)));
            if (!p.waves && (F32 || !odd)) consider(5, time(fwd[5], 128, tiled_cols, true, odd ? 1.2f : 1.f));
            if (!p.waves && !F32) consider(6, time(fwd[6], 128, 128, true, odd ? 1.1f : 1.f));
        }
        if (best == 0) return launch_rows<DT, ST, HALF, 1, 1, GRAD>(p, st);
        if (best == 1) return launch_rows<DT, ST, HALF, 1, 2, GRAD>(p, st);
        if constexpr (!F32) {
            if (best == 2) return launch_rows<DT, ST, HALF, 2, 2, GRAD>(p, st);
            if (best == 4) return launch_rows<DT, ST, HALF, 4, 4, GRAD>(p, st);
        }
        if (best == 3) return launch_rows<DT, ST, HALF, 2, 4, GRAD>(p, st);
    } else {
        // a workgroup's row tiles share one group: its scales go to the activations
        const int most = p.gsteps % 4 == 0 ? 8 : p.gsteps % 2 == 0 ? 4 : 2;
        consider(0, time(grad[0], 32, 16, false, 1.f));
        if (most >= 4) consider(1, time(grad[1], 64, 16, false, 1.f));
        if (p.N > 16) {
            if (most == 8) consider(2, time(grad[2], 128, 32, true, 1.f));
            if (!p.waves) consider(3, time(grad[3], 128, tiled_cols, true, 1.f));
        }
        if (best == 0) return launch_rows<DT, ST, HALF, 1, 2, GRAD>(p, st);
        if (best == 1) return launch_rows<DT, ST, HALF, 1, 4, GRAD>(p, st);
        if (best == 2) return launch_rows<DT, ST, HALF, 2, 8, GRAD>(p, st);
    }
    if constexpr (DT == GR_DT_F32 || (GRAD && DT == GR_DT_F16)) return launch_gemm<DT, ST, HALF, GRAD, 4, 2, 2, 4, 1>(p, st);
    else if constexpr (GRAD) return launch_gemm<DT, ST, HALF, GRAD, 4, 4, 2, 4, 1>(p, st);
    else if (best == 6) return launch_gemm<DT, ST, HALF, GRAD, 4, 2, 2, 4, 2>(p, st);
    else return launch_gemm<DT, ST, HALF, GRAD, 4, 4, 2, 4, 2>(p, st);
}
template <int DT, bool HALF>
static hipError_t launch_any(const W4Params& p, int scale_type, bool grad, hipStream_t st) {
    if (scale_type == GR_DT_F32) return grad ? launch_typed<DT, GR_DT_F32, HALF, true>(p, st) : launch_typed<DT, GR_DT_F32, HALF, false>(p, st);
    if (scale_type == GR_DT_BF16) return grad ? launch_typed<DT, GR_DT_BF16, HALF, true>(p, st) : launch_typed<DT, GR_DT_BF16, HALF, false>(p, st);
    return grad ? launch_typed<DT, GR_DT_F16, HALF, true>(p, st) : launch_typed<DT, GR_DT_F16, HALF, false>(p, st);
}
#endif
