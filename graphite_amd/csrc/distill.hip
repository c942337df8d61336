// distill.hip -- distillation loss against a teacher's top logits, and its gradient (gr_distill_topk).
//
// With c = log2(e) / tau and, over the classes the teacher leaves unnamed (open form; closed form: over all classes),
//   mr = max z_i,  w_i = exp2((z_i - mr) c),  Sr = sum w_i                                   one pass, running maximum and sum
//   M = max(mr, max of the named z),  St = Sr exp2((mr - M) c) + sum over named of exp2((z_j - M) c)
// the student's log-probabilities are  log q_j = (z_j - M) c ln2 - ln St  and  log q_rest = ln Sr + (mr - M) c ln2 - ln St, and
//   d loss / d z_i = tau (P q_i - p_rest w_i / Sr),  q_i = w_i exp2((mr - M) c) / St   unnamed,   tau (P q_j - p_j)   named,
// P = what the loss's terms hold of the teacher: 1, but the sum of the named p_j where no p_rest enters (it is 0, p_j of rounded
// logits adding up to 1 or more, or no unnamed class can take it): the softmax's normaliser then has that much weight.
// The unnamed sum has its own maximum, so q_rest keeps its digits when the named classes hold nearly everything (a difference
// 1 - sum q_j would not).  The teacher's few values are handled in 64 bits: p_rest IS a difference, next to zero.
#include "common.h"
#include <limits.h>
#include <math.h>

namespace {

constexpr int KD_MAX_K = 1024;

template <int DT> struct KdType;
template <> struct KdType<GR_DT_F32> { typedef float T; };
template <> struct KdType<GR_DT_BF16> { typedef __bf16 T; };
template <> struct KdType<GR_DT_F16> { typedef _Float16 T; };

struct KdParams {
    const void* z; void* grad;
    const int64_t* index; const void* value; int vt;
    const float *lse, *grad_loss; float* loss;
    int64_t N, ldz, ldg, ld_top;
    int64_t n0;              // first row of this launch
    int V, k;
    float tau;
    double inv_tau;
    float c_hi, c_lo;        // log2(e) / tau = c_hi + c_lo, both positive
    int bits;                // closed form: look for repeated classes with one bit per class (V <= 2^20)
};

__device__ __forceinline__ double kd_value(const void* v, int t, int64_t i) {
    if (t == GR_DT_F32) return (double)((const float*)v)[i];
    if (t == GR_DT_BF16) return (double)(float)((const __bf16*)v)[i];
    return (double)(float)((const _Float16*)v)[i];
}
typedef unsigned kd_u32x4 __attribute__((ext_vector_type(4)));

// exp2((v - m) * log2(e) / tau), the constant in two parts: in one, its rounding would tilt every exponent the same way.
// Both parts are positive, so that -inf stays -inf through the fma.
struct KdExp {
    float hi, lo;
    __device__ __forceinline__ float arg(float v, float m) const {
        const float d = v - m;
        return __builtin_fmaf(d, hi, d * lo);
    }
    __device__ __forceinline__ float operator()(float v, float m) const { return __builtin_amdgcn_exp2f(arg(v, m)); }
};

// 16 bytes of a row as floats, and back
template <int DT>
__device__ __forceinline__ void kd_unpack(kd_u32x4 r, float (&f)[DT == GR_DT_F32 ? 4 : 8]) {
    if constexpr (DT == GR_DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(r[i]);
    } else if constexpr (DT == GR_DT_BF16) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(r[i] << 16);
            f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    } else {
        union { kd_u32x4 u; _Float16 h[8]; } c;
        c.u = r;
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = (float)c.h[i];
    }
}
template <int DT>
__device__ __forceinline__ kd_u32x4 kd_packed(const float (&f)[DT == GR_DT_F32 ? 4 : 8]) {
    typedef typename KdType<DT>::T T;
    union { kd_u32x4 u; T t[16 / sizeof(T)]; } c;
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); i++) c.t[i] = (T)f[i];
    return c.u;
}
// the elements of a vector whose bit is set become -inf
template <int DT>
__device__ __forceinline__ kd_u32x4 kd_drop(kd_u32x4 r, unsigned bits) {
    if (bits) {
        if constexpr (DT == GR_DT_F32) {
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = (bits >> i & 1u) ? 0xff800000u : r[i];
        } else {
            const unsigned ninf = DT == GR_DT_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (bits >> (2 * i) & 1u) r[i] = (r[i] & 0xffff0000u) | ninf;
                if (bits >> (2 * i + 1) & 1u) r[i] = (r[i] & 0xffffu) | (ninf << 16);
            }
        }
    }
    return r;
}

// Reductions over a wave by data-parallel moves (lane 63 collects), the result in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float kd_move(float x, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double kd_move(double x, double none) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(__double2hiint(none), __double2hiint(x), CTRL, ROWS, 0xf, false),
                            __builtin_amdgcn_update_dpp(__double2loint(none), __double2loint(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float kd_last(float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63)); }
__device__ __forceinline__ double kd_last(double x) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), 63), __builtin_amdgcn_readlane(__double2loint(x), 63));
}
template <typename F, typename OP>
__device__ __forceinline__ F kd_wave(F x, F none, OP op) {
    x = op(x, kd_move<0x111, 0xf>(x, none));                // row_shr:1, 2, 4, 8
    x = op(x, kd_move<0x112, 0xf>(x, none));
    x = op(x, kd_move<0x114, 0xf>(x, none));
    x = op(x, kd_move<0x118, 0xf>(x, none));
    x = op(x, kd_move<0x142, 0xa>(x, none));                // row_bcast:15 into rows 1 and 3
    x = op(x, kd_move<0x143, 0xc>(x, none));                // row_bcast:31 into rows 2 and 3
    return kd_last(x);
}
// ... and over the workgroup; `slots` (one float per wave, 16-byte aligned) is not used again before the next barrier
template <int NT, typename OP>
__device__ __forceinline__ float kd_block(float x, float none, float* slots, OP op) {
    x = kd_wave(x, none, op);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = x;
        __syncthreads();
        x = slots[0];
#pragma unroll
        for (int w = 1; w < NT / 64; w++) x = op(x, slots[w]);
    }
    return x;
}

// One workgroup per row.  VPT 16-byte vectors per thread of the row stay in registers between the pass that finds its maximum,
// the one that sums and the one that writes the gradient, so the row is read from memory once; what does not fit (BIG) is read
// again, mostly from the caches.  Bound by memory: 4096 x 32768 bf16 120 us = 4.5 TB/s, a copy of that size takes 100 us.
// The teacher's few classes are the first wave's work.
// LDS (dynamic): p [k] double | z [k] float | i [k] int | bits, one per class (OPEN), bit 32 = the first aligned element.
template <int DT, int NT, int VPT, bool BIG, bool OPEN>
__global__ __launch_bounds__(NT) void k_distill(KdParams p) {
    typedef typename KdType<DT>::T T;
    constexpr int VE = 16 / (int)sizeof(T);
    constexpr float NINF = -__builtin_inff();
    extern __shared__ __attribute__((aligned(16))) unsigned char kd_lds[];
    __shared__ __attribute__((aligned(16))) float s_max[NT / 64], s_sum[NT / 64];
    __shared__ int s_flags;
    __shared__ float s_named, s_part;                       // maximum of the named logits, their sum of exp2
    __shared__ double s_mass;                               // sum of the teacher's exp
    double* s_p = (double*)kd_lds;
    float* s_z = (float*)(s_p + p.k);
    int* s_i = (int*)(s_z + p.k);
    unsigned* s_bits = (unsigned*)(s_i + p.k);
    const int64_t n = p.n0 + blockIdx.x;
    const int tid = threadIdx.x, V = p.V, k = p.k;
    const T* z = (const T*)p.z + n * p.ldz;
    T* g = p.grad ? (T*)p.grad + n * p.ldg : nullptr;
    const KdExp ex{p.c_hi, p.c_lo};
    const auto add = [](auto a, auto b) { return a + b; };
    const auto mx = [](auto a, auto b) { return a > b ? a : b; };

    // the row: h elements up to the first 16-byte border, nv vectors, the rest; thread t < h + rest also has ONE of the loose ones
    int h = (int)((16 - (uintptr_t)z % 16) % 16 / sizeof(T));
    if (h > V) h = V;
    const int nv = (V - h) / VE, loose = V - nv * VE;
    const int li = tid < h ? tid : nv * VE + tid;
    const kd_u32x4* zv = (const kd_u32x4*)(z + h);
    // vector tid + b of the row, b uniform: a scalar base and one 32-bit offset for all of a thread's vectors
    const unsigned toff = (unsigned)tid * 16u;
    const auto vec = [&](int b) { return *(const kd_u32x4*)((const char*)(zv + b) + toff); };
    kd_u32x4 r[VPT];
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        r[v] = kd_drop<DT>(kd_u32x4{0, 0, 0, 0}, 0xffu);
        if (tid < nv - v * NT) r[v] = vec(v * NT);
    }
    float lz = tid < loose ? (float)z[li] : NINF;

    // ---- the teacher's row, while those loads are under way
    const bool bits = OPEN || p.bits;
    if (bits) {
        for (int i = tid; i < (V - h + 63) / 32; i += NT) s_bits[i] = 0u;
        __syncthreads();
    }
    const bool first_wave = tid < 64;
    if (first_wave) {
        const int64_t* ix = p.index + n * p.ld_top;
        int flags = 0;                                      // 1: a slot is live, 2: a bad index, 4: a class may be named twice
        double top = -__builtin_inf();
        for (int j = tid; j < k; j += 64) {
            const int64_t i = ix[j];
            const double t = kd_value(p.value, p.vt, n * p.ld_top + j) * p.inv_tau;
            const bool on = i >= 0 && i < V;
            if (!on && i != -1) flags |= 2;
            s_i[j] = on ? (int)i : -1;
            s_z[j] = on ? (float)z[i] : 0.f;
            s_p[j] = on ? t : -__builtin_inf();
            if (on) {
                if (bits) {
                    const int b = (int)i - h + 32;
                    if (atomicOr(&s_bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u) flags |= 4;
                } else {
                    flags |= 4;                             // not known: compare them all
                }
                if (OPEN || !(t == -__builtin_inf())) flags |= 1;
                top = t > top ? t : top;
            }
        }
        flags = (__ballot(flags & 1) ? 1 : 0) | (__ballot(flags & 2) ? 2 : 0) | (__ballot(flags & 4) ? 4 : 0);
        top = OPEN ? (double)p.lse[p.ld_top ? n : 0] : kd_wave(top, -__builtin_inf(), mx);
        double sum = 0;
        float mn = NINF;
        for (int j = tid; j < k; j += 64) {
            const double e = s_i[j] < 0 ? 0. : exp(s_p[j] - top);
            s_p[j] = e;
            sum += e;
            if (OPEN && s_i[j] >= 0) mn = s_z[j] > mn ? s_z[j] : mn;
        }
        sum = kd_wave(sum, 0., add);
        mn = kd_wave(mn, NINF, mx);
        if (tid == 0) { s_flags = flags; s_mass = sum; s_named = mn; }
    }
    __syncthreads();
    const int flags = s_flags;
    const float gl = p.grad_loss ? p.grad_loss[n] : 1.f;
    if ((flags & 2) || !(flags & 1)) {
        const float v = (flags & 2) ? __builtin_nanf("") : 0.f;
        if (p.loss && tid == 0) p.loss[n] = v;
        if (g)
            for (int i = tid; i < V; i += NT) g[i] = (T)v;
        return;
    }

    // ---- the unnamed classes: running maximum and sum of what is not kept, maximum of what is
    constexpr int VW = 32 / VE;                              // vectors in a word of bits
    static_assert(NT % VW == 0, "");
    const int tw = tid / VW + 1, tb = tid % VW * VE;
    const auto named = [&](int b) { return (s_bits[tw + b / VW] >> tb) & ((1u << VE) - 1u); };      // of vector tid + b
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        if (OPEN && tid < nv - v * NT) r[v] = kd_drop<DT>(r[v], named(v * NT));
        __builtin_amdgcn_sched_barrier(0);
    }
    if (OPEN) {
        const int b = li - h + 32;
        if (tid < loose && (s_bits[b >> 5] >> (b & 31) & 1u)) lz = NINF;
    }
    // Between the passes the vectors are made opaque: otherwise the compiler keeps their unpacked floats, twice the registers.
    const auto forget = [&]() {
#pragma unroll
        for (int v = 0; v < VPT; v++) asm volatile("" : "+v"(r[v]));
    };
    float m = lz;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        float f[VE];
        kd_unpack<DT>(r[v], f);
#pragma unroll
        for (int e = 0; e < VE; e++) m = f[e] > m ? f[e] : m;
    }
    forget();
    float bm = NINF, bs = 0.f;
    if (BIG) {
        for (int b = VPT * NT; tid < nv - b; b += NT) {
            kd_u32x4 q = vec(b);
            if (OPEN) q = kd_drop<DT>(q, named(b));
            float f[VE], mn = bm, t = 0.f;
            kd_unpack<DT>(q, f);
#pragma unroll
            for (int e = 0; e < VE; e++) mn = f[e] > mn ? f[e] : mn;
            const float base = mn == NINF ? 0.f : mn;
#pragma unroll
            for (int e = 0; e < VE; e++) t += ex(f[e], base);
            bs = bs * ex(bm, base) + t;
            bm = mn;
        }
        m = bm > m ? bm : m;
    }
    m = kd_block<NT>(m, NINF, s_max, mx);
    const double mass = s_mass, inv = OPEN ? 1. : 1. / mass;
    double rest = OPEN ? 1. - mass : 0.;
    if (rest < 0.) rest = 0.;
    const bool none = m == NINF;                            // no unnamed class, or none with a finite logit
    const float mr = none ? 0.f : m;
    const float named_max = s_named;
    const float M = OPEN && named_max > m ? named_max : m;

    float acc[VE], Sr = 0.f;
#pragma unroll
    for (int e = 0; e < VE; e++) acc[e] = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        float f[VE];
        kd_unpack<DT>(r[v], f);
#pragma unroll
        for (int e = 0; e < VE; e++) acc[e] += ex(f[e], mr);
        __builtin_amdgcn_sched_barrier(0);
    }
    forget();
#pragma unroll
    for (int e = 0; e < VE; e++) Sr += acc[e];
    Sr += ex(lz, mr);
    if (BIG) Sr += bs * ex(bm, mr);
    if (OPEN && first_wave) {                               // every named class once
        float part = 0.f;
        for (int j = tid; j < k; j += 64) {
            bool first = s_i[j] >= 0;
            if (flags & 4)
                for (int i = 0; i < j && first; i++) first = s_i[i] != s_i[j];
            if (first) part += ex(s_z[j], M);
        }
        part = kd_wave(part, 0.f, add);
        if (tid == 0) s_part = part;
    }
    Sr = kd_block<NT>(Sr, 0.f, s_sum, add);
    if (NT == 64) __syncthreads();
    const float part = OPEN ? s_part : 0.f;
    const float shift = none ? 0.f : ex(mr, M);
    const float St = part + Sr * shift;
    const bool tail = OPEN && !(rest <= 0.) && !(none && Sr == 0.f);
    const float a0 = gl * p.tau;
    const float P = OPEN && !tail ? (float)mass : 1.f;
    // Unnamed gradients are a0 w_i / Sr (q_rest - p_rest): where the two are near 1, their difference is taken from what the
    // named classes hold on either side, else directly.
    const float q_rest = Sr * shift / St;
    const float A = !tail ? a0 * P * (shift / St) : a0 / Sr * (rest > 0.5 ? (float)mass - part / St : q_rest - (float)rest);
    if (g) {
        const bool same = (uintptr_t)(g + h) % 16 == 0;
        kd_u32x4* gv = (kd_u32x4*)(g + h);
        const auto put = [&](int b, kd_u32x4 q) {
            float f[VE];
            kd_unpack<DT>(q, f);
#pragma unroll
            for (int e = 0; e < VE; e++) f[e] = A * ex(f[e], mr);
            if (same) *(kd_u32x4*)((char*)(gv + b) + toff) = kd_packed<DT>(f);
            else
#pragma unroll
                for (int e = 0; e < VE; e++) (g + h + (int64_t)b * VE)[tid * VE + e] = (T)f[e];
        };
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            if (tid < nv - v * NT) put(v * NT, r[v]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (BIG)
            for (int b = VPT * NT; tid < nv - b; b += NT) {
                kd_u32x4 q = vec(b);
                if (OPEN) q = kd_drop<DT>(q, named(b));
                put(b, q);
            }
        if (tid < loose) g[li] = (T)(A * ex(lz, mr));
    }
    __syncthreads();                                        // the named classes are written over; s_p is read across lanes
    if (!first_wave) return;
    // At high temperatures the loss takes the normaliser St again, in 64 bits but for Sr: then the q of its logarithms add up to
    // 1, and an error of Sr moves the loss by (q_rest - p_rest) of it, next to nothing where student and teacher are alike; tau^2
    // would lift one float rounding of St over the whole loss (43 classes, loss 0.3: off by 3e-7 at tau = 4, 3e-6 at 20, 5e-3 at
    // 1000; so 8e-8 and 6e-6).  Closed form: where every class is named.  Up to 4 it is left out: 8192 rows of 43 classes 16.3 us
    // without, 17.9 with it.
    double Ur = (double)Sr * (double)shift, named_sum = (double)part;
    bool whole = false;                                     // closed form: the named classes are all there are
    if (p.tau > 4.f && p.loss && (OPEN || k >= V)) {
        named_sum = 0;
        float count = 0.f;
        for (int j = tid; j < k; j += 64) {
            bool first = s_i[j] >= 0;
            if (flags & 4)
                for (int i = 0; i < j && first; i++) first = s_i[i] != s_i[j];
            if (first) { named_sum += exp(((double)s_z[j] - (double)M) * p.inv_tau); count += 1.f; }
        }
        named_sum = kd_wave(named_sum, 0., add);
        if (OPEN) Ur = (double)Sr * (none ? 0. : exp(((double)mr - (double)M) * p.inv_tau));
        else whole = kd_wave(count, 0.f, add) == (float)V;
    }
    const double lnS = log(OPEN ? named_sum + Ur : whole ? named_sum : Ur);
    double kl = 0;
    for (int j = tid; j < k; j += 64) {                     // the first slot of a class takes all its mass
        const int ij = s_i[j];
        bool first = ij >= 0;
        double pj = s_p[j];
        if (flags & 4) {
            for (int i = 0; i < j && first; i++) first = s_i[i] != ij;
            for (int i = j + 1; i < k && first; i++) pj += s_i[i] == ij ? s_p[i] : 0.;
        }
        if (!first) continue;
        pj *= inv;
        const float d = ex.arg(s_z[j], M);
        if (pj > 0. || pj != pj) kl += pj * (log(pj) - (((double)s_z[j] - (double)M) * p.inv_tau - lnS));
        if (g) g[ij] = (T)(a0 * (P * (__builtin_amdgcn_exp2f(d) / St) - (float)pj));
    }
    if (p.loss) {
        kl = kd_wave(kl, 0., add);
        // log q_rest: as -log1p when it is near 0, where a difference of logarithms would lose it
        if (tail) kl += rest * (log(rest) + (q_rest > 0.5f ? log1p(named_sum / Ur) : lnS - (log((double)Sr) + ((double)mr - (double)M) * p.inv_tau)));
        if (tid == 0) p.loss[n] = (float)((double)p.tau * (double)p.tau * kl);
    }
}

template <int DT, int NT, int VPT, bool BIG, bool OPEN>
hipError_t launch1(KdParams p, hipStream_t st) {
    const size_t lds = (size_t)p.k * 16 + (p.bits ? ((size_t)p.V + 95) / 32 * 4 : 0);
    auto kern = &k_distill<DT, NT, VPT, BIG, OPEN>;
    if (lds > 64 * 1024) {                                  // 2^20 classes: 128 KB of bits
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    constexpr int64_t MOST = 0xffffffffu / NT;              // a launch's threads are counted in 32 bits
    for (; p.n0 < p.N; p.n0 += MOST) {
        const int64_t rows = p.N - p.n0 < MOST ? p.N - p.n0 : MOST;
        hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3(NT), lds, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <int DT, bool OPEN>
hipError_t launch(const KdParams& p, hipStream_t st) {
    const int64_t nv = (int64_t)p.V * (int64_t)sizeof(typename KdType<DT>::T) / 16;
    // A row costs a workgroup four barriers and the first wave's work on the teacher's classes, so short rows take few waves
    // (8192 rows of 2048 bf16: 64 threads 27 us, 256 45, 1024 146); long ones need loads in flight, and few rows many waves
    // (4096 rows of 32768 bf16: 256 threads with the row in registers 125 us, 1024 130; 1 row of 131072 f32: 1024 threads 26 us,
    // 256 66).  Rows beyond 64 KB are read twice rather than held by 1024 threads x 16 vectors, which spill (4096 x 32768 f32
    // 238 us against 260, 515 x 100003 135 against 143); 512 such workgroups run at a time, so the last 3 of 515 rows run alone.
    if (nv <= 64 * 4) return launch1<DT, 64, 4, false, OPEN>(p, st);
    if (nv <= 256 * 4) return launch1<DT, 256, 4, false, OPEN>(p, st);
    if (nv <= 1024 * 4) return p.N >= 512 ? launch1<DT, 256, 16, false, OPEN>(p, st) : launch1<DT, 1024, 4, false, OPEN>(p, st);
    return launch1<DT, 1024, 4, true, OPEN>(p, st);
}

}  // namespace

extern "C" int gr_distill_topk(gr_ctx* ctx, const void* z, int dtype, int64_t N, int V, int64_t ldz, const int64_t* index,
                               const void* value, int value_type, int k, int64_t ld_top, const float* teacher_lse, float tau,
                               const float* grad_loss, float* loss, void* grad, int64_t ldg, void* stream) {
    if (!ctx) return GR_EINVAL;
    GR_HIP(ctx, hipSetDevice(ctx->device));
    auto ok = [](int t) { return t == GR_DT_F32 || t == GR_DT_BF16 || t == GR_DT_F16; };
    auto size = [](int t) { return (uintptr_t)(t == GR_DT_F32 ? 4 : 2); };
    if (!ok(dtype) || !ok(value_type)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: unknown element type");
    if (N < 0 || N > INT_MAX || V <= 0 || V > INT_MAX - 65536) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: %lld rows of %d classes", (long long)N, V);
    if (k < 1 || k > KD_MAX_K) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: k = %d is not in [1, %d]", k, KD_MAX_K);
    if (!(tau >= 1e-6f && tau <= 1e6f)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: tau must lie in [1e-6, 1e6]");
    if (teacher_lse && V > (1 << 20)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: at most 2^20 classes with teacher_lse");
    if (ldz < V || (grad && ldg < V) || (ld_top != 0 && ld_top < k)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: a row stride is shorter than its row");
    if (N == 0) return GR_OK;                          // empty batch: nothing to do (pointers may be null)
    if (!z || !index || !value || (!loss && !grad)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: null pointer");
    if (((uintptr_t)z | (uintptr_t)grad) % size(dtype) || (uintptr_t)value % size(value_type))
        return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: misaligned tensor");
    if (grad == z && ldg != ldz) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: in place needs ldg == ldz");
    KdParams p = {z, grad, index, value, value_type, teacher_lse, grad_loss, loss, N, ldz, ldg, ld_top, 0, V, k, tau, 1.0 / (double)tau, 0, 0, V <= (1 << 20)};
    const double c = 1.4426950408889634074 / (double)tau;
    p.c_hi = (float)c;
    if ((double)p.c_hi >= c) p.c_hi = nextafterf(p.c_hi, 0.f);
    p.c_lo = (float)(c - (double)p.c_hi);
    hipStream_t st = (hipStream_t)stream;
    const double nv = (double)N * V, es = (double)size(dtype);
    ProfScope ps(ctx, "k_distill", st, 6.0 * nv, nv * es * (grad ? 2 : 1));
    const bool open = teacher_lse != nullptr;
    hipError_t e;
    if (dtype == GR_DT_F32) e = open ? launch<GR_DT_F32, true>(p, st) : launch<GR_DT_F32, false>(p, st);
    else if (dtype == GR_DT_BF16) e = open ? launch<GR_DT_BF16, true>(p, st) : launch<GR_DT_BF16, false>(p, st);
    else e = open ? launch<GR_DT_F16, true>(p, st) : launch<GR_DT_F16, false>(p, st);
    GR_HIP(ctx, e);
    return GR_OK;
}
