// distill.hip -- distillation loss against a teacher's top logits, and its gradient (gr_distill_topk).
//
// With c = log2(e) / tau and, over the classes the teacher leaves unnamed (open form; closed form: over all classes),
//   mr = max z_i,  w_i = exp2((z_i - mr) c),  Sr = sum w_i                                   one pass, running maximum and sum
//   M = max(mr, max of the named z),  St = Sr exp2((mr - M) c) + sum over named of exp2((z_j - M) c)
// the student's log-probabilities are  log q_j = (z_j - M) c ln2 - ln St  and  log q_rest = ln Sr + (mr - M) c ln2 - ln St, and
//   d loss / d z_i = tau (w_i exp2((mr - M) c) / St - p_rest w_i / Sr)   unnamed,   tau (q_j - p_j)   named.
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
    int V, k;
    float tau;
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

// Reductions over the workgroup of two values at once; every thread gets the results.  `buf` holds two slots per wave.
template <int NT, typename A, typename B, typename OA, typename OB>
__device__ __forceinline__ void kd_reduce2(A& a, B& b, double* buf, OA oa, OB ob) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a = oa(a, __shfl_xor(a, o));
        b = ob(b, __shfl_xor(b, o));
    }
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) {
            buf[(threadIdx.x >> 6) * 2] = (double)a;
            buf[(threadIdx.x >> 6) * 2 + 1] = (double)b;
        }
        __syncthreads();
        a = (A)buf[0];
        b = (B)buf[1];
#pragma unroll
        for (int w = 1; w < NT / 64; w++) {
            a = oa(a, (A)buf[w * 2]);
            b = ob(b, (B)buf[w * 2 + 1]);
        }
        __syncthreads();
    }
}

// One workgroup per row.  VPT 16-byte vectors per thread of the row stay in registers between the pass that finds its maximum
// and sum and the one that writes the gradient, so the row is read from memory once; what does not fit (BIG) is read again.
// LDS (dynamic): p [k] double | z [k] float | i [k] int | bits, one per class (OPEN), bit 32 = the first aligned element.
template <int DT, int NT, int VPT, bool BIG, bool OPEN>
__global__ __launch_bounds__(NT) void k_distill(KdParams p) {
    typedef typename KdType<DT>::T T;
    constexpr int VE = 16 / (int)sizeof(T);
    constexpr float NINF = -__builtin_inff();
    extern __shared__ __attribute__((aligned(16))) unsigned char kd_lds[];
    __shared__ double s_red[2 * (NT / 64)];
    double* s_p = (double*)kd_lds;
    float* s_z = (float*)(s_p + p.k);
    int* s_i = (int*)(s_z + p.k);
    unsigned* s_bits = (unsigned*)(s_i + p.k);
    const int64_t n = blockIdx.x;
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
    kd_u32x4 r[VPT];
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        const int i = tid + v * NT;
        if (i < nv) r[v] = zv[i];
        else r[v] = kd_drop<DT>(kd_u32x4{0, 0, 0, 0}, 0xffu);
    }
    float lz = tid < loose ? (float)z[li] : NINF;

    // ---- the teacher's row, while those loads are under way
    const bool bits = OPEN || p.bits;
    if (bits) {
        for (int i = tid; i < (V - h + 63) / 32; i += NT) s_bits[i] = 0u;
        __syncthreads();
    }
    const int64_t* ix = p.index + n * p.ld_top;
    int flags = 0;                                          // 1: a slot is live, 2: a bad index, 4: a class may be named twice
    double top = -__builtin_inf();
    for (int j = tid; j < k; j += NT) {
        const int64_t i = ix[j];
        const double t = kd_value(p.value, p.vt, n * p.ld_top + j) / (double)p.tau;
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
                flags |= 4;                                 // not known: compare them all
            }
            if (OPEN || !(t == -__builtin_inf())) flags |= 1;
            top = t > top ? t : top;
        }
    }
    kd_reduce2<NT>(top, flags, s_red, mx, [](int a, int b) { return a | b; });
    if (NT == 64) __syncthreads();                          // the slots, for the wave's other lanes
    const float gl = p.grad_loss ? p.grad_loss[n] : 1.f;
    if ((flags & 2) || !(flags & 1)) {
        const float v = (flags & 2) ? __builtin_nanf("") : 0.f;
        if (p.loss && tid == 0) p.loss[n] = v;
        if (g)
            for (int i = tid; i < V; i += NT) g[i] = (T)v;
        return;
    }
    if (OPEN) top = (double)p.lse[p.ld_top ? n : 0];
    double sum = 0;
    float M = NINF;                                         // maximum of the named logits
    for (int j = tid; j < k; j += NT) {
        const double e = s_i[j] < 0 ? 0. : exp(s_p[j] - top);
        s_p[j] = e;
        sum += e;
        if (OPEN && s_i[j] >= 0) M = s_z[j] > M ? s_z[j] : M;
    }

    // ---- the unnamed classes: running maximum and sum of what is not kept, maximum of what is
    const auto named = [&](int i) {                         // the bits of vector i
        return VE == 8 ? (s_bits[(i >> 2) + 1] >> ((i & 3) * 8)) & 0xffu : (s_bits[(i >> 3) + 1] >> ((i & 7) * 4)) & 0xfu;
    };
    if (OPEN) {
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int i = tid + v * NT;
            if (i < nv) r[v] = kd_drop<DT>(r[v], named(i));
        }
        const int b = li - h + 32;
        if (tid < loose && (s_bits[b >> 5] >> (b & 31) & 1u)) lz = NINF;
    }
    float m = lz;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        float f[VE];
        kd_unpack<DT>(r[v], f);
#pragma unroll
        for (int e = 0; e < VE; e++) m = f[e] > m ? f[e] : m;
    }
    float bm = NINF, bs = 0.f;
    if (BIG) {
        for (int i = tid + VPT * NT; i < nv; i += NT) {
            kd_u32x4 q = zv[i];
            if (OPEN) q = kd_drop<DT>(q, named(i));
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
    kd_reduce2<NT>(sum, m, s_red, add, mx);
    const double inv = OPEN ? 1. : 1. / sum;
    double rest = OPEN ? 1. - sum : 0.;
    if (rest < 0.) rest = 0.;
    const bool none = m == NINF;                            // no unnamed class, or none with a finite logit
    const float mr = none ? 0.f : m;
    if (OPEN) {
        float dummy = 0.f;
        M = m > M ? m : M;
        kd_reduce2<NT>(M, dummy, s_red, mx, add);
    } else {
        M = m;
    }

    float acc[VE], Sr = 0.f, part = 0.f;
#pragma unroll
    for (int e = 0; e < VE; e++) acc[e] = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        float f[VE];
        kd_unpack<DT>(r[v], f);
#pragma unroll
        for (int e = 0; e < VE; e++) acc[e] += ex(f[e], mr);
    }
#pragma unroll
    for (int e = 0; e < VE; e++) Sr += acc[e];
    Sr += ex(lz, mr);
    if (BIG) Sr += bs * ex(bm, mr);
    // merged probabilities: the first slot of a class takes them all, the others step back
    for (int j = tid; j < k; j += NT) {
        bool first = s_i[j] >= 0;
        if (flags & 4)
            for (int i = 0; i < j && first; i++) first = s_i[i] != s_i[j];
        if (OPEN && first) part += ex(s_z[j], M);
    }
    kd_reduce2<NT>(Sr, part, s_red, add, add);
    const float shift = none ? 0.f : ex(mr, M);
    const float St = part + Sr * shift;
    const bool tail = OPEN && !(rest <= 0.) && !(none && Sr == 0.f);
    const float a0 = gl * p.tau;
    const float A = a0 * (shift / St - (tail ? (float)rest / Sr : 0.f));
    if (g) {
        const bool same = (uintptr_t)(g + h) % 16 == 0;
        kd_u32x4* gv = (kd_u32x4*)(g + h);
        const auto put = [&](int i, kd_u32x4 q) {
            float f[VE];
            kd_unpack<DT>(q, f);
#pragma unroll
            for (int e = 0; e < VE; e++) f[e] = A * ex(f[e], mr);
            if (same) gv[i] = kd_packed<DT>(f);
            else
#pragma unroll
                for (int e = 0; e < VE; e++) g[h + i * VE + e] = (T)f[e];
        };
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int i = tid + v * NT;
            if (i < nv) put(i, r[v]);
        }
        if (BIG)
            for (int i = tid + VPT * NT; i < nv; i += NT) {
                kd_u32x4 q = zv[i];
                if (OPEN) q = kd_drop<DT>(q, named(i));
                put(i, q);
            }
        if (tid < loose) g[li] = (T)(A * ex(lz, mr));
    }
    __syncthreads();                                        // the named classes are written over; s_p is read across lanes
    const double lnS = log((double)St);
    constexpr double LN2 = 0.69314718055994530942;
    double kl = 0;
    for (int j = tid; j < k; j += NT) {
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
        if (pj > 0. || pj != pj) kl += pj * (log(pj) - ((double)d * LN2 - lnS));
        if (g) g[ij] = (T)(a0 * (__builtin_amdgcn_exp2f(d) / St - (float)pj));
    }
    if (p.loss) {
        double dummy = 0;
        kd_reduce2<NT>(kl, dummy, s_red, add, add);
        if (tail) kl += rest * (log(rest) - (log((double)Sr) + (double)ex.arg(mr, M) * LN2 - lnS));
        if (tid == 0) p.loss[n] = (float)((double)p.tau * (double)p.tau * kl);
    }
}

template <int DT, int NT, int VPT, bool BIG, bool OPEN>
hipError_t launch1(const KdParams& p, hipStream_t st) {
    const size_t lds = (size_t)p.k * 16 + (p.bits ? ((size_t)p.V + 95) / 32 * 4 : 0);
    auto kern = &k_distill<DT, NT, VPT, BIG, OPEN>;
    if (lds > 64 * 1024) {                                  // 2^20 classes: 128 KB of bits
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)p.N), dim3(NT), lds, st, p);
    return hipGetLastError();
}
template <int DT, bool OPEN>
hipError_t launch(const KdParams& p, hipStream_t st) {
    const int64_t nv = (int64_t)p.V * (int64_t)sizeof(typename KdType<DT>::T) / 16;
    if (nv <= 64 * 4) return launch1<DT, 64, 4, false, OPEN>(p, st);
    if (nv <= 256 * 4) return launch1<DT, 256, 4, false, OPEN>(p, st);
    if (nv <= 256 * 16) return launch1<DT, 256, 16, false, OPEN>(p, st);
    if (nv <= 512 * 16) return launch1<DT, 512, 16, false, OPEN>(p, st);
    if (nv <= 1024 * 16) return launch1<DT, 1024, 16, false, OPEN>(p, st);
    return launch1<DT, 1024, 16, true, OPEN>(p, st);
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
    KdParams p = {z, grad, index, value, value_type, teacher_lse, grad_loss, loss, N, ldz, ldg, ld_top, V, k, tau, 0, 0, V <= (1 << 20)};
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
