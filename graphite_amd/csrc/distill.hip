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

namespace {

constexpr int KD_MAX_K = 1024;
constexpr float LN2 = 0.69314718055994530942f;

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
};

__device__ __forceinline__ double kd_value(const void* v, int t, int64_t i) {
    if (t == GR_DT_F32) return (double)((const float*)v)[i];
    if (t == GR_DT_BF16) return (double)(float)((const __bf16*)v)[i];
    return (double)(float)((const _Float16*)v)[i];
}
__device__ __forceinline__ float kd_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// reductions over the workgroup; every thread gets the result.  `buf` has one slot per wave and is reused by the next call.
template <typename F, typename OP>
__device__ __forceinline__ F kd_reduce(F v, F* buf, OP op) {
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    const int nw = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = buf[0];
    for (int w = 1; w < nw; w++) v = op(v, buf[w]);
    __syncthreads();
    return v;
}

// One workgroup per row.
template <int DT, bool OPEN>
__global__ __launch_bounds__(256) void k_distill(KdParams p) {
    typedef typename KdType<DT>::T T;
    extern __shared__ unsigned kd_named[];                  // OPEN: bit i = class i is named
    __shared__ double s_p[KD_MAX_K];
    __shared__ int s_i[KD_MAX_K];
    __shared__ float s_z[KD_MAX_K];                         // the named logits (grad may overwrite z)
    __shared__ double s_red[16];
    __shared__ float s_redf[16];
    const int64_t n = blockIdx.x;
    const int tid = threadIdx.x, nt = blockDim.x, V = p.V;
    const T* z = (const T*)p.z + n * p.ldz;
    const float c = 1.44269504088896340736f / p.tau;
    const auto add = [](auto a, auto b) { return a + b; };
    const auto mx = [](auto a, auto b) { return a > b ? a : b; };

    // ---- the teacher's row
    if (OPEN) {
        for (int i = tid; i < (V + 31) / 32; i += nt) kd_named[i] = 0u;
    }
    __syncthreads();
    const int64_t* ix = p.index + n * p.ld_top;
    const int64_t vrow = n * p.ld_top;
    double bad = 0, top = -__builtin_inf(), live = 0;
    for (int j = tid; j < p.k; j += nt) {
        const int64_t i = ix[j];
        const double t = kd_value(p.value, p.vt, vrow + j) / (double)p.tau;
        if (i < -1 || i >= V) bad = 1;
        const bool on = i >= 0 && i < V;
        s_i[j] = on ? (int)i : -1;
        s_z[j] = on ? (float)z[i] : 0.f;
        s_p[j] = on ? t : -__builtin_inf();
        if (on) {
            if (OPEN) { live = 1; atomicOr(&kd_named[i >> 5], 1u << (i & 31)); }
            else if (!(t == -__builtin_inf())) live = 1;
            top = t > top ? t : top;
        }
    }
    bad = kd_reduce(bad, s_red, mx);
    live = kd_reduce(live, s_red, mx);
    top = OPEN ? (double)p.lse[p.ld_top ? n : 0] : kd_reduce(top, s_red, mx);
    const float gl = p.grad_loss ? p.grad_loss[n] : 1.f;
    T* g = p.grad ? (T*)p.grad + n * p.ldg : nullptr;
    if (bad != 0 || live == 0) {
        const float v = bad != 0 ? __builtin_nanf("") : 0.f;
        if (p.loss && tid == 0) p.loss[n] = v;
        if (g)
            for (int i = tid; i < V; i += nt) g[i] = (T)v;
        return;
    }
    double sum = 0;
    for (int j = tid; j < p.k; j += nt) {
        const double e = exp(s_p[j] - top);
        s_p[j] = s_i[j] < 0 ? 0. : e;
        sum += s_p[j];
    }
    sum = kd_reduce(sum, s_red, add);
    const double inv = OPEN ? 1. : 1. / sum;
    double rest = OPEN ? 1. - sum : 0.;
    if (rest < 0.) rest = 0.;

    // ---- the student's unnamed classes
    float m = -__builtin_inff(), s = 0.f;
    for (int i = tid; i < V; i += nt) {
        if (OPEN && (kd_named[i >> 5] >> (i & 31) & 1u)) continue;
        const float v = (float)z[i];
        const float mn = v > m ? v : m, base = mn == -__builtin_inff() ? 0.f : mn;
        s = s * kd_exp2((m - base) * c) + kd_exp2((v - base) * c);
        m = mn;
    }
    float mr = kd_reduce(m, s_redf, mx);
    const bool none = mr == -__builtin_inff();
    if (none) mr = 0.f;
    const float Sr = kd_reduce(s * kd_exp2((m - mr) * c), s_redf, add);

    // ---- the named ones: merged probabilities (first slot of a class), their logits
    float M = none ? -__builtin_inff() : mr;
    if (OPEN) {
        float t = M;
        for (int j = tid; j < p.k; j += nt)
            if (s_i[j] >= 0) { const float v = s_z[j]; t = v > t ? v : t; }
        M = kd_reduce(t, s_redf, mx);
    }
    float part = 0.f;
    double kl = 0;
    if (OPEN) {
        for (int j = tid; j < p.k; j += nt) {
            bool first = s_i[j] >= 0;
            for (int i = 0; i < j && first; i++) first = s_i[i] != s_i[j];
            if (first) part += kd_exp2((s_z[j] - M) * c);
        }
        part = kd_reduce(part, s_redf, add);
    }
    const float shift = none ? 0.f : kd_exp2((mr - M) * c);
    const float St = (OPEN ? part : 0.f) + Sr * shift;
    const float lnS = logf(St);
    const double tt = (double)p.tau * (double)p.tau;
    const bool tail = OPEN && !(rest <= 0.) && !(none && Sr == 0.f);
    const float a0 = gl * p.tau;
    const float A = a0 * (shift / St - (tail ? (float)rest / Sr : 0.f));
    if (g) {
        for (int i = tid; i < V; i += nt) g[i] = (T)(A * kd_exp2(((float)z[i] - mr) * c));
        __syncthreads();                                   // the named classes are written over
    }
    for (int j = tid; j < p.k; j += nt) {
        const int ij = s_i[j];
        bool first = ij >= 0;
        for (int i = 0; i < j && first; i++) first = s_i[i] != ij;
        if (!first) continue;
        double pj = s_p[j];
        for (int i = j + 1; i < p.k; i++) pj += s_i[i] == ij ? s_p[i] : 0.;
        pj *= inv;
        const float d = (s_z[j] - M) * c;
        const double lq = (double)(d * LN2) - (double)lnS;
        if (pj > 0. || pj != pj) kl += pj * (log(pj) - lq);
        if (g) g[ij] = (T)(a0 * (kd_exp2(d) / St - (float)pj));
    }
    if (p.loss) {
        kl = kd_reduce(kl, s_red, add);
        if (tail) kl += rest * (log(rest) - ((double)logf(Sr) + (double)((mr - M) * c * LN2) - (double)lnS));
        if (tid == 0) p.loss[n] = (float)(tt * kl);
    }
}

template <int DT>
hipError_t launch(const KdParams& p, hipStream_t st) {
    if (!p.lse) {
        hipLaunchKernelGGL((k_distill<DT, false>), dim3((unsigned)p.N), dim3(256), 0, st, p);
        return hipGetLastError();
    }
    const size_t lds = (size_t)(p.V + 31) / 32 * 4;
    static bool big = false;                               // 2^20 classes: 128 KB of bits
    if (!big) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_distill<DT, true>), hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
        if (e != hipSuccess) return e;
        big = true;
    }
    hipLaunchKernelGGL((k_distill<DT, true>), dim3((unsigned)p.N), dim3(256), lds, st, p);
    return hipGetLastError();
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
    if (!(tau > 0.f) || tau > 3e38f) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: tau must be positive and finite");
    if (teacher_lse && V > (1 << 20)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: at most 2^20 classes with teacher_lse");
    if (ldz < V || (grad && ldg < V) || (ld_top != 0 && ld_top < k)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: a row stride is shorter than its row");
    if (N == 0) return GR_OK;                          // empty batch: nothing to do (pointers may be null)
    if (!z || !index || !value || (!loss && !grad)) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: null pointer");
    if (((uintptr_t)z | (uintptr_t)grad) % size(dtype) || (uintptr_t)value % size(value_type))
        return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: misaligned tensor");
    if (grad == z && ldg != ldz) return gr_fail(ctx, GR_EINVAL, "gr_distill_topk: in place needs ldg == ldz");
    const KdParams p = {z, grad, index, value, value_type, teacher_lse, grad_loss, loss, N, ldz, ldg, ld_top, V, k, tau};
    hipStream_t st = (hipStream_t)stream;
    const double nv = (double)N * V, es = (double)size(dtype);
    ProfScope ps(ctx, "k_distill", st, 6.0 * nv, nv * es * (grad ? 2 : 1));
    GR_HIP(ctx, dtype == GR_DT_F32 ? launch<GR_DT_F32>(p, st) : dtype == GR_DT_BF16 ? launch<GR_DT_BF16>(p, st) : launch<GR_DT_F16>(p, st));
    return GR_OK;
}
