// w4.hip -- linear layers whose weights are 4-bit integers with group scales: packing, forward, input gradient.
#include "common.h"
#include "w4.h"
#include <limits.h>
#include <new>

struct gr_w4 {
    gr_ctx* ctx = nullptr;
    int M = 0, K = 0, group = 0, G = 0, st = 0, Mp = 0, Kp = 0;
    bool has_zeros = false;              // else `zeros` is one row of eights
    char* mem = nullptr;                 // one allocation: pack | transposed pack | scales | zeros | bias
    w4_u32x4 *pack = nullptr, *packT = nullptr;
    void* scales = nullptr;
    uint8_t* zeros = nullptr;
    float* bias = nullptr;
};

static inline size_t dt_size(int dt) { return dt == GR_DT_F32 ? 4 : 2; }
static inline bool dt_ok(int dt) { return dt == GR_DT_F32 || dt == GR_DT_BF16 || dt == GR_DT_F16; }

// One packed dword (w4.h): eight contraction steps of one row.  TRANSPOSED: rows = k, steps = m.
template <bool TRANSPOSED>
__global__ void k_w4_pack(const uint8_t* __restrict__ q, int64_t ldq, int M, int K, int chunks, int64_t ndwords,
                          unsigned* __restrict__ out) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= ndwords) return;
    const int i = (int)(id & 3), lane = (int)(id >> 2) & 63;
    const int64_t tile = id >> 8;
    const int c = (int)(tile % chunks);
    const int64_t row = tile / chunks * 16 + (lane & 15);
    const int s0 = c * W4_CHUNK + i * 32 + (lane >> 4) * 8;
    unsigned w = 0;
    for (int e = 0; e < 8; e++) {
        const int64_t m = TRANSPOSED ? s0 + e : row, k = TRANSPOSED ? row : s0 + e;
        unsigned v = 0;
        if (m < M && k < K) v = (q[m * ldq + (k >> 1)] >> (4 * (k & 1))) & 15u;
        w |= v << (4 * ((e >> 1) + 4 * (e & 1)));
    }
    out[id] = w;
}
// scales / zeros [M][G] -> [G][Mp] (group-major: a tile's rows are contiguous), zero beyond M; bias copied
template <typename T>
__global__ void k_w4_scales(const T* __restrict__ s, int64_t lds, const uint8_t* __restrict__ z, int64_t ldz, int M, int G,
                            int Mp, T* __restrict__ so, uint8_t* __restrict__ zo) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= (int64_t)G * Mp) return;
    const int m = (int)(id % Mp), g = (int)(id / Mp);
    so[id] = m < M ? s[m * lds + g] : (T)0;
    if (z) zo[id] = m < M ? z[m * ldz + g] & 15 : 0;
    else if (g == 0) zo[id] = 8;
}

gr_ctx* w4_ctx(const gr_w4* w) { return w->ctx; }
int w4_out_features(const gr_w4* w) { return w->M; }
int w4_in_features(const gr_w4* w) { return w->K; }

extern "C" void gr_w4_destroy(gr_w4* w) {
    if (!w) return;
    if (w->mem) (void)hipFree(w->mem);       // the memory knows its device; the caller's current one stays
    delete w;
}

extern "C" int gr_w4_create(gr_ctx* ctx, const uint8_t* q, int64_t ldq, const void* scales, int scale_type, int64_t lds,
                            const uint8_t* zeros, int64_t ldz, const float* bias, int out_features, int in_features, int group,
                            int input_grad, void* stream, gr_w4** out) {
    if (!ctx) return GR_EINVAL;
    GR_HIP(ctx, hipSetDevice(ctx->device));
    if (!q || !scales || !out) return gr_fail(ctx, GR_EINVAL, "gr_w4_create: null pointer");
    *out = nullptr;
    const int M = out_features, K = in_features;
    if (M <= 0 || K <= 0 || M > INT_MAX - 256 || K > INT_MAX - 256) return gr_fail(ctx, GR_EINVAL, "gr_w4_create: %d x %d weights", M, K);
    if (group <= 0 || group % 32) return gr_fail(ctx, GR_EINVAL, "gr_w4_create: group %d is not a positive multiple of 32", group);
    if (!dt_ok(scale_type)) return gr_fail(ctx, GR_EINVAL, "gr_w4_create: unknown scale type %d", scale_type);
    const int G = (int)(((int64_t)K + group - 1) / group);
    if (ldq < ((int64_t)K + 1) / 2 || lds < G || (zeros && ldz < G))
        return gr_fail(ctx, GR_EINVAL, "gr_w4_create: a row stride is shorter than its row");
    // the packing kernels take a thread per eight weights, which a launch counts in 32 bits
    if (((int64_t)M + 127) / 128 * 128 * (((int64_t)K + 127) / 128 * 128) / 8 > 0xffffff00ll)
        return gr_fail(ctx, GR_EINVAL, "gr_w4_create: %d x %d are too many weights", M, K);
    hipStream_t st = (hipStream_t)stream;
    gr_w4* w = new (std::nothrow) gr_w4();
    if (!w) return gr_fail(ctx, GR_ENOMEM, "gr_w4_create: out of host memory");
    w->ctx = ctx; w->M = M; w->K = K; w->group = group; w->G = G; w->st = scale_type; w->has_zeros = zeros != nullptr;
    w->Mp = (M + 127) / 128 * 128; w->Kp = (K + 127) / 128 * 128;
    const size_t pk = (size_t)w->Mp * w->Kp / 2, ssz = gr_align((size_t)G * w->Mp * dt_size(scale_type));
    const size_t zsz = gr_align((size_t)(zeros ? G : 1) * w->Mp), bsz = bias ? gr_align((size_t)M * 4) : 0;
    hipError_t e = hipMalloc((void**)&w->mem, pk * (input_grad ? 2 : 1) + ssz + zsz + bsz);
    if (e != hipSuccess) {
        w->mem = nullptr;
        gr_w4_destroy(w);
        return gr_fail(ctx, GR_ENOMEM, "gr_w4_create: hipMalloc: %s", hipGetErrorString(e));
    }
    char* m = w->mem;
    w->pack = (w4_u32x4*)m; m += pk;
    if (input_grad) { w->packT = (w4_u32x4*)m; m += pk; }
    w->scales = m; m += ssz;
    w->zeros = (uint8_t*)m; m += zsz;
    const int64_t nd = (int64_t)(pk / 4), ns = (int64_t)G * w->Mp;
    const dim3 gp((unsigned)((nd + 255) / 256)), gs((unsigned)((ns + 255) / 256));
    hipLaunchKernelGGL(k_w4_pack<false>, gp, dim3(256), 0, st, q, ldq, M, K, w->Kp / W4_CHUNK, nd, (unsigned*)w->pack);
    if (input_grad)
        hipLaunchKernelGGL(k_w4_pack<true>, gp, dim3(256), 0, st, q, ldq, M, K, w->Mp / W4_CHUNK, nd, (unsigned*)w->packT);
    if (scale_type == GR_DT_F32)
        hipLaunchKernelGGL(k_w4_scales<float>, gs, dim3(256), 0, st, (const float*)scales, lds, zeros, ldz, M, G, w->Mp, (float*)w->scales, w->zeros);
    else
        hipLaunchKernelGGL(k_w4_scales<uint16_t>, gs, dim3(256), 0, st, (const uint16_t*)scales, lds, zeros, ldz, M, G, w->Mp, (uint16_t*)w->scales, w->zeros);
    e = hipGetLastError();
    if (bias && e == hipSuccess) {
        w->bias = (float*)m;
        e = hipMemcpyAsync(w->bias, bias, (size_t)M * 4, hipMemcpyDeviceToDevice, st);
    }
    if (e == hipSuccess) e = hipStreamSynchronize(st);       // the object may be used on any stream from here on
    if (e != hipSuccess) { gr_w4_destroy(w); return gr_fail(ctx, GR_EHIP, "gr_w4_create: %s", hipGetErrorString(e)); }
    *out = w;
    return GR_OK;
}

static hipError_t w4_launch(const W4Params& p, int dt, int scale_type, bool grad, hipStream_t st) {
    if (dt == GR_DT_F32) return w4_launch_f32(p, scale_type, grad, st);
    const bool half = (uintptr_t)p.x % 4 || (p.N > 1 && p.ldx % 2);       // some row begins in the middle of a dword
    if (dt == GR_DT_BF16) return half ? w4_launch_bf16_half(p, scale_type, grad, st) : w4_launch_bf16(p, scale_type, grad, st);
    return half ? w4_launch_f16_half(p, scale_type, grad, st) : w4_launch_f16(p, scale_type, grad, st);
}

static int w4_run(gr_ctx* ctx, const gr_w4* w, const char* who, bool grad, const void* x, int dt, int64_t N, int64_t ldx, const void* gate,
                  int64_t ldg, int relu, void* y, int64_t ldy, int waves, hipStream_t st) {
    if (!w) return gr_fail(ctx, GR_EINVAL, "%s: null layer", who);
    if (w->ctx != ctx) return gr_fail(ctx, GR_ESTATE, "%s: the layer belongs to another context", who);
    if (!dt_ok(dt)) return gr_fail(ctx, GR_EINVAL, "%s: unknown element type %d", who, dt);
    if (grad && !w->packT) return gr_fail(ctx, GR_ESTATE, "%s: the layer was created without input_grad", who);
    if (N < 0) return gr_fail(ctx, GR_EINVAL, "%s: negative batch", who);
    if (N == 0) return GR_OK;                          // empty batch: nothing to do (pointers may be null)
    W4Params p = {};
    p.C = grad ? w->M : w->K;
    p.R = grad ? w->K : w->M;
    if (!x || !y) return gr_fail(ctx, GR_EINVAL, "%s: null pointer", who);
    if (ldx < p.C || ldy < p.R || (gate && ldg < p.R)) return gr_fail(ctx, GR_EINVAL, "%s: a row stride is shorter than its row", who);
    const size_t es = dt_size(dt);
    if (((uintptr_t)x | (uintptr_t)y | (uintptr_t)gate) % es) return gr_fail(ctx, GR_EINVAL, "%s: misaligned tensor", who);
    if ((int64_t)((p.R + 15) / 16) * ((N + 15) / 16) > INT_MAX) return gr_fail(ctx, GR_EINVAL, "%s: batch too large", who);
    p.pack = grad ? w->packT : w->pack;
    p.scales = w->scales; p.zeros = w->zeros; p.Mp = w->Mp;
    p.zstride = w->has_zeros ? w->Mp : 0;
    p.chunks = (grad ? w->Mp : w->Kp) / W4_CHUNK;
    p.gsteps = w->group / 32;
    p.x = x; p.y = y; p.bias = w->bias; p.gate = gate;
    p.N = N; p.ldx = ldx; p.ldy = ldy; p.ldg = ldg; p.relu = relu; p.waves = waves;
    const double fl = 2.0 * (double)N * w->M * w->K;
    const double by = (double)w->M * w->K / 2 + (double)w->M * w->G * (dt_size(w->st) + (w->has_zeros ? 1 : 0)) + (double)N * (w->M + w->K) * es;
    ProfScope ps(ctx, grad ? "k_w4_grad" : "k_w4_forward", st, fl, by);
    const hipError_t e = w4_launch(p, dt, w->st, grad, st);
    GR_HIP(ctx, e);
    return GR_OK;
}

extern "C" int gr_linear_w4(gr_ctx* ctx, const gr_w4* w, const void* x, int dtype, int64_t N, int64_t ldx, int relu, void* y,
                            int64_t ldy, void* stream) {
    if (!ctx) return GR_EINVAL;
    GR_HIP(ctx, hipSetDevice(ctx->device));
    return w4_run(ctx, w, "gr_linear_w4", false, x, dtype, N, ldx, nullptr, 0, relu, y, ldy, 0, (hipStream_t)stream);
}
extern "C" int gr_linear_w4_input_grad(gr_ctx* ctx, const gr_w4* w, const void* grad_y, int dtype, int64_t N, int64_t ldgy,
                                       const void* gate, int64_t ldgate, void* grad_x, int64_t ldgx, void* stream) {
    if (!ctx) return GR_EINVAL;
    GR_HIP(ctx, hipSetDevice(ctx->device));
    return w4_run(ctx, w, "gr_linear_w4_input_grad", true, grad_y, dtype, N, ldgy, gate, ldgate, 0, grad_x, ldgx, 0, (hipStream_t)stream);
}

// Waves of a model's layers: the few-row kernels add in an order that only their number decides (a wave's chunks in turn, then
// the waves), so with a fixed one an image's logits and gradient are the same bits in every chunk, like the float layers'.
// GTSRBNet, groups of 64, us: 1 image 314 with 4 waves, 313 with 8 and 313 with the layers' own choice; 8192 images 13548,
// 13635 and 13370 (the tiled kernel, whose order is another).
constexpr int W4_MODEL_WAVES = 4;
int w4_model_forward(gr_ctx* ctx, const gr_w4* w, const float* x, int64_t N, int64_t ldx, int relu, float* y, int64_t ldy, hipStream_t st) {
    return w4_run(ctx, w, "gr_linear_w4", false, x, GR_DT_F32, N, ldx, nullptr, 0, relu, y, ldy, W4_MODEL_WAVES, st);
}
int w4_model_input_grad(gr_ctx* ctx, const gr_w4* w, const float* grad_y, int64_t N, int64_t ldgy, const float* gate, int64_t ldgate,
                        float* grad_x, int64_t ldgx, hipStream_t st) {
    return w4_run(ctx, w, "gr_linear_w4_input_grad", true, grad_y, GR_DT_F32, N, ldgy, gate, ldgate, 0, grad_x, ldgx, W4_MODEL_WAVES, st);
}
