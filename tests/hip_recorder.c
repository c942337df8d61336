/* A HIP runtime that runs nothing: it keeps two pretend devices, hands out addresses without memory behind them, and records
 * kernel launches (name, grid, block, LDS bytes, the first eight bytes of the first argument).  Loaded in front of libgraphite_hip.so it shows on the CPU
 * what the host code of an entry point asks the runtime for.  Launches are refused where the runtime refuses them: 2^32 or more
 * threads in a dimension, more than 1024 in a workgroup, no workgroup at all. */
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>
#include <stdint.h>
#include <string.h>

enum { MAX_KERNELS = 1 << 18, MAX_LAUNCHES = 65536 };
typedef struct { const void* fn; const char* name; } Kernel;
typedef struct { const char* name; unsigned grid[3], block[3]; size_t lds; uint64_t arg; } Launch;
static Kernel kernels[MAX_KERNELS];
static Launch launches[MAX_LAUNCHES];
static int nkernels, nlaunches, device;
static hipError_t last;
static uintptr_t next = (uintptr_t)1 << 44;
static struct { dim3 g, b; size_t lds; hipStream_t st; } conf;

int rec_device(void) { return device; }
int rec_kernels(void) { return nkernels; }
const char* rec_kernel(int i) { return kernels[i].name; }
int rec_launches(void) { return nlaunches; }
void rec_clear(void) { nlaunches = 0; }
const char* rec_name(int i) { return launches[i].name; }
const unsigned* rec_grid(int i) { return launches[i].grid; }
const unsigned* rec_block(int i) { return launches[i].block; }
size_t rec_lds(int i) { return launches[i].lds; }
uint64_t rec_arg(int i) { return launches[i].arg; }

static hipError_t done(hipError_t e) { if (e != hipSuccess) last = e; return e; }
void** __hipRegisterFatBinary(const void* d) { (void)d; static void* h; return &h; }
void __hipUnregisterFatBinary(void** h) { (void)h; }
void __hipRegisterVar(void** h, void* v, char* a, char* b, int c, size_t d, int e, int f) { (void)h; (void)v; (void)a; (void)b; (void)c; (void)d; (void)e; (void)f; }
void __hipRegisterFunction(void** h, const void* fn, char* dev, const char* name, unsigned t, void* a, void* b, void* c, void* d, int* w) {
    (void)h; (void)dev; (void)t; (void)a; (void)b; (void)c; (void)d; (void)w;
    if (nkernels < MAX_KERNELS) { kernels[nkernels].fn = fn; kernels[nkernels++].name = name; }
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t st) { conf.g = g; conf.b = b; conf.lds = lds; conf.st = st; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* st) { *g = conf.g; *b = conf.b; *lds = conf.lds; *st = conf.st; return hipSuccess; }
hipError_t hipLaunchKernel(const void* fn, dim3 g, dim3 b, void** args, size_t lds, hipStream_t st) {
    (void)st;
    const uint64_t top = (uint64_t)1 << 32;
    if (!g.x || !g.y || !g.z || !b.x || !b.y || !b.z || (uint64_t)b.x * b.y * b.z > 1024 || lds > 160 * 1024 ||
        (uint64_t)g.x * b.x >= top || (uint64_t)g.y * b.y >= top || (uint64_t)g.z * b.z >= top) return done(hipErrorInvalidConfiguration);
    if (nlaunches == MAX_LAUNCHES) return done(hipErrorOutOfMemory);
    Launch* l = &launches[nlaunches++];
    memset(l, 0, sizeof *l);
    for (int i = 0; i < nkernels; i++) if (kernels[i].fn == fn) l->name = kernels[i].name;
    l->grid[0] = g.x; l->grid[1] = g.y; l->grid[2] = g.z;
    l->block[0] = b.x; l->block[1] = b.y; l->block[2] = b.z;
    l->lds = lds;
    if (args && args[0]) memcpy(&l->arg, args[0], 8);
    return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void* fn, hipFuncAttribute a, int v) { (void)fn; (void)a; return done(v > 160 * 1024 ? hipErrorInvalidValue : hipSuccess); }
hipError_t hipGetDeviceCount(int* n) { *n = 2; return hipSuccess; }
hipError_t hipSetDevice(int d) { if (d < 0 || d > 1) return done(hipErrorInvalidDevice); device = d; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = device; return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int d) { (void)d; memset(p, 0, sizeof *p); strcpy(p->gcnArchName, "gfx950"); return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void* s) { (void)s; *p = (void*)next; next += 256; return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { *p = (void*)next; next += (n + 511) & ~(size_t)255; return hipSuccess; }
hipError_t hipFree(void* p) { (void)p; return hipSuccess; }
hipError_t hipGetLastError(void) { const hipError_t e = last; last = hipSuccess; return e; }
const char* hipGetErrorString(hipError_t e) { return e == hipErrorInvalidConfiguration ? "invalid configuration" : "error"; }
hipError_t hipDeviceSynchronize(void) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t s) { (void)s; return hipSuccess; }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind k) { (void)d; (void)s; (void)n; (void)k; return hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind k, hipStream_t st) { (void)st; return hipMemcpy(d, s, n, k); }
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t st) { (void)d; (void)v; (void)n; (void)st; return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { *e = (hipEvent_t)next; next += 256; return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t e) { (void)e; return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) { (void)e; (void)s; return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t e) { (void)e; return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t a, hipEvent_t b) { (void)a; (void)b; *ms = 0.f; return hipSuccess; }
