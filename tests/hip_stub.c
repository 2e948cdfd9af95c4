/* A HIP runtime without a GPU for tests of failure handling: memory is host memory, kernels do not run, and a test says which copy
 * fails, which device is current for a thread and whether a capture is under way. Loaded with RTLD_GLOBAL before the library, whose calls
 * it then takes. */
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>
#include <stdlib.h>
#include <string.h>

static _Thread_local int device;
static _Thread_local hipError_t last;
static int devices = 2, capturing, launches, memsets, live, copies, fail_copy = -1, sticky = 1;

static hipError_t done(hipError_t e) {
    if (e != hipSuccess || !sticky) last = e;
    return e;
}
/* The n-th copy from now on fails (0: the next one; -1: none). keep: hipGetLastError keeps an error until it is read (ROCm 7), else a call that
 * succeeds clears it. */
void stub_fail_copy(int n, int keep) { fail_copy = n < 0 ? -1 : copies + n; sticky = keep; last = hipSuccess; }
void stub_stale_error(void) { last = hipErrorInvalidValue; }
void stub_capture(int on) { capturing = on; }
int stub_live(void) { return live; }
int stub_launches(void) { return launches; }
int stub_memsets(void) { return memsets; }          /* asynchronous ones: nodes of a graph under capture */
int stub_device(void) { return device; }
void stub_set_device(int d) { device = d; }

hipError_t hipGetDeviceCount(int * n) { *n = devices; return done(hipSuccess); }
hipError_t hipSetDevice(int d) { if (d < 0 || d >= devices) return done(hipErrorInvalidDevice); device = d; return done(hipSuccess); }
hipError_t hipGetDevice(int * d) { *d = device; return done(hipSuccess); }
hipError_t hipGetDeviceProperties(hipDeviceProp_t * p, int d) {
    (void) d;
    memset(p, 0, sizeof *p);
    p->multiProcessorCount = 256;
    p->sharedMemPerBlock = 160 << 10;
    return done(hipSuccess);
}
hipError_t hipGetLastError(void) { hipError_t e = last; last = hipSuccess; return e; }
const char * hipGetErrorString(hipError_t e) { return e == hipSuccess ? "no error" : "an error of the stub"; }
hipError_t hipDeviceSynchronize(void) { return done(hipSuccess); }
hipError_t hipStreamSynchronize(hipStream_t s) { (void) s; return done(hipSuccess); }
hipError_t hipStreamCreateWithFlags(hipStream_t * s, unsigned f) { (void) f; *s = (hipStream_t) malloc(1); return done(hipSuccess); }
hipError_t hipStreamDestroy(hipStream_t s) { free((void *) s); return done(hipSuccess); }
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus * c) { (void) s; *c = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone; return done(hipSuccess); }
hipError_t hipGetSymbolAddress(void ** p, const void * symbol) { *p = (void *) symbol; return done(hipSuccess); }
hipError_t hipFuncSetAttribute(const void * f, hipFuncAttribute a, int v) { (void) f; (void) a; (void) v; return done(hipSuccess); }
hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int * n, const void * f, int b, size_t l) { (void) f; (void) b; (void) l; *n = 2; return done(hipSuccess); }
/* while a capture is under way an allocation or a copy ends it with an error, as the runtime's default mode does */
static hipError_t take(void ** p, size_t n) {
    if (capturing) return done(hipErrorStreamCaptureUnsupported);
    if (!(*p = calloc(1, n ? n : 1))) return done(hipErrorOutOfMemory);
    ++live;
    return done(hipSuccess);
}
hipError_t hipMalloc(void ** p, size_t n) { return take(p, n); }
hipError_t hipHostMalloc(void ** p, size_t n, unsigned f) { (void) f; return take(p, n); }
hipError_t hipFree(void * p) {
    if (!p) return done(hipSuccess);
    if (capturing) return done(hipErrorStreamCaptureUnsupported);
    free(p);
    --live;
    return done(hipSuccess);
}
hipError_t hipMemcpy(void * to, const void * from, size_t n, hipMemcpyKind k) {
    (void) k;
    if (capturing) return done(hipErrorStreamCaptureUnsupported);
    if (copies++ == fail_copy) return done(hipErrorUnknown);
    memcpy(to, from, n);
    return done(hipSuccess);
}
hipError_t hipMemcpyAsync(void * to, const void * from, size_t n, hipMemcpyKind k, hipStream_t s) { (void) s; (void) k; memcpy(to, from, n); return done(hipSuccess); }
hipError_t hipMemcpy2D(void * to, size_t tp, const void * from, size_t fp, size_t w, size_t h, hipMemcpyKind k) {
    (void) k;
    if (capturing) return done(hipErrorStreamCaptureUnsupported);
    if (copies++ == fail_copy) return done(hipErrorUnknown);
    for (size_t i = 0; i < h; ++i) memcpy((char *) to + i * tp, (const char *) from + i * fp, w);
    return done(hipSuccess);
}
hipError_t hipMemset(void * p, int v, size_t n) { memset(p, v, n); return done(hipSuccess); }
hipError_t hipMemsetAsync(void * p, int v, size_t n, hipStream_t s) { (void) s; ++memsets; memset(p, v, n); return done(hipSuccess); }
hipError_t hipLaunchKernel(const void * f, dim3 g, dim3 b, void ** a, size_t l, hipStream_t s) { (void) f; (void) g; (void) b; (void) a; (void) l; (void) s; ++launches; return done(hipSuccess); }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t l, hipStream_t s) { (void) g; (void) b; (void) l; (void) s; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 * g, dim3 * b, size_t * l, hipStream_t * s) { memset(g, 0, sizeof *g); memset(b, 0, sizeof *b); *l = 0; *s = 0; return hipSuccess; }
