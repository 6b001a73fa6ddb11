/* A CUDA runtime of host memory for tests of the library's host code without a GPU: preloaded
 * before libijb200.so, its allocations are the heap's, its copies memcpy, its kernels nothing.
 * It keeps a log of calls, and a test can make one of them fail. */
#include <cuda_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#define MAX_LOG (1 << 16)
static const char *log_name[MAX_LOG];
static size_t log_value[MAX_LOG];
static int log_n;
static char fail_name[64], fail_after[64];
static int fail_armed;      /* 1: waiting for fail_after, 2: the next fail_name fails */
static int largest_cluster = 16;

int fake_calls(void) { return log_n; }
const char *fake_call(int i) { return log_name[i]; }
size_t fake_value(int i) { return log_value[i]; }
void fake_fail(const char *name, const char *after) {
    snprintf(fail_name, sizeof(fail_name), "%s", name);
    snprintf(fail_after, sizeof(fail_after), "%s", after);
    fail_armed = 1;
}
void fake_largest_cluster(int n) { largest_cluster = n; }

static cudaError_t call(const char *name, size_t value) {
    if (log_n < MAX_LOG) {
        log_name[log_n] = name;
        log_value[log_n++] = value;
    }
    if (fail_armed == 2 && strcmp(name, fail_name) == 0) {
        fail_armed = 0;
        return cudaErrorLaunchOutOfResources;
    }
    if (fail_armed == 1 && strcmp(name, fail_after) == 0) fail_armed = 2;
    return cudaSuccess;
}
#define CALL(value) call(__func__, value)

static cudaError_t take(const char *name, void **p, size_t n) {
    const cudaError_t e = call(name, n);
    if (e == cudaSuccess) *p = aligned_alloc(256, (n + 255) / 256 * 256);
    if (e == cudaSuccess) memset(*p, 0, (n + 255) / 256 * 256);
    return e;
}
cudaError_t cudaMalloc(void **p, size_t n) { return take(__func__, p, n); }
cudaError_t cudaHostAlloc(void **p, size_t n, unsigned flags) { return take(__func__, p, n); }
cudaError_t cudaFree(void *p) { free(p); return cudaSuccess; }
cudaError_t cudaFreeHost(void *p) { free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void *d, const void *s, size_t n, enum cudaMemcpyKind k) {
    memcpy(d, s, n);
    return CALL(n);
}
cudaError_t cudaMemcpyAsync(void *d, const void *s, size_t n, enum cudaMemcpyKind k, cudaStream_t t) {
    memcpy(d, s, n);
    return CALL(n);
}
cudaError_t cudaMemcpy2D(void *d, size_t dp, const void *s, size_t sp, size_t w, size_t h, enum cudaMemcpyKind k) {
    return CALL(w * h);
}
cudaError_t cudaMemcpy2DAsync(void *d, size_t dp, const void *s, size_t sp, size_t w, size_t h, enum cudaMemcpyKind k,
                              cudaStream_t t) {
    return CALL(w * h);
}
cudaError_t cudaMemset(void *d, int v, size_t n) { memset(d, v, n); return CALL(n); }
cudaError_t cudaMemsetAsync(void *d, int v, size_t n, cudaStream_t t) { memset(d, v, n); return CALL(n); }
cudaError_t cudaDeviceGetAttribute(int *v, enum cudaDeviceAttr a, int dev) {
    *v = a == cudaDevAttrMultiProcessorCount ? 148 : 232448;
    return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize(void) { return CALL(0); }
cudaError_t cudaGetDevice(int *dev) { *dev = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int dev) { return CALL((size_t)dev); }
cudaError_t cudaEventCreate(cudaEvent_t *e) { *e = (cudaEvent_t)1; return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t *e, unsigned f) { *e = (cudaEvent_t)1; return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t e) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float *ms, cudaEvent_t a, cudaEvent_t b) { *ms = 1.f; return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { return CALL(0); }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t *s, unsigned f) { *s = (cudaStream_t)2; return cudaSuccess; }
cudaError_t cudaStreamDestroy(cudaStream_t s) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return CALL(0); }
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned f) { return cudaSuccess; }
cudaError_t cudaStreamBeginCapture(cudaStream_t s, enum cudaStreamCaptureMode m) { return CALL(0); }
cudaError_t cudaStreamEndCapture(cudaStream_t s, cudaGraph_t *g) { *g = (cudaGraph_t)3; return CALL(0); }
cudaError_t cudaGraphInstantiate(cudaGraphExec_t *x, cudaGraph_t g, unsigned long long f) {
    *x = (cudaGraphExec_t)4;
    return CALL(0);
}
cudaError_t cudaGraphLaunch(cudaGraphExec_t x, cudaStream_t s) { return CALL(0); }
cudaError_t cudaGraphDestroy(cudaGraph_t g) { return cudaSuccess; }
cudaError_t cudaGraphExecDestroy(cudaGraphExec_t x) { return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
const char *cudaGetErrorString(cudaError_t e) { return e == cudaSuccess ? "no error" : "made by the test"; }
cudaError_t cudaFuncGetAttributes(struct cudaFuncAttributes *a, const void *f) {
    memset(a, 0, sizeof(*a));
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void *f, enum cudaFuncAttribute a, int v) { return cudaSuccess; }
cudaError_t cudaGetSymbolAddress(void **p, const void *s) { return take(__func__, p, 1 << 20); }
cudaError_t cudaGetDriverEntryPoint(const char *n, void **p, unsigned long long f, enum cudaDriverEntryPointQueryResult *q) {
    return cudaErrorNotSupported;
}
static int cluster(const cudaLaunchConfig_t *c) {
    for (unsigned i = 0; i < c->numAttrs; ++i)
        if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) return (int)c->attrs[i].val.clusterDim.x;
    return 1;
}
cudaError_t cudaOccupancyMaxActiveClusters(int *n, const void *f, const cudaLaunchConfig_t *c) {
    *n = cluster(c) <= largest_cluster ? 4 : 0;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t smem, cudaStream_t s) { return CALL(1); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *c, const void *f, void **args) {
    const cudaError_t e = CALL((size_t)cluster(c));
    return e == cudaSuccess && cluster(c) > largest_cluster ? cudaErrorInvalidConfiguration : e;
}
