// The CUDA runtime calls that runtime.cu makes, over host memory and two devices that
// are not there, so that its host logic can be tested without a GPU.
#include <cuda_runtime.h>
#include <stdlib.h>
#include <string.h>

namespace {
thread_local int current = 0;
constexpr int kDevices = 2;
// As the runtime does: a call that fails leaves its error for cudaGetLastError.
thread_local cudaError_t last = cudaSuccess;
cudaError_t fail(cudaError_t e) { return last = e; }
}  // namespace

extern "C" {

cudaError_t cudaGetDeviceCount(int* n) { return *n = kDevices, cudaSuccess; }
cudaError_t cudaSetDevice(int id) {
    if (id < 0 || id >= kDevices) return fail(cudaErrorInvalidDevice);
    return current = id, cudaSuccess;
}
cudaError_t cudaGetDevice(int* id) { return *id = current, cudaSuccess; }
cudaError_t cudaGetDeviceProperties(cudaDeviceProp* p, int) {
    memset(p, 0, sizeof *p);
    p->multiProcessorCount = 148;
    return cudaSuccess;
}
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { return *p = malloc(n), cudaSuccess; }
cudaError_t cudaMallocHost(void** p, size_t n) { return *p = malloc(n), cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { return free(p), cudaSuccess; }
cudaError_t cudaMallocAsync(void** p, size_t n, cudaStream_t) {
    if (n >= (size_t)1 << 37) return fail(cudaErrorMemoryAllocation);
    return *p = malloc(n), cudaSuccess;
}
cudaError_t cudaFreeAsync(void* p, cudaStream_t) { return free(p), cudaSuccess; }
cudaError_t cudaFree(void* p) { return free(p), cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) {
    return memcpy(d, s, n), cudaSuccess;
}
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void*) {
    return memset(a, 0, sizeof *a), cudaSuccess;
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) {
    return *s = (cudaStream_t)malloc(8), cudaSuccess;
}
cudaError_t cudaStreamDestroy(cudaStream_t s) { return free(s), cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
    return *s = cudaStreamCaptureStatusNone, cudaSuccess;
}
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return *e = nullptr, cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaDeviceGetDefaultMemPool(cudaMemPool_t* p, int) { return *p = nullptr, cudaSuccess; }
cudaError_t cudaMemPoolSetAttribute(cudaMemPool_t, cudaMemPoolAttr, void*) { return cudaSuccess; }
cudaError_t cudaMemPoolTrimTo(cudaMemPool_t, size_t) { return cudaSuccess; }
cudaError_t cudaGetLastError(void) {
    const cudaError_t e = last;
    return last = cudaSuccess, e;
}
const char* cudaGetErrorString(cudaError_t) { return "fake"; }

}  // extern "C"
