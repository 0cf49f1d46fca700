// The runtime calls of one object of the library, without a device: they answer as they are told to and note what is launched.
#include <cuda_runtime_api.h>

static int g_large = 1, g_clusters = 4, g_launches = 0, g_cluster[16];

extern "C" {
void fake_set(int large, int clusters) { g_large = large, g_clusters = clusters, g_launches = 0; }
int fake_launches() { return g_launches; }
int fake_cluster(int i) { return g_cluster[i]; }

cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute attr, int) {
  return attr == cudaFuncAttributeNonPortableClusterSizeAllowed && !g_large ? cudaErrorNotSupported : cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t*) {
  *n = g_clusters;
  return g_clusters < 0 ? cudaErrorInvalidClusterSize : cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void*, void**) {
  int size = 1;
  for (unsigned i = 0; i < c->numAttrs; ++i)
    if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) size = static_cast<int>(c->attrs[i].val.clusterDim.x);
  if (size > 8 && (!g_large || g_clusters < 1)) return cudaErrorInvalidClusterSize;
  g_cluster[g_launches++ % 16] = size;
  return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { return *v = 148, cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t cudaMemcpyFromSymbolAsync(void*, const void*, size_t, size_t, cudaMemcpyKind, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t cudaMemcpyToSymbolAsync(const void*, const void*, size_t, size_t, cudaMemcpyKind, cudaStream_t) { return cudaErrorUnknown; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaErrorUnknown; }
void** __cudaRegisterFatBinary(void*) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
unsigned __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return 1; }
}
