// A stand-in for the CUDA runtime: linked with the library's own objects it lets the host side of the decode-step entry
// points run where there is no GPU.  It places nothing and runs nothing; it keeps a list of what was asked and refuses the
// requests it is told to refuse.
#include <cuda_runtime_api.h>

#include <cstdio>
#include <cstring>
#include <map>
#include <string>

#define EXPORT extern "C" __attribute__((visibility("default")))

namespace {
std::map<const void *, std::string> &Names() {  // host function -> mangled kernel name; filled before main()
    static std::map<const void *, std::string> names;
    return names;
}
std::string asked;  // one line per attribute and launch
int device = 0, largest_cluster = 16, refuse_launch = -1, refuse_attribute = -1, launches = 0, attributes = 0;
cudaError_t last = cudaSuccess;

cudaError_t Fail(cudaError_t e) { return last = e; }

cudaError_t Launch(const void *func, unsigned grid, size_t smem, int cluster) {
    char line[512];
    std::snprintf(line, sizeof line, "launch %s grid=%u smem=%zu cluster=%d\n", Names()[func].c_str(), grid, smem, cluster);
    asked += line;
    return launches++ == refuse_launch ? Fail(cudaErrorInvalidConfiguration) : cudaSuccess;
}
}  // namespace

// What the tests say and ask.  A new device forgets what the library remembers per device.
EXPORT void fake_begin(int new_device, int cluster, int launch, int attribute) {
    device = new_device;
    largest_cluster = cluster;
    refuse_launch = launch;
    refuse_attribute = attribute;
    launches = attributes = 0;
    asked.clear();
    last = cudaSuccess;
}
EXPORT const char *fake_asked() { return asked.c_str(); }

extern "C" {
void **__cudaRegisterFatBinary(void *) {
    static void *handle;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *host, char *, const char *name, int, void *, void *, void *, void *, int *) {
    Names()[host] = name;
}

static dim3 pushed_grid;
static size_t pushed_smem;
unsigned __cudaPushCallConfiguration(dim3 grid, dim3, size_t smem, void *) {
    pushed_grid = grid;
    pushed_smem = smem;
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3 *grid, dim3 *, size_t *smem, void *) {
    *grid = pushed_grid;
    *smem = pushed_smem;
    return cudaSuccess;
}

cudaError_t cudaGetDevice(int *d) {
    *d = device;
    return cudaSuccess;
}
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaMemGetInfo(size_t *, size_t *) { return cudaErrorNotSupported; }
cudaError_t cudaGetDeviceProperties(cudaDeviceProp *prop, int) {  // the header maps the name to the one with its version
    std::memset(prop, 0, sizeof *prop);
    prop->multiProcessorCount = 148;
    prop->l2CacheSize = 126 << 20;
    return cudaSuccess;
}
cudaError_t cudaGetLastError() {
    const cudaError_t e = last;
    last = cudaSuccess;
    return e;
}
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute attribute, int) {
    asked += attribute == cudaFuncAttributeNonPortableClusterSizeAllowed ? "attribute cluster\n" : "attribute smem\n";
    return attributes++ == refuse_attribute ? Fail(cudaErrorInvalidValue) : cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveClusters(int *n, const void *, const cudaLaunchConfig_t *cfg) {
    *n = static_cast<int>(cfg->attrs[0].val.clusterDim.x) <= largest_cluster ? 1 : 0;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void *func, dim3 grid, dim3, void **, size_t smem, cudaStream_t) {
    return Launch(func, grid.x, smem, 1);
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *cfg, const void *func, void **) {
    int cluster = 1;
    for (unsigned i = 0; i < cfg->numAttrs; ++i) {
        if (cfg->attrs[i].id == cudaLaunchAttributeClusterDimension) cluster = static_cast<int>(cfg->attrs[i].val.clusterDim.x);
    }
    return Launch(func, cfg->gridDim.x, cfg->dynamicSmemBytes, cluster);
}
}
