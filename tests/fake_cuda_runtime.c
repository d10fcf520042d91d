/* A CUDA runtime with a device of 148 SMs and no GPU behind it, preloaded
 * before the library under test: launches are written down instead of made.
 * FAKE_CTAS_AN_SM=footprint: the occupancy calls count as many CTAs an SM as
 * its shared memory holds; otherwise one, whatever they take, as driver
 * 580.159 does for these kernels. */
#include <cuda_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static struct { const void* fn; const char* name; int smem; } kernels[1024];
static int n_kernels;
static char text[1 << 16];
static size_t used;

const char* fake_launches(void) { return text; }
void fake_forget(void) { text[used = 0] = 0; }

static int find(const void* fn) {
    for (int i = 0; i < n_kernels; ++i)
        if (kernels[i].fn == fn) return i;
    return -1;
}

void** __cudaRegisterFatBinary(void* bin) { static void* handle; (void)bin; return &handle; }
void __cudaRegisterFatBinaryEnd(void** h) { (void)h; }
void __cudaUnregisterFatBinary(void** h) { (void)h; }
void __cudaRegisterFunction(void** h, const char* host, char* dev, const char* name, int limit, uint3* tid, uint3* bid,
                            dim3* bd, dim3* gd, int* w) {
    (void)h, (void)dev, (void)limit, (void)tid, (void)bid, (void)bd, (void)gd, (void)w;
    if (n_kernels < 1024) kernels[n_kernels].fn = host, kernels[n_kernels++].name = name;
}

cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, enum cudaDeviceAttr a, int d) {
    (void)d;
    if (a != cudaDevAttrMultiProcessorCount) return cudaErrorInvalidValue;
    *v = 148;
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* fn, enum cudaFuncAttribute a, int v) {
    const int i = find(fn);
    if (i < 0 || a != cudaFuncAttributeMaxDynamicSharedMemorySize || v > 227 * 1024) return cudaErrorInvalidValue;
    kernels[i].smem = v;
    return cudaSuccess;
}

static int ctas_an_sm(size_t smem) {
    const char* how = getenv("FAKE_CTAS_AN_SM");
    return how && !strcmp(how, "footprint") ? (int)(228 * 1024 / (smem + 1024)) : 1;
}

cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void* fn, int threads, size_t smem, unsigned flags) {
    (void)threads, (void)flags;
    const int i = find(fn);
    if (i < 0 || smem > (size_t)kernels[i].smem) return cudaErrorInvalidValue;
    *n = ctas_an_sm(smem);
    return cudaSuccess;
}

cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* fn, const cudaLaunchConfig_t* c) {
    static const int clusters[] = {0, 148, 74, 45, 33, 26, 22, 15, 15}; /* as a B200 has them */
    const int i = find(fn);
    if (i < 0 || c->dynamicSmemBytes > (size_t)kernels[i].smem) return cudaErrorInvalidValue;
    if (c->attrs[0].val.clusterDim.x > 8) return cudaErrorInvalidValue;
    *n = ctas_an_sm(c->dynamicSmemBytes) * clusters[c->attrs[0].val.clusterDim.x];
    return cudaSuccess;
}

cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* fn, void** args) {
    (void)args;
    const int i = find(fn);
    if (i < 0 || c->dynamicSmemBytes > (size_t)kernels[i].smem) return cudaErrorInvalidValue;
    if (c->gridDim.x > 2147483647u || c->gridDim.y > 65535u || c->gridDim.z > 65535u) return cudaErrorInvalidConfiguration;
    unsigned cluster = 0;
    for (unsigned j = 0; j < c->numAttrs; ++j)
        if (c->attrs[j].id == cudaLaunchAttributeClusterDimension) cluster = c->attrs[j].val.clusterDim.x;
    if (!cluster || c->gridDim.x % cluster) return cudaErrorInvalidConfiguration;
    used += (size_t)snprintf(text + used, sizeof text - used, "%s %u %u %u\n", kernels[i].name, c->gridDim.x, c->gridDim.y, cluster);
    return cudaSuccess;
}

/* cuTensorMapEncodeTiled, its documented limits on what these maps use checked */
static int encode(void* map, int type, unsigned rank, void* at, const unsigned long long* dims, const unsigned long long* strides,
                  const unsigned* box, const unsigned* es, int interleave, int swizzle, int promotion, int fill) {
    (void)type, (void)interleave, (void)swizzle, (void)promotion, (void)fill;
    if ((size_t)at % 16) return 1;
    for (unsigned i = 0; i < rank; ++i)
        if (!dims[i] || dims[i] > 1ull << 32 || !box[i] || box[i] > 256 || es[i] != 1) return 1;
    for (unsigned i = 0; i + 1 < rank; ++i)
        if (strides[i] % 16 || strides[i] >= 1ull << 40) return 1;
    memset(map, 0, 128);
    memcpy(map, &at, sizeof at); /* not all zeros, as no map is */
    return 0;
}

cudaError_t cudaGetDriverEntryPointByVersion(const char* name, void** fn, unsigned version, unsigned long long flags,
                                             enum cudaDriverEntryPointQueryResult* q) {
    (void)version, (void)flags;
    if (strcmp(name, "cuTensorMapEncodeTiled")) return cudaErrorInvalidValue;
    *fn = (void*)encode;
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
