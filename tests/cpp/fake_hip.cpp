// fake_hip.cpp -- a HIP runtime that runs nothing, for CPU tests of the host
// layer: linked with tmac_attn.cpp instead of libamdhip64.  Device memory is host
// memory, streams are always idle (or capturing, fake_set_capturing), and a launch
// is only written down: fake_launch_name(i) and fake_launch_grid(i, d) give its
// kernel and grid, fake_launch_prefix(i, field) how a prefix kernel's work is cut.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "attn_args.h"

namespace {
struct Launch {
    std::string name;
    unsigned grid[3], block;
    int prefix[3];  // tmac_prefix_*: most runs of a prefix, workgroups that share the units, most blocks of columns
};
std::vector<Launch> g_launches;
std::vector<std::string*> g_names;  // hipFunction_t values
bool g_capturing = false;
char g_handle[8];
}  // namespace

// Code objects and the scratch array: only their existence matters.
extern "C" {
static const unsigned char kBlob[1] = {0};
extern const unsigned char* const tmac_attn_code_objects[5];
extern const uint64_t tmac_attn_code_object_sizes[5];
const unsigned char* const tmac_attn_code_objects[5] = {kBlob, kBlob, kBlob, kBlob, kBlob};
const uint64_t tmac_attn_code_object_sizes[5] = {1, 1, 1, 1, 1};
int tmac_scratch_setup(int, void** ptr) {
    static void* p = std::malloc(16u << 20);
    *ptr = p;
    return 0;
}

int fake_launches() { return (int)g_launches.size(); }
void fake_clear() { g_launches.clear(); }
const char* fake_launch_name(int i) { return g_launches[(size_t)i].name.c_str(); }
unsigned fake_launch_grid(int i, int d) { return g_launches[(size_t)i].grid[d]; }
int fake_launch_prefix(int i, int field) { return g_launches[(size_t)i].prefix[field]; }
unsigned fake_launch_block(int i) { return g_launches[(size_t)i].block; }
void fake_set_capturing(int on) { g_capturing = on != 0; }

hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { *e = (hipEvent_t)g_handle; return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { *ms = 0; return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { return (*p = std::calloc(1, n)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void* p) { std::free(p); return hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset(p, 0, sizeof(*p));
    p->multiProcessorCount = 256;
    std::strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
    return hipSuccess;
}
const char* hipGetErrorString(hipError_t) { return "fake"; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipGraphExecUpdate(hipGraphExec_t, hipGraph_t, hipGraphNode_t*, hipGraphExecUpdateResult*) { return hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t, hipGraphNode_t*, char*, size_t) {
    *e = (hipGraphExec_t)g_handle;
    return hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { return hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { std::memcpy(d, s, n); return hipSuccess; }
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t) { std::memset(d, v, n); return hipSuccess; }
hipError_t hipModuleLoadData(hipModule_t* m, const void*) { *m = (hipModule_t)g_handle; return hipSuccess; }
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
    g_names.push_back(new std::string(name));
    *f = (hipFunction_t)g_names.back();
    return hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned, unsigned,
                                 unsigned, hipStream_t, void** params, void**) {
    Launch l{};
    l.name = *reinterpret_cast<std::string*>(f);
    l.grid[0] = gx;
    l.grid[1] = gy;
    l.grid[2] = gz;
    l.block = bx;
    if (l.name.rfind("tmac_prefix_", 0) == 0) {
        const auto* a = static_cast<const tmac::PagedAttnArgs*>(params[0]);
        l.prefix[0] = a->prefix_splits;
        l.prefix[1] = a->prefix_groups;
        l.prefix[2] = a->prefix_blocks;
    }
    g_launches.push_back(l);
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) { return hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) { *g = (hipGraph_t)g_handle; return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { *s = (hipStream_t)g_handle; return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
}
