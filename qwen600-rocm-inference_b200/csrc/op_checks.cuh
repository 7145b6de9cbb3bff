// op_checks.cuh — what the entry points of the operators on caller-owned memory
// share: failures as status codes, checks of pointers, facts about the device.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <initializer_list>
#include <string>

#include "../../include/qwen_b200.h"

int qwen_internal_fail(int code, const std::string& msg);

namespace {

int fail(int code, const std::string& msg) { return qwen_internal_fail(code, msg); }
#define CU(call)                                                                                        \
    do {                                                                                                \
        cudaError_t e_ = (call);                                                                        \
        if (e_ != cudaSuccess) return fail(QWEN_E_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
    } while (0)
#define TRY(call)                          \
    do {                                   \
        int rc_ = (call);                  \
        if (rc_ != QWEN_OK) return rc_;    \
    } while (0)

struct Ptr {
    const void* p;
    const char* name;
    size_t align;
    bool used;   // false: may be anything
};
// NULL and alignment (no GPU needed).
int check_places(std::initializer_list<Ptr> ptrs) {
    for (const Ptr& a : ptrs) {
        if (!a.used) continue;
        if (!a.p) return fail(QWEN_E_ARG, std::string(a.name) + " is NULL");
        if ((uintptr_t)a.p % a.align) return fail(QWEN_E_ARG, std::string(a.name) + " must be " + std::to_string(a.align) + "-byte aligned");
    }
    return QWEN_OK;
}
// These first, then: device memory of the current device, *dev.
int check_ptrs(std::initializer_list<Ptr> ptrs, int* dev) {
    TRY(check_places(ptrs));
    CU(cudaGetDevice(dev));
    for (const Ptr& a : ptrs) {
        if (!a.used) continue;
        cudaPointerAttributes at;
        const cudaError_t e = cudaPointerGetAttributes(&at, a.p);
        if (e != cudaSuccess) cudaGetLastError();   // not left behind for the caller's next query
        if (e != cudaSuccess || (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged))
            return fail(QWEN_E_ARG, std::string(a.name) + " is not device memory");
        if (at.type == cudaMemoryTypeDevice && at.device != *dev)
            return fail(QWEN_E_ARG, std::string(a.name) + " lies on another device than the current one");
    }
    return QWEN_OK;
}
bool is16(int t) { return t == QWEN_BF16 || t == QWEN_FP16; }
bool is8(int t) { return t == QWEN_E4M3 || t == QWEN_INT8; }

int sm_count(int dev, int* n) {
    static std::atomic<int> known[64];
    if (dev < 0 || dev >= 64) return fail(QWEN_E_ARG, "device index beyond 63");
    int v = known[dev].load();
    if (!v) {
        CU(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
        known[dev].store(v);
    }
    *n = v;
    return QWEN_OK;
}
// Sets a kernel's shared-memory limit once per device (not a stream operation: allowed during capture).
template <typename K>
int smem_limit(K kernel, std::atomic<uint64_t>& done, int dev, int bytes) {
    if (!((done.load() >> dev) & 1)) {
        CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(1ull << dev);
    }
    return QWEN_OK;
}

}  // namespace
