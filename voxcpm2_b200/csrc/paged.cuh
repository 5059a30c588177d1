// What the paged KV cache operators (pages.cu, qk_rows.cu, sparse_attn.cu) share: the C entries'
// error mapping and argument checks, and the device view of a cache.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <new>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/voxcpm2_cuda.h"
#include "common.cuh"

void vxc_internal_set_error(const char* msg);

namespace vxc {

struct PagedOom : std::runtime_error {
    using std::runtime_error::runtime_error;
};

inline void paged_ck(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return;
    cudaGetLastError();
    if (e == cudaErrorMemoryAllocation) throw PagedOom(std::string(what) + ": " + cudaGetErrorString(e));
    throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

inline void paged_require(bool ok, const char* msg) {
    if (!ok) throw std::invalid_argument(msg);
}

// Exceptions -> status codes; nothing is thrown through the C ABI.
template <typename F>
int32_t paged_guard(F&& f) noexcept {
    try {
        f();
        return VXC_STATUS_OK;
    } catch (const std::invalid_argument& e) {
        vxc_internal_set_error(e.what());
        return VXC_STATUS_INVALID_ARGUMENT;
    } catch (const PagedOom& e) {
        vxc_internal_set_error(e.what());
        return VXC_STATUS_OUT_OF_MEMORY;
    } catch (const std::bad_alloc&) {
        vxc_internal_set_error("native allocation failed");
        return VXC_STATUS_OUT_OF_MEMORY;
    } catch (const std::exception& e) {
        vxc_internal_set_error(e.what());
        return VXC_STATUS_RUNTIME_ERROR;
    } catch (...) {
        vxc_internal_set_error("unknown native exception");
        return VXC_STATUS_RUNTIME_ERROR;
    }
}

constexpr int kMaxPool = 1 << 20;
constexpr int kMaxSeqs = 4096;
constexpr int kMaxSeqPages = 16384;
constexpr int kMaxKvHeads = 256;

inline int dtype_size(int dtype) { return dtype == VXC_F32 ? 4 : 2; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Sizes of a cache (no pointer is looked at).
inline void check_page_sizes(const vxc_pages* p) {
    paged_require(p != nullptr, "null argument");
    paged_require(p->dtype == VXC_F32 || p->dtype == VXC_F16 || p->dtype == VXC_BF16, "pages: dtype must be f32, f16 or bf16");
    paged_require(p->layers > 0 && p->layers <= 65536, "pages: layers must be 1 to 65536");
    paged_require(p->n_pages > 0 && p->n_pages <= kMaxPool, "pages: n_pages must be 1 to 2^20");
    paged_require(p->kv_heads > 0 && p->kv_heads <= kMaxKvHeads, "pages: kv_heads must be 1 to 256");
    paged_require(p->page_size == 16 || p->page_size == 32 || p->page_size == 64 || p->page_size == 128,
                  "pages: page_size must be 16, 32, 64 or 128");
    paged_require(p->head_dim == 64 || p->head_dim == 128, "pages: head_dim must be 64 or 128");
    paged_require(p->n_seqs > 0 && p->n_seqs <= kMaxSeqs, "pages: n_seqs must be 1 to 4096");
    paged_require(p->max_pages > 0 && p->max_pages <= kMaxSeqPages, "pages: max_pages must be 1 to 16384");
}

// Refuses arrays that are not memory of the current device: a kernel would fault on them. Arrays of one
// allocation (an allocator's small ones) are asked about once. A question takes 0.05 us; the host time of whole calls
// from Python (4 to 12 us each) is the same with and without.
class DeviceMemory {
public:
    explicit DeviceMemory(const char* call) : call_(call) { paged_ck(cudaGetDevice(&dev_), "cudaGetDevice"); }
    // null: an optional array that the call goes without
    void require(const void* ptr, const char* name) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(ptr);
        if (!ptr) return;
        for (int i = 0; i < kKept; ++i)
            if (at - start_[i] < size_[i]) return;
        unsigned type = 0;
        int dev = -1, managed = 0;
        CUdeviceptr start = 0;
        size_t size = 0;
        CUpointer_attribute what[] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                      CU_POINTER_ATTRIBUTE_IS_MANAGED, CU_POINTER_ATTRIBUTE_RANGE_START_ADDR,
                                      CU_POINTER_ATTRIBUTE_RANGE_SIZE};
        void* to[] = {&type, &dev, &managed, &start, &size};
        if (query()(5, what, to, static_cast<CUdeviceptr>(at)) != CUDA_SUCCESS)
            throw std::runtime_error(std::string(call_) + ": the driver does not know " + name);
        if (!managed && !(type == CU_MEMORYTYPE_DEVICE && dev == dev_))
            throw std::invalid_argument(std::string(call_) + ": " + name + " is not memory of the current device");
        start_[next_] = start;
        size_[next_] = size;
        next_ = (next_ + 1) % kKept;
    }

private:
    using Query = CUresult (*)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
    static Query query() {
        static const Query fn = [] {
            void* f = nullptr;
            cudaDriverEntryPointQueryResult q;
            paged_ck(cudaGetDriverEntryPointByVersion("cuPointerGetAttributes", &f, 12000, cudaEnableDefault, &q),
                     "cuPointerGetAttributes");
            if (q != cudaDriverEntryPointSuccess || !f) throw std::runtime_error("cuPointerGetAttributes is not there");
            return reinterpret_cast<Query>(f);
        }();
        return fn;
    }
    static constexpr int kKept = 4;
    const char* call_;
    int dev_ = 0, next_ = 0;
    uintptr_t start_[kKept] = {};
    size_t size_[kKept] = {};
};

inline void check_page_arrays(const vxc_pages* p) {
    check_page_sizes(p);
    paged_require(p->k && p->v && p->bounds && p->table && p->lens && p->refs && p->status && p->work,
                  "pages: null array");
    paged_require(aligned32(p->k) && aligned32(p->v) && aligned16(p->bounds) && aligned16(p->refs) && aligned16(p->work),
                  "pages: k and v must start on 32-byte, bounds, refs and work on 16-byte boundaries");
    paged_require(aligned4(p->table) && aligned4(p->lens) && aligned4(p->status), "pages: misaligned int32 array");
}
// After all other checks of a call.
inline void check_page_memory(const vxc_pages* p, DeviceMemory& mem) {
    mem.require(p->k, "pages.k");
    mem.require(p->v, "pages.v");
    mem.require(p->bounds, "pages.bounds");
    mem.require(p->table, "pages.table");
    mem.require(p->lens, "pages.lens");
    mem.require(p->refs, "pages.refs");
    mem.require(p->status, "pages.status");
    mem.require(p->work, "pages.work");
}

// Lets a kernel take the dynamic shared memory that a launch asks for. Always up to the same limit, so that
// calls at the same time do not take it from one another between this and their launches.
constexpr int kDynamicLimit = 232448 - 8192;  // an SM's 227 KB less what the kernels hold statically
inline void allow_dynamic_smem(const void* kernel, size_t need, const char* what) {
    if (need <= 40 * 1024) return;
    paged_require(need <= kDynamicLimit, "shared memory of the call exceeds an SM's");
    paged_ck(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDynamicLimit), what);
}

// Launch with programmatic dependent launch: every kernel of these operators waits
// (pdl_wait) before it touches memory, so its launch overlaps the tail of the one before.
template <typename... KArgs, typename... Args>
void paged_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, const char* what,
                  Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    paged_ck(cudaLaunchKernelEx(&cfg, kernel, KArgs(std::forward<Args>(args))...), what);
}

// The first code reported stays.
__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, 0, code); }

}  // namespace vxc
