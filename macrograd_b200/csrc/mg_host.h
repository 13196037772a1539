// mg_host.h -- what the library's translation units share on the host side:
// errors, the device's state, scratch memory, launch counting and the tensor-map
// encoder. Defined in mg_gemm.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <cstddef>
#include <cstdint>

#include "mg_gemm.h"

namespace mg {
namespace host {

// Sets this thread's mg_last_error() and returns `s`.
mg_status fail(mg_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

struct Device {
    int ordinal = 0;
    int sm_count = 0;
    int max_smem = 0;
    int* status = nullptr;         // {status, detail} of mg_device_status()
    cudaMemPool_t pool = nullptr;
};

// State of the current device (MG_ERR_UNSUPPORTED if it is not sm_100).
mg_status device(Device* out);

void count_launch();

// Per-call scratch: from the registered allocator or the library's pool,
// given back stream-ordered when the call ends.
class Scratch {
public:
    Scratch(const Device& dev, void* stream) : pool_(dev.pool), stream_(stream) {}
    ~Scratch();
    Scratch(const Scratch&) = delete;
    Scratch& operator=(const Scratch&) = delete;
    void* get(size_t bytes);

private:
    cudaMemPool_t pool_;
    void* stream_;
    void* ptrs_[8];
    int n_ = 0;
};

// cuTensorMapEncodeTiled of a 16-bit matrix stack: dims[rank] innermost first,
// strides[rank - 1] in bytes, 128-byte swizzle.
mg_status encode_bf16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                      const uint32_t* box);

struct Range {
    explicit Range(const char* name) { nvtxRangePushA(name); }
    ~Range() { nvtxRangePop(); }
    Range(const Range&) = delete;
    Range& operator=(const Range&) = delete;
};

}  // namespace host
}  // namespace mg

#define MG_HOST_TRY(call)                                                                       \
    do {                                                                                        \
        cudaError_t e_ = (call);                                                                \
        if (e_ != cudaSuccess)                                                                  \
            return mg::host::fail(MG_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_)); \
    } while (0)
