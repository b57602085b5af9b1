// Host helpers shared by the translation units of libctct_b200.so: launches, error text, sizes.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include <utility>

namespace ctct {

// CTCT_OK, or CTCT_ERR_LAUNCH after recording the text that ctct_b200_strerror returns (ctct_abi.cu)
int check_launch(const char *what);

// Launch with programmatic stream serialisation: the kernel may be set up, and start, while the
// kernel before it in the stream drains; it must call pdl_wait() before touching that kernel's output.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

inline int sm_count() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace ctct
