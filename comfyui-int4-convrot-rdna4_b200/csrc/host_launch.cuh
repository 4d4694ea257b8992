// Host-side launch helpers shared by the library's translation units.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace convrot {

bool aligned16(const void* p);
int sm_count();

// cuTensorMapEncodeTiled through the runtime's driver entry point; null when
// the driver does not provide it.
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

// Launch with programmatic stream serialization: the kernel may start its
// prologue while the previous kernel in the stream drains; every kernel of this
// library calls griddep_wait() before touching memory another kernel wrote.
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                       Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

template <typename KernelT>
cudaError_t ensure_smem(KernelT kernel, int bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace convrot
