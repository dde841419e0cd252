// Whether a range of device memory lies inside the allocation its first byte belongs to: what zyxb_buffer_import asks of the CUDA
// driver's cuMemGetAddressRange before it hands out an id, so that no program reads or writes behind the allocation.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace zyxb {

// nullptr, or why the range cannot be used.  address_range: the driver's entry point; without it nothing is known of the allocation.
inline const char* import_refusal(void* address_range, uint64_t at, uint64_t bytes) {
  if (!address_range) return "the CUDA driver offers no cuMemGetAddressRange to check the range with";
  CUdeviceptr base = 0;
  size_t size = 0;
  if (reinterpret_cast<CUresult (*)(CUdeviceptr*, size_t*, CUdeviceptr)>(address_range)(&base, &size, (CUdeviceptr)at) != CUDA_SUCCESS || at < base)
    return "range exceeds the allocation";
  const uint64_t offset = at - base;
  return offset <= size && bytes <= size - offset ? nullptr : "range exceeds the allocation";
}

}  // namespace zyxb
