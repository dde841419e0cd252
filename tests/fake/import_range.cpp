// import_refusal with stand-ins of the driver's entry point: one allocation [0x10000, 0x10000 + 4096), and a call that fails.
#include <string.h>

#include "../../zyx_b200/csrc/import_range.h"

static CUresult one_allocation(CUdeviceptr* base, size_t* size, CUdeviceptr at) {
  if (at < 0x10000 || at >= 0x11000) return CUDA_ERROR_NOT_FOUND;
  *base = 0x10000; *size = 4096;
  return CUDA_SUCCESS;
}
static CUresult fails(CUdeviceptr*, size_t*, CUdeviceptr) { return CUDA_ERROR_INVALID_VALUE; }

// entry: 0 none, 1 the allocation, 2 the call that fails
extern "C" const char* refusal(int entry, uint64_t at, uint64_t bytes) {
  return zyxb::import_refusal(entry == 0 ? nullptr : entry == 1 ? (void*)one_allocation : (void*)fails, at, bytes);
}
