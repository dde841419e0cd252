// Sends RMS norm launches of many widths and row counts through the library's own dispatch in a process without a GPU, where a launch
// that is accepted ends in the driver's "no device" error, and prints those that end in any other.
//   rms_dispatch ROWS...
#include <stdio.h>
#include <stdlib.h>

#include <string>
#include <vector>

#include "../../zyx_b200/csrc/internal.h"

using namespace zyxb;

int main(int argc, char** argv) {
  std::vector<uint64_t> bytes(8, 1ull << 60);
  std::vector<void*> ptrs;
  for (int i = 0; i < 8; ++i) ptrs.push_back((void*)((uintptr_t)(i + 1) << 24));
  uint64_t launches = 0, tried = 0;
  LaunchCtx lc{};
  lc.sm_count = 148; lc.scratch_bytes = 320ull << 20; lc.launch_counter = &launches;
  cudaGetLastError();
  const std::string no_device[] = {cudaGetErrorString(cudaErrorNoDevice), cudaGetErrorString(cudaErrorInsufficientDriver)};
  auto look = [&](const zyxb_rmsnorm_desc& d, bool backward, int st, const std::string& err) {
    ++tried;
    for (const std::string& text : no_device)
      if (st == ZYXB_ERR_KERNEL_LAUNCH && err.size() >= text.size() && err.compare(err.size() - text.size(), text.size(), text) == 0) return;
    printf("%s dtype %d rows %llu cols %llu quant %d: %d %s\n", backward ? "backward" : "forward", d.dtype, (unsigned long long)d.rows,
           (unsigned long long)d.cols, d.quant, st, err.c_str());
  };
  for (int i = 1; i < argc; ++i)
    for (uint64_t cols = 1; cols <= 16384; ++cols)
      for (int dtype : {ZYXB_F32, ZYXB_BF16}) {
        zyxb_rmsnorm_desc d{};
        std::string err;
        d.dtype = dtype; d.rows = strtoull(argv[i], nullptr, 10); d.cols = cols; d.eps = 1e-6f;
        d.has_weight = 1;
        look(d, true, launch_rmsnorm_bwd(d, ptrs.data(), bytes.data(), 5, lc, err), err);
        d.has_weight = 0;
        for (int residual = 0; residual < 2; ++residual) {
          d.has_residual = residual;
          err.clear();
          look(d, false, launch_rmsnorm(d, ptrs.data(), bytes.data(), residual ? 4 : 2, lc, err), err);
        }
      }
  fprintf(stderr, "%llu launches\n", (unsigned long long)tried);
  return 0;
}
