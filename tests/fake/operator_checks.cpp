// The argument checks of the embedding, RMS norm and Muon programs without a device: validation, then the launcher's own checks,
// which come before its first CUDA call.  Loaded by tests/fake/operator_checks.py in a process that sees no GPU, so that arguments
// which pass all checks end in a launch error and never reach one.
#include <string.h>

#include "../../zyx_b200/csrc/internal.h"

using namespace zyxb;

extern "C" __attribute__((visibility("default"))) int32_t check_operator(const zyxb_kernel_desc* d, void* const* args, const uint64_t* bytes, int32_t n_args,
                                                                         char* text, int32_t size) {
  std::string err;
  int st = ZYXB_OK;
  switch (d->kind) {
    case ZYXB_KIND_EMBEDDING: case ZYXB_KIND_EMBEDDING_BWD: st = validate_embedding(d->u.embedding, d->kind == ZYXB_KIND_EMBEDDING_BWD, err); break;
    case ZYXB_KIND_RMSNORM: case ZYXB_KIND_RMSNORM_BWD: st = validate_rmsnorm(d->u.rmsnorm, d->kind == ZYXB_KIND_RMSNORM_BWD, err); break;
    default: st = validate_muon(d->u.muon, err);
  }
  uint64_t launches = 0;
  LaunchCtx lc{};
  lc.sm_count = 148; lc.scratch_bytes = 320ull << 20; lc.launch_counter = &launches;
  if (st == ZYXB_OK && n_args >= 0) {
    switch (d->kind) {
      case ZYXB_KIND_EMBEDDING: st = launch_embedding(d->u.embedding, args, bytes, n_args, lc, err); break;
      case ZYXB_KIND_EMBEDDING_BWD: st = launch_embedding_bwd(d->u.embedding, args, bytes, n_args, lc, err); break;
      case ZYXB_KIND_RMSNORM: st = launch_rmsnorm(d->u.rmsnorm, args, bytes, n_args, lc, err); break;
      case ZYXB_KIND_RMSNORM_BWD: st = launch_rmsnorm_bwd(d->u.rmsnorm, args, bytes, n_args, lc, err); break;
      default: st = launch_muon(d->u.muon, d->u.muon.rows, d->u.muon.cols, nullptr, args, bytes, n_args, lc, err);
    }
  }
  strncpy(text, err.c_str(), (size_t)size - 1);
  text[size - 1] = 0;
  return st;
}
