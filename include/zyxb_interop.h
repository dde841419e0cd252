/* Device memory shared with other libraries of the process (libzyxb.so).  Apart from zyxb.h because a stand-in of that ABI without a
 * device has nothing to import. */
#ifndef ZYXB_INTEROP_H
#define ZYXB_INTEROP_H
#include "zyxb.h"

#ifdef __cplusplus
extern "C" {
#endif

/* An id for device memory that another library of this process owns (a tensor of it, say): programs then read and write it in
 * place.  device_ptr is 256-byte aligned and [device_ptr, device_ptr + bytes) lies inside one allocation on this device.
 * zyxb_free releases only the id; the owner keeps the memory alive until this library's work on it has finished.  The library's
 * streams know nothing of the owner's: either both use one stream (zyxb_use_stream), or the caller synchronises with the owner's
 * stream before a launch and with this device (zyxb_sync / zyxb_device_sync) before the owner reads what a launch wrote, or gives
 * its memory away. */
int32_t zyxb_buffer_import(zyxb_ctx* ctx, int32_t dev, void* device_ptr, uint64_t bytes, uint32_t* out_buf);

/* The device's kernels, memsets and copies that do not come from the host run on `stream` (a cudaStream_t of this device; NULL is the
 * legacy default stream) instead of the context's own, in order with what others put there before and after: imported memory then needs
 * no synchronisation.  ZYXB_OWN_STREAM goes back.  What was launched before the call stays in front of what is launched after it.  The
 * stream has to live until the context uses another one or is shut down.  Refused between zyxb_capture_begin and zyxb_capture_end, for
 * a stream that is being captured and for the per-thread default stream; the legacy default stream cannot be captured. */
#define ZYXB_OWN_STREAM ((void*)(intptr_t)-1)
int32_t zyxb_use_stream(zyxb_ctx* ctx, int32_t dev, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ZYXB_INTEROP_H */
