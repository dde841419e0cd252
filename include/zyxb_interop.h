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
 * streams know nothing of the owner's: synchronise with the owner's stream before a launch, and with this device (zyxb_sync /
 * zyxb_device_sync) before the owner reads what a launch wrote. */
int32_t zyxb_buffer_import(zyxb_ctx* ctx, int32_t dev, void* device_ptr, uint64_t bytes, uint32_t* out_buf);

#ifdef __cplusplus
}
#endif
#endif /* ZYXB_INTEROP_H */
