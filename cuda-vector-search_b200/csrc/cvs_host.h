// Host helpers of the C ABI's translation units: status and message of a failed
// call, the current device, tensor maps.
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include "cvs.h"

namespace cvs {

struct DeviceInfo {
  int sms = 0;
  int major = 0;
  int minor = 0;
  int* err = nullptr;  // device address of the device error word
};

// Records the message cvs_last_error returns on this thread and passes the status on.
cvs_status fail(cvs_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
cvs_status cuda_fail(cudaError_t e, const char* what);

// The current device; CVS_ERR_UNSUPPORTED unless it is an sm_100 GPU.
cvs_status device_info(DeviceInfo* out, int* dev_out = nullptr);

// Tensor map of a half-precision matrix [rows][cols], rows `stride` elements apart, in
// boxes of 64 columns (one 128-byte swizzled row) x box_rows rows. Works in any host thread.
cvs_status make_half_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int64_t cols, int64_t stride,
                         int box_rows);

}  // namespace cvs
