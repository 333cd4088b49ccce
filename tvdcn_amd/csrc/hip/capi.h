// What the files of the C ABI share (defined in capi.hip): the thread's last error and the kernel timer.
#pragma once

#include <hip/hip_runtime.h>

#include <functional>
#include <string>

#include "../../../include/tvdcn_hip.h"

namespace tvdcn_hip {

tvdcn_status api_fail(tvdcn_status st, const std::string &msg);
void api_clear_error();
// runs `launch` between the kernel timer's events; its error becomes TVDCN_STATUS_HIP_ERROR
tvdcn_status api_launch(int family, hipStream_t s, const std::function<hipError_t()> &launch);

}  // namespace tvdcn_hip
