// The checks of arguments that the C ABI's operators on channels-last maps share (capi_maps.hip, capi_rows.hip).
#pragma once

#include <initializer_list>
#include <string>

#include "capi.h"

namespace tvdcn_hip {
namespace {

constexpr int64_t MOST_CHANNELS = 1 << 20;
constexpr int64_t MOST_ELEMENTS = (int64_t)1 << 40;   // of a map: its bytes, and its workspace's, fit 64 bits

inline tvdcn_status invalid(const std::string &msg) { return api_fail(TVDCN_STATUS_INVALID_ARGUMENT, msg); }

inline tvdcn_status check_type(const char *what, int32_t dtype, int32_t activation = TVDCN_ACT_NONE) {
    if (dtype < 0 || dtype > 3) return invalid(std::string(what) + ": unknown dtype");
    if (dtype == TVDCN_DTYPE_FLOAT64)
        return api_fail(TVDCN_STATUS_NOT_SUPPORTED, std::string(what) + ": float32, float16 and bfloat16 only");
    if (activation < TVDCN_ACT_NONE || activation > TVDCN_ACT_GELU) return invalid(std::string(what) + ": unknown activation");
    return TVDCN_STATUS_SUCCESS;
}

inline tvdcn_status check_map(const char *what, int64_t rows, int64_t channels) {
    if (rows < 0) return invalid(std::string(what) + ": negative size");
    if (channels <= 0) return invalid(std::string(what) + ": channels must be positive");
    if (channels > MOST_CHANNELS)
        return api_fail(TVDCN_STATUS_NOT_SUPPORTED, std::string(what) + ": more than 2^20 channels");
    if (rows > MOST_ELEMENTS / channels) return api_fail(TVDCN_STATUS_NOT_SUPPORTED, std::string(what) + ": map too large");
    return TVDCN_STATUS_SUCCESS;
}

inline tvdcn_status check_pointers(const char *what, std::initializer_list<const void *> needed,
                            std::initializer_list<const void *> optional) {
    for (const void *p : needed)
        if (!p) return invalid(std::string(what) + ": null tensor");
    for (auto list : {needed, optional})
        for (const void *p : list)
            if (reinterpret_cast<uintptr_t>(p) & 15) return invalid("tensor pointers must be 16-byte aligned");
    return TVDCN_STATUS_SUCCESS;
}

// statistics: single floats
inline tvdcn_status check_floats(std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (reinterpret_cast<uintptr_t>(p) & 3) return invalid("statistics must be 4-byte aligned");
    return TVDCN_STATUS_SUCCESS;
}

inline tvdcn_status check_workspace(const void *workspace, size_t have, size_t need) {
    if (have < need || (need > 0 && !workspace))
        return api_fail(TVDCN_STATUS_WORKSPACE_TOO_SMALL, "workspace too small: " + std::to_string(have) + " bytes, " +
                                                              std::to_string(need) + " needed");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return invalid("workspace must be 16-byte aligned");
    return TVDCN_STATUS_SUCCESS;
}

#define RETURN_IF(expr) \
    if (const tvdcn_status st_ = (expr)) return st_

}  // namespace
}  // namespace tvdcn_hip
