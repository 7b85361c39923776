// moa_checks.h -- host checks of the paged cache's and the search calls' arguments: the reason is recorded, the code returned.
#pragma once

#include <string>

#include "../../include/moa_ops.h"
#include "moa_internal.h"

namespace moa {

inline int bad_value(const std::string& msg) { return set_error(MOA_ERROR_INVALID_VALUE, msg.c_str()); }

inline int check_ptr(const void* p, const char* name, size_t align) {
    if (!p) return bad_value(std::string(name) + " is NULL");
    if (reinterpret_cast<uintptr_t>(p) % align)
        return set_error(MOA_ERROR_MISALIGNED, (std::string(name) + " is not " + std::to_string(align) + "-byte aligned").c_str());
    return MOA_SUCCESS;
}

inline int check_range(int v, int lo, int hi, const char* name) {
    if (v >= lo && v <= hi) return MOA_SUCCESS;
    return bad_value(std::string(name) + " must be in [" + std::to_string(lo) + ", " + std::to_string(hi) + "], got " + std::to_string(v));
}

}  // namespace moa
