// What the library's C entry points share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

namespace dz {
// Sets the thread's message (dz_last_error) and returns `code`.
int32_t api_fail(int32_t code, const std::string& msg);
// The same for a failed HIP call (DZ_ERR_HIP); clears the runtime's record of the error.
int32_t api_hip_fail(hipError_t e, const char* what);
// DZ_OK if [p, p + bytes) lies inside one device allocation.
int32_t api_check_range(const void* p, uint64_t bytes, const char* what);
}  // namespace dz
