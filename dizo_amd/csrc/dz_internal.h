// What the library's C entry points share.
#pragma once
#include <stdint.h>

#include <string>

namespace dz {
// Sets the thread's message (dz_last_error) and returns `code`.
int32_t api_fail(int32_t code, const std::string& msg);
// DZ_OK if [p, p + bytes) lies inside one device allocation.
int32_t api_check_range(const void* p, uint64_t bytes, const char* what);
}  // namespace dz
