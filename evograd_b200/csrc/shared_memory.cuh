// Dynamic shared memory beyond the 48 KB that a launch may ask for without leave.
#pragma once

#include <cstddef>

namespace evg {

// Lets `kernel` be launched with `bytes` of dynamic shared memory on the current device; false
// where that does not fit. The limit is a property of the kernel and the device, not of a launch:
// it is raised to the largest size that fits beside the kernel's static shared memory and never
// lowered, so a call from another thread cannot take it away between here and the launch.
bool allow_shared_memory(const void* kernel, size_t bytes);

}  // namespace evg
