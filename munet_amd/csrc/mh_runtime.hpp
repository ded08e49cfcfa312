// Host runtime helpers shared by the C ABI and the engine: error type, HIP
// status checks, per-device error flags and growable workspace.
#pragma once

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

namespace mh {

struct Error : std::runtime_error {
  explicit Error(const std::string &m) : std::runtime_error(m) {}
};

void set_last_error(const std::string &msg);
void hip_check(hipError_t e, const char *what);
int current_device();
// The embedding's flag, which an engine takes for its own, and (right behind it)
// that of the paged cache's calls, which an engine's run leaves alone.
int *device_error_flag();
int *serving_error_flag();
// Grow-only scratch on the current device (may hipMalloc; never under capture).
void *workspace(size_t bytes);
void set_last_kernel_time_us(double us);

}  // namespace mh
