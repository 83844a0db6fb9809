// The device accounts' entry points over host memory, their kernels followed thread by thread (hip/hip_runtime.h beside this file).
#include <hip/hip_runtime.h>

#include <cstdarg>

#include "../../kv-project_amd/csrc/page_tables.hip"

namespace kvq {
void set_error(const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vfprintf(stderr, fmt, args);
  va_end(args);
}
}  // namespace kvq

extern "C" void lockstep_order(int order) { lockstep::order = order; }
extern "C" const char* lockstep_error() {     // since the last call
  const char* e = lockstep::error;
  lockstep::error = nullptr;
  return e;
}
