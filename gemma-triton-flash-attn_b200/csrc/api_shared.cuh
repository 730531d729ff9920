// Host helpers shared by the translation units of the C ABI (defined in
// gqa_fa_api.cu): error reporting, device binding, the device status word and
// the wait settings of later launches.
#pragma once
#include <cuda_runtime.h>

namespace gqafa {

// Record a message for gqafa_last_error and return `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();
// Make the device of `stream` (the current one for the legacy stream) current.
int bind_device(cudaStream_t stream);
// Device address of the current device's status word (nullptr on failure).
int* status_ptr();
// Bound of every mbarrier wait in clock cycles, and the test switch that keeps
// the producers idle (gqafa_set_test_waits).
long long wait_limit_setting();
int no_loads_setting();

}  // namespace gqafa
