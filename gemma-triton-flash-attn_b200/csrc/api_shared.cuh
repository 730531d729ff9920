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

// Forward whose batch elements have their own lengths (int32 device arrays,
// see ragged_lens): q [B, Hq, N, D] with strides, k and v contiguous
// [B, Hkv, Nk, D], lse (may be null) [B, Hq, N]. Arguments are the caller's to
// check; the device is bound.
struct RaggedForward {
  const void* q;
  const long long* q_strides;
  const void *k, *v;
  void* o;
  const long long* o_strides;
  float* lse;
  const int *kv_lens, *q_lens;
  int B, Hq, Hkv, N, Nk, D, kv_cap, causal, window;
  float scale;
  bool bf16;
};
int ragged_forward(const RaggedForward& r, cudaStream_t stream);

}  // namespace gqafa
