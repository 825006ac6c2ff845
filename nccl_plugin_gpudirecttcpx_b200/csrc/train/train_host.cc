// Error text of the training operators' C ABI.
#include <cstdarg>
#include <cstdio>

#include <cuda_runtime.h>

#include "tcpxb/train.h"

namespace tcpxb_train {

static thread_local char g_error[256];

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return code;
}

int use(int device) {
  const cudaError_t e = cudaSetDevice(device);
  return e == cudaSuccess ? TCPXB_T_OK : fail(TCPXB_T_CUDA, "device %d: %s", device, cudaGetErrorString(e));
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TCPXB_T_OK : fail(TCPXB_T_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace tcpxb_train

extern "C" const char* tcpxb_train_last_error(void) { return tcpxb_train::g_error; }
