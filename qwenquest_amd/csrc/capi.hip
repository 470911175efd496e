// Library-level entry points: version, error reporting, a stream's capture.
#include <stdarg.h>
#include <string.h>

#include "qq_common.h"

namespace qq {
namespace {
thread_local char g_last_error[1024] = "";
}

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(QQ_EHIP, "%s: %s", what, hipGetErrorString(e));
  return QQ_OK;
}

}  // namespace qq

extern "C" int qq_version(void) { return 100; }

extern "C" const char* qq_last_error(void) { return qq::g_last_error; }

extern "C" int64_t qq_stream_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return -1;
  }
  if (status == hipStreamCaptureStatusNone) return 0;
  return status == hipStreamCaptureStatusActive ? (int64_t)(id + 1) : -1;
}
