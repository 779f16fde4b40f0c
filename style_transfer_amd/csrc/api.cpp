// Library-level entry points of libst_hip.so.
#include "common.h"

namespace st {
char* error_buffer() {
  static thread_local char buf[512] = {0};
  return buf;
}
}  // namespace st

extern "C" int st_version(void) { return 122; }  // 0.1.22: + st_capture_id

extern "C" const char* st_last_error(void) { return st::error_buffer(); }

extern "C" unsigned long long st_capture_id(st_stream_t stream) {
  if (!stream) return 0;                                          // the null stream cannot be captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
}
