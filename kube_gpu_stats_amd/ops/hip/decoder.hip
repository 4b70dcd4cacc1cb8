// Error reporting shared by the decoder block's entries (decoder.h).
#include "decoder.h"

#include <cstdio>

#include "decoder_common.h"

namespace kgs {

thread_local char g_decoder_error[256];

int fail(const char* what, const char* why) {
  std::snprintf(g_decoder_error, sizeof g_decoder_error, "%s: %s", what, why);
  return -1;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(what, hipGetErrorString(e));
}

}  // namespace kgs

extern "C" const char* kgs_decoder_last_error() { return kgs::g_decoder_error; }
