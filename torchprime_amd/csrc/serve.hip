// What every entry point of libtprime_hip.so shares (error plumbing, version query), and the operators that answer with a model:
// the paged key-value cache, attention over it, sampling.
#include "kv_cache.hpp"
#include "paged_attn.hpp"
#include "sample.hpp"

namespace tp {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

int check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return TP_ERR_LAUNCH;
  }
  return TP_OK;
}

}  // namespace tp

extern "C" int tp_version(void) { return 100; }
extern "C" const char* tp_last_error(void) { return tp::g_err; }
