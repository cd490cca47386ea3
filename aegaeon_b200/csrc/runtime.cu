// Library-wide host utilities: thread-local error text, version, SM count cache and the
// sticky device error word reader.
#include "aeg_common.cuh"

#include <mutex>
#include <vector>

namespace aeg {

namespace {
thread_local std::string t_last_error;
}

int set_error(int code, const char* fmt, ...) {
  char buf[1024];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  t_last_error.assign(buf);
  return code;
}

int num_sms() {
  static std::mutex mu;
  static std::vector<int> cache;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= static_cast<int>(cache.size())) cache.resize(dev + 1, 0);
  if (cache[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cache[dev] = n;
  }
  return cache[dev];
}

// Per device the stream, and the capture on it (0: none), whose last noted launch is an attention; one at a
// time, so that another stream's attention makes this one's writes start their successors later, never sooner.
namespace {
constexpr int kTailDevices = 64;
struct Tail {
  bool any = false;
  cudaStream_t stream = nullptr;
  unsigned long long capture = 0;
};
std::mutex g_tail_mu;
Tail g_tail[kTailDevices];

// The current device's entry and the capture on `s`; false where either cannot be told.
bool find_tail(cudaStream_t s, Tail** t, unsigned long long* capture) {
  int dev = 0;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kTailDevices ||
      cudaStreamGetCaptureInfo(s, &status, &id) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  *t = &g_tail[dev];
  *capture = status == cudaStreamCaptureStatusNone ? 0 : id;
  return true;
}
}  // namespace

bool follows_attention(cudaStream_t s) {
  Tail* t = nullptr;
  unsigned long long capture = 0;
  if (!find_tail(s, &t, &capture)) return false;
  std::lock_guard<std::mutex> lock(g_tail_mu);
  return t->any && t->stream == s && t->capture == capture;
}

void note_launch(cudaStream_t s, bool attention) {
  Tail* t = nullptr;
  unsigned long long capture = 0;
  const bool known = find_tail(s, &t, &capture);
  std::lock_guard<std::mutex> lock(g_tail_mu);
  if (!known) {
    for (Tail& x : g_tail) x.any = false;
  } else if (attention) {
    *t = Tail{true, s, capture};
  } else if (t->stream == s && t->capture == capture) {
    t->any = false;
  }
}

}  // namespace aeg

extern "C" {

int aeg_version(void) { return 100; }

const char* aeg_last_error(void) { return aeg::t_last_error.c_str(); }

int aeg_read_device_errors(void* stream, uint32_t* flags) {
  AEG_CHECK_ARG(flags != nullptr, "aeg_read_device_errors: flags is NULL");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e[7] = {cudaSuccess, cudaSuccess, cudaSuccess, cudaSuccess, cudaSuccess, cudaSuccess, cudaSuccess};
  uint32_t f = aeg::deverr_read_and_clear_copy(s, &e[0]);
  f |= aeg::deverr_read_and_clear_cache(s, &e[1]);
  f |= aeg::deverr_read_and_clear_attn(s, &e[2]);
  f |= aeg::deverr_read_and_clear_step(s, &e[3]);
  f |= aeg::deverr_read_and_clear_prefill(s, &e[4]);
  f |= aeg::deverr_read_and_clear_int4(s, &e[5]);
  f |= aeg::deverr_read_and_clear_pool(s, &e[6]);
  for (cudaError_t x : e)
    if (x != cudaSuccess)
      return aeg::set_error(AEG_ERR_CUDA, "aeg_read_device_errors: %s", cudaGetErrorString(x));
  *flags = f;
  return AEG_OK;
}

}  // extern "C"
