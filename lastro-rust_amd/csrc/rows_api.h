// What the entry points over a caller's buffers share: statuses, rows, the buffers' device.
#pragma once
#include "../../include/moert.h"
#include "kv8.h"

namespace moert {

int set_error(int code, const char* fmt, ...);

#define KV_CFG(cond, ...) \
  do {                    \
    if (!(cond)) return set_error(MOERT_E_CONFIG, __VA_ARGS__); \
  } while (0)

#define KV_HIP(expr)                                                                                            \
  do {                                                                                                          \
    const hipError_t e_ = (expr);                                                                               \
    if (e_ != hipSuccess)                                                                                       \
      return set_error(MOERT_E_DEVICE, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)

#define KV_TRY(expr)             \
  do {                           \
    const int rc_ = (expr);      \
    if (rc_ != MOERT_OK) return rc_; \
  } while (0)

// Rows that a call reads or (out) writes, of one of `types` (a bit each).
inline int rows(const char* what, const moert_rows* r, int types, int n_seqs, int n, int heads, int d, bool out,
                KvRows* k) {
  KV_CFG(r && r->data_dev, "%s: null rows", what);
  KV_CFG(r->dtype >= 0 && r->dtype < 31 && types >> r->dtype & 1, "%s: rows of dtype %d", what, r->dtype);
  KV_CFG((uintptr_t)r->data_dev % (r->dtype == MOERT_F32 ? 4 : 2) == 0, "%s: rows not aligned to their type", what);
  if (out) {
    // each axis, from the one with the least stride on, has to clear all that the ones before it span
    struct Axis {
      long long stride;
      int count;
    } a[3] = {{r->seq_stride, n_seqs}, {r->pos_stride, n}, {r->head_stride, heads}};
    for (int i = 0; i < 2; i++)
      for (int j = 0; j < 2 - i; j++)
        if (a[j].stride > a[j + 1].stride) {
          const Axis t = a[j];
          a[j] = a[j + 1];
          a[j + 1] = t;
        }
    __int128 span = d;
    for (const Axis& x : a)
      if (x.count > 1) {
        KV_CFG(x.stride >= span, "%s: rows to be written overlap (strides %lld, %lld, %lld)", what, r->seq_stride,
               r->pos_stride, r->head_stride);
        span += (__int128)x.stride * (x.count - 1);
      }
  }
  *k = KvRows{r->data_dev, r->dtype == MOERT_F16 ? 1 : r->dtype == MOERT_BF16 ? 2 : 0, r->seq_stride, r->pos_stride, r->head_stride};
  return MOERT_OK;
}

// Makes the buffers' device the current one while the call lasts. An error that an earlier call of the caller's has
// left in the thread is dropped: the launchers ask for the last error, and it would pass for a launch's.
class OnDevice {
 public:
  ~OnDevice() {
    if (back_ >= 0) (void)hipSetDevice(back_);
  }
  int enter(const char* what, const void* p) {
    (void)hipGetLastError();
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
      (void)hipGetLastError();  // an address that the runtime does not know is no device error
      return set_error(MOERT_E_CONFIG, "%s: the cache is not in device memory", what);
    }
    KV_CFG(a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged, "%s: the cache is not in device memory",
           what);
    int now = -1;
    KV_HIP(hipGetDevice(&now));
    if (now != a.device) {
      KV_HIP(hipSetDevice(a.device));
      back_ = now;
    }
    return MOERT_OK;
  }

 private:
  int back_ = -1;
};

}  // namespace moert
