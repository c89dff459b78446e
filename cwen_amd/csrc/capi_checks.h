// Argument checks that the serving operators' entry points share (host code).
#pragma once
#include "cwen_internal.h"

namespace {

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }
bool aligned4(const void *p) { return ((uintptr_t)p & 3u) == 0; }
int elem_size(int type) { return type == CWEN_T_F32 ? 4 : type == CWEN_T_F16 || type == CWEN_T_BF16 ? 2 : 0; }

// The context's device for the length of a call, whatever device the caller
// has current.
struct OnDevice {
  int before = -1, rc = CWEN_OK;
  explicit OnDevice(int device) {
    if (hipGetDevice(&before) != hipSuccess) {
      rc = CWEN_EHIP;
      before = -1;
    } else if (before == device) {
      before = -1;
    } else if (hipSetDevice(device) != hipSuccess) {
      rc = CWEN_EHIP;
    }
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// Rows of n_head heads of dim elements (strides in elements).
bool ok_rows(const void *p, long long ts, long long row) {
  return p && aligned16(p) && ts % 8 == 0 && ts >= row;
}
bool overlap(const void *a, long long abytes, const void *b, long long bbytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + (uintptr_t)bbytes && y < x + (uintptr_t)abytes;
}

// Whether rows of xr bytes at x keep clear of T rows of yr bytes at y: no common memory at all,
// or (`inside`) rows of the same stride that lie side by side, as the parts of one product do.
bool clear_of(const void *x, long long x_ts, long long xr, const void *y, long long y_ts, long long yr, int T, bool inside) {
  if (!overlap(x, (T - 1) * x_ts + xr, y, (T - 1) * y_ts + yr)) return true;
  if (!inside || T == 1 || x_ts != y_ts) return false;
  long long off = (long long)((intptr_t)x - (intptr_t)y) % y_ts;
  if (off < 0) off += y_ts;
  return off >= yr && off + xr <= y_ts;
}

}  // namespace
