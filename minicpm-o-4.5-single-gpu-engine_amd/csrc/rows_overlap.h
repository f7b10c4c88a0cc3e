// Whether two sets of equally wide rows in memory share a byte: for argument checks of calls whose operands may be slices of one
// buffer (queries and keys of a joint projection lie between each other without sharing anything).
#pragma once

#include <stdint.h>

namespace t2w {

struct Rows {
  const void* p;
  long long ld, width;  // bytes between rows and bytes of a row; width <= ld where there are several
  long long n;
};

// true where they may meet: exact for equal strides, by the spans' ends otherwise
inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.n <= 0 || b.n <= 0 || a.width <= 0 || b.width <= 0) return false;
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  const uintptr_t xe = x + (uintptr_t)(a.ld * (a.n - 1) + a.width), ye = y + (uintptr_t)(b.ld * (b.n - 1) + b.width);
  if (x >= ye || y >= xe) return false;
  if (a.n == 1 || b.n == 1 || a.ld != b.ld) {
    // one row against rows it may lie between, or strides that differ: only a row between two others is told apart
    const Rows& many = a.n > 1 ? a : b;
    const Rows& one = a.n > 1 ? b : a;
    if (one.n > 1 || many.n == 1) return true;
    const uintptr_t m = (uintptr_t)many.p, o = (uintptr_t)one.p;
    if (o < m) return true;
    const uintptr_t at = (o - m) % (uintptr_t)many.ld;
    return !(at >= (uintptr_t)many.width && at + (uintptr_t)one.width <= (uintptr_t)many.ld);
  }
  const uintptr_t ld = (uintptr_t)a.ld, d = y >= x ? (y - x) % ld : (ld - (x - y) % ld) % ld;  // b's rows behind a's, modulo a row
  return !(d >= (uintptr_t)a.width && d + (uintptr_t)b.width <= ld);
}

}  // namespace t2w
