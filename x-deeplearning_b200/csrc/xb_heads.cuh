// What the kernels of the attention over lists share: rows of several heads and whether two sets of them meet.
#pragma once

#include "xb_common.cuh"
#include "xb_ssm.cuh"

namespace xb {

// element c of head h of row t: at + t * row + h * head + c
struct Heads {
  const void* at;
  int64_t row, head;
  template <typename T>
  __device__ __forceinline__ const T* get(int64_t t, int h) const { return static_cast<const T*>(at) + t * row + h * head; }
};

// (elements of a row of n heads of width d, from the first to behind the last)
inline int64_t heads_width(int64_t head, int n, int d) { return (n - 1) * head + d; }
// Whether two sets of rows share memory, by where they begin and end; strides in elements of `size` bytes
inline bool heads_meet_ends(const Heads& a, int na, int da, int64_t rows_a, const Heads& b, int nb, int db, int64_t rows_b, int64_t size) {
  if (!a.at || !b.at || rows_a < 1 || rows_b < 1) return false;
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.at), q = reinterpret_cast<uintptr_t>(b.at);
  return p < q + (uintptr_t)(((rows_b - 1) * b.row + heads_width(b.head, nb, db)) * size) && q < p + (uintptr_t)(((rows_a - 1) * a.row + heads_width(a.head, na, da)) * size);
}
// Whether two sets of rows share memory. Told exactly where both have one row stride and the heads of a row
// lie within it (one set may take other columns than the other), else by where they begin and end (one row's stride says nothing).
inline bool heads_meet(const Heads& a, int na, int da, const Heads& b, int nb, int db, int64_t rows, int64_t size) {
  if (!a.at || !b.at || rows < 1 || na < 1 || nb < 1) return false;
  const int64_t wa = heads_width(a.head, na, da), wb = heads_width(b.head, nb, db);
  if (rows > 1 && a.row == b.row && wa <= a.row && wb <= b.row) return rows_meet(a.at, a.row * size, wa * size, b.at, b.row * size, wb * size, rows);
  return heads_meet_ends(a, na, da, rows, b, nb, db, rows, size);
}
inline bool heads_whole(const Heads& a, int64_t size, int64_t unit) {
  return reinterpret_cast<uintptr_t>(a.at) % unit == 0 && a.row * size % unit == 0 && a.head * size % unit == 0;
}
// Outputs of several heads: different (row, head) share no element
inline bool heads_apart(const Heads& a, int n, int d, int64_t rows) {
  if (n > 1 && a.head < d) return false;
  if (rows <= 1) return true;
  return a.row >= heads_width(a.head, n, d) || (n > 1 ? a.row >= d && a.head >= (rows - 1) * a.row + d : a.row >= d);
}

}  // namespace xb
