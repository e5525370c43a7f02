// Whether two matrices share memory. Plain C++, no CUDA.
#pragma once
#include <stdint.h>

namespace sx {

// Rows of a matrix as byte ranges: `rows` of `bytes` each, `stride` bytes apart (stride >= bytes).
struct ByteRows {
  const void* p;
  long long rows, bytes, stride;
};
inline ByteRows one_row(const void* p, long long bytes) { return {p, p != nullptr ? 1 : 0, bytes, bytes}; }
// Whether a byte belongs to both: an output that other rows or CTAs still read as input. Rows of one matrix may lie between another's.
inline bool share_bytes(const ByteRows& a, const ByteRows& b) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (a.rows <= 0 || b.rows <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
  if (pa + (a.rows - 1) * a.stride + a.bytes <= pb || pb + (b.rows - 1) * b.stride + b.bytes <= pa) return false;
  if (a.stride == b.stride) {  // two views of one buffer: the same for every pair of rows
    if (pb < pa) return share_bytes(b, a);
    const long long q = (long long)(pb - pa) / a.stride, r = (long long)(pb - pa) % a.stride;
    return (q < a.rows && r < a.bytes) || (q + 1 < a.rows && r + b.bytes > a.stride);
  }
  for (long long i = 0, j = 0; i < a.rows && j < b.rows;) {
    const uintptr_t ra = pa + i * a.stride, rb = pb + j * b.stride;
    if (ra < rb + b.bytes && rb < ra + a.bytes) return true;
    if (ra < rb) ++i;
    else ++j;
  }
  return false;
}

}  // namespace sx
