// Host-side helpers shared by the C entry points: the device of a call, the library's launch counter and the
// calling thread's last CUDA error (both kept in swiglu_capi.cu), extents of strided tensors.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "swiglu_b200.h"

namespace swiglu_b200 {

// Counts one kernel launch in swiglu_b200_launch_count().
void note_launch();
// Records `e` for swiglu_b200_last_cuda_error() and returns `code`.
int note_cuda_error(int code, cudaError_t e);
// The code of a launch that was just made, which is counted.
inline int launched() {
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_LAUNCH, err);
  note_launch();
  return SWIGLU_B200_OK;
}

// Makes `device` current for the duration of a call (no-op for -1 or when it already is).
struct CallDevice {
  int prev = -1;
  bool switched = false;
  cudaError_t err = cudaSuccess;
  explicit CallDevice(int device) {
    if (device < 0) return;
    err = cudaGetDevice(&prev);
    if (err != cudaSuccess) return;
    if (prev != device) {
      err = cudaSetDevice(device);
      switched = (err == cudaSuccess);
    }
  }
  ~CallDevice() {
    if (switched) cudaSetDevice(prev);
  }
  CallDevice(const CallDevice&) = delete;
  CallDevice& operator=(const CallDevice&) = delete;
};

inline unsigned long long address(const void* p) { return (unsigned long long)(uintptr_t)p; }

// Bytes [lo, hi) touched by `rows` rows of `row_bytes` bytes whose starts are `pitch_bytes` apart.
struct ByteRange {
  unsigned long long lo, hi;
};
inline ByteRange byte_range(const void* p, long long rows, long long row_bytes, long long pitch_bytes) {
  return ByteRange{address(p), address(p) + (unsigned long long)((rows - 1) * pitch_bytes + row_bytes)};
}
inline bool overlap(const ByteRange& a, const ByteRange& b) { return a.lo < b.hi && b.lo < a.hi; }
// Whether two sets of rows at one pitch share a byte.  Their rows may lie between one another's, as the two halves of a
// packed tensor do.
inline bool rows_overlap(const void* p, const void* q, long long rows, long long row_bytes, long long pitch_bytes) {
  const unsigned long long a = address(p), b = address(q);
  const unsigned long long apart = a < b ? b - a : a - b;
  if (rows <= 1) return apart < (unsigned long long)row_bytes;
  const unsigned long long skipped = apart / (unsigned long long)pitch_bytes;  // rows before the one it falls into
  const unsigned long long into = apart % (unsigned long long)pitch_bytes;
  return (skipped < (unsigned long long)rows && into < (unsigned long long)row_bytes) ||
         (skipped + 1 < (unsigned long long)rows && into + (unsigned long long)row_bytes > (unsigned long long)pitch_bytes);
}

// True when rows * pitch (in bytes) and everything derived from it stays within 62 bits.
inline bool fits_address_space(long long rows, long long pitch, long long element) {
  if (pitch > (1LL << 56) || rows > (1LL << 56)) return false;
  return rows == 0 || pitch * element <= (1LL << 62) / rows;
}

}  // namespace swiglu_b200
