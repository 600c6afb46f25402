// What the C entries of the operators for batches share: their device, their errors, checks of arguments.
#pragma once
#include <exception>

#include "../../include/spx.h"
#include "internal.h"

namespace spx {

// The context's device for the length of a call, the caller's afterwards.
struct OnDevice {
  int was = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&was);
    if (err == hipSuccess && was != device) err = hipSetDevice(device);
    else was = -1;
  }
  ~OnDevice() { if (was >= 0) (void)hipSetDevice(was); }
};

// No exception leaves a C entry (error texts allocate).
template <class F>
inline int entry(F f) {
  try {
    return f();
  } catch (const std::exception &) {
    return -1;
  }
}

inline int log2_of(int v) { return 31 - __builtin_clz((unsigned)v); }
inline bool row_type(int t) { return t == SPX_F32 || t == SPX_F16 || t == SPX_BF16; }
inline int64_t size_of(int t) { return t == SPX_F32 ? 4 : 2; }
inline bool aligned(const void *p, int64_t a) { return (uintptr_t)p % (uintptr_t)a == 0; }
// Arrays of 32-bit numbers. (Kernels read some of them by scalar loads, which drop an address's last two bits.)
template <class... T>
inline bool words(T... p) { return (aligned(p, 4) && ...); }

}  // namespace spx
