// Element types of the layer operators (norm.hip, attention*.hip): float32, bfloat16 and float16 rows, float32 sums.
#pragma once
#include <string.h>

#include "../../include/vsn.h"
#include "common.h"

namespace vsn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct vec8;
template <>
struct vec8<float> {
  typedef f32x8 type;
};
template <>
struct vec8<__bf16> {
  typedef bf16x8 type;
};
template <>
struct vec8<_Float16> {
  typedef f16x8 type;
};

// Makes a device current for the length of a call and puts the caller's back.  (A failure is the return code's to report:
// left behind, the runtime's last error would be taken for one of the next call's, here or in torch.)
struct DeviceScope {
  int before = -1;
  bool ok = false;
  explicit DeviceScope(int device) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    ok = before == device || hipSetDevice(device) == hipSuccess;
    if (!ok) (void)hipGetLastError();
    if (before == device) before = -1;
  }
  ~DeviceScope() {
    if (ok && before >= 0) (void)hipSetDevice(before);
  }
};

}  // namespace vsn
