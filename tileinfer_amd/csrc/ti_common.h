// Shared host/device helpers of the gfx950 paged KV-cache library.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/tileinfer_amd.h"

namespace ti {

// Records a printf-style message as the calling thread's last error and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Checks the launch that was just enqueued; returns TI_OK or TI_ELAUNCH with the runtime's text.
int check_launch(const char* what);

// Number of compute units of the current device (cached per device id).
int device_cu_count();

// Workgroups of at most 256 threads that a launch takes along x: its work items there are counted in 32 bits.
constexpr int64_t kMaxGridX = (int64_t(1) << 24) - 1;

// Scores are scaled by scale * log2 e in 32 bits; a larger scale (or an infinite one, as a host double beyond 32 bits
// becomes) leaves them.
constexpr float kMaxScale = 1e30f;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 4 x 32-bit registers: one 16-byte global access, or the 8 x 16-bit operand of a
// 16x16x32 MFMA.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

}  // namespace ti
