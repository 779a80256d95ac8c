// What the kernels that stage tiles in LDS and read them as MFMA operands share: loads straight into LDS,
// transposed reads, and the reductions of a softmax row that is spread over the wave's four 16-lane rows.
#pragma once

#include "decode_common.h"

namespace ti {

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// One 1 KiB load into LDS: lane i's 16 bytes at rsrc + voff land at LDS byte lds + 16 i. Issued
// as assembly, which the compiler's wait insertion does not see: its own waits for the loads it
// knows stay at least as strict (vector memory operations complete in issue order, so hidden
// loads only add to what a count waits for), and the kernel waits for these loads explicitly
// before each stage barrier. The builtin form instead makes the compiler wait for every load
// into a stage array before reading that array, all loads issued since included, which defeats
// a pipeline that keeps two tiles in flight. Nor does the compiler's hazard recogniser see it: a
// descriptor word written by v_readfirstlane or v_readlane (VALU) must be five wait states old when
// a buffer instruction reads it, and m0 one, which the s_nop provides.
__device__ __forceinline__ void load_lds16(u32x4 rsrc, uint32_t voff, const uint16_t* lds) {
  const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(m0)
               : "memory");
}

// The cache row at byte offset `off` from `base`.
__device__ __forceinline__ const uint16_t* at_bytes(const uint16_t* base, uint64_t off) {
  return reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(base) + off);
}

// Buffer descriptor words of [base, base + bytes) (raw, no stride), uniform.
__device__ __forceinline__ u32x4 rsrc_words(const uint16_t* base, uint32_t bytes) {
  const uint64_t addr = reinterpret_cast<uint64_t>(base);
  return u32x4{uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(addr)))),
               uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(addr >> 32) & 0xffffu))),
               uint32_t(__builtin_amdgcn_readfirstlane(int(bytes))), uint32_t(kBufferRsrcWord3)};
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// ds_read_b64_tr_b16 (measured on gfx950): within each 16-lane group, output lane j receives
// element j % 4 of the 8-byte rows addressed by lanes j/4, j/4 + 4, j/4 + 8, j/4 + 12.
__device__ __forceinline__ u32x2 lds_read_tr4(const uint16_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}

// Maxima without the quieting of NaN operands that fmaxf costs (v_maximum3 gives a NaN for one). Not as assembly:
// an accumulator must be some wait states old when an instruction outside the matrix unit reads it, and the
// compiler counts them only up to instructions that it knows.
__device__ __forceinline__ float max2(float x, float y) { return __builtin_elementwise_maximum(x, y); }
__device__ __forceinline__ float max3(float x, float y, float z) { return max2(max2(x, y), z); }

// Max over the four 16-lane rows of the wave (lanes n, n+16, n+32, n+48).
__device__ __forceinline__ float row_group_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_group_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// LDS places of 16-byte chunk c of row r: c ^ swz16(r) in rows of whole 256-byte blocks, c ^ swz8(r) in rows of 128
// bytes. A ds_read_b128 serves rows {0-3, 12-15} of one chunk with rows {4-11} of its neighbour, a transposed read two
// neighbouring chunks of eight rows; either way these are 16 different bank quads.
__device__ __forceinline__ int swz16(int r) { return ((2 * r) & 15) ^ ((r & 8) ? 9 : 0); }
__device__ __forceinline__ int swz8(int r) {
  const int u = (r >> 1) & 7;
  return ((2 * u) & 7) ^ ((u & 4) ? 5 : 0);
}

// A list of `total` tiles cut into at most `most` runs of at least `shortest`, the first `rest` of them one tile longer.
// All in 32 bits (the host refuses or does not cut longer lists): a 64-bit division takes about half a microsecond at
// the start of every workgroup.
struct Runs {
  uint32_t runs, base, rest;
  __device__ __forceinline__ Runs(uint32_t most, uint32_t total, uint32_t shortest) {
    runs = max(1u, min(most, total / shortest));
    base = total / runs;
    rest = total - base * runs;
  }
  __device__ __forceinline__ uint32_t start(uint32_t i) const { return i * base + min(i, rest); }
  __device__ __forceinline__ uint32_t holding(uint32_t u) const {  // the run of position u
    const uint32_t longer = rest * (base + 1);
    return u < longer ? u / (base + 1) : rest + (u - longer) / base;
  }
};

// Exp2 units by which softmax weights are lifted before they are rounded to 16 bits; the sums carry the same factor, which
// the division by l takes out. An fp16 weight has steps of 2^-24 at least, so that 60,000 of 2^-25.6 of their row's
// greatest (the tail behind a first token that takes most of the attention) would all round to zero, while l counts
// them. Seven, and the eight by which a maximum may rise before it is taken over, stay below fp16's 2^16. bf16 has the
// exponents of 32 bits and needs none.
__device__ __forceinline__ constexpr float weight_lift(Bf16) { return 0.f; }
__device__ __forceinline__ constexpr float weight_lift(F16) { return 7.f; }

}  // namespace ti
