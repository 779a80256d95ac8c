// The input side of a step whose positions have several axes (time, height, width of image and video tokens), in
// one launch (gfx950): for every token t
//   x'  = x * rsqrt(mean x^2 + eps) * (offset + w)                     (queries and keys; without weights x' = x)
//   a_i = positions[axes[i], t] * inv_freq[i],   i < rotary_dim / 2 = half
//   y_i = x'_i cos a_i - x'_{i + half} sin a_i,   y_{i + half} = x'_{i + half} cos a_i + x'_i sin a_i
// the rest of x' as it is; queries to q_out, keys and values (unchanged) to the cache rows at slot_mapping.
// Everything in 32 bits and rounded once; an angle is formed in 64 bits, in turns, and only its fraction of a turn
// becomes 32 bits: a position of 10^6 times a frequency of 1 has no bits left for the fraction in 32.
//
// A row is D / 8 lanes of 16 bytes, so that a wave takes 2 (D = 256) or 4 (D = 128) rows at a time; a wave takes P such
// passes over the rows of one token (its q, k and v heads), all loaded at once. Lane i computes the angle of frequency
// i (and of i + 64) once a wave, the lanes of a row read theirs back from LDS: a sine for every value instead would cost
// more time than the row's bytes. Bound: HBM and the vector work of the norms for long chunks (8,191 tokens with 24/4 heads
// of 256 and norms 56 to 59 us, 4.6 to 4.8 TB/s; without norms 50, 5.3 TB/s), the launch for short ones (48 tokens 7 to
// 8 us). The norms' sums by DPP and partners exchanged as 16-bit pairs, where both had been shuffles of 32-bit values: 58.5
// to 57.1 us in turn, 47.5 to 45.1 for 32/8 heads of 128. Loads with the nt bit made no difference.
#include <type_traits>

#include "decode_common.h"

namespace ti {
namespace {

constexpr int kMaxAxes = 4;

struct RopeAxesArgs {
  const uint16_t* q;  // [T, hq, D]
  int64_t q_st, q_sh;
  const uint16_t* k;  // [T, hkv, D]
  int64_t k_st, k_sh;
  const uint16_t* v;
  int64_t v_st, v_sh;
  const void* positions;  // [axes, T] int32 or int64
  int64_t pos_sa;
  const float* inv_freq;   // [half]
  const int32_t* axis_of;  // [half] or nullptr: all axis 0
  const uint16_t* q_w;     // [D] or nullptr
  const uint16_t* k_w;
  uint16_t* q_out;
  int64_t o_st, o_sh;
  uint16_t* k_cache;
  uint16_t* v_cache;
  int64_t cache_row, num_slots;
  const int32_t* slots;
  int32_t tokens, hq, hkv, rotary, axes, wide;  // wide: 64-bit positions
  int32_t parts;                                // waves of a token
  float eps, offset;
};

// Sum over the 16 (LPR 16) or 32 lanes of a row, in all of them.
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  auto turned = [](float v, auto by) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + decltype(by)::value, 0xf, 0xf, false));
  };
  x += turned(x, std::integral_constant<int, 8>{});  // row_ror
  x += turned(x, std::integral_constant<int, 4>{});
  x += turned(x, std::integral_constant<int, 2>{});
  x += turned(x, std::integral_constant<int, 1>{});
  if constexpr (LPR == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

template <int D, int P, typename Tag>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxesArgs a) {
  constexpr int LPR = D / 8;
  constexpr int RPW = 64 / LPR;
  constexpr int MAX_HALF = D / 2;  // frequencies
  __shared__ __align__(16) float s_cs[4][2][MAX_HALF];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t item = blockIdx.x * 4u + uint32_t(wave);
  const uint32_t parts = uint32_t(a.parts);
  const int t = int(item / parts);
  if (t >= a.tokens) return;  // uniform; no barrier below
  const int part = int(item - uint32_t(t) * parts);
  const int l = lane & (LPR - 1);
  const int rows = a.hq + 2 * a.hkv;

  u32x4 x[P];
  int row[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    row[i] = (part * P + i) * RPW + lane / LPR;
    const int r = min(row[i], rows - 1);  // lanes behind the last row repeat it and store nothing
    const uint16_t* src;
    if (r < a.hq) src = a.q + t * a.q_st + r * a.q_sh;
    else if (r < a.hq + a.hkv) src = a.k + t * a.k_st + (r - a.hq) * a.k_sh;
    else src = a.v + t * a.v_st + (r - a.hq - a.hkv) * a.v_sh;
    x[i] = load16(src + 8 * l);
  }
  const int half = a.rotary / 2;
  const bool low = 8 * l < half, turned = 8 * l < a.rotary;
  // The lane that holds a lane's partners; its own where it turns nothing.
  const int partner = turned ? (lane & ~(LPR - 1)) | (low ? l + half / 8 : l - half / 8) : lane;
  u32x4 wq = {}, wk = {}, pq = {}, pk = {};  // this lane's weights and its partners'
  if (a.q_w) {
    wq = load16(a.q_w + 8 * l);
    wk = load16(a.k_w + 8 * l);
    pq = load16(a.q_w + 8 * (partner & (LPR - 1)));
    pk = load16(a.k_w + 8 * (partner & (LPR - 1)));
  }
  const int64_t slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.num_slots;

#pragma unroll 1
  for (int f = lane; f < half; f += 64) {  // once; twice for more than 128 turned values
    const int axis = a.axis_of ? min(max(a.axis_of[f], 0), a.axes - 1) : 0;
    const int64_t at = axis * a.pos_sa + t;
    const double pos = a.wide ? double(static_cast<const int64_t*>(a.positions)[at])
                              : double(static_cast<const int32_t*>(a.positions)[at]);
    const double turns = pos * (double(a.inv_freq[f]) * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * float(turns - rint(turns)), &s, &c);
    s_cs[wave][0][f] = c;
    s_cs[wave][1][f] = s;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int at = turned ? (low ? 8 * l : 8 * l - half) : 0;
  f32x4 c[2], s[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    c[j] = *reinterpret_cast<const f32x4*>(&s_cs[wave][0][at + 4 * j]);
    s[j] = *reinterpret_cast<const f32x4*>(&s_cs[wave][1][at + 4 * j]);
    s[j] = low ? -s[j] : s[j];
    if (!turned) {
      c[j] = f32x4{1.f, 1.f, 1.f, 1.f};
      s[j] = f32x4{};
    }
  }

#pragma unroll
  for (int i = 0; i < P; ++i) {
    const bool is_q = row[i] < a.hq, is_v = row[i] >= a.hq + a.hkv;
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = unpack2(x[i][j], Tag{});
      y[2 * j] = p.x;
      y[2 * j + 1] = p.y;
    }
    float r = 1.f;
    if (a.q_w) {  // uniform
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
      r = rsqrtf(row_sum<LPR>(ss) / float(D) + a.eps);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 w = unpack2(is_q ? wq[j] : wk[j], Tag{});
        y[2 * j] *= r * (a.offset + w.x);
        y[2 * j + 1] *= r * (a.offset + w.y);
      }
    }
    // The rotation's partners come as 16-bit pairs, and are normalised here again: half the exchange.
    u32x4 res;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 other = unpack2(uint32_t(__shfl(int(x[i][j]), partner, 64)), Tag{});
      if (a.q_w) {
        const float2 w = unpack2(is_q ? pq[j] : pk[j], Tag{});
        other.x *= r * (a.offset + w.x);
        other.y *= r * (a.offset + w.y);
      }
      // Past the rotation the value itself: a partner that is not finite stays out of it.
      const float u = turned ? other.x * s[j >> 1][2 * j & 3] : -0.f;
      const float v = turned ? other.y * s[j >> 1][(2 * j & 3) + 1] : -0.f;
      res[j] = pack_fma2(y[2 * j], c[j >> 1][2 * j & 3], u, y[2 * j + 1], c[j >> 1][(2 * j & 3) + 1], v, Tag{});
    }
    if (row[i] >= rows) continue;
    uint16_t* dst;
    if (is_q) {
      dst = a.q_out + t * a.o_st + row[i] * a.o_sh;
    } else {
      if (!stored) continue;
      const int h = row[i] - a.hq - (is_v ? a.hkv : 0);
      dst = (is_v ? a.v_cache : a.k_cache) + slot * a.cache_row + int64_t(h) * D;
    }
    *reinterpret_cast<u32x4*>(dst + 8 * l) = is_v ? x[i] : res;
  }
}

bool vec_rows(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
}

template <int D, int P, typename Tag>
void launch_rope_axes(RopeAxesArgs a, hipStream_t s) {
  a.parts = int32_t(ceil_div(a.hq + 2 * int64_t(a.hkv), P * (64 / (D / 8))));
  const unsigned blocks = unsigned(ceil_div(int64_t(a.tokens) * a.parts, 4));
  hipLaunchKernelGGL((rope_axes_kernel<D, P, Tag>), dim3(blocks), dim3(256), 0, s, a);
}

// Passes of a wave: four where the rows fill the GPU several times over (the angles once for four passes, four loads
// in flight), one where they do not and each pass would wait for the one before. With 24/4 heads of 256, one against four:
// 8,191 tokens 87 us against 56, 1,024 (where the rule changes) 13.1 against 11.4, up to 512 8.1 to 8.6 either way.
template <int D, typename Tag>
void launch_rope_axes_dim(const RopeAxesArgs& a, hipStream_t s) {
  const int64_t passes = int64_t(a.tokens) * ceil_div(a.hq + 2 * int64_t(a.hkv), 64 / (D / 8));
  if (passes >= 64 * int64_t(device_cu_count())) launch_rope_axes<D, 4, Tag>(a, s);
  else launch_rope_axes<D, 1, Tag>(a, s);
}

}  // namespace
}  // namespace ti

extern "C" int ti_rope_axes_append(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                   int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                   int64_t v_stride_h, const void* positions, int64_t pos_stride_a,
                                   int32_t position_bits, const float* inv_freq, const int32_t* axis_of,
                                   const void* q_weight, const void* k_weight, float weight_offset, void* q_out,
                                   int64_t out_stride_t, int64_t out_stride_h, void* k_cache, void* v_cache,
                                   int64_t cache_row_stride, int64_t num_slots, const int32_t* slot_mapping,
                                   int32_t n_tokens, int32_t num_axes, int32_t num_q_heads, int32_t num_kv_heads,
                                   int32_t head_dim, int32_t rotary_dim, float eps, int32_t dtype, void* stream) {
  using namespace ti;
  const char* who = "ti_rope_axes_append";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  if (head_dim != 128 && head_dim != 256) {
    return fail(TI_EUNSUPPORTED, "%s: head_dim %d not built (128, 256)", who, head_dim);
  }
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0) {
    return fail(TI_EUNSUPPORTED, "%s: rotary_dim %d is not a multiple of 16 up to head_dim", who, rotary_dim);
  }
  if (position_bits != 32 && position_bits != 64) {
    return fail(TI_EUNSUPPORTED, "%s: positions of %d bits (32, 64)", who, position_bits);
  }
  const int64_t heads = int64_t(num_q_heads) + 2 * int64_t(num_kv_heads);
  if (n_tokens < 0 || num_axes < 1 || num_axes > kMaxAxes || num_q_heads <= 0 || num_kv_heads <= 0 || num_slots < 0 ||
      heads > (1 << 20) || ceil_div(int64_t(n_tokens) * heads, 4) > kMaxGridX) {
    return fail(TI_EINVAL, "%s: bad sizes n_tokens=%d num_axes=%d heads=%d/%d (at most 2^26 rows)", who, n_tokens,
                num_axes, num_q_heads, num_kv_heads);
  }
  if (n_tokens == 0) return TI_OK;
  if (!q || !k || !v || !q_out || !k_cache || !v_cache || !slot_mapping ||
      (rotary_dim > 0 && (!positions || !inv_freq)) || !q_weight != !k_weight) {
    return fail(TI_EINVAL, "%s: null pointer (the weights are both given or both not)", who);
  }
  if (!vec_rows(q, q_stride_t, q_stride_h) || !vec_rows(k, k_stride_t, k_stride_h) ||
      !vec_rows(v, v_stride_t, v_stride_h) || !vec_rows(q_out, out_stride_t, out_stride_h) ||
      !vec_rows(k_cache, cache_row_stride, 0) || !vec_rows(v_cache, cache_row_stride, 0) ||
      !vec_rows(q_weight, 0, 0) || !vec_rows(k_weight, 0, 0)) {
    return fail(TI_EINVAL, "%s: rows must be 16-byte aligned", who);
  }
  if (cache_row_stride < int64_t(num_kv_heads) * head_dim) {
    return fail(TI_EINVAL, "%s: cache rows of %d x %d values at stride %lld", who, num_kv_heads, head_dim,
                static_cast<long long>(cache_row_stride));
  }
  RopeAxesArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = static_cast<const uint16_t*>(k);
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v = static_cast<const uint16_t*>(v);
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.positions = positions;
  a.pos_sa = pos_stride_a;
  a.inv_freq = inv_freq;
  a.axis_of = axis_of;
  a.q_w = static_cast<const uint16_t*>(q_weight);
  a.k_w = static_cast<const uint16_t*>(k_weight);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.cache_row = cache_row_stride;
  a.num_slots = num_slots;
  a.slots = slot_mapping;
  a.tokens = n_tokens;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.rotary = rotary_dim;
  a.axes = num_axes;
  a.wide = position_bits == 64;
  a.eps = eps;
  a.offset = weight_offset;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == TI_DTYPE_BF16;
  if (head_dim == 256) {
    if (bf16) launch_rope_axes_dim<256, Bf16>(a, s);
    else launch_rope_axes_dim<256, F16>(a, s);
  } else {
    if (bf16) launch_rope_axes_dim<128, Bf16>(a, s);
    else launch_rope_axes_dim<128, F16>(a, s);
  }
  return check_launch(who);
}
