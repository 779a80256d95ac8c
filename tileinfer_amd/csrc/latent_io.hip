// The input side of a latent-attention layer in one launch (gfx950): for every token
//   row[slot] = [ c * rsqrt(mean c^2 + eps) * (offset + w) | rotate(k_r) ],   q_out = rotate(q_r)
// with c the latent (L values), k_r the key's rotated part that all heads share and q_r the queries'
// rotated part (64 values a head). Statistics, scale and rotation in 32 bits, each value rounded once to
// 16. The rotation pairs i with i + 32 and takes cos/sin[0 .. 32) of the token.
//
// Bound: HBM for long chunks (8,191 tokens with 24 heads 12.4 us, 5.7 TB/s), the launch for a decode step (33
// tokens 5.7 us). Every row is whole 16-byte vectors: a latent
// row is L / 8 lanes, a rotated row 8 lanes, so that a wave takes 64 / (L / 8) latent rows or 8 rotated
// ones (those of the key and of the heads are one list, token by token), and the partners of a rotation
// are 4 lanes apart.
#include "decode_common.h"

namespace ti {
namespace {

constexpr int kRope = 64;

struct LatentInArgs {
  const uint16_t* q;  // [T, H, 64] at q_st, q_sh; H may be 0
  int64_t q_st, q_sh;
  uint16_t* q_out;
  int64_t o_st, o_sh;
  const uint16_t* c;  // [T, L]
  int64_t c_st;
  const uint16_t* k;  // [T, 64]
  int64_t k_st;
  const uint16_t* w;  // [L]
  const uint16_t* cos;
  const uint16_t* sin;
  int64_t cs_st;
  uint16_t* cache;  // rows [num_slots][L + 64] at cache_row
  int64_t cache_row, num_slots;
  const int32_t* slots;
  int32_t tokens, heads;
  float offset, eps;
  int64_t latent_waves;  // waves that take latent rows, the others take rotated ones
};

template <int L, typename Tag>
__global__ __launch_bounds__(256) void latent_in_kernel(LatentInArgs a) {
  constexpr int LPR = L / 8;         // lanes of a latent row
  constexpr int ROWS = 64 / LPR;     // latent rows of a wave
  const int lane = threadIdx.x & 63;
  const int64_t wave = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave < a.latent_waves) {
    const int l = lane & (LPR - 1);
    const int64_t t = wave * ROWS + lane / LPR;
    const bool in = t < a.tokens;
    const u32x4 w = load16(a.w + 8 * l);
    const u32x4 x = in ? load16(a.c + t * a.c_st + 8 * l) : u32x4{};
    const int64_t slot = in ? a.slots[t] : -1;
    float v[8], ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = unpack2(x[j], Tag{});
      v[2 * j] = p.x;
      v[2 * j + 1] = p.y;
      ss = fmaf(p.x, p.x, fmaf(p.y, p.y, ss));
    }
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) ss += __shfl_xor(ss, d, 64);
    const float r = rsqrtf(ss / float(L) + a.eps);
    u32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = unpack2(w[j], Tag{});
      y[j] = pack_mul2(v[2 * j] * r, a.offset + p.x, v[2 * j + 1] * r, a.offset + p.y, Tag{});
    }
    if (slot >= 0 && slot < a.num_slots) {
      *reinterpret_cast<u32x4*>(a.cache + slot * a.cache_row + 8 * l) = y;
    }
    return;
  }
  // Rotated rows: token t's are its key (row 0) and its heads (rows 1 .. H).
  const int64_t item = (wave - a.latent_waves) * 8 + (lane >> 3);
  const int per = a.heads + 1;
  const int64_t t = item / per;
  const int h = int(item - t * per) - 1;
  const int l = lane & 7;
  const bool in = t < a.tokens;
  u32x4 x = {}, c = {}, s = {};
  uint16_t* dst = nullptr;
  if (in) {
    x = load16((h < 0 ? a.k + t * a.k_st : a.q + t * a.q_st + h * a.q_sh) + 8 * l);
    c = load16(a.cos + t * a.cs_st + 8 * (l & 3));
    s = load16(a.sin + t * a.cs_st + 8 * (l & 3));
    if (h >= 0) {
      dst = a.q_out + t * a.o_st + h * a.o_sh;
    } else {
      const int64_t slot = a.slots[t];
      if (slot >= 0 && slot < a.num_slots) dst = a.cache + slot * a.cache_row + L;
    }
  }
  const bool low = l < 4;
  u32x4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 own = unpack2(x[j], Tag{});
    const float2 other = unpack2(uint32_t(__shfl_xor(int(x[j]), 4, 64)), Tag{});
    const float2 cc = unpack2(c[j], Tag{}), sn = unpack2(s[j], Tag{});
    const float px = other.x * sn.x, py = other.y * sn.y;
    y[j] = pack_fma2(own.x, cc.x, low ? -px : px, own.y, cc.y, low ? -py : py, Tag{});
  }
  if (dst) *reinterpret_cast<u32x4*>(dst + 8 * l) = y;
}

// Pointers and strides of whole 16-byte vectors.
bool vec_rows(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
}

template <typename Tag>
void launch_latent_in(const LatentInArgs& a, int latent, unsigned blocks, hipStream_t s) {
  if (latent == 512) hipLaunchKernelGGL((latent_in_kernel<512, Tag>), dim3(blocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((latent_in_kernel<256, Tag>), dim3(blocks), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace ti

extern "C" int ti_latent_rope_append(const void* q_rope, int64_t q_stride_t, int64_t q_stride_h,
                                     void* q_out, int64_t out_stride_t, int64_t out_stride_h,
                                     const void* latent, int64_t latent_stride_t, const void* key_rope,
                                     int64_t key_stride_t, const void* weight, float weight_offset,
                                     const void* cos, const void* sin, int64_t cs_stride_t,
                                     void* latent_cache, int64_t cache_row_stride, int64_t num_slots,
                                     const int32_t* slot_mapping, int32_t n_tokens, int32_t num_heads,
                                     int32_t latent_dim, int32_t rope_dim, float eps, int32_t dtype,
                                     void* stream) {
  using namespace ti;
  const char* who = "ti_latent_rope_append";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  if (latent_dim != 512 && latent_dim != 256) {
    return fail(TI_EUNSUPPORTED, "%s: latent_dim %d not built (256, 512)", who, latent_dim);
  }
  if (rope_dim != kRope) return fail(TI_EUNSUPPORTED, "%s: rope_dim %d not built (64)", who, rope_dim);
  if (n_tokens < 0 || num_heads < 0 || num_slots < 0 || int64_t(n_tokens) * (num_heads + 1) > INT32_MAX) {
    return fail(TI_EINVAL, "%s: bad sizes tokens=%d heads=%d", who, n_tokens, num_heads);
  }
  if (n_tokens == 0) return TI_OK;
  if (!latent || !key_rope || !weight || !cos || !sin || !latent_cache || !slot_mapping ||
      (num_heads > 0 && (!q_rope || !q_out))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (cache_row_stride < latent_dim + kRope) {
    return fail(TI_EINVAL, "%s: cache rows of %d at stride %lld", who, latent_dim + kRope,
                static_cast<long long>(cache_row_stride));
  }
  if (!vec_rows(latent, latent_stride_t, 0) || !vec_rows(key_rope, key_stride_t, 0) ||
      !vec_rows(weight, 0, 0) || !vec_rows(cos, cs_stride_t, 0) || !vec_rows(sin, cs_stride_t, 0) ||
      !vec_rows(latent_cache, cache_row_stride, 0) ||
      (num_heads > 0 && (!vec_rows(q_rope, q_stride_t, q_stride_h) ||
                         !vec_rows(q_out, out_stride_t, out_stride_h)))) {
    return fail(TI_EINVAL, "%s: rows must be 16-byte aligned", who);
  }
  const int64_t latent_waves = ceil_div(n_tokens, 512 / latent_dim);
  const int64_t rope_waves = ceil_div(int64_t(n_tokens) * (num_heads + 1), 8);
  const int64_t blocks = ceil_div(latent_waves + rope_waves, 4);
  if (blocks > kMaxGridX) {
    return fail(TI_EINVAL, "%s: %d tokens of %d heads are more than one call takes", who, n_tokens, num_heads);
  }
  LatentInArgs a{};
  a.q = static_cast<const uint16_t*>(q_rope);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.c = static_cast<const uint16_t*>(latent);
  a.c_st = latent_stride_t;
  a.k = static_cast<const uint16_t*>(key_rope);
  a.k_st = key_stride_t;
  a.w = static_cast<const uint16_t*>(weight);
  a.cos = static_cast<const uint16_t*>(cos);
  a.sin = static_cast<const uint16_t*>(sin);
  a.cs_st = cs_stride_t;
  a.cache = static_cast<uint16_t*>(latent_cache);
  a.cache_row = cache_row_stride;
  a.num_slots = num_slots;
  a.slots = slot_mapping;
  a.tokens = n_tokens;
  a.heads = num_heads;
  a.offset = weight_offset;
  a.eps = eps;
  a.latent_waves = latent_waves;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == TI_DTYPE_BF16) launch_latent_in<Bf16>(a, latent_dim, unsigned(blocks), s);
  else launch_latent_in<F16>(a, latent_dim, unsigned(blocks), s);
  return check_launch(who);
}
