// Latent attention over packed chunks, expanded form (gfx950): every head has its own key and value,
// k_j = [kn_j | k_r_j] and v_j, where kn and v are the up-projected latent (one product of the caller,
// kv [tokens, H, 2 DN] = [kn | v]) and k_r the rotated part that all heads share:
//   s_ij = scale * (qn_i . kn_j + q_r_i . k_r_j),  p_i = softmax_j(s_ij),  o_i = sum_j p_ij v_j
// for the queries i and keys j of one sequence, causal and aligned to the last key (query i sees the
// keys j <= k_len - q_len + i). A first chunk has k_len = q_len, a continuation more keys than queries.
//
// Work unit: (sequence, head, 128 query rows), one workgroup of four waves of 32 rows. Keys come in tiles
// of 64, loaded straight into LDS one tile ahead and read by all waves:
//   S^T[64 keys x 32 rows]  = K[64 x (DN + 64)] . Q^T        (16x16x32, Q in registers)
//   O^T[DN x 32 rows]      += V^T[DN x 64] . P^T             (16x16x32, V by transposed reads)
// with an accumulator's row its lane's column, as in the paged prefill. Two workgroups fit a CU, so that
// one's softmax runs beside the other's products. The last query blocks, which see the most keys, come
// first; the blocks of one head follow each other at a distance of H, so with a multiple of 8 heads they
// share an XCD's L2.
#include "lds_tiles.h"

namespace ti {
namespace {

constexpr int kKeys = 64;      // keys of a tile
constexpr int kRows = 128;     // query rows of a workgroup
constexpr int kRope = 64;
constexpr float kSlack = 8.f;  // exp2 units a row maximum may rise before O is rescaled

struct ExpandedArgs {
  const uint16_t* q;  // [total_q, H, DN + 64]
  int64_t q_st, q_sh;
  const uint16_t* kv;  // [total_k, H, 2 DN]
  int64_t kv_st, kv_sh;
  const uint16_t* kr;  // [total_k, 64]
  int64_t kr_st;
  uint16_t* out;  // [total_q, H, DN]
  int64_t o_st, o_sh;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int32_t total_q, total_k, causal;
  float scale_log2;
};

// LDS places of 16-byte chunk c of row r: c ^ swz16(r) in rows of whole 256-byte blocks (kn and v),
// c ^ swz8(r) in the 128-byte rows of k_r. A ds_read_b128 serves rows {0-3, 12-15} of one chunk with rows
// {4-11} of its neighbour, a transposed read two neighbouring chunks of eight rows; either way these
// are 16 different bank quads.
__device__ __forceinline__ int swz16(int r) { return ((2 * r) & 15) ^ ((r & 8) ? 9 : 0); }
__device__ __forceinline__ int swz8(int r) {
  const int u = (r >> 1) & 7;
  return ((2 * u) & 7) ^ ((u & 4) ? 5 : 0);
}

template <int DN, typename Tag>
__global__ __launch_bounds__(256, 2) void latent_prefill_kernel(ExpandedArgs a) {
  constexpr int KN = DN / 32;               // k-steps of the unrotated part
  constexpr int NDT = DN / 16;
  constexpr int ROW = 2 * DN;               // elements of a [kn | v] row
  constexpr int CH = ROW / 8;
  constexpr int NKV = kKeys * CH / 256;     // loads of a wave and tile
  constexpr int NKR = kKeys * 8 / 256;
  constexpr int NL = NKV + NKR;
  constexpr int kStage = kKeys * (ROW + kRope);
  static_assert(CH % 16 == 0);
  __shared__ __align__(16) uint16_t s_tile[2 * kStage];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int h = blockIdx.x, b = blockIdx.z;

  // The sequence's extent, within the tensors whatever the offsets say.
  const int q0 = min(max(a.cu_q[b], 0), a.total_q);
  const int q_len = min(max(a.cu_q[b + 1], q0), a.total_q) - q0;
  const int k0 = min(max(a.cu_k[b], 0), a.total_k);
  const int k_len = min(max(a.cu_k[b + 1], k0), a.total_k) - k0;
  const int blocks = (q_len + kRows - 1) / kRows;
  if (int(blockIdx.y) >= blocks) return;
  const int qb0 = (blocks - 1 - int(blockIdx.y)) * kRows;
  const int rows = min(kRows, q_len - qb0);
  const int offset = k_len - q_len;  // query i sits at key position offset + i
  const int k_end = a.causal ? min(k_len, offset + qb0 + rows) : k_len;
  const int nt = k_end > 0 ? (k_end + kKeys - 1) / kKeys : 0;

  // Q operands of this wave's rows; rows behind the last repeat it and are not stored.
  u32x4 q[2][KN + 2];
  int limit[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int r = min(qb0 + wave * 32 + rt * 16 + n, q_len - 1);
    limit[rt] = a.causal ? offset + r : k_len - 1;
    const uint16_t* src = a.q + int64_t(q0 + r) * a.q_st + h * a.q_sh + 8 * g;
#pragma unroll
    for (int kk = 0; kk < KN + 2; ++kk) q[rt][kk] = load16(src + 32 * kk);
  }

  // Byte offsets of this lane's loads within a tile.
  uint32_t kv_at[NKV], kr_at[NKR];
#pragma unroll
  for (int i = 0; i < NKV; ++i) {
    const int f = (wave * NKV + i) * 64 + lane, r = f / CH;
    kv_at[i] = uint32_t(r) * uint32_t(a.kv_st * 2) + 16 * ((f % CH) ^ swz16(r));
  }
#pragma unroll
  for (int i = 0; i < NKR; ++i) {
    const int f = (wave * NKR + i) * 64 + lane, r = f >> 3;
    kr_at[i] = uint32_t(r) * uint32_t(a.kr_st * 2) + 16 * ((f & 7) ^ swz8(r));
  }
  auto issue = [&](int t, int stage) {
    const int valid = min(kKeys, k_end - t * kKeys);  // keys past it read as zero
    const uint16_t* kv = a.kv + int64_t(k0 + t * kKeys) * a.kv_st + h * a.kv_sh;
    const uint16_t* kr = a.kr + int64_t(k0 + t * kKeys) * a.kr_st;
    const u32x4 rkv = rsrc_words(kv, uint32_t(valid - 1) * uint32_t(a.kv_st * 2) + ROW * 2);
    const u32x4 rkr = rsrc_words(kr, uint32_t(valid - 1) * uint32_t(a.kr_st * 2) + kRope * 2);
    uint16_t* to = s_tile + stage * kStage;
#pragma unroll
    for (int i = 0; i < NKV; ++i) load_lds16(rkv, kv_at[i], to + (wave * NKV + i) * 512);
#pragma unroll
    for (int i = 0; i < NKR; ++i) load_lds16(rkr, kr_at[i], to + kKeys * ROW + (wave * NKR + i) * 512);
  };

  // Operand reads of row n (K) and of row 4 g + n / 4 (V), elements.
  int k_at[KN], r_at[2], v_at[NDT];
#pragma unroll
  for (int kk = 0; kk < KN; ++kk) k_at[kk] = n * ROW + 8 * ((4 * kk + g) ^ swz16(n));
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) r_at[kk] = kKeys * ROW + n * kRope + 8 * ((4 * kk + g) ^ swz8(n));
  {
    const int r = 4 * g + (n >> 2);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      v_at[dt] = r * ROW + 8 * ((DN / 8 + 2 * dt + ((lane >> 1) & 1)) ^ swz16(r)) + 4 * (lane & 1);
    }
  }

  f32x4 o[NDT][2];
  float m[2], l[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt][rt] = f32x4{};
  }
  // The rows this wave has, the keys its first and its last row see.
  const int wrow = qb0 + wave * 32;
  const int see_first = a.causal ? offset + wrow : k_len - 1;
  const int see_last = a.causal ? offset + min(wrow + 31, q_len - 1) : k_len - 1;
  const bool active = wrow < q_len;

  __builtin_amdgcn_s_waitcnt(0);  // q has landed: the loop below has waits of its own alone
  if (nt > 0) issue(0, 0);
  if (nt > 1) issue(1, 1);
  for (int t = 0; t < nt; ++t) {
    if (t + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(NL) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    const uint16_t* tile = s_tile + (t & 1) * kStage;
    if (active && t * kKeys <= see_last) {  // uniform
      f32x4 s[4][2];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        s[tt][0] = f32x4{};
        s[tt][1] = f32x4{};
      }
#pragma unroll
      for (int kk = 0; kk < KN + 2; ++kk) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const int at = kk < KN ? k_at[kk < KN ? kk : 0] + 16 * tt * ROW
                                 : r_at[kk < KN ? 0 : kk - KN] + 16 * tt * kRope;
          const u32x4 k = *reinterpret_cast<const u32x4*>(tile + at);
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) s[tt][rt] = mfma16x16x32(k, q[rt][kk], s[tt][rt], Tag{});
        }
      }
      const bool whole = t * kKeys + kKeys - 1 <= see_first && (t + 1) * kKeys <= k_end;
      u32x4 pb[2][2];
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = s[e >> 2][rt][e & 3] * a.scale_log2;
        if (!whole) {
          const int lim = min(limit[rt], k_end - 1) - t * kKeys - 4 * g;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (16 * (e >> 2) + (e & 3) > lim) x[e] = -INFINITY;
          }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 15; e += 2) top = max3(top, x[e], x[e + 1]);
        top = row_group_max(max2(top, x[15]));
        if (__builtin_amdgcn_ballot_w64(top > m[rt] + kSlack)) {  // m = -inf at first
          const float mn = fmaxf(m[rt], top);
          const float c = mn == -INFINITY ? 1.f : fast_exp2(m[rt] - mn);
          m[rt] = mn;
          l[rt] *= c;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt][rt] *= c;
        }
        const float base = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] = fast_exp2(x[e] - base);
          l[rt] += x[e];
        }
        // P is rounded to the inputs' type for the matrix unit, as in the paged prefill: at most half a
        // step of each weight, while l sums the unrounded ones in 32 bits.
#pragma unroll
        for (int e = 0; e < 8; ++e) pb[rt][e >> 2][e & 3] = pack2(x[2 * e], x[2 * e + 1], Tag{});
      }
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const uint16_t* at = tile + v_at[dt] + 32 * kp * ROW;
          const u32x2 lo = lds_read_tr4(at), hi = lds_read_tr4(at + 16 * ROW);
          const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) o[dt][rt] = mfma16x16x32(v, pb[rt][kp], o[dt][rt], Tag{});
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stage is read
    if (t + 2 < nt) issue(t + 2, t & 1);
  }
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int r = wrow + rt * 16 + n;
    const float lt = row_group_sum(l[rt]);
    if (r >= q_len) continue;
    const float inv = lt != 0.f ? 1.f / lt : 0.f;  // a row that sees nothing is zero
    uint16_t* dst = a.out + int64_t(q0 + r) * a.o_st + h * a.o_sh + 4 * g;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const f32x4 y = o[dt][rt] * inv;
      *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
    }
  }
}

bool vec_rows(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
}

}  // namespace
}  // namespace ti

extern "C" int ti_latent_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* kv,
                                 int64_t kv_stride_t, int64_t kv_stride_h, const void* key_rope,
                                 int64_t key_stride_t, const int32_t* cu_seqlens_q,
                                 const int32_t* cu_seqlens_k, void* out, int64_t out_stride_t,
                                 int64_t out_stride_h, int32_t batch, int32_t total_q, int32_t total_k,
                                 int32_t max_seqlen_q, int32_t num_heads, int32_t head_dim,
                                 int32_t rope_dim, int32_t causal, float scale, int32_t dtype,
                                 void* stream) {
  using namespace ti;
  const char* who = "ti_latent_prefill";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  if (head_dim != 128 && head_dim != 64) {
    return fail(TI_EUNSUPPORTED, "%s: head_dim %d not built (64, 128)", who, head_dim);
  }
  if (rope_dim != kRope) return fail(TI_EUNSUPPORTED, "%s: rope_dim %d not built (64)", who, rope_dim);
  if (batch < 0 || total_q < 0 || total_k < 0 || max_seqlen_q < 0 || num_heads <= 0 || batch > 65535 ||
      num_heads > 65535) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d total_q=%d total_k=%d max_seqlen_q=%d heads=%d", who, batch,
                total_q, total_k, max_seqlen_q, num_heads);
  }
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return TI_OK;
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || (total_k > 0 && (!kv || !key_rope))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (!vec_rows(q, q_stride_t, q_stride_h) || !vec_rows(kv, kv_stride_t, kv_stride_h) ||
      !vec_rows(key_rope, key_stride_t, 0) || !vec_rows(out, out_stride_t, out_stride_h)) {
    return fail(TI_EINVAL, "%s: rows must be 16-byte aligned", who);
  }
  // A tile's rows are reached by 32-bit offsets.
  if (kv_stride_t < 0 || key_stride_t < 0 || kv_stride_t >= (1 << 24) || key_stride_t >= (1 << 24)) {
    return fail(TI_EINVAL, "%s: token strides %lld, %lld of kv and key_rope must be in [0, 2^24)", who,
                static_cast<long long>(kv_stride_t), static_cast<long long>(key_stride_t));
  }
  ExpandedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.kv = static_cast<const uint16_t*>(kv);
  a.kv_st = kv_stride_t;
  a.kv_sh = kv_stride_h;
  a.kr = static_cast<const uint16_t*>(key_rope);
  a.kr_st = key_stride_t;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.total_q = total_q;
  a.total_k = total_k;
  a.causal = causal;
  a.scale_log2 = scale * 1.4426950408889634f;
  const int64_t longest = max_seqlen_q < total_q ? max_seqlen_q : total_q;
  const dim3 grid(unsigned(num_heads), unsigned(ceil_div(longest, kRows)), unsigned(batch));
  if (grid.y > 65535) return fail(TI_EINVAL, "%s: max_seqlen_q %d too long", who, max_seqlen_q);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == TI_DTYPE_BF16;
  if (head_dim == 128) {
    if (bf16) hipLaunchKernelGGL((latent_prefill_kernel<128, Bf16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((latent_prefill_kernel<128, F16>), grid, dim3(256), 0, s, a);
  } else {
    if (bf16) hipLaunchKernelGGL((latent_prefill_kernel<64, Bf16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((latent_prefill_kernel<64, F16>), grid, dim3(256), 0, s, a);
  }
  return check_launch(who);
}
