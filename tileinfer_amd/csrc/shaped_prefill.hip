// Paged prefill with shaped scores (gfx950): the queries of a sequence's chunk over its cached tokens, the chunk's own
// among them, straight from the pages. Query i at position p_i = seqlen - q_len + i sees the keys
//   first_i <= j <= last_i, p_i - j < window
// (documents: first_i the first token of its document; a prefix or an image attended both ways: last_i its end; without
// the arrays 0 and p_i), with the scores
//   s_ij = cap tanh(scale q_i . k_j / cap) - slope_h |p_i - j|
// The kernel is that of shaped_rows.h, a workgroup for 128 rows of a (sequence, KV head); here are its launch shapes.
#include "shaped_rows.h"

namespace ti {
namespace {

bool vec_rows(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
}

struct ShapedSizes {
  int32_t blocks, splits, slots;
  int64_t units, whole, o_floats, ml_floats, bytes;
};

// How units are cut. A CU holds one workgroup at D = 256, two at 128 (slots). Where the units do not fill the slots, all
// are cut into as many parts as fill them; where they fill them some times over and the units of a chunk are alike
// (one sequence, at least as much context as chunk), those of the last, partial round are. Parts have at least four
// tiles, and only units that exist have them: at most as many as fill the slots, 34 MB. Cut against whole, 24/4 heads of
// 256, capped: 64 queries over 8,256 keys 45 us against 277; 2,048 over 10,240, whose last round is cut, 553 against 641,
// in a window of 4,096 276 against 317; but the last round of a first chunk of 2,048, its shortest units, 99 against 86.
ShapedSizes shaped_sizes(int32_t batch, int32_t total_q, int32_t max_q, int32_t hq, int32_t hkv, int32_t head_dim,
                         int64_t max_k) {
  ShapedSizes z{};
  const int64_t group = hq / hkv, longest = max_q < total_q ? max_q : total_q;
  z.blocks = int32_t(ceil_div(longest * group, kRows));
  z.units = int64_t(batch) * z.blocks * hkv;
  z.whole = z.units;
  z.splits = 1;
  const int64_t slots = int64_t(device_cu_count()) * (head_dim == 256 ? 1 : 2), most = max_k / (4 * kKeys);
  const int64_t real = batch == 1 ? z.units : hkv * (ceil_div(total_q * group, kRows) + batch - 1);
  int64_t cut = 0;  // units to cut
  if (real < slots) cut = z.units;
  else if (batch == 1 && max_k >= 2 * longest) cut = z.units % slots;
  if (cut > 0) {
    int64_t splits = slots / (cut == z.units ? real : cut);
    splits = splits > most ? most : splits;
    splits = splits > kMaxParts ? kMaxParts : splits;
    // A padded batch's workgroups: 16,384 of head_dim 128, 8,192 of 256, most of which have no rows to take.
    if (splits > 1 && cut * splits * kRows * head_dim <= int64_t(1) << 28) {
      z.whole = z.units - cut;
      z.splits = int32_t(splits);
      z.slots = int32_t(cut == z.units && real < cut ? real : cut);
      const int64_t rows = z.slots * splits * kRows;
      z.o_floats = rows * head_dim;
      z.ml_floats = rows * 2;
      z.bytes = (z.o_floats + z.ml_floats) * 4;
    }
  }
  return z;
}

int check_shaped(const char* who, int32_t batch, int32_t total_q, int32_t max_q, int32_t hq, int32_t hkv,
                 int32_t head_dim, int64_t max_k) {
  if (head_dim != 128 && head_dim != 256) {
    return fail(TI_EUNSUPPORTED, "%s: head_dim %d not built (128, 256)", who, head_dim);
  }
  if (batch < 0 || batch > 65535 || total_q < 0 || max_q < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || hq > 65535 ||
      max_k < 0 || int64_t(total_q) * (hq / hkv) > INT32_MAX - 2 * kRows) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d total_q=%d max_seqlen_q=%d heads=%d/%d (at most 65535 sequences and "
                "heads, 2^31 rows a KV head)", who, batch, total_q, max_q, hq, hkv);
  }
  return TI_OK;
}

}  // namespace
}  // namespace ti

extern "C" int ti_gqa_prefill_shaped_workspace_bytes(int32_t batch, int32_t total_q, int32_t max_seqlen_q,
                                                     int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                     int64_t max_seqlen_k, int64_t* workspace_bytes_out) {
  using namespace ti;
  const char* who = "ti_gqa_prefill_shaped_workspace_bytes";
  const int rc = check_shaped(who, batch, total_q, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, max_seqlen_k);
  if (rc != TI_OK) return rc;
  if (!workspace_bytes_out) return fail(TI_EINVAL, "%s: null output", who);
  const bool none = batch == 0 || total_q == 0 || max_seqlen_q == 0;
  *workspace_bytes_out = none ? 0 : shaped_sizes(batch, total_q, max_seqlen_q, num_q_heads, num_kv_heads, head_dim,
                                                 max_seqlen_k).bytes;
  return TI_OK;
}

extern "C" int ti_gqa_prefill_shaped(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                                     const void* v_cache, const int32_t* block_table, int64_t block_table_stride,
                                     const int32_t* cu_seqlens_q, const int32_t* seqlen_k, const int32_t* first_key,
                                     const int32_t* last_key, const float* slopes, void* out, int64_t out_stride_t,
                                     int64_t out_stride_h, void* workspace, int64_t workspace_bytes, int32_t batch,
                                     int32_t total_q, int32_t max_seqlen_q, int32_t num_q_heads, int32_t num_kv_heads,
                                     int32_t head_dim, int32_t page_size, int64_t num_blocks,
                                     int32_t max_blocks_per_seq, int64_t max_seqlen_k, int32_t causal, float scale,
                                     float softcap, int32_t window, int32_t dtype, void* stream) {
  using namespace ti;
  const char* who = "ti_gqa_prefill_shaped";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  const int rc = check_shaped(who, batch, total_q, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, max_seqlen_k);
  if (rc != TI_OK) return rc;
  if (!shape_ok(scale, softcap)) {
    return fail(TI_EINVAL, "%s: scale %g must be positive, at most 1e30, softcap %g zero (none) or 1e-3 to 1e4", who,
                double(scale), double(softcap));
  }
  if (window < 0) return fail(TI_EINVAL, "%s: window %d is negative", who, window);
  if (page_size <= 0 || num_blocks < 0 || max_blocks_per_seq < 0 || num_blocks > INT32_MAX / page_size) {
    return fail(TI_EINVAL, "%s: bad cache page_size=%d num_blocks=%lld max_blocks_per_seq=%d (at most "
                "2^31 - 1 rows)", who, page_size, static_cast<long long>(num_blocks), max_blocks_per_seq);
  }
  const int64_t tokens = int64_t(max_blocks_per_seq) * page_size;
  if (tokens > INT32_MAX - 1024) {  // tiles ahead of the last one are counted too
    return fail(TI_EINVAL, "%s: max_blocks_per_seq %d x page_size %d exceeds 2^31", who, max_blocks_per_seq, page_size);
  }
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return TI_OK;
  if (!q || !out || !cu_seqlens_q || !seqlen_k || (max_blocks_per_seq > 0 && (!k_cache || !v_cache || !block_table))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (!vec_rows(q, q_stride_t, q_stride_h) || !vec_rows(out, out_stride_t, out_stride_h) || !vec_rows(k_cache, 0, 0) ||
      !vec_rows(v_cache, 0, 0)) {
    return fail(TI_EINVAL, "%s: rows must be 16-byte aligned", who);
  }
  ShapedSizes z = shaped_sizes(batch, total_q, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, max_seqlen_k);
  if (!workspace) {
    z.splits = 1;
    z.whole = z.units;
  } else if (z.bytes > 0 && (workspace_bytes < z.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    return fail(TI_EINVAL, "%s: workspace %lld < %lld bytes, or not 16-byte aligned", who,
                static_cast<long long>(workspace_bytes), static_cast<long long>(z.bytes));
  }
  if (z.whole + (z.units - z.whole) * (z.splits > kRows / 16 ? z.splits : kRows / 16) > kMaxGridX / 2) {
    return fail(TI_EINVAL, "%s: batch %d x max_seqlen_q %d x heads %d/%d is more than one call takes", who, batch,
                max_seqlen_q, num_q_heads, num_kv_heads);
  }
  RowsArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_cache = static_cast<const uint16_t*>(k_cache);
  a.v_cache = static_cast<const uint16_t*>(v_cache);
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.cu_q = cu_seqlens_q;
  a.seqlen = seqlen_k;
  a.first_key = first_key;
  a.last_key = last_key;
  a.slopes = slopes;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + z.o_floats;
  a.units = int32_t(z.units);
  a.whole = int32_t(z.whole);
  a.total_q = total_q;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.blocks = z.blocks;
  a.splits = z.splits;
  a.slots = z.slots;
  a.num_blocks32 = int32_t(num_blocks);
  set_page(a, page_size);
  a.max_blocks = max_blocks_per_seq;
  a.causal = causal;
  a.window = window > tokens + int64_t(total_q) ? 0 : window;  // wider than any distance
  a.shape = score_shape(scale, softcap);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == TI_DTYPE_BF16;
  if (head_dim == 256) {
    if (bf16) launch_rows<256, false, Bf16>(a, s);
    else launch_rows<256, false, F16>(a, s);
  } else {
    if (bf16) launch_rows<128, false, Bf16>(a, s);
    else launch_rows<128, false, F16>(a, s);
  }
  return check_launch(who);
}
