// The cache rows of accepted drafts, moved behind the context (gfx950): a sequence's last num_drafts tokens are a
// drafted tree; the path accepted[b] = a_0 < a_1 < ... of it becomes the sequence's next tokens, so that
//   row(C + j) = row(C + a_j),  C = seqlen[b] - num_drafts,  new_seqlen[b] = C + (number of accepted drafts)
// in every plane (a layer's keys or values) of the cache, in place.
//
// A path ascends, so a_j >= j and the moves go down: a thread owns 16 bytes of one plane's rows and takes the moves in
// order, eight loads before their eight stores (a store of this or a later group lands at or below the group's last j,
// which no later move reads: those have a_k >= k). Drafts that stay (a_j = j, always the path's first ones) cost
// nothing. Bound: the launch and a chain of four dependent loads (lengths and paths, block ids, rows) for small batches
// (four sequences, 32 planes of 4 x 256 values: 5.4 us), those and HBM for large ones (64 with 32 drafts 13 us, 4 TB/s).
#include "decode_common.h"

namespace ti {
namespace {

constexpr int kMaxDrafts = 64;  // a lane for each

struct KeepArgs {
  uint16_t* cache;  // [planes][num_blocks * page_size] rows of `row` elements
  int64_t plane, row;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seqlen;
  const int32_t* accepted;  // [B, width] at acc_stride
  int64_t acc_stride;
  int32_t* new_seqlen;
  int32_t drafts, width, page_size, num_blocks32, max_blocks, blocks_per_seq, planes;
};

__global__ __launch_bounds__(256) void keep_drafts_kernel(KeepArgs a) {
  const int lane = threadIdx.x & 63;
  const int b = int(blockIdx.x / unsigned(a.blocks_per_seq));
  const int part = int(blockIdx.x - unsigned(b) * unsigned(a.blocks_per_seq));
  const int len = a.seqlen[b], context = len - a.drafts;
  const int id = lane < a.width ? a.accepted[b * a.acc_stride + lane] : -1;
  const int before = __shfl_up(id, 1, 64);
  const bool good = id >= 0 && id < a.drafts && (lane == 0 || id > before);
  const uint64_t bad = ~__builtin_amdgcn_ballot_w64(good);
  const int count = bad ? __builtin_ctzll(bad) : 64;
  if (part == 0 && threadIdx.x == 0) a.new_seqlen[b] = context < 0 ? len : context + count;
  if (context < 0) return;
  const uint64_t moved = __builtin_amdgcn_ballot_w64(good && lane < count && id != lane);
  if (moved == 0) return;
  const int first = __builtin_ctzll(moved);
  auto row_at = [&](int64_t pos) {  // -1: no such row
    if (pos >= int64_t(a.max_blocks) * a.page_size) return -1;
    const int block = a.block_table[b * a.bt_stride + pos / a.page_size];
    return uint32_t(block) < uint32_t(a.num_blocks32) ? int(block * a.page_size + pos % a.page_size) : -1;
  };
  int from = -1, to = -1;
  if (lane >= first && lane < count) {
    from = row_at(int64_t(context) + id);
    to = row_at(int64_t(context) + lane);
  }
  const int64_t cols = a.row / 8, all = cols * a.planes;
  const int64_t item = int64_t(part) * 256 + threadIdx.x;
  const bool live = item < all;
  const int64_t plane = live ? item / cols : 0, col = live ? item - plane * cols : 0;
  uint16_t* const base = a.cache + plane * a.plane + col * 8;
  for (int j = first; j < count; j += 8) {
    u32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = min(j + i, 63);
      const int src = __builtin_amdgcn_readlane(from, k);
      if (live && j + i < count && src >= 0) x[i] = load16(base + src * a.row);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = min(j + i, 63);
      const int src = __builtin_amdgcn_readlane(from, k), dst = __builtin_amdgcn_readlane(to, k);
      if (live && j + i < count && src >= 0 && dst >= 0) *reinterpret_cast<u32x4*>(base + dst * a.row) = x[i];
    }
  }
}

}  // namespace
}  // namespace ti

extern "C" int ti_keep_drafts(void* cache, const int32_t* block_table, int64_t block_table_stride,
                              const int32_t* seqlen, const int32_t* accepted, int64_t accepted_stride,
                              int32_t* new_seqlen, int32_t batch, int32_t num_drafts, int32_t accepted_width,
                              int32_t planes, int64_t row_elems, int32_t page_size, int64_t num_blocks,
                              int32_t max_blocks_per_seq, void* stream) {
  using namespace ti;
  const char* who = "ti_keep_drafts";
  if (num_drafts < 1 || num_drafts > kMaxDrafts) {
    return fail(TI_EUNSUPPORTED, "%s: num_drafts %d not in 1 .. %d", who, num_drafts, kMaxDrafts);
  }
  if (batch < 0 || accepted_width < 0 || planes < 0 || row_elems <= 0 || row_elems > INT32_MAX || row_elems % 8 != 0 ||
      page_size <= 0 || num_blocks < 0 || num_blocks > INT32_MAX / page_size || max_blocks_per_seq < 0 ||
      int64_t(max_blocks_per_seq) * page_size > INT32_MAX) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d width=%d planes=%d row_elems=%lld page_size=%d num_blocks=%lld "
                "max_blocks_per_seq=%d (rows of a multiple of 8 values, at most 2^31 - 1 of them)", who, batch,
                accepted_width, planes, static_cast<long long>(row_elems), page_size, static_cast<long long>(num_blocks),
                max_blocks_per_seq);
  }
  const int64_t threads = row_elems / 8 * planes;
  const int64_t per_seq = planes == 0 ? 1 : ceil_div(threads, 256);
  if (per_seq > kMaxGridX || per_seq * batch > kMaxGridX) {
    return fail(TI_EINVAL, "%s: batch %d x planes %d x %lld values is more than one call takes", who, batch, planes,
                static_cast<long long>(row_elems));
  }
  if (batch == 0) return TI_OK;
  if (!seqlen || !new_seqlen || (accepted_width > 0 && !accepted) ||
      (planes > 0 && num_blocks > 0 && !cache) || (max_blocks_per_seq > 0 && !block_table)) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (reinterpret_cast<uintptr_t>(cache) & 15) return fail(TI_EINVAL, "%s: cache must be 16-byte aligned", who);
  // A sequence's workgroups read its length while the first of them stores the new one.
  const uintptr_t old_at = reinterpret_cast<uintptr_t>(seqlen), new_at = reinterpret_cast<uintptr_t>(new_seqlen);
  if (old_at < new_at + 4 * uintptr_t(batch) && new_at < old_at + 4 * uintptr_t(batch)) {
    return fail(TI_EINVAL, "%s: new_seqlen and seqlen overlap", who);
  }
  KeepArgs a{};
  a.cache = static_cast<uint16_t*>(cache);
  a.plane = num_blocks * page_size * row_elems;
  a.row = row_elems;
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.seqlen = seqlen;
  a.accepted = accepted;
  a.acc_stride = accepted_stride;
  a.new_seqlen = new_seqlen;
  a.drafts = num_drafts;
  a.width = accepted_width < kMaxDrafts ? accepted_width : kMaxDrafts;
  a.page_size = page_size;
  a.num_blocks32 = int32_t(num_blocks);
  a.max_blocks = max_blocks_per_seq;
  a.blocks_per_seq = int32_t(per_seq);
  a.planes = planes;
  hipLaunchKernelGGL(keep_drafts_kernel, dim3(unsigned(per_seq * batch)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch(who);
}
