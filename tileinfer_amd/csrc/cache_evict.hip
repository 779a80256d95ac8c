// Cutting a paged cache to its heaviest tokens (gfx950). For every (sequence, KV head) of n tokens:
//   keep all of them if n <= budget, else the `budget` tokens that rank first, where the first `sinks` and
//   the last `recent` tokens rank before all others and those by their mass, ties to the lowest position;
//   kept[j] = the kept positions in ascending order, mass_out[j] = mass[kept[j]],
//   and the head's K (and V) row of token kept[j] is copied to slot j of the sequence's new block table.
// Heads of one sequence keep different tokens, all the same number. A bit copy; no arithmetic on values.
//
// Selection (one workgroup per (sequence, KV head)): masses become unsigned keys of the same order, the
// budget-th largest key is found digit by digit (11, 11 and 10 bits, a histogram in LDS each), then each
// wave walks a contiguous range of positions and numbers the kept ones by ballots, so the order is the
// positions'. Bound: the latency of four passes over the masses, which stay in L2 after the first.
// Copy: every 16-byte vector of the new rows by one lane. Bound: HBM.
#include "decode_common.h"

namespace ti {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;

struct EvictArgs {
  uint16_t* k_cache;  // rows [num_blocks * page_size][hkv][D]
  uint16_t* v_cache;  // the same, or nullptr
  const float* mass;  // [B, hkv, capacity] at m_sb, m_sh
  int64_t m_sb, m_sh;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* new_table;
  int64_t nt_stride;
  const int32_t* seqlen;
  int32_t* kept;        // [B, hkv, budget], -1 behind the last
  int32_t* new_seqlen;  // [B]
  float* mass_out;      // [B, hkv, capacity], 0 behind the last
  int32_t hkv, head_dim, num_blocks32, page_size, max_blocks, budget, sinks, recent;
  int64_t capacity;
};

__device__ __forceinline__ int evict_len(const EvictArgs& a, int b) {
  const int64_t cap = min(int64_t(a.max_blocks) * a.page_size, a.capacity);
  const int n = max(a.seqlen[b], 0);
  return int64_t(n) > cap ? int(cap) : n;
}

// Unsigned keys in the order of the ranks: tokens always kept first, then by mass (-0 as 0), NaN last.
__device__ __forceinline__ uint32_t rank_key(const EvictArgs& a, const float* mass, int t, int n) {
  if (t < a.sinks || t >= n - a.recent) return 0xffffffffu;
  const float x = mass[t] + 0.f;
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ int s_hist[kBins];
  __shared__ int s_wave[kWaves][2];
  __shared__ int s_found[2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = evict_len(a, b);
  const int keep = min(n, a.budget);
  const int64_t row = int64_t(b) * a.hkv + h;
  const float* mass = a.mass + b * a.m_sb + h * a.m_sh;
  int32_t* kept = a.kept + row * a.budget;
  float* out = a.mass_out + row * a.capacity;
  if (h == 0 && threadIdx.x == 0) a.new_seqlen[b] = keep;
  for (int j = keep + int(threadIdx.x); j < a.budget; j += kThreads) kept[j] = -1;
  for (int64_t j = keep + int64_t(threadIdx.x); j < a.capacity; j += kThreads) out[j] = 0.f;
  if (keep == n) {
    for (int t = threadIdx.x; t < n; t += kThreads) {
      kept[t] = t;
      out[t] = mass[t];
    }
    return;
  }
  // The keep-th largest key: `prefix` is its digits so far, `need` how many of the keys with that prefix
  // (and the digits to come) are still to be kept.
  uint32_t prefix = 0, fixed = 0;
  int need = keep;
  for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {
    const uint32_t bins = shift == 0 ? 1024 : 2048;
    // shifts 21, 10, 0: digits of 11, 11 and 10 bits
    for (int i = threadIdx.x; i < kBins; i += kThreads) s_hist[i] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < n; t += kThreads) {
      const uint32_t key = rank_key(a, mass, t, n);
      if ((key & fixed) == prefix) atomicAdd(&s_hist[(key >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // Bins from the greatest: thread i holds bins 2 i and 2 i + 1 of that order.
    const int hi = s_hist[kBins - 1 - 2 * int(threadIdx.x)], lo = s_hist[kBins - 2 - 2 * int(threadIdx.x)];
    int incl = hi + lo;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(incl, d, 64);
      if (lane >= d) incl += y;
    }
    if (lane == 63) s_wave[wave][0] = incl;
    __syncthreads();
    int before = incl - hi - lo;
    for (int w = 0; w < wave; ++w) before += s_wave[w][0];
    if (before < need && need <= before + hi) {
      s_found[0] = kBins - 1 - 2 * int(threadIdx.x);
      s_found[1] = need - before;
    } else if (before + hi < need && need <= before + hi + lo) {
      s_found[0] = kBins - 2 - 2 * int(threadIdx.x);
      s_found[1] = need - before - hi;
    }
    __syncthreads();
    prefix |= uint32_t(s_found[0]) << shift;
    fixed |= (bins - 1) << shift;
    need = s_found[1];
    if (shift == 0) break;
  }
  // Kept: keys above `prefix`, and the first `need` that equal it. Each wave numbers a contiguous range.
  const int per = ((n + kWaves - 1) / kWaves + 63) & ~63;
  const int w0 = min(n, wave * per), w1 = min(n, w0 + per);
  int above = 0, equal = 0;
  for (int t0 = w0; t0 < w1; t0 += 64) {
    const int t = t0 + lane;
    const uint32_t key = t < w1 ? rank_key(a, mass, t, n) : 0u;
    above += __popcll(__builtin_amdgcn_ballot_w64(t < w1 && key > prefix));
    equal += __popcll(__builtin_amdgcn_ballot_w64(t < w1 && key == prefix));
  }
  __syncthreads();  // s_wave is read
  if (lane == 0) {
    s_wave[wave][0] = above;
    s_wave[wave][1] = equal;
  }
  __syncthreads();
  int seen_above = 0, seen_equal = 0;
  for (int w = 0; w < wave; ++w) {
    seen_above += s_wave[w][0];
    seen_equal += s_wave[w][1];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  for (int t0 = w0; t0 < w1; t0 += 64) {
    const int t = t0 + lane;
    const uint32_t key = t < w1 ? rank_key(a, mass, t, n) : 0u;
    const bool is_above = t < w1 && key > prefix, is_equal = t < w1 && key == prefix;
    const uint64_t ma = __builtin_amdgcn_ballot_w64(is_above), me = __builtin_amdgcn_ballot_w64(is_equal);
    const int eq = seen_equal + __popcll(me & below);
    if (is_above || (is_equal && eq < need)) {
      const int j = seen_above + __popcll(ma & below) + min(eq, need);
      kept[j] = t;
      out[j] = mass[t];
    }
    seen_above += __popcll(ma);
    seen_equal += __popcll(me);
  }
}

// Vectors [16 bytes] of the kept rows of one (sequence, KV head), a grid of them.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int keep = min(evict_len(a, b), a.budget);
  const int vecs = a.head_dim / 8;
  const int64_t row = int64_t(b) * a.hkv + h;
  const int64_t total = int64_t(keep) * vecs;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int j = int(i / vecs), c = int(i - int64_t(j) * vecs);
    const int t = a.kept[row * a.budget + j];
    const int from = a.block_table[b * a.bt_stride + t / a.page_size];
    const int into = a.new_table[b * a.nt_stride + j / a.page_size];
    if (uint32_t(from) >= uint32_t(a.num_blocks32) || uint32_t(into) >= uint32_t(a.num_blocks32)) continue;
    const int64_t s = ((int64_t(from) * a.page_size + t % a.page_size) * a.hkv + h) * a.head_dim + 8 * c;
    const int64_t d = ((int64_t(into) * a.page_size + j % a.page_size) * a.hkv + h) * a.head_dim + 8 * c;
    *reinterpret_cast<u32x4*>(a.k_cache + d) = load16(a.k_cache + s);
    if (a.v_cache) *reinterpret_cast<u32x4*>(a.v_cache + d) = load16(a.v_cache + s);
  }
}

}  // namespace
}  // namespace ti

extern "C" int ti_evict_kvcache(void* k_cache, void* v_cache, const float* mass, int64_t mass_stride_b,
                                int64_t mass_stride_h, int64_t mass_capacity, const int32_t* block_table,
                                int64_t block_table_stride, const int32_t* seqlen,
                                const int32_t* new_block_table, int64_t new_table_stride, int32_t* kept,
                                int32_t* new_seqlen, float* mass_out, int32_t batch, int32_t num_kv_heads,
                                int32_t head_dim, int32_t page_size, int64_t num_blocks,
                                int32_t max_blocks_per_seq, int32_t new_blocks_per_seq, int32_t budget,
                                int32_t sinks, int32_t recent, int32_t dtype, void* stream) {
  using namespace ti;
  const char* who = "ti_evict_kvcache";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  if (batch < 0 || batch > 65535 || num_kv_heads <= 0 || num_kv_heads > 65535 || head_dim <= 0 ||
      head_dim % 8 != 0 || head_dim > (1 << 16) || page_size <= 0 || num_blocks < 0 || num_blocks > INT32_MAX ||
      max_blocks_per_seq < 0 || new_blocks_per_seq < 0) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d num_kv_heads=%d head_dim=%d page_size=%d (head_dim a "
                "multiple of 8)", who, batch, num_kv_heads, head_dim, page_size);
  }
  if (budget <= 0 || sinks < 0 || recent < 0 || int64_t(sinks) + recent > budget) {
    return fail(TI_EINVAL, "%s: budget %d must be positive and hold sinks %d and recent %d", who, budget, sinks,
                recent);
  }
  const int64_t tokens = int64_t(max_blocks_per_seq) * page_size;
  if (tokens > INT32_MAX - 1024 || int64_t(batch) * num_kv_heads * budget > (int64_t(1) << 40)) {
    return fail(TI_EINVAL, "%s: max_blocks_per_seq %d x page_size %d exceeds 2^31", who, max_blocks_per_seq,
                page_size);
  }
  if (mass_capacity < tokens || mass_stride_h < mass_capacity || mass_stride_b < 0) {
    return fail(TI_EINVAL, "%s: mass rows of %lld floats for sequences of up to %lld tokens", who,
                static_cast<long long>(mass_capacity), static_cast<long long>(tokens));
  }
  const int64_t most = tokens < budget ? tokens : budget;
  if (int64_t(new_blocks_per_seq) * page_size < most) {
    return fail(TI_EINVAL, "%s: the new table's %d blocks hold fewer than %lld tokens", who, new_blocks_per_seq,
                static_cast<long long>(most));
  }
  if (batch == 0) return TI_OK;
  if (!seqlen || !kept || !new_seqlen || (mass_capacity > 0 && (!mass || !mass_out)) ||
      (tokens > 0 && (!k_cache || !block_table || !new_block_table))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) != 0) {
    return fail(TI_EINVAL, "%s: caches must be 16-byte aligned", who);
  }
  EvictArgs a{};
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.mass = mass;
  a.m_sb = mass_stride_b;
  a.m_sh = mass_stride_h;
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.new_table = new_block_table;
  a.nt_stride = new_table_stride;
  a.seqlen = seqlen;
  a.kept = kept;
  a.new_seqlen = new_seqlen;
  a.mass_out = mass_out;
  a.hkv = num_kv_heads;
  a.head_dim = head_dim;
  a.num_blocks32 = int32_t(num_blocks);
  a.page_size = page_size;
  a.max_blocks = max_blocks_per_seq;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.capacity = mass_capacity;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3(unsigned(num_kv_heads), unsigned(batch)), dim3(kThreads), 0, s, a);
  if (most > 0) {
    const int64_t blocks = ceil_div(most * (head_dim / 8), 256);
    const dim3 grid(unsigned(blocks < 4096 ? blocks : 4096), unsigned(num_kv_heads), unsigned(batch));
    hipLaunchKernelGGL(evict_copy_kernel, grid, dim3(256), 0, s, a);
  }
  return check_launch(who);
}
