// Cutting a paged cache to its heaviest tokens (gfx950). For every (sequence, KV head) of n tokens:
//   keep all of them if n <= budget, else the `budget` tokens that rank first, where the first `sinks` and
//   the last `recent` tokens rank before all others and those by their mass, ties to the lowest position;
//   kept[j] = the kept positions in ascending order, mass_out[j] = mass[kept[j]],
//   and the head's K (and V) row of token kept[j] is copied to slot j of the sequence's new block table.
// Heads of one sequence keep different tokens, all the same number. A bit copy; no arithmetic on values.
//
// Selection (one workgroup per (sequence, KV head)): masses become unsigned keys of the same order, held in
// registers (up to 32,768 tokens; longer sequences read theirs again for every pass), the budget-th largest
// key is found digit by digit (11, 11 and 10 bits, a histogram in LDS each), then each wave walks a
// contiguous range of positions and numbers the kept ones by ballots, so the order is the positions'. Summed
// weights have few exponents and many zeros, so a histogram has four copies of each bin, for lanes of
// different remainders. Bound: the issue of its passes on one CU, and their barriers (11 us for one head of 6,001
// tokens, 21 us for 32 of up to 32,768).
// Copy: every 16-byte vector of the new rows by one lane, and the kept masses (read back by the selection they
// were one load after the other: 4 us at 32,768 tokens). Bound: HBM (48 us, 5.6 TB/s, for 8 x 4 heads of 4,096
// kept tokens of 256 dimensions).
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
  int32_t hkv, head_dim, num_blocks32, page_size, page_shift, max_blocks, budget, sinks, recent;
  int64_t capacity;
};

__device__ __forceinline__ int evict_len(const EvictArgs& a, int b) {
  const int64_t cap = min(int64_t(a.max_blocks) * a.page_size, a.capacity);
  const int n = max(a.seqlen[b], 0);
  return int64_t(n) > cap ? int(cap) : n;
}

// Unsigned keys in the order of the ranks: tokens always kept first, then by mass (-0 as 0), NaN last. Zero is
// none of them: it stands for no token.
__device__ __forceinline__ uint32_t rank_key(const EvictArgs& a, float mass, int t, int n) {
  const float x = mass + 0.f;
  const uint32_t u = __float_as_uint(x);
  const uint32_t key = x != x ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
  return t < a.sinks || t >= n - a.recent ? 0xffffffffu : key;
}

constexpr int kCopies = 4;   // of every bin
constexpr int kHeld = 32;    // keys that a thread holds in registers,
constexpr int kGroup = 4;    // in groups that a wave takes or leaves
typedef int i32x4 __attribute__((ext_vector_type(4)));
static_assert(kCopies == 4 && kBins == 2 * kThreads);

// Sum over the waves before this one.
__device__ __forceinline__ int before_wave(const i32x4* of_waves, int wave) {
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kWaves / 4; ++k) {
    const i32x4 v = of_waves[k];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += 4 * k + e < wave ? v[e] : 0;
  }
  return sum;
}

template <bool HELD>
__global__ __launch_bounds__(kThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ i32x4 s_hist[kBins];
  __shared__ i32x4 s_wave[2][kWaves / 4];
  __shared__ int s_found[2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = evict_len(a, b);
  const int keep = min(n, a.budget);
  const int64_t row = int64_t(b) * a.hkv + h;
  const float* mass = a.mass + b * a.m_sb + h * a.m_sh;
  int32_t* kept = a.kept + row * a.budget;
  if (h == 0 && threadIdx.x == 0) a.new_seqlen[b] = keep;
  if (HELD ? n > kHeld * kThreads : n <= kHeld * kThreads) return;  // the other form's
  if (keep == n) {
    for (int t = threadIdx.x; t < n; t += kThreads) kept[t] = t;
    return;
  }
  // Wave w's tokens are [w per, (w + 1) per), 64 a round.
  const int per = ((n + kWaves - 1) / kWaves + 63) & ~63;
  const int w0 = min(n, wave * per), w1 = min(n, w0 + per);
  const int rounds = (w1 - w0 + 63) >> 6;
  uint32_t keys[HELD ? kHeld : 1];
  // f(group) for the groups of rounds that the wave has. Whole groups: a condition for every round becomes part of
  // that round's lane mask, and all 32 are issued (6,001 tokens: 14.4 us of selection against 10.6).
  auto groups = [&](auto f) __attribute__((always_inline)) {
    int here = rounds;
    asm volatile("" : "+s"(here));  // compared anew: conditions kept from pass to pass do not fit the registers
#pragma unroll
    for (int i0 = 0; i0 < kHeld; i0 += kGroup) {
      if (i0 < here) f(i0);
    }
  };
  if constexpr (HELD) {
    groups([&](int i0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = i0; i < i0 + kGroup; ++i) keys[i] = __float_as_uint(mass[min(w0 + 64 * i + lane, n - 1)]);
    });  // all of them in flight
    groups([&](int i0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = i0; i < i0 + kGroup; ++i) {
        const int t = w0 + 64 * i + lane;
        keys[i] = t < w1 ? rank_key(a, __uint_as_float(keys[i]), t, n) : 0u;
      }
    });
  }
  // f(round, key) for the wave's tokens; lanes behind its last one have key 0.
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (HELD) {
      groups([&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = i0; i < i0 + kGroup; ++i) f(i, keys[i]);
      });
    } else {
      for (int i = 0; i < rounds; ++i) {
        const int t = w0 + 64 * i + lane;
        f(i, t < w1 ? rank_key(a, mass[min(t, n - 1)], t, n) : 0u);
      }
    }
  };
  s_hist[threadIdx.x] = i32x4{};
  s_hist[kThreads + threadIdx.x] = i32x4{};
  __syncthreads();
  // The keep-th largest key: `prefix` is its digits so far, `need` how many of the keys with that prefix
  // (and the digits to come) are still to be kept. Digits of 11, 11 and 10 bits.
  uint32_t prefix = 0, fixed = 0;
  int need = keep;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    int* const copy = reinterpret_cast<int*>(s_hist) + (lane & (kCopies - 1));
    each([&](int, uint32_t key) {
      if (key != 0 && (key & fixed) == prefix) atomicAdd(copy + ((key >> shift) & mask) * kCopies, 1);
    });
    __syncthreads();
    // Bins from the greatest: thread i holds bins 2 i and 2 i + 1 of that order, and clears them.
    i32x4* const bins = s_hist + (kBins - 2 - 2 * int(threadIdx.x));
    const i32x4 l4 = bins[0], h4 = bins[1];
    bins[0] = i32x4{};
    bins[1] = i32x4{};
    const int hi = (h4[0] + h4[1]) + (h4[2] + h4[3]), lo = (l4[0] + l4[1]) + (l4[2] + l4[3]);
    const int incl = wave_prefix_sum(hi + lo);
    if (lane == 63) reinterpret_cast<int*>(s_wave[0])[wave] = incl;
    __syncthreads();
    const int before = incl - hi - lo + before_wave(s_wave[0], wave);
    if (before < need && need <= before + hi) {
      s_found[0] = kBins - 1 - 2 * int(threadIdx.x);
      s_found[1] = need - before;
    } else if (before + hi < need && need <= before + hi + lo) {
      s_found[0] = kBins - 2 - 2 * int(threadIdx.x);
      s_found[1] = need - before - hi;
    }
    __syncthreads();
    prefix |= uint32_t(s_found[0]) << shift;
    fixed |= mask << shift;
    need = s_found[1];
  }
  // Kept: keys above `prefix`, and the first `need` that equal it.
  int above = 0, equal = 0;
  each([&](int, uint32_t key) {
    above += __popcll(__builtin_amdgcn_ballot_w64(key > prefix));
    equal += __popcll(__builtin_amdgcn_ballot_w64(key == prefix));
  });
  __syncthreads();  // s_wave is read
  if (lane == 0) {
    reinterpret_cast<int*>(s_wave[0])[wave] = above;
    reinterpret_cast<int*>(s_wave[1])[wave] = equal;
  }
  __syncthreads();
  int seen_above = before_wave(s_wave[0], wave), seen_equal = before_wave(s_wave[1], wave);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  each([&](int i, uint32_t key) {
    const uint64_t ma = __builtin_amdgcn_ballot_w64(key > prefix), me = __builtin_amdgcn_ballot_w64(key == prefix);
    if (ma | me) {  // uniform
      const int eq = seen_equal + __popcll(me & below);
      if (key > prefix || (key == prefix && eq < need)) {
        kept[seen_above + __popcll(ma & below) + min(eq, need)] = w0 + 64 * i + lane;
      }
      seen_above += __popcll(ma);
      seen_equal += __popcll(me);
    }
  });
}

// Vectors [16 bytes] of the kept rows of one (sequence, KV head), a grid of them, their masses, and what lies
// behind the last.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int keep = min(evict_len(a, b), a.budget);
  const int vecs = a.head_dim / 8;
  const int64_t row = int64_t(b) * a.hkv + h;
  const int first = int(blockIdx.x) * 256 + int(threadIdx.x), stride = int(gridDim.x) * 256;  // at most 2^20
  auto page_of = [&](int t) { return a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size; };
  // Vector `first` and every stride-th one after it, as (place, vector of its row).
  const int step_rows = stride / vecs, step_vecs = stride - step_rows * vecs;
  int64_t j = first / vecs;
  int c = first - int(j) * vecs;
  while (j < keep) {
    const int t = a.kept[row * a.budget + j];
    const int page = page_of(t), new_page = page_of(int(j));
    const int from = a.block_table[b * a.bt_stride + page], into = a.new_table[b * a.nt_stride + new_page];
    if (uint32_t(from) < uint32_t(a.num_blocks32) && uint32_t(into) < uint32_t(a.num_blocks32)) {
      const int64_t src = int64_t(from) * a.page_size + (t - page * a.page_size);
      const int64_t dst = int64_t(into) * a.page_size + (int(j) - new_page * a.page_size);
      const int64_t s = (src * a.hkv + h) * a.head_dim + 8 * c, d = (dst * a.hkv + h) * a.head_dim + 8 * c;
      const u32x4 k = load16(a.k_cache + s);
      if (a.v_cache) {
        const u32x4 v = load16(a.v_cache + s);
        __builtin_amdgcn_sched_barrier(0);  // both loads before the first store waits
        *reinterpret_cast<u32x4*>(a.v_cache + d) = v;
      }
      *reinterpret_cast<u32x4*>(a.k_cache + d) = k;
    }
    j += step_rows;
    c += step_vecs;
    if (c >= vecs) {
      c -= vecs;
      ++j;
    }
  }
  const float* mass = a.mass + b * a.m_sb + h * a.m_sh;
  for (int64_t i = first; i < a.capacity; i += stride) {
    a.mass_out[row * a.capacity + i] = i < keep ? mass[a.kept[row * a.budget + i]] : 0.f;
  }
  for (int64_t i = keep + first; i < a.budget; i += stride) a.kept[row * a.budget + i] = -1;
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
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(unsigned(page_size)) : -1;
  a.max_blocks = max_blocks_per_seq;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.capacity = mass_capacity;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 sel{unsigned(num_kv_heads), unsigned(batch)};
  hipLaunchKernelGGL(evict_select_kernel<true>, sel, dim3(kThreads), 0, s, a);
  if (tokens > kHeld * kThreads) hipLaunchKernelGGL(evict_select_kernel<false>, sel, dim3(kThreads), 0, s, a);
  int64_t work = most * (head_dim / 8);
  work = work > budget ? work : budget;
  work = work > mass_capacity ? work : mass_capacity;
  const int64_t blocks = ceil_div(work, 256);
  const dim3 grid(unsigned(blocks < 4096 ? blocks : 4096), unsigned(num_kv_heads), unsigned(batch));
  hipLaunchKernelGGL(evict_copy_kernel, grid, dim3(256), 0, s, a);
  return check_launch(who);
}
