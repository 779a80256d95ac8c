// Attention weight that each cached token receives from a sequence's last queries (gfx950): for sequence b
// and KV head g, over the rows r = (query i of the last `new`, head of the group),
//   mass[b, g, t] += sum_r softmax_t( scale * q_r . K[t] ),  query i seeing t <= seqlen - new + i,
// the running sums by which a cache is cut to its heaviest tokens (cache_evict.hip). Everything past the
// products of 16-bit values is 32 bits; a token's sum is made by one lane in a fixed order, so calls repeat
// bit for bit.
//
// A wave takes 16 TT tokens of one KV head, whose K rows it reads from the pages into registers as MFMA
// operands (lane l: row l % 16, 8 values of k-group l / 16), and multiplies them with 16 rows of queries at
// a time, S^T[16 tokens x 16 rows] as in the paged decode.
//   Up to 16 rows (a decode step): the scores are kept, 4 bytes a row and token against 2 D of the K row,
//     beside each workgroup's (max, sum) of every row; a second kernel joins those and adds the weights.
//     K is read once.
//   More rows (a window of queries): scores would outweigh K, so they are computed twice: once for the
//     (max, sum) of every workgroup and row, joined by a small kernel, and once for the weights. A
//     workgroup's K rows stay in registers while the queries come 32 rows at a time through LDS, the next
//     ones on their way, so that a wave reads each operand once for all its tokens.
#include "lds_tiles.h"

namespace ti {
namespace {

struct MassArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;  // q [B, new, Hq, D] strides (elements)
  const uint16_t* k_cache;   // rows [num_blocks * page_size][hkv][D]
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seqlen;
  float* mass;  // [B, hkv, >= max_blocks * page_size]
  int64_t m_sb, m_sh;
  float* scores;  // [B, hkv, rows][tokens]  (up to 16 rows)
  float* part;    // [B, hkv][parts][rows][2]  (max, sum) of a workgroup's tokens, max in exp2 units
  float* stats;   // [B, hkv][rows][2]  (max, 1 / sum)  (more than 16 rows)
  int32_t new_tokens, hkv, group, rows, num_blocks32, page_size, page_shift, max_blocks;
  int32_t parts;   // parts of a sequence of the greatest length
  int64_t tokens;  // that length, a multiple of 4
  float scale_log2;
};

constexpr int kFewRows = 16;

__device__ __forceinline__ int mass_len(const MassArgs& a, int b) {
  const int64_t cap = int64_t(a.max_blocks) * a.page_size;
  const int n = max(a.seqlen[b], 0);
  return int64_t(n) > cap ? int(cap) : n;
}

__device__ __align__(16) uint16_t g_zero_key[576] = {};

// The K operands of tokens t0 + 16 tt + (0 .. 15), as lane (n, g) holds them, and whether this lane's
// accumulator tokens (4 g + e of each tile) exist.
template <int D, int TT>
struct KeyTile {
  u32x4 k[TT][D / 32];
  uint32_t there[TT];  // bit j: token 16 tt + j is in the sequence and its block in the cache
};

template <int D, int TT>
__device__ __forceinline__ void load_keys(const MassArgs& a, int b, int h, int len, int t0, KeyTile<D, TT>& x) {
  const int lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  // All ids, then all rows: no load waits for another one's, and none is conditional (a branch around each would
  // order them). An absent token is a row of zeros, whatever the cache holds there.
  int id[TT], in_page[TT];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const int t = min(t0 + 16 * tt + n, len - 1);
    const int page = a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size;
    in_page[tt] = t - page * a.page_size;
    id[tt] = a.block_table[b * a.bt_stride + page];
  }
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const bool ok = t0 + 16 * tt + n < len && uint32_t(id[tt]) < uint32_t(a.num_blocks32);
    x.there[tt] = uint32_t(__builtin_amdgcn_ballot_w64(ok)) & 0xffffu;
    const uint16_t* row = a.k_cache + ((int64_t(id[tt]) * a.page_size + in_page[tt]) * a.hkv + h) * D;
    const uint16_t* src = (ok ? row : g_zero_key) + 8 * g;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) x.k[tt][kk] = load16(src + 32 * kk);
  }
}

// Scores, in exp2 units, of the tile's tokens (4 g + e of each 16) and row r0 + n; -inf where the row does
// not see the token. Rows behind the last are all -inf.
template <int D, int TT, typename Tag>
__device__ __forceinline__ void score_rows(const MassArgs& a, int b, int h, int len, int t0, int r0,
                                           const KeyTile<D, TT>& x, float (&s)[TT][4]) {
  const int lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int r = min(r0 + n, a.rows - 1);
  const int tok = r / a.group, head = h * a.group + (r - tok * a.group);
  const uint16_t* src = a.q + b * a.q_sb + tok * a.q_st + head * a.q_sh + 8 * g;
  u32x4 q[D / 32];
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) q[kk] = load16(src + 32 * kk);
  f32x4 acc[TT];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) acc[tt] = f32x4{};
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) {
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[tt] = mfma16x16x32(x.k[tt][kk], q[kk], acc[tt], Tag{});
  }
  const int last = r0 + n < a.rows ? len - a.new_tokens + tok : -1;
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 4 * g + e;
      const bool seen = ((x.there[tt] >> j) & 1) && t0 + 16 * tt + j <= last;
      s[tt][e] = seen ? acc[tt][e] * a.scale_log2 : -INFINITY;
    }
  }
}

// (max, sum) of each row over the wave's tokens, of scores s * scale (a scale is positive).
template <int TT>
__device__ __forceinline__ void row_stats(const float (&s)[TT][4], float scale, float& m, float& l) {
  float top = max2(max3(s[0][0], s[0][1], s[0][2]), s[0][3]);
#pragma unroll
  for (int tt = 1; tt < TT; ++tt) top = max3(max3(top, s[tt][0], s[tt][1]), s[tt][2], s[tt][3]);
  top = row_group_max(top);
  m = top == -INFINITY ? -INFINITY : top * scale;  // nothing seen, whatever the scale
  const float base = m == -INFINITY ? 0.f : m;
  float part[4] = {};
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
    for (int e = 0; e < 4; ++e) part[e] += fast_exp2(fmaf(s[tt][e], scale, -base));
  }
  l = row_group_sum((part[0] + part[1]) + (part[2] + part[3]));
}

// Up to 16 rows: scores of 64 TT tokens a workgroup, and its (max, sum) of every row.
template <int D, int TT, typename Tag>
__global__ __launch_bounds__(256) void mass_scores_kernel(MassArgs a) {
  __shared__ float s_ml[4][16][2];
  const int b = blockIdx.y, chunk = int(blockIdx.x / unsigned(a.hkv)), h = int(blockIdx.x) - chunk * a.hkv;
  const int len = mass_len(a, b);
  const int wg0 = chunk * 64 * TT;
  if (wg0 >= len) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & 15, g = lane >> 4;
  const int t0 = wg0 + wave * 16 * TT;
  KeyTile<D, TT> x;
  load_keys<D, TT>(a, b, h, len, t0, x);
  // All of them in flight before the first product waits (16 x U[512, 8k], D = 256: 34.5 us against 36.9); 144
  // registers of them would leave two waves a SIMD (16 x 4,000 latent rows 27.5 us against 24.6).
  if constexpr (D <= 320) __builtin_amdgcn_sched_barrier(0);
  float s[TT][4], m, l;
  score_rows<D, TT, Tag>(a, b, h, len, t0, 0, x, s);
  if (n < a.rows) {
    float* dst = a.scores + ((int64_t(b) * a.hkv + h) * a.rows + n) * a.tokens + t0 + 4 * g;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      if (t0 + 16 * tt + 4 * g < len) {
        *reinterpret_cast<f32x4*>(dst + 16 * tt) = f32x4{s[tt][0], s[tt][1], s[tt][2], s[tt][3]};
      }
    }
  }
  row_stats<TT>(s, 1.f, m, l);
  if (g == 0) {
    s_ml[wave][n][0] = m;
    s_ml[wave][n][1] = l;
  }
  __syncthreads();
  if (threadIdx.x < unsigned(a.rows)) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[w][threadIdx.x][0]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < 4; ++w) sum += s_ml[w][threadIdx.x][1] * fast_exp2(s_ml[w][threadIdx.x][0] - base);
    float* dst = a.part + (((int64_t(b) * a.hkv + h) * a.parts + chunk) * a.rows + threadIdx.x) * 2;
    dst[0] = top;
    dst[1] = sum;
  }
}

// (max, 1 / sum) of a row from its parts; 16 lanes of consecutive threads join one row.
__device__ __forceinline__ void join_parts(const float* part, int parts, int64_t stride, int lane16, float& m,
                                           float& inv) {
  m = -INFINITY;
  float l = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 64) {  // four loads in flight a lane
    float2 ml[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      ml[k] = *reinterpret_cast<const float2*>(part + min(p0 + 16 * k + lane16, parts - 1) * stride);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float pm = p0 + 16 * k + lane16 < parts ? ml[k].x : -INFINITY;
      const float mn = fmaxf(m, pm);
      const float base = mn == -INFINITY ? 0.f : mn;
      l = l * fast_exp2(m - base) + (pm == -INFINITY ? 0.f : ml[k].y) * fast_exp2(pm - base);
      m = mn;
    }
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    const float om = __shfl_xor(m, d, 64), ol = __shfl_xor(l, d, 64);
    const float mn = fmaxf(m, om);
    const float base = mn == -INFINITY ? 0.f : mn;
    l = l * fast_exp2(m - base) + ol * fast_exp2(om - base);
    m = mn;
  }
  inv = l != 0.f ? 1.f / l : 0.f;  // a row that sees nothing gives nothing
}

constexpr int kAddTokens = 1024;  // tokens of a workgroup of mass_add_kernel

// The weights of up to 16 rows from their scores, added to the sums.
__global__ __launch_bounds__(256) void mass_add_kernel(MassArgs a, int part_tokens) {
  __shared__ float s_stat[kFewRows][2];
  const int b = blockIdx.z, h = blockIdx.y;
  const int len = mass_len(a, b);
  const int wg0 = int(blockIdx.x) * kAddTokens;
  if (wg0 >= len) return;
  const int t = wg0 + 4 * int(threadIdx.x);
  float* dst = a.mass + b * a.m_sb + h * a.m_sh;
  float before[4];  // on their way beside the scores, not one after the other behind them
#pragma unroll
  for (int e = 0; e < 4; ++e) before[e] = dst[min(t + e, len - 1)];
  const int64_t bh = int64_t(b) * a.hkv + h;
  const int parts = (len + part_tokens - 1) / part_tokens;
  const int row = threadIdx.x >> 4;
  if (row < a.rows) {
    float m, inv;
    join_parts(a.part + (bh * a.parts * a.rows + row) * 2, parts, 2 * int64_t(a.rows), threadIdx.x & 15, m, inv);
    if ((threadIdx.x & 15) == 0) {
      s_stat[row][0] = m == -INFINITY ? 0.f : m;
      s_stat[row][1] = inv;
    }
  }
  __syncthreads();
  if (t >= len) return;
  const float* src = a.scores + bh * a.rows * a.tokens + t;
  float w[4] = {};
  for (int r0 = 0; r0 < a.rows; r0 += 8) {
    f32x4 s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = *reinterpret_cast<const f32x4*>(src + min(r0 + i, a.rows - 1) * a.tokens);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (r0 + i >= a.rows) break;  // uniform
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] += fast_exp2(s[i][e] - s_stat[r0 + i][0]) * s_stat[r0 + i][1];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (t + e < len) dst[t + e] = before[e] + w[e];
  }
}

// More than 16 rows: queries through LDS, kQRows at a time in two or three stages. Place of 16-byte chunk c of row r: c ^
// its swizzle, so that the operand reads (16 rows of a chunk and its neighbour) hit every bank quad once;
// rows of whole 256-byte blocks start on the same bank, the others 32 banks apart.
constexpr int kQRows = 32;

template <int D>
__device__ __forceinline__ int q_place(int r) {
  return D % 128 == 0 ? swz16(r) : swz8(r);
}

// STATS: the rows' (max, 1 / sum) come too, behind the queries, a copy for each wave.
template <int D, bool STATS>
struct QueryStages {
  static constexpr int CH = D / 8, QLOADS = kQRows * CH / 256, LOADS = QLOADS + (STATS ? 1 : 0);
  static constexpr int STAGE = kQRows * D + (STATS ? 4 * kQRows * 4 : 0);  // 16-bit elements
  static constexpr int STAGES = D <= 320 ? 3 : 2;  // three: one barrier a block

  // This lane's part of the loads, block after block: address and place in the group of its rows. They advance
  // without a division or a product, which would take as long as the block's scores.
  const uint16_t* at[QLOADS];
  int head[QLOADS];
  const uint16_t* first;
  const float* stats;
  int next = 0;  // first row of the block to load next
  int64_t step, wrap;
  int step_heads, lane, wave;

  __device__ __forceinline__ QueryStages(const MassArgs& a, int b, int h)
      : lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
    first = a.q + b * a.q_sb + int64_t(h) * a.group * a.q_sh;
    stats = STATS ? a.stats + (int64_t(b) * a.hkv + h) * a.rows * 2 : nullptr;
    const int toks = kQRows / a.group;
    step_heads = kQRows - toks * a.group;
    step = toks * a.q_st + step_heads * a.q_sh;
    wrap = a.q_st - a.group * a.q_sh;
#pragma unroll
    for (int i = 0; i < QLOADS; ++i) {
      const int f = (wave * QLOADS + i) * 64 + lane, row = f / CH;
      const int tok = row / a.group;
      head[i] = row - tok * a.group;
      at[i] = first + tok * a.q_st + head[i] * a.q_sh + 8 * ((f % CH) ^ q_place<D>(row));
    }
  }

  // The next kQRows queries of the group into a stage; in place of rows behind the last, its first one.
  __device__ __forceinline__ void issue(const MassArgs& a, uint16_t* stage) {
#pragma unroll
    for (int i = 0; i < QLOADS; ++i) {
      const int f = (wave * QLOADS + i) * 64 + lane;
      const uint16_t* src = next + f / CH < a.rows ? at[i] : first + 8 * (f % CH);
      const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(stage + (wave * QLOADS + i) * 512)));
      asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
      head[i] += step_heads;
      const bool over = head[i] >= a.group;
      at[i] += step + (over ? wrap : 0);
      head[i] -= over ? a.group : 0;
    }
    if constexpr (STATS) {
      static_assert(2 * kQRows == 64);
      const float* src = stats + min(2 * next + lane, 2 * a.rows - 1);
      const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(stage + kQRows * D + wave * 128)));
      asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "{m0}"(m0) : "memory");
    }
    next += kQRows;
  }

  // Products of the wave's tokens and rows r0 + 16 rt + n, -inf where the row does not see the token. whole: every
  // token exists and every row sees it.
  template <int TT, typename Tag>
  static __device__ __forceinline__ void scores(const MassArgs& a, int len, int t0, int r0, int rt, bool whole,
                                                const uint16_t* stage, const KeyTile<D, TT>& x,
                                                float (&s)[TT][4]) {
    const int lane = threadIdx.x & 63;
    const int n = lane & 15, g = lane >> 4;
    u32x4 q[D / 32];
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      q[kk] = *reinterpret_cast<const u32x4*>(stage + (16 * rt + n) * D + 8 * ((4 * kk + g) ^ q_place<D>(n)));
    }
    f32x4 acc[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[tt] = f32x4{};
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) acc[tt] = mfma16x16x32(x.k[tt][kk], q[kk], acc[tt], Tag{});
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[tt][e] = acc[tt][e];
    }
    const int r = r0 + 16 * rt + n;
    if (!whole || r0 + kQRows > a.rows) {  // uniform
      const int last = r < a.rows ? len - a.new_tokens + r / a.group : -1;
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * g + e;
          if (!((x.there[tt] >> j) & 1) || t0 + 16 * tt + j > last) s[tt][e] = -INFINITY;
        }
      }
    }
  }

  // Calls f(i, r0, stage) for every block of queries, the next ones on their way; past(i) behind the barrier
  // that ends block i.
  template <typename F, typename P>
  __device__ __forceinline__ void for_blocks(const MassArgs& a, uint16_t* stages, F f, P past) {
    issue(a, stages);
    if (kQRows < a.rows) issue(a, stages + STAGE);
    // The keys (and whatever else the compiler knows of) have landed, so that it places no wait of its own,
    // which would also wait for the stage in flight, in the loop.
    __builtin_amdgcn_s_waitcnt(0);
    int stage = 0;
    const int blocks = (a.rows + kQRows - 1) / kQRows;
    for (int i = 0; i < blocks; ++i) {
      if (i + 1 < blocks) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (STAGES == 3 && i + 2 < blocks) {  // the stage of block i - 1 is read
        issue(a, stages + (stage == 0 ? 2 : stage - 1) * STAGE);
      }
      if (i > 0) past(i - 1);
      f(i, i * kQRows, stages + stage * STAGE);
      if (STAGES == 2) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (i + 2 < blocks) issue(a, stages + stage * STAGE);
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    past(blocks - 1);
  }
};

// Whether every token of the wave's tiles exists and every query sees it (uniform).
template <int D, int TT>
__device__ __forceinline__ bool all_seen(const MassArgs& a, int len, int t0, const KeyTile<D, TT>& x) {
  uint32_t all = 0xffffu;
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) all &= x.there[tt];
  return all == 0xffffu && t0 + 16 * TT <= len - a.new_tokens + 1;
}

// Waves of a SIMD: what the K rows leave of the registers. They are what hides a workgroup's start (its blocks'
// ids, then its keys): 32 queries of 32/8 heads of 128 over 4 x U[2k, 16k] tokens, both passes, 92 us with
// three of 64 tokens each, 67 with five of 32. At D = 128 five leave the second pass one register short (one value
// of scratch a lane, stored and read once).
constexpr int mass_waves(int d) { return d <= 128 ? 5 : d <= 256 ? 3 : 2; }

// First pass: (max, sum) of every workgroup and row.
template <int D, int TT, typename Tag>
__global__ __launch_bounds__(256, mass_waves(D)) void mass_stats_kernel(MassArgs a) {
  using Q = QueryStages<D, false>;
  __shared__ __align__(16) uint16_t s_q[Q::STAGES * Q::STAGE];
  __shared__ float2 s_ml[2][4][kQRows];
  const int b = blockIdx.y, chunk = int(blockIdx.x / unsigned(a.hkv)), h = int(blockIdx.x) - chunk * a.hkv;
  const int len = mass_len(a, b);
  if (chunk * 64 * TT >= len) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = (chunk * 4 + wave) * 16 * TT;
  Q queries(a, b, h);
  KeyTile<D, TT> x;
  load_keys<D, TT>(a, b, h, len, t0, x);
  const bool whole = all_seen<D, TT>(a, len, t0, x);
  float2* dst = reinterpret_cast<float2*>(a.part) + ((int64_t(b) * a.hkv + h) * a.parts + chunk) * a.rows;
  queries.for_blocks(
      a, s_q,
      [&](int i, int r0, const uint16_t* stage) {
#pragma unroll
        for (int rt = 0; rt < kQRows / 16; ++rt) {
          float s[TT][4], m, l;
          Q::template scores<TT, Tag>(a, len, t0, r0, rt, whole, stage, x, s);
          row_stats<TT>(s, a.scale_log2, m, l);
          if (lane < 16) s_ml[i & 1][wave][16 * rt + lane] = make_float2(m, l);
        }
      },
      [&](int i) {  // the waves' parts are there
        const int r = i * kQRows + lane;
        if (wave != (i & 3) || lane >= kQRows || r >= a.rows) return;
        float2 ml[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) ml[w] = s_ml[i & 1][w][lane];
        const float top = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += ml[w].y * fast_exp2(ml[w].x - base);
        dst[r] = make_float2(top, sum);
      });
}

__global__ __launch_bounds__(256) void mass_join_kernel(MassArgs a, int part_tokens) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int parts = (mass_len(a, b) + part_tokens - 1) / part_tokens;
  const int row = int(blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (row >= a.rows) return;
  const int64_t bh = int64_t(b) * a.hkv + h;
  float m, inv;
  join_parts(a.part + (bh * a.parts * a.rows + row) * 2, parts, 2 * int64_t(a.rows), threadIdx.x & 15, m, inv);
  if ((threadIdx.x & 15) == 0) {
    float* dst = a.stats + (bh * a.rows + row) * 2;
    dst[0] = m == -INFINITY ? 0.f : m;
    dst[1] = inv;
  }
}

// Second pass: the weights, added to the sums.
template <int D, int TT, typename Tag>
__global__ __launch_bounds__(256, mass_waves(D)) void mass_weights_kernel(MassArgs a) {
  using Q = QueryStages<D, true>;
  __shared__ __align__(16) uint16_t s_q[Q::STAGES * Q::STAGE];
  const int b = blockIdx.y, chunk = int(blockIdx.x / unsigned(a.hkv)), h = int(blockIdx.x) - chunk * a.hkv;
  const int len = mass_len(a, b);
  if (chunk * 64 * TT >= len) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int t0 = (chunk * 4 + wave) * 16 * TT;
  Q queries(a, b, h);
  KeyTile<D, TT> x;
  load_keys<D, TT>(a, b, h, len, t0, x);
  const bool whole = all_seen<D, TT>(a, len, t0, x);
  float w[TT][4] = {};
  queries.for_blocks(a, s_q, [&](int, int r0, const uint16_t* stage) {
#pragma unroll
    for (int rt = 0; rt < kQRows / 16; ++rt) {
      float s[TT][4];
      Q::template scores<TT, Tag>(a, len, t0, r0, rt, whole, stage, x, s);
      const float2 ml = reinterpret_cast<const float2*>(stage + kQRows * D + wave * 128)[16 * rt + n];
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[tt][e] = fmaf(fast_exp2(fmaf(s[tt][e], a.scale_log2, -ml.x)), ml.y, w[tt][e]);
        }
      }
    }
  }, [](int) {});
  // The 16 lanes of a group hold 4 TT tokens' sums over their own rows: halves change hands until every lane has
  // one token's (or one of 16 / (4 TT) copies of it), v[0] of token 16 (i / 4) + 4 g + i % 4, i the bits of n.
  float v[4 * TT];
#pragma unroll
  for (int i = 0; i < 4 * TT; ++i) v[i] = w[i >> 2][i & 3];
#pragma unroll
  for (int half = 2 * TT, d = 8; d > 0; half >>= 1, d >>= 1) {
    if (half > 0) {
      const bool up = n & d;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float mine = up ? v[i + half] : v[i], other = up ? v[i] : v[i + half];
        v[i] = mine + __shfl_xor(other, d, 64);
      }
    } else {
      v[0] += __shfl_xor(v[0], d, 64);
    }
  }
  const int i = n / (4 / TT);
  const int t = t0 + 16 * (i >> 2) + 4 * g + (i & 3);
  if (n % (4 / TT) == 0 && t < len) a.mass[b * a.m_sb + h * a.m_sh + t] += v[0];
}

// 16-token tiles of a wave: what its K rows leave of the registers.
// (Few rows, us with 1 / 2 / 4: a step of 16 x U[512, 8k] tokens, 24/4 heads of 256, 43.8 / 43.5 / 46.9, one of
// 8,000 14.7 / 14.0 / 16.0, 16 x 4,000 latent rows 30.6 / 27.3 / 27.1. 32 queries over 4 x 4,000 latent rows:
// 89 with 1 against 134 with 2, whose query addresses no longer fit the registers.)
constexpr int tiles_of(int d, bool few) { return few || d <= 320 ? 2 : 1; }

struct MassSizes {
  int32_t part_tokens, parts;
  int64_t tokens, scores, part, stats, bytes;  // floats, bytes
};

MassSizes mass_sizes(int32_t batch, int32_t hkv, int32_t rows, int32_t d, int64_t tokens) {
  MassSizes s;
  const bool few = rows <= kFewRows;
  s.part_tokens = 64 * tiles_of(d, few);
  s.parts = int32_t(ceil_div(tokens, s.part_tokens));
  s.tokens = ceil_div(tokens, 4) * 4;
  const int64_t bh = int64_t(batch) * hkv;
  s.scores = few ? bh * rows * s.tokens : 0;
  s.part = bh * s.parts * rows * 2;
  s.stats = few ? 0 : bh * rows * 2;
  s.bytes = ((s.scores + s.part + s.stats) * 4 + 15) & ~int64_t(15);
  return s;
}

int check_mass(const char* who, int32_t batch, int32_t new_tokens, int32_t hq, int32_t hkv, int32_t d,
               int32_t page_size, int32_t max_blocks) {
  if (d != 128 && d != 256 && d != 320 && d != 576) {
    return fail(TI_EUNSUPPORTED, "%s: head_dim %d not built (128, 256, 320, 576)", who, d);
  }
  if (batch < 0 || batch > 65535 || new_tokens <= 0 || hq <= 0 || hkv <= 0 || hkv > 65535 || hq % hkv != 0 ||
      int64_t(new_tokens) * (hq / hkv) > (1 << 20)) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d new_tokens=%d heads=%d/%d", who, batch, new_tokens, hq, hkv);
  }
  const int part_tokens = 64 * tiles_of(d, new_tokens * (hq / hkv) <= kFewRows);
  if (page_size <= 0 || max_blocks < 0 || int64_t(max_blocks) * page_size > INT32_MAX - 1024 ||
      ceil_div(int64_t(max_blocks) * page_size, part_tokens) * hkv > kMaxGridX) {
    return fail(TI_EINVAL, "%s: bad cache page_size=%d max_blocks_per_seq=%d", who, page_size, max_blocks);
  }
  return TI_OK;
}

template <int D, typename Tag>
void launch_mass(const MassArgs& a, const MassSizes& sz, unsigned batch, hipStream_t s) {
  const unsigned hkv = unsigned(a.hkv);
  // The heads of a token range follow each other: together they read whole rows of the cache.
  const dim3 grid(unsigned(ceil_div(a.tokens, sz.part_tokens)) * hkv, batch);
  if (a.rows <= kFewRows) {
    hipLaunchKernelGGL((mass_scores_kernel<D, tiles_of(D, true), Tag>), grid, dim3(256), 0, s, a);
    hipLaunchKernelGGL(mass_add_kernel, dim3(unsigned(ceil_div(a.tokens, kAddTokens)), hkv, batch), dim3(256), 0,
                       s, a, sz.part_tokens);
    return;
  }
  constexpr int TT = tiles_of(D, false);
  hipLaunchKernelGGL((mass_stats_kernel<D, TT, Tag>), grid, dim3(256), 0, s, a);
  hipLaunchKernelGGL(mass_join_kernel, dim3(unsigned(ceil_div(a.rows, 16)), hkv, batch), dim3(256), 0, s, a,
                     sz.part_tokens);
  hipLaunchKernelGGL((mass_weights_kernel<D, TT, Tag>), grid, dim3(256), 0, s, a);
}

template <typename Tag>
void launch_mass_dim(const MassArgs& a, const MassSizes& sz, int d, unsigned batch, hipStream_t s) {
  if (d == 128) launch_mass<128, Tag>(a, sz, batch, s);
  else if (d == 256) launch_mass<256, Tag>(a, sz, batch, s);
  else if (d == 320) launch_mass<320, Tag>(a, sz, batch, s);
  else launch_mass<576, Tag>(a, sz, batch, s);
}

}  // namespace
}  // namespace ti

extern "C" int ti_cache_mass_workspace_bytes(int32_t batch, int32_t new_tokens, int32_t num_q_heads,
                                             int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                             int32_t max_blocks_per_seq, int64_t* workspace_bytes_out) {
  using namespace ti;
  const char* who = "ti_cache_mass_workspace_bytes";
  int rc = check_mass(who, batch, new_tokens, num_q_heads, num_kv_heads, head_dim, page_size, max_blocks_per_seq);
  if (rc != TI_OK) return rc;
  if (!workspace_bytes_out) return fail(TI_EINVAL, "%s: null output", who);
  *workspace_bytes_out = mass_sizes(batch, num_kv_heads, new_tokens * (num_q_heads / num_kv_heads), head_dim,
                                    int64_t(max_blocks_per_seq) * page_size).bytes;
  return TI_OK;
}

extern "C" int ti_cache_mass(const void* q, int64_t q_stride_b, int64_t q_stride_t, int64_t q_stride_h,
                             const void* k_cache, const int32_t* block_table, int64_t block_table_stride,
                             const int32_t* seqlen, float* mass, int64_t mass_stride_b, int64_t mass_stride_h,
                             void* workspace, int64_t workspace_bytes, int32_t batch, int32_t new_tokens,
                             int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                             int64_t num_blocks, int32_t max_blocks_per_seq, float scale, int32_t dtype,
                             void* stream) {
  using namespace ti;
  const char* who = "ti_cache_mass";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  int rc = check_mass(who, batch, new_tokens, num_q_heads, num_kv_heads, head_dim, page_size, max_blocks_per_seq);
  if (rc != TI_OK) return rc;
  if (!(scale > 0.f && scale <= kMaxScale)) {
    return fail(TI_EINVAL, "%s: scale %g is not positive or beyond 1e30", who, double(scale));
  }
  if (num_blocks < 0 || num_blocks > INT32_MAX) {
    return fail(TI_EINVAL, "%s: bad cache num_blocks=%lld", who, static_cast<long long>(num_blocks));
  }
  const int64_t tokens = int64_t(max_blocks_per_seq) * page_size;
  if (mass_stride_h < tokens || mass_stride_b < 0) {
    return fail(TI_EINVAL, "%s: mass rows of %lld floats for sequences of up to %lld tokens", who,
                static_cast<long long>(mass_stride_h), static_cast<long long>(tokens));
  }
  if (batch == 0 || tokens == 0) return TI_OK;
  const int32_t rows = new_tokens * (num_q_heads / num_kv_heads);
  const MassSizes sz = mass_sizes(batch, num_kv_heads, rows, head_dim, tokens);
  if (!q || !k_cache || !block_table || !seqlen || !mass || !workspace) return fail(TI_EINVAL, "%s: null pointer", who);
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
        reinterpret_cast<uintptr_t>(workspace)) & 15) != 0 ||
      q_stride_b % 8 != 0 || q_stride_t % 8 != 0 || q_stride_h % 8 != 0) {
    return fail(TI_EINVAL, "%s: q, cache and workspace must be 16-byte aligned, q strides multiples of 8", who);
  }
  if (workspace_bytes < sz.bytes) {
    return fail(TI_EINVAL, "%s: workspace %lld < %lld bytes", who, static_cast<long long>(workspace_bytes),
                static_cast<long long>(sz.bytes));
  }
  MassArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_stride_b;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_cache = static_cast<const uint16_t*>(k_cache);
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.seqlen = seqlen;
  a.mass = mass;
  a.m_sb = mass_stride_b;
  a.m_sh = mass_stride_h;
  a.scores = static_cast<float*>(workspace);
  a.part = a.scores + sz.scores;
  a.stats = a.part + sz.part;
  a.new_tokens = new_tokens;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.rows = rows;
  a.num_blocks32 = int32_t(num_blocks);
  a.page_size = page_size;
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(unsigned(page_size)) : -1;
  a.max_blocks = max_blocks_per_seq;
  a.parts = sz.parts;
  a.tokens = sz.tokens;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == TI_DTYPE_BF16) launch_mass_dim<Bf16>(a, sz, head_dim, unsigned(batch), s);
  else launch_mass_dim<F16>(a, sz, head_dim, unsigned(batch), s);
  return check_launch(who);
}
