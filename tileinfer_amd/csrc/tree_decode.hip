// Attention of drafted trees over the paged cache (gfx950): the last N <= 64 tokens of every sequence are its queries,
// N drafts behind a context of C = seqlen - N tokens (N = 1: a decode step). Draft i sees the context and those drafts j
// whose bit is set in its 64-bit mask (its ancestors and itself):
//   s_j = cap tanh(scale q . k_j / cap) - slope |p_i - p_j|,  p = softmax(s),  o = sum_j p_j v_j
// The position of a context token is its place, that of draft i is C + (number of other drafts it sees), its depth in the
// tree, and a window keeps the keys with p_i - p_j < window.
//
// Work: the rows of a KV head are the (draft, query head of its group) pairs. A workgroup of eight waves holds RB = 16 RG
// rows of one (sequence, KV head) and walks its tokens in tiles of 8192 / D, staged in LDS:
//   S^T[16 tokens x 16 rows] = K[16 x D] . Q^T[D x 16]        (16x16x32) cut over the waves by tokens, rows and k
//   O^T[16 d x 16 rows]     += V^T[16 d x 32] . P^T[32 x 16]  every wave its 16 rows and D RG / 8 columns
// in which an accumulator's row is its lane's column, as in the paged prefill. The parts of S go through LDS, every wave of
// a row group adds them up in the same order and keeps the same statistics; the next tile's scores are computed beside
// this tile's output, one barrier a tile.
//
// The batch's tiles are one list, cut into runs of equal length; a run is taken by one workgroup for each KV head, side
// by side, since the heads' rows of a token lie side by side in memory. A sequence that lies in one run is written by it,
// others leave (m, l, o) parts in 32 bits that a second kernel joins in the order of the runs.
//
// Bound: HBM for long batches (a step of 32 x 16,384 tokens with 32/8 heads of 128, capped, 331 to 342 us, 6.3 to 6.5 TB/s;
// with 24/4 heads of 256 320 us, 6.7 TB/s), the start of a run and the join's launch for short ones (16 sequences of 512 to
// 8,192 tokens with one token of 24/4 heads 57 us, with eight 77 to 79, where the scores, statistics and products of four
// row groups follow one another in a tile; one of 700 tokens with eight 16).
//
// Trees of more than 64 rows a KV head go to the kernel of shaped_rows.h (kFewRows).
#include <type_traits>

#include "shaped_rows.h"

namespace ti {
namespace {

constexpr int kWaves = 8;
constexpr int kKStages = 3;    // K tiles in LDS: one in use, two on their way
constexpr int kVStages = 4;    // V is used a tile later

struct TreeArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;  // q [B, N, hq, D] strides (elements)
  const uint16_t* k_cache;   // rows [num_blocks * page_size][hkv * D]
  const uint16_t* v_cache;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seqlen;
  const int64_t* mask;  // [B, N] at mask_sb, or nullptr: draft i sees the drafts j <= i
  int64_t mask_sb;
  const float* slopes;  // [hq] or nullptr
  uint16_t* out;        // [B, N, hq, D]
  float* part_o;        // [runs][hkv][2][RB][D] unnormalised rows
  float* part_ml;       // [runs][hkv][2][RB][2] their (m, l), m in exp2 units
  int32_t* first_tile;  // [B + 1] each sequence's first tile, and the total
  int32_t batch, drafts, hq, hkv, group, rows, num_blocks32, page_size, max_blocks;
  uint32_t page_magic, page_shift;  // as RowsArgs has them
  int32_t runs, window;  // window 0: none
  ScoreShape shape;
};

__device__ __forceinline__ int tree_len(const TreeArgs& a, int b) {
  const int64_t cap = int64_t(a.max_blocks) * a.page_size;
  const int n = max(a.seqlen[b], 0);
  return int64_t(n) > cap ? int(cap) : n;
}
// A sequence's tiles: from the first that any of its queries may see.
__device__ __forceinline__ int tile_begin(const TreeArgs& a, int len, int tile) {
  return a.window > 0 ? max(len - a.drafts - a.window + 1, 0) / tile : 0;
}
__device__ __forceinline__ int tile_count(const TreeArgs& a, int len, int tile) {
  return (len + tile - 1) / tile - tile_begin(a, len, tile);
}

// Calls of at least this many 32 KiB tiles load their rows with the streaming policy; shorter ones, which the last-level
// cache may still hold, keep the default one. Streamed against not, 32 sequences with 32/8 heads of 128: of 16,384 tokens
// 331 us against 379, of 2,400 (9,600 tiles) 58 against 65, of 600 (where the rule changes) 21.9 against 22.6; below it the
// look for shared blocks costs more than it gains (8 sequences of 2,000 tokens with eight drafts of 24/4 heads of 256 37.5
// against 34.3, 128 of 150 tokens 40.7 against 38.9).
constexpr int64_t kStreamTiles = 2400;

__device__ __forceinline__ Runs runs_of(const TreeArgs& a, uint32_t total) { return Runs(uint32_t(a.runs), total, 1u); }

// As load_lds16_at. STREAM: with the nt bit, for bytes that are read once.
template <bool STREAM>
__device__ __forceinline__ void load_lds16_as(uint64_t src, const uint16_t* lds) {
  if constexpr (STREAM) {
    const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(src), "{m0}"(m0) : "memory");
  } else {
    load_lds16_at(src, lds);
  }
}

template <int N>
__device__ __forceinline__ void wait_loads_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int D>
struct TreeTile {
  static constexpr int T = 8192 / D;  // tokens: 16 KiB of K, 16 of V
};

// RG: row groups of 16. CAP: the scores are capped, by the waves that compute them, each its own once (beside the output
// every wave of a row group would cap all of them: 32 x 16,384 tokens with 32/8 heads of 128 405 us against 333).
template <int D, int RG, int CAP, typename Tag>
__global__ __launch_bounds__(64 * kWaves, 2) void tree_decode_kernel(TreeArgs a) {
  constexpr int T = TreeTile<D>::T, TT = T / 16, KP = T / 32;
  constexpr int KS = CAP || TT * RG >= kWaves ? 1 : kWaves / (TT * RG);  // parts of k in the first product
  constexpr int KK = D / 32 / KS;                                        // k-steps of a wave
  constexpr int QW = TT * RG * KS < kWaves ? TT * RG * KS : kWaves;      // waves of the first product
  constexpr int JW = TT * RG * KS / QW;                                  // their 16 x 16 score tiles
  constexpr int DG = kWaves / RG;                                 // column groups
  constexpr int NDT = D / 16 / DG;                                // 16-column tiles of a wave
  constexpr int RB = RG * 16;
  constexpr int CH = D / 8, RPL = 64 / CH;    // 16-byte chunks of a row, rows of a load
  constexpr int NLD = T / RPL / kWaves;       // loads of a wave and tile, of K and of V each
  constexpr int kTileElems = T * D;
  static_assert(NLD == 2 && JW >= 1 && TT % JW == 0);

  __shared__ __align__(16) uint16_t s_k[kKStages * kTileElems];
  __shared__ __align__(16) uint16_t s_v[kVStages * kTileElems];
  __shared__ f32x4 s_s[2][KS][RG][TT][64];  // scores of the next tile and of this one
  __shared__ int s_ids[kIdSlots];
  __shared__ int s_depth[kMaxDrafts];
  __shared__ __align__(16) uint64_t s_from[4][T][2];  // addresses of a tile's tokens in K and in V
  __shared__ uint64_t s_here[8];                      // and which of them exist

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rg = wave % RG, dg = wave / RG;  // of the second product
  const int q_tt = wave % QW * JW % TT, q_rest = wave % QW * JW / TT;  // of the first
  const int q_rg = q_rest % RG, q_ks = q_rest / RG;

  const int run = int(blockIdx.x) / a.hkv, kvh = int(blockIdx.x) - run * a.hkv;

  // The batch's tiles, this run's share of them, and the sequence in which it starts.
  uint32_t total = 0;
  int nt = 0, incl = 0;  // of the last 64 sequences looked at
  auto count = [&](int b) { return b < a.batch ? tile_count(a, tree_len(a, b), T) : 0; };
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    nt = count(b0 + lane);
    incl = wave_prefix_sum(nt);
    if (blockIdx.x == 0 && wave == 0 && b0 + lane < a.batch) a.first_tile[b0 + lane] = int(total) + incl - nt;
    total += uint32_t(__builtin_amdgcn_readlane(incl, 63));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.first_tile[a.batch] = int(total);
  const Runs runs = runs_of(a, total);
  if (uint32_t(run) >= runs.runs || total == 0) return;
  const uint32_t start = runs.start(run), end = runs.start(run + 1);
  int b = 0;
  uint32_t unit0 = 0;  // position of sequence b's first tile
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) {
      nt = count(b0 + lane);
      incl = wave_prefix_sum(nt);
    }
    const uint32_t sum = uint32_t(__builtin_amdgcn_readlane(incl, 63));
    if (unit0 + sum > start) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(unit0 + uint32_t(incl) > start);
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      unit0 += uint32_t(__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(nt, l));
      break;
    }
    unit0 += sum;
  }

  // Load j of a wave takes the tile's rows kStep j + load_row; chunk c of row r lies at c ^ swz16(r), the same in rows 16
  // apart.
  constexpr int kStep = kWaves * RPL;
  static_assert(kStep % 16 == 0);
  const int load_row = wave * RPL + lane / CH;
  const uint32_t lane_off = 16 * ((lane % CH) ^ swz16(load_row));
  // Its operand reads (elements): of K rows 16 (q_tt + j) + n each k-step, of V row 4 g + n / 4.
  int k_at[KK], v_at[NDT];
#pragma unroll
  for (int i = 0; i < KK; ++i) k_at[i] = (16 * q_tt + n) * D + 8 * ((4 * (q_ks * KK + i) + g) ^ swz16(n));
  {
    const int r = 4 * g + (n >> 2);
#pragma unroll
    for (int o = 0; o < NDT; ++o) {
      v_at[o] = r * D + 8 * ((2 * (dg * NDT + o) + ((lane >> 1) & 1)) ^ swz16(r)) + 4 * (lane & 1);
    }
  }
  uint64_t zero_row = reinterpret_cast<uint64_t>(g_zero_row);
  asm("" : "+s"(zero_row));  // held, not looked up again for every tile

  // This lane's row of the second product: its draft, head and slope (rows behind the last repeat it, not stored).
  const int row = rg * 16 + n;
  const int tok = min(row, a.rows - 1) / a.group, head = kvh * a.group + min(row, a.rows - 1) - tok * a.group;
  const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
  const uint64_t exist = a.drafts == 64 ? ~uint64_t(0) : (uint64_t(1) << a.drafts) - 1;
  auto mask_of = [&](int b, int i) {  // of draft i
    return exist & (a.mask ? uint64_t(a.mask[b * a.mask_sb + i]) : (uint64_t(2) << i) - 1);
  };
  auto depth_of = [](uint64_t m, int i) { return __builtin_popcountll(m & ~(uint64_t(1) << i)); };

  for (uint32_t p = start; p < end;) {
    const int len = tree_len(a, b);
    const int tiles = tile_count(a, len, T), tile0 = tile_begin(a, len, T);
    const uint32_t rel = p - unit0;
    if (rel >= uint32_t(tiles)) {
      unit0 += uint32_t(tiles);
      ++b;
      continue;
    }
    const int t0 = int(rel), t1 = min(tiles, t0 + int(end - p));

    u32x4 q[KK];
    {
      const int r = min(q_rg * 16 + n, a.rows - 1);
      const int i = r / a.group, h = kvh * a.group + r - i * a.group;
      const uint16_t* src = a.q + b * a.q_sb + i * a.q_st + h * a.q_sh + 32 * KK * q_ks + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[kk] = load16(src + 32 * kk);
    }
    uint64_t seen = mask_of(b, tok);
    const int context = len - a.drafts;  // may be negative: then the drafts before 0 do not exist
    const int position = context + depth_of(seen, tok);
    if (a.window > 0) {  // uniform
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last sequence's depths are read
      if (int(threadIdx.x) < a.drafts) s_depth[threadIdx.x] = depth_of(mask_of(b, threadIdx.x), threadIdx.x);
      __syncthreads();
      seen = drafts_near(seen, s_depth, a.drafts, position - context, a.window);
    }
    // Tiles below this one are seen whole by every row if all their tokens are there and the window reaches.
    const int reach = a.window > 0 ? context + a.drafts - a.window : 0;
    // Rows that no other sequence reads are streamed (kPolicyStream). A sequence whose first block another one also starts
    // with shares pages with it (prefix caching shares whole chains of blocks from the first on).
    bool stream = int64_t(total) * a.hkv >= kStreamTiles;
    if (stream) {
      const int first = a.block_table[b * a.bt_stride];
      for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int other = b0 + lane;
        if (__builtin_amdgcn_ballot_w64(other < a.batch && other != b &&
                                        a.block_table[min(other, a.batch - 1) * a.bt_stride] == first)) {
          stream = false;
        }
      }
    }
    f32x4 o[NDT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x4{};

    // Tiles in pieces whose block ids fit s_ids.
    const int piece = int(min(int64_t(1) << 24, int64_t(kIdSlots - 2) * a.page_size / T));
    for (int a0 = tile0 + t0; a0 < tile0 + t1; a0 += piece) {
      const int a1 = min(tile0 + t1, a0 + piece);
      const int page0 = a0 * T / a.page_size;
      const int pages = (min(a1 * T, len) - 1) / a.page_size - page0 + 1;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last piece is read
      for (int i = threadIdx.x; i < pages; i += 64 * kWaves) {
        s_ids[i] = a.block_table[b * a.bt_stride + page0 + i];
      }
      if (int(threadIdx.x) < a.drafts) s_depth[threadIdx.x] = depth_of(mask_of(b, threadIdx.x), threadIdx.x);
      // Everything that the compiler knows of has landed too, q among it, so that it places no wait of its
      // own (which would also wait for the tiles in flight) in the loop below.
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("s_barrier" ::: "memory");

      // One wave's work for a tile: the addresses of its tokens' rows of this KV head, from which all loads follow; absent
      // tokens are zeros, not what the cache may hold there.
      auto find = [&](int t) __attribute__((always_inline)) {
        const int at = t * T + lane, page = int(__umulhi(2u * uint32_t(at), a.page_magic) >> a.page_shift);
        const int id = s_ids[min(page - page0, kIdSlots - 1)];
        const bool ok = lane < T && at < min(len, a1 * T) && uint32_t(id) < uint32_t(a.num_blocks32);
        const uint64_t off = uint64_t(uint32_t(id * a.page_size + at - page * a.page_size)) * (uint32_t(a.hkv) * (2 * D)) +
                             uint32_t(kvh) * (2 * D);
        const uint64_t here = __builtin_amdgcn_ballot_w64(ok);
        if (lane < T) {
          s_from[t & 3][lane][0] = ok ? reinterpret_cast<uint64_t>(a.k_cache) + off : zero_row;
          s_from[t & 3][lane][1] = ok ? reinterpret_cast<uint64_t>(a.v_cache) + off : zero_row;
        }
        if (lane == 0) s_here[t & 7] = here;
      };
      auto issue_as = [&](auto policy, int t) __attribute__((always_inline)) {  // tile t
        constexpr bool STREAM = decltype(policy)::value;
        const int i = t - a0;
        uint16_t* const to_k = s_k + int(unsigned(i) % kKStages) * kTileElems;
        uint16_t* const to_v = s_v + (i & (kVStages - 1)) * kTileElems;
        uint64_t from[NLD][2];
#pragma unroll
        for (int j = 0; j < NLD; ++j) {
          from[j][0] = s_from[t & 3][load_row + j * kStep][0] + lane_off;
          from[j][1] = s_from[t & 3][load_row + j * kStep][1] + lane_off;
        }
#pragma unroll
        for (int j = 0; j < NLD; ++j) load_lds16_as<STREAM>(from[j][0], to_k + (wave * RPL + j * kStep) * D);
#pragma unroll
        for (int j = 0; j < NLD; ++j) load_lds16_as<STREAM>(from[j][1], to_v + (wave * RPL + j * kStep) * D);
      };
      auto issue = [&](int t) __attribute__((always_inline)) {
        if (stream) issue_as(std::true_type{}, t);
        else issue_as(std::false_type{}, t);
      };
      // Waits for this wave's loads of K of tile t + 1 and of V of tile t, and for the others'. V of a tile is needed a tile
      // later than its K and is loaded behind it.
      auto landed = [&](int t) {
        if (t + 2 < a1) wait_loads_barrier<3 * NLD>();
        else if (t + 1 < a1) wait_loads_barrier<NLD>();
        else wait_loads_barrier<0>();
      };
      // The first product of tile a0 + i. All reads before the first MFMA (sched_barrier: left to itself the
      // compiler reads each operand right before its MFMA and waits for it).
      u32x4 k[JW][KK];
      auto read_keys = [&](int i) {
        const uint16_t* tile = s_k + int(unsigned(i) % kKStages) * kTileElems;
#pragma unroll
        for (int w = 0; w < JW; ++w) {
#pragma unroll
          for (int j = 0; j < KK; ++j) k[w][j] = *reinterpret_cast<const u32x4*>(tile + k_at[j] + 16 * w * D);
        }
      };
      auto score = [&](int i) {
#pragma unroll
        for (int w = 0; w < JW; ++w) {
          f32x4 s[2] = {};
#pragma unroll
          for (int j = 0; j < KK; ++j) s[j & 1] = mfma16x16x32(k[w][j], q[j], s[j & 1], Tag{});
          s[0] += s[1];
          if constexpr (CAP) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][e] = CAP == kWideCap ? capped_wide(s[0][e], a.shape) : capped(s[0][e], a.shape);
          }
          s_s[i & 1][q_ks][q_rg][q_tt + w][lane] = s[0];
        }
      };
      if (wave < 4) find(a0 + wave);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if (a0 + i < a1) issue(a0 + i);
      }
      if (a0 + 2 < a1) wait_loads_barrier<5 * NLD>();  // K of the first tile
      else if (a0 + 1 < a1) wait_loads_barrier<3 * NLD>();
      else wait_loads_barrier<NLD>();
      if (wave < QW) read_keys(0);
      __builtin_amdgcn_sched_barrier(0);
      if (wave < QW) score(0);
      landed(a0);
      for (int t = a0; t < a1; ++t) {
        // Here the scores of tile t, its V and the K of tile t + 1 are in LDS; the stages that tile t + 3 takes are free.
        const int i = t - a0;
        if (t + 3 < a1) issue(t + 3);
        if (wave == (i & (kWaves - 1))) find(t + 4);
        f32x4 y[KS][TT];
#pragma unroll
        for (int j = 0; j < KS; ++j) {
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) y[j][tt] = s_s[i & 1][j][rg][tt][lane];
        }
        if (wave < QW) read_keys(i + 1);  // behind the last tile, of what is there: those scores are not used
        u32x2 v[KP][NDT][2];
        const uint16_t* tile = s_v + (i & (kVStages - 1)) * kTileElems;
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            v[kp][dt][0] = lds_read_tr4(tile + v_at[dt] + 32 * kp * D);
            v[kp][dt][1] = lds_read_tr4(tile + v_at[dt] + (32 * kp + 16) * D);
          }
        }
        const uint64_t mask = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(s_here[t & 7]))))) |
                              uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(s_here[t & 7] >> 32))))) << 32;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 1; j < KS; ++j) {
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) y[0][tt] += y[j][tt];
        }
        float x[4 * TT];
#pragma unroll
        for (int e = 0; e < 4 * TT; ++e) x[e] = CAP ? y[0][e >> 2][e & 3] : y[0][e >> 2][e & 3] * a.shape.scale_log2;
        const int first = t * T;
        constexpr uint64_t kAll = T == 64 ? ~uint64_t(0) : (uint64_t(1) << (T & 63)) - 1;
        if ((mask & kAll) == kAll && first + T <= context && first >= reach) {  // uniform
          if (a.slopes) {
            const float far = float(first + 4 * g - position);
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) x[e] = fmaf(slope, far + float(16 * (e >> 2) + (e & 3)), x[e]);
          }
        } else {
          const int base = first + 4 * g - context;  // draft number of this lane's first key; negative: context
          if (a.slopes) {
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) {
              const int draft = base + 16 * (e >> 2) + (e & 3);
              int depth = s_depth[min(max(draft, 0), kMaxDrafts - 1)];
              asm("" : "+v"(depth));  // read for every lane, not in a branch of those with a draft
              x[e] = fmaf(-slope, float(abs(position - context - (draft < 0 ? draft : depth))), x[e]);
            }
          }
          const int from = a.window > 0 ? position - a.window + 1 - first - 4 * g : 0;
          const uint64_t vis = ((mask & kAll) >> (4 * g)) & tree_seen(base, from, seen);
#pragma unroll
          for (int e = 0; e < 4 * TT; ++e) {
            if (!((vis >> (16 * (e >> 2) + (e & 3))) & 1)) x[e] = -INFINITY;
          }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e + 1 < 4 * TT; e += 2) top = max3(top, x[e], x[e + 1]);
        top = row_group_max(max2(top, x[4 * TT - 1]));
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {  // m = -inf at first
          const float mn = fmaxf(m, top);
          const float c = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
          m = mn;
          l *= c;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt] *= c;
        }
        const float base = m == -INFINITY ? 0.f : m - weight_lift(Tag{});
        if (wave < QW) score(i + 1);
        float sum[4] = {};
#pragma unroll
        for (int e = 0; e < 4 * TT; ++e) {
          x[e] = fast_exp2(x[e] - base);
          sum[e & 3] += x[e];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        // P is rounded to the cache's type for the matrix unit, as in the paged decode: at most half a
        // step of each weight (lifted in fp16, weight_lift), while l sums the unrounded ones in 32 bits.
        u32x4 pb[KP];
#pragma unroll
        for (int e = 0; e < 2 * TT; ++e) pb[e >> 2][e & 3] = pack2(x[2 * e], x[2 * e + 1], Tag{});
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            o[dt] = mfma16x16x32(u32x4{v[kp][dt][0][0], v[kp][dt][0][1], v[kp][dt][1][0], v[kp][dt][1][1]}, pb[kp], o[dt],
                                 Tag{});
          }
        }
        landed(t + 1);  // and every wave is done with tile t
      }
    }

    l = row_group_sum(l);
    if (row < a.rows) {
      if (t0 == 0 && t1 == tiles) {
        const float inv = l != 0.f ? 1.f / l : 0.f;  // a row that sees nothing is zero
        uint16_t* dst = a.out + ((int64_t(b) * a.drafts + tok) * a.hq + head) * D + dg * NDT * 16 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const f32x4 y = o[dt] * inv;
          *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
        }
      } else {
        const int64_t part = (int64_t(run) * a.hkv + kvh) * 2 + (p == start ? 0 : 1);
        float* dst = a.part_o + (part * RB + rg * 16 + n) * D + dg * NDT * 16 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = o[dt];
        if (g == 0 && dg == 0) {
          *reinterpret_cast<float2*>(a.part_ml + (part * RB + rg * 16 + n) * 2) = make_float2(m, l);
        }
      }
    }
    p += uint32_t(t1 - t0);
  }
}

// Joins the parts of sequences that several runs share, each workgroup a few rows, in the order of the runs; rows of
// sequences without tokens are zero.
constexpr int kMergeParts = 1024;  // parts of a row, at most the runs

template <int D, typename Tag>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int rb_rows, int per_group) {
  constexpr int COLS = D / 4, GROUPS = 256 / COLS;
  __shared__ float s_c[kMergeParts];
  __shared__ float s_red[4][2];
  __shared__ f32x4 s_o[GROUPS - 1][COLS];
  const int col = threadIdx.x % COLS, group = threadIdx.x / COLS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per_seq = a.drafts * a.hq;
  const uint32_t total = uint32_t(a.first_tile[a.batch]);
  const Runs runs = runs_of(a, total);
  const int64_t rows = int64_t(a.batch) * per_seq;
  for (int64_t at = int64_t(blockIdx.x) * per_group; at < min(rows, int64_t(blockIdx.x + 1) * per_group); ++at) {
    const int b = int(at / per_seq), rest = int(at - int64_t(b) * per_seq);
    const int tok = rest / a.hq, head = rest - tok * a.hq;
    const int kvh = head / a.group, r = tok * a.group + head - kvh * a.group;
    const uint32_t u0 = uint32_t(a.first_tile[b]), nt = uint32_t(a.first_tile[b + 1]) - u0;
    uint16_t* dst = a.out + at * D + 4 * col;
    if (nt == 0) {
      if (group == 0) *reinterpret_cast<u32x2*>(dst) = u32x2{0, 0};
      continue;
    }
    const int i0 = int(runs.holding(u0)), i1 = int(runs.holding(u0 + nt - 1));
    if (i0 == i1) continue;  // written by its run
    const int parts = i1 - i0 + 1;
    // Part i0 is that run's first one (slot 0) if the sequence begins with the run, else its last (slot 1).
    const int64_t step = int64_t(a.hkv) * 2 * rb_rows;
    const int64_t row0 = i0 * step + int64_t(kvh) * 2 * rb_rows + r;
    const int64_t row_first = row0 + (runs.start(i0) == u0 ? 0 : rb_rows);
    auto part = [&](int i) { return i == 0 ? row_first : row0 + i * step; };
    float top = -INFINITY;
    float m[kMergeParts / 256], l[kMergeParts / 256];
#pragma unroll
    for (int k = 0; k < kMergeParts / 256; ++k) {
      const int i = 256 * k + int(threadIdx.x);
      m[k] = -INFINITY;
      l[k] = 0.f;
      if (i < parts) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + part(i) * 2);
        m[k] = ml.x;
        l[k] = ml.y;
      }
      top = fmaxf(top, m[k]);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    __syncthreads();  // the last row's sums are read
    if (lane == 0) s_red[wave][0] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_red[0][0], s_red[1][0]), fmaxf(s_red[2][0], s_red[3][0]));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kMergeParts / 256; ++k) {
      const float c = fast_exp2(m[k] - base);
      s_c[256 * k + threadIdx.x] = c;
      sum += c * l[k];
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) s_red[wave][1] = sum;
    __syncthreads();
    sum = (s_red[0][1] + s_red[1][1]) + (s_red[2][1] + s_red[3][1]);
    f32x4 o = {};
#pragma unroll 8
    for (int i = group; i < parts; i += GROUPS) {
      o += s_c[i] * *reinterpret_cast<const f32x4*>(a.part_o + part(i) * D + 4 * col);
    }
    if (group > 0) s_o[group - 1][col] = o;
    __syncthreads();
    if (group > 0) continue;
#pragma unroll
    for (int k = 0; k + 1 < GROUPS; ++k) o += s_o[k][col];
    o *= sum != 0.f ? 1.f / sum : 0.f;
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1], Tag{}), pack2(o[2], o[3], Tag{})};
  }
}

int rows_per_block(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

int64_t align16(int64_t x) { return (x + 15) & ~int64_t(15); }

struct TreeSizes {
  int32_t rb, runs;  // rows of a workgroup of this file's kernel, runs of either
  int32_t blocks;    // many rows (blocks > 0): of 128 in the kernel of shaped_rows.h
  int64_t units, o_floats, ml_floats, bytes;
};

// Rows of a KV head beyond which the tree goes to the kernel of shaped_rows.h, whose workgroups take 128 rows at a time:
// row blocks of 64 would each read the cache and repeat the wait for its tiles (16 sequences of 512 to 8,192 tokens with
// 96 rows 133 us in two such blocks, 95 there; 24 of up to 6,000 with 256 rows 340 against 186).
constexpr int kFewRows = 64;

TreeSizes tree_sizes(int32_t batch, int32_t drafts, int32_t hq, int32_t hkv, int32_t head_dim) {
  TreeSizes s{};
  const int64_t rows = int64_t(drafts) * (hq / hkv);
  if (rows > kFewRows) {
    s.blocks = int32_t(ceil_div(rows, kRows));
    s.units = int64_t(batch) * s.blocks * hkv;
    const int64_t lists = int64_t(hkv) * s.blocks;  // workgroups of a run
    const int64_t runs = device_cu_count() * (head_dim == 256 ? 1 : 2) / lists;  // of the workgroups that a GPU holds
    s.runs = int32_t(runs < 1 ? 1 : runs > kMaxParts ? kMaxParts : runs);
    s.o_floats = s.runs * lists * 2 * kRows * head_dim;
    s.ml_floats = s.runs * lists * 2 * kRows * 2;
    s.bytes = align16((s.o_floats + s.ml_floats) * 4 + (int64_t(batch) + 1) * 4);
    return s;
  }
  s.rb = rows_per_block(rows);
  const int64_t runs = device_cu_count() / hkv;  // a workgroup for each KV head, one a CU: its LDS
  s.runs = int32_t(runs < 1 ? 1 : runs > kMergeParts ? kMergeParts : runs);
  s.o_floats = int64_t(s.runs) * hkv * 2 * s.rb * head_dim;
  s.ml_floats = int64_t(s.runs) * hkv * 2 * s.rb * 2;
  s.bytes = align16((s.o_floats + s.ml_floats) * 4 + (int64_t(batch) + 1) * 4);
  return s;
}

int check_tree(const char* who, int32_t batch, int32_t drafts, int32_t hq, int32_t hkv, int32_t head_dim) {
  if (head_dim != 128 && head_dim != 256) {
    return fail(TI_EUNSUPPORTED, "%s: head_dim %d not built (128, 256)", who, head_dim);
  }
  if (drafts < 1 || drafts > kMaxDrafts) {
    return fail(TI_EUNSUPPORTED, "%s: %d drafts not in 1 .. %d", who, drafts, kMaxDrafts);
  }
  if (batch < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || hq > 65536 ||
      int64_t(batch) * drafts * hq > kMaxGridX) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d drafts=%d heads=%d/%d (at most 65536 heads, below 2^24 rows in all)",
                who, batch, drafts, hq, hkv);
  }
  return TI_OK;
}

template <int D, int CAP, typename Tag>
void launch_tree(const TreeArgs& a, int rb, hipStream_t s) {
  const dim3 grid(unsigned(a.runs) * unsigned(a.hkv)), block(64 * kWaves);
  if (rb == 16) hipLaunchKernelGGL((tree_decode_kernel<D, 1, CAP, Tag>), grid, block, 0, s, a);
  else if (rb == 32) hipLaunchKernelGGL((tree_decode_kernel<D, 2, CAP, Tag>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((tree_decode_kernel<D, 4, CAP, Tag>), grid, block, 0, s, a);
  const int64_t rows = int64_t(a.batch) * a.drafts * a.hq;
  const int per_group = int(ceil_div(rows, 8192));
  hipLaunchKernelGGL((tree_merge_kernel<D, Tag>), dim3(unsigned(ceil_div(rows, per_group))), dim3(256), 0, s, a, rb,
                     per_group);
}

}  // namespace
}  // namespace ti

extern "C" int ti_gqa_tree_workspace_bytes(int32_t batch, int32_t num_drafts, int32_t num_q_heads, int32_t num_kv_heads,
                                           int32_t head_dim, int64_t* workspace_bytes_out) {
  using namespace ti;
  const char* who = "ti_gqa_tree_workspace_bytes";
  const int rc = check_tree(who, batch, num_drafts, num_q_heads, num_kv_heads, head_dim);
  if (rc != TI_OK) return rc;
  if (!workspace_bytes_out) return fail(TI_EINVAL, "%s: null output", who);
  *workspace_bytes_out = tree_sizes(batch, num_drafts, num_q_heads, num_kv_heads, head_dim).bytes;
  return TI_OK;
}

extern "C" int ti_gqa_tree_paged(const void* q, int64_t q_stride_b, int64_t q_stride_t, int64_t q_stride_h,
                                 const void* k_cache, const void* v_cache, const int32_t* block_table,
                                 int64_t block_table_stride, const int32_t* seqlen, const int64_t* tree_mask,
                                 int64_t mask_stride_b, const float* slopes, void* out, void* workspace,
                                 int64_t workspace_bytes, int32_t batch, int32_t num_drafts, int32_t num_q_heads,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int64_t num_blocks,
                                 int32_t max_blocks_per_seq, float scale, float softcap, int32_t window, int32_t dtype,
                                 void* stream) {
  using namespace ti;
  const char* who = "ti_gqa_tree_paged";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  const int rc = check_tree(who, batch, num_drafts, num_q_heads, num_kv_heads, head_dim);
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
  // Tiles ahead of the last one and a draft's position lie some hundred tokens behind it; all stays in 32 bits.
  const int64_t tokens = int64_t(max_blocks_per_seq) * page_size;
  if (tokens > INT32_MAX - 1024 ||
      int64_t(batch) * (ceil_div(tokens, 8192 / head_dim) + 1) > INT32_MAX) {
    return fail(TI_EINVAL, "%s: batch %d x max_blocks_per_seq %d x page_size %d is more than one call takes", who, batch,
                max_blocks_per_seq, page_size);
  }
  if (batch == 0) return TI_OK;
  const TreeSizes sz = tree_sizes(batch, num_drafts, num_q_heads, num_kv_heads, head_dim);
  if (sz.units * (ceil_div(tokens, kKeys) + 1) > INT32_MAX) {  // the list is counted in 32 bits
    return fail(TI_EINVAL, "%s: batch %d x %lld tokens x %d x %d heads is more than one call takes", who, batch,
                static_cast<long long>(tokens), num_drafts, num_q_heads);
  }
  if (!q || !seqlen || !out || !workspace || (max_blocks_per_seq > 0 && (!k_cache || !v_cache || !block_table))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
        reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0 ||
      q_stride_b % 8 != 0 || q_stride_t % 8 != 0 || q_stride_h % 8 != 0) {
    return fail(TI_EINVAL, "%s: q, caches, out and workspace must be 16-byte aligned, q strides multiples of 8", who);
  }
  if (workspace_bytes < sz.bytes) {
    return fail(TI_EINVAL, "%s: workspace %lld < %lld bytes", who, static_cast<long long>(workspace_bytes),
                static_cast<long long>(sz.bytes));
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == TI_DTYPE_BF16;
  const int32_t near = window > tokens + kMaxDrafts ? 0 : window;  // none where it is wider than any distance
  if (sz.blocks > 0) {
    RowsArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_sb = q_stride_b;
    a.q_st = q_stride_t;
    a.q_sh = q_stride_h;
    a.k_cache = static_cast<const uint16_t*>(k_cache);
    a.v_cache = static_cast<const uint16_t*>(v_cache);
    a.block_table = block_table;
    a.bt_stride = block_table_stride;
    a.seqlen = seqlen;
    a.slopes = slopes;
    a.out = static_cast<uint16_t*>(out);
    a.o_sh = head_dim;
    a.o_st = int64_t(num_q_heads) * head_dim;
    a.o_sb = a.o_st * num_drafts;
    a.mask = tree_mask;
    a.mask_sb = mask_stride_b;
    a.drafts = num_drafts;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + sz.o_floats;
    a.first_tile = reinterpret_cast<int32_t*>(a.part_ml + sz.ml_floats);
    a.units = int32_t(sz.units);
    a.runs = sz.runs;
    a.batch = batch;
    a.blocks = sz.blocks;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.group = num_q_heads / num_kv_heads;
    a.num_blocks32 = int32_t(num_blocks);
    set_page(a, page_size);
    a.max_blocks = max_blocks_per_seq;
    a.window = near;
    a.shape = score_shape(scale, softcap);
    if (head_dim == 256) {
      if (bf16) launch_rows<256, true, Bf16>(a, s);
      else launch_rows<256, true, F16>(a, s);
    } else {
      if (bf16) launch_rows<128, true, Bf16>(a, s);
      else launch_rows<128, true, F16>(a, s);
    }
    return check_launch(who);
  }
  TreeArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_stride_b;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_cache = static_cast<const uint16_t*>(k_cache);
  a.v_cache = static_cast<const uint16_t*>(v_cache);
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.seqlen = seqlen;
  a.mask = tree_mask;
  a.mask_sb = mask_stride_b;
  a.slopes = slopes;
  a.out = static_cast<uint16_t*>(out);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + sz.o_floats;
  a.first_tile = reinterpret_cast<int32_t*>(a.part_ml + sz.ml_floats);
  a.batch = batch;
  a.drafts = num_drafts;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.rows = num_drafts * a.group;
  a.num_blocks32 = int32_t(num_blocks);
  set_page(a, page_size);
  a.max_blocks = max_blocks_per_seq;
  a.runs = sz.runs;
  a.window = near;
  a.shape = score_shape(scale, softcap);
  const int cap = cap_of(a.shape);
  auto launch = [&](auto tag) {
    using Tag = decltype(tag);
    if (head_dim == 256) {
      if (cap == kWideCap) launch_tree<256, kWideCap, Tag>(a, sz.rb, s);
      else if (cap == kCap) launch_tree<256, kCap, Tag>(a, sz.rb, s);
      else launch_tree<256, kNoCap, Tag>(a, sz.rb, s);
    } else {
      if (cap == kWideCap) launch_tree<128, kWideCap, Tag>(a, sz.rb, s);
      else if (cap == kCap) launch_tree<128, kCap, Tag>(a, sz.rb, s);
      else launch_tree<128, kNoCap, Tag>(a, sz.rb, s);
    }
  };
  if (bf16) launch(Bf16{});
  else launch(F16{});
  return check_launch(who);
}
