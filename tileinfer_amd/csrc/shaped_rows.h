// Attention of many query rows over the paged cache with shaped scores (gfx950): the kernel behind the shaped prefill
// (queries of packed chunks, each with an interval of keys) and behind wide trees of drafts (TREE: the last tokens of
// every sequence, each with a mask of drafts). A row is a (token, query head) pair of one KV head:
//   s_j = cap tanh(scale q . k_j / cap) - slope |p - p_j|,   o = sum_j softmax(s)_j v_j
//
// Work unit: (sequence, KV head, 128 rows). The tiles of 64 keys that any row sees are loaded straight from the pages
// into LDS and read by all waves, each with 16 C rows (C = 1 of eight waves at D = 256, 2 of four at D = 128):
//   S^T[64 keys x rows] = K . Q^T      (16x16x32, Q in registers)
//   O^T[D x rows]      += V^T . P^T    (16x16x32, V by transposed reads)
// with an accumulator's row its lane's column, so that the softmax stays in the lane. A score of the cap costs three
// exponential-unit instructions, so that the softmax takes as many cycles as the products; it runs beside them, cut in
// two: while the matrix unit computes the scores of tile t + 1, the vector unit turns those of tile t into weights, and
// beside the output of tile t it caps the scores of tile t + 1. One barrier a tile; K is two tiles ahead, V one.
//
// Bound, at D = 256: LDS (each wave reads all of K and V for its 16 rows: 512 KB a tile at some 215 bytes a cycle, and the
// loads write 64 KB) and the loads' way through the CU's address unit (1,250 to 1,350 cycles of a loading wave's 4,600 a
// tile, capped 5,100), the matrix unit being busy 38 % of the time, capped 35 %: 2,048 queries over 10,240 keys within a
// window of 4,096 with 24/4 heads 244 us (845 TFLOP/s), capped 254 to 281; a first chunk of 2,048 82, capped 81 to 92.
// Waves of 32 rows (half the reads) do not fit 256 registers with the softmax beside the products; with 512 (four waves a
// CU) the compiler moved them between register files (379 us against 274 then), without the overlap 279. At D = 128: the
// vector unit (capped 180 us, 150 without, 918 TFLOP/s for the same chunk with 32/8 heads) and unit starts: 12 chunks of
// packed documents with 32/8 heads 76 to 84 us.
#pragma once

#include "lds_tiles.h"
#include "score_shape.h"

namespace ti {
namespace {

constexpr int kRows = 128;     // rows of a unit
constexpr int kKeys = 64;      // keys of a tile
constexpr int kIdSlots = 512;  // block ids staged at a time
constexpr float kSlack = 8.f;  // exp2 units a row maximum may rise before O is rescaled
constexpr int kMaxDrafts = 64;
constexpr int kMaxParts = 512;  // parts of a row

struct RowsArgs {
  const uint16_t* q;  // [tokens, hq, D] at q_st, q_sh; TREE: [B, drafts, hq, D], q_sb too
  int64_t q_sb, q_st, q_sh;
  const uint16_t* k_cache;  // rows [num_blocks * page_size][hkv * D]
  const uint16_t* v_cache;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seqlen;
  const float* slopes;  // [hq] or nullptr
  uint16_t* out;        // as q
  int64_t o_sb, o_st, o_sh;
  // Prefill
  const int32_t* cu_q;
  const int32_t* first_key;  // [total_q] or nullptr
  const int32_t* last_key;
  int32_t total_q, causal;
  // TREE
  const int64_t* mask;  // [B, drafts] at mask_sb, or nullptr: draft i sees the drafts j <= i
  int64_t mask_sb;
  int32_t drafts;
  // Prefill: units in the order of (sequence, block from the last one, KV head). The first `whole` of them are a workgroup's
  // each, the keys of the others are cut into `splits` parts, of which a second kernel joins [part_slot][splits]. There are
  // `slots` of them: units that exist, where `units` counts the longest chunk's for every sequence.
  // TREE: the sequences' tiles are one list, cut into `runs` of equal length, each taken by a workgroup for each KV head and
  // block of rows, side by side: the heads' rows of a token lie side by side in memory, and the blocks (on one XCD) read
  // the same ones. A sequence that lies in one run is written by it, the parts of others [run][block][KV head][first or
  // last one] are joined by a second kernel in the order of the runs. (One list of all heads' and blocks' tiles, 24 trees
  // of 64 over up to 6,000 tokens with 32/8 heads: 258 us; of all heads', the blocks side by side: 237; so 197.)
  float* part_o;   // [..][128][D] unnormalised rows
  float* part_ml;  // [..][128][2] their (m, l), m in exp2 units
  int32_t* first_tile;  // TREE: [B + 1] each sequence's first tile of one unit, and the total
  int32_t units, whole, splits, slots, blocks, runs, batch;
  int32_t hq, hkv, group, num_blocks32, page_size, max_blocks, window;  // window 0: none
  // at / page_size = mulhi(2 at, page_magic) >> page_shift for at below 2^31: page_shift = ceil(log2 page_size),
  // page_magic = ceil(2^(31 + page_shift) / page_size)
  uint32_t page_magic, page_shift;
  ScoreShape shape;
};

__device__ __align__(16) uint16_t g_zero_row[256] = {};

// A sequence's queries, within the tensors whatever the offsets say, and its cached tokens.
template <bool TREE>
struct Queries {
  int q0, q_len, kv_len, offset;
  __device__ __forceinline__ Queries(const RowsArgs& a, int b) {
    if constexpr (TREE) {
      q0 = 0;
      q_len = a.drafts;
    } else {
      q0 = min(max(a.cu_q[b], 0), a.total_q);
      q_len = min(max(a.cu_q[b + 1], q0), a.total_q) - q0;
    }
    const int64_t cap = int64_t(a.max_blocks) * a.page_size;
    const int n = max(a.seqlen[b], 0);
    kv_len = int64_t(n) > cap ? int(cap) : n;
    offset = kv_len - q_len;  // query i's row sits at position offset + i; TREE: the context's length
  }
};

// Prefill: the place of a cut unit's parts. In one sequence its place behind the whole ones; of several, all cut, its place
// among the units that exist, by a wave's sum over the sequences before. Offsets that go back may have more units than
// the rows say, and than there are slots: those behind the last one are not cut.
__device__ __forceinline__ int part_slot(const RowsArgs& a, int b, int qb, int kvh) {
  if (a.batch == 1) return (a.blocks - 1 - qb) * a.hkv + kvh - a.whole;
  int before = 0;
  for (int b0 = 0; b0 < b; b0 += 64) {
    const int other = b0 + int(threadIdx.x & 63);
    const Queries<false> s(a, min(other, b));
    const int n = other < b ? min((s.q_len * a.group + kRows - 1) / kRows, a.blocks) : 0;
    before += __builtin_amdgcn_readlane(wave_prefix_sum(n), 63);
  }
  return (before + qb) * a.hkv + kvh;
}

// TREE: the tiles of a unit, from the first that any of its rows may see.
__device__ __forceinline__ int tree_tile0(const RowsArgs& a, const Queries<true>& s) {
  return a.window > 0 ? max(s.offset - a.window + 1, 0) / kKeys : 0;
}
__device__ __forceinline__ int tree_tiles(const RowsArgs& a, int b) {
  if (b >= a.batch) return 0;
  const Queries<true> s(a, b);
  return (s.kv_len + kKeys - 1) / kKeys - tree_tile0(a, s);
}
// Tiles of a run at least: 32 drafts over 700 tokens with 24/4 heads of 256 30.6 us, with runs of one tile 32.3; long lists
// take the same either way.
constexpr uint32_t kMinRun = 2;
__device__ __forceinline__ Runs tree_runs(const RowsArgs& a, uint32_t total) {
  return Runs(uint32_t(a.runs), total, kMinRun);
}

__device__ __forceinline__ void load_lds16_at(uint64_t src, const uint16_t* lds) {
  const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}

__device__ __forceinline__ uint64_t drafts_seen(const RowsArgs& a, int b, int i) {
  const uint64_t exist = a.drafts == 64 ? ~uint64_t(0) : (uint64_t(1) << a.drafts) - 1;
  return exist & (a.mask ? uint64_t(a.mask[b * a.mask_sb + i]) : (uint64_t(2) << i) - 1);
}

// Bits [0, n) of 64.
__device__ __forceinline__ uint64_t low_bits(int n) {
  return n <= 0 ? 0 : n > 63 ? ~uint64_t(0) : (uint64_t(1) << (n & 63)) - 1;
}

// Which of the keys from draft number `base` on (negative: context) a row sees that sees the drafts of a mask, and the
// context from its bit `from` on. Bits, not a test for each key: a branch for each takes longer than the tile.
__device__ __forceinline__ uint64_t tree_seen(int base, int from, uint64_t drafts) {
  const uint64_t context = low_bits(-base) & ~low_bits(from);
  const uint64_t shifted = base >= 0 ? drafts >> (base & 63) : drafts << (-base & 63);
  return context | (base > 63 || base < -63 ? 0 : shifted);
}

// The drafts of a mask that a window leaves to the draft at `depth` (s_depth: that of each).
__device__ __forceinline__ uint64_t drafts_near(uint64_t mask, const int* s_depth, int drafts, int depth, int window) {
  for (int k = 0; k < drafts; ++k) {
    if (depth - s_depth[k] >= window) mask &= ~(uint64_t(1) << k);
  }
  return mask;
}

template <int D>
struct RowsShape {
  static constexpr int C = D == 256 ? 1 : 2;  // row tiles of a wave
  static constexpr int W = kRows / 16 / C;    // waves
  static constexpr int THREADS = 64 * W;
};

// CAP: how the scores are capped. SLOPES: they are biased (kWideCap: they may be).
template <int D, int CAP, bool SLOPES, bool TREE, typename Tag>
__global__ __launch_bounds__(RowsShape<D>::THREADS, 2) void shaped_rows_kernel(RowsArgs a) {
  constexpr int C = RowsShape<D>::C, W = RowsShape<D>::W;
  constexpr int TT = kKeys / 16, KP = kKeys / 32;
  constexpr int KK = D / 32, NDT = D / 16;
  constexpr int CH = D / 8, RPL = 64 / CH;  // 16-byte chunks of a row, rows of a load
  constexpr int LW = 4;                     // waves that load
  constexpr int NLD = kKeys / RPL / LW;     // their loads of a tile, of K and of V each
  constexpr int kTile = kKeys * D;
  __shared__ __align__(16) uint16_t s_k[2 * kTile];
  __shared__ __align__(16) uint16_t s_v[2 * kTile];
  __shared__ int s_ids[kIdSlots];
  __shared__ int s_range[W][2];
  __shared__ __align__(16) uint64_t s_from[4][kKeys][2];  // addresses of a tile's tokens in K and in V
  __shared__ uint64_t s_here[4];                          // and which of them exist
  __shared__ int4 s_row[kRows];  // (first key, last key, position, slope) of every row
  __shared__ uint64_t s_seen[TREE ? kRows : 1];
  __shared__ int s_depth[TREE ? kMaxDrafts : 1];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  int b = 0, qb = 0, kvh = 0, split = 0, splits = 1, cut = 0;
  uint32_t p = 0, start = 0, end = 0, run = 0, seq0 = 0;  // TREE: places in the list; where sequence b begins
  if constexpr (TREE) {
    uint32_t total = 0;
    int nt = 0, incl = 0;  // of the last 64 sequences looked at
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      nt = tree_tiles(a, b0 + lane);
      incl = wave_prefix_sum(nt);
      if (blockIdx.x == 0 && wave == 0 && b0 + lane < a.batch) a.first_tile[b0 + lane] = int(total) + incl - nt;
      total += uint32_t(__builtin_amdgcn_readlane(incl, 63));
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.first_tile[a.batch] = int(total);
    const Runs runs = tree_runs(a, total);
    const uint32_t pair = blockIdx.x / unsigned(a.hkv);
    kvh = int(blockIdx.x - pair * unsigned(a.hkv));
    qb = int(pair / unsigned(a.runs));
    run = pair - unsigned(qb) * unsigned(a.runs);
    if (run >= runs.runs || total == 0) return;
    start = p = runs.start(run);
    end = runs.start(run + 1);
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (a.batch > 64) {
        nt = tree_tiles(a, b0 + lane);
        incl = wave_prefix_sum(nt);
      }
      const uint32_t sum = uint32_t(__builtin_amdgcn_readlane(incl, 63));
      if (seq0 + sum > start) {
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(seq0 + uint32_t(incl) > start));
        b = b0 + l;
        seq0 += uint32_t(__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(nt, l));
        break;
      }
      seq0 += sum;
    }
  } else {
    int unit = blockIdx.x;
    if (unit >= a.whole) {
      const int rest = a.units - a.whole, i = unit - a.whole;
      split = i / rest;
      unit = a.whole + i - split * rest;
      splits = a.splits;
    }
    const int per_seq = a.blocks * a.hkv;
    b = unit / per_seq;
    const int in_seq = unit - b * per_seq;
    qb = a.blocks - 1 - in_seq / a.hkv;
    kvh = in_seq % a.hkv;
  }

  while (true) {
    const Queries<TREE> sq(a, b);
    const int rows = sq.q_len * a.group;
    int nt = 0, t_rel = 0;  // TREE: the unit's tiles, the run's first one of them
    if constexpr (TREE) {
      nt = tree_tiles(a, b);
      const uint32_t rel = p - seq0;
      if (rel >= uint32_t(nt)) {
        seq0 += uint32_t(nt);
        ++b;
        continue;
      }
      t_rel = int(rel);
    } else {
      if (qb * kRows >= rows) return;
      if (splits > 1) {
        cut = part_slot(a, b, qb, kvh);
        if (cut >= a.slots) {
          if (split > 0) return;
          splits = 1;
        }
      }
    }

    if constexpr (TREE) {
      if (int(threadIdx.x) < a.drafts) {
        s_depth[threadIdx.x] = __builtin_popcountll(drafts_seen(a, b, threadIdx.x) & ~(uint64_t(1) << threadIdx.x));
      }
      __syncthreads();
    }
    // This lane's rows and the keys they see, which stay in LDS: only tiles that a limit or a slope touches need them.
    const int row0 = qb * kRows + wave * 16 * C + n;
    // Everything that the limits come from is loaded first, at once, and Q behind it: loads land in order, and one after the
    // other (each row's queries, then its limits) they took 4 of a short unit's 18 us.
    int tok[C], head[C], first_of[C], last_of[C];
    uint64_t mask_of[C];
    float slope[C];
#pragma unroll
    for (int rt = 0; rt < C; ++rt) {
      const int r = min(row0 + 16 * rt, rows - 1);  // rows behind the last repeat it, not stored
      tok[rt] = r / a.group;
      head[rt] = kvh * a.group + r - tok[rt] * a.group;
    }
    if (SLOPES) {
#pragma unroll
      for (int rt = 0; rt < C; ++rt) slope[rt] = CAP == kWideCap && !a.slopes ? 0.f : a.slopes[head[rt]];
    }
    if constexpr (TREE) {
#pragma unroll
      for (int rt = 0; rt < C; ++rt) mask_of[rt] = drafts_seen(a, b, tok[rt]);
    } else {
      if (a.first_key) {
#pragma unroll
        for (int rt = 0; rt < C; ++rt) first_of[rt] = a.first_key[sq.q0 + tok[rt]];
      }
      if (a.last_key) {
#pragma unroll
        for (int rt = 0; rt < C; ++rt) last_of[rt] = a.last_key[sq.q0 + tok[rt]];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4 q[C][KK];
#pragma unroll
    for (int rt = 0; rt < C; ++rt) {
      const uint16_t* src = a.q + (TREE ? b * a.q_sb : sq.q0 * a.q_st) + tok[rt] * a.q_st + head[rt] * a.q_sh + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[rt][kk] = load16(src + 32 * kk);
    }
    __builtin_amdgcn_sched_barrier(0);
    int some_lo = INT32_MAX, some_hi = -1, all_lo = 0, all_hi = INT32_MAX;
#pragma unroll
    for (int rt = 0; rt < C; ++rt) {
      int pos = sq.offset + tok[rt], lo = 0, hi;
      if constexpr (TREE) {
        uint64_t seen = mask_of[rt];
        const int depth = __builtin_popcountll(seen & ~(uint64_t(1) << tok[rt]));
        pos = sq.offset + depth;
        hi = sq.offset - 1;  // of the context; the drafts by their bits
        if (a.window > 0) seen = drafts_near(seen, s_depth, a.drafts, depth, a.window);
        if (g == 0) s_seen[wave * 16 * C + rt * 16 + n] = seen;
      } else {
        if (a.first_key) lo = max(first_of[rt], 0);
        hi = min(a.last_key ? last_of[rt] : a.causal ? pos : sq.kv_len - 1, sq.kv_len - 1);
      }
      if (a.window > 0 && pos >= a.window) lo = max(lo, pos - a.window + 1);
      if (!TREE && lo > hi) {  // sees nothing
        lo = INT32_MAX;
        hi = -1;
      }
      if (g == 0) {
        s_row[wave * 16 * C + rt * 16 + n] = make_int4(lo, hi, pos, SLOPES ? __float_as_int(slope[rt] * kLog2e) : 0);
      }
      some_lo = min(some_lo, lo);
      some_hi = max(some_hi, hi);
      all_lo = max(all_lo, lo);
      all_hi = min(all_hi, hi);
    }
    // Over the wave's rows: the keys that some row sees, and those that every row sees.
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      some_lo = min(some_lo, __shfl_xor(some_lo, d, 64));
      some_hi = max(some_hi, __shfl_xor(some_hi, d, 64));
      all_lo = max(all_lo, __shfl_xor(all_lo, d, 64));
      all_hi = min(all_hi, __shfl_xor(all_hi, d, 64));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    if (lane == 0) {
      s_range[wave][0] = some_lo;
      s_range[wave][1] = some_hi;
    }
    __syncthreads();
    int key_lo = INT32_MAX, key_hi = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      key_lo = min(key_lo, s_range[w][0]);
      key_hi = max(key_hi, s_range[w][1]);
    }
    key_lo = __builtin_amdgcn_readfirstlane(key_lo);
    key_hi = __builtin_amdgcn_readfirstlane(key_hi);
    int t0, t1;
    if constexpr (TREE) {
      const int tile0 = tree_tile0(a, sq);
      t0 = tile0 + t_rel;
      t1 = min(tile0 + nt, t0 + int(end - p));
    } else {
      const int tile0 = key_hi < 0 ? 0 : key_lo / kKeys, tiles = key_hi < 0 ? 0 : key_hi / kKeys + 1 - tile0;
      t0 = tile0 + int(int64_t(tiles) * split / splits);
      t1 = tile0 + int(int64_t(tiles) * (split + 1) / splits);
    }

    // Operand reads of K row n and of V row 4 g + n / 4 (elements): those of k-step kk and column tile dt are at these with
    // the bits of kk and dt flipped, which the rows' places leave alone.
    const int k_at = n * D + 8 * (g ^ swz16(n));
    const int v_row = 4 * g + (n >> 2);
    const int v_at = v_row * D + 8 * (((lane >> 1) & 1) ^ swz16(v_row)) + 4 * (lane & 1);
    // Load j of a wave takes the tile's rows kStep j + load_row: a lane's chunk is the same in rows 16 apart, in rows 8
    // apart 9 places on.
    constexpr int kStep = LW * RPL;
    static_assert(kStep == 16 || kStep == 8);
    const int load_row = (wave & (LW - 1)) * RPL + lane / CH;
    const uint32_t lane_off = 16 * ((lane % CH) ^ swz16(load_row));
    uint64_t zero_row = reinterpret_cast<uint64_t>(g_zero_row);
    asm("" : "+s"(zero_row));  // held, not looked up again for every tile

    f32x4 o[NDT][C];
    float m[C], l[C];
#pragma unroll
    for (int rt = 0; rt < C; ++rt) {
      m[rt] = -INFINITY;
      l[rt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt][rt] = f32x4{};
    }
    // The scores x between the products are what is cheapest to make and to compare: with a slope the scores in exp2
    // units; with a cap alone r = 1 / (1 + e^2y), of which the score is cap (1 - 2 r) and whose minimum is the
    // maximum of the scores; else the dot products. A weight is exp2(mul x + add).
    constexpr bool kInverse = CAP && !SLOPES;
    constexpr float kMasked = kInverse ? INFINITY : -INFINITY;
    const float mul = SLOPES ? 1.f : CAP ? -2.f * a.shape.cap_log2 : a.shape.scale_log2;
    const float add = kInverse ? a.shape.cap_log2 : 0.f;

    // From the last tile, the nearest keys, to the first: a slope's scores fall from tile to tile that way, where they would
    // rise, and O be brought to a new maximum, with each (24 trees of 64 over up to 6,000 tokens 199 us against 192). Tiles
    // are counted from there, in pieces whose block ids fit s_ids.
    const int piece = int(min(int64_t(1) << 24, int64_t(kIdSlots - 2) * a.page_size / kKeys));
    for (int a0 = 0; a0 < t1 - t0; a0 += piece) {
      const int a1 = min(t1 - t0, a0 + piece);  // tiles t1 - 1 - a0 down to t1 - a1
      const int page0 = (t1 - a1) * kKeys / a.page_size;
      const int pages = (min((t1 - a0) * kKeys, sq.kv_len) - 1) / a.page_size - page0 + 1;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last piece is read
      for (int i = threadIdx.x; i < pages; i += 64 * W) s_ids[i] = a.block_table[b * a.bt_stride + page0 + i];
      __builtin_amdgcn_s_waitcnt(0);  // q has landed too: the loop below has waits of its own alone
      asm volatile("s_barrier" ::: "memory");

      // One wave's work for a tile: the addresses of its 64 tokens' rows of this KV head, from which all loads follow (each
      // wave by itself took 1,000 cycles a tile for its rows); absent tokens are zeros, not what the cache may hold there.
      auto find = [&](int t) __attribute__((always_inline)) {
        const int at = max(t1 - 1 - t, 0) * kKeys + lane;
        const int page = int(__umulhi(2u * uint32_t(at), a.page_magic) >> a.page_shift);
        const int id = s_ids[min(max(page - page0, 0), kIdSlots - 1)];
        const bool ok = t < a1 && at < sq.kv_len && uint32_t(id) < uint32_t(a.num_blocks32);
        const uint64_t off = uint64_t(uint32_t(id * a.page_size + at - page * a.page_size)) * (uint32_t(a.hkv) * (2 * D)) +
                             uint32_t(kvh) * (2 * D);
        const uint64_t here = __builtin_amdgcn_ballot_w64(ok);
        s_from[t & 3][lane][0] = ok ? reinterpret_cast<uint64_t>(a.k_cache) + off : zero_row;
        s_from[t & 3][lane][1] = ok ? reinterpret_cast<uint64_t>(a.v_cache) + off : zero_row;
        if (lane == 0) s_here[t & 3] = here;
      };
      // Loads tile t of K (kv 0) or V (1).
      auto issue = [&](int kv, int t, uint16_t* to) __attribute__((always_inline)) {
        const uint64_t* const from = &s_from[t & 3][load_row][kv];
        uint64_t at[NLD];
#pragma unroll
        for (int j = 0; j < NLD; ++j) at[j] = from[2 * kStep * j];
#pragma unroll
        for (int j = 0; j < NLD; ++j) {
          load_lds16_at(at[j] + (kStep == 8 && (j & 1) ? lane_off ^ (16 * 9) : lane_off),
                        to + ((wave & (LW - 1)) * RPL + j * kStep) * D);
        }
      };

      f32x4 s[TT][C];
      // One k-step of the scores of the tile in K stage `k_off` (its reads a step ahead of the products).
      u32x4 k[2][TT];
      auto read_keys = [&](int k_off, int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          k[kk & 1][tt] = *reinterpret_cast<const u32x4*>(s_k + (k_off ^ (32 * kk)) + 16 * tt * D);
        }
      };
      auto multiply_keys = [&](f32x4 (&to)[TT][C], int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
          for (int rt = 0; rt < C; ++rt) {
            to[tt][rt] = mfma16x16x32(k[kk & 1][tt], q[rt][kk], kk == 0 ? f32x4{} : to[tt][rt], Tag{});
          }
        }
      };
      // A dot product as the score that is kept (without its slope).
      auto shape_of = [&](float dot) __attribute__((always_inline)) {
        if constexpr (CAP == kWideCap) {
          return capped_wide(dot, a.shape);
        } else if constexpr (CAP) {
          const float r = __builtin_amdgcn_rcpf(1.f + fast_exp2(dot * a.shape.cap_in));
          return kInverse ? r : fmaf(-2.f * a.shape.cap_log2, r, a.shape.cap_log2);
        } else {
          return SLOPES ? dot * a.shape.scale_log2 : dot;
        }
      };
      // The slopes and limits of tile t on its scores; the rows' maxima, and O brought to new ones.
      auto limit = [&](int t) __attribute__((always_inline)) {
        const int first = (t1 - 1 - t) * kKeys;
        const uint64_t here = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(s_here[t & 3]))))) |
                              uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(s_here[t & 3] >> 32))))) << 32;
        bool whole = here == ~uint64_t(0) && first >= all_lo && first + kKeys - 1 <= all_hi;  // uniform
        if constexpr (SLOPES) {
          if (!TREE || whole) {
#pragma unroll
            for (int rt = 0; rt < C; ++rt) {
              const int4 row = s_row[wave * 16 * C + rt * 16 + n];
              const float far = float(first + 4 * g - row.z), slope = __int_as_float(row.w);
#pragma unroll
              for (int e = 0; e < 4 * TT; ++e) {
                s[e >> 2][rt][e & 3] = fmaf(-slope, fabsf(far + float(16 * (e >> 2) + (e & 3))), s[e >> 2][rt][e & 3]);
              }
            }
          }
        }
        if (!whole) {
          const uint64_t mine = here >> (4 * g);
#pragma unroll
          for (int rt = 0; rt < C; ++rt) {
            const int4 row = s_row[wave * 16 * C + rt * 16 + n];
            const int from = row.x - first - 4 * g;
            uint64_t seen;  // bit j: key first + 4 g + j
            if constexpr (TREE) {
              const int base = first + 4 * g - sq.offset;
              seen = mine & tree_seen(base, from, s_seen[wave * 16 * C + rt * 16 + n]);
              if constexpr (SLOPES) {
#pragma unroll
                for (int e = 0; e < 4 * TT; ++e) {
                  const int draft = base + 16 * (e >> 2) + (e & 3);
                  int depth = s_depth[min(max(draft, 0), kMaxDrafts - 1)];
                  asm("" : "+v"(depth));  // read for every lane, not in a branch of those with a draft
                  const int dist = row.z - sq.offset - (draft < 0 ? draft : depth);
                  s[e >> 2][rt][e & 3] = fmaf(-__int_as_float(row.w), float(abs(dist)), s[e >> 2][rt][e & 3]);
                }
              }
            } else {
              seen = mine & ~low_bits(from) & low_bits(row.y - first - 4 * g + 1);
            }
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) {
              if (!((seen >> (16 * (e >> 2) + (e & 3))) & 1)) s[e >> 2][rt][e & 3] = kMasked;
            }
          }
        }
        float top[C];
        bool rise = false;
#pragma unroll
        for (int rt = 0; rt < C; ++rt) {
          float x = kInverse ? -s[0][rt][0] : s[0][rt][0];
#pragma unroll
          for (int e = 1; e < 4 * TT - 1; e += 2) {
            const float y = s[e >> 2][rt][e & 3], z = s[(e + 1) >> 2][rt][(e + 1) & 3];
            x = kInverse ? max3(x, -y, -z) : max3(x, y, z);
          }
          const float y = s[TT - 1][rt][3];
          x = row_group_max(max2(x, kInverse ? -y : y));
          top[rt] = fmaf(kInverse ? -mul : mul, x, add);  // a scale is positive
          rise |= top[rt] > m[rt] + kSlack;  // m = -inf at first
        }
        // One condition for all row tiles, so that their exponentials are one block.
        if (__builtin_amdgcn_ballot_w64(rise)) {
#pragma unroll
          for (int rt = 0; rt < C; ++rt) {
            const float mn = fmaxf(m[rt], top[rt]);
            const float c = mn == -INFINITY ? 1.f : fast_exp2(m[rt] - mn);
            m[rt] = mn;
            l[rt] *= c;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt][rt] *= c;
          }
        }
      };

      // Prologue: K of the first two tiles, V of the first; the first tile's scores.
      if (wave < 3) find(a0 + wave);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (wave < LW) {
        issue(0, a0, s_k + (a0 & 1) * kTile);
        issue(1, a0, s_v + (a0 & 1) * kTile);
        if (a0 + 1 < a1) issue(0, a0 + 1, s_k + ((a0 + 1) & 1) * kTile);
      }
      if (a0 + 1 < a1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NLD) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NLD) : "memory");
      {
        const int k_off = (a0 & 1) * kTile + k_at;
        read_keys(k_off, 0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          if (kk + 1 < KK) read_keys(k_off, kk + 1);
          __builtin_amdgcn_sched_barrier(0);
          multiply_keys(s, kk);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int rt = 0; rt < C; ++rt) {
#pragma unroll
          for (int e = 0; e < 4 * TT; ++e) s[e >> 2][rt][e & 3] = shape_of(s[e >> 2][rt][e & 3]);
        }
        limit(a0);
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

      for (int t = a0; t < a1; ++t) {
        // Here K of tile t + 1 and V of tile t are in LDS, s holds the scores of tile t; every wave is done with K of tile
        // t and V of tile t - 1.
        const int stage = t & 1;
        // The oldest wave of each SIMD, which the SIMD serves first and which would wait for the others at the barrier,
        // loads: the loads pass the CU's address unit at 64 bytes a cycle, and a wave stands still meanwhile.
        if (wave < LW) {
          if (t + 2 < a1) issue(0, t + 2, s_k + stage * kTile);
          if (D == 256 && t + 1 < a1) issue(1, t + 1, s_v + (stage ^ 1) * kTile);
        }
        if (wave == W - 1) find(t + 3);

        int k_off = (stage ^ 1) * kTile + k_at, v_off = stage * kTile + v_at;
        asm("" : "+v"(k_off), "+v"(v_off));  // the places of each k-step and column tile are computed, not held
        // The scores of tile t + 1 (behind the last tile, of what is there: they are not used) beside the weights of tile t.
        f32x4 ns[TT][C];
        u32x4 pb[C][KP];
        float base[C];
#pragma unroll
        for (int rt = 0; rt < C; ++rt) base[rt] = add - (m[rt] == -INFINITY ? 0.f : m[rt] - weight_lift(Tag{}));
        read_keys(k_off, 0);
        constexpr int EK = 4 * TT / KK;  // weights of a row tile beside a k-step
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          if (kk + 1 < KK) read_keys(k_off, kk + 1);
          multiply_keys(ns, kk);
#pragma unroll
          for (int rt = 0; rt < C; ++rt) {
#pragma unroll
            for (int i = 0; i < EK; i += 2) {
              const int e = kk * EK + i;
              const float x = fast_exp2(fmaf(s[e >> 2][rt][e & 3], mul, base[rt]));
              const float y = fast_exp2(fmaf(s[e >> 2][rt][(e & 3) + 1], mul, base[rt]));
              l[rt] += x + y;
              // P is rounded to the inputs' type for the matrix unit, as in the paged prefill: at most half a
              // step of each weight (lifted in fp16, weight_lift), while l sums the unrounded ones in 32 bits.
              pb[rt][e >> 3][(e >> 1) & 3] = pack2(x, y, Tag{});
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (D == 128 && wave < LW && t + 1 < a1) issue(1, t + 1, s_v + (stage ^ 1) * kTile);
        // The output of tile t beside the cap of tile t + 1: V in groups of VG column tiles, read a group ahead.
        constexpr int VG = 4, GROUPS = KP * NDT / VG, EV = 4 * TT / GROUPS;
        u32x2 v[2][VG][2];
        auto read_values = [&](int i) __attribute__((always_inline)) {  // group i: of keys 32 (i / (NDT / VG))
          const int kp = i / (NDT / VG), d0 = i % (NDT / VG) * VG;
#pragma unroll
          for (int j = 0; j < VG; ++j) {
            const uint16_t* from = s_v + (v_off ^ (16 * (d0 + j))) + 32 * kp * D;
            v[i & 1][j][0] = lds_read_tr4(from);
            v[i & 1][j][1] = lds_read_tr4(from + 16 * D);
          }
        };
        read_values(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
          const int kp = i / (NDT / VG), d0 = i % (NDT / VG) * VG;
          if (i + 1 < GROUPS) read_values(i + 1);
#pragma unroll
          for (int j = 0; j < VG; ++j) {
            const u32x4 vv = {v[i & 1][j][0][0], v[i & 1][j][0][1], v[i & 1][j][1][0], v[i & 1][j][1][1]};
#pragma unroll
            for (int rt = 0; rt < C; ++rt) o[d0 + j][rt] = mfma16x16x32(vv, pb[rt][kp], o[d0 + j][rt], Tag{});
          }
#pragma unroll
          for (int rt = 0; rt < C; ++rt) {
#pragma unroll
            for (int j = 0; j < EV; ++j) {
              const int e = i * EV + j;
              s[e >> 2][rt][e & 3] = shape_of(ns[e >> 2][rt][e & 3]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (t + 1 < a1) limit(t + 1);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
    }

    const bool complete = TREE ? t_rel == 0 && t1 - t0 == nt : splits == 1;
#pragma unroll
    for (int rt = 0; rt < C; ++rt) {
      const float lt = row_group_sum(l[rt]);
      const int r = row0 + 16 * rt;
      if (r >= rows) continue;
      if (complete) {
        const float inv = lt != 0.f ? 1.f / lt : 0.f;  // a row that sees nothing is zero
        const int tok = r / a.group, head = kvh * a.group + r - tok * a.group;
        uint16_t* dst = a.out + (TREE ? b * a.o_sb : sq.q0 * a.o_st) + tok * a.o_st + head * a.o_sh + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const f32x4 y = o[dt][rt] * inv;
          *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
        }
      } else {
        const int64_t slot = TREE ? ((int64_t(run) * a.blocks + qb) * a.hkv + kvh) * 2 + (p == start ? 0 : 1)
                                  : int64_t(cut) * splits + split;
        const int64_t part = slot * kRows + r - qb * kRows;
        float* dst = a.part_o + part * D + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = o[dt][rt];
        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(m[rt], lt);
      }
    }
    if constexpr (!TREE) return;
    p += uint32_t(t1 - t0);
    if (p >= end) return;
    __syncthreads();  // the unit's limits are read
  }
}

// Joins the parts of a cut unit's rows in their order (of its splits, of the runs), and writes zeros for sequences without
// tokens: one workgroup for 16 rows.
template <int D, bool TREE, typename Tag>
__global__ __launch_bounds__(256) void shaped_merge_kernel(RowsArgs a) {
  constexpr int COLS = D / 4, PAR = 256 / COLS;
  const int item = int(blockIdx.x) / (kRows / 16), r0 = int(blockIdx.x) % (kRows / 16) * 16;
  const int unit = TREE ? item : a.whole + item, per_seq = a.blocks * a.hkv;
  const int b = unit / per_seq, in_seq = unit - b * per_seq;
  const int qb = TREE ? in_seq % a.blocks : a.blocks - 1 - in_seq / a.hkv;
  const int kvh = TREE ? in_seq / a.blocks : in_seq % a.hkv;
  const Queries<TREE> sq(a, b);
  const int rows = sq.q_len * a.group;
  if (qb * kRows + r0 >= rows) return;
  int parts = a.splits;
  int64_t row_first = 0, row_next = 0, step = kRows;
  if constexpr (!TREE) {
    const int slot = part_slot(a, b, qb, kvh);
    if (slot >= a.slots) return;  // not cut
    row_first = row_next = int64_t(slot) * a.splits * kRows;
  } else {
    const uint32_t f0 = uint32_t(a.first_tile[b]), nt = uint32_t(a.first_tile[b + 1]) - f0;
    parts = 0;
    if (nt > 0) {
      const Runs runs = tree_runs(a, uint32_t(a.first_tile[a.batch]));
      const uint32_t i0 = runs.holding(f0), i1 = runs.holding(f0 + nt - 1);
      if (i0 == i1) return;  // written by its run
      parts = int(i1 - i0) + 1;
      // Part i0 is that run's first one (slot 0) if the sequence begins with the run, else its last (slot 1).
      row_next = ((int64_t(i0) * a.blocks + qb) * a.hkv + kvh) * 2 * kRows;
      row_first = row_next + (runs.start(i0) == f0 ? 0 : kRows);
      step = int64_t(a.blocks) * a.hkv * 2 * kRows;
    }
  }
  __shared__ float s_c[PAR][kMaxParts];
  const int col = threadIdx.x % COLS;  // a row's lanes are one wave's
  for (int k = threadIdx.x / COLS; k < 16; k += PAR) {
    const int r = qb * kRows + r0 + k;
    if (r >= rows) break;
    auto part = [&](int i) { return (i == 0 ? row_first : row_next + i * step) + r0 + k; };
    // The parts' weights first, a lane of the row's each (one latency for all of them), then their sum, eight in flight.
    float top = -INFINITY;
    for (int i = col; i < parts; i += COLS) {
      s_c[k % PAR][i] = a.part_ml[part(i) * 2];
      top = fmaxf(top, s_c[k % PAR][i]);
    }
#pragma unroll
    for (int d = COLS / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float base = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    for (int i = col; i < parts; i += COLS) {
      const float c = fast_exp2(s_c[k % PAR][i] - base);
      s_c[k % PAR][i] = c;
      l += c * a.part_ml[part(i) * 2 + 1];
    }
#pragma unroll
    for (int d = COLS / 2; d > 0; d >>= 1) l += __shfl_xor(l, d, 64);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x4 o = {};
#pragma unroll 8
    for (int i = 0; i < parts; ++i) o += s_c[k % PAR][i] * *reinterpret_cast<const f32x4*>(a.part_o + part(i) * D + 4 * col);
    __builtin_amdgcn_wave_barrier();  // the weights are read before the next row's are written
    o *= l != 0.f ? 1.f / l : 0.f;
    const int tok = r / a.group, head = kvh * a.group + r - tok * a.group;
    uint16_t* dst = a.out + (TREE ? b * a.o_sb : sq.q0 * a.o_st) + tok * a.o_st + head * a.o_sh + 4 * col;
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1], Tag{}), pack2(o[2], o[3], Tag{})};
  }
}

template <typename Args>
void set_page(Args& a, int32_t page_size) {
  a.page_size = page_size;
  a.page_shift = page_size == 1 ? 0 : 32 - uint32_t(__builtin_clz(unsigned(page_size) - 1));
  a.page_magic = uint32_t(((uint64_t(1) << (31 + a.page_shift)) + page_size - 1) / uint64_t(page_size));
}

template <int D, bool TREE, typename Tag>
void launch_rows(const RowsArgs& a, hipStream_t s) {
  const dim3 block(RowsShape<D>::THREADS);
  const dim3 grid(unsigned(TREE ? a.runs * a.blocks * a.hkv : a.whole + (a.units - a.whole) * a.splits));
  const int cap = cap_of(a.shape);
  const bool slopes = a.slopes != nullptr;
  if (cap == kWideCap) hipLaunchKernelGGL((shaped_rows_kernel<D, kWideCap, true, TREE, Tag>), grid, block, 0, s, a);
  else if (cap && slopes) hipLaunchKernelGGL((shaped_rows_kernel<D, kCap, true, TREE, Tag>), grid, block, 0, s, a);
  else if (cap) hipLaunchKernelGGL((shaped_rows_kernel<D, kCap, false, TREE, Tag>), grid, block, 0, s, a);
  else if (slopes) hipLaunchKernelGGL((shaped_rows_kernel<D, kNoCap, true, TREE, Tag>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((shaped_rows_kernel<D, kNoCap, false, TREE, Tag>), grid, block, 0, s, a);
  const int joined = TREE ? a.units : a.splits > 1 ? a.units - a.whole : 0;
  if (joined > 0) {
    hipLaunchKernelGGL((shaped_merge_kernel<D, TREE, Tag>), dim3(unsigned(joined) * (kRows / 16)), dim3(256), 0, s, a);
  }
}

}  // namespace
}  // namespace ti
