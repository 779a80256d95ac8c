// Latent attention on the paged cache, absorbed form (gfx950): each cached token is one vector
// [c | k_r] of L + 64 values (a normalised latent and a rotated key that all heads share), queries are
// given in the same space (q_nope times the key's up-projection, beside the rotated part), and
//   s_j = scale * q . [c_j | k_r_j],  p = softmax(s),  o = sum_j p_j c_j
// so keys and values are the same bytes, read once for every head. A sequence's last `new_tokens` tokens
// are its queries (one when decoding, a few drafted ones when verifying): query i of them sees the
// tokens before position seqlen - new_tokens + i + 1. The caller multiplies o by the value's
// up-projection.
//
// Work: the rows of a sequence are its (query, head) pairs. A workgroup of eight waves holds RB = 16 RG rows
// of one sequence and walks its tokens in tiles of 32, staged in LDS once and read twice, as K and as V:
//   S^T[16 tokens x 16 rows] = K[16 x E] . Q^T[E x 16]     (16x16x32) cut over the waves by tokens, rows and
//                              k (KS parts of E), Q in registers; the parts go through LDS
//   O^T[16 d x 16 rows]     += V^T[16 d x 32] . P^T[32 x 16]   every wave its 16 rows and L RG / 8 columns
// in which an accumulator's row is its lane's column. The waves of a row group add the parts of S up in the
// same order and keep the same statistics, so the softmax stays in the lane, as in the paged prefill; P
// goes to the second product as S^T lies (the order of a tile's tokens is the same in P and in the
// transposed reads of V). No product is computed twice, so that the waves' LDS reads (178 KB a tile at L = 512)
// take a third of the time in which the tile's 36 KB come from HBM; the next tile's scores are computed beside
// this tile's output, with one barrier a tile. Bound: HBM for long batches (64 sequences of 16,384 tokens with 32
// heads 196 us, 6.2 TB/s), else the start of a run, a tile's chain of reads, products and softmax (1.2 us), and
// the join's launch (16 sequences of 512 to 8,192 tokens with 24 heads 38 us; one of 700 tokens 14 us). Sequences of
// more than 32 rows read their cache once for every 32, and not from L2, since the runs of their row blocks start
// far apart: 64 sequences of 16,384 tokens with 128 heads fetch 4.8 GB of a cache of 1.2, in 675 us (7.2 TB/s, 433
// TFLOP/s); with 64 heads 361 us.
//
// The batch's tiles (row blocks times sequences times tiles) are one list, cut into runs of equal length,
// one for each workgroup; a unit (sequence, row block) that lies in one run is written by it, others
// leave (m, l, o) parts in 32 bits that a second kernel joins in the order of the runs.
#include <type_traits>

#include "lds_tiles.h"

namespace ti {
namespace {

constexpr int kTile = 32;       // tokens of a tile
constexpr int kWaves = 8;
constexpr int kStages = 4;      // latents of tiles in LDS: two in use, two on their way
constexpr int kRopeStages = 3;  // rotated parts: one in use, two on their way
constexpr int kRope = 64;       // rotated dimensions beside the latent
constexpr int kIdSlots = 512;   // block ids staged at a time
constexpr float kSlack = 8.f;   // exp2 units a row maximum may rise before O is rescaled

struct LatentArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;  // q [B, new, H, E] strides (elements)
  const uint16_t* cache;     // rows [num_blocks * page_size][E]
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* seqlen;
  uint16_t* out;  // [B, new, H, L]
  float* part_o;  // [runs][2][RB][L] unnormalised rows
  float* part_ml;  // [runs][2][RB][2] their (m, l), m in exp2 units
  int32_t* first_tile;  // [B + 1] each sequence's first tile, and the total
  int32_t batch, new_tokens, heads, rows, row_blocks, num_blocks32, page_size, page_shift, max_blocks;
  int32_t runs;
  float scale_log2;
};

__device__ __align__(16) uint16_t g_zero_latent[512 + kRope] = {};

__device__ __forceinline__ int latent_len(const LatentArgs& a, int b) {
  const int64_t cap = int64_t(a.max_blocks) * a.page_size;
  const int n = max(a.seqlen[b], 0);
  return int64_t(n) > cap ? int(cap) : n;
}

// Lists of at least this many tiles (75 MB at L = 512) load their rows with the streaming policy: 64 sequences of
// 16,384 tokens 203 us against 224, 64 of 100 to 4,000 in turn with others 58.1 against 61.9; shorter ones,
// which the last-level cache may still hold, keep the default one (one of 32,000: 29.6 us against 31.7).
constexpr uint32_t kStreamTiles = 2048;

// Shortest run of tiles: two, or one where the list is so short that its first tiles' latency is all there is
// (one sequence of 700 tokens, 24 heads: 14.3 us against 16.1 with two; four of 1,000: 16.4 against 15.6).
constexpr uint32_t kShortTiles = 48;

__device__ __forceinline__ Runs runs_of(const LatentArgs& a, uint32_t total) {
  return Runs(uint32_t(a.runs), total, total <= kShortTiles ? 1u : 2u);
}

// One load of 16 bytes a lane into LDS, from base + off of each lane: lane i's land at byte lds + 16 i.
// STREAM: with the nt bit, for bytes that are read once.
template <bool STREAM>
__device__ __forceinline__ void load_lds16_from(uint64_t base, uint32_t off, const uint16_t* lds) {
  const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
  if constexpr (STREAM) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(m0) : "memory");
  } else {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(m0) : "memory");
  }
}
template <bool STREAM>
__device__ __forceinline__ void load_lds16_at(uint64_t src, const uint16_t* lds) {
  const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
  if constexpr (STREAM) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(src), "{m0}"(m0) : "memory");
  } else {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
  }
}

template <int N>
__device__ __forceinline__ void wait_loads_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// L: latent size. RG: row groups of 16. KS: parts of E in the first product.
template <int L, int RG, int KS, typename Tag>
__global__ __launch_bounds__(64 * kWaves, 2) void latent_decode_kernel(LatentArgs a) {
  constexpr int E = L + kRope;
  constexpr int KK = E / 32 / KS;                   // k-steps of a wave
  constexpr int CH = L / 8;                         // 16-byte chunks of a latent
  constexpr int NLAT = kTile * CH / 64 / kWaves;    // loads of a wave and tile: of latents,
  constexpr int kRopeWaves = kTile * 8 / 64;        // and in the first waves one of rotated parts
  constexpr int DG = kWaves / RG;                   // column groups
  constexpr int NDT = L / 16 / DG;                  // 16-column tiles of a wave
  constexpr int RB = RG * 16;
  constexpr int kLat = kTile * L, kRot = kTile * kRope;
  static_assert(2 * RG * KS <= kWaves && KK * KS * 32 == E);

  __shared__ __align__(16) uint16_t s_lat[kStages * kLat];
  __shared__ __align__(16) uint16_t s_rot[kRopeStages * kRot];
  __shared__ f32x4 s_s[2][KS][RG][2][64];  // scores of the next tile and of this one
  __shared__ int s_ids[kIdSlots];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rg = wave % RG, dg = wave / RG;                  // of the second product
  const int q_tt = wave & 1, q_rg = (wave >> 1) % RG;       // of the first
  const int q_ks = min(wave / (2 * RG), KS - 1);             // waves without a part of it repeat one

  // The batch's tiles, this run's share of them, and the sequence in which it starts.
  uint32_t total = 0;
  int nt = 0, incl = 0;  // of the last 64 sequences looked at
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    nt = b0 + lane < a.batch ? (latent_len(a, b0 + lane) + kTile - 1) / kTile : 0;
    incl = wave_prefix_sum(nt);
    if (blockIdx.x == 0 && wave == 0 && b0 + lane < a.batch) a.first_tile[b0 + lane] = int(total) + incl - nt;
    total += uint32_t(__builtin_amdgcn_readlane(incl, 63));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.first_tile[a.batch] = int(total);
  total *= uint32_t(a.row_blocks);
  const Runs runs = runs_of(a, total);
  if (blockIdx.x >= runs.runs || total == 0) return;
  const uint32_t start = runs.start(blockIdx.x), end = runs.start(blockIdx.x + 1);
  int b = 0;
  uint32_t unit0 = 0;  // position of sequence b's first tile
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) {
      nt = b0 + lane < a.batch ? (latent_len(a, b0 + lane) + kTile - 1) / kTile : 0;
      incl = wave_prefix_sum(nt);
    }
    const uint32_t sum = uint32_t(__builtin_amdgcn_readlane(incl, 63));
    if (unit0 + sum * a.row_blocks > start) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(unit0 + uint32_t(incl) * a.row_blocks > start);
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      unit0 += uint32_t(__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(nt, l)) * a.row_blocks;
      break;
    }
    unit0 += sum * a.row_blocks;
  }

  // This lane's part of a tile's loads. Row r's latent is chunks [CH r, CH (r + 1)) of the stage, its
  // rotated part 8 chunks behind the latents; a wave's load takes 64 chunks. Chunk c lies at c ^ swz16(r), of a rotated
  // part at c ^ swz8(r).
  uint32_t lat_off[NLAT];
#pragma unroll
  for (int i = 0; i < NLAT; ++i) {
    const int f = (wave * NLAT + i) * 64 + lane;
    lat_off[i] = 16 * ((f % CH) ^ swz16(f / CH));
  }
  const int rope_row = (wave * 8 + (lane >> 3)) & (kTile - 1);
  const uint32_t rope_off = 2 * L + 16 * ((lane & 7) ^ swz8(rope_row));
  // Its operand reads (elements): of K row 16 q_tt + n each k-step, of V row 4 g + n / 4 chunk
  // 2 dt + (lane & 2) / 2 by dt % 8.
  int k_at[KK], v_at[NDT];
#pragma unroll
  for (int i = 0; i < KK; ++i) {
    const int kk = q_ks * KK + i, r = 16 * q_tt + n;
    k_at[i] = kk < L / 32 ? r * L + 8 * ((4 * kk + g) ^ swz16(n))
                          : r * kRope + 8 * ((4 * (kk - L / 32) + g) ^ swz8(n));
  }
  {
    const int r = 4 * g + (n >> 2);
#pragma unroll
    for (int o = 0; o < NDT; ++o) {
      v_at[o] = r * L + 8 * ((2 * (dg * NDT + o) + ((lane >> 1) & 1)) ^ swz16(r)) + 4 * (lane & 1);
    }
  }
  uint64_t zero_row = reinterpret_cast<uint64_t>(g_zero_latent);
  asm("" : "+s"(zero_row));  // held, not looked up again for every tile

  for (uint32_t p = start; p < end;) {
    const int len = latent_len(a, b);
    const int tiles = (len + kTile - 1) / kTile;
    const uint32_t rel = p - unit0;
    if (rel >= uint32_t(tiles) * a.row_blocks) {
      unit0 += uint32_t(tiles) * a.row_blocks;
      ++b;
      continue;
    }
    const int rb = a.row_blocks == 1 ? 0 : int(rel / uint32_t(tiles));
    const int t0 = int(rel) - rb * tiles;
    const int t1 = min(tiles, t0 + int(end - p));

    u32x4 q[KK];
    {
      const int r = min(rb * RB + q_rg * 16 + n, a.rows - 1);  // rows behind the last are not stored
      const int tok = r / a.heads, h = r - tok * a.heads;
      const uint16_t* src = a.q + b * a.q_sb + tok * a.q_st + h * a.q_sh + 32 * KK * q_ks + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[kk] = load16(src + 32 * kk);
    }
    // Rows that no other workgroup reads are streamed (kPolicyStream). A sequence whose first block another one
    // also starts with shares pages with it (prefix caching shares whole chains of blocks from the first on).
    bool stream = a.row_blocks == 1 && total >= kStreamTiles;
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
    const int row = rb * RB + rg * 16 + n;
    const int limit = len - a.new_tokens + min(row, a.rows - 1) / a.heads;  // last position that it sees
    f32x4 o[NDT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x4{};

    // Tiles in pieces whose block ids fit s_ids.
    const int piece = int(min(int64_t(1) << 24, int64_t(kIdSlots - 2) * a.page_size / kTile));
    for (int a0 = t0; a0 < t1; a0 += piece) {
      const int a1 = min(t1, a0 + piece);
      const int page0 = a0 * kTile / a.page_size;
      const int pages = (min(a1 * kTile, len) - 1) / a.page_size - page0 + 1;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last piece is read
      for (int i = threadIdx.x; i < pages; i += 64 * kWaves) {
        s_ids[i] = a.block_table[b * a.bt_stride + page0 + i];
      }
      // Everything that the compiler knows of has landed too, q among it, so that it places no wait of its
      // own (which would also wait for the tiles in flight) in the loop below.
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("s_barrier" ::: "memory");

      // Token lane % 32 of the tile to load next: position, slot of its block id, place in the block. They
      // advance tile by tile, without a division.
      int pos = a0 * kTile + (lane & (kTile - 1));
      int slot = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page_size;
      int in_page = pos - slot * a.page_size;
      slot -= page0;
      const int step_slots = kTile / a.page_size, step_rest = kTile % a.page_size;
      auto read_id = [&]() { return s_ids[min(slot, kIdSlots - 1)]; };
      // Address of that token's row given its block id, and on to the next tile; zeros for an absent token,
      // not what the cache may hold there.
      uint32_t here = 0;  // the tile's tokens that exist
      auto row_of = [&](int id) {
        const bool ok = pos < min(len, a1 * kTile) && uint32_t(id) < uint32_t(a.num_blocks32);
        here = uint32_t(__builtin_amdgcn_ballot_w64(ok));
        const uint64_t at = reinterpret_cast<uint64_t>(a.cache) +
                            uint64_t(uint32_t(id * a.page_size + in_page)) * (2 * E);
        pos += kTile;
        slot += step_slots;
        in_page += step_rest;
        const bool over = in_page >= a.page_size;
        slot += over ? 1 : 0;
        in_page -= over ? a.page_size : 0;
        return ok ? at : zero_row;
      };
      auto issue_as = [&](auto policy, uint64_t at, int i) __attribute__((always_inline)) {  // tile a0 + i
        constexpr bool STREAM = decltype(policy)::value;
        const int lo = int(uint32_t(at)), hi = int(uint32_t(at >> 32));
        uint16_t* to = s_lat + (i & (kStages - 1)) * kLat;
        if constexpr (CH == 64) {  // a load is one row: its address is uniform
#pragma unroll
          for (int j = 0; j < NLAT; ++j) {
            const int r = wave * NLAT + j;
            const uint64_t src = uint64_t(uint32_t(__builtin_amdgcn_readlane(lo, r))) |
                                 uint64_t(uint32_t(__builtin_amdgcn_readlane(hi, r))) << 32;
            load_lds16_from<STREAM>(src, lat_off[j], to + r * 512);
          }
        } else {
#pragma unroll
          for (int j = 0; j < NLAT; ++j) {
            const int r = ((wave * NLAT + j) * 64 + lane) / CH;
            const uint64_t src = uint64_t(uint32_t(__shfl(lo, r, 64))) | uint64_t(uint32_t(__shfl(hi, r, 64))) << 32;
            load_lds16_at<STREAM>(src + lat_off[j], to + (wave * NLAT + j) * 512);
          }
        }
        if (wave < kRopeWaves) {
          const uint64_t src = uint64_t(uint32_t(__shfl(lo, rope_row, 64))) |
                               uint64_t(uint32_t(__shfl(hi, rope_row, 64))) << 32;
          load_lds16_at<STREAM>(src + rope_off, s_rot + int(unsigned(i) % kRopeStages) * kRot + wave * 512);
        }
      };
      auto issue = [&](uint64_t at, int i) __attribute__((always_inline)) {
        if (stream) issue_as(std::true_type{}, at, i);
        else issue_as(std::false_type{}, at, i);
      };
      // Waits until all but this wave's loads of the `more` newest tiles have landed, and for the others' too.
      auto landed = [&](int more) {
        if (wave < kRopeWaves) {
          if (more >= 2) wait_loads_barrier<2 * (NLAT + 1)>();
          else if (more == 1) wait_loads_barrier<NLAT + 1>();
          else wait_loads_barrier<0>();
        } else {
          if (more >= 2) wait_loads_barrier<2 * NLAT>();
          else if (more == 1) wait_loads_barrier<NLAT>();
          else wait_loads_barrier<0>();
        }
      };
      // The first product of tile a0 + i. All reads before the first MFMA (sched_barrier: left to itself the
      // compiler reads each operand right before its MFMA and waits for it).
      u32x4 k[KK];
      auto read_keys = [&](int i) {
        const uint16_t* lat = s_lat + (i & (kStages - 1)) * kLat;
        const uint16_t* rot = s_rot + int(unsigned(i) % kRopeStages) * kRot;
#pragma unroll
        for (int j = 0; j < KK; ++j) {
          // the last part's last two k-steps are the rotated ones
          const uint16_t* from = j < KK - 2 ? lat : q_ks == KS - 1 ? rot : lat;
          k[j] = *reinterpret_cast<const u32x4*>(from + k_at[j]);
        }
      };
      auto score = [&](int i) {
        f32x4 s[2] = {};
#pragma unroll
        for (int j = 0; j < KK; ++j) s[j & 1] = mfma16x16x32(k[j], q[j], s[j & 1], Tag{});
        if (wave < 2 * RG * KS) s_s[i & 1][q_ks][q_rg][q_tt][lane] = s[0] + s[1];
      };
      uint32_t there[kStages - 1];  // of tiles t, t + 1 and t + 2
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) {
        const uint64_t at = row_of(read_id());
        there[i] = here;
        if (a0 + i < a1) issue(at, i);
      }
      uint64_t next = row_of(read_id());
      uint32_t next_there = here;
      landed(a1 - 1 - a0);
      read_keys(0);
      __builtin_amdgcn_sched_barrier(0);
      score(0);
      landed(min(1, a1 - 2 - a0));
      for (int t = a0; t < a1; ++t) {
        // Here the scores of tile t, its V and the K of tile t + 1 are in LDS and tile t - 1 is free.
        const int i = t - a0;
        if (t + kStages - 1 < a1) issue(next, i + kStages - 1);
        const uint32_t mask = there[0];
        there[0] = there[1];
        there[1] = there[2];
        there[2] = next_there;
        const int next_id = read_id();
        f32x4 y[KS][2];
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          y[j][0] = s_s[i & 1][j][rg][0][lane];
          y[j][1] = s_s[i & 1][j][rg][1][lane];
        }
        read_keys(i + 1);  // behind the last tile, of what is there: those scores are not used
        u32x2 v[NDT][2];
        const uint16_t* lat = s_lat + (i & (kStages - 1)) * kLat;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          v[dt][0] = lds_read_tr4(lat + v_at[dt]);
          v[dt][1] = lds_read_tr4(lat + v_at[dt] + 16 * L);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 1; j < KS; ++j) {
          y[0][0] += y[j][0];
          y[0][1] += y[j][1];
        }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[0][e >> 2][e & 3] * a.scale_log2;
        if (mask != 0xffffffffu || t * kTile + kTile - 1 > len - a.new_tokens) {  // uniform
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = 16 * (e >> 2) + 4 * g + (e & 3);
            if (!((mask >> j) & 1) || t * kTile + j > limit) x[e] = -INFINITY;
          }
        }
        float top = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max2(x[6], x[7]));
        top = row_group_max(top);
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {  // m = -inf at first
          const float mn = fmaxf(m, top);
          const float c = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
          m = mn;
          l *= c;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt] *= c;
        }
        const float base = m == -INFINITY ? 0.f : m - weight_lift(Tag{});
        score(i + 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fast_exp2(x[e] - base);
        l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        // P is rounded to the cache's type for the matrix unit, as in the paged decode: at most half a
        // step of each weight (lifted in fp16, weight_lift), while l sums the unrounded ones in 32 bits.
        const u32x4 pb = {pack2(x[0], x[1], Tag{}), pack2(x[2], x[3], Tag{}), pack2(x[4], x[5], Tag{}),
                          pack2(x[6], x[7], Tag{})};
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          o[dt] = mfma16x16x32(u32x4{v[dt][0][0], v[dt][0][1], v[dt][1][0], v[dt][1][1]}, pb, o[dt], Tag{});
        }
        next = row_of(next_id);
        next_there = here;
        landed(t + kStages - 1 < a1 ? 1 : 0);  // tile t + 2, and every wave is done with tile t
      }
    }

    l = row_group_sum(l);
    if (row < a.rows) {
      if (t0 == 0 && t1 == tiles) {
        const float inv = l != 0.f ? 1.f / l : 0.f;  // a row that sees nothing is zero
        uint16_t* dst = a.out + (int64_t(b) * a.rows + row) * L + dg * NDT * 16 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const f32x4 y = o[dt] * inv;
          *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
        }
      } else {
        const int64_t part = (int64_t(blockIdx.x) * 2 + (p == start ? 0 : 1)) * RB + rg * 16 + n;
        float* dst = a.part_o + part * L + dg * NDT * 16 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = o[dt];
        if (g == 0 && dg == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(m, l);
      }
    }
    p += uint32_t(t1 - t0);
  }
}

// Joins the parts of units that several runs share, one workgroup for each row, in a fixed order; rows of
// sequences without tokens are zero. The parts' weights first (one latency for all of them), then
// 1024 / L groups of threads each sum every so many-th part, eight in flight, and add up through LDS.
constexpr int kMergeParts = 1024;  // parts of a unit whose weights are held at a time

template <int L, typename Tag>
__global__ __launch_bounds__(256) void latent_merge_kernel(LatentArgs a, int rb_rows) {
  constexpr int COLS = L / 4, GROUPS = 256 / COLS;
  __shared__ float s_c[kMergeParts];
  __shared__ float s_red[4][2];
  __shared__ f32x4 s_o[GROUPS - 1][COLS];
  const int b = blockIdx.x / a.rows, r = blockIdx.x - b * a.rows;
  const int rb = r / rb_rows, rr = r - rb * rb_rows;
  const int f0 = a.first_tile[b], f1 = a.first_tile[b + 1];
  const uint32_t total = uint32_t(a.first_tile[a.batch]) * a.row_blocks;
  const uint32_t nt = uint32_t(f1 - f0);
  const int col = threadIdx.x % COLS, group = threadIdx.x / COLS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint16_t* dst = a.out + (int64_t(b) * a.rows + r) * L + 4 * col;
  if (nt == 0) {
    if (group == 0) *reinterpret_cast<u32x2*>(dst) = u32x2{0, 0};
    return;
  }
  const Runs runs = runs_of(a, total);
  const uint32_t u0 = uint32_t(f0) * a.row_blocks + rb * nt;
  const int i0 = int(runs.holding(u0)), i1 = int(runs.holding(u0 + nt - 1));
  if (i0 == i1) return;  // written by its run
  const int parts = i1 - i0 + 1;  // at most the runs, of which there are no more than kMergeParts
  // Part i0 is that run's first one (slot 0) if the unit begins with the run, else its last (slot 1).
  const int64_t row0 = int64_t(i0) * 2 * rb_rows + rr;
  const int64_t row_first = row0 + (runs.start(i0) == u0 ? 0 : rb_rows);
  auto part = [&](int i) { return i == 0 ? row_first : row0 + int64_t(i) * 2 * rb_rows; };
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
    o += s_c[i] * *reinterpret_cast<const f32x4*>(a.part_o + part(i) * L + 4 * col);
  }
  if (group > 0) s_o[group - 1][col] = o;
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int k = 0; k + 1 < GROUPS; ++k) o += s_o[k][col];
  o *= sum != 0.f ? 1.f / sum : 0.f;
  *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1], Tag{}), pack2(o[2], o[3], Tag{})};
}

// Rows of a workgroup for a sequence's rows. Blocks of 64 would halve the passes over the cache, but at L = 512 need
// 130 registers more than a wave has; at L = 256 64 sequences of 10,000 tokens with 64 rows took 124 us against 178,
// but eight of 1,000 20.2 against 17.6 and 24 of up to 6,000 with 96 rows 59 against 52.
int rows_per_block(int32_t rows) { return rows <= 16 ? 16 : 32; }

int64_t align16(int64_t x) { return (x + 15) & ~int64_t(15); }

struct LatentSizes {
  int32_t rb, row_blocks, runs;
  int64_t o_floats, ml_floats, bytes;
};

LatentSizes latent_sizes(int32_t batch, int32_t new_tokens, int32_t heads, int32_t latent) {
  LatentSizes s;
  const int32_t rows = new_tokens * heads;
  s.rb = rows_per_block(rows);
  s.row_blocks = int32_t(ceil_div(rows, s.rb));
  s.runs = device_cu_count() < kMergeParts ? device_cu_count() : kMergeParts;  // one workgroup a CU: its LDS
  s.o_floats = int64_t(s.runs) * 2 * s.rb * latent;
  s.ml_floats = int64_t(s.runs) * 2 * s.rb * 2;
  s.bytes = align16((s.o_floats + s.ml_floats) * 4 + (int64_t(batch) + 1) * 4);
  return s;
}

int check_latent(const char* who, int32_t batch, int32_t new_tokens, int32_t heads, int32_t latent,
                 int32_t rope) {
  if (latent != 512 && latent != 256) {
    return fail(TI_EUNSUPPORTED, "%s: latent_dim %d not built (256, 512)", who, latent);
  }
  if (rope != kRope) return fail(TI_EUNSUPPORTED, "%s: rope_dim %d not built (64)", who, rope);
  // The join has a workgroup for each row.
  if (batch < 0 || new_tokens <= 0 || heads <= 0 || int64_t(new_tokens) * heads > kMaxGridX ||
      int64_t(batch) * new_tokens * heads > kMaxGridX) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d new_tokens=%d heads=%d (below 2^24 rows in all)", who, batch,
                new_tokens, heads);
  }
  return TI_OK;
}

template <int L, typename Tag>
void launch_latent(const LatentArgs& a, int rb, hipStream_t s) {
  const dim3 grid(unsigned(a.runs)), block(64 * kWaves);
  if (rb == 16) hipLaunchKernelGGL((latent_decode_kernel<L, 1, L == 512 ? 3 : 2, Tag>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((latent_decode_kernel<L, 2, 2, Tag>), grid, block, 0, s, a);
  hipLaunchKernelGGL((latent_merge_kernel<L, Tag>), dim3(unsigned(a.batch * a.rows)), dim3(256), 0, s, a, rb);
}

}  // namespace
}  // namespace ti

extern "C" int ti_latent_decode_workspace_bytes(int32_t batch, int32_t new_tokens, int32_t num_heads,
                                                int32_t latent_dim, int64_t* workspace_bytes_out) {
  using namespace ti;
  const char* who = "ti_latent_decode_workspace_bytes";
  int rc = check_latent(who, batch, new_tokens, num_heads, latent_dim, kRope);
  if (rc != TI_OK) return rc;
  if (!workspace_bytes_out) return fail(TI_EINVAL, "%s: null output", who);
  *workspace_bytes_out = latent_sizes(batch, new_tokens, num_heads, latent_dim).bytes;
  return TI_OK;
}

extern "C" int ti_latent_decode_paged(const void* q, int64_t q_stride_b, int64_t q_stride_t,
                                      int64_t q_stride_h, const void* latent_cache,
                                      const int32_t* block_table, int64_t block_table_stride,
                                      const int32_t* seqlen, void* out, void* workspace,
                                      int64_t workspace_bytes, int32_t batch, int32_t new_tokens,
                                      int32_t num_heads, int32_t latent_dim, int32_t rope_dim,
                                      int32_t page_size, int64_t num_blocks, int32_t max_blocks_per_seq,
                                      float scale, int32_t dtype, void* stream) {
  using namespace ti;
  const char* who = "ti_latent_decode_paged";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  int rc = check_latent(who, batch, new_tokens, num_heads, latent_dim, rope_dim);
  if (rc != TI_OK) return rc;
  if (!(scale > 0.f && scale <= kMaxScale)) {
    return fail(TI_EINVAL, "%s: scale %g is not positive or beyond 1e30", who, double(scale));
  }
  if (page_size <= 0 || num_blocks < 0 || max_blocks_per_seq < 0 ||
      num_blocks * page_size > INT32_MAX) {
    return fail(TI_EINVAL, "%s: bad cache page_size=%d num_blocks=%lld max_blocks_per_seq=%d (at most "
                "2^31 - 1 rows)", who, page_size, static_cast<long long>(num_blocks), max_blocks_per_seq);
  }
  if (int64_t(max_blocks_per_seq) * page_size > INT32_MAX - kTile) {
    return fail(TI_EINVAL, "%s: max_blocks_per_seq %d x page_size %d exceeds 2^31", who,
                max_blocks_per_seq, page_size);
  }
  const LatentSizes sz = latent_sizes(batch, new_tokens, num_heads, latent_dim);
  if (int64_t(batch) * sz.row_blocks * (ceil_div(int64_t(max_blocks_per_seq) * page_size, kTile) + 1) > INT32_MAX) {
    return fail(TI_EINVAL, "%s: batch %d x %d tokens x %d rows is more than one call takes", who, batch,
                max_blocks_per_seq * page_size, new_tokens * num_heads);
  }
  if (batch == 0) return TI_OK;
  if (!q || !seqlen || !out || !workspace || (max_blocks_per_seq > 0 && (!latent_cache || !block_table))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(latent_cache) |
        reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0 ||
      q_stride_b % 8 != 0 || q_stride_t % 8 != 0 || q_stride_h % 8 != 0) {
    return fail(TI_EINVAL, "%s: q, cache, out and workspace must be 16-byte aligned, q strides multiples of 8", who);
  }
  if (workspace_bytes < sz.bytes) {
    return fail(TI_EINVAL, "%s: workspace %lld < %lld bytes", who, static_cast<long long>(workspace_bytes),
                static_cast<long long>(sz.bytes));
  }
  LatentArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_stride_b;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.cache = static_cast<const uint16_t*>(latent_cache);
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.seqlen = seqlen;
  a.out = static_cast<uint16_t*>(out);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + sz.o_floats;
  a.first_tile = reinterpret_cast<int32_t*>(a.part_ml + sz.ml_floats);
  a.batch = batch;
  a.new_tokens = new_tokens;
  a.heads = num_heads;
  a.rows = new_tokens * num_heads;
  a.row_blocks = sz.row_blocks;
  a.num_blocks32 = int32_t(num_blocks);
  a.page_size = page_size;
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(unsigned(page_size)) : -1;
  a.max_blocks = max_blocks_per_seq;
  a.runs = sz.runs;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (latent_dim == 512) {
    if (dtype == TI_DTYPE_BF16) launch_latent<512, Bf16>(a, sz.rb, s);
    else launch_latent<512, F16>(a, sz.rb, s);
  } else {
    if (dtype == TI_DTYPE_BF16) launch_latent<256, Bf16>(a, sz.rb, s);
    else launch_latent<256, F16>(a, sz.rb, s);
  }
  return check_launch(who);
}
