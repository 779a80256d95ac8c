// Latent attention on the paged cache, absorbed form (gfx950): each cached token is one vector
// [c | k_r] of L + 64 values (a normalised latent and a rotated key that all heads share), queries are
// given in the same space (q_nope times the key's up-projection, beside the rotated part), and
//   s_j = scale * q . [c_j | k_r_j],  p = softmax(s),  o = sum_j p_j c_j
// so keys and values are the same bytes, read once for every head. A sequence's last `new_tokens` tokens
// are its queries (one when decoding, a few drafted ones when verifying): query i of them sees the
// tokens before position seqlen - new_tokens + i + 1. The caller multiplies o by the value's
// up-projection.
//
// Work: the rows of a sequence are its (query, head) pairs. A workgroup's four waves hold RB rows of one
// sequence and walk its tokens in tiles of 32, which are staged in LDS once and read twice, as K and as
// V. Waves are RG row groups times DS column groups: a wave computes the scores of its group's rows
// (every column group the same ones, so neither scores nor softmax statistics cross waves) and its
// L / DS columns of the output:
//   S^T[32 tokens x 16 rows] = K[32 x E] . Q^T[E x 16]     (16x16x32, E/32 steps, Q in registers)
//   O^T[16 d x 16 rows]     += V^T[16 d x 32] . P^T[32 x 16]
// in which an accumulator's row is its lane's column and the softmax stays in the lane, as in the paged
// prefill; P goes to the second product as the first one left it (the order of a tile's tokens is the
// same in P and in the transposed reads of V).
//
// The batch's tiles (row blocks times sequences times tiles) are one list, cut into runs of equal length,
// one for each workgroup; a unit (sequence, row block) that lies in one run is written by it, others
// leave (m, l, o) parts in 32 bits that a second kernel joins in the order of the runs.
#include "lds_tiles.h"

namespace ti {
namespace {

constexpr int kTile = 32;       // tokens of a tile
constexpr int kRope = 64;       // rotated dimensions beside the latent
constexpr int kIdSlots = 1024;  // block ids staged at a time
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
  int32_t runs, min_tiles;
  float scale_log2;
};

__device__ __align__(16) uint16_t g_zero_latent[512 + kRope] = {};

__device__ __forceinline__ int latent_len(const LatentArgs& a, int b) {
  const int64_t cap = int64_t(a.max_blocks) * a.page_size;
  const int n = max(a.seqlen[b], 0);
  return int64_t(n) > cap ? int(cap) : n;
}

// Runs in use and the run that holds position u of the list (runs are [floor(i T / R), floor((i + 1) T / R))).
__device__ __forceinline__ int64_t runs_of(const LatentArgs& a, int64_t total) {
  return max(int64_t(1), min(int64_t(a.runs), total / a.min_tiles));
}
__device__ __forceinline__ int64_t run_at(int64_t u, int64_t total, int64_t runs) {
  return ((u + 1) * runs - 1) / total;
}

__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

// One load of 16 bytes a lane into LDS: lane i's land at byte lds + 16 i.
__device__ __forceinline__ void load_lds16_at(const uint16_t* src, const uint16_t* lds) {
  const uint32_t m0 = uint32_t(__builtin_amdgcn_readfirstlane(int(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)))));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}

// LDS place of 16-byte chunk c of a tile's row r is c ^ swz8(r) (rows of L + 64 values start 32 banks
// apart). A ds_read_b128 serves rows {0-3, 12-15} of one chunk with rows {4-11} of its neighbour, a
// transposed read two neighbouring chunks of eight rows: both hit every bank quad once.
__device__ __forceinline__ int swz8(int r) {
  const int u = (r >> 1) & 7;
  return ((2 * u) & 7) ^ ((u & 4) ? 5 : 0);
}

template <int N>
__device__ __forceinline__ void wait_loads_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// L: latent size. RT: 16-row tiles of a wave. RG: row groups, DS: column groups (RG * DS = 4 waves).
template <int L, int RT, int RG, int DS, int STAGES, typename Tag>
__global__ __launch_bounds__(256, RT == 1 ? 2 : 1) void latent_decode_kernel(LatentArgs a) {
  constexpr int E = L + kRope;
  constexpr int KK = E / 32;
  constexpr int CH = E / 8;                    // 16-byte chunks of a row
  constexpr int NL = kTile * CH / 64 / 4;      // loads of a wave and tile
  constexpr int NDT = L / 16 / DS;             // 16-column tiles of a wave
  constexpr int RB = RG * RT * 16;
  constexpr int kStageElems = kTile * E;
  static_assert(RG * DS == 4 && kTile * CH % 256 == 0 && STAGES >= 2);

  __shared__ __align__(16) uint16_t s_kv[STAGES * kStageElems];
  __shared__ int s_ids[kIdSlots];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rg = wave / DS, ds = wave % DS;

  // The batch's tiles, this run's share of them, and the sequence in which it starts.
  int64_t total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int nt = b0 + lane < a.batch ? (latent_len(a, b0 + lane) + kTile - 1) / kTile : 0;
    const int incl = wave_scan(nt, lane);
    if (blockIdx.x == 0 && wave == 0 && b0 + lane < a.batch) a.first_tile[b0 + lane] = int(total) + incl - nt;
    total += __builtin_amdgcn_readlane(incl, 63);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.first_tile[a.batch] = int(total);
  total *= a.row_blocks;
  const int64_t runs = runs_of(a, total);
  if (int64_t(blockIdx.x) >= runs || total == 0) return;
  const int64_t start = blockIdx.x * total / runs, end = (blockIdx.x + 1) * total / runs;
  int b = 0;
  int64_t unit0 = 0;  // position of sequence b's first tile
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int nt = b0 + lane < a.batch ? (latent_len(a, b0 + lane) + kTile - 1) / kTile : 0;
    const int incl = wave_scan(nt, lane);
    const int sum = __builtin_amdgcn_readlane(incl, 63);
    if (unit0 + int64_t(sum) * a.row_blocks > start) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(unit0 + int64_t(incl) * a.row_blocks > start);
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      unit0 += int64_t(__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(nt, l)) * a.row_blocks;
      break;
    }
    unit0 += int64_t(sum) * a.row_blocks;
  }

  // This lane's part of a tile's loads: row and byte of the row, and its operand reads.
  int load_row[NL], load_off[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int f = (wave * NL + i) * 64 + lane;
    load_row[i] = f / CH;
    load_off[i] = 8 * ((f % CH) ^ swz8(load_row[i]));
  }
  int k_at[2];  // K chunk 4 kk + g of row n, for even and odd kk (elements)
#pragma unroll
  for (int o = 0; o < 2; ++o) k_at[o] = n * E + 8 * ((4 * o + g) ^ swz8(n));
  int v_at[4];  // V chunk 2 dt + (lane & 2) / 2 of row 4 g + n / 4, for dt % 4
  {
    const int r = 4 * g + (n >> 2);
#pragma unroll
    for (int o = 0; o < 4; ++o) v_at[o] = r * E + 8 * ((2 * o + ((lane >> 1) & 1)) ^ swz8(r)) + 4 * (lane & 1);
  }

  for (int64_t p = start; p < end;) {
    const int len = latent_len(a, b);
    const int nt = (len + kTile - 1) / kTile;
    const int64_t rel = p - unit0;
    if (rel >= int64_t(nt) * a.row_blocks) {
      unit0 += int64_t(nt) * a.row_blocks;
      ++b;
      continue;
    }
    const int rb = int(rel / nt);
    const int t0 = int(rel - int64_t(rb) * nt);
    const int t1 = int(min(int64_t(nt), t0 + (end - p)));
    const int row0 = rb * RB + rg * RT * 16;

    u32x4 q[RT][KK];
    int limit[RT];  // last position that this lane's rows see
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = min(row0 + rt * 16 + n, a.rows - 1);  // rows behind the last are not stored
      const int tok = r / a.heads, h = r - tok * a.heads;
      limit[rt] = len - a.new_tokens + tok;
      const uint16_t* src = a.q + b * a.q_sb + tok * a.q_st + h * a.q_sh + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[rt][kk] = load16(src + 32 * kk);
    }
    f32x4 o[NDT][RT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -INFINITY;
      l[rt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt][rt] = f32x4{};
    }

    // Tiles in pieces whose block ids fit s_ids.
    const int piece = int(min(int64_t(1) << 30, int64_t(kIdSlots - 2) * a.page_size / kTile));
    for (int a0 = t0; a0 < t1; a0 += piece) {
      const int a1 = min(t1, a0 + piece);
      const int page0 = a0 * kTile / a.page_size;
      const int pages = (min(a1 * kTile, len) - 1) / a.page_size - page0 + 1;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last piece is read
      for (int i = threadIdx.x; i < pages; i += 256) s_ids[i] = a.block_table[b * a.bt_stride + page0 + i];
      // Everything that the compiler knows of has landed too, q among it, so that it places no wait of its
      // own (which would also wait for the tiles in flight) in the loop below.
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("s_barrier" ::: "memory");

      uint32_t there[STAGES];  // the staged tiles' tokens that exist, next tile first
      auto issue = [&](int t, int stage) {
        const int pos = t * kTile + (lane & 31);
        int row = -1;
        if (pos < len) {
          const int page = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page_size;
          const int id = s_ids[page - page0];
          if (uint32_t(id) < uint32_t(a.num_blocks32)) row = id * a.page_size + (pos - page * a.page_size);
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          // An absent token's row is zeros, not what the cache may hold there.
          const int r = __shfl(row, load_row[i], 64);
          const uint16_t* base = r >= 0 ? a.cache : g_zero_latent;
          load_lds16_at(base + (uint64_t(uint32_t(max(r, 0))) * E + load_off[i]),
                        s_kv + stage * kStageElems + (wave * NL + i) * 512);
        }
        return uint32_t(__builtin_amdgcn_ballot_w64(row >= 0));
      };
      int stage = 0;
      constexpr int kAhead = STAGES == 2 ? 2 : STAGES - 1;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (a0 + i < a1) there[i] = issue(a0 + i, i);
      }
      for (int t = a0; t < a1; ++t) {
        // Tile t has landed in every wave's part of the stage.
        if constexpr (STAGES == 2) {
          if (t + 1 < a1) wait_loads_barrier<NL>();
          else wait_loads_barrier<0>();
        } else {
          const int more = min(kAhead - 1, a1 - 1 - t);
          if (more >= 2) wait_loads_barrier<2 * NL>();
          else if (more == 1) wait_loads_barrier<NL>();
          else wait_loads_barrier<0>();
        }
        const uint32_t mask = there[0];
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) there[i] = there[i + 1];
        if constexpr (STAGES > 2) {
          const int into = stage == 0 ? STAGES - 1 : stage - 1;
          if (t + kAhead < a1) there[kAhead - 1] = issue(t + kAhead, into);
        }
        const uint16_t* kv = s_kv + stage * kStageElems;

        f32x4 s[2][RT];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[tt][rt] = f32x4{};
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(kv + k_at[kk & 1] + 64 * (kk >> 1) + 16 * tt * E);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[tt][rt] = mfma16x16x32(k, q[rt][kk], s[tt][rt], Tag{});
          }
        }
        const bool whole = mask == 0xffffffffu && t * kTile + kTile - 1 <= len - a.new_tokens;
        u32x4 pb[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][rt][e & 3] * a.scale_log2;
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int j = 16 * (e >> 2) + 4 * g + (e & 3);
              if (!((mask >> j) & 1) || t * kTile + j > limit[rt]) x[e] = -INFINITY;
            }
          }
          float top = x[0];
#pragma unroll
          for (int e = 1; e < 8; ++e) top = max2(top, x[e]);
          top = row_group_max(top);
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
          for (int e = 0; e < 8; ++e) {
            x[e] = fast_exp2(x[e] - base);
            l[rt] += x[e];
          }
          // P is rounded to the cache's type for the matrix unit, as in the paged decode: at most half a
          // step of each weight, while l sums the unrounded ones in 32 bits.
#pragma unroll
          for (int e = 0; e < 4; ++e) pb[rt][e] = pack2(x[2 * e], x[2 * e + 1], Tag{});
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const int at = v_at[dt & 3] + 64 * (dt >> 2) + ds * NDT * 16;
          const u32x2 lo = lds_read_tr4(kv + at), hi = lds_read_tr4(kv + at + 16 * E);
          const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) o[dt][rt] = mfma16x16x32(v, pb[rt], o[dt][rt], Tag{});
        }
        if constexpr (STAGES == 2) {
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stage is read
          if (t + 2 < a1) there[1] = issue(t + 2, stage);
        }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
      }
    }

    const bool complete = t0 == 0 && t1 == nt;
    const int64_t part = (int64_t(blockIdx.x) * 2 + (p == start ? 0 : 1)) * RB + rg * RT * 16;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + n;
      const float lt = row_group_sum(l[rt]);
      if (r >= a.rows) continue;
      if (complete) {
        const float inv = lt != 0.f ? 1.f / lt : 0.f;  // a row that sees nothing is zero
        uint16_t* dst = a.out + (int64_t(b) * a.rows + r) * L + ds * NDT * 16 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const f32x4 y = o[dt][rt] * inv;
          *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
        }
      } else {
        float* dst = a.part_o + (part + rt * 16 + n) * L + ds * NDT * 16 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = o[dt][rt];
        if (g == 0 && ds == 0) {
          float* ml = a.part_ml + (part + rt * 16 + n) * 2;
          ml[0] = m[rt];
          ml[1] = lt;
        }
      }
    }
    p += t1 - t0;
  }
}

// Joins the parts of units that several runs share, one workgroup of L / 4 threads for each row, in the
// order of the runs; rows of sequences without tokens are zero.
template <int L, typename Tag>
__global__ __launch_bounds__(L / 4) void latent_merge_kernel(LatentArgs a, int rb_rows) {
  const int b = blockIdx.x / a.rows, r = blockIdx.x - b * a.rows;
  const int rb = r / rb_rows, rr = r - rb * rb_rows;
  const int f0 = a.first_tile[b], f1 = a.first_tile[b + 1];
  const int64_t total = int64_t(a.first_tile[a.batch]) * a.row_blocks;
  const int64_t nt = f1 - f0;
  uint16_t* dst = a.out + (int64_t(b) * a.rows + r) * L + 4 * threadIdx.x;
  if (nt == 0) {
    *reinterpret_cast<u32x2*>(dst) = u32x2{0, 0};
    return;
  }
  const int64_t runs = runs_of(a, total);
  const int64_t u0 = int64_t(f0) * a.row_blocks + rb * nt;
  const int64_t i0 = run_at(u0, total, runs), i1 = run_at(u0 + nt - 1, total, runs);
  if (i0 == i1) return;  // written by its run
  const int64_t first = (i0 * 2 + (i0 * total / runs == u0 ? 0 : 1)) * rb_rows + rr;
  auto part = [&](int64_t i) { return i == i0 ? first : i * 2 * rb_rows + rr; };
  float top = -INFINITY;
  for (int64_t i = i0; i <= i1; ++i) top = fmaxf(top, a.part_ml[part(i) * 2]);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 o = {};
  float l = 0.f;
#pragma unroll 8
  for (int64_t i = i0; i <= i1; ++i) {
    const int64_t at = part(i);
    const float c = fast_exp2(a.part_ml[at * 2] - base);
    l += c * a.part_ml[at * 2 + 1];
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + at * L + 4 * threadIdx.x);
    o += c * x;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  o *= inv;
  *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1], Tag{}), pack2(o[2], o[3], Tag{})};
}

// Rows of a workgroup for a sequence's rows.
int rows_per_block(int32_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

int plan_runs(int32_t rb) { return device_cu_count() * (rb <= 32 ? 2 : 1); }

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
  s.runs = plan_runs(s.rb);
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
  if (batch < 0 || new_tokens <= 0 || heads <= 0 || int64_t(new_tokens) * heads > (1 << 24) ||
      int64_t(batch) * new_tokens * heads > INT32_MAX) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d new_tokens=%d heads=%d", who, batch, new_tokens, heads);
  }
  return TI_OK;
}

template <int L, typename Tag>
void launch_latent(const LatentArgs& a, int rb, hipStream_t s) {
  const dim3 grid(unsigned(a.runs)), block(256);
  if (rb == 16) hipLaunchKernelGGL((latent_decode_kernel<L, 1, 1, 4, 2, Tag>), grid, block, 0, s, a);
  else if (rb == 32) hipLaunchKernelGGL((latent_decode_kernel<L, 1, 2, 2, 2, Tag>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((latent_decode_kernel<L, 2, 2, 2, 3, Tag>), grid, block, 0, s, a);
  hipLaunchKernelGGL((latent_merge_kernel<L, Tag>), dim3(unsigned(a.batch * a.rows)), dim3(L / 4), 0, s, a, rb);
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
  if (page_size <= 0 || num_blocks < 0 || max_blocks_per_seq < 0 ||
      num_blocks * page_size > INT32_MAX) {
    return fail(TI_EINVAL, "%s: bad cache page_size=%d num_blocks=%lld max_blocks_per_seq=%d (at most "
                "2^31 - 1 rows)", who, page_size, static_cast<long long>(num_blocks), max_blocks_per_seq);
  }
  if (int64_t(max_blocks_per_seq) * page_size > INT32_MAX - kTile) {
    return fail(TI_EINVAL, "%s: max_blocks_per_seq %d x page_size %d exceeds 2^31", who,
                max_blocks_per_seq, page_size);
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
  const LatentSizes sz = latent_sizes(batch, new_tokens, num_heads, latent_dim);
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
  a.min_tiles = 4;
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
