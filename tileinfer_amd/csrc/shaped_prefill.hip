// Paged prefill with shaped scores (gfx950): the queries of a sequence's chunk over its cached tokens, the chunk's own
// among them, straight from the pages. Query i at position p_i = seqlen - q_len + i sees the keys
//   first_i <= j <= last_i, p_i - j < window
// (documents: first_i the first token of its document; a prefix or an image attended both ways: last_i its end; without
// the arrays 0 and p_i), with the scores
//   s_ij = cap tanh(scale q_i . k_j / cap) - slope_h |p_i - j|
//
// Work unit: (sequence, KV head, 128 rows), a row a (token, query head of the group) pair. A workgroup of four waves of
// 32 rows walks the tiles of 8192 / D keys that any of its rows sees, loaded straight into LDS one tile ahead:
//   S^T[keys x 32 rows] = K . Q^T          (16x16x32, Q in registers)
//   O^T[D x 32 rows]   += V^T . P^T        (16x16x32, V by transposed reads)
// with an accumulator's row its lane's column, as in the paged prefill. Two workgroups fit a CU, so that one's softmax
// runs beside the other's products. Units' tiles may be cut into equal splits, joined by a second kernel in their order,
// where the units do not fill the CUs.
#include "lds_tiles.h"
#include "score_shape.h"

namespace ti {
namespace {

constexpr int kRows = 128;     // rows of a workgroup
constexpr int kStages = 2;
constexpr int kIdSlots = 512;  // block ids staged at a time
constexpr float kSlack = 8.f;  // exp2 units a row maximum may rise before O is rescaled

struct ShapedArgs {
  const uint16_t* q;  // [total_q, hq, D] strides (elements)
  int64_t q_st, q_sh;
  const uint16_t* k_cache;  // rows [num_blocks * page_size][hkv * D]
  const uint16_t* v_cache;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* seqlen;
  const int32_t* first_key;  // [total_q] or nullptr
  const int32_t* last_key;
  const float* slopes;  // [hq] or nullptr
  uint16_t* out;
  int64_t o_st, o_sh;
  float* part_o;   // [batch][blocks][hkv][splits][128][D] unnormalised rows, with splits > 1
  float* part_ml;  // the same without D: (m, l), m in exp2 units
  int32_t total_q, batch, hq, hkv, group, blocks, splits, num_blocks32, page_size, page_shift, max_blocks, causal, window;
  ScoreShape shape;
};

__device__ __align__(16) uint16_t g_zero_row[256] = {};

// A sequence's chunk, within the tensors whatever the offsets say.
struct Chunk {
  int q0, q_len, kv_len, offset;
  __device__ __forceinline__ Chunk(const ShapedArgs& a, int b) {
    q0 = min(max(a.cu_q[b], 0), a.total_q);
    q_len = min(max(a.cu_q[b + 1], q0), a.total_q) - q0;
    const int64_t cap = int64_t(a.max_blocks) * a.page_size;
    const int n = max(a.seqlen[b], 0);
    kv_len = int64_t(n) > cap ? int(cap) : n;
    offset = kv_len - q_len;  // query i sits at position offset + i
  }
};

__device__ __forceinline__ void load_lds16_at(uint64_t src, const uint16_t* lds) {
  const uint32_t m0 = uint32_t(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds)));
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}

template <int D>
struct ShapedTile {
  static constexpr int T = 8192 / D;  // keys: 16 KiB of K, 16 of V
};

template <int D, typename Tag>
__global__ __launch_bounds__(256, 2) void shaped_prefill_kernel(ShapedArgs a) {
  constexpr int T = ShapedTile<D>::T, TT = T / 16, KP = T / 32;
  constexpr int KK = D / 32, NDT = D / 16;
  constexpr int CH = D / 8, RPL = 64 / CH;  // 16-byte chunks of a row, rows of a load
  constexpr int NLD = T / RPL / 4;          // loads of a wave and tile, of K and of V each
  constexpr int kTileElems = T * D;
  __shared__ __align__(16) uint16_t s_k[kStages * kTileElems];
  __shared__ __align__(16) uint16_t s_v[kStages * kTileElems];
  __shared__ int s_ids[kIdSlots];
  __shared__ int s_range[4][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x, b = blockIdx.z;
  const int qb = a.blocks - 1 - int(blockIdx.y) / a.splits, split = int(blockIdx.y) % a.splits;
  const Chunk ch(a, b);
  const int rows = ch.q_len * a.group;
  if (qb * kRows >= rows) return;

  // This lane's two rows: token, head, position and the keys it sees.
  int tok[2], head[2], pos[2], lo[2], hi[2];
  float slope[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int r = min(qb * kRows + wave * 32 + rt * 16 + n, rows - 1);  // rows behind the last repeat it, not stored
    tok[rt] = r / a.group;
    head[rt] = kvh * a.group + r - tok[rt] * a.group;
    pos[rt] = ch.offset + tok[rt];
    lo[rt] = a.first_key ? max(a.first_key[ch.q0 + tok[rt]], 0) : 0;
    if (a.window > 0 && pos[rt] >= a.window) lo[rt] = max(lo[rt], pos[rt] - a.window + 1);
    hi[rt] = min(a.last_key ? a.last_key[ch.q0 + tok[rt]] : a.causal ? pos[rt] : ch.kv_len - 1, ch.kv_len - 1);
    slope[rt] = a.slopes ? a.slopes[head[rt]] * kLog2e : 0.f;
    if (lo[rt] > hi[rt]) {  // sees nothing
      lo[rt] = INT32_MAX;
      hi[rt] = -1;
    }
  }
  // Over the wave's rows: the keys that some row sees, and those that every row sees.
  int some_lo = min(lo[0], lo[1]), some_hi = max(hi[0], hi[1]);
  int all_lo = max(lo[0], lo[1]), all_hi = min(hi[0], hi[1]);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    some_lo = min(some_lo, __shfl_xor(some_lo, d, 64));
    some_hi = max(some_hi, __shfl_xor(some_hi, d, 64));
    all_lo = max(all_lo, __shfl_xor(all_lo, d, 64));
    all_hi = min(all_hi, __shfl_xor(all_hi, d, 64));
  }
  some_lo = __builtin_amdgcn_readfirstlane(some_lo);
  some_hi = __builtin_amdgcn_readfirstlane(some_hi);
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  if (lane == 0) {
    s_range[wave][0] = some_lo;
    s_range[wave][1] = some_hi;
  }
  __syncthreads();
  const int key_lo = __builtin_amdgcn_readfirstlane(min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0])));
  const int key_hi = __builtin_amdgcn_readfirstlane(max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1])));
  const int tile0 = key_hi < 0 ? 0 : key_lo / T, tiles = key_hi < 0 ? 0 : key_hi / T + 1 - tile0;
  const int t0 = tile0 + int(int64_t(tiles) * split / a.splits), t1 = tile0 + int(int64_t(tiles) * (split + 1) / a.splits);

  u32x4 q[2][KK];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const uint16_t* src = a.q + int64_t(ch.q0 + tok[rt]) * a.q_st + head[rt] * a.q_sh + 8 * g;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) q[rt][kk] = load16(src + 32 * kk);
  }

  // This lane's part of a tile's loads: chunk c of row r lies at c ^ swz16(r).
  uint32_t src_off[NLD];
  int src_row[NLD];
#pragma unroll
  for (int i = 0; i < NLD; ++i) {
    src_row[i] = (wave * NLD + i) * RPL + lane / CH;
    src_off[i] = uint32_t(kvh) * (2 * D) + 16 * ((lane % CH) ^ swz16(src_row[i]));
  }
  // Operand reads of K row n and of V row 4 g + n / 4 (elements): those of k-step kk and column tile dt are at these with
  // the bits of kk and dt flipped, which the rows' places leave alone.
  const int k_at = n * D + 8 * (g ^ swz16(n));
  const int v_row = 4 * g + (n >> 2);
  const int v_at = v_row * D + 8 * (((lane >> 1) & 1) ^ swz16(v_row)) + 4 * (lane & 1);
  const uint64_t row_bytes = uint64_t(a.hkv) * (2 * D);
  uint64_t zero_row = reinterpret_cast<uint64_t>(g_zero_row);
  asm("" : "+s"(zero_row));  // held, not looked up again for every tile
  constexpr uint64_t kAll = T == 64 ? ~uint64_t(0) : (uint64_t(1) << (T & 63)) - 1;

  f32x4 o[NDT][2];
  float m[2], l[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt][rt] = f32x4{};
  }
  // A capped or biased score is in exp2 units when it is compared, a plain one still has to be scaled.
  const bool shaped = a.shape.cap_log2 > 0.f || a.slopes != nullptr;
  const float mul = shaped ? 1.f : a.shape.scale_log2;

  // Tiles in pieces whose block ids fit s_ids.
  const int piece = int(min(int64_t(1) << 24, int64_t(kIdSlots - 2) * a.page_size / T));
  for (int a0 = t0; a0 < t1; a0 += piece) {
    const int a1 = min(t1, a0 + piece);
    const int page0 = a0 * T / a.page_size;
    const int pages = (min(a1 * T, ch.kv_len) - 1) / a.page_size - page0 + 1;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last piece is read
    for (int i = threadIdx.x; i < pages; i += 256) s_ids[i] = a.block_table[b * a.bt_stride + page0 + i];
    __builtin_amdgcn_s_waitcnt(0);  // q has landed too: the loop below has waits of its own alone
    asm volatile("s_barrier" ::: "memory");

    // Token lane % T of the tile to load next: position, slot of its block id, place in the block.
    int at = a0 * T + (lane & (T - 1));
    int slot = a.page_shift >= 0 ? at >> a.page_shift : at / a.page_size;
    int in_page = at - slot * a.page_size;
    slot -= page0;
    const int step_slots = T / a.page_size, step_rest = T % a.page_size;
    uint64_t there[kStages];
    // Loads the next tile into `stage`; zeros for an absent token, not what the cache may hold there.
    auto issue = [&](int stage) __attribute__((always_inline)) {
      const int id = s_ids[min(slot, kIdSlots - 1)];
      const bool ok = at < min(ch.kv_len, a1 * T) && uint32_t(id) < uint32_t(a.num_blocks32);
      const uint64_t here = __builtin_amdgcn_ballot_w64(ok) & kAll;
      const int row = ok ? id * a.page_size + in_page : -1;
      at += T;
      slot += step_slots;
      in_page += step_rest;
      const bool over = in_page >= a.page_size;
      slot += over ? 1 : 0;
      in_page -= over ? a.page_size : 0;
#pragma unroll
      for (int j = 0; j < NLD; ++j) {
        const int r = __shfl(row, src_row[j], 64);
        const uint64_t from = uint64_t(uint32_t(r)) * row_bytes + src_off[j];
        load_lds16_at(r >= 0 ? reinterpret_cast<uint64_t>(a.k_cache) + from : zero_row,
                      s_k + stage * kTileElems + (wave * NLD + j) * 512);
        load_lds16_at(r >= 0 ? reinterpret_cast<uint64_t>(a.v_cache) + from : zero_row,
                      s_v + stage * kTileElems + (wave * NLD + j) * 512);
      }
      return here;
    };
    there[0] = issue(0);
    there[1] = a0 + 1 < a1 ? issue(1) : 0;
    for (int t = a0; t < a1; ++t) {
      const int stage = (t - a0) & 1;
      if (t + 1 < a1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NLD) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const uint16_t* const tk = s_k + stage * kTileElems;
      const uint16_t* const tv = s_v + stage * kTileElems;
      const int first = t * T;
      const uint64_t here = there[0];
      if (first <= some_hi && first + T > some_lo) {  // uniform
        f32x4 s[TT][2];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          s[tt][0] = f32x4{};
          s[tt][1] = f32x4{};
        }
        // The next k-step's reads go out before the products of the last one (sched_barrier: left to itself the
        // compiler reads each operand right before its MFMAs and waits for it).
        u32x4 k[2][TT];
        auto read_keys = [&](int kk, u32x4 (&to)[TT]) {
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) to[tt] = *reinterpret_cast<const u32x4*>(tk + (k_at ^ (32 * kk)) + 16 * tt * D);
        };
        read_keys(0, k[0]);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          if (kk + 1 < KK) read_keys(kk + 1, k[(kk + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) s[tt][rt] = mfma16x16x32(k[kk & 1][tt], q[rt][kk], s[tt][rt], Tag{});
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (a.shape.cap_log2 > 0.f) {  // uniform
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) s[e >> 2][rt][e & 3] = capped(s[e >> 2][rt][e & 3], a.shape);
          }
        } else if (shaped) {
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) s[e >> 2][rt][e & 3] *= a.shape.scale_log2;
          }
        }
        if (a.slopes) {
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            const float far = float(first + 4 * g - pos[rt]);
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) {
              s[e >> 2][rt][e & 3] = fmaf(-slope[rt], fabsf(far + float(16 * (e >> 2) + (e & 3))), s[e >> 2][rt][e & 3]);
            }
          }
        }
        if (!(first >= all_lo && first + T - 1 <= all_hi)) {  // uniform
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            const int from = lo[rt] - first - 4 * g, to = hi[rt] - first - 4 * g;
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) {
              const int j = 16 * (e >> 2) + (e & 3);
              if (j < from || j > to) s[e >> 2][rt][e & 3] = -INFINITY;
            }
          }
        }
        if (here != kAll) {  // uniform: a block outside the cache, or the last tile
#pragma unroll
          for (int e = 0; e < 4 * TT; ++e) {
            if (!((here >> (16 * (e >> 2) + 4 * g + (e & 3))) & 1)) s[e >> 2][0][e & 3] = s[e >> 2][1][e & 3] = -INFINITY;
          }
        }
        float top[2];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          top[rt] = s[0][rt][0];
#pragma unroll
          for (int e = 1; e < 4 * TT - 1; e += 2) {
            top[rt] = max3(top[rt], s[e >> 2][rt][e & 3], s[(e + 1) >> 2][rt][(e + 1) & 3]);
          }
          top[rt] = row_group_max(max2(top[rt], s[TT - 1][rt][3])) * mul;  // a scale is positive
        }
        // One condition for both row tiles, so that their exponentials are one block.
        if (__builtin_amdgcn_ballot_w64(top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {  // m = -inf at first
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            const float mn = fmaxf(m[rt], top[rt]);
            const float c = mn == -INFINITY ? 1.f : fast_exp2(m[rt] - mn);
            m[rt] = mn;
            l[rt] *= c;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt][rt] *= c;
          }
        }
        u32x4 pb[2][KP];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          const float base = m[rt] == -INFINITY ? 0.f : m[rt] - weight_lift(Tag{});
          float x[4 * TT];
#pragma unroll
          for (int e = 0; e < 4 * TT; ++e) {
            x[e] = fast_exp2(fmaf(s[e >> 2][rt][e & 3], mul, -base));
            l[rt] += x[e];
          }
          // P is rounded to the inputs' type for the matrix unit, as in the paged prefill: at most half a
          // step of each weight (lifted in fp16, weight_lift), while l sums the unrounded ones in 32 bits.
#pragma unroll
          for (int e = 0; e < 2 * TT; ++e) pb[rt][e >> 2][e & 3] = pack2(x[2 * e], x[2 * e + 1], Tag{});
        }
        // V in groups of eight column tiles: more at once do not fit the registers beside O and Q at D = 256.
        constexpr int VG = NDT < 8 ? NDT : 8;
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
#pragma unroll
          for (int d0 = 0; d0 < NDT; d0 += VG) {
            u32x2 v[VG][2];
#pragma unroll
            for (int i = 0; i < VG; ++i) {
              const uint16_t* from = tv + (v_at ^ (16 * (d0 + i))) + 32 * kp * D;
              v[i][0] = lds_read_tr4(from);
              v[i][1] = lds_read_tr4(from + 16 * D);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < VG; ++i) {
              const u32x4 vv = {v[i][0][0], v[i][0][1], v[i][1][0], v[i][1][1]};
#pragma unroll
              for (int rt = 0; rt < 2; ++rt) o[d0 + i][rt] = mfma16x16x32(vv, pb[rt][kp], o[d0 + i][rt], Tag{});
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stage is read
      there[0] = there[1];
      if (t + kStages < a1) there[1] = issue(stage);
    }
  }

#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const float lt = row_group_sum(l[rt]);
    const int r = qb * kRows + wave * 32 + rt * 16 + n;
    if (r >= rows) continue;
    if (a.splits == 1) {
      const float inv = lt != 0.f ? 1.f / lt : 0.f;  // a row that sees nothing is zero
      uint16_t* dst = a.out + int64_t(ch.q0 + tok[rt]) * a.o_st + head[rt] * a.o_sh + 4 * g;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const f32x4 y = o[dt][rt] * inv;
        *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
      }
    } else {
      const int64_t unit = (int64_t(b) * a.blocks + qb) * a.hkv + kvh;
      const int64_t part = (unit * a.splits + split) * kRows + r - qb * kRows;
      float* dst = a.part_o + part * D + 4 * g;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = o[dt][rt];
      if (g == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(m[rt], lt);
    }
  }
}

// Joins the splits of a unit's rows in their order: one workgroup for 16 rows.
template <int D, typename Tag>
__global__ __launch_bounds__(256) void shaped_merge_kernel(ShapedArgs a) {
  constexpr int COLS = D / 4, PAR = 256 / COLS;
  const int kvh = blockIdx.x, b = blockIdx.z;
  const int qb = int(blockIdx.y) / (kRows / 16), r0 = int(blockIdx.y) % (kRows / 16) * 16;
  const Chunk ch(a, b);
  const int rows = ch.q_len * a.group;
  const int col = threadIdx.x % COLS;
  const int64_t unit = (int64_t(b) * a.blocks + qb) * a.hkv + kvh;
  for (int k = threadIdx.x / COLS; k < 16; k += PAR) {
    const int r = qb * kRows + r0 + k;
    if (r >= rows) break;
    const int64_t part0 = unit * a.splits * kRows + r0 + k;
    float top = -INFINITY;
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, a.part_ml[(part0 + i * kRows) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 o = {};
    float l = 0.f;
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) {
      const int64_t part = part0 + i * kRows;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + part * 2);
      const float c = fast_exp2(ml.x - base);
      l += c * ml.y;
      o += c * *reinterpret_cast<const f32x4*>(a.part_o + part * D + 4 * col);
    }
    o *= l != 0.f ? 1.f / l : 0.f;
    const int tok = r / a.group, head = kvh * a.group + r - tok * a.group;
    uint16_t* dst = a.out + int64_t(ch.q0 + tok) * a.o_st + head * a.o_sh + 4 * col;
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1], Tag{}), pack2(o[2], o[3], Tag{})};
  }
}

bool vec_rows(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
}

struct ShapedSizes {
  int32_t blocks, splits;
  int64_t o_floats, ml_floats, bytes;
};

// Splits of a unit: as many as bring the call's units to the two workgroups that each CU holds, of at least eight tiles.
ShapedSizes shaped_sizes(int32_t batch, int32_t total_q, int32_t max_q, int32_t hq, int32_t hkv, int32_t head_dim,
                         int64_t max_k) {
  ShapedSizes z{};
  const int64_t group = hq / hkv, longest = max_q < total_q ? max_q : total_q;
  z.blocks = int32_t(ceil_div(longest * group, kRows));
  const int64_t units = hkv * (ceil_div(total_q * group, kRows) + batch - 1);
  int64_t splits = 2 * int64_t(device_cu_count()) / (units < 1 ? 1 : units);
  const int64_t most = max_k / (8 * (8192 / head_dim));
  splits = splits > most ? most : splits;
  splits = splits > 64 ? 64 : splits;
  z.splits = int32_t(splits < 1 ? 1 : splits);
  if (z.splits > 1) {
    const int64_t rows = int64_t(batch) * z.blocks * hkv * z.splits * kRows;
    z.o_floats = rows * head_dim;
    z.ml_floats = rows * 2;
    z.bytes = (z.o_floats + z.ml_floats) * 4;
    if (z.bytes > int64_t(1) << 30) {  // ragged beyond use
      z.splits = 1;
      z.o_floats = z.ml_floats = z.bytes = 0;
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

template <int D, typename Tag>
void launch_shaped(const ShapedArgs& a, hipStream_t s) {
  const dim3 grid(unsigned(a.hkv), unsigned(a.blocks) * unsigned(a.splits), unsigned(a.batch));
  hipLaunchKernelGGL((shaped_prefill_kernel<D, Tag>), grid, dim3(256), 0, s, a);
  if (a.splits > 1) {
    const dim3 merge(unsigned(a.hkv), unsigned(a.blocks) * (kRows / 16), unsigned(a.batch));
    hipLaunchKernelGGL((shaped_merge_kernel<D, Tag>), merge, dim3(256), 0, s, a);
  }
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
  *workspace_bytes_out = batch == 0 || total_q == 0 || max_seqlen_q == 0
                             ? 0
                             : shaped_sizes(batch, total_q, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, max_seqlen_k).bytes;
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
  if (tokens > INT32_MAX - 256) {
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
  } else if (z.bytes > 0 && (workspace_bytes < z.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
    return fail(TI_EINVAL, "%s: workspace %lld < %lld bytes, or not 16-byte aligned", who,
                static_cast<long long>(workspace_bytes), static_cast<long long>(z.bytes));
  }
  if (int64_t(z.blocks) * (z.splits > kRows / 16 ? z.splits : kRows / 16) > 65535) {
    return fail(TI_EINVAL, "%s: max_seqlen_q %d too long", who, max_seqlen_q);
  }
  ShapedArgs a{};
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
  a.total_q = total_q;
  a.batch = batch;
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.blocks = z.blocks;
  a.splits = z.splits;
  a.num_blocks32 = int32_t(num_blocks);
  a.page_size = page_size;
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(unsigned(page_size)) : -1;
  a.max_blocks = max_blocks_per_seq;
  a.causal = causal;
  a.window = window > tokens + int64_t(total_q) ? 0 : window;  // wider than any distance
  a.shape = score_shape(scale, softcap);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == TI_DTYPE_BF16;
  if (head_dim == 256) {
    if (bf16) launch_shaped<256, Bf16>(a, s);
    else launch_shaped<256, F16>(a, s);
  } else {
    if (bf16) launch_shaped<128, Bf16>(a, s);
    else launch_shaped<128, F16>(a, s);
  }
  return check_launch(who);
}
