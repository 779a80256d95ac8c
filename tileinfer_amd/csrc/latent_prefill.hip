// Latent attention over packed chunks, expanded form (gfx950): every head has its own key and value,
// k_j = [kn_j | k_r_j] and v_j, where kn and v are the up-projected latent (one product of the caller,
// kv [tokens, H, 2 DN] = [kn | v]) and k_r the rotated part that all heads share:
//   s_ij = scale * (qn_i . kn_j + q_r_i . k_r_j),  p_i = softmax_j(s_ij),  o_i = sum_j p_ij v_j
// for the queries i and keys j of one sequence, causal and aligned to the last key (query i sees the
// keys j <= k_len - q_len + i). A first chunk has k_len = q_len, a continuation more keys than queries.
//
// Work unit: (head, sequence, 128 query rows). A workgroup of four waves of 32 rows walks a unit's keys in
// tiles of 64, loaded straight into LDS one tile ahead and read by all waves:
//   S^T[64 keys x 32 rows]  = K[64 x (DN + 64)] . Q^T        (16x16x32, Q in registers)
//   O^T[DN x 32 rows]      += V^T[DN x 64] . P^T             (16x16x32, V by transposed reads)
// with an accumulator's row its lane's column, as in the paged prefill. Two workgroups fit a CU, so that
// one's softmax runs beside the other's products. A workgroup of eight waves gives each half of a tile's keys
// to four of them and joins the two sums through LDS at the unit's end.
//
// Schedules. Per unit: one workgroup each, the last query blocks, which see the most keys, first, and long
// sequences in the order of their keys; no workspace.
// Balanced: the tiles of all units are one list (by head, sequence, block), cut into equal runs, one for each of
// the workgroups that fit the GPU; a unit that lies in one run is written by it, others leave (m, l, o) parts in
// 32 bits that a second kernel joins in the order of the runs. It is for calls whose units do not fill the CUs.
// Consecutive runs go to the same XCD, whose L2 then serves a head's keys to its blocks.
//
// Bound: the matrix units and the softmax's vector work for long chunks (8,192 queries with 24 heads 470 us,
// 1,100 TFLOP/s), the longest unit for a first chunk (2,048 queries 50 us, 650 TFLOP/s), starts of units for short
// ones (24 of 17 to 700 68 us).
#include "lds_tiles.h"

namespace ti {
namespace {

constexpr int kKeys = 64;      // keys of a tile
constexpr int kRope = 64;
constexpr float kSlack = 8.f;  // exp2 units a row maximum may rise before O is rescaled

struct ExpandedArgs {
  const uint16_t* q;  // [total_q, H, DN + 64]
  int64_t q_st, q_sh;
  const uint16_t* kv;  // [total_k, H, 2 DN]
  int64_t kv_st, kv_sh;
  const uint16_t* kr;  // [total_k, 64]
  int64_t kr_st;
  uint16_t* out;  // [total_q, H, DN]
  int64_t o_st, o_sh;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int32_t total_q, total_k, causal, batch, heads, key_groups, by_length;
  float scale_log2;
  // Balanced schedule (runs > 0): parts of cut units, and each sequence's first tile within a head's.
  int32_t runs;
  float* part_o;      // [runs][2][128][DN] unnormalised rows
  float* part_ml;     // [runs][2][128][2] their (m, l), m in exp2 units
  int32_t* seq_tile;  // [B + 1]
};

constexpr int kRows = 128;  // query rows of a workgroup
constexpr int kXcds = 8;

// A sequence's extent, within the tensors whatever the offsets say, and its units' tiles.
struct Seq {
  int q0, q_len, k0, k_len, offset, blocks, shift;
  bool causal;
  __device__ __forceinline__ Seq(const ExpandedArgs& a, int b) {
    q0 = min(max(a.cu_q[b], 0), a.total_q);
    q_len = min(max(a.cu_q[b + 1], q0), a.total_q) - q0;
    k0 = min(max(a.cu_k[b], 0), a.total_k);
    k_len = min(max(a.cu_k[b + 1], k0), a.total_k) - k0;
    offset = k_len - q_len;  // query i sits at key position offset + i
    blocks = (q_len + kRows - 1) / kRows;
    shift = (offset + (offset > 0 ? kKeys - 1 : 0)) / kKeys;  // offset / 64 rounded up
    causal = a.causal;
  }
  // Keys that block qb sees: all under no mask, and to the last one for the last block.
  __device__ __forceinline__ int key_end(int qb) const {
    const int end = !causal || qb == blocks - 1 ? k_len : offset + kRows * (qb + 1);
    return end > 0 ? end : 0;
  }
  __device__ __forceinline__ int tiles(int qb) const { return (key_end(qb) + kKeys - 1) / kKeys; }
  // Tiles of the blocks before qb. Under the mask those of block i < blocks - 1 are 2 (i + 1) + shift, if
  // positive.
  __device__ __forceinline__ int before(int qb) const {
    const int n = max(min(qb, blocks - 1), 0);
    int sum;
    if (causal) {
      const int none = min(max(-shift / 2, 0), n);
      sum = n * (n + 1 + shift) - none * (none + 1 + shift);
    } else {
      sum = n * ((k_len + kKeys - 1) / kKeys);
    }
    return qb == blocks && blocks > 0 ? sum + tiles(blocks - 1) : sum;
  }
};

constexpr uint32_t kMinRun = 4;  // tiles of a run (the host takes the other schedule for lists beyond 32 bits)

// KG: key groups of four waves each; a group takes 64 / KG keys of a tile.
template <int DN, int KG, bool BALANCED, typename Tag>
__global__ __launch_bounds__(256 * KG, 2) void latent_prefill_kernel(ExpandedArgs a) {
  constexpr int TT = 4 / KG, KP = 2 / KG;   // 16-key and 32-key tiles of a wave
  constexpr int STAGES = KG == 1 ? 2 : 3;
  constexpr int KN = DN / 32;               // k-steps of the unrotated part
  constexpr int NDT = DN / 16;
  constexpr int ROW = 2 * DN;               // elements of a [kn | v] row
  constexpr int CH = ROW / 8;
  constexpr int NKV = kKeys * CH / 256 / KG;  // loads of a wave and tile
  constexpr int NKR = kKeys * 8 / 256 / KG;
  constexpr int NL = NKV + NKR;
  constexpr int kStage = kKeys * (ROW + kRope);
  static_assert(CH % 16 == 0);
  static_assert(KG == 1 || STAGES * kStage * 2 >= 4 * (2 * NDT * 1024 + 2 * 512), "the stages hold a group's sums");
  __shared__ __align__(16) uint16_t s_tile[STAGES * kStage];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rw = wave & 3, key0 = 32 * (wave >> 2);  // rows and keys of a tile that this wave takes

  int h, b, qb;
  uint32_t p = 0, start = 0, end = 1;  // the run's positions in the list, and the next one
  int t_first = 0;                     // first tile of the next unit
  uint32_t run = 0;
  if constexpr (BALANCED) {
    int per_head = 0, nt = 0, incl = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      nt = 0;
      if (b0 + lane < a.batch) {
        const Seq s(a, b0 + lane);
        nt = s.before(s.blocks);
      }
      incl = wave_prefix_sum(nt);
      if (blockIdx.x == 0 && wave == 0 && b0 + lane < a.batch) a.seq_tile[b0 + lane] = per_head + incl - nt;
      per_head += __builtin_amdgcn_readlane(incl, 63);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.seq_tile[a.batch] = per_head;
    const uint32_t total = uint32_t(per_head) * a.heads;
    const Runs runs(uint32_t(a.runs), total, kMinRun);
    run = blockIdx.x;
    if (run >= runs.runs || total == 0) return;
    if (runs.runs % kXcds == 0) run = run % kXcds * (runs.runs / kXcds) + run / kXcds;
    start = p = runs.start(run);
    end = runs.start(run + 1);
    h = int(p / uint32_t(per_head));
    int rel = int(p - uint32_t(h) * per_head);
    b = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (a.batch > 64) {
        nt = 0;
        if (b0 + lane < a.batch) {
          const Seq s(a, b0 + lane);
          nt = s.before(s.blocks);
        }
        incl = wave_prefix_sum(nt);
      }
      const int sum = __builtin_amdgcn_readlane(incl, 63);
      if (sum > rel) {
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > rel));
        b = b0 + l;
        rel -= __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(nt, l);
        break;
      }
      rel -= sum;
    }
    const Seq s(a, b);
    int lo = 0, hi = s.blocks - 1;  // the first block whose end lies behind rel
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s.before(mid + 1) > rel) hi = mid;
      else lo = mid + 1;
    }
    qb = lo;
    t_first = rel - s.before(qb);
  } else {
    // A sequence's last blocks first; its blocks stay side by side, for their keys in L2 (last blocks of all
    // sequences first: 24 chunks of up to 300 over up to 4,000 keys 274 us against 196). Long sequences in the
    // order of their keys, so that the last units to start are short: 12 ragged chunks over up to 4,000 keys 129 us
    // against 148 (one box; 126 to 140 over several), four prompts of 500 to 3,000 104 against 115. The order costs a
    // unit about a microsecond: prompts of 17 to 700 stay as they come (67 us against 72).
    h = blockIdx.x;
    b = blockIdx.z;
    if (a.by_length) {
      const int len = lane < a.batch ? Seq(a, lane).k_len : -1;
      int rank = 0;
      for (int i = 0; i < a.batch; ++i) {
        const int other = __builtin_amdgcn_readlane(len, i);
        rank += other > len || (other == len && i < lane) ? 1 : 0;
      }
      b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.batch && rank == int(blockIdx.z)));
    }
    qb = Seq(a, b).blocks - 1 - int(blockIdx.y);
    if (qb < 0) return;
  }

  // Byte offsets of this lane's loads within a tile: chunk c of row r lies at c ^ swz16(r) of its [kn | v], at c ^ swz8(r)
  // of its k_r.
  uint32_t kv_at[NKV], kr_at[NKR];
#pragma unroll
  for (int i = 0; i < NKV; ++i) {
    const int f = (wave * NKV + i) * 64 + lane, r = f / CH;
    kv_at[i] = uint32_t(r) * uint32_t(a.kv_st * 2) + 16 * ((f % CH) ^ swz16(r));
  }
#pragma unroll
  for (int i = 0; i < NKR; ++i) {
    const int f = (wave * NKR + i) * 64 + lane, r = f >> 3;
    kr_at[i] = uint32_t(r) * uint32_t(a.kr_st * 2) + 16 * ((f & 7) ^ swz8(r));
  }
  // Operand reads of row n (K) and of row 4 g + n / 4 (V), elements: those of k-step kk and column tile dt are
  // at these with the bits of kk and dt flipped, which the rows' places leave alone.
  const int k_at = (key0 + n) * ROW + 8 * (g ^ swz16(n));
  const int r_at = kKeys * ROW + (key0 + n) * kRope + 8 * (g ^ swz8(n));
  const int v_row = 4 * g + (n >> 2);
  const int v_at = (key0 + v_row) * ROW + 8 * ((DN / 8 + ((lane >> 1) & 1)) ^ swz16(v_row)) + 4 * (lane & 1);

  while (true) {
    const Seq sq(a, b);
    const int tiles = sq.tiles(qb), k_end = sq.key_end(qb);
    const int t0 = BALANCED ? t_first : 0;
    const int t1 = BALANCED ? min(tiles, t0 + int(end - p)) : tiles;

    // Q operands of this wave's rows; rows behind the last repeat it and are not stored.
    u32x4 q[2][KN + 2];
    int limit[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const int r = min(qb * kRows + rw * 32 + rt * 16 + n, sq.q_len - 1);
      limit[rt] = a.causal ? sq.offset + r : sq.k_len - 1;
      const uint16_t* src = a.q + int64_t(sq.q0 + r) * a.q_st + h * a.q_sh + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KN + 2; ++kk) q[rt][kk] = load16(src + 32 * kk);
    }

    auto issue = [&](int t, int stage) {
      const int valid = min(kKeys, k_end - t * kKeys);  // keys past it read as zero
      const uint16_t* kv = a.kv + int64_t(sq.k0 + t * kKeys) * a.kv_st + h * a.kv_sh;
      const uint16_t* kr = a.kr + int64_t(sq.k0 + t * kKeys) * a.kr_st;
      const u32x4 rkv = rsrc_words(kv, uint32_t(valid - 1) * uint32_t(a.kv_st * 2) + ROW * 2);
      const u32x4 rkr = rsrc_words(kr, uint32_t(valid - 1) * uint32_t(a.kr_st * 2) + kRope * 2);
      uint16_t* to = s_tile + stage * kStage;
#pragma unroll
      for (int i = 0; i < NKV; ++i) load_lds16(rkv, kv_at[i], to + (wave * NKV + i) * 512);
#pragma unroll
      for (int i = 0; i < NKR; ++i) load_lds16(rkr, kr_at[i], to + kKeys * ROW + (wave * NKR + i) * 512);
    };

    f32x4 o[NDT][2];
    float m[2], l[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      m[rt] = -INFINITY;
      l[rt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt][rt] = f32x4{};
    }
    // The rows this wave has, the keys its first and its last row see.
    const int wrow = qb * kRows + rw * 32;
    const int see_first = a.causal ? sq.offset + wrow : sq.k_len - 1;
    const int see_last = a.causal ? sq.offset + min(wrow + 31, sq.q_len - 1) : sq.k_len - 1;
    const bool active = wrow < sq.q_len;

    __builtin_amdgcn_s_waitcnt(0);  // q has landed: the loop below has waits of its own alone
    constexpr int kAhead = 2;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (t0 + i < t1) issue(t0 + i, i);
    }
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      if (t + 1 < t1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NL) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if constexpr (STAGES == 3) {  // every wave has read tile t - 1
        if (t + kAhead < t1) issue(t + kAhead, stage == 0 ? STAGES - 1 : stage - 1);
      }
      const uint16_t* tile = s_tile + stage * kStage;
      const int first_key = t * kKeys + key0;
      if (active && first_key <= see_last) {  // uniform
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
          for (int tt = 0; tt < TT; ++tt) {
            const int at = kk < KN ? (k_at ^ (32 * kk)) + 16 * tt * ROW : (r_at ^ (32 * (kk - KN))) + 16 * tt * kRope;
            to[tt] = *reinterpret_cast<const u32x4*>(tile + at);
          }
        };
        read_keys(0, k[0]);
#pragma unroll
        for (int kk = 0; kk < KN + 2; ++kk) {
          if (kk + 1 < KN + 2) read_keys(kk + 1, k[(kk + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) s[tt][rt] = mfma16x16x32(k[kk & 1][tt], q[rt][kk], s[tt][rt], Tag{});
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        // V of the first 32 keys is read beside the softmax, the others' beside its products.
        u32x2 v[KP][NDT][2];
        auto read_values = [&](int kp) __attribute__((always_inline)) {
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            const uint16_t* at = tile + (v_at ^ (16 * dt)) + 32 * kp * ROW;
            v[kp][dt][0] = lds_read_tr4(at);
            v[kp][dt][1] = lds_read_tr4(at + 16 * ROW);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        read_values(0);
        const bool whole = first_key + 16 * TT - 1 <= see_first && first_key + 16 * TT <= k_end;
        if (!whole) {
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            const int lim = min(limit[rt], k_end - 1) - first_key - 4 * g;
#pragma unroll
            for (int e = 0; e < 4 * TT; ++e) {
              if (16 * (e >> 2) + (e & 3) > lim) s[e >> 2][rt][e & 3] = -INFINITY;
            }
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
          top[rt] = row_group_max(max2(top[rt], s[TT - 1][rt][3])) * a.scale_log2;  // a scale is positive
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
            x[e] = fast_exp2(fmaf(s[e >> 2][rt][e & 3], a.scale_log2, -base));
            l[rt] += x[e];
          }
          // P is rounded to the inputs' type for the matrix unit, as in the paged prefill: at most half a
          // step of each weight (lifted in fp16, weight_lift), while l sums the unrounded ones in 32 bits.
#pragma unroll
          for (int e = 0; e < 2 * TT; ++e) pb[rt][e >> 2][e & 3] = pack2(x[2 * e], x[2 * e + 1], Tag{});
        }
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
          if (kp + 1 < KP) read_values(kp + 1);
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            const u32x4 vv = {v[kp][dt][0][0], v[kp][dt][0][1], v[kp][dt][1][0], v[kp][dt][1][1]};
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) o[dt][rt] = mfma16x16x32(vv, pb[rt][kp], o[dt][rt], Tag{});
          }
        }
      }
      if constexpr (STAGES == 2) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stage is read
        if (t + kAhead < t1) issue(t + kAhead, stage);
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }

    l[0] = row_group_sum(l[0]);
    l[1] = row_group_sum(l[1]);
    if constexpr (KG == 2) {
      // The second key group's sums go to the first through the stages.
      f32x4* const s_o = reinterpret_cast<f32x4*>(s_tile) + rw * 2 * NDT * 64 + lane;
      float2* const s_ml = reinterpret_cast<float2*>(reinterpret_cast<f32x4*>(s_tile) + 4 * 2 * NDT * 64) + rw * 128 + lane;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stages are read
      if (key0 != 0) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) s_o[64 * (NDT * rt + dt)] = o[dt][rt];
          s_ml[64 * rt] = make_float2(m[rt], l[rt]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (key0 == 0) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          const float2 other = s_ml[64 * rt];
          const float mn = fmaxf(m[rt], other.x);
          const float base = mn == -INFINITY ? 0.f : mn;
          const float c0 = fast_exp2(m[rt] - base), c1 = fast_exp2(other.x - base);
          m[rt] = mn;
          l[rt] = l[rt] * c0 + other.y * c1;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt][rt] = o[dt][rt] * c0 + s_o[64 * (NDT * rt + dt)] * c1;
        }
      }
    }
    const bool complete = t0 == 0 && t1 == tiles;
    const int64_t part = (int64_t(run) * 2 + (p == start ? 0 : 1)) * kRows + rw * 32 + n;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const int r = wrow + rt * 16 + n;
      const float lt = l[rt];
      if (r >= sq.q_len || key0 != 0) continue;
      if (!BALANCED || complete) {
        const float inv = lt != 0.f ? 1.f / lt : 0.f;  // a row that sees nothing is zero
        uint16_t* dst = a.out + int64_t(sq.q0 + r) * a.o_st + h * a.o_sh + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const f32x4 y = o[dt][rt] * inv;
          *reinterpret_cast<u32x2*>(dst + 16 * dt) = u32x2{pack2(y[0], y[1], Tag{}), pack2(y[2], y[3], Tag{})};
        }
      } else {
        float* dst = a.part_o + (part + 16 * rt) * DN + 4 * g;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4*>(dst + 16 * dt) = o[dt][rt];
        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + (part + 16 * rt) * 2) = make_float2(m[rt], lt);
      }
    }
    if constexpr (!BALANCED) return;
    p += uint32_t(t1 - t0);
    if (p >= end) return;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the sums are read
    // The next unit that has tiles: the run holds more of them, so there is one.
    t_first = 0;
    do {
      if (++qb >= Seq(a, b).blocks) {
        qb = 0;
        do {
          if (++b == a.batch) {
            b = 0;
            ++h;
          }
        } while (Seq(a, b).blocks == 0);
      }
    } while (Seq(a, b).tiles(qb) == 0);
  }
}

// Joins the parts of units that several runs share, in the order of the runs, and writes zeros for rows that see
// nothing: one workgroup for 16 rows of a unit.
template <int DN, typename Tag>
__global__ __launch_bounds__(256) void latent_prefill_merge_kernel(ExpandedArgs a) {
  constexpr int COLS = DN / 4;          // threads of a row
  constexpr int PAR = 256 / COLS;       // rows at a time
  const int h = blockIdx.y, b = blockIdx.z;
  const int qb = int(blockIdx.x) / (kRows / 16), r0 = int(blockIdx.x) % (kRows / 16) * 16;
  const Seq s(a, b);
  if (qb >= s.blocks || qb * kRows + r0 >= s.q_len) return;
  const int nt = s.tiles(qb);
  const int col = threadIdx.x % COLS;
  const uint32_t per_head = uint32_t(a.seq_tile[a.batch]);
  int parts = 0;
  int64_t row_first = 0, row_next = 0;
  if (nt > 0) {
    const Runs runs(uint32_t(a.runs), per_head * a.heads, kMinRun);
    const uint32_t u0 = uint32_t(h) * per_head + uint32_t(a.seq_tile[b] + s.before(qb));
    const uint32_t i0 = runs.holding(u0), i1 = runs.holding(u0 + nt - 1);
    if (i0 == i1) return;  // written by its run
    parts = int(i1 - i0) + 1;
    // Part i0 is that run's first one (slot 0) if the unit begins with the run, else its last (slot 1).
    row_first = (int64_t(i0) * 2 + (runs.start(i0) == u0 ? 0 : 1)) * kRows;
    row_next = int64_t(i0) * 2 * kRows;
  }
  auto part = [&](int i) { return i == 0 ? row_first : row_next + int64_t(i) * 2 * kRows; };
  for (int k = threadIdx.x / COLS; k < 16; k += PAR) {
    const int rr = r0 + k, r = qb * kRows + rr;
    if (r >= s.q_len) break;
    float top = -INFINITY;
    for (int i = 0; i < parts; ++i) top = fmaxf(top, a.part_ml[(part(i) + rr) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 o = {};
    float l = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const int64_t at = part(i) + rr;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
      const float c = fast_exp2(ml.x - base);
      l += c * ml.y;
      o += c * *reinterpret_cast<const f32x4*>(a.part_o + at * DN + 4 * col);
    }
    o *= l != 0.f ? 1.f / l : 0.f;
    uint16_t* dst = a.out + int64_t(s.q0 + r) * a.o_st + h * a.o_sh + 4 * col;
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1], Tag{}), pack2(o[2], o[3], Tag{})};
  }
}

bool vec_rows(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
}

struct PrefillSizes {
  int32_t runs;
  int64_t o_floats, ml_floats, bytes;
};

// The balanced schedule's runs and workspace; 0 where the call takes one workgroup per unit. Cutting units
// costs their parts' way through memory and a second launch, so it is for calls whose units do not fill the
// CUs: 1,024 queries over 9,216 keys with 24 heads (192 units) 167 us against 225 per unit, but a first chunk
// of 2,048 (384 units) 76 against 66 and 24 prompts of 17 to 700 (1,800 units) 116 against 72.
PrefillSizes prefill_sizes(int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t head_dim) {
  PrefillSizes z{};
  const int64_t cus = device_cu_count(), slots = 2 * cus, blocks = ceil_div(total_q, kRows);
  if (batch > 65535 || blocks * heads > cus) return z;
  // The list is counted in 32 bits on the device. Offsets that go back may give every sequence all blocks and keys.
  if (batch * blocks * ceil_div(total_k, kKeys) * heads > INT32_MAX) return z;
  z.runs = int32_t(slots);
  z.o_floats = slots * 2 * kRows * head_dim;
  z.ml_floats = slots * 2 * kRows * 2;
  z.bytes = ((z.o_floats + z.ml_floats + batch + 1) * 4 + 15) & ~int64_t(15);
  return z;
}

// Key groups of a workgroup. Two share a unit's rows and halve its tiles' time. They are for first chunks of few
// units, where the time is that of the last, longest unit. At head_dim 128 such a workgroup fills a CU, at 64 two
// fit; us with one group against two:
//   head_dim 128: one of 2,048 with 24 heads (384 units) 60 / 50, one of 4,096 with 12 108 / 90, one of 1,100 with 40
//     36 / 34, two of 2,048 with 16 77 / 61, two of 1,024 with 24 37 / 37; but four of 2,048 with 8 76 / 85, three of
//     1,600 with 12 56 / 66, four of 1,024 with 16 45 / 51;
//   head_dim 64: 45 / 42, 79 / 73 and 26 / 25 for the first three; but two of 2,048 55 / 58, two of 1,024 26 / 30, four
//     of 2,048 55 / 58, four of 1,024 32 / 34.
// More units gain nothing or lose (2,800 with 24 heads, 528 units: 82 / 85, 59 / 58; 8,192 with 24: 461 / 551, 311 /
// 336), nor do units of one length (2,048 behind 8,192: 316 / 366) and short ones (24 of 90, 20 heads: 15 / 20).
int32_t prefill_key_groups(int32_t batch, int32_t total_q, int32_t total_k, int32_t heads, int32_t head_dim,
                           int32_t causal) {
  const bool few = ceil_div(total_q, kRows) * heads <= 2 * device_cu_count();
  const bool long_ones = total_q / 8 / kRows >= batch && batch <= (head_dim == 128 ? 2 : 1);
  return causal && total_q == total_k && long_ones && few ? 2 : 1;
}

template <int DN, typename Tag>
void launch_prefill(const ExpandedArgs& a, int64_t longest, hipStream_t s) {
  const unsigned blocks = unsigned(ceil_div(longest, kRows));
  const unsigned heads = unsigned(a.heads), batch = unsigned(a.batch);
  if (a.runs == 0) {
    const dim3 grid(heads, blocks, batch);
    if (a.key_groups == 2) hipLaunchKernelGGL((latent_prefill_kernel<DN, 2, false, Tag>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((latent_prefill_kernel<DN, 1, false, Tag>), grid, dim3(256), 0, s, a);
    return;
  }
  hipLaunchKernelGGL((latent_prefill_kernel<DN, 1, true, Tag>), dim3(unsigned(a.runs)), dim3(256), 0, s, a);
  hipLaunchKernelGGL((latent_prefill_merge_kernel<DN, Tag>), dim3(blocks * (kRows / 16), heads, batch), dim3(256), 0,
                     s, a);
}

}  // namespace
}  // namespace ti

extern "C" int ti_latent_prefill_workspace_bytes(int32_t batch, int32_t total_q, int32_t total_k,
                                                 int32_t num_heads, int32_t head_dim,
                                                 int64_t* workspace_bytes_out) {
  using namespace ti;
  const char* who = "ti_latent_prefill_workspace_bytes";
  if (batch < 0 || total_q < 0 || total_k < 0 || num_heads <= 0 || (head_dim != 128 && head_dim != 64)) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d total_q=%d total_k=%d heads=%d head_dim=%d", who, batch, total_q,
                total_k, num_heads, head_dim);
  }
  if (!workspace_bytes_out) return fail(TI_EINVAL, "%s: null output", who);
  *workspace_bytes_out = batch == 0 || total_q == 0 ? 0 : prefill_sizes(batch, total_q, total_k, num_heads, head_dim).bytes;
  return TI_OK;
}

extern "C" int ti_latent_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* kv,
                                 int64_t kv_stride_t, int64_t kv_stride_h, const void* key_rope,
                                 int64_t key_stride_t, const int32_t* cu_seqlens_q,
                                 const int32_t* cu_seqlens_k, void* out, int64_t out_stride_t,
                                 int64_t out_stride_h, void* workspace, int64_t workspace_bytes,
                                 int32_t batch, int32_t total_q, int32_t total_k, int32_t max_seqlen_q, int32_t num_heads, int32_t head_dim,
                                 int32_t rope_dim, int32_t causal, float scale, int32_t dtype,
                                 void* stream) {
  using namespace ti;
  const char* who = "ti_latent_prefill";
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_F16) {
    return fail(TI_EUNSUPPORTED, "%s: dtype code %d is not bf16/fp16", who, dtype);
  }
  if (head_dim != 128 && head_dim != 64) {
    return fail(TI_EUNSUPPORTED, "%s: head_dim %d not built (64, 128)", who, head_dim);
  }
  if (rope_dim != kRope) return fail(TI_EUNSUPPORTED, "%s: rope_dim %d not built (64)", who, rope_dim);
  if (batch < 0 || total_q < 0 || total_k < 0 || max_seqlen_q < 0 || num_heads <= 0 || batch > 65535 ||
      num_heads > 65535) {
    return fail(TI_EINVAL, "%s: bad sizes batch=%d total_q=%d total_k=%d max_seqlen_q=%d heads=%d", who, batch,
                total_q, total_k, max_seqlen_q, num_heads);
  }
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return TI_OK;
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || (total_k > 0 && (!kv || !key_rope))) {
    return fail(TI_EINVAL, "%s: null pointer", who);
  }
  if (!vec_rows(q, q_stride_t, q_stride_h) || !vec_rows(kv, kv_stride_t, kv_stride_h) ||
      !vec_rows(key_rope, key_stride_t, 0) || !vec_rows(out, out_stride_t, out_stride_h)) {
    return fail(TI_EINVAL, "%s: rows must be 16-byte aligned", who);
  }
  if (!(scale > 0.f && scale <= kMaxScale)) {
    return fail(TI_EINVAL, "%s: scale %g is not positive or beyond 1e30", who, double(scale));
  }
  // A tile's rows are reached by 32-bit offsets.
  if (kv_stride_t < 0 || key_stride_t < 0 || kv_stride_t >= (1 << 24) || key_stride_t >= (1 << 24)) {
    return fail(TI_EINVAL, "%s: token strides %lld, %lld of kv and key_rope must be in [0, 2^24)", who,
                static_cast<long long>(kv_stride_t), static_cast<long long>(key_stride_t));
  }
  ExpandedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.kv = static_cast<const uint16_t*>(kv);
  a.kv_st = kv_stride_t;
  a.kv_sh = kv_stride_h;
  a.kr = static_cast<const uint16_t*>(key_rope);
  a.kr_st = key_stride_t;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.total_q = total_q;
  a.total_k = total_k;
  a.causal = causal;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.batch = batch;
  a.heads = num_heads;
  const PrefillSizes z = prefill_sizes(batch, total_q, total_k, num_heads, head_dim);
  if (workspace && z.bytes > 0) {
    if (workspace_bytes < z.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
      return fail(TI_EINVAL, "%s: workspace %lld < %lld bytes, or not 16-byte aligned", who,
                  static_cast<long long>(workspace_bytes), static_cast<long long>(z.bytes));
    }
    a.runs = z.runs;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + z.o_floats;
    a.seq_tile = reinterpret_cast<int32_t*>(a.part_ml + z.ml_floats);
  }
  const int64_t longest = max_seqlen_q < total_q ? max_seqlen_q : total_q;
  a.by_length = batch > 1 && batch <= 64 && total_k / 1024 >= batch;
  a.key_groups = prefill_key_groups(batch, total_q, total_k, num_heads, head_dim, causal);
  if (ceil_div(longest, kRows) > 65535) return fail(TI_EINVAL, "%s: max_seqlen_q %d too long", who, max_seqlen_q);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == TI_DTYPE_BF16;
  if (head_dim == 128) {
    if (bf16) launch_prefill<128, Bf16>(a, longest, s);
    else launch_prefill<128, F16>(a, longest, s);
  } else {
    if (bf16) launch_prefill<64, Bf16>(a, longest, s);
    else launch_prefill<64, F16>(a, longest, s);
  }
  return check_launch(who);
}
