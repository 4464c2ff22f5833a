// Attention of a few query rows against a 4-bit key / value cache with grouped
// heads (sm_100a), head dims 64 and 128 in groups of 64.
//
// With codes n, scales s and minima m per (row t, group g) and normalised
// queries q:
//   score_t = sum_g s_tg (q_g . n_tg) + m_tg sum(q_g)
//   o_d     = sum_t (p_t s_tg) n_td + sum_t p_t m_tg
// so that the tensor cores multiply integers: the query with the codes, and the
// weights p s (rounded to fp16, or to bf16 where scales lie far apart) with the
// codes.  The second sums stay in fp32.
//
// A block owns up to 16 query rows of a (sequence, key / value head) and a stretch
// of its keys, then the next one's (Kv4Line).  Each of its four warps takes every fourth 32-row tile on its own:
// tiles arrive by cp.async in a ring private to the warp, so that the loop has
// no block-wide barrier, and the codes go from shared memory to matrix operands
// in registers.  The 8 query rows (two tiles of 8 for up to 16) are the n side of
// tensor-core products, 16 keys the m side of the scores, 16 value dims the m side
// of the output; a byte permute pairs the codes of two keys before they become
// operands (kv4_device.cuh).
//
// The running maximum moves only when a score exceeds it by 2^8, which keeps
// the shuffles and the rescaling out of most tiles.
//
// Measured: 64 sequences x 8192 keys, 48 query heads on 8 of 128: 142 - 147 us, 4.1 TB/s
// (63 % of the measured copy bandwidth).  Bound by the instruction mix: ALU 51 %,
// tensor 23 %, FMA 17 %, LSU 21 % of their cycles, which overlap little; 314
// instructions per 16 keys.  One sequence of 8192 keys: 11.7 us, of 130 keys: 5.1 us.
#include <algorithm>

#include "kv4_device.cuh"

namespace omni {

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;       // keys per tile of a warp
constexpr float kSlack = 8.f;   // log2 units a score may exceed the running maximum by

template <int D, int NT>
struct HeadsCfg {
  static constexpr int NG = D / 64;
  static constexpr int kStages = 3;   // and three blocks per SM: 149 us, two stages and four blocks 155 us
  static constexpr int kRow = D / 2;
  static constexpr int kCodes = kTile * kRow;
  static constexpr int kParams = kTile * NG * 4;
  static constexpr int kStage = 2 * (kCodes + kParams);
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kRows = 8 * NT;
  static constexpr int kMerge = kWarps * kRows * (D + 2) * 4;
  static constexpr int kQ = kRing > kMerge ? kRing : kMerge;      // byte offset of the queries
  static constexpr int kSmem = kQ + kRows * D * 2 + kRows * (NG + 1) * 4;
};

__device__ __forceinline__ void load_params(uint32_t at, uint32_t (&p)[1]) { p[0] = lds32(at); }
__device__ __forceinline__ void load_params(uint32_t at, uint32_t (&p)[2]) {
  const uint2 v = lds64(at);
  p[0] = v.x;
  p[1] = v.y;
}

template <int D, int NT, int TYPE>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) kv4_heads_kernel(const Kv4Attend a, const Kv4Line line) {
  using C = HeadsCfg<D, NT>;
  constexpr int NG = C::NG;
  extern __shared__ __align__(16) uint8_t smem[];
  uint2* sq = reinterpret_cast<uint2*>(smem + C::kQ);                       // [kRows][D / 8 words][2]
  float* sqs = reinterpret_cast<float*>(smem + C::kQ + C::kRows * D * 2);   // [kRows][NG]: sum(q_g) 2^-24
  float* srs = sqs + C::kRows * NG;                                         // [kRows]: factor of the scores
  const int lane = lane_id(), warp = warp_id(), i = lane >> 2, j = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStage;
  wait_for_previous_grid();
  launch_dependents();
  __shared__ Kv4Walk walk;
  int share = 0;
  int2 span = walk.begin<kWarps * 32, kTile>(a, line, &share);

  while (span.x < span.y) {
  Kv4Piece piece = walk.next<kTile>(a, line, share, &span);
  const int b = piece.b, hk = line.row_blocks.of(piece.segment), row0 = (piece.segment - hk * line.row_blocks.d) * C::kRows;
  const int nrows = min(C::kRows, line.rows.d - row0);
  const Kv4View see = kv4_rows<kTile>(a, line, &piece, row0, nrows);
  const int sink_tiles = piece.sink_tiles, first = piece.first;
  const int t0 = piece.step0 * kWarps, t1 = min(piece.tiles, piece.step1 * kWarps);
  // place of query row r in q and in the output, in heads
  auto head_of = [&](int r) {
    const int t = line.group.of(row0 + r);
    return ((long long)b * a.Tn + t) * a.H + hk * line.group.d + row0 + r - t * line.group.d;
  };
  auto row_of = [&](int tile) { return (tile < sink_tiles ? tile : first + tile - sink_tiles) * kTile; };

  const uint8_t* kc = a.k.codes + b * a.k.c_b + hk * a.k.c_h;
  const uint8_t* vc = a.v.codes + b * a.v.c_b + hk * a.v.c_h;
  const uint8_t* kp = a.k.params + b * a.k.p_b + hk * a.k.p_h;
  const uint8_t* vp = a.v.params + b * a.v.p_b + hk * a.v.p_h;
  // A tile is contiguous in memory.  In shared memory row t lies at t ^ bit2(t), and rows of 64
  // bytes have their halves swapped where bit1(t) is set: the 8 (scores) and 4 (output) rows that
  // one load touches then fall into different banks.
  auto issue = [&](int tile, int stage) {
    const long long r0 = row_of(tile);
    const uint32_t dst = ring + stage * C::kStage;
    constexpr int kPieces = C::kCodes / 16, kPer = C::kRow / 16;
#pragma unroll
    for (int n = 0; n < kPieces / 32; ++n) {
      const int idx = lane + 32 * n, t = idx / kPer;
      int c = idx % kPer;
      if (D == 128) c ^= ((t >> 1) & 1) << 1;
      const uint32_t at = dst + (t ^ ((t >> 2) & 1)) * C::kRow + c * 16;
      kv4_cp16(at, kc + r0 * C::kRow + idx * 16);
      kv4_cp16(at + C::kCodes, vc + r0 * C::kRow + idx * 16);
    }
    constexpr int kPp = C::kParams / 16;  // 16 or 8 pieces each of k and v
    const bool is_v = lane >= 16;
    if ((lane & 15) < kPp)
      kv4_cp16(dst + 2 * C::kCodes + (is_v ? C::kParams : 0) + (lane & 15) * 16,
               (is_v ? vp : kp) + r0 * (NG * 4) + (lane & 15) * 16);
  };
  int next = t0 + warp;
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) {
    if (next < t1) issue(next, s);
    kv4_cp_commit();
    next += kWarps;
  }

  // ---- queries: normalised fp16 rows, group sums, score factors; a lane takes the eight
  // dims of a code word, a warp two or four rows ----------------------------------------------------
  constexpr int kWords = D / 8, kAtOnce = 32 / kWords;
  for (int r = warp * kAtOnce + lane / kWords; r < C::kRows; r += kWarps * kAtOnce) {
    const int w = lane % kWords;
    float x[8] = {}, amax = 0.f, un;
    if (r < nrows) kv4_load8<TYPE>(a.q, head_of(r) * D + w * 8, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
    for (int o = 1; o < kWords; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float sc = q_normaliser(amax, &un);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= sc;
    float sum = query_pairs(x, sq + (r * kWords + w) * 2);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((w & 7) == 0) sqs[r * NG + (w >> 3)] = sum * (1.f / kKv4Codes);
    if (w == 0) srs[r] = un * (a.scale * kKv4Log2e);
  }
  __syncthreads();
  // operand of the scores: lane (i, j) holds query row i against the 16 dims that it reads of each group
  uint2 qf[NG][4][NT];
  float qs[NG][NT][2], rs[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) qf[g][ks][nt] = sq[((nt * 8 + i) * (D / 8) + g * 8 + 2 * j) * 2 + ks];
#pragma unroll
      for (int c = 0; c < 2; ++c) qs[g][nt][c] = sqs[(nt * 8 + 2 * j + c) * NG + g];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rs[nt][c] = srs[nt * 8 + 2 * j + c];
    }
  }
  const bool huge = kv4_score_factors<NT>(rs);

  float f[NG];                     // the values' power of two; 0 before any
#pragma unroll
  for (int g = 0; g < NG; ++g) f[g] = 0.f;
  float acc[NG][4][NT][4], accm[NG][NT][2], lsum[NT][2];
  float limit[NT][2], ref[NT][2];  // running maximum + slack, running maximum (0 before any key)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) acc[g][mm][nt][c] = 0.f;
      accm[g][nt][0] = accm[g][nt][1] = 0.f;
    }
    lsum[nt][0] = lsum[nt][1] = 0.f;
    limit[nt][0] = limit[nt][1] = -INFINITY;
    ref[nt][0] = ref[nt][1] = 0.f;
  }

  uint32_t k_at[NG], v_at0[NG], v_at1[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    k_at[g] = (i ^ ((i >> 2) & 1)) * C::kRow + j * 8 + ((g ^ (D == 128 ? (i >> 1) & 1 : 0)) * 32);
    const uint32_t at = C::kCodes + i * 4 + (g ^ (D == 128 ? j & 1 : 0)) * 32;
    v_at0[g] = at + ((2 * j) ^ ((j >> 1) & 1)) * C::kRow;
    v_at1[g] = at + ((2 * j + 1) ^ ((j >> 1) & 1)) * C::kRow;
  }

  int stage = 0;
  for (int tile = t0 + warp; tile < t1; tile += kWarps, next += kWarps) {
    kv4_cp_wait<C::kStages - 2>();
    __syncwarp();  // every lane's pieces have landed, and every lane has left the stage refilled below
    if (next < t1) issue(next, stage == 0 ? C::kStages - 1 : stage - 1);
    kv4_cp_commit();
    const int r0 = row_of(tile);
    const bool masked = huge || !(r0 + kTile <= a.n_sink || (r0 >= see.lo_max && r0 + kTile <= see.hi_min));
    uint32_t st = ring + stage * C::kStage, sp = st + 2 * C::kCodes + i * NG * 4;
    // ---- do the scales of the tile's values fit their power of two?  Lane: key r0 + lane ----
    bool slow[NG];
    {
      uint32_t v[NG];
      load_params(st + 2 * C::kCodes + C::kParams + lane * NG * 4, v);
      const int r = r0 + lane;
      const bool used = !masked || r < a.n_sink || (r >= see.lo_min && r < see.hi_max);
      bool fit = true;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        slow[g] = false;
        fit = fit && (!used || kv4_in_range(bf16_lo(v[g]), f[g]));
      }
      if (!__all_sync(0xffffffffu, fit)) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float sc = bf16_lo(v[g]);
          const uint32_t e = __reduce_max_sync(0xffffffffu, used && sc <= 3.4e38f ? __float_as_uint(sc) >> 23 : 0u);
          if (e > 0) {  // largest scale in [2^3, 2^4); sums made before move along
            const float now = __uint_as_float(min(257u - e, 254u) << 23);
            const float move = f[g] == 0.f ? 0.f : now / f[g];
            float most = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int mm = 0; mm < 4; ++mm) most = fmaxf(most, fabsf(acc[g][mm][nt][c]));
            if (__all_sync(0xffffffffu, most * move < kKv4Room)) {
              f[g] = now;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                  for (int mm = 0; mm < 4; ++mm) acc[g][mm][nt][c] *= move;
            }
          }
          slow[g] = !__all_sync(0xffffffffu, !used || kv4_in_range(sc, f[g]));
        }
      }
    }
    // Rolled: the loop's code must stay in the instruction cache next to the scheduler.
#pragma unroll 1
    for (int r = r0 + i; r < r0 + kTile; r += 16, st += 16 * C::kRow, sp += 16 * NG * 4) {
      // ---- scores of 16 keys (this lane: keys r and r + 8), in units of log2 ------------
      uint32_t pa[NG], pb[NG];
      load_params(sp, pa);
      load_params(sp + 8 * NG * 4, pb);
      float s[NT][4];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint2 wa = lds64(st + k_at[g]), wb = lds64(st + k_at[g] + 8 * C::kRow);
        float d[NT][4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t xa = (ks < 2 ? wa.x : wa.y) >> ((ks & 1) * 8), xb = (ks < 2 ? wb.x : wb.y) >> ((ks & 1) * 8);
          const uint32_t a0 = xa & 0x000f000fu, a1 = xb & 0x000f000fu, a2 = xa & 0x00f000f0u, a3 = xb & 0x00f000f0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 q = qf[g][ks][nt];
            if (ks == 0) mma_f16_zero(d[nt], a0, a1, a2, a3, q.x, q.y);
            else mma_f16(d[nt], a0, a1, a2, a3, q.x, q.y);
          }
        }
        const float sa = bf16_lo(pa[g]), ma = bf16_hi(pa[g]), sb = bf16_lo(pb[g]), mb = bf16_hi(pb[g]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float m = qs[g][nt][c & 1] * (c < 2 ? ma : mb);
            s[nt][c] = fmaf(d[nt][c], c < 2 ? sa : sb, g == 0 ? m : m + s[nt][c]);
          }
      }
      bool above = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][c] *= rs[nt][c & 1];
      uint32_t hidden = 0;   // bit 4 nt + c: the row does not see the key
      if (masked) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int lo = __shfl_sync(0xffffffffu, see.seen.lo, nt * 8 + 2 * j + c);
            const int hi = __shfl_sync(0xffffffffu, see.seen.hi, nt * 8 + 2 * j + c);
            if (huge) {
              s[nt][c] *= kKv4Lift;
              s[nt][c + 2] *= kKv4Lift;
            }
            if (!(r < a.n_sink || (r >= lo && r < hi))) {
              s[nt][c] = -INFINITY;
              hidden |= 1u << (4 * nt + c);
            }
            if (!(r + 8 < a.n_sink || (r + 8 >= lo && r + 8 < hi))) {
              s[nt][c + 2] = -INFINITY;
              hidden |= 4u << (4 * nt + c);
            }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[nt][c] = fmaxf(s[nt][c], s[nt][c + 2]);
          above |= top[nt][c] > limit[nt][c];
        }
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float old = limit[nt][c] - kSlack;
            float x = fmaxf(top[nt][c], old);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            limit[nt][c] = x + kSlack;
            // what was summed is in units of 2^ref, whatever limit - kSlack rounds to
            const float now = x == -INFINITY ? 0.f : x;
            const float alpha = old == -INFINITY ? 0.f : fast_exp2(ref[nt][c] - now);
            ref[nt][c] = now;
            lsum[nt][c] *= alpha;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              accm[g][nt][c] *= alpha;
#pragma unroll
              for (int mm = 0; mm < 4; ++mm) {
                acc[g][mm][nt][c] *= alpha;
                acc[g][mm][nt][c + 2] *= alpha;
              }
            }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s[nt][c] = fast_exp2(s[nt][c] - ref[nt][c]);
          s[nt][c + 2] = fast_exp2(s[nt][c + 2] - ref[nt][c]);
          lsum[nt][c] += s[nt][c] + s[nt][c + 2];
        }

      // ---- output -----------------------------------------------------------------
      load_params(sp + C::kParams, pa);
      load_params(sp + C::kParams + 8 * NG * 4, pb);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float sa = bf16_lo(pa[g]), sb = bf16_lo(pb[g]);
        const float ma = bf16_hi(pa[g]), mb = bf16_hi(pb[g]);
        float x[NT][4];
        const float fa = sa * f[g], fb = sb * f[g];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 4; ++c) x[nt][c] = s[nt][c] * (c < 2 ? fa : fb);
          if (masked) {  // a key that a row does not see may hold anything; one that it sees counts, whatever its weight
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (hidden >> (4 * nt + c) & 1) x[nt][c] = 0.f;
              else accm[g][nt][c & 1] = fmaf(s[nt][c], c < 2 ? ma : mb, accm[g][nt][c & 1]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) accm[g][nt][c & 1] = fmaf(s[nt][c], c < 2 ? ma : mb, accm[g][nt][c & 1]);
          }
        }
        const uint32_t w0 = lds32(st + v_at0[g]), w1 = lds32(st + v_at1[g]);
        const uint32_t w8 = lds32(st + v_at0[g] + 8 * C::kRow), w9 = lds32(st + v_at1[g] + 8 * C::kRow);
        const uint32_t l0 = __byte_perm(w0, w1, 0x5410), h0 = __byte_perm(w0, w1, 0x7632);
        const uint32_t l8 = __byte_perm(w8, w9, 0x5410), h8 = __byte_perm(w8, w9, 0x7632);
        uint32_t bw[NT][2];
        if (!slow[g]) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            bw[nt][0] = movmatrix_trans(pack_f16x2(x[nt][0], x[nt][1]));
            bw[nt][1] = movmatrix_trans(pack_f16x2(x[nt][2], x[nt][3]));
          }
          mma_values<0, NT>(acc[g][0], l0, h0, l8, h8, bw);
          mma_values<1, NT>(acc[g][1], l0, h0, l8, h8, bw);
          mma_values<2, NT>(acc[g][2], l0, h0, l8, h8, bw);
          mma_values<3, NT>(acc[g][3], l0, h0, l8, h8, bw);
        } else {
          float sums[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            bw[nt][0] = movmatrix_trans(pack_bf16x2(x[nt][0], x[nt][1]));
            bw[nt][1] = movmatrix_trans(pack_bf16x2(x[nt][2], x[nt][3]));
            mma_bf16_zero(sums[nt], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, bw[nt][0], bw[nt][1]);
#pragma unroll
            for (int c = 0; c < 4; ++c)  // p 8 s: these weights meet n - 8
              if (x[nt][c] != 0.f) accm[g][nt][c & 1] = fmaf(s[nt][c], 8.f * (c < 2 ? sa : sb), accm[g][nt][c & 1]);
          }
          mma_values_bf16<0, NT>(acc[g][0], l0, h0, l8, h8, bw, sums);
          mma_values_bf16<1, NT>(acc[g][1], l0, h0, l8, h8, bw, sums);
          mma_values_bf16<2, NT>(acc[g][2], l0, h0, l8, h8, bw, sums);
          mma_values_bf16<3, NT>(acc[g][3], l0, h0, l8, h8, bw, sums);
        }
      }
    }
    stage = stage + 1 == C::kStages ? 0 : stage + 1;
  }

  // ---- join the warps (the ring's memory is free: all copies have landed) -----------
  kv4_cp_wait<0>();
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);          // [kWarps][kRows][D]
  float* sml = so + kWarps * C::kRows * D;             // [kWarps][kRows][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = warp * C::kRows + nt * 8 + 2 * j + c;
      float l = lsum[nt][c];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (i == 0) {
        sml[2 * r] = limit[nt][c] == -INFINITY ? -INFINITY : ref[nt][c];
        sml[2 * r + 1] = l;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float m = accm[g][nt][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        const float unit = f[g] == 0.f ? 0.f : 1.f / f[g];
        float* o = so + r * D + g * 64 + 8 * i;
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) {
          o[mm] = fmaf(acc[g][mm][nt][c], unit * value_unit(mm), m);
          o[4 + mm] = fmaf(acc[g][mm][nt][c + 2], unit * value_unit(mm), m);
        }
      }
    }
  __syncthreads();
  // a segment that this block holds alone is finished; otherwise its piece goes to a slot
  const bool alone = piece.step0 == 0 && piece.step1 == piece.steps;
  float* part = a.part + (size_t)(2 * blockIdx.x + (piece.step0 == 0)) * C::kRows * (D + 2);
  for (int idx = threadIdx.x; idx < nrows * (D / 2); idx += kWarps * 32) {
    const int r = idx / (D / 2), d = (idx % (D / 2)) * 2;
    float top = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sml[2 * (w * C::kRows + r)]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int at = w * C::kRows + r;
      const float f = fast_exp2(sml[2 * at] - ref);
      l = fmaf(f, sml[2 * at + 1], l);
      x = fmaf(f, so[at * D + d], x);
      y = fmaf(f, so[at * D + d + 1], y);
    }
    if (alone) {
      const long long head = head_of(r);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      reinterpret_cast<uint32_t*>(a.out)[(head * D + d) / 2] = kv4_pack2<TYPE>(x * inv, y * inv);
    } else {
      *reinterpret_cast<float2*>(part + r * D + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(part + C::kRows * D + 2 * r) = make_float2(top, l);
    }
  }
  __syncthreads();  // the next segment refills shared memory
  }
}

template <int D, int NT, int TYPE>
void launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  auto kern = kv4_heads_kernel<D, NT, TYPE>;
  constexpr int smem = HeadsCfg<D, NT>::kSmem;
  ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  kv4_launch(kern, dim3((unsigned)p.blocks), kWarps * 32, smem, s, a, kv4_line(a, p));
}

template <int TYPE>
void launch_dims(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  if (a.W == 128)
    p.row_tiles == 1 ? launch<128, 1, TYPE>(a, p, s) : launch<128, 2, TYPE>(a, p, s);
  else
    p.row_tiles == 1 ? launch<64, 1, TYPE>(a, p, s) : launch<64, 2, TYPE>(a, p, s);
}

}  // namespace

void kv4_heads_plan(const Kv4Attend& a, Kv4Plan& p) {
  const int R = a.Tn * (a.H / a.Hk);
  p.kernel = 1;
  // 8 query rows per block and three blocks per SM, or 16 and two: that reads the codes once for twice the
  // rows, but a block takes 4.5 us longer to start and to end.  Measured, us 8 / 16 rows (cold): 6 rows of
  // 64 x 8 heads x 64 steps 155 / 226; 12 rows of 16 x 8 x 32 steps 56 / 48, of 1 x 8 x 64 steps 21.5 / 23.6;
  // 16 rows of 64 x 4 x 32 steps 93 / 81; heads of 64, 12 rows of 64 x 8 x 32 steps 106 / 93, of 8 x 8 x 8
  // steps 17.4 / 19.5.  That is 2.2 and 2.0 us per step of a block.
  const double steps = (double)kv4_plan_steps(a) * a.B * a.Hk;
  const double one = 2.2 * steps * ((R + 7) / 8) / (148 * 3), two = 2.0 * steps * ((R + 15) / 16) / (148 * 2) + 4.5;
  p.row_tiles = one <= two ? 1 : 2;
  p.row_blocks = (R + 8 * p.row_tiles - 1) / (8 * p.row_tiles);
  kv4_line_plan(a, p, 148 * (p.row_tiles == 1 ? 3 : 2), 3);
}

void kv4_heads_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  if (a.type == KV4_F16) launch_dims<KV4_F16>(a, p, s);
  else launch_dims<KV4_BF16>(a, p, s);
  if (p.restart > 0) kv4_combine(a, p, s);
}

}  // namespace omni
