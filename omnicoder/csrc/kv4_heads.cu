// Attention of a few query rows against a 4-bit key / value cache with grouped
// heads (sm_100a), head dims 64 and 128 in groups of 64.
//
// With codes n, scales s and minima m per (row t, group g) and normalised
// queries q:
//   score_t = sum_g s_tg (q_g . n_tg) + m_tg sum(q_g)
//   o_d     = sum_t (p_t s_tg) (n_td - 8) + sum_t p_t (m_tg + 8 s_tg)
// so that the tensor cores multiply integers: the query with the codes, and the
// weights p s (rounded to bf16, the only rounding before the output's) with the
// codes.  The second sums stay in fp32; the weights meet n - 8 instead of n
// because the rounding error then scales with at most 8 steps, not 15.
//
// A block owns (sequence, key / value head, up to 16 query rows, one split of
// the keys).  Each of its four warps takes every fourth 32-row tile on its own:
// tiles arrive by cp.async in a ring private to the warp, so that the loop has
// no block-wide barrier, and the codes go from shared memory to matrix operands
// in registers.  The 8 query rows (two tiles of 8 for up to 16) are the n side of
// m16n8k16, 16 keys the m side of the scores, 16 value dims the m side of the
// output: one mma for 256 codes.  Nibbles as fp16 bits are subnormals n 2^-24
// (or n 2^-20 one nibble up), which the fp16 product takes exactly: one AND for
// two key codes.  Value codes become bf16 16 + n by a shift and a LOP3 after a
// byte permute has paired two keys; the constant 24 = 16 + 8 is taken out
// through the sum of the rounded weights, an mma against ones.
//
// The running maximum moves only when a score exceeds it by 2^8, which keeps
// the shuffles and the rescaling out of most tiles.
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
  static constexpr int kStages = 3;
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

template <int D, int NT, int TYPE>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) kv4_heads_kernel(const Kv4Attend a, const int splits) {
  using C = HeadsCfg<D, NT>;
  constexpr int NG = C::NG;
  extern __shared__ __align__(16) uint8_t smem[];
  __half* sq = reinterpret_cast<__half*>(smem + C::kQ);                     // [kRows][D]
  float* sqs = reinterpret_cast<float*>(smem + C::kQ + C::kRows * D * 2);   // [kRows][NG]: sum(q_g) 2^-24
  float* srs = sqs + C::kRows * NG;                                         // [kRows]: factor of the scores
  const int lane = lane_id(), warp = warp_id(), i = lane >> 2, j = lane & 3;
  const int split = blockIdx.x % splits, row0 = (blockIdx.x / splits) * C::kRows, hk = blockIdx.y, b = blockIdx.z;
  const int G = a.H / a.Hk, R = a.Tn * G, nrows = min(C::kRows, R - row0);

  // ---- the rows each query sees; lane r holds query row r --------------------
  Kv4Seen seen{0, 0};
  if (lane < nrows) seen = kv4_seen(a, b, (row0 + lane) / G);
  const int lo_min = __reduce_min_sync(0xffffffffu, lane < nrows ? seen.lo : a.L);
  const int hi_max = __reduce_max_sync(0xffffffffu, lane < nrows ? seen.hi : 0);
  const int lo_max = __reduce_max_sync(0xffffffffu, lane < nrows ? seen.lo : 0);
  const int hi_min = __reduce_min_sync(0xffffffffu, lane < nrows ? seen.hi : a.L);
  const int sink_tiles = (a.n_sink + kTile - 1) / kTile;
  const int first = max(lo_min / kTile, sink_tiles);
  const int tiles = sink_tiles + max(0, hi_max > lo_min ? (hi_max + kTile - 1) / kTile - first : 0);
  const int per = (tiles + splits - 1) / splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  auto row_of = [&](int tile) { return (tile < sink_tiles ? tile : first + tile - sink_tiles) * kTile; };

  const uint8_t* kc = a.k.codes + b * a.k.c_b + hk * a.k.c_h;
  const uint8_t* vc = a.v.codes + b * a.v.c_b + hk * a.v.c_h;
  const uint8_t* kp = a.k.params + b * a.k.p_b + hk * a.k.p_h;
  const uint8_t* vp = a.v.params + b * a.v.p_b + hk * a.v.p_h;
  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStage;

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

  // ---- queries: normalised fp16 rows, group sums, score factors --------------
  for (int r = warp; r < C::kRows; r += kWarps) {
    constexpr int kPerLane = D / 32;
    float x[kPerLane], amax = 0.f, sum = 0.f, un;
    const int row = row0 + r;
    const long long at = (((long long)b * a.Tn + row / G) * a.H + hk * G + row % G) * D + lane * kPerLane;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      x[e] = r < nrows ? kv4_load1<TYPE>(a.q, at + e) : 0.f;
      amax = fmaxf(amax, fabsf(x[e]));
    }
    const float sc = q_normaliser(warp_max(amax), &un);
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      const __half h = __float2half_rn(x[e] * sc);
      sq[r * D + lane * kPerLane + e] = h;
      sum += __half2float(h);
    }
#pragma unroll
    for (int o = 16 / NG; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane % (32 / NG) == 0) sqs[r * NG + lane / (32 / NG)] = sum * 5.9604644775390625e-8f;
    if (lane == 0) srs[r] = un * (a.scale * (kKv4Log2e * kKv4Codes));
  }
  __syncthreads();
  // operand of the scores: lane (i, j) holds query row i against the 16 dims that it reads of each
  // group; dims one nibble up count 16-fold
  uint32_t qf[NG][4][NT][2];
  float qs[NG][NT][2], rs[NT][2];
  int lo[NT][2], hi[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const __half* q = sq + (nt * 8 + i) * D + g * 64 + j * 16;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const __half* p = q + (ks >> 1) * 8 + (ks & 1) * 2;
        const __half2 even = __halves2half2(p[0], p[4]), odd = __halves2half2(p[1], p[5]);
        const __half2 odd16 = __hmul2(odd, __float2half2_rn(0.0625f));
        qf[g][ks][nt][0] = *reinterpret_cast<const uint32_t*>(&even);
        qf[g][ks][nt][1] = *reinterpret_cast<const uint32_t*>(&odd16);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) qs[g][nt][c] = sqs[(nt * 8 + 2 * j + c) * NG + g];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rs[nt][c] = srs[nt * 8 + 2 * j + c];
      lo[nt][c] = __shfl_sync(0xffffffffu, seen.lo, nt * 8 + 2 * j + c);
      hi[nt][c] = __shfl_sync(0xffffffffu, seen.hi, nt * 8 + 2 * j + c);
    }
  }

  float acc[NG][4][NT][4], accr[NG][NT][4], accm[NG][NT][2], lsum[NT][2], mx[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        accr[g][nt][c] = 0.f;
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) acc[g][mm][nt][c] = 0.f;
      }
      accm[g][nt][0] = accm[g][nt][1] = 0.f;
    }
    lsum[nt][0] = lsum[nt][1] = 0.f;
    mx[nt][0] = mx[nt][1] = -INFINITY;
  }

  const uint32_t k_at = (i ^ ((i >> 2) & 1)) * C::kRow + j * 8, k_swap = D == 128 ? ((i >> 1) & 1) * 32 : 0;
  const uint32_t v_at0 = C::kCodes + ((2 * j) ^ ((j >> 1) & 1)) * C::kRow + i * 4;
  const uint32_t v_at1 = C::kCodes + ((2 * j + 1) ^ ((j >> 1) & 1)) * C::kRow + i * 4;
  const uint32_t v_swap = D == 128 ? (j & 1) * 32 : 0;

  int stage = 0;
  for (int tile = t0 + warp; tile < t1; tile += kWarps, next += kWarps) {
    kv4_cp_wait<C::kStages - 2>();
    __syncwarp();  // every lane's pieces have landed, and every lane has left the stage refilled below
    if (next < t1) issue(next, stage == 0 ? C::kStages - 1 : stage - 1);
    kv4_cp_commit();
    const uint32_t st = ring + stage * C::kStage;
    const uint32_t sp = st + 2 * C::kCodes;
    const int r0 = row_of(tile);

    // ---- scores, in units of log2 ---------------------------------------------
    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[mt][nt][c] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint2 wa = lds64(st + mt * 16 * C::kRow + k_at + ((g * 32) ^ k_swap));
        const uint2 wb = lds64(st + (mt * 16 + 8) * C::kRow + k_at + ((g * 32) ^ k_swap));
        const uint32_t pa = lds32(sp + ((mt * 16 + i) * NG + g) * 4), pb = lds32(sp + ((mt * 16 + i + 8) * NG + g) * 4);
        float d[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) d[nt][c] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t xa = (ks < 2 ? wa.x : wa.y) >> ((ks & 1) * 8), xb = (ks < 2 ? wb.x : wb.y) >> ((ks & 1) * 8);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_f16(d[nt], xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u, qf[g][ks][nt][0],
                    qf[g][ks][nt][1]);
        }
        const float sa = bf16_lo(pa), ma = bf16_hi(pa), sb = bf16_lo(pb), mb = bf16_hi(pb);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[mt][nt][0] = fmaf(d[nt][0], sa, fmaf(qs[g][nt][0], ma, s[mt][nt][0]));
          s[mt][nt][1] = fmaf(d[nt][1], sa, fmaf(qs[g][nt][1], ma, s[mt][nt][1]));
          s[mt][nt][2] = fmaf(d[nt][2], sb, fmaf(qs[g][nt][0], mb, s[mt][nt][2]));
          s[mt][nt][3] = fmaf(d[nt][3], sb, fmaf(qs[g][nt][1], mb, s[mt][nt][3]));
        }
      }
    }
    const bool masked = !(r0 + kTile <= a.n_sink || (r0 >= lo_max && r0 + kTile <= hi_min));
    bool above = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = r0 + mt * 16 + i + (c >> 1) * 8;
          s[mt][nt][c] *= rs[nt][c & 1];
          if (masked && !(r < a.n_sink || (r >= lo[nt][c & 1] && r < hi[nt][c & 1]))) s[mt][nt][c] = -INFINITY;
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[nt][c] = fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2]));
        above |= top[nt][c] > mx[nt][c] + kSlack;
      }
    }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(top[nt][c], mx[nt][c]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          const float alpha = x == -INFINITY ? 1.f : fast_exp2(mx[nt][c] - x);
          mx[nt][c] = x;
          lsum[nt][c] *= alpha;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            accm[g][nt][c] *= alpha;
            accr[g][nt][c] *= alpha;
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
        const float ref = mx[nt][c] == -INFINITY ? 0.f : mx[nt][c];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          s[mt][nt][c] = fast_exp2(s[mt][nt][c] - ref);
          s[mt][nt][c + 2] = fast_exp2(s[mt][nt][c + 2] - ref);
          lsum[nt][c] += s[mt][nt][c] + s[mt][nt][c + 2];
        }
      }

    // ---- output -----------------------------------------------------------------
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t pa = lds32(sp + C::kParams + ((mt * 16 + i) * NG + g) * 4);
        const uint32_t pb = lds32(sp + C::kParams + ((mt * 16 + i + 8) * NG + g) * 4);
        const float sa = bf16_lo(pa), sb = bf16_lo(pb);
        const float ca = fmaf(8.f, sa, bf16_hi(pa)), cb = fmaf(8.f, sb, bf16_hi(pb));
        uint32_t bw[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float* p = s[mt][nt];
          float x0 = p[0] * sa, x1 = p[1] * sa, x2 = p[2] * sb, x3 = p[3] * sb;
          if (masked) {  // a key that a row does not see may hold anything
            x0 = p[0] == 0.f ? 0.f : x0;
            x1 = p[1] == 0.f ? 0.f : x1;
            x2 = p[2] == 0.f ? 0.f : x2;
            x3 = p[3] == 0.f ? 0.f : x3;
            accm[g][nt][0] += (p[0] == 0.f ? 0.f : p[0] * ca) + (p[2] == 0.f ? 0.f : p[2] * cb);
            accm[g][nt][1] += (p[1] == 0.f ? 0.f : p[1] * ca) + (p[3] == 0.f ? 0.f : p[3] * cb);
          } else {
            accm[g][nt][0] = fmaf(p[0], ca, fmaf(p[2], cb, accm[g][nt][0]));
            accm[g][nt][1] = fmaf(p[1], ca, fmaf(p[3], cb, accm[g][nt][1]));
          }
          bw[nt][0] = movmatrix_trans(pack_bf16x2(x0, x1));
          bw[nt][1] = movmatrix_trans(pack_bf16x2(x2, x3));
          mma_bf16(accr[g][nt], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, bw[nt][0], bw[nt][1]);
        }
        const uint32_t at = st + mt * 16 * C::kRow + ((g * 32) ^ v_swap);
        const uint32_t w0 = lds32(at + v_at0), w1 = lds32(at + v_at1);
        const uint32_t w8 = lds32(at + v_at0 + 8 * C::kRow), w9 = lds32(at + v_at1 + 8 * C::kRow);
        const uint32_t l0 = __byte_perm(w0, w1, 0x5410), h0 = __byte_perm(w0, w1, 0x7632);
        const uint32_t l8 = __byte_perm(w8, w9, 0x5410), h8 = __byte_perm(w8, w9, 0x7632);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_bf16(acc[g][0][nt], nibbles_bf16<0>(l0), nibbles_bf16<0>(h0), nibbles_bf16<0>(l8), nibbles_bf16<0>(h8),
                   bw[nt][0], bw[nt][1]);
          mma_bf16(acc[g][1][nt], nibbles_bf16<1>(l0), nibbles_bf16<1>(h0), nibbles_bf16<1>(l8), nibbles_bf16<1>(h8),
                   bw[nt][0], bw[nt][1]);
          mma_bf16(acc[g][2][nt], nibbles_bf16<2>(l0), nibbles_bf16<2>(h0), nibbles_bf16<2>(l8), nibbles_bf16<2>(h8),
                   bw[nt][0], bw[nt][1]);
          mma_bf16(acc[g][3][nt], nibbles_bf16<3>(l0), nibbles_bf16<3>(h0), nibbles_bf16<3>(l8), nibbles_bf16<3>(h8),
                   bw[nt][0], bw[nt][1]);
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
        sml[2 * r] = mx[nt][c];
        sml[2 * r + 1] = l;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float m = accm[g][nt][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        m = fmaf(-24.f, accr[g][nt][c], m);
        float* o = so + r * D + g * 64 + 8 * i;
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) {
          o[mm] = acc[g][mm][nt][c] + m;
          o[4 + mm] = acc[g][mm][nt][c + 2] + m;
        }
      }
    }
  __syncthreads();
  float* pml = a.part + (size_t)a.B * a.Tn * a.H * splits * D;
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
    const int row = row0 + r;
    const long long head = ((long long)b * a.Tn + row / G) * a.H + hk * G + row % G;
    if (splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      reinterpret_cast<uint32_t*>(a.out)[(head * D + d) / 2] = kv4_pack2<TYPE>(x * inv, y * inv);
    } else {
      const long long at = head * splits + split;
      *reinterpret_cast<float2*>(a.part + at * D + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(pml + at * 2) = make_float2(top, l);
    }
  }
}

template <int D, int NT, int TYPE>
void launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  auto kern = kv4_heads_kernel<D, NT, TYPE>;
  constexpr int smem = HeadsCfg<D, NT>::kSmem;
  ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  kern<<<dim3((unsigned)(p.splits * p.row_blocks), (unsigned)a.Hk, (unsigned)a.B), kWarps * 32, smem, s>>>(a, p.splits);
}

template <int TYPE>
void launch_dims(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  if (a.W == 128)
    p.row_tiles == 1 ? launch<128, 1, TYPE>(a, p, s) : launch<128, 2, TYPE>(a, p, s);
  else
    p.row_tiles == 1 ? launch<64, 1, TYPE>(a, p, s) : launch<64, 2, TYPE>(a, p, s);
}

// One output row (sequence, token, head) per block: join its splits.
template <int TYPE>
__global__ void kv4_combine_kernel(const Kv4Attend a, const int splits) {
  const long long row = blockIdx.x;
  const float* pml = a.part + (size_t)a.B * a.Tn * a.H * splits * a.V + row * splits * 2;
  float top = -INFINITY;
  for (int k = 0; k < splits; ++k) top = fmaxf(top, pml[2 * k]);
  const float ref = top == -INFINITY ? 0.f : top;
  const int d = threadIdx.x * 2;
  float l = 0.f, x = 0.f, y = 0.f;
  for (int k = 0; k < splits; ++k) {
    const float f = fast_exp2(pml[2 * k] - ref);
    const float2 v = *reinterpret_cast<const float2*>(a.part + (row * splits + k) * a.V + d);
    l = fmaf(f, pml[2 * k + 1], l);
    x = fmaf(f, v.x, x);
    y = fmaf(f, v.y, y);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  reinterpret_cast<uint32_t*>(a.out)[(row * a.V + d) / 2] = kv4_pack2<TYPE>(x * inv, y * inv);
}

}  // namespace

void kv4_combine(const Kv4Attend& a, int splits, cudaStream_t s) {
  const unsigned rows = (unsigned)((long long)a.B * a.Tn * a.H);
  if (a.type == KV4_F16) kv4_combine_kernel<KV4_F16><<<rows, a.V / 2, 0, s>>>(a, splits);
  else kv4_combine_kernel<KV4_BF16><<<rows, a.V / 2, 0, s>>>(a, splits);
}

void kv4_heads_plan(const Kv4Attend& a, Kv4Plan& p) {
  const int R = a.Tn * (a.H / a.Hk);
  p.kernel = 1;
  p.row_tiles = R <= 8 ? 1 : 2;
  p.row_blocks = (R + 8 * p.row_tiles - 1) / (8 * p.row_tiles);
  // The host knows the cache's size, not the sequences' lengths: plan for a full cache (or window).
  // Cost of a split count: waves of blocks times the tiles a warp walks, plus about four tiles' time
  // to start and to join a block.
  const long long rows = std::min<long long>(a.L - a.sink_rows, a.window > 0 ? a.window + a.Tn : 1 << 30);
  const int tiles = (a.n_sink + kTile - 1) / kTile + (int)((rows + kTile - 1) / kTile) + 1;
  const long long blocks = (long long)a.B * a.Hk * p.row_blocks, slots = 148 * (p.row_tiles == 1 ? 3 : 2);
  long long best = -1;
  for (int sp = 1; sp <= 64 && (sp == 1 || tiles >= sp * kWarps); ++sp) {
    const long long waves = (blocks * sp + slots - 1) / slots;
    const long long per_warp = ((tiles + sp - 1) / sp + kWarps - 1) / kWarps;
    const long long cost = waves * (per_warp + 4) + (sp > 1 ? 6 : 0);
    if (best < 0 || cost < best) {
      best = cost;
      p.splits = sp;
    }
  }
  p.floats = p.splits > 1 ? (size_t)a.B * a.Tn * a.H * p.splits * (a.V + 2) : 0;
}

void kv4_heads_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  if (a.type == KV4_F16) launch_dims<KV4_F16>(a, p, s);
  else launch_dims<KV4_BF16>(a, p, s);
  if (p.splits > 1) kv4_combine(a, p.splits, s);
}

}  // namespace omni
