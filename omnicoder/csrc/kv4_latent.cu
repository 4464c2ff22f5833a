// Attention of a few query rows against a 4-bit latent cache (sm_100a): every
// head reads the same rows of W = r + 64 dims, whose first r dims are the value
// (r = 512 or 256, groups of 64).  The algebra is that of kv4_heads.cu:
//   score_t = sum_g s_tg (q_g . n_tg) + sum_g m_tg sum(q_g)
//   o_d     = sum_t (p_t s_tg) (n_td - 8) + sum_t p_t (m_tg + 8 s_tg)
//
// 16 rows of up to 576 + 512 products per key are too much output for one warp's
// registers, so the four warps of a block share a tile of 128 keys: each warp
// scores 32 of them over all groups, then the weights go through shared memory
// and each warp accumulates a quarter of the value dims over all 128.  A tile is
// one contiguous piece of memory and arrives by two bulk copies on an mbarrier.
// The sum over groups of m sum(q_g) is a product of its own, keys x groups, with
// m in bf16 as stored and sum(q_g) split into three bf16 terms: nine
// multiply-adds per score less.
#include <algorithm>

#include "kv4_device.cuh"

namespace omni {

void* status_ptr();  // bindings.cpp

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 128;
constexpr int kStages = 2;
constexpr int kRows = 16;       // query rows of a block (two mma columns of 8)
constexpr int NT = kRows / 8;
constexpr float kSlack = 8.f;
constexpr int kPRow = kTile + 8;  // floats per row of weights: rows 32 bytes apart modulo 128

template <int V>
struct LatentCfg {
  static constexpr int W = V + 64;
  static constexpr int NG = W / 64;                  // key groups
  static constexpr int VG = V / 64 / kWarps;         // value groups of a warp
  static constexpr int kRow = W / 2;
  static constexpr int kCodes = kTile * kRow;
  static constexpr int kParams = kTile * NG * 4;
  static constexpr int kStage = kCodes + kParams;
  static constexpr int kQf = kStages * kStage;       // query operands [NG * 4][32 lanes][4]
  static constexpr int kP = kQf + NG * 4 * 32 * 16;  // weights [kRows][kPRow]
  static constexpr int kMisc = kP + kRows * kPRow * 4;  // sums of q, factors, maxima, barriers
  static constexpr int kSmem = kMisc + kRows * (16 + 1 + kWarps + 1) * 4 + kRows * 2 * 4 + kStages * 8;
};

template <int V, int TYPE>
__global__ void __launch_bounds__(kWarps * 32, 2) kv4_latent_kernel(const Kv4Attend a, const Kv4Line line, StatusBlock* st) {
  using C = LatentCfg<V>;
  constexpr int W = C::W, NG = C::NG, VG = C::VG;
  extern __shared__ __align__(128) uint8_t smem[];
  uint32_t* sqf = reinterpret_cast<uint32_t*>(smem + C::kQf);
  float* sp = reinterpret_cast<float*>(smem + C::kP);
  float* sqs = reinterpret_cast<float*>(smem + C::kMisc);  // [kRows][16]: sum(q_g) 2^-24, zero from NG on
  float* srs = sqs + kRows * 16;                           // [kRows]: factor of the scores
  float* smx = srs + kRows;                                // [kWarps][kRows]
  float* sal = smx + kWarps * kRows;                       // [kRows]: rescaling of this tile
  int* slo = reinterpret_cast<int*>(sal + kRows);          // [kRows], then hi
  int* shi = slo + kRows;
  uint64_t* full = reinterpret_cast<uint64_t*>(shi + kRows);
  const int tid = threadIdx.x, lane = lane_id(), warp = warp_id(), i = lane >> 2, j = lane & 3;
  const int R = a.Tn * a.H;
  if (tid == 0) {
    for (int k = 0; k < kStages; ++k) mbar_init(&full[k], 1);
    fence_barrier_init();
  }
  if (line.min_steps > 0) launch_dependents();
  Kv4Walk walk;
  walk.begin(a, line);
  int used = 0;     // tiles that went through the stages
  bool ok = true;

  while (walk.at < walk.end) {
  int t0, step1;
  const Kv4Piece piece = walk.next(a, line, kRows, &t0, &step1);
  const int b = piece.b, row0 = piece.segment * kRows, nrows = min(kRows, R - row0);
  const int sink_tiles = piece.sink_tiles, first = piece.first, t1 = min(piece.tiles, step1);
  Kv4Seen seen{0, 0};
  if (lane < nrows) seen = kv4_seen(a, b, (row0 + lane) / a.H);
  const int lo_max = __reduce_max_sync(0xffffffffu, lane < nrows ? seen.lo : 0);
  const int hi_min = __reduce_min_sync(0xffffffffu, lane < nrows ? seen.hi : a.L);
  auto row_of = [&](int tile) { return (tile < sink_tiles ? tile : first + tile - sink_tiles) * kTile; };

  const uint8_t* kc = a.k.codes + b * a.k.c_b;
  const uint8_t* kp = a.k.params + b * a.k.p_b;
  auto issue = [&](int tile, int stage) {  // one thread; rows behind the cache's end are not copied
    const long long r0 = row_of(tile);
    const uint32_t n = (uint32_t)min((long long)kTile, a.L - r0);
    uint8_t* dst = smem + stage * C::kStage;
    mbar_arrive_expect_tx(&full[stage], n * (C::kRow + NG * 4));
    bulk_load(dst, kc + r0 * C::kRow, n * C::kRow, &full[stage]);
    bulk_load(dst + C::kCodes, kp + r0 * (NG * 4), n * NG * 4, &full[stage]);
  };
  if (tid == 0)
    for (int k = 0; k < kStages; ++k)
      if (t0 + k < t1) issue(t0 + k, (used + k) % kStages);

  // ---- queries: normalised fp16, laid out as the operands of the scores ------------
  for (int r = warp; r < kRows; r += kWarps) {
    float x[W / 32], amax = 0.f, un;
    const long long at = ((long long)b * R + row0 + r) * W;
#pragma unroll
    for (int e = 0; e < W / 32; ++e) {
      x[e] = r < nrows ? kv4_load1<TYPE>(a.q, at + lane + 32 * e) : 0.f;
      amax = fmaxf(amax, fabsf(x[e]));
    }
    const float sc = q_normaliser(warp_max(amax), &un);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = lane + 32 * e;                   // dim of the group: lane d / 16 reads words d / 8
        const __half h = __float2half_rn(x[2 * g + e] * sc);
        sum += __half2float(h);
        const int jj = d >> 4, ks = ((d >> 3) & 1) * 2 + ((d >> 1) & 1), odd = d & 1, hi = (d >> 2) & 1;
        const __half v = odd ? __hmul(h, __float2half_rn(0.0625f)) : h;
        // [g, ks][lane (r & 7, jj)][row tile, even / odd nibble][low / high half]
        reinterpret_cast<__half*>(sqf)[(((g * 4 + ks) * 32 + (r & 7) * 4 + jj) * 4 + (r >> 3) * 2 + odd) * 2 + hi] = v;
      }
      sum = warp_sum(sum);
      if (lane == 0) sqs[r * 16 + g] = sum * 5.9604644775390625e-8f;
    }
    if (lane >= NG && lane < 16) sqs[r * 16 + lane] = 0.f;
    if (lane == 0) srs[r] = un * (a.scale * (kKv4Log2e * kKv4Codes));
  }
  if (warp == 0 && lane < kRows) {
    slo[lane] = seen.lo;
    shi[lane] = seen.hi;
  }
  __syncthreads();

  // operands of the minima's product: three bf16 terms of sum(q_g), row i, groups 2j, 2j + 1, +8, +9
  uint32_t qm[3][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float u = sqs[(nt * 8 + i) * 16 + 8 * h + 2 * j], v = sqs[(nt * 8 + i) * 16 + 8 * h + 2 * j + 1];
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        qm[k][nt][h] = pack_bf16x2(u, v);
        u -= bf16_lo(qm[k][nt][h]);
        v -= bf16_hi(qm[k][nt][h]);
      }
    }
  float rs[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) rs[nt][c] = srs[nt * 8 + 2 * j + c];

  float acc[VG][4][NT][4], accr[VG][NT][4], accm[VG][NT], lsum[NT][2], mx[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int g = 0; g < VG; ++g) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        accr[g][nt][c] = 0.f;
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) acc[g][mm][nt][c] = 0.f;
      }
      accm[g][nt] = 0.f;
    }
    lsum[nt][0] = lsum[nt][1] = 0.f;
    mx[nt][0] = mx[nt][1] = -INFINITY;
  }

  // Row t of an mma tile of 16 keys is key t ^ bit2(t): the rows that one load touches then start in
  // different 32-byte slots of the banks (rows are 32 bytes apart modulo 128).
  const int key_i = i ^ ((i >> 2) & 1);
  const int key_0 = (2 * j) ^ ((j >> 1) & 1), key_1 = (2 * j + 1) ^ ((j >> 1) & 1);

  for (int tile = t0; tile < t1; ++tile) {
    const int stage = (used + tile - t0) % kStages;
    ok = mbar_wait(&full[stage], ((used + tile - t0) / kStages) & 1, st, STATUS_TIMEOUT_TMA_FULL) && ok;
    const uint32_t codes = smem_u32(smem + stage * C::kStage), params = codes + C::kCodes;
    const int r0 = row_of(tile);

    // ---- scores of this warp's 32 keys ---------------------------------------------
    float s[2][NT][4];
    const uint32_t k_at = codes + (warp * 32 + key_i) * C::kRow + j * 8;
    const uint32_t p_at = params + (warp * 32 + key_i) * NG * 4;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[mt][nt][c] = 0.f;
      uint32_t m[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {  // keys i, i + 8 against groups 2j, 2j + 1, then + 8
        const uint32_t at = p_at + (mt * 16 + (h & 1) * 8) * NG * 4;
        const int g = 2 * j + (h >> 1) * 8;
        m[h] = __byte_perm(g < NG ? lds32(at + g * 4) : 0u, g + 1 < NG ? lds32(at + g * 4 + 4) : 0u, 0x7632);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 3; ++k) mma_bf16(s[mt][nt], m[0], m[1], m[2], m[3], qm[k][nt][0], qm[k][nt][1]);
    }
    // rolled, as the loop over the values below: the code must stay in the instruction cache
#pragma unroll 1
    for (int g = 0; g < NG; ++g) {
      uint2 wa[2], wb[2];
      float d[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        wa[mt] = lds64(k_at + mt * 16 * C::kRow + g * 32);
        wb[mt] = lds64(k_at + (mt * 16 + 8) * C::kRow + g * 32);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) d[mt][nt][c] = 0.f;
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint4 q = *reinterpret_cast<const uint4*>(sqf + ((g * 4 + ks) * 32 + lane) * 4);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t xa = (ks < 2 ? wa[mt].x : wa[mt].y) >> ((ks & 1) * 8);
          const uint32_t xb = (ks < 2 ? wb[mt].x : wb[mt].y) >> ((ks & 1) * 8);
          mma_f16(d[mt][0], xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u, q.x, q.y);
          mma_f16(d[mt][1], xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u, q.z, q.w);
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float sa = bf16_lo(lds32(p_at + (mt * 16 * NG + g) * 4));
        const float sb = bf16_lo(lds32(p_at + ((mt * 16 + 8) * NG + g) * 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[mt][nt][0] = fmaf(d[mt][nt][0], sa, s[mt][nt][0]);
          s[mt][nt][1] = fmaf(d[mt][nt][1], sa, s[mt][nt][1]);
          s[mt][nt][2] = fmaf(d[mt][nt][2], sb, s[mt][nt][2]);
          s[mt][nt][3] = fmaf(d[mt][nt][3], sb, s[mt][nt][3]);
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
          const int r = r0 + warp * 32 + mt * 16 + key_i + (c >> 1) * 8, q = nt * 8 + 2 * j + (c & 1);
          s[mt][nt][c] *= rs[nt][c & 1];
          if (masked && !(r < a.n_sink || (r >= slo[q] && r < shi[q]))) s[mt][nt][c] = -INFINITY;
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[nt][c] = fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2]));
        above |= top[nt][c] > mx[nt][c] + kSlack;
      }
    }
    // also the barrier behind the previous tile's reads of the weights
    if (__syncthreads_or(above)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = top[nt][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          if (i == 0) smx[warp * kRows + nt * 8 + 2 * j + c] = x;
        }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = nt * 8 + 2 * j + c;
          float x = mx[nt][c];
#pragma unroll
          for (int w = 0; w < kWarps; ++w) x = fmaxf(x, smx[w * kRows + q]);
          const float alpha = x == -INFINITY ? 1.f : fast_exp2(mx[nt][c] - x);
          mx[nt][c] = x;
          lsum[nt][c] *= alpha;
          if (warp == 0 && i == 0) sal[q] = alpha;
#pragma unroll
          for (int g = 0; g < VG; ++g) {
            accr[g][nt][c] *= alpha;
#pragma unroll
            for (int mm = 0; mm < 4; ++mm) {
              acc[g][mm][nt][c] *= alpha;
              acc[g][mm][nt][c + 2] *= alpha;
            }
          }
        }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < VG; ++g) accm[g][nt] *= sal[nt * 8 + i];
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float ref = mx[nt][c] == -INFINITY ? 0.f : mx[nt][c];
        float* o = sp + (nt * 8 + 2 * j + c) * kPRow + warp * 32 + i;   // by mma row, not by key
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float x = fast_exp2(s[mt][nt][c] - ref), y = fast_exp2(s[mt][nt][c + 2] - ref);
          lsum[nt][c] += x + y;
          o[mt * 16] = x;
          o[mt * 16 + 8] = y;
        }
      }
    __syncthreads();

    // ---- output: this warp's value groups over all keys of the tile -------------------
#pragma unroll 1
    for (int kt = 0; kt < kTile / 16; ++kt) {
      float2 p0[NT], p8[NT];  // weights of row i at mma rows 2j, 2j + 1 and + 8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float* p = sp + (nt * 8 + i) * kPRow + kt * 16 + 2 * j;
        p0[nt] = *reinterpret_cast<const float2*>(p);
        p8[nt] = *reinterpret_cast<const float2*>(p + 8);
      }
      const uint32_t c0 = codes + (kt * 16 + key_0) * C::kRow + i * 4, c1 = codes + (kt * 16 + key_1) * C::kRow + i * 4;
      const uint32_t q0 = params + (kt * 16 + key_0) * NG * 4, q1 = params + (kt * 16 + key_1) * NG * 4;
#pragma unroll
      for (int g = 0; g < VG; ++g) {
        const int vg = warp * VG + g;
        const uint32_t w0 = lds32(c0 + vg * 32), w1 = lds32(c1 + vg * 32);
        const uint32_t w8 = lds32(c0 + 8 * C::kRow + vg * 32), w9 = lds32(c1 + 8 * C::kRow + vg * 32);
        const uint32_t u0 = lds32(q0 + vg * 4), u1 = lds32(q1 + vg * 4);
        const uint32_t u8 = lds32(q0 + (8 * NG + vg) * 4), u9 = lds32(q1 + (8 * NG + vg) * 4);
        const float s0 = bf16_lo(u0), s1 = bf16_lo(u1), s8 = bf16_lo(u8), s9 = bf16_lo(u9);
        const float m0 = fmaf(8.f, s0, bf16_hi(u0)), m1 = fmaf(8.f, s1, bf16_hi(u1));
        const float m8 = fmaf(8.f, s8, bf16_hi(u8)), m9 = fmaf(8.f, s9, bf16_hi(u9));
        uint32_t bw[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (masked) {  // a key that a row does not see may hold anything
            auto times = [](float p, float x) { return p == 0.f ? 0.f : p * x; };
            bw[nt][0] = pack_bf16x2(times(p0[nt].x, s0), times(p0[nt].y, s1));
            bw[nt][1] = pack_bf16x2(times(p8[nt].x, s8), times(p8[nt].y, s9));
            accm[g][nt] += times(p0[nt].x, m0) + times(p0[nt].y, m1) + times(p8[nt].x, m8) + times(p8[nt].y, m9);
          } else {
            bw[nt][0] = pack_bf16x2(p0[nt].x * s0, p0[nt].y * s1);
            bw[nt][1] = pack_bf16x2(p8[nt].x * s8, p8[nt].y * s9);
            accm[g][nt] = fmaf(p0[nt].x, m0, fmaf(p0[nt].y, m1, fmaf(p8[nt].x, m8, fmaf(p8[nt].y, m9, accm[g][nt]))));
          }
          mma_bf16(accr[g][nt], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, bw[nt][0], bw[nt][1]);
        }
        const uint32_t l0 = __byte_perm(w0, w1, 0x5410), h0 = __byte_perm(w0, w1, 0x7632);
        const uint32_t l8 = __byte_perm(w8, w9, 0x5410), h8 = __byte_perm(w8, w9, 0x7632);
        mma_values<0, NT>(acc[g][0], l0, h0, l8, h8, bw);
        mma_values<1, NT>(acc[g][1], l0, h0, l8, h8, bw);
        mma_values<2, NT>(acc[g][2], l0, h0, l8, h8, bw);
        mma_values<3, NT>(acc[g][3], l0, h0, l8, h8, bw);
      }
    }
    if (tile + kStages < t1) {
      __syncthreads();  // every warp has left the stage
      if (tid == 0) issue(tile + kStages, stage);
    }
  }
  used += max(0, t1 - t0);

  // ---- join: row maxima are the block's already; sums over the warps' keys -------------
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = lsum[nt][c];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (i == 0) smx[warp * kRows + nt * 8 + 2 * j + c] = l;
    }
  // sums of p (m + 8 s): lane (i, j) holds row i over the keys of j
#pragma unroll
  for (int g = 0; g < VG; ++g)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float m = accm[g][nt];
      m += __shfl_xor_sync(0xffffffffu, m, 1);
      m += __shfl_xor_sync(0xffffffffu, m, 2);
      if (j == 0) sp[(warp * VG + g) * kRows + nt * 8 + i] = m;
    }
  __syncthreads();
  const bool alone = t0 == 0 && step1 == piece.steps;
  float* part = a.part + (size_t)(2 * blockIdx.x + (t0 == 0)) * kRows * (V + 2);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int q = nt * 8 + 2 * j + c;
      if (q >= nrows) continue;
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) l += smx[w * kRows + q];
      const float inv = !alone ? 1.f : (l == 0.f ? 0.f : 1.f / l);
#pragma unroll
      for (int g = 0; g < VG; ++g) {
        const float m = fmaf(-24.f, accr[g][nt][c], sp[(warp * VG + g) * kRows + q]);
        float o[8];
#pragma unroll
        for (int mm = 0; mm < 4; ++mm) {
          o[mm] = (acc[g][mm][nt][c] + m) * inv;
          o[4 + mm] = (acc[g][mm][nt][c + 2] + m) * inv;
        }
        const int d = (warp * VG + g) * 64 + 8 * i;
        if (!alone) {
          float4* p = reinterpret_cast<float4*>(part + q * V + d);
          p[0] = make_float4(o[0], o[1], o[2], o[3]);
          p[1] = make_float4(o[4], o[5], o[6], o[7]);
        } else {
          *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + ((long long)b * R + row0 + q) * V + d) =
              make_uint4(kv4_pack2<TYPE>(o[0], o[1]), kv4_pack2<TYPE>(o[2], o[3]), kv4_pack2<TYPE>(o[4], o[5]),
                         kv4_pack2<TYPE>(o[6], o[7]));
        }
      }
      if (!alone && warp == 0 && i == 0)
        *reinterpret_cast<float2*>(part + kRows * V + 2 * q) = make_float2(mx[nt][c], l);
    }
  __syncthreads();  // the next segment refills shared memory
  }
  (void)ok;
}

template <int V, int TYPE>
void launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  auto kern = kv4_latent_kernel<V, TYPE>;
  constexpr int smem = LatentCfg<V>::kSmem;
  ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  kern<<<p.blocks, kWarps * 32, smem, s>>>(a, kv4_line(a, p, kTile),
                                           reinterpret_cast<StatusBlock*>(status_ptr()));
}

}  // namespace

void kv4_latent_plan(const Kv4Attend& a, Kv4Plan& p) {
  p.kernel = 2;
  p.row_tiles = NT;
  p.row_blocks = (a.Tn * a.H + kRows - 1) / kRows;
  kv4_line_plan(a, p, 148 * 2, 1);
}

void kv4_latent_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  if (a.type == KV4_F16)
    a.V == 512 ? launch<512, KV4_F16>(a, p, s) : launch<256, KV4_F16>(a, p, s);
  else
    a.V == 512 ? launch<512, KV4_BF16>(a, p, s) : launch<256, KV4_BF16>(a, p, s);
  if (p.min_steps > 0) kv4_combine(a, p, s);
}

}  // namespace omni
