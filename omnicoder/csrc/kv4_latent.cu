// Attention of a few query rows against a 4-bit latent cache (sm_100a): every
// head reads the same rows of W = r + 64 dims, whose first r dims are the value
// (r = 512 or 256, groups of 64).  The algebra is that of kv4_heads.cu:
//   score_t = sum_g s_tg (q_g . n_tg) + sum_g m_tg sum(q_g)
//   o_d     = sum_t (p_t s_tg) n_td + sum_t p_t m_tg
//
// 16 rows of up to 576 + 512 products per key are too much output for one warp's
// registers, so the eight warps of a block share a tile of 128 keys: each warp
// scores 16 of them over all groups, then the weights go through shared memory
// and each warp accumulates one group of the value dims over all 128 (r = 256: over
// half of them, 31 us for 8 x 4 tokens where half a group's dims took 33).  A tile is one contiguous piece of memory and arrives by two bulk
// copies on an mbarrier.
// The sum over groups of m sum(q_g) is a product of its own, keys x groups, with
// m in bf16 as stored and sum(q_g) split into three bf16 terms: nine
// multiply-adds per score less.
//
// Measured: 64 sequences x 4160 rows of 512 + 64 dims, 16 heads: 70 us, 1.3 TB/s.
// Bound by tensor (33 %), ALU (41 %) and FMA (17 %) issue together and the three
// phases' latency, which two blocks per SM do not hide; a third does not fit in
// shared memory.  Their 128 registers spill 56 and 40 bytes (256 value dims: 8 and 8).
// Four warps of two key tiles each took 78 us.  One sequence of 8192 rows: 13.7 us.
#include <algorithm>

#include "kv4_device.cuh"

namespace omni {

void* status_ptr();  // bindings.cpp

namespace {

constexpr int kWarps = 8;
constexpr int kTile = 16 * kWarps;
constexpr int kStages = 2;
constexpr int kRows = 16;       // query rows of a block (two mma columns of 8)
constexpr int NT = kRows / 8;
constexpr float kSlack = 8.f;
constexpr int kPRow = kTile + 8;  // floats per row of weights: rows 32 bytes apart modulo 128

template <int V>
struct LatentCfg {
  static constexpr int W = V + 64;
  static constexpr int NG = W / 64;                  // key groups
  static constexpr int VG = V / 64;                  // value groups: one per warp,
  static constexpr int KS = kWarps / VG;             // or per pair of warps that halve the keys
  static constexpr int kRow = W / 2;
  static constexpr int kCodes = kTile * kRow;
  static constexpr int kParams = kTile * NG * 4;
  static constexpr int kStage = kCodes + kParams;
  static constexpr int kQf = kStages * kStage;       // query operands [NG * 4 k steps][32 lanes][row tile]
  static constexpr int kP = kQf + NG * 4 * 32 * 16;  // weights [kRows][kPRow]
  static constexpr int kMisc = kP + kRows * kPRow * 4;  // sums of q, factors, maxima, barriers
  static constexpr int kSmem = kMisc + kRows * (16 + 1 + kWarps + 1) * 4 + kRows * 2 * 4 + kStages * 8;
};

template <int V, int TYPE, int PER_SM>
__global__ void __launch_bounds__(kWarps * 32, PER_SM) kv4_latent_kernel(const Kv4Attend a, const Kv4Line line, StatusBlock* st) {
  using C = LatentCfg<V>;
  constexpr int W = C::W, NG = C::NG, KS = C::KS;
  extern __shared__ __align__(128) uint8_t smem[];
  uint2* sqf = reinterpret_cast<uint2*>(smem + C::kQf);
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
  wait_for_previous_grid();
  launch_dependents();
  __shared__ Kv4Walk walk;
  int share = 0;
  int2 span = walk.begin<kWarps * 32, kTile>(a, line, &share);
  int used = 0;     // tiles that went through the stages
  // Behind a wait that ran out (uniform over the block): nothing is copied or read any more, and this
  // piece and the block's later ones become NaN; their places are noted all the same.
  bool dead = false;

  while (span.x < span.y) {
  Kv4Piece piece = walk.next<kTile>(a, line, share, &span);
  const int b = piece.b, row0 = piece.segment * kRows, nrows = min(kRows, R - row0);
  // query rows, two per warp, a lane eight dims (a code word); asked for before anything waits
  constexpr int kWords = W / 8, kPer = (2 * kWords + 31) / 32;
  float x[kPer][8] = {};
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int at = lane + 32 * e, second = at >= kWords, r = 2 * warp + second, w = at - second * kWords;
    if (w < kWords && r < nrows) kv4_load8<TYPE>(a.q, ((long long)b * R + row0 + r) * W + w * 8, x[e]);
  }
  const Kv4View see = kv4_rows<kTile>(a, line, &piece, row0, nrows);
  const int sink_tiles = piece.sink_tiles, first = piece.first, t0 = piece.step0;
  const int t1 = dead ? t0 : min(piece.tiles, piece.step1);
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

  // ---- queries: normalised fp16, laid out as the operands of the scores ---------------------------
  {
    static_assert(kRows == 2 * kWarps && kWords % 8 == 0, "two rows a warp, groups within eight lanes");
    const int r0 = 2 * warp;
    float amax[2] = {}, sc[2], un[2];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const bool second = lane + 32 * e >= kWords;
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[e][k]));
      if (second) amax[1] = fmaxf(amax[1], top);
      else amax[0] = fmaxf(amax[0], top);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = q_normaliser(warp_max(amax[h]), &un[h]);
      if (lane == h) srs[r0 + h] = un[h] * (a.scale * kKv4Log2e);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int at = lane + 32 * e, second = at >= kWords, r = r0 + second, w = at - second * kWords, g = w >> 3;
      float sum = 0.f;
      if (w < kWords) {
        const float by = second ? sc[1] : sc[0];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[e][k] *= by;
        uint2 q[2];
        sum = query_pairs(x[e], q);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          sqf[((g * 4 + (w & 1) * 2 + k) * 32 + (r & 7) * 4 + ((w >> 1) & 3)) * NT + (r >> 3)] = q[k];
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if ((lane & 7) == 0 && w < kWords) sqs[r * 16 + g] = sum * (1.f / kKv4Codes);
    }
    if ((lane & 15) >= NG) sqs[(r0 + (lane >> 4)) * 16 + (lane & 15)] = 0.f;
  }
  if (warp == 0 && lane < kRows) {
    slo[lane] = see.seen.lo;
    shi[lane] = see.seen.hi;
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
  const bool huge = kv4_score_factors<NT>(rs);

  // acc[mm]: value dims mm and 4 + mm of a lane's eight; accm: sums of p m
  float f = 0.f;   // the values' power of two; 0 before any
  float acc[4][NT][4], accm[NT], lsum[NT][2], limit[NT][2], ref[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mm = 0; mm < 4; ++mm)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[mm][nt][c] = 0.f;
    accm[nt] = 0.f;
    lsum[nt][0] = lsum[nt][1] = dead ? __int_as_float(0x7fffffff) : 0.f;
    limit[nt][0] = limit[nt][1] = -INFINITY;
    ref[nt][0] = ref[nt][1] = 0.f;
  }

  // Row t of an mma tile of 16 keys is key t ^ bit2(t): the rows that one load touches then start in
  // different 32-byte slots of the banks (rows are 32 bytes apart modulo 128).
  const int key_i = i ^ ((i >> 2) & 1);
  // this warp's value group and, of the tile's key tiles, its share
  const int vg = warp % C::VG, kt0 = warp / C::VG * (kTile / 16 / KS);
  const int key_0 = (2 * j) ^ ((j >> 1) & 1), key_1 = (2 * j + 1) ^ ((j >> 1) & 1);

  auto landed = [&](int tile, int code) {
    const int n = used + tile - t0;
    return mbar_wait(&full[n % kStages], (n / kStages) & 1, st, code);
  };
  for (int tile = t0; tile < t1; ++tile) {
    const int stage = (used + tile - t0) % kStages;
    const bool late = !landed(tile, STATUS_TIMEOUT_TMA_FULL);
    const uint32_t codes = smem_u32(smem + stage * C::kStage), params = codes + C::kCodes;
    const int r0 = row_of(tile);

    // ---- scores of this warp's 16 keys (this lane: mma rows i and i + 8) ----------------
    const uint32_t k_at = codes + (warp * 16 + key_i) * C::kRow + j * 8;
    const uint32_t p_at = params + (warp * 16 + key_i) * NG * 4;
    float s[NT][4];
    uint32_t m[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {  // keys i, i + 8 against groups 2j, 2j + 1, then + 8
      const uint32_t at = p_at + (h & 1) * 8 * NG * 4;
      const int g = 2 * j + (h >> 1) * 8;
      m[h] = __byte_perm(g < NG ? lds32(at + g * 4) : 0u, g + 1 < NG ? lds32(at + g * 4 + 4) : 0u, 0x7632);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 3; ++k) mma_bf16(s[nt], m[0], m[1], m[2], m[3], qm[k][nt][0], qm[k][nt][1]);
    }
#pragma unroll(PER_SM == 1 ? NG : 3)
    for (int g = 0; g < NG; ++g) {
      const uint2 wa = lds64(k_at + g * 32), wb = lds64(k_at + 8 * C::kRow + g * 32);
      const float sa = bf16_lo(lds32(p_at + g * 4)), sb = bf16_lo(lds32(p_at + (8 * NG + g) * 4));
      float d[NT][4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint4 q = *reinterpret_cast<const uint4*>(sqf + ((g * 4 + ks) * 32 + lane) * NT);
        const uint32_t xa = (ks < 2 ? wa.x : wa.y) >> ((ks & 1) * 8), xb = (ks < 2 ? wb.x : wb.y) >> ((ks & 1) * 8);
        const uint32_t a0 = xa & 0x000f000fu, a1 = xb & 0x000f000fu, a2 = xa & 0x00f000f0u, a3 = xb & 0x00f000f0u;
        if (ks == 0) {
          mma_f16_zero(d[0], a0, a1, a2, a3, q.x, q.y);
          mma_f16_zero(d[1], a0, a1, a2, a3, q.z, q.w);
        } else {
          mma_f16(d[0], a0, a1, a2, a3, q.x, q.y);
          mma_f16(d[1], a0, a1, a2, a3, q.z, q.w);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][c] = fmaf(d[nt][c], c < 2 ? sa : sb, s[nt][c]);
    }
    const bool masked = huge || !(r0 + kTile <= a.n_sink || (r0 >= see.lo_max && r0 + kTile <= see.hi_min));
    bool above = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[nt][c] *= rs[nt][c & 1];
    if (masked) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = r0 + warp * 16 + key_i + (c >> 1) * 8, q = nt * 8 + 2 * j + (c & 1);
          if (huge) s[nt][c] *= kKv4Lift;
          if (!(r < a.n_sink || (r >= slo[q] && r < shi[q]))) s[nt][c] = -INFINITY;
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[nt][c] = fmaxf(s[nt][c], s[nt][c + 2]);
        above |= top[nt][c] > limit[nt][c];
      }
    // also the barrier behind the previous tile's reads of the weights
    if (__syncthreads_or(above || late)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = top[nt][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          if (i == 0) smx[warp * kRows + nt * 8 + 2 * j + c] = x;
        }
      if (__syncthreads_or(late)) {
        dead = true;
        for (int k = tile; k < min(tile + kStages, t1); ++k) landed(k, STATUS_TIMEOUT_DRAIN);  // copies in flight
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) lsum[nt][0] = lsum[nt][1] = __int_as_float(0x7fffffff);
        break;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = nt * 8 + 2 * j + c;
          const float old = limit[nt][c] - kSlack;
          float x = old;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) x = fmaxf(x, smx[w * kRows + q]);
          limit[nt][c] = x + kSlack;
          // what was summed is in units of 2^ref, whatever limit - kSlack rounds to
          const float now = x == -INFINITY ? 0.f : x;
          const float alpha = old == -INFINITY ? 0.f : fast_exp2(ref[nt][c] - now);
          ref[nt][c] = now;
          lsum[nt][c] *= alpha;
          if (warp == 0 && i == 0) sal[q] = alpha;
#pragma unroll
          for (int mm = 0; mm < 4; ++mm) {
            acc[mm][nt][c] *= alpha;
            acc[mm][nt][c + 2] *= alpha;
          }
        }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) accm[nt] *= sal[nt * 8 + i];
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* o = sp + (nt * 8 + 2 * j + c) * kPRow + warp * 16 + i;   // by mma row, not by key
        const float x = fast_exp2(s[nt][c] - ref[nt][c]), y = fast_exp2(s[nt][c + 2] - ref[nt][c]);
        lsum[nt][c] += x + y;
        o[0] = x;
        o[8] = y;
      }
    __syncthreads();

    // ---- do the scales of the tile's values fit their power of two?  Lane: every 32nd of the warp's keys ----
    bool slow = false;
    {
      constexpr int kOwn = kTile / 32 / KS;   // keys per lane
      float sc[kOwn];
      bool used[kOwn], fit = true;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const int r = kt0 * 16 + lane + 32 * k;
        sc[k] = bf16_lo(lds32(params + (r * NG + vg) * 4));
        used[k] = !masked || r0 + r < a.n_sink || (r0 + r >= see.lo_min && r0 + r < see.hi_max);
        fit = fit && (!used[k] || kv4_in_range(sc[k], f));
      }
      if (!__all_sync(0xffffffffu, fit)) {
        uint32_t e = 0;
#pragma unroll
        for (int k = 0; k < kOwn; ++k)
          if (used[k] && sc[k] <= 3.4e38f) e = max(e, __float_as_uint(sc[k]) >> 23);
        e = __reduce_max_sync(0xffffffffu, e);
        if (e > 0) {  // largest scale in [2^3, 2^4); sums made before move along
          const float now = __uint_as_float(min(257u - e, 254u) << 23);
          const float move = f == 0.f ? 0.f : now / f;
          float most = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int mm = 0; mm < 4; ++mm) most = fmaxf(most, fabsf(acc[mm][nt][c]));
          if (__all_sync(0xffffffffu, most * move < kKv4Room)) {
            f = now;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int mm = 0; mm < 4; ++mm) acc[mm][nt][c] *= move;
          }
        }
        fit = true;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) fit = fit && (!used[k] || kv4_in_range(sc[k], f));
        slow = !__all_sync(0xffffffffu, fit);
      }
    }
    // ---- output: this warp's value dims over its keys of the tile ---------------------
#pragma unroll(PER_SM == 1 ? 4 : 1)
    for (int kt = kt0; kt < kt0 + kTile / 16 / KS; ++kt) {
      const uint32_t c0 = codes + (kt * 16 + key_0) * C::kRow + i * 4 + vg * 32;
      const uint32_t c1 = codes + (kt * 16 + key_1) * C::kRow + i * 4 + vg * 32;
      const uint32_t q0 = params + ((kt * 16 + key_0) * NG + vg) * 4, q1 = params + ((kt * 16 + key_1) * NG + vg) * 4;
      const uint32_t w0 = lds32(c0), w1 = lds32(c1), w8 = lds32(c0 + 8 * C::kRow), w9 = lds32(c1 + 8 * C::kRow);
      const uint32_t u0 = lds32(q0), u1 = lds32(q1), u8 = lds32(q0 + 8 * NG * 4), u9 = lds32(q1 + 8 * NG * 4);
      const float s0 = bf16_lo(u0), s1 = bf16_lo(u1), s8 = bf16_lo(u8), s9 = bf16_lo(u9);
      const float m0 = bf16_hi(u0), m1 = bf16_hi(u1), m8 = bf16_hi(u8), m9 = bf16_hi(u9);
      const float f0 = s0 * f, f1 = s1 * f, f8 = s8 * f, f9 = s9 * f;
      float x[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {  // weights of row i at mma rows 2j, 2j + 1 and + 8
        const float* p = sp + (nt * 8 + i) * kPRow + kt * 16 + 2 * j;
        const float2 p0 = *reinterpret_cast<const float2*>(p), p8 = *reinterpret_cast<const float2*>(p + 8);
        x[nt][0] = p0.x * f0;
        x[nt][1] = p0.y * f1;
        x[nt][2] = p8.x * f8;
        x[nt][3] = p8.y * f9;
        if (masked) {  // a key that a row does not see may hold anything
          auto times = [](float p, float x) { return p == 0.f ? 0.f : p * x; };
          if (p0.x == 0.f) x[nt][0] = 0.f;
          if (p0.y == 0.f) x[nt][1] = 0.f;
          if (p8.x == 0.f) x[nt][2] = 0.f;
          if (p8.y == 0.f) x[nt][3] = 0.f;
          accm[nt] += times(p0.x, m0) + times(p0.y, m1) + times(p8.x, m8) + times(p8.y, m9);
        } else {
          accm[nt] = fmaf(p0.x, m0, fmaf(p0.y, m1, fmaf(p8.x, m8, fmaf(p8.y, m9, accm[nt]))));
        }
      }
      const uint32_t l0 = __byte_perm(w0, w1, 0x5410), h0 = __byte_perm(w0, w1, 0x7632);
      const uint32_t l8 = __byte_perm(w8, w9, 0x5410), h8 = __byte_perm(w8, w9, 0x7632);
      uint32_t bw[NT][2];
      if (!slow) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bw[nt][0] = pack_f16x2(x[nt][0], x[nt][1]);
          bw[nt][1] = pack_f16x2(x[nt][2], x[nt][3]);
        }
        mma_values<0, NT>(acc[0], l0, h0, l8, h8, bw);
        mma_values<1, NT>(acc[1], l0, h0, l8, h8, bw);
        mma_values<2, NT>(acc[2], l0, h0, l8, h8, bw);
        mma_values<3, NT>(acc[3], l0, h0, l8, h8, bw);
      } else {
        float sums[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bw[nt][0] = pack_bf16x2(x[nt][0], x[nt][1]);
          bw[nt][1] = pack_bf16x2(x[nt][2], x[nt][3]);
          mma_bf16_zero(sums[nt], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, bw[nt][0], bw[nt][1]);
          // p 8 s: these weights meet n - 8
          accm[nt] = fmaf(f == 0.f ? 0.f : 8.f / f, (x[nt][0] + x[nt][1]) + (x[nt][2] + x[nt][3]), accm[nt]);
        }
        mma_values_bf16<0, NT>(acc[0], l0, h0, l8, h8, bw, sums);
        mma_values_bf16<1, NT>(acc[1], l0, h0, l8, h8, bw, sums);
        mma_values_bf16<2, NT>(acc[2], l0, h0, l8, h8, bw, sums);
        mma_values_bf16<3, NT>(acc[3], l0, h0, l8, h8, bw, sums);
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
  // sums of p m: lane (i, j) holds row i over the keys of j
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float m = accm[nt];
    m += __shfl_xor_sync(0xffffffffu, m, 1);
    m += __shfl_xor_sync(0xffffffffu, m, 2);
    if (j == 0) sp[warp * kRows + nt * 8 + i] = m;
  }
  __syncthreads();
  const bool alone = t0 == 0 && piece.step1 == piece.steps;
  float* part = a.part + (size_t)(2 * blockIdx.x + (t0 == 0)) * kRows * (V + 2);
  const float unit = f == 0.f ? 0.f : 1.f / f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int mm = 0; mm < 4; ++mm)
        acc[mm][nt][c] = fmaf(acc[mm][nt][c], unit * value_unit(mm), sp[warp * kRows + nt * 8 + 2 * j + (c & 1)]);
  if (KS == 2) {  // the stages' memory is free: the second warp of a pair hands over its sums
    float* to = reinterpret_cast<float*>(smem) + (warp % C::VG) * 32 * 32 + lane;
#pragma unroll
    for (int n = 0; n < 32; ++n)
      if (warp >= C::VG) to[n * 32] = acc[n >> 3][(n >> 2) & 1][n & 3];
    // ordinary stores to bytes that the next segment's bulk copies (another proxy) write: a barrier
    // alone does not order the two
    fence_proxy_async_smem();
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 32; ++n)
      if (warp < C::VG) acc[n >> 3][(n >> 2) & 1][n & 3] += to[n * 32];
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int q = nt * 8 + 2 * j + c;
      if (q >= nrows || warp >= C::VG) continue;
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) l += smx[w * kRows + q];
      const float inv = !alone ? 1.f : (l == 0.f ? 0.f : 1.f / l);
      const int d = vg * 64 + 8 * i;
      float o[8];
#pragma unroll
      for (int mm = 0; mm < 4; ++mm) {
        o[mm] = acc[mm][nt][c] * inv;
        o[4 + mm] = acc[mm][nt][c + 2] * inv;
      }
      if (!alone) {
        float4* p = reinterpret_cast<float4*>(part + q * V + d);
        p[0] = make_float4(o[0], o[1], o[2], o[3]);
        p[1] = make_float4(o[4], o[5], o[6], o[7]);
        if (warp == 0 && i == 0)
          *reinterpret_cast<float2*>(part + kRows * V + 2 * q) = make_float2(limit[nt][c] == -INFINITY ? -INFINITY : ref[nt][c], l);
      } else {
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + ((long long)b * R + row0 + q) * V + d) =
            make_uint4(kv4_pack2<TYPE>(o[0], o[1]), kv4_pack2<TYPE>(o[2], o[3]), kv4_pack2<TYPE>(o[4], o[5]),
                       kv4_pack2<TYPE>(o[6], o[7]));
      }
    }
  __syncthreads();  // the next segment refills shared memory
  }
}

template <int V, int TYPE, int PER_SM>
void launch_per_sm(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  auto kern = kv4_latent_kernel<V, TYPE, PER_SM>;
  constexpr int smem = LatentCfg<V>::kSmem;
  ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  kv4_launch(kern, dim3((unsigned)p.blocks), kWarps * 32, smem, s, a, kv4_line(a, p),
             reinterpret_cast<StatusBlock*>(status_ptr()));
}

// No more blocks than SMs: twice the registers, loops unrolled.  Measured, us one / two blocks per SM:
// 1 sequence of 128, 256, 8192 rows of 576 8.1 / 9.1, 11.8 / 13.2, 13.1 / 13.9; 16 of 1024 14.9 / 14.4,
// rows of 320 12.0 / 14.4.
template <int V, int TYPE>
void launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  p.blocks <= 148 ? launch_per_sm<V, TYPE, 1>(a, p, s) : launch_per_sm<V, TYPE, 2>(a, p, s);
}

}  // namespace

void kv4_latent_plan(const Kv4Attend& a, Kv4Plan& p) {
  p.kernel = 2;
  p.row_tiles = NT;
  p.row_blocks = (a.Tn * a.H + kRows - 1) / kRows;
  // One block per SM of up to two steps, or two blocks that share it.  Measured, us: 4 x 64 steps 17.3 /
  // 18.2, rows of 320 13.4 / 14.1; 16 x 33 steps 26.3 / 27.2, rows of 320 18.9 / 18.6; 64 x 33 71 / 64.
  const long long steps = kv4_plan_steps(a) * a.B * p.row_blocks;
  kv4_line_plan(a, p, steps <= 148 * 2 ? 148 : 148 * 2, 1);
}

void kv4_latent_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  if (a.type == KV4_F16)
    a.V == 512 ? launch<512, KV4_F16>(a, p, s) : launch<256, KV4_F16>(a, p, s);
  else
    a.V == 512 ? launch<512, KV4_BF16>(a, p, s) : launch<256, KV4_BF16>(a, p, s);
  if (p.restart > 0) kv4_combine(a, p, s);
}

}  // namespace omni
