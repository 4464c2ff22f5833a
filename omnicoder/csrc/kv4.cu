// 4-bit key / value cache (sm_100a): rows quantised as they are written, read
// back, and attended over.
//
//   codes  [B, Hk, L, W / 2]     byte i of a row: dim 2i (low nibble), 2i + 1
//   params [B, Hk, L, W / g, 2]  bf16 (scale s, minimum m) per group of g dims
//   value  x = n * s + m, n = 0 .. 15
//
// Position p of a sequence lies in row offset + p.  In the attention, rows
// [0, n_sink) are compressed memory that every query sees, and query (b, t)
// sees the positions p < kv_len[b], p <= q_pos[b, t] and, with a window,
// p > q_pos[b, t] - window.
#include <algorithm>

#include "kv4_device.cuh"

namespace omni {

namespace {

using bf16 = __nv_bfloat16;

constexpr float kMinScale = 7.52316384526264e-37f;  // 2^-120

// ---------------------------------------------------------------------------
// Sixteen consecutive values of one type <-> fp32
// ---------------------------------------------------------------------------
constexpr int kPiece = 16;

// Ordinary loads: the read-only path is for memory that nobody writes while the kernel lives, and this one
// is alive before its predecessor has written the rows.
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
  *reinterpret_cast<uint4*>(w + 4) = *(reinterpret_cast<const uint4*>(p) + 1);
}
// Rows to read into are allocated by the call and start on 32-byte boundaries.
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Words of sixteen values, and the values.
template <int TYPE>
__device__ __forceinline__ void load_words(const void* base, long long i, uint32_t* w) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(base) + i * (TYPE == KV4_F32 ? 4 : 2);
#pragma unroll
  for (int k = 0; k < (TYPE == KV4_F32 ? 2 : 1); ++k) load32(p + 32 * k, w + 8 * k);
}
template <int TYPE>
__device__ __forceinline__ void words_to_floats(const uint32_t* w, float* x) {
#pragma unroll
  for (int k = 0; k < (TYPE == KV4_F32 ? 16 : 8); ++k) {
    if (TYPE == KV4_F32) {
      x[k] = __uint_as_float(w[k]);
    } else if (TYPE == KV4_BF16) {
      x[2 * k] = bf16_lo(w[k]);
      x[2 * k + 1] = bf16_hi(w[k]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
}

template <int TYPE>
__device__ __forceinline__ void store_piece(void* base, long long i, const float* x) {
  constexpr int kWords = TYPE == KV4_F32 ? 16 : 8;
  uint8_t* p = reinterpret_cast<uint8_t*>(base) + i * (TYPE == KV4_F32 ? 4 : 2);
  uint32_t w[kWords];
#pragma unroll
  for (int k = 0; k < kWords; ++k)
    w[k] = TYPE == KV4_F32 ? __float_as_uint(x[k]) : kv4_pack2<TYPE>(x[2 * k], x[2 * k + 1]);
#pragma unroll
  for (int k = 0; k < kWords / 8; ++k) store32(p + 32 * k, w + 8 * k);
}

template <int TYPE>
__device__ __forceinline__ void store1(void* base, long long i, float x) {
  if (TYPE == KV4_BF16)
    reinterpret_cast<bf16*>(base)[i] = __float2bfloat16_rn(x);
  else
    reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
}

// ---------------------------------------------------------------------------
// Append and read back.  A thread owns sixteen dims (writing groups of 32 and 64:
// 32 dims) of up to kPasses rows; the threads of a group of g dims are neighbours in
// a warp, and a block's rows run over the tokens of one head and then the next, so
// that a warp writes whole sectors of the codes.  Measured: 8 x 8192 rows of 576
// bf16 values written in 24 us (4.1 TB/s) and read back in 18.5 us (5.2 TB/s); the
// write is bound by its instructions, the read by memory.  Single tokens of 64
// sequences: 2.5 and 1.5 us.  Writing 16 dims per thread took 29 us: 312 instead of
// 215 instructions per 16 values, for addresses, minimum and maximum.
// ---------------------------------------------------------------------------
constexpr int kIoThreads = 256;
constexpr int kPasses = 4;

struct IoGrid {
  Kv4Div pieces, tokens;       // threads of a row; T
  int rows_per_pass, passes;
  int total;                   // rows Hk * T of a sequence
  int groups, lanes_shift;     // groups of a row; 2^lanes_shift threads hold one
};

struct IoRow {
  int h, t;
  long long row;  // of the cache; -1: nothing to do
};

__device__ __forceinline__ IoRow io_row(const Kv4IO& a, const IoGrid& g, int r) {
  IoRow x;
  x.h = g.tokens.of(r);
  x.t = r - x.h * a.T;
  x.row = a.row_offset + kv4_load_pos(a.pos, a.pos64, (long long)blockIdx.y * a.T + x.t);
  if (x.row < 0 || x.row >= a.L) x.row = -1;
  return x;
}

__device__ __forceinline__ uint8_t* io_codes(const Kv4IO& a, const Kv4Cache& c, const IoRow& x, int piece) {
  return c.codes + blockIdx.y * c.c_b + x.h * c.c_h + x.row * (a.W / 2) + piece * 8;
}
__device__ __forceinline__ uint32_t* io_params(const Kv4Cache& c, const IoGrid& g, const IoRow& x, int piece) {
  return reinterpret_cast<uint32_t*>(c.params + blockIdx.y * c.p_b + x.h * c.p_h + (x.row * g.groups + (piece >> g.lanes_shift)) * 4);
}

// Round (x - m) / s, .. < 15.5, decided as if the quotient were exact: d + e = x - m exactly,
// r = d - n s exactly for n next to it (n s has at most 12 significant bits), and r + e is compared
// with half a step; ties to even.
__device__ __forceinline__ uint32_t kv4_code_exact(float x, float m, float s, float inv) {
  const float d = x - m, back = d - x, half = 0.5f * s;
  const float e = (x - (d - back)) - (m + back);
  float n = rintf(d * inv);
  const float r = fmaf(-n, s, d);
  const bool odd = ((int)n & 1) != 0;
  if (r > half || (r == half && (e > 0.f || (e == 0.f && odd)))) n += 1.f;
  else if (r < -half || (r == -half && (e < 0.f || (e == 0.f && odd)))) n -= 1.f;
  return (uint32_t)fminf(fmaxf(n, 0.f), 15.f);
}

// Two fp32 numbers in one instruction.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
  return x;
}
__device__ __forceinline__ float2 split2(uint64_t x) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(x));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t x;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(a), "l"(b), "l"(c));
  return x;
}

// Sixteen codes from q', the quotient (x - m) / s with one residual correction (Markstein, 1990):
// within 2^-20 of it, and exactly k + 1/2 where the quotient is that and x - m is exact.  Adding
// 2^23 rounds it, ties to even.  That decides as an exact quotient would
//   - for a bf16 value that is 0 or at least 2^-16 of the range R, where m is too: x, m and s are then
//     multiples of 2^-24 R, x - m is exact, and a quotient that is not halfway between two codes is
//     2^-24 R / s > 2^-21 or more away, half a unit of the quotient's last place;
//   - for any value whose quotient is not within 2^-16 of halfway (kv4_near_border, whose quotient
//     lacks the correction: within 2^-18).
// Other values are rounded again (kv4_code_exact).
// The two words of codes go side by side, dims i and i + 8; four codes join as a number below 2^16.
template <int TYPE>
__device__ __forceinline__ uint64_t kv4_codes16(const float* x, float m, float s, float inv) {
  const uint64_t m2 = pair2(-m, -m), s2 = pair2(-s, -s), inv2 = pair2(inv, inv), sixteen = pair2(16.f, 16.f);
  const uint64_t up = pair2(8388608.f, 8388608.f), down = pair2(-8388608.f, -8388608.f);
  uint64_t half[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint64_t acc = 0;
#pragma unroll
    for (int i = 4 * h + 3; i >= 4 * h; --i) {
      const uint64_t d = add2(pair2(x[i], x[i + 8]), m2), q = mul2(d, inv2);
      uint64_t q1 = fma2(fma2(q, s2, d), inv2, q);
      if (TYPE != KV4_BF16) {  // the minimum was rounded to bf16
        const float2 v = split2(q1);
        q1 = pair2(fminf(fmaxf(v.x, 0.f), 15.f), fminf(fmaxf(v.y, 0.f), 15.f));
      }
      const uint64_t n = add2(add2(q1, up), down);
      acc = i == 4 * h + 3 ? n : fma2(acc, sixteen, n);
    }
    half[h] = add2(acc, up);
  }
  const float2 lo = split2(half[0]), hi = split2(half[1]);
  const uint32_t w0 = __byte_perm(__float_as_uint(lo.x), __float_as_uint(hi.x), 0x5410);
  const uint32_t w1 = __byte_perm(__float_as_uint(lo.y), __float_as_uint(hi.y), 0x5410);
  return (uint64_t)w0 | ((uint64_t)w1 << 32);
}

// Is the quotient within 2^-16 of halfway between two codes?
__device__ __forceinline__ bool kv4_near_border(float x, float m, float inv) {
  const float t = fminf(fmaxf((x - m) * inv, 0.f), 15.f);
  return fabsf(t - ((t + 8388608.f) - 8388608.f)) > 0.4999847412109375f;
}

template <int TYPE, int PIECES>
__global__ void __launch_bounds__(kIoThreads) kv4_write_kernel(const Kv4IO a, const IoGrid g) {
  wait_for_previous_grid();
  launch_dependents();
  constexpr int kWords = TYPE == KV4_F32 ? 16 : 8;   // of a piece
  const int b = blockIdx.y, r_in = g.pieces.of(threadIdx.x), piece = threadIdx.x - r_in * g.pieces.d;
  const Kv4Cache& c = a.cache[blockIdx.z];
  const Kv4Rows& src = a.rows[blockIdx.z];
  const int lanes = 1 << g.lanes_shift;  // 1 or 2 neighbouring threads hold a group
  const int first = blockIdx.x * (g.rows_per_pass * g.passes) + r_in;
  const bool idle = r_in >= g.rows_per_pass;
#pragma unroll 1
  for (int k = 0; k < g.passes; ++k) {
    const int r = first + k * g.rows_per_pass;
    uint32_t w[PIECES * kWords];
    const IoRow row = io_row(a, g, min(r, g.total - 1));   // threads behind the last row repeat it and write nothing
    const long long at = b * src.x_b + row.t * src.x_t + row.h * src.x_h + piece * (PIECES * kPiece);
#pragma unroll
    for (int n = 0; n < PIECES; ++n) load_words<TYPE>(src.x, at + n * kPiece, w + n * kWords);
    float lo, hi, probe, least = 0.f;  // probe: NaN behind a NaN or an infinity; least |x|
    if (TYPE == KV4_BF16) {
      const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(w);
      const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
      __nv_bfloat162 l = v[0], h = v[0], p = __hmul2(v[0], zero), q = __habs2(v[0]);
#pragma unroll
      for (int i = 1; i < PIECES * kWords; ++i) {
        l = __hmin2(l, v[i]);
        h = __hmax2(h, v[i]);
        p = __hfma2(v[i], zero, p);
        q = __hmin2(q, __habs2(v[i]));
      }
      lo = fminf(__low2float(l), __high2float(l));
      hi = fmaxf(__low2float(h), __high2float(h));
      probe = __low2float(p) + __high2float(p);
      least = fminf(__low2float(q), __high2float(q));
    } else {
      lo = INFINITY;
      hi = -INFINITY;
      probe = 0.f;
#pragma unroll
      for (int n = 0; n < PIECES; ++n) {
        float x[kPiece];
        words_to_floats<TYPE>(w + n * kWords, x);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          lo = fminf(lo, x[i]);
          hi = fmaxf(hi, x[i]);
          probe = fmaf(x[i], 0.f, probe);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < PIECES; o <<= 1) {  // groups of 16 are a thread's own
      const float l2 = __shfl_xor_sync(0xffffffffu, lo, o), h2 = __shfl_xor_sync(0xffffffffu, hi, o);
      const float p2 = __shfl_xor_sync(0xffffffffu, probe, o);
      if (o < lanes) {
        lo = fminf(lo, l2);
        hi = fmaxf(hi, h2);
        probe += p2;
      }
    }
    // m is exact for bf16 rows; the scale is taken from the rounded minimum, as a product with
    // fp32(1 / 15): where the quotient by 15 would lie halfway between two bf16 numbers (0.05 % of random
    // bf16 ranges) that decides which of the two is stored.  The codes refer to the stored one.
    const bf16 mb = __float2bfloat16_rn(lo);
    const float m = __bfloat162float(mb);
    const float range = hi - m;
    bf16 sb = __float2bfloat16_rn(range * (1.f / 15.f));
    float s = __bfloat162float(sb);
    const bool bad = probe != 0.f || !(fabsf(m) <= 3.3895314e38f) || !(s <= 3.3895314e38f);
    if (!(s >= kMinScale)) {
      s = 0.f;
      sb = __float2bfloat16_rn(0.f);
    }
    uint64_t code[PIECES];
#pragma unroll
    for (int n = 0; n < PIECES; ++n) code[n] = 0;
    if (!bad && s > 0.f) {
      float inv;  // within 2^-23: candidates and residual corrections need no more
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
      // the values to look at: all, or bf16 ones below 2^-16 of the range
      const float small = range * 1.52587890625e-5f;
      const float limit = TYPE != KV4_BF16 || s < 1e-27f || (m != 0.f && fabsf(m) < small) ? INFINITY : small;
      uint32_t again = 0;
#pragma unroll
      for (int n = 0; n < PIECES; ++n) {
        float x[kPiece];
        words_to_floats<TYPE>(w + n * kWords, x);
        if (TYPE != KV4_BF16 || least < limit) {
#pragma unroll
          for (int i = 0; i < kPiece; ++i)
            if (fabsf(x[i]) < limit && kv4_near_border(x[i], m, inv)) again |= 1u << (n * kPiece + i);
        }
        code[n] = kv4_codes16<TYPE>(x, m, s, inv);
      }
      if (s < 1e-27f) again = 0xffffffffu >> (32 - PIECES * kPiece);
      while (again != 0) {  // few values of few threads: read again
        const int i = __ffs(again) - 1, shift = 4 * (i & 15);
        again &= again - 1;
        const uint64_t exact = (uint64_t)kv4_code_exact(kv4_load1<TYPE>(src.x, at + i), m, s, inv) << shift;
        const uint64_t keep = ~(15ull << shift);
        if (PIECES == 1 || i < kPiece) code[0] = (code[0] & keep) | exact;
        else code[PIECES - 1] = (code[PIECES - 1] & keep) | exact;
      }
    }
    if (row.row < 0 || idle || r >= g.total) continue;
    uint8_t* to = io_codes(a, c, row, piece * PIECES);
    if (PIECES == 2)
      *reinterpret_cast<ulonglong2*>(to) = make_ulonglong2(code[0], code[PIECES - 1]);
    else
      *reinterpret_cast<uint64_t*>(to) = code[0];
    if ((piece & (lanes - 1)) == 0) {
      const uint32_t word = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(mb) << 16);
      *io_params(c, g, row, piece) = bad ? 0x7fc07fc0u : word;
    }
  }
}

template <int TYPE>
__global__ void __launch_bounds__(kIoThreads) kv4_read_kernel(const Kv4IO a, const IoGrid g) {
  wait_for_previous_grid();
  launch_dependents();
  const int b = blockIdx.y, r_in = g.pieces.of(threadIdx.x), piece = threadIdx.x - r_in * g.pieces.d;
  if (r_in >= g.rows_per_pass) return;
  const Kv4Cache& c = a.cache[blockIdx.z];
  const Kv4Rows& dst = a.rows[blockIdx.z];
  const int first = blockIdx.x * (g.rows_per_pass * g.passes) + r_in;
  uint2 code[kPasses];
  uint32_t word[kPasses];
  IoRow row[kPasses];
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int r = first + k * g.rows_per_pass;
    code[k] = make_uint2(0, 0);  // rows outside the cache read as zeros
    word[k] = 0;
    if (k < g.passes && r < g.total) {
      row[k] = io_row(a, g, r);
      if (row[k].row >= 0) {
        code[k] = *reinterpret_cast<const uint2*>(io_codes(a, c, row[k], piece));
        word[k] = *io_params(c, g, row[k], piece);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    if (k >= g.passes || first + k * g.rows_per_pass >= g.total) break;
    const long long at = b * dst.x_b + row[k].t * dst.x_t + row[k].h * dst.x_h + piece * kPiece;
    if (TYPE == KV4_BF16) {
      // n s + m in one bf16 multiply-add, rounded once; nibbles 0..3 of both halves of a code word as
      // 128 + n give the dims e and e + 4
      const uint32_t s2 = __byte_perm(word[k], word[k], 0x1010), m2 = __byte_perm(word[k], word[k], 0x3232);
      uint32_t v[8];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t u = (((w ? code[k].y : code[k].x) >> (4 * e)) & 0x000f000fu) | 0x43004300u;
          const __nv_bfloat162 n = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(128.f));
          const __nv_bfloat162 x = __hfma2(n, *reinterpret_cast<const __nv_bfloat162*>(&s2), *reinterpret_cast<const __nv_bfloat162*>(&m2));
          v[4 * w + e] = *reinterpret_cast<const uint32_t*>(&x);
        }
      uint32_t o[8];
#pragma unroll
      for (int w = 0; w < 8; w += 4) {  // (0, 4), (1, 5), .. -> (0, 1), (2, 3), (4, 5), (6, 7)
        o[w] = __byte_perm(v[w], v[w + 1], 0x5410);
        o[w + 1] = __byte_perm(v[w + 2], v[w + 3], 0x5410);
        o[w + 2] = __byte_perm(v[w], v[w + 1], 0x7632);
        o[w + 3] = __byte_perm(v[w + 2], v[w + 3], 0x7632);
      }
      store32(reinterpret_cast<uint16_t*>(dst.x) + at, o);
    } else {
      const float s = bf16_lo(word[k]), m = bf16_hi(word[k]);
      float x[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        // 2^23 + n as bits, less 2^23: the code as a float
        const uint32_t n = ((i < 8 ? code[k].x : code[k].y) >> (4 * (i & 7))) & 15u;
        x[i] = fmaf(__uint_as_float(n | 0x4b000000u) - 8388608.f, s, m);
      }
      store_piece<TYPE>(dst.x, at, x);
    }
  }
}

// Enough blocks first, then several rows per thread.  Measured, 1, 2 and up to 4 rows, us written /
// read back: 8 x 8192 rows of 576 in bf16 27.6 / 23.4, 25.8 / 19.8, 26.0 / 18.5, in fp32 74 / 35, 61 / 31,
// 54 / 31; 3 x 4001 x 8 heads of 128 and a token of 64 sequences within 4 %.
dim3 io_grid(const Kv4IO& a, int dims, IoGrid* g) {
  g->pieces = Kv4Div(a.W / dims);
  g->tokens = Kv4Div(a.T);
  g->rows_per_pass = kIoThreads / g->pieces.d;
  g->total = a.T * a.Hk;
  g->groups = a.W / a.group;
  g->lanes_shift = a.group == 4 * dims ? 2 : a.group == 2 * dims ? 1 : 0;
  const long long blocks1 = (g->total + g->rows_per_pass - 1) / g->rows_per_pass;
  g->passes = (int)std::min<long long>(kPasses, std::max<long long>(1, blocks1 * a.B * a.count / (148 * 4)));
  const long long per_block = (long long)g->rows_per_pass * g->passes;
  return dim3((unsigned)((g->total + per_block - 1) / per_block), (unsigned)a.B, (unsigned)a.count);
}

// ---------------------------------------------------------------------------
// Attention, one block per query row: any row width and group.  Eight warps
// take 32-row tiles in turn; a lane owns a row for the scores and every 32nd
// value dim for the output.  Statistics and sums in fp32.
// ---------------------------------------------------------------------------
constexpr int kRowWarps = 8;
constexpr int kRowDims = 32;  // value dims of a lane: V <= 1024

template <int TYPE>
__global__ void __launch_bounds__(kRowWarps * 32) kv4_row_kernel(const Kv4Attend a) {
  wait_for_previous_grid();
  launch_dependents();
  extern __shared__ float sm[];
  float* sq = sm;                              // [W]
  float* so = sq + a.W;                        // [kRowWarps][V]
  float* sml = so + kRowWarps * a.V;           // [kRowWarps][2]
  const int row = blockIdx.x, b = blockIdx.y, lane = lane_id(), warp = warp_id();
  const int t = row / a.H, h = row % a.H, hk = h / (a.H / a.Hk);
  const long long qi = ((long long)b * a.Tn * a.H + row) * a.W;
  for (int i = threadIdx.x; i < a.W; i += kRowWarps * 32) sq[i] = kv4_load1<TYPE>(a.q, qi + i) * a.scale * kKv4Log2e;
  __syncthreads();
  const Kv4Seen seen = kv4_seen(a, b, t);
  const uint8_t* kc = a.k.codes + b * a.k.c_b + hk * a.k.c_h;
  const uint8_t* kp = a.k.params + b * a.k.p_b + hk * a.k.p_h;
  const bool latent = a.v.codes == nullptr;
  const uint8_t* vc = latent ? kc : a.v.codes + b * a.v.c_b + hk * a.v.c_h;
  const uint8_t* vp = latent ? kp : a.v.params + b * a.v.p_b + hk * a.v.p_h;
  const int groups = a.W / a.group, half = a.W / 2;
  float o[kRowDims];
#pragma unroll
  for (int i = 0; i < kRowDims; ++i) o[i] = 0.f;
  float mx = -INFINITY, sum = 0.f;
  Kv4Piece piece;
  kv4_tiles<32>(a, seen, &piece);
  for (int tile = warp; tile < piece.tiles; tile += kRowWarps) {
    const int r0 = (tile < piece.sink_tiles ? tile : piece.first + tile - piece.sink_tiles) * 32;
    const int r = r0 + lane;
    const bool vis = r < a.n_sink || (r >= seen.lo && r < seen.hi);
    const uint32_t seen_rows = __ballot_sync(0xffffffffu, vis);
    float s = -INFINITY;
    if (vis) {
      s = 0.f;
      for (int g = 0; g < groups; ++g) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(kp + ((long long)r * groups + g) * 4);
        const float sc = bf16_lo(word), mn = bf16_hi(word);
        for (int i = 0; i < a.group / 8; ++i) {
          const int d = g * a.group + i * 8;
          const uint32_t code = *reinterpret_cast<const uint32_t*>(kc + (long long)r * half + d / 2);
#pragma unroll
          for (int e = 0; e < 8; ++e) s = fmaf(sq[d + e], fmaf((float)((code >> (4 * e)) & 15u), sc, mn), s);
        }
      }
    }
    const float top = fmaxf(mx, warp_max(s));
    const float ref = top == -INFINITY ? 0.f : top;
    const float alpha = fast_exp2(mx - ref);
    const float p = fast_exp2(s - ref);
    sum = sum * alpha + p;
    mx = top;
#pragma unroll
    for (int i = 0; i < kRowDims; ++i) o[i] *= alpha;
    for (int k = 0; k < 32; ++k) {
      const float pk = __shfl_sync(0xffffffffu, p, k);
      if (!(seen_rows >> k & 1)) continue;  // whatever they hold
      const long long rk = r0 + k;
#pragma unroll
      for (int i = 0; i < kRowDims; ++i) {
        const int d = lane + 32 * i;
        if (d < a.V) {
          const uint32_t word = *reinterpret_cast<const uint32_t*>(vp + (rk * groups + d / a.group) * 4);
          const int n = (vc[rk * half + d / 2] >> (4 * (d & 1))) & 15;
          o[i] = fmaf(pk, fmaf((float)n, bf16_lo(word), bf16_hi(word)), o[i]);
        }
      }
    }
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int i = 0; i < kRowDims; ++i)
    if (lane + 32 * i < a.V) so[warp * a.V + lane + 32 * i] = o[i];
  if (lane == 0) {
    sml[2 * warp] = mx;
    sml[2 * warp + 1] = sum;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.f, w[kRowWarps];
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) top = fmaxf(top, sml[2 * i]);
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) {
    w[i] = fast_exp2(sml[2 * i] - (top == -INFINITY ? 0.f : top));
    total += w[i] * sml[2 * i + 1];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;  // a row that sees nothing gives zeros
  for (int d = threadIdx.x; d < a.V; d += kRowWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) x = fmaf(w[i], so[i * a.V + d], x);
    store1<TYPE>(a.out, ((long long)b * a.Tn * a.H + row) * a.V + d, x * inv);
  }
}

template <int TYPE>
void launch_rows(const Kv4Attend& a, cudaStream_t s) {
  auto kern = kv4_row_kernel<TYPE>;
  const int smem = (a.W + kRowWarps * (a.V + 2)) * 4;
  ensure_smem_attr(reinterpret_cast<const void*>(kern), smem);
  kv4_launch(kern, dim3((unsigned)(a.Tn * a.H), (unsigned)a.B), kRowWarps * 32, smem, s, a);
}

}  // namespace

void kv4_write(const Kv4IO& a, cudaStream_t s) {
  IoGrid g{Kv4Div(1), Kv4Div(1), 0, 0, 0, 0, 0};
  const bool two = a.group >= 32;
  const dim3 grid = io_grid(a, two ? 32 : 16, &g);
  auto go = [&](auto one_piece, auto two_pieces) { kv4_launch(two ? two_pieces : one_piece, grid, kIoThreads, 0, s, a, g); };
  if (a.type == KV4_F32) go(kv4_write_kernel<KV4_F32, 1>, kv4_write_kernel<KV4_F32, 2>);
  else if (a.type == KV4_F16) go(kv4_write_kernel<KV4_F16, 1>, kv4_write_kernel<KV4_F16, 2>);
  else go(kv4_write_kernel<KV4_BF16, 1>, kv4_write_kernel<KV4_BF16, 2>);
}

void kv4_read(const Kv4IO& a, cudaStream_t s) {
  IoGrid g{Kv4Div(1), Kv4Div(1), 0, 0, 0, 0, 0};
  const dim3 grid = io_grid(a, kPiece, &g);
  if (a.type == KV4_F32) kv4_launch(kv4_read_kernel<KV4_F32>, grid, kIoThreads, 0, s, a, g);
  else if (a.type == KV4_F16) kv4_launch(kv4_read_kernel<KV4_F16>, grid, kIoThreads, 0, s, a, g);
  else kv4_launch(kv4_read_kernel<KV4_BF16>, grid, kIoThreads, 0, s, a, g);
}

// The tensor-core kernels take heads of 64 and 128 dims and latents of 512 + 64 and 256 + 64 (the dense,
// draft, long-context and 24-layer presets); any other width goes to one block per query row, with a
// sequence's keys in one block: heads of 32 (tiny_moe) and latents of 160 + 64 and 128 + 48 (the mobile
// presets).  There the int8 cache's kernel, which splits them, can be faster; us int4 / int8, 4096 rows, 8
// query heads: 8 heads of 32, 1 sequence 498 / 221, 16 535 / 3317; latent of 128 + 48, 1 sequence 722 / 73, 16
// 754 / 415; latent of 160 + 64 775 (int8 does not take it).  Measured, us tensor / row kernel (cold): 1 sequence of 32 rows, 2 heads of 64 9.1 / 47; 8 x 130
// rows, 8 heads of 128 11 / 66; 1 x 130 latent rows, 16 heads 20 / 100; 64 x 8192, 48 on 8 heads of 128
// 147 / 19979.
Kv4Plan kv4_plan(const Kv4Attend& a) {
  Kv4Plan p{};
  if (a.v.codes != nullptr && a.group == 64 && (a.W == 64 || a.W == 128)) kv4_heads_plan(a, p);
  if (a.v.codes == nullptr && a.group == 64 && a.W == a.V + 64 && (a.V == 256 || a.V == 512)) kv4_latent_plan(a, p);
  return p;
}

void kv4_attend(const Kv4Attend& a, const Kv4Plan& plan, cudaStream_t s) {
  if (plan.kernel == 1) kv4_heads_launch(a, plan, s);
  else if (plan.kernel == 2) kv4_latent_launch(a, plan, s);
  else if (a.type == KV4_F16) launch_rows<KV4_F16>(a, s);
  else launch_rows<KV4_BF16>(a, s);
}

}  // namespace omni
