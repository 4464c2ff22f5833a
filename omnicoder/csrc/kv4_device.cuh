// Device helpers shared by the attention kernels over a 4-bit cache.
#pragma once
#include "common.cuh"
#include "kv4.h"

namespace omni {

constexpr float kKv4Log2e = 1.4426950408889634f;

__device__ __forceinline__ long long kv4_load_pos(const void* p, bool is64, long long i) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}
// Positions of the attention, beyond any cache row (L < 2^30) cut off.
__device__ __forceinline__ int kv4_load_near(const void* p, bool is64, long long i) {
  if (!is64) return min(max(reinterpret_cast<const int*>(p)[i], -(1 << 30)), 1 << 30);
  return (int)min(max(reinterpret_cast<const long long*>(p)[i], -(1ll << 30)), 1ll << 30);
}

template <int TYPE>
__device__ __forceinline__ float kv4_load1(const void* base, long long i) {
  if (TYPE == KV4_F32) return reinterpret_cast<const float*>(base)[i];
  if (TYPE == KV4_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(reinterpret_cast<const __half*>(base)[i]);
}

template <int TYPE>
__device__ __forceinline__ uint32_t kv4_pack2(float a, float b) {
  if (TYPE == KV4_BF16) return pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Rows that a query sees besides the memory rows [0, n_sink): [lo, hi).
struct Kv4Seen {
  int lo, hi;
};

__device__ __forceinline__ Kv4Seen kv4_seen(const Kv4Attend& a, int b, int t) {
  const int len = kv4_load_near(a.kv_len, a.len64, b);
  const int qp = kv4_load_near(a.q_pos, a.pos64, (long long)b * a.Tn + t), room = a.L - a.sink_rows;
  const int end = max(min(min(len, qp + 1), room), 0);
  const int first = a.window > 0 ? max(qp - a.window + 1, 0) : 0;
  Kv4Seen s;
  s.lo = a.sink_rows + min(first, room);
  s.hi = max(a.sink_rows + end, s.lo);
  return s;
}

// ---- tensor-core tiles on registers ---------------------------------------------
// Codes become matrix operands in registers, straight from the 4-bit tile in
// shared memory.  tcgen05 operands would have to be written back to shared or
// tensor memory first: as 16-bit tiles four times the bytes of the codes; as 8-bit
// ones (a nibble in a byte is the e4m3 number n 2^-9) twice, with the queries and the
// weights each split into two or three such numbers.  Neither was built.
//
// The two low nibbles of a 16-bit half, masked out, are the fp16 subnormals n 2^-24
// and 16 n 2^-24, which the fp16 product takes exactly: two codes per AND.  (The
// 8-bit float product of this family, mma.sync, is emulated here: 29 cycles against 8
// for the fp16 one.)
__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = A B
__device__ __forceinline__ void mma_f16_zero(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_zero(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit elements spread over the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Nibble MM of both 16-bit halves as the bf16 pair (16 + n, 16 + n'): bits 3..6 of a
// bf16 mantissa at exponent 2^4 count in ones.
template <int MM>
__device__ __forceinline__ uint32_t nibbles_bf16(uint32_t x) {
  const uint32_t y = MM == 0 ? x << 3 : x >> (MM == 0 ? 0 : 4 * MM - 3);
  return (y & 0x00780078u) | 0x41804180u;
}

// Weights meet value codes as x = p s f in fp16, f a power of two for which every scale s of the
// keys at hand has s f in [2^-8, 2^6], or 0: then x < 2^14 (p < 2^8), its rounding is 2^-11 of it
// down to 2^-14 and 2^-25 below, 2^-17 of a row's largest weight.  Where the scales of
// neighbouring keys lie further apart, x is rounded to bf16 instead (slow).
// Smaller scales raise f only as far as the sums in it leave room for.
constexpr float kKv4Low = 0.00390625f, kKv4High = 64.f, kKv4Room = 1.2676506e30f;  // 2^100

// f = 0: none yet.  A NaN or an infinity fits any f: it stays one, for the queries that see it.
__device__ __forceinline__ bool kv4_in_range(float s, float f) {
  return !(s * f < kKv4Low && s > 0.f) && !(s * f > kKv4High && s <= 3.4e38f);
}

// acc[mm][nt] += 16 value dims x 16 keys (nibble mm of a lane's paired words: dims mm in the low, 4 + mm
// in the high halves of its eight) times the weights w of row tile nt.  The sums are in units of
// 2^-24, 2^-20 for odd mm.
template <int MM, int NT>
__device__ __forceinline__ void mma_values(float (*acc)[4], uint32_t l0, uint32_t h0, uint32_t l8, uint32_t h8,
                                           const uint32_t (*w)[2]) {
  constexpr uint32_t kMask = MM & 1 ? 0x00f000f0u : 0x000f000fu;
  const uint32_t a0 = (l0 >> (MM & 2) * 4) & kMask, a1 = (h0 >> (MM & 2) * 4) & kMask;
  const uint32_t a2 = (l8 >> (MM & 2) * 4) & kMask, a3 = (h8 >> (MM & 2) * 4) & kMask;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt], a0, a1, a2, a3, w[nt][0], w[nt][1]);
}

// The same for bf16 weights, whose sum sums[nt][] over the keys is known, and codes n - 8: the
// rounding of a weight then counts for eight steps at most.
template <int MM, int NT>
__device__ __forceinline__ void mma_values_bf16(float (*acc)[4], uint32_t l0, uint32_t h0, uint32_t l8, uint32_t h8,
                                                const uint32_t (*w)[2], const float (*sums)[4]) {
  const uint32_t a0 = nibbles_bf16<MM>(l0), a1 = nibbles_bf16<MM>(h0), a2 = nibbles_bf16<MM>(l8), a3 = nibbles_bf16<MM>(h8);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float d[4];
    mma_bf16_zero(d, a0, a1, a2, a3, w[nt][0], w[nt][1]);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc[nt][c] = fmaf(fmaf(-24.f, sums[nt][c & 1], d[c]), MM & 1 ? 9.5367431640625e-7f : 5.9604644775390625e-8f, acc[nt][c]);
  }
}
__device__ __forceinline__ float value_unit(int mm) { return mm & 1 ? 1048576.f : 16777216.f; }

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void kv4_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void kv4_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void kv4_cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// Query rows enter the fp16 product with codes as q 2^e, the largest |q| of the
// row in [2^14, 2^15).  What fp16 rounds off is at most 2^-39 of it in even dims and, as odd
// ones are stored a sixteenth as large (query_pairs), 2^-35 in odd ones.
// `unscale` is 2^-e; the codes' 2^-24 is undone separately (kKv4Codes).
constexpr float kKv4Codes = 16777216.f;
__device__ __forceinline__ float q_normaliser(float amax, float* unscale) {
  const uint32_t e = min(max((__float_as_uint(amax) >> 23) & 255u, 40u), 254u);
  *unscale = __uint_as_float((e - 14u) << 23);  // 2^(e - 127 - 14)
  return __uint_as_float((268u - e) << 23);     // 2^(14 - (e - 127))
}

// Factor of a row's raw scores: the row's unscale, the softmax scale, log2 e and kKv4Codes.  That can
// leave fp32 where the scores do not (|q| scale from 2^117 on, small keys), so rows are prepared without
// kKv4Codes, and where one of a block's is kKv4Huge or more, all are multiplied in two steps: here by
// kKv4Codes / kKv4Lift and, in the loop's branch for tiles that some row does not see whole, by kKv4Lift.
constexpr float kKv4Huge = 1.2676506e30f, kKv4Lift = 4294967296.f;  // 2^100, 2^32
template <int N>
__device__ __forceinline__ bool kv4_score_factors(float (*rs)[2]) {  // this lane's; the warp holds every row
  bool huge = false;
#pragma unroll
  for (int n = 0; n < N; ++n) huge = huge || fabsf(rs[n][0]) >= kKv4Huge || fabsf(rs[n][1]) >= kKv4Huge;
  huge = __any_sync(0xffffffffu, huge);
  const float by = huge ? kKv4Codes / kKv4Lift : kKv4Codes;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    rs[n][0] *= by;
    rs[n][1] *= by;
  }
  return huge;
}

// Eight dims of a normalised query, the partners of a code word: operands of two k steps (nibbles
// 0 and 4 with 1 and 5, 2 and 6 with 3 and 7; the second pair of each counts 16-fold); -> their sum,
// of the dims before that rounding: the minima meet the query as it is.
__device__ __forceinline__ float query_pairs(const float* x, uint2* out) {
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const __half2 even = __floats2half2_rn(x[2 * k], x[2 * k + 4]), odd = __floats2half2_rn(x[2 * k + 1], x[2 * k + 5]);
    const __half2 odd16 = __hmul2(odd, __float2half2_rn(0.0625f));
    sum += (x[2 * k] + x[2 * k + 4]) + (x[2 * k + 1] + x[2 * k + 5]);
    out[k] = make_uint2(*reinterpret_cast<const uint32_t*>(&even), *reinterpret_cast<const uint32_t*>(&odd16));
  }
  return sum;
}

// Eight consecutive fp16 or bf16 values.
template <int TYPE>
__device__ __forceinline__ void kv4_load8(const void* base, long long i, float* x) {
  const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + i);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = TYPE == KV4_BF16 ? make_float2(bf16_lo(u[k]), bf16_hi(u[k]))
                                      : __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
    x[2 * k] = f.x;
    x[2 * k + 1] = f.y;
  }
}

// ---- work of the blocks ---------------------------------------------------------
// A segment is (sequence, key / value head, row block): its keys are walked in
// steps of 128 rows.  Few steps, or very many segments: a block each.  Otherwise
// the blocks that stay resident share them in one of two ways, chosen on the
// device from the lengths:
//   - every segment in equal parts, a block each;
//   - the steps of all segments in one line, cut into consecutive pieces equal to one step,
//     so that uneven lengths and segment counts that do not fill the GPU cost
//     nothing, but a block that goes on to a second segment starts anew.
// A block then holds at most two pieces that it shares with others, the first (of
// a segment begun by an earlier block) and the last; those go to slots 2 * block
// and 2 * block + 1 of the workspace, and the block that begins a segment notes
// its first and last block for the kernel that joins them.
constexpr int kKv4Step = 128;

// n / d for 0 <= n < 2^31 as a multiplication.
struct Kv4Div {
  int d;
  uint32_t mul, shift;
  explicit Kv4Div(int n) : d(n), mul(0), shift(0) {  // mul = ceil(2^(32 + shift) / d), shift = ceil(log2 d) - 1
    while ((2ull << shift) < (unsigned long long)d) ++shift;
    if (d > 1) mul = (uint32_t)(((1ull << (32 + shift)) + d - 1) / d);
  }
  __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
};

struct Kv4Line {
  Kv4Div segments;    // of one sequence: Hk * row_blocks
  Kv4Div row_blocks, group, rows;  // row blocks of a head, heads that share one, query rows of it: Tn * group
  int restart;        // what a second segment costs a block, in steps; 0: a block per segment
  int blocks;
  int2* meta;         // [B * segments] first and last block
  int* begun;         // [blocks] the segment that begins in a block and goes on in others, or -1
};

constexpr int kKv4MaxLine = 256;   // sequences on a line

struct Kv4Piece {
  int b, segment;                  // sequence, segment of it
  int steps, step0, step1;         // of the segment; the block's own
  int sink_tiles, first, tiles;    // tiles over the memory rows; first tile behind them; all
};

// Rows [lo, hi) that any query of a sequence sees.
__device__ __forceinline__ Kv4Seen kv4_union(const Kv4Attend& a, int b) {
  Kv4Seen u{a.L, 0};
  for (int t = 0; t < a.Tn; ++t) {
    const Kv4Seen s = kv4_seen(a, b, t);
    if (s.hi > s.lo) {
      u.lo = min(u.lo, s.lo);
      u.hi = max(u.hi, s.hi);
    }
  }
  return u;
}

template <int kTile>
__device__ __forceinline__ void kv4_tiles(const Kv4Attend& a, Kv4Seen u, Kv4Piece* p) {
  p->sink_tiles = (a.n_sink + kTile - 1) / kTile;
  p->first = max(u.lo / kTile, p->sink_tiles);
  p->tiles = p->sink_tiles + max(0, u.hi > u.lo ? (u.hi + kTile - 1) / kTile - p->first : 0);
  constexpr int kPerStep = kKv4Step / kTile;
  p->steps = max(1, (p->tiles + kPerStep - 1) / kPerStep);  // a sequence that sees nothing still writes zeros
}

// The pieces of one block, in turn; every thread of the block calls both functions.
// Shared memory: for each sequence the steps up to its end, its first tile and its tiles.
struct Kv4Walk {
  int end[kKv4MaxLine], first[kKv4MaxLine], tiles[kKv4MaxLine], sums[32], most[32];

  // -> first and last step of the block on the line.  share: steps of a block (or one more), or minus
  // the parts that every segment is cut into
  template <int kThreads, int kTile>
  __device__ __forceinline__ int2 begin(const Kv4Attend& a, const Kv4Line& l, int* share) {
    if (l.restart == 0) return make_int2(0, 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int before = 0, longest = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      Kv4Piece q;
      q.steps = 0;
      if (b0 + tid < a.B) kv4_tiles<kTile>(a, kv4_union(a, b0 + tid), &q);
      int sum = q.steps;  // inclusive prefix over the threads
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const int top = __reduce_max_sync(0xffffffffu, q.steps);
      if (lane == 31) {
        sums[warp] = sum;
        most[warp] = top;
      }
      __syncthreads();
      int all = before;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) sum += sums[w];
        all += sums[w];
        longest = max(longest, most[w]);
      }
      if (b0 + tid < a.B) {
        end[b0 + tid] = before + sum;
        first[b0 + tid] = q.first;
        tiles[b0 + tid] = q.tiles;
      }
      before = all;
      __syncthreads();
    }
    const int total = before * l.segments.d;
    if (threadIdx.x == 0) l.begun[blockIdx.x] = -1;
    const int blocks = gridDim.x, at = blockIdx.x, each = total / blocks, parts = blocks / (a.B * l.segments.d);
    if (parts > 0 && (longest + parts - 1) / parts <= each + l.restart) {
      *share = -parts;
      return make_int2(0, at < a.B * l.segments.d * parts);
    }
    *share = each;
    const int more = total - each * blocks;   // blocks of one step more come first
    return make_int2(at * each + min(at, more), (at + 1) * each + min(at + 1, more));
  }

  // The segment that holds step span.x; moves span.x behind it.  A block per segment: tiles and
  // steps are left to kv4_tiles() of the rows that its queries see.
  template <int kTile>
  __device__ __forceinline__ Kv4Piece next(const Kv4Attend& a, const Kv4Line& l, int share, int2* span) {
    Kv4Piece p;
    if (l.restart == 0) {
      p.b = l.segments.of(blockIdx.x);
      p.segment = blockIdx.x - p.b * l.segments.d;
      p.steps = p.step0 = p.step1 = p.sink_tiles = p.first = p.tiles = 0;
      span->x = span->y;
      return p;
    }
    p.sink_tiles = (a.n_sink + kTile - 1) / kTile;
    int last = blockIdx.x;
    if (share < 0) {
      const int place = blockIdx.x / -share, part = blockIdx.x + place * share;
      p.b = l.segments.of(place);
      p.segment = place - p.b * l.segments.d;
      p.steps = end[p.b] - (p.b > 0 ? end[p.b - 1] : 0);
      const int each = (p.steps - share - 1) / -share;
      p.step0 = min(p.steps, part * each);
      p.step1 = min(p.steps, p.step0 + each);
      last += (p.steps - 1) / each;   // of part 0
      span->x = span->y;
    } else {
      int lo = 0, hi = a.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] * l.segments.d > span->x) hi = mid;
        else lo = mid + 1;
      }
      const int start = lo > 0 ? end[lo - 1] : 0;
      p.b = lo;
      p.steps = end[lo] - start;
      p.segment = (span->x - start * l.segments.d) / p.steps;
      const int at = start * l.segments.d + p.segment * p.steps;   // the segment's first step on the line
      p.step0 = span->x - at;
      p.step1 = min(p.steps, span->y - at);
      span->x = at + p.steps;
      if (p.step0 == 0 && p.step1 < p.steps && threadIdx.x == 0) {   // the block of the segment's last step
        const int step = at + p.steps - 1, more = end[a.B - 1] * l.segments.d - share * (int)gridDim.x;
        const int cut = more * (share + 1);
        last = step < cut ? step / (share + 1) : more + (step - cut) / share;
      }
    }
    p.first = first[p.b];
    p.tiles = tiles[p.b];
    if (p.step0 == 0 && threadIdx.x == 0) {
      const int place = p.b * l.segments.d + p.segment;
      l.meta[place] = make_int2(blockIdx.x, last);
      if (last > (int)blockIdx.x) l.begun[blockIdx.x] = place;
    }
    return p;
  }
};

// What the queries of a block see.  Lane r holds query row r; the other numbers are the warp's.
struct Kv4View {
  Kv4Seen seen;
  int lo_min, hi_max;   // rows that any of them sees
  int lo_max, hi_min;   // rows that all of them see
};

template <int kTile>
__device__ __forceinline__ Kv4View kv4_rows(const Kv4Attend& a, const Kv4Line& l, Kv4Piece* p, int row0, int nrows) {
  Kv4View r{Kv4Seen{0, 0}, 0, 0, 0, 0};
  const int lane = lane_id();
  const bool valid = lane < nrows;
  if (valid) r.seen = kv4_seen(a, p->b, l.group.of(row0 + lane));
  const bool any = valid && r.seen.hi > r.seen.lo;
  r.lo_min = __reduce_min_sync(0xffffffffu, any ? r.seen.lo : a.L);
  r.hi_max = __reduce_max_sync(0xffffffffu, any ? r.seen.hi : 0);
  r.lo_max = __reduce_max_sync(0xffffffffu, valid ? r.seen.lo : 0);
  r.hi_min = __reduce_min_sync(0xffffffffu, valid ? r.seen.hi : a.L);
  if (l.restart == 0) {
    kv4_tiles<kTile>(a, Kv4Seen{r.lo_min, r.hi_max}, p);
    p->step1 = p->steps;
  }
  return r;
}

// Every kernel of this family may be set up while its predecessor in the stream still runs: it
// waits for that one's end, and its memory, before it touches any.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
void kv4_launch(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Steps of a segment in a full cache (or window): the host does not know the sequences' lengths.
long long kv4_plan_steps(const Kv4Attend& a);
// Grid and workspace: slots blocks stay resident; a block's start costs it about restart steps.
void kv4_line_plan(const Kv4Attend& a, Kv4Plan& p, int slots, int restart);
Kv4Line kv4_line(const Kv4Attend& a, const Kv4Plan& p);
// Joins the pieces: 8 * row_tiles rows of V sums and then (max, sum) pairs per slot.
void kv4_combine(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s);
void kv4_heads_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s);
void kv4_heads_plan(const Kv4Attend& a, Kv4Plan& p);
void kv4_latent_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s);
void kv4_latent_plan(const Kv4Attend& a, Kv4Plan& p);

}  // namespace omni
