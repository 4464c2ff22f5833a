// How the attention kernels over a 4-bit cache share their keys, and the kernel
// that joins what they shared.
#include <algorithm>
#include <cmath>

#include "kv4_device.cuh"

namespace omni {

namespace {

constexpr int kThreads = 256;

// A thread holds four value dims of a query row; GROUPS threads take every GROUPS-th
// piece each and are summed in a fixed order.
template <int TYPE, int GROUPS>
__global__ void __launch_bounds__(kThreads) kv4_combine_kernel(const Kv4Attend a, const Kv4Line line, const Kv4Div cols,
                                                              const int rows_per_block, const bool by_block) {
  constexpr int kItems = kThreads / GROUPS;
  __shared__ float4 s_sum[kThreads];
  __shared__ float2 s_ml[kThreads];
  const int item = threadIdx.x % kItems, group = threadIdx.x / kItems, at = blockIdx.x * kItems + item;
  const int place0 = cols.of(at), col = at - place0 * cols.d;   // four dims of a row
  wait_for_previous_grid();
  launch_dependents();
  // by segment: place is (sequence, head, row); by block: (block, row of the segment begun there)
  int2 range = make_int2(0, 0);
  int b = 0, hk = 0, row = 0;
  if (by_block) {
    const int block = place0 / rows_per_block, segment = block < line.blocks ? line.begun[block] : -1;
    if (segment >= 0) {
      b = line.segments.of(segment);
      const int in = segment - b * line.segments.d;
      hk = line.row_blocks.of(in);
      row = (in - hk * line.row_blocks.d) * rows_per_block + place0 % rows_per_block;
      if (row < line.rows.d) range = line.meta[segment];
    }
  } else {
    const int head = line.rows.of(place0);
    row = place0 - head * line.rows.d;
    b = head / a.Hk;
    hk = head - b * a.Hk;
    if (b < a.B) range = line.meta[b * line.segments.d + hk * line.row_blocks.d + row / rows_per_block];
  }
  const int t = line.group.of(row), r = row & (rows_per_block - 1);
  const bool join = range.x != range.y;  // otherwise one block held the segment and has written the row
  const size_t slot = (size_t)rows_per_block * (a.V + 2);
  float top = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (join) {
#pragma unroll 4
    for (int k = range.x + group; k <= range.y; k += GROUPS) {
      const float* p = a.part + (2 * (size_t)k + (k == range.x)) * slot;
      const float2 ml = *reinterpret_cast<const float2*>(p + rows_per_block * a.V + 2 * r);
      const float4 v = *reinterpret_cast<const float4*>(p + r * a.V + 4 * col);
      const float m = fmaxf(top, ml.x), ref = m == -INFINITY ? 0.f : m;
      const float f0 = fast_exp2(top - ref), f1 = fast_exp2(ml.x - ref);
      l = l * f0 + ml.y * f1;
      o.x = o.x * f0 + v.x * f1;
      o.y = o.y * f0 + v.y * f1;
      o.z = o.z * f0 + v.z * f1;
      o.w = o.w * f0 + v.w * f1;
      top = m;
    }
  }
  s_sum[threadIdx.x] = o;
  s_ml[threadIdx.x] = make_float2(top, l);
  __syncthreads();
  if (group != 0 || !join) return;
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) top = fmaxf(top, s_ml[g * kItems + item].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  l = 0.f;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const float2 ml = s_ml[g * kItems + item];
    const float4 v = s_sum[g * kItems + item];
    const float f = fast_exp2(ml.x - ref);
    l = fmaf(f, ml.y, l);
    x.x = fmaf(f, v.x, x.x);
    x.y = fmaf(f, v.y, x.y);
    x.z = fmaf(f, v.z, x.z);
    x.w = fmaf(f, v.w, x.w);
  }
  const long long out = ((long long)b * a.Tn + t) * a.H + hk * line.group.d + row - t * line.group.d;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + out * a.V + 4 * col) =
      make_uint2(kv4_pack2<TYPE>(x.x * inv, x.y * inv), kv4_pack2<TYPE>(x.z * inv, x.w * inv));
}

template <int TYPE, int GROUPS>
void launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  const long long segments = (long long)a.B * a.Hk * p.row_blocks, rows = 8 * p.row_tiles;
  const bool by_block = p.blocks < segments;   // at most one shared segment begins in a block
  const long long items = (by_block ? p.blocks * rows : (long long)a.B * a.Tn * a.H) * (a.V / 4), per = kThreads / GROUPS;
  kv4_launch(kv4_combine_kernel<TYPE, GROUPS>, dim3((unsigned)((items + per - 1) / per)), kThreads, 0, s, a, kv4_line(a, p),
             Kv4Div(a.V / 4), (int)rows, by_block);
}

}  // namespace

Kv4Line kv4_line(const Kv4Attend& a, const Kv4Plan& p) {
  const size_t sums = (size_t)p.blocks * 2 * 8 * p.row_tiles * (a.V + 2), segments = (size_t)a.B * a.Hk * p.row_blocks;
  const int group = a.H / a.Hk;
  int2* meta = reinterpret_cast<int2*>(a.part + sums);
  return Kv4Line{Kv4Div(a.Hk * p.row_blocks), Kv4Div(p.row_blocks), Kv4Div(group), Kv4Div(a.Tn * group), p.restart, p.blocks,
                 meta, reinterpret_cast<int*>(meta + segments)};
}

long long kv4_plan_steps(const Kv4Attend& a) {
  const long long rows = a.n_sink + std::min<long long>(a.L - a.sink_rows, a.window > 0 ? (long long)a.window + a.Tn : 1 << 30);
  return (rows + kKv4Step - 1) / kKv4Step;
}

// A block per segment costs the steps of the SM with the most of them, the blocks of an SM sharing its
// pipes; shared steps cost their share, and about `restart` steps more to find the places and to join the
// pieces.  Measured, one query row a sequence, us shared / a block each: 8 heads of 128, 1 sequence of 2,
// 4, 8 steps 6.7 / 4.9, 7.3 / 7.2, 7.3 / 11.5, 64 of 8 steps 30.9 / 27.5, 256 of 16 150 / 141; one latent
// head, 1 sequence of 1, 2, 4 steps 10.2 / 7.9, 11.2 / 11.6, 11.8 / 18.5, 64 of 8 25 / 34, 256 of 16
// 112 / 105, of up to 16 88 / 103.  Many sequences or new tokens make the places on the line dear to
// find: a block each.
void kv4_line_plan(const Kv4Attend& a, Kv4Plan& p, int slots, int restart) {
  const long long steps = kv4_plan_steps(a), segments = (long long)a.B * a.Hk * p.row_blocks;
  const double each = steps * std::max(1.0, (segments + 147) / 148 * 148.0 / slots);
  const double shared = std::max(1.0, std::ceil((double)steps * segments / slots)) + restart;
  if (each <= shared || a.B > kKv4MaxLine || a.Tn > 16 || segments * (steps + 1) > (1 << 30) ||
      (long long)a.B * a.Tn * a.H * a.V > (1 << 30)) {
    p.restart = 0;
    p.blocks = (int)segments;
    p.floats = 0;
    return;
  }
  p.restart = restart;
  p.blocks = (int)std::min<long long>(slots, segments * (steps + 1));
  p.floats = (size_t)p.blocks * (2 * 8 * p.row_tiles * (a.V + 2) + 1) + 2 * (size_t)segments;
}

void kv4_combine(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s) {
  // A segment has about blocks / segments + 1 pieces.  Measured, 16 and 2 threads for the pieces of four
  // dims, us of the whole call: 55 pieces 13.0 / 16.8, 17 pieces 8.8 / 10.9, 5 pieces 8.3 / 8.6 and,
  // of many rows (32768 times four dims), 9 pieces 19.5 / 14.8, 18 pieces 27.5 / 27.7.
  const long long segments = (long long)a.B * a.Hk * p.row_blocks;
  const bool many = p.blocks > 6 * segments && (long long)a.B * a.Tn * a.H * (a.V / 4) <= 16384;
  if (a.type == KV4_F16) many ? launch<KV4_F16, 16>(a, p, s) : launch<KV4_F16, 2>(a, p, s);
  else many ? launch<KV4_BF16, 16>(a, p, s) : launch<KV4_BF16, 2>(a, p, s);
}

}  // namespace omni
