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
// Eight consecutive values of one type <-> fp32
// ---------------------------------------------------------------------------
template <int TYPE>
__device__ __forceinline__ void load8(const void* base, long long i, float* x) {
  if (TYPE == KV4_F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + i);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (TYPE == KV4_BF16) {
        x[2 * k] = bf16_lo(u[k]);
        x[2 * k + 1] = bf16_hi(u[k]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
        x[2 * k] = f.x;
        x[2 * k + 1] = f.y;
      }
    }
  }
}

template <int TYPE>
__device__ __forceinline__ void store8(void* base, long long i, const float* x) {
  if (TYPE == KV4_F32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + i) =
        make_uint4(kv4_pack2<TYPE>(x[0], x[1]), kv4_pack2<TYPE>(x[2], x[3]), kv4_pack2<TYPE>(x[4], x[5]), kv4_pack2<TYPE>(x[6], x[7]));
  }
}

template <int TYPE>
__device__ __forceinline__ void store1(void* base, long long i, float x) {
  if (TYPE == KV4_BF16)
    reinterpret_cast<bf16*>(base)[i] = __float2bfloat16_rn(x);
  else
    reinterpret_cast<__half*>(base)[i] = __float2half_rn(x);
}

// ---------------------------------------------------------------------------
// Append and read back.  A thread owns eight dims (one 16-byte piece of a
// 16-bit row, four bytes of codes); the threads of a group of g dims are
// neighbours in a warp.  Threads run over (head, token, piece) of a sequence
// with the token in the middle, so that a warp writes whole sectors of one
// head's rows.  Both are bound by memory, single tokens by the launch.
// ---------------------------------------------------------------------------
constexpr int kIoThreads = 256;

struct IoIndex {
  int h, t, piece;
  long long row;
  bool active;
};

__device__ __forceinline__ IoIndex io_index(const Kv4IO& a) {
  const int pieces = a.W / 8, per_head = a.T * pieces;
  const int total = per_head * a.Hk;
  const long long i = (long long)blockIdx.x * kIoThreads + threadIdx.x;
  IoIndex x;
  x.active = i < total;
  const int k = x.active ? (int)i : 0;
  x.h = k / per_head;
  const int r = k - x.h * per_head;
  x.t = r / pieces;
  x.piece = r - x.t * pieces;
  x.row = a.row_offset + kv4_load_pos(a.pos, a.pos64, (long long)blockIdx.y * a.T + x.t);
  return x;
}

// Round (x - m) / s, decided as if the quotient were exact: d + e = x - m
// exactly, r = d - n s exactly (n s has at most 12 significant bits and lies
// within s of d), and r + e is compared with half a step.
__device__ __forceinline__ int kv4_code(float x, float m, float s, float inv) {
  const float d = x - m;
  const float back = d - x;
  const float e = (x - (d - back)) - (m + back);
  float n = rintf(d * inv);
  const float r = fmaf(-n, s, d), half = 0.5f * s;
  const bool odd = ((int)n & 1) != 0;
  if (r > half || (r == half && (e > 0.f || (e == 0.f && odd)))) n += 1.f;
  else if (r < -half || (r == -half && (e < 0.f || (e == 0.f && odd)))) n -= 1.f;
  return (int)fminf(fmaxf(n, 0.f), 15.f);
}

template <int TYPE>
__global__ void __launch_bounds__(kIoThreads) kv4_write_kernel(const Kv4IO a) {
  const IoIndex ix = io_index(a);
  const int b = blockIdx.y;
  const Kv4Cache& c = a.cache[blockIdx.z];
  const Kv4Rows& src = a.rows[blockIdx.z];
  float x[8];
  load8<TYPE>(src.x, b * src.x_b + ix.t * src.x_t + ix.h * src.x_h + ix.piece * 8, x);
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad |= (__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u;
  }
  const int lanes = a.group / 8;  // 2, 4 or 8 neighbouring threads hold a group
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    const float l2 = __shfl_xor_sync(0xffffffffu, lo, o), h2 = __shfl_xor_sync(0xffffffffu, hi, o);
    const int b2 = __shfl_xor_sync(0xffffffffu, (int)bad, o);
    if (o < lanes) {
      lo = fminf(lo, l2);
      hi = fmaxf(hi, h2);
      bad |= b2 != 0;
    }
  }
  // m: exact for 16-bit rows whose type is bf16; the scale is taken from the rounded minimum
  const bf16 mb = __float2bfloat16_rn(lo);
  const float m = __bfloat162float(mb);
  bf16 sb = __float2bfloat16_rn(__fdiv_rn(hi - m, 15.f));
  float s = __bfloat162float(sb);
  bad |= !(fabsf(m) <= 3.3895314e38f) || !(s <= 3.3895314e38f);
  if (s < kMinScale) {
    s = 0.f;
    sb = __float2bfloat16_rn(0.f);
  }
  uint32_t code = 0;
  if (!bad && s > 0.f) {
    const float inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) code |= (uint32_t)kv4_code(x[i], m, s, inv) << (4 * i);
  }
  if (!ix.active || ix.row < 0 || ix.row >= a.L) return;
  *reinterpret_cast<uint32_t*>(c.codes + b * c.c_b + ix.h * c.c_h + ix.row * (a.W / 2) + ix.piece * 4) = code;
  if (ix.piece % lanes == 0) {
    const uint32_t word = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(mb) << 16);
    *reinterpret_cast<uint32_t*>(c.params + b * c.p_b + ix.h * c.p_h + (ix.row * (a.W / a.group) + ix.piece / lanes) * 4) =
        bad ? 0x7fc07fc0u : word;
  }
}

template <int TYPE>
__global__ void __launch_bounds__(kIoThreads) kv4_read_kernel(const Kv4IO a) {
  const IoIndex ix = io_index(a);
  if (!ix.active) return;
  const int b = blockIdx.y;
  const Kv4Cache& c = a.cache[blockIdx.z];
  const Kv4Rows& dst = a.rows[blockIdx.z];
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (ix.row >= 0 && ix.row < a.L) {
    const uint32_t code =
        *reinterpret_cast<const uint32_t*>(c.codes + b * c.c_b + ix.h * c.c_h + ix.row * (a.W / 2) + ix.piece * 4);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(
        c.params + b * c.p_b + ix.h * c.p_h + (ix.row * (a.W / a.group) + ix.piece * 8 / a.group) * 4);
    const float s = bf16_lo(word), m = bf16_hi(word);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((code >> (4 * i)) & 15u), s, m);
  }
  store8<TYPE>(dst.x, b * dst.x_b + ix.t * dst.x_t + ix.h * dst.x_h + ix.piece * 8, x);
}

dim3 io_grid(const Kv4IO& a) {
  const long long n = (long long)a.T * a.Hk * (a.W / 8);
  return dim3((unsigned)((n + kIoThreads - 1) / kIoThreads), (unsigned)a.B, (unsigned)a.count);
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
  const int tiles = (a.L + 31) / 32;
  for (int tile = warp; tile < tiles; tile += kRowWarps) {
    const int r0 = tile * 32;
    if (r0 >= a.n_sink && (r0 + 32 <= seen.lo || r0 >= seen.hi)) continue;
    const int r = r0 + lane;
    const bool vis = r < a.n_sink || (r >= seen.lo && r < seen.hi);
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
      if (pk == 0.f) continue;  // unseen rows, whatever they hold
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
  kern<<<dim3((unsigned)(a.Tn * a.H), (unsigned)a.B), kRowWarps * 32, smem, s>>>(a);
}

}  // namespace

void kv4_write(const Kv4IO& a, cudaStream_t s) {
  if (a.type == KV4_F32) kv4_write_kernel<KV4_F32><<<io_grid(a), kIoThreads, 0, s>>>(a);
  else if (a.type == KV4_F16) kv4_write_kernel<KV4_F16><<<io_grid(a), kIoThreads, 0, s>>>(a);
  else kv4_write_kernel<KV4_BF16><<<io_grid(a), kIoThreads, 0, s>>>(a);
}

void kv4_read(const Kv4IO& a, cudaStream_t s) {
  if (a.type == KV4_F32) kv4_read_kernel<KV4_F32><<<io_grid(a), kIoThreads, 0, s>>>(a);
  else if (a.type == KV4_F16) kv4_read_kernel<KV4_F16><<<io_grid(a), kIoThreads, 0, s>>>(a);
  else kv4_read_kernel<KV4_BF16><<<io_grid(a), kIoThreads, 0, s>>>(a);
}

Kv4Plan kv4_plan(const Kv4Attend& a) {
  Kv4Plan p{};
  p.splits = 1;
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
