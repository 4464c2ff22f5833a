// Device helpers shared by the attention kernels over a 4-bit cache.
#pragma once
#include "common.cuh"
#include "kv4.h"

namespace omni {

constexpr float kKv4Log2e = 1.4426950408889634f;

__device__ __forceinline__ long long kv4_load_pos(const void* p, bool is64, long long i) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
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
  const long long len = kv4_load_pos(a.kv_len, a.len64, b);
  const long long qp = kv4_load_pos(a.q_pos, a.pos64, (long long)b * a.Tn + t);
  const long long room = a.L - a.sink_rows;
  const long long end = max(min(min(len, qp + 1), room), 0ll);
  const long long first = a.window > 0 ? max(qp - a.window + 1, 0ll) : 0ll;
  Kv4Seen s;
  s.lo = a.sink_rows + (int)min(first, room);
  s.hi = max(a.sink_rows + (int)end, s.lo);
  return s;
}

// ---- legacy tensor-core tiles on registers -----------------------------------
// Codes become matrix operands in registers, straight from the 4-bit tile in
// shared memory; tcgen05 operands would have to be written back to shared or
// tensor memory as 16-bit tiles first, four times the bytes of the codes, for a
// product of 8 or 16 columns that the memory-bound kernel does not wait for.
__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Nibble `mm` of both 16-bit halves as the bf16 pair (16 + n, 16 + n'): bits 3..6
// of a bf16 mantissa at exponent 2^4 count in ones.
template <int MM>
__device__ __forceinline__ uint32_t nibbles_bf16(uint32_t x) {
  const uint32_t y = MM == 0 ? x << 3 : x >> (MM == 0 ? 0 : 4 * MM - 3);
  return (y & 0x00780078u) | 0x41804180u;
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

// Query rows enter the fp16 product with codes as q * 2^e, the largest |q| of the
// row in [2^14, 2^15): bf16 and fp16 values keep every bit down to 2^-39 of it.
// `unscale` is 2^-e; the codes' 2^-24 is undone separately (kKv4Codes).
constexpr float kKv4Codes = 16777216.f;
__device__ __forceinline__ float q_normaliser(float amax, float* unscale) {
  const uint32_t e = min(max((__float_as_uint(amax) >> 23) & 255u, 40u), 254u);
  *unscale = __uint_as_float((e - 14u) << 23);  // 2^(e - 127 - 14)
  return __uint_as_float((268u - e) << 23);     // 2^(14 - (e - 127))
}

// Workspace of the splits: rows [B, Hk, R, splits] of V sums, then (max, sum) pairs.
void kv4_combine(const Kv4Attend& a, int splits, cudaStream_t s);
void kv4_heads_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s);
void kv4_heads_plan(const Kv4Attend& a, Kv4Plan& p);
void kv4_latent_launch(const Kv4Attend& a, const Kv4Plan& p, cudaStream_t s);
void kv4_latent_plan(const Kv4Attend& a, Kv4Plan& p);

}  // namespace omni
