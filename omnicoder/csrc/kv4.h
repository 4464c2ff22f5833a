// Host interface of the 4-bit key / value cache kernels (kv4.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace omni {

enum Kv4Type : int { KV4_F32 = 0, KV4_F16 = 1, KV4_BF16 = 2 };

// One cache: codes [B, Hk, L, W / 2] and params [B, Hk, L, W / group, 2] with contiguous rows;
// strides in bytes.
struct Kv4Cache {
  uint8_t* codes;
  uint8_t* params;
  long long c_b, c_h, p_b, p_h;
};

// Rows of values beside it: x [B, T, Hk, W] with contiguous rows, strides in elements.
struct Kv4Rows {
  void* x;
  long long x_b, x_t, x_h;
};

struct Kv4IO {
  Kv4Cache cache[2];
  Kv4Rows rows[2];
  int count;             // 1, or 2 for keys and values
  const void* pos;       // [B, T] int32 or int64
  bool pos64;
  int B, T, Hk, L, W, group;
  long long row_offset;
  int type;              // Kv4Type of the rows
};
void kv4_write(const Kv4IO& a, cudaStream_t s);
void kv4_read(const Kv4IO& a, cudaStream_t s);

struct Kv4Attend {
  const void* q;         // [B, Tn, H, W], fp16 or bf16, contiguous
  int type;
  Kv4Cache k, v;         // v.codes == nullptr: latent cache, the value is the first V dims of a row
  const void* q_pos;     // [B, Tn]
  const void* kv_len;    // [B]
  bool pos64, len64;
  void* out;             // [B, Tn, H, V]
  float* part;           // workspace of kv4_plan().floats
  int B, Tn, H, Hk, L, W, V, group;
  int window, sink_rows, n_sink;
  float scale;
};
struct Kv4Plan {
  int kernel;            // 0: one block per query row, 1: grouped heads, 2: latent
  int row_tiles;         // 8-row query tiles per block
  int row_blocks;        // blocks that share a key / value head's query rows
  int blocks;            // grid: blocks that share the key tiles of all of them
  int restart;           // what a block's start costs it, in steps of 128 keys; 0: a block per (sequence, head, rows)
  size_t floats;         // workspace
};
Kv4Plan kv4_plan(const Kv4Attend& a);
void kv4_attend(const Kv4Attend& a, const Kv4Plan& plan, cudaStream_t s);

}  // namespace omni
