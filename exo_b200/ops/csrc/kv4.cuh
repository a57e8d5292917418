// Layout of a 4-bit KV cache unit (16 tokens of one head, 10 D bytes), shared by the kernels that write and read it.
// exo_b200/ops/kv4.py defines the format; the orders below put a lane's operands next to each other:
//   keys    words [D/128][16 tokens][4 t][4 g], word (t, g) = dims 32 g + 8 t .. +7
//   values  halfwords [D/128][16 places][8 slots][4 g], halfword g of slot c = dims 32 g + 4 c' .. +3
// (64-wide heads have 2 groups: [16][4][2] words, [16][8][2] halfwords, no slot swizzle).
#pragma once
#include <cuda_fp16.h>
#include <cstring>
#include "common.cuh"

namespace kv4 {

constexpr int GROUP = 32;
constexpr int UNIT = 16;      // tokens
constexpr float LARGEST = 65280.f;      // of a cached value: 15 s + m then fits fp16

template <int D> struct Geo {
  static constexpr int BYTES = 10 * D;          // of a unit
  static constexpr int CODES = 8 * D;           // of them codes
  static constexpr int G = D / GROUP;           // groups of a row
  static constexpr int PER = G < 4 ? G : 4;     // groups that a word order interleaves
  static constexpr int HALVES = D / (PER * GROUP);
};

__host__ __device__ constexpr int v_place(int tok) { return (tok & 8) | ((tok & 1) << 2) | ((tok >> 1) & 3); }

// byte of the code of (tok, dim) in a unit; dims 2i, 2i + 1 share it, the even one in the low nibble
template <int D> __device__ __forceinline__ int k_byte(int tok, int dim) {
  constexpr int P = Geo<D>::PER;
  const int h = dim / (P * GROUP), r = dim % (P * GROUP), g = r / GROUP, i = r % GROUP;
  return ((h * UNIT + tok) * 4 + i / 8) * (4 * P) + 4 * g + (i % 8) / 2;
}
template <int D> __device__ __forceinline__ int v_slot(int place, int c) { return D == 64 ? c : c ^ ((place & 2) << 1); }
template <int D> __device__ __forceinline__ int v_byte(int tok, int dim) {
  constexpr int P = Geo<D>::PER;
  const int h = dim / (P * GROUP), r = dim % (P * GROUP), g = r / GROUP, i = r % GROUP;
  const int place = v_place(tok);
  return ((h * UNIT + place) * 8 + v_slot<D>(place, i / 4)) * (2 * P) + 2 * g + (i % 4) / 2;
}
// index of the scale of (tok, group) among the unit's fp16 numbers (which start behind the codes); the least value's is
// 16 G further on
template <int D> __device__ __forceinline__ int k_meta(int tok, int g) { return tok * Geo<D>::G + g; }
template <int D> __device__ __forceinline__ int v_meta(int tok, int g) { return ((tok >> 1) * Geo<D>::G + g) * 2 + (tok & 1); }

// where the unit of a slot starts: block, head, unit of the block
__device__ __forceinline__ size_t unit_index(long block, int head, int n_kv, int units_per_block, int unit) {
  return ((size_t)block * n_kv + head) * units_per_block + unit;
}

// x / d and x % d for 0 <= x < 2^31 without a division: x m >> p with m = ceil(2^p / d), p = 31 + ceil(log2 d)
struct FastDiv {
  uint32_t m, d;
  int p;
  __host__ __device__ FastDiv() : m(0), d(1), p(0) {}
  explicit FastDiv(int by) : d((uint32_t)by), p(31) {
    while ((1u << (p - 31)) < d) p++;
    m = (uint32_t)((((unsigned long long)1 << p) + d - 1) / d);
  }
  __device__ __forceinline__ int div(int x) const { return (int)(((unsigned long long)(uint32_t)x * m) >> p); }
};

// Arguments of the entry points, as one block of memory: a Python caller packs them at once (22 to 30 arguments through ctypes take
// 5 to 8 us, a block and two arguments 2).
struct AppendCall {
  const void *q, *k, *v;
  long sq, sk, sv;
  const int *positions, *axes;
  const float* inv_freq;
  void *q_out, *kcache, *vcache;
  const int* slots;
  const void *q_norm, *k_norm;
  long n_slots;
  float mscale, eps;
  int n_axes, n_q, n_kv, head_dim, rot, block_size, T, dtype, v_unit, quantized;
};
struct ReadCall {
  const void *kcache, *vcache;
  const int* slots;
  void *kout, *vout;
  long rows, n_slots;
  int n_kv, head_dim, block_size, dtype;
};
struct AttnCall {
  const void *q, *kcache, *vcache;
  const int *tables, *seq_lens, *cu_q;
  void *out, *ws;
  int* tickets;                 // decode
  const void* sinks;
  float scale;
  int splits;                   // prompt
  int T, B, Hq, Hkv, D, n_blocks, max_blocks, block_size, window, sink_dtype;
};
// false: the block is not one of these
template <typename C> inline bool unpack_call(C& c, const void* block, int bytes) {
  if (!block || bytes != (int)sizeof(C)) return false;
  memcpy(&c, block, sizeof(C));
  return true;
}

// the sequence that row `t` of a ragged batch belongs to (cu_q[b] <= t < cu_q[b + 1]), -1 behind the last one
__device__ __forceinline__ int seq_of_row(const int* cu_q, int B, int t) {
  if (t >= cu_q[B]) return -1;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

}  // namespace kv4
