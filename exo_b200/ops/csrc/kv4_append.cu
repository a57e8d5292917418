// What writes a 4-bit KV cache, and what reads its rows back.
//
// The append takes the fused q/k/v projection of T tokens and does, per head of a token and without leaving registers:
//   x <- x * rsqrt(mean x^2 + eps) * w          (q and k, optional)
//   (x_i, x_{i+r}) <- rotation by p[axis(i)] * f_i   (q and k; r = half the rotated dims; one or several position axes)
//   q: stored;  k, v: 32-dim groups -> m = fp16 rounded down of the least value, s = fp16 rounded up of (max - m) / 15,
//   codes rint((x - m) / s), stored in the operand order of kv4.cuh.
// Nothing is rounded between the three steps.  The quotients are rounded as a division rounds them: bf16 rows hit exact halves
// of a step often (their values have few bits), and a product with a rounded reciprocal would decide those ties at random.  One
// correctly rounded reciprocal a group and Markstein's correction (q = a r, q + r (a - q s): correctly rounded) make that three
// instructions a value; adding 1.5 2^23 leaves the code in the sum's low bits.
//
// One block = one token, a warp = one head at a time, the next head's row on its way meanwhile.  The sines and cosines of a
// token are the same for all its heads: they are taken once per block (angle in 64 bits, reduced to one turn, then the fp32
// functions) and kept in shared memory.
// Bound by instructions, not bytes, until they were counted: 240 a row at first (two 64-bit divisions by the block size, five
// IEEE divisions, conversions through the slow unit).
#include "kv4.cuh"

namespace {

using namespace kv4;

struct AppendParams {
  const void *q, *k, *v;                 // first q / k / v head of token 0
  long sq, sk, sv;                       // elements between tokens
  const int* positions;                  // [T], or [axes][T]
  const int* axes;                       // [rot / 2] position axis of each pair, or null
  const float* inv_freq;
  float mscale;
  int n_q, n_kv, rot;
  void* q_out;                           // [T, n_q, D]
  void *kcache, *vcache;                 // 4-bit units, or rows [slots, n_kv, D]
  const int* slots;
  long n_slots;
  int block_size;
  FastDiv by_block;
  const void *q_norm, *k_norm;
  float eps;
  int T, v_unit, heads_per_block;
};

// E neighbouring values as they are in memory
template <typename T, int E> struct Raw { uint32_t w[E * sizeof(T) / 4]; };
template <typename T, int E> __device__ __forceinline__ Raw<T, E> load_raw(const T* p) {
  constexpr int N = E * sizeof(T) / 4;
  Raw<T, E> r;
  if constexpr (N == 1) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r.w[0] = u.x; r.w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
      r.w[i] = u.x; r.w[i + 1] = u.y; r.w[i + 2] = u.z; r.w[i + 3] = u.w;
    }
  }
  return r;
}
template <typename T, int E> __device__ __forceinline__ void unpack_raw(const Raw<T, E>& r, float* v) {
#pragma unroll
  for (int i = 0; i < E * (int)sizeof(T) / 4; i++) {
    if constexpr (sizeof(T) == 2) {
      v[2 * i] = __uint_as_float(r.w[i] << 16);
      v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    } else {
      v[i] = __uint_as_float(r.w[i]);
    }
  }
}

template <typename T, int E> __device__ __forceinline__ void store_row(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    if constexpr (E == 2) *reinterpret_cast<uint32_t*>(p) = w[0];
    else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<float2*>(p + e) = make_float2(v[e], v[e + 1]);
  }
}

// either is NaN
__device__ __forceinline__ bool nan2(float a, float b) {
  int r;
  asm("{\n\t.reg .pred p;\n\tsetp.nan.f32 p, %1, %2;\n\tselp.s32 %0, 1, 0, p;\n\t}" : "=r"(r) : "f"(a), "f"(b));
  return r != 0;
}
// a / s, rounded as IEEE division rounds it, where r is 1 / s so rounded
__device__ __forceinline__ float quotient(float a, float s, float r) {
  const float q = a * r;
  return fmaf(fmaf(-q, s, a), r, q);
}

// Quantises the row that a warp holds (E neighbouring dims a lane) into token `tok` of a unit.
template <int D, bool VALUES> __device__ __forceinline__ void quantize_row(const float* x, uint8_t* unit, int tok, int lane) {
  constexpr int E = D / 32, LG = GROUP / E;      // lanes of a group
  bool nan = false;
  float v[E], lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 0; e < E; e += 2) nan |= nan2(x[e], x[e + 1]);
#pragma unroll
  for (int e = 0; e < E; e++) {
    v[e] = x[e];
    lo = fminf(lo, v[e]);
    hi = fmaxf(hi, v[e]);
  }
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  nan = __any_sync(0xffffffffu, nan);            // one NaN makes the whole row NaN
  if (__any_sync(0xffffffffu, !(lo >= -LARGEST && hi <= LARGEST))) {
    lo = fminf(fmaxf(lo, -LARGEST), LARGEST);
    hi = fminf(fmaxf(hi, -LARGEST), LARGEST);
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = fminf(fmaxf(v[e], -LARGEST), LARGEST);
  }
  __half mh = __float2half_rd(lo);
  const float m = __half2float(mh);
  __half sh = __float2half_ru(quotient(hi - m, 15.f, 1.f / 15.f));
  const float s = __half2float(sh), r = s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t code = 0;
#pragma unroll
  for (int e = E - 1; e >= 0; e--)               // 0 <= (v - m) / s <= 15: m and s are rounded outwards
    code = code << 4 | (__float_as_uint(quotient(v[e] - m, s, r) + 12582912.f) & 15u);
  if (nan) { code = 0; sh = __ushort_as_half(0); mh = __ushort_as_half(0x7e00); }
  const int dim = lane * E, g = dim / GROUP;
  const int at = VALUES ? v_byte<D>(tok, dim) : k_byte<D>(tok, dim);
  if constexpr (E == 2) unit[at] = (uint8_t)code;
  else if constexpr (E == 4) *reinterpret_cast<uint16_t*>(unit + at) = (uint16_t)code;
  else if constexpr (!VALUES) *reinterpret_cast<uint32_t*>(unit + at) = code;
  else {
    *reinterpret_cast<uint16_t*>(unit + at) = (uint16_t)code;
    *reinterpret_cast<uint16_t*>(unit + v_byte<D>(tok, dim + 4)) = (uint16_t)(code >> 16);
  }
  if (lane % LG == 0) {
    __half* meta = reinterpret_cast<__half*>(unit + Geo<D>::CODES);
    const int i = VALUES ? v_meta<D>(tok, g) : k_meta<D>(tok, g);
    meta[i] = sh;
    meta[i + UNIT * Geo<D>::G] = mh;
  }
}

template <typename T, int D, bool Q4>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams p) {
  constexpr int E = D / 32;
  __shared__ float2 turn[D / 2];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.rot >> 1, hl = half / E;            // lanes of each rotated half
  pdl_trigger();
  pdl_wait();
  for (int i = threadIdx.x; i < half; i += 256) {
    const long ax = p.axes ? p.axes[i] : 0;
    const double a = (double)p.positions[ax * p.T + t] * (double)p.inv_freq[i];
    const double r = a - rint(a * 0.15915494309189535) * 6.283185307179586;     // one turn: 1 / 2 pi, 2 pi
    float s, c;
    sincosf((float)r, &s, &c);
    turn[i] = make_float2(c * p.mscale, s * p.mscale);
  }
  __syncthreads();
  const int slot = p.n_kv ? p.slots[t] : -1;
  const bool kept = slot >= 0 && slot < p.n_slots;
  // the token's unit of head 0 (units of a block: [head][unit])
  const int units = p.block_size / UNIT, block = kept ? p.by_block.div(slot) : 0, in = kept ? slot - block * p.block_size : 0;
  const size_t unit0 = unit_index(block, 0, p.n_kv, units, in / UNIT) * Geo<D>::BYTES;
  const int heads = p.n_q + 2 * p.n_kv, n_qk = p.n_q + p.n_kv;
  const int h_end = min(heads, (int)(blockIdx.y + 1) * p.heads_per_block);
  auto row_at = [&](int h) {
    return h < p.n_q ? (const T*)p.q + t * p.sq + (size_t)h * D : h < n_qk ? (const T*)p.k + t * p.sk + (size_t)(h - p.n_q) * D
                                                                         : (const T*)p.v + t * p.sv + (size_t)(h - n_qk) * D;
  };
  const bool first = lane < hl, turned = lane < 2 * hl;
  const int other = !turned ? lane : first ? lane + hl : lane - hl, pair = (first ? lane : lane - hl) * E;
  int h = blockIdx.y * p.heads_per_block + warp;
  Raw<T, E> next;
  if (h < h_end) next = load_raw<T, E>(row_at(h) + lane * E);
  for (; h < h_end; h += 8) {
    const Raw<T, E> now = next;
    if (h + 8 < h_end) next = load_raw<T, E>(row_at(h + 8) + lane * E);
    const bool is_q = h < p.n_q, is_v = h >= n_qk;
    float v[E];
    unpack_raw<T, E>(now, v);
    const T* nw = (const T*)(is_q ? p.q_norm : is_v ? nullptr : p.k_norm);
    if (nw || (is_v && p.v_unit)) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) ss += v[e] * v[e];
      const float rstd = rsqrtf(warp_sum(ss) / D + p.eps);
      if (nw) {
        float w[E];
        unpack_raw<T, E>(load_raw<T, E>(nw + lane * E), w);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] *= rstd * w[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] *= rstd;
      }
    }
    if (!is_v && half) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float o = __shfl_sync(0xffffffffu, v[e], other);
        if (turned) {
          const float2 cs = turn[pair + e];
          v[e] = fmaf(v[e], cs.x, first ? -o * cs.y : o * cs.y);
        }
      }
    }
    if (is_q) {
      store_row<T, E>((T*)p.q_out + ((size_t)t * p.n_q + h) * D + lane * E, v);
    } else if (kept) {
      const int hd = is_v ? h - n_qk : h - p.n_q;
      if constexpr (Q4) {
        uint8_t* unit = (uint8_t*)(is_v ? p.vcache : p.kcache) + unit0 + (size_t)hd * units * Geo<D>::BYTES;
        if (is_v) quantize_row<D, true>(v, unit, in % UNIT, lane);
        else quantize_row<D, false>(v, unit, in % UNIT, lane);
      } else {
        store_row<T, E>((T*)(is_v ? p.vcache : p.kcache) + ((size_t)slot * p.n_kv + hd) * D + lane * E, v);
      }
    }
  }
}

// Rows back out of the cache: a warp per slot, D / 8 lanes per row of a head (8 values a lane, 16 bytes of bf16), keys then values.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* kcache, const uint8_t* vcache, const int* slots, T* kout,
                                                       T* vout, long rows, int n_kv, int block_size, FastDiv by_block, long n_slots,
                                                       int warps_a_row) {
  constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;           // lanes of a row, rows of a warp
  pdl_trigger();
  pdl_wait();
  const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long r = w / warps_a_row;
  if (r >= rows) return;
  const int lane = threadIdx.x & 31, first = (int)(w - r * warps_a_row) * AT_ONCE + lane / LANES, dim = lane % LANES * 8;
  const int slot = slots[r];
  const bool kept = slot >= 0 && slot < n_slots;
  const int units = block_size / UNIT, block = kept ? by_block.div(slot) : 0, in = kept ? slot - block * block_size : 0, tok = in % UNIT;
  const size_t unit0 = unit_index(block, 0, n_kv, units, in / UNIT) * Geo<D>::BYTES;
  const int g = dim / GROUP, k_at = k_byte<D>(tok, dim), v_at = v_byte<D>(tok, dim), v_at2 = v_byte<D>(tok, dim + 4);
  const int k_num = Geo<D>::CODES + 2 * k_meta<D>(tok, g), v_num = Geo<D>::CODES + 2 * v_meta<D>(tok, g);
#pragma unroll 4
  for (int i = first; i < 2 * n_kv; i += AT_ONCE * warps_a_row) {
    const bool values = i >= n_kv;
    const int h = values ? i - n_kv : i;
    const uint8_t* unit = (values ? vcache : kcache) + unit0 + (size_t)h * units * Geo<D>::BYTES;
    uint32_t code = 0;
    float s = 0.f, m = 0.f;
    if (kept) {
      code = values ? *reinterpret_cast<const uint16_t*>(unit + v_at) | (uint32_t)*reinterpret_cast<const uint16_t*>(unit + v_at2) << 16
                    : *reinterpret_cast<const uint32_t*>(unit + k_at);
      const __half* num = reinterpret_cast<const __half*>(unit + (values ? v_num : k_num));
      s = __half2float(num[0]);
      m = __half2float(num[UNIT * Geo<D>::G]);
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++)                  // 2^23 + n less 2^23: n without a conversion
      v[e] = fmaf(__uint_as_float((code >> (4 * e) & 15u) | 0x4b000000u) - 8388608.f, s, m);
    store_row<T, 8>((values ? vout : kout) + ((size_t)r * n_kv + h) * D + dim, v);
  }
}

template <typename T, int D, bool Q4> int launch_append(AppendParams p, cudaStream_t st) {
  const int heads = p.n_q + 2 * p.n_kv;
  // A warp takes one head while there are few tokens (the card is filled by heads), and up to all the heads of its eighth
  // when there are many (the sines are then taken once per token).
  const int all = (heads + 7) / 8;
  int rounds = (int)((long)p.T * all / (148 * 8));
  rounds = rounds < 1 ? 1 : rounds > all ? all : rounds;
  p.heads_per_block = 8 * rounds;
  const dim3 grid(p.T, (heads + p.heads_per_block - 1) / p.heads_per_block);
  const cudaError_t e = launch_pdl(kv4_append_kernel<T, D, Q4>, grid, dim3(256), 0, st, p);
  if (e != cudaSuccess) return (int)e;
  EXO_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// q / k / v: the first head of token 0 of each part, `s*` elements between tokens (rows may be slices of a wider tensor;
// every row must start on E * sizeof(T) bytes, E = head_dim / 32).  `quantized`: the caches are 4-bit units, else rows of T.
EXO_API int exo_kv4_append(const void* q, const void* k, const void* v, long sq, long sk, long sv, const int* positions,
                           const int* axes, const float* inv_freq, float mscale, int n_q, int n_kv, int head_dim, int rot,
                           void* q_out, void* kcache, void* vcache, const int* slots, long n_slots, int block_size,
                           const void* q_norm, const void* k_norm, float eps, int T_, int dtype, int v_unit, int quantized,
                           cudaStream_t st) {
  if (T_ == 0 || n_q + 2 * n_kv == 0) return 0;
  if (T_ < 0 || rot < 0 || rot > head_dim || rot % (head_dim / 16) || block_size <= 0 || (quantized && block_size % UNIT) || n_slots > 0x7fffffffL) return -2;
  AppendParams p{q, k, v, sq, sk, sv, positions, axes, inv_freq, mscale, n_q, n_kv, rot, q_out, kcache, vcache, slots, n_slots,
                 block_size, FastDiv(block_size), q_norm, k_norm, eps, T_, v_unit, 0};
#define BY_CACHE(TT, DD) return quantized ? launch_append<TT, DD, true>(p, st) : launch_append<TT, DD, false>(p, st)
#define BY_DIM(TT)                       \
  if (head_dim == 64) BY_CACHE(TT, 64);   \
  if (head_dim == 128) BY_CACHE(TT, 128); \
  if (head_dim == 256) BY_CACHE(TT, 256); \
  return -2
  if (dtype == EXO_BF16) { BY_DIM(__nv_bfloat16); }
  if (dtype == EXO_F32) { BY_DIM(float); }
#undef BY_DIM
#undef BY_CACHE
  return -2;
}

// Rows of the cache at `slots` as T: kout / vout [rows, n_kv, D]; a slot outside the cache gives zeros.
EXO_API int exo_kv4_read(const void* kcache, const void* vcache, const int* slots, void* kout, void* vout, long rows, int n_kv,
                         int head_dim, int block_size, long n_slots, int dtype, cudaStream_t st) {
  if (rows == 0 || n_kv == 0) return 0;
  if (rows < 0 || block_size <= 0 || block_size % UNIT || n_slots > 0x7fffffffL) return -2;
  // all heads of a slot by one warp where slots fill the card, else spread
  const int most = (2 * n_kv * (head_dim / 8) + 31) / 32;
  const int warps = rows >= 148 * 32 ? 1 : most;
  const long blocks = (rows * warps + 7) / 8;
  if (blocks > 0x7fffffffL) return -2;
  const FastDiv by_block(block_size);
  cudaError_t e;
#define READ(TT, DD)                                                                                                          \
  e = launch_pdl(kv4_read_kernel<TT, DD>, dim3((unsigned)blocks), dim3(256), 0, st, (const uint8_t*)kcache,                    \
                 (const uint8_t*)vcache, slots, (TT*)kout, (TT*)vout, rows, n_kv, block_size, by_block, n_slots, warps)
#define BY_DIM(TT)                    \
  if (head_dim == 64) READ(TT, 64);   \
  else if (head_dim == 128) READ(TT, 128); \
  else if (head_dim == 256) READ(TT, 256); \
  else return -2
  if (dtype == EXO_BF16) { BY_DIM(__nv_bfloat16); }
  else if (dtype == EXO_F32) { BY_DIM(float); }
  else return -2;
#undef BY_DIM
#undef READ
  if (e != cudaSuccess) return (int)e;
  EXO_CHECK_LAUNCH();
  return 0;
}
