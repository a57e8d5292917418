// What writes a 4-bit KV cache, and what reads its rows back.
//
// The append takes the fused q/k/v projection of T tokens and does, per head of a token and without leaving registers:
//   x <- x * rsqrt(mean x^2 + eps) * w          (q and k, optional)
//   (x_i, x_{i+r}) <- rotation by p[axis(i)] * f_i   (q and k; r = half the rotated dims; one or several position axes)
//   q: stored;  k, v: 32-dim groups -> m = fp16 rounded down of the least value, s = fp16 rounded up of (max - m) / 15,
//   codes rint((x - m) / s), stored in the operand order of kv4.cuh.
// Nothing is rounded between the three steps.  The quotients are IEEE divisions: bf16 rows hit exact halves of a step
// often (their values have few bits), and a product with a rounded reciprocal would decide those ties at random.
//
// One block = one token, a warp = one head at a time.  The sines and cosines of a token are the same for all its heads: they
// are taken once per block (angle in 64 bits, reduced to one turn, then the fp32 functions) and kept in shared memory.
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
  const void *q_norm, *k_norm;
  float eps;
  int T, v_unit, heads_per_block;
};

template <typename T, int E> __device__ __forceinline__ void load_row(const T* p, float* v) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (E == 2) {
      const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(p);
      v[0] = __low2float(a); v[1] = __high2float(a);
    } else if constexpr (E == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
      v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 u = *reinterpret_cast<const float2*>(p + e);
      v[e] = u.x; v[e + 1] = u.y;
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

// Quantises the row that a warp holds (E neighbouring dims a lane) into token `tok` of a unit.
template <int D, bool VALUES> __device__ __forceinline__ void quantize_row(const float* x, uint8_t* unit, int tok, int lane) {
  constexpr int E = D / 32, LG = GROUP / E;      // lanes of a group
  bool nan = false;
  float v[E], lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e++) {
    nan |= x[e] != x[e];
    v[e] = fminf(fmaxf(x[e], -LARGEST), LARGEST);
    lo = fminf(lo, v[e]);
    hi = fmaxf(hi, v[e]);
  }
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  nan = __any_sync(0xffffffffu, nan);            // one NaN makes the whole row NaN
  __half mh = __float2half_rd(lo);
  const float m = __half2float(mh);
  __half sh = __float2half_ru(__fdiv_rn(hi - m, 15.f));
  const float s = __half2float(sh);
  uint32_t code = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float n = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(v[e] - m, s)), 0.f), 15.f) : 0.f;
    code |= (uint32_t)n << (4 * e);
  }
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
  const long slot = p.n_kv ? p.slots[t] : -1;
  const bool kept = slot >= 0 && slot < p.n_slots;
  const int heads = p.n_q + 2 * p.n_kv;
  const int h_end = min(heads, (int)(blockIdx.y + 1) * p.heads_per_block);
  for (int h = blockIdx.y * p.heads_per_block + warp; h < h_end; h += 8) {
    const bool is_q = h < p.n_q, is_k = !is_q && h < p.n_q + p.n_kv;
    const int hd = is_q ? h : is_k ? h - p.n_q : h - p.n_q - p.n_kv;
    const T* src = is_q ? (const T*)p.q + t * p.sq : is_k ? (const T*)p.k + t * p.sk : (const T*)p.v + t * p.sv;
    float v[E];
    load_row<T, E>(src + (size_t)hd * D + lane * E, v);
    const T* nw = (const T*)(is_q ? p.q_norm : is_k ? p.k_norm : nullptr);
    if (nw || (!is_q && !is_k && p.v_unit)) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) ss += v[e] * v[e];
      const float rstd = rsqrtf(warp_sum(ss) / D + p.eps);
      float w[E];
#pragma unroll
      for (int e = 0; e < E; e++) w[e] = 1.f;
      if (nw) load_row<T, E>(nw + lane * E, w);
#pragma unroll
      for (int e = 0; e < E; e++) v[e] *= rstd * w[e];
    }
    if ((is_q || is_k) && half) {
      const bool first = lane < hl, turned = lane < 2 * hl;
      const int other = !turned ? lane : first ? lane + hl : lane - hl;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float o = __shfl_sync(0xffffffffu, v[e], other);
        if (turned) {
          const float2 cs = turn[(first ? lane : lane - hl) * E + e];
          v[e] = first ? v[e] * cs.x - o * cs.y : v[e] * cs.x + o * cs.y;
        }
      }
    }
    if (is_q) {
      store_row<T, E>((T*)p.q_out + ((size_t)t * p.n_q + hd) * D + lane * E, v);
    } else if (kept) {
      void* cache = is_k ? p.kcache : p.vcache;
      if constexpr (Q4) {
        const int in = (int)(slot % p.block_size);
        uint8_t* unit = (uint8_t*)cache + unit_index(slot / p.block_size, hd, p.n_kv, p.block_size / UNIT, in / UNIT) * Geo<D>::BYTES;
        if (is_k) quantize_row<D, false>(v, unit, in % UNIT, lane);
        else quantize_row<D, true>(v, unit, in % UNIT, lane);
      } else {
        store_row<T, E>((T*)cache + ((size_t)slot * p.n_kv + hd) * D + lane * E, v);
      }
    }
  }
}

// Rows back out of the cache: a warp per (slot, head, keys or values).
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* kcache, const uint8_t* vcache, const int* slots, T* kout,
                                                       T* vout, long rows, int n_kv, int block_size, long n_slots) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= rows * n_kv * 2) return;
  const bool values = w & 1;
  const long r = (w >> 1) / n_kv;
  const int h = (int)((w >> 1) % n_kv);
  const long slot = slots[r];
  float v[E];
#pragma unroll
  for (int e = 0; e < E; e++) v[e] = 0.f;
  if (slot >= 0 && slot < n_slots) {
    const int in = (int)(slot % block_size), tok = in % UNIT, dim = lane * E, g = dim / GROUP;
    const uint8_t* unit = (values ? vcache : kcache) + unit_index(slot / block_size, h, n_kv, block_size / UNIT, in / UNIT) * Geo<D>::BYTES;
    const int at = values ? v_byte<D>(tok, dim) : k_byte<D>(tok, dim);
    const __half* meta = reinterpret_cast<const __half*>(unit + Geo<D>::CODES) + (values ? v_meta<D>(tok, g) : k_meta<D>(tok, g));
    uint32_t code;
    if constexpr (E == 2) code = unit[at];
    else if constexpr (E == 4) code = *reinterpret_cast<const uint16_t*>(unit + at);
    else code = values ? *reinterpret_cast<const uint16_t*>(unit + at) |
                             (uint32_t)*reinterpret_cast<const uint16_t*>(unit + v_byte<D>(tok, dim + 4)) << 16
                       : *reinterpret_cast<const uint32_t*>(unit + at);
    const float s = __half2float(meta[0]), m = __half2float(meta[UNIT * Geo<D>::G]);
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = fmaf((float)((code >> (4 * e)) & 15), s, m);
  }
  store_row<T, E>((values ? vout : kout) + ((size_t)r * n_kv + h) * D + lane * E, v);
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
  if (T_ < 0 || rot < 0 || rot > head_dim || rot % (head_dim / 16) || (quantized && block_size % UNIT)) return -2;
  AppendParams p{q, k, v, sq, sk, sv, positions, axes, inv_freq, mscale, n_q, n_kv, rot, q_out, kcache, vcache, slots, n_slots,
                 block_size, q_norm, k_norm, eps, T_, v_unit, 0};
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
  const long blocks = (rows * n_kv * 2 + 7) / 8;
  if (rows < 0 || blocks > 0x7fffffffL || block_size % UNIT) return -2;
  cudaError_t e;
#define READ(TT, DD)                                                                                                          \
  e = launch_pdl(kv4_read_kernel<TT, DD>, dim3((unsigned)blocks), dim3(256), 0, st, (const uint8_t*)kcache,                    \
                 (const uint8_t*)vcache, slots, (TT*)kout, (TT*)vout, rows, n_kv, block_size, n_slots)
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
