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
// What bounds it: bytes would (8192 tokens of 32 + 16 heads of 128: 178 MB, 27 us), but the kernel takes 70 us: some 140 instructions a
// row fill 58% of the issue slots (240 a row at first, with two 64-bit divisions by the block size and five IEEE divisions:
// 120 us), and the rest is the latency of a block's one pass (positions, sines, barrier, six rows a warp) with five blocks an
// SM.  Tried without gain: weight and rotation folded into two factors a dim (72 us), CTAs that walk tokens and fetch the next
// one's rows meanwhile (80 to 92), four tokens a block (102 with the read), four rows ahead (68 to 74), three to six blocks an SM.
// Copying the queries alone, with neither norm nor rotation, takes 36.  kv4_read: 12 to 16 us for 8192 slots of 16 heads (44 MB, 7 us).
#include <type_traits>
#include "kv4.cuh"

namespace {

using namespace kv4;

struct AppendParams {
  const void *q, *k, *v;                 // first q / k / v head of token 0
  long sq, sk, sv;                       // elements between tokens
  const int* positions;                  // [T], or [axes][T]
  const int* axes;                       // [rot / 2] position axis of each pair, or null
  int n_axes;                            // rows of positions; another axis than 0 .. n_axes - 1 is taken as the nearest of them
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
// `at` (and `at2`, for the upper half of 8 values): the bytes of the lane's codes; `num`: of its group's scale.
template <int D, bool VALUES> __device__ __forceinline__ void quantize_row(const float* x, uint8_t* unit, int at, int at2, int num, int lane) {
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
  if constexpr (E == 2) unit[at] = (uint8_t)code;
  else if constexpr (E == 4) *reinterpret_cast<uint16_t*>(unit + at) = (uint16_t)code;
  else if constexpr (!VALUES) *reinterpret_cast<uint32_t*>(unit + at) = code;
  else {
    *reinterpret_cast<uint16_t*>(unit + at) = (uint16_t)code;
    *reinterpret_cast<uint16_t*>(unit + at2) = (uint16_t)(code >> 16);
  }
  if (lane % LG == 0) {
    __half* meta = reinterpret_cast<__half*>(unit + num);
    meta[0] = sh;
    meta[UNIT * Geo<D>::G] = mh;
  }
}

template <typename T, int D, bool Q4>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendParams p) {
  constexpr int E = D / 32;
  __shared__ __align__(16) float2 turn[D / 2];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.rot >> 1, hl = half / E;            // lanes of each rotated half
  const int dim = lane * E, g = dim / GROUP, units = p.block_size / UNIT;
  const int h0 = blockIdx.y * p.heads_per_block, h1 = h0 + p.heads_per_block;
  pdl_trigger();
  pdl_wait();
  // The block's heads of a part (0 q, 1 k, 2 v) are heads [lo, hi) of the token; a warp has every eighth.  The first rows of all
  // three are on their way while the sines are taken.
  const int ends[4] = {0, p.n_q, p.n_q + p.n_kv, p.n_q + 2 * p.n_kv};
  const T* src[3] = {(const T*)p.q + t * p.sq + dim, (const T*)p.k + t * p.sk + dim, (const T*)p.v + t * p.sv + dim};
  int start[3], stop[3];
  Raw<T, E> raw[3];
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const int from = max(ends[i], h0);
    start[i] = from + ((warp - (from - h0)) & 7);
    stop[i] = min(ends[i + 1], h1);
    if (start[i] < stop[i]) raw[i] = load_raw<T, E>(src[i] + (size_t)(start[i] - ends[i]) * D);
  }
  for (int i = threadIdx.x; i < half; i += 256) {
    const long ax = p.axes ? min(max(p.axes[i], 0), p.n_axes - 1) : 0;
    const double a = (double)p.positions[ax * p.T + t] * (double)p.inv_freq[i];
    const double r = a - rint(a * 0.15915494309189535) * 6.283185307179586;     // one turn: 1 / 2 pi, 2 pi
    float s, c;
    sincosf((float)r, &s, &c);
    turn[i] = make_float2(c * p.mscale, s * p.mscale);
  }
  __syncthreads();
  const bool first = lane < hl, turned = lane < 2 * hl;
  const int other = !turned ? lane : first ? lane + hl : lane - hl;
  const float2* cs = turn + (turned ? (first ? lane : lane - hl) * E : 0);
  const int slot = p.n_kv ? p.slots[t] : -1;
  const bool kept = slot >= 0 && slot < p.n_slots;
  // the token's unit of head 0 (units of a block: [head][unit])
  const int block = kept ? p.by_block.div(slot) : 0, in = kept ? slot - block * p.block_size : 0, tok = in % UNIT;
  const size_t unit0 = unit_index(block, 0, p.n_kv, units, in / UNIT) * Geo<D>::BYTES;

  auto part = [&](auto kind) {
    constexpr int KIND = decltype(kind)::value;
    const int lo = ends[KIND], to = stop[KIND];
    int h = start[KIND];
    if (h >= to) return;
    const T* nw = (const T*)(KIND == 0 ? p.q_norm : KIND == 1 ? p.k_norm : nullptr);
    const bool normed = KIND == 2 ? p.v_unit != 0 : nw != nullptr;
    Raw<T, E> weight, next = raw[KIND];
    if (KIND != 2 && nw) weight = load_raw<T, E>(nw + dim);
    const int at = KIND == 1 ? k_byte<D>(tok, dim) : v_byte<D>(tok, dim), at2 = v_byte<D>(tok, dim + (E == 8 ? 4 : 0));
    const int num = Geo<D>::CODES + 2 * (KIND == 1 ? k_meta<D>(tok, g) : v_meta<D>(tok, g));
    [[maybe_unused]] uint8_t* units0 = (uint8_t*)(KIND == 1 ? p.kcache : p.vcache) + unit0;
    T* rows0 = KIND == 0 ? (T*)p.q_out + (size_t)t * p.n_q * D + dim : (T*)(KIND == 1 ? p.kcache : p.vcache) + (size_t)(kept ? slot : 0) * p.n_kv * D + dim;
    for (; h < to; h += 8) {
      float v[E];
      unpack_raw<T, E>(next, v);
      if (h + 8 < to) next = load_raw<T, E>(src[KIND] + (size_t)(h + 8 - lo) * D);
      if (normed) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) ss = fmaf(v[e], v[e], ss);
        const float rstd = rsqrtf(warp_sum(ss) * (1.f / D) + p.eps);
        if constexpr (KIND == 2) {
#pragma unroll
          for (int e = 0; e < E; e++) v[e] *= rstd;
        } else {
          float w[E];
          unpack_raw<T, E>(weight, w);
#pragma unroll
          for (int e = 0; e < E; e++) v[e] *= rstd * w[e];
        }
      }
      if (KIND != 2 && half) {
        float o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = __shfl_sync(0xffffffffu, v[e], other);
        if (turned) {
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float4 c = *reinterpret_cast<const float4*>(cs + e);       // (cos, sin) of two pairs
            v[e] = fmaf(v[e], c.x, first ? -o[e] * c.y : o[e] * c.y);
            v[e + 1] = fmaf(v[e + 1], c.z, first ? -o[e + 1] * c.w : o[e + 1] * c.w);
          }
        }
      }
      if constexpr (KIND == 0) {
        store_row<T, E>(rows0 + (size_t)h * D, v);
      } else if (kept) {
        if constexpr (Q4) quantize_row<D, KIND == 2>(v, units0 + (size_t)(h - lo) * units * Geo<D>::BYTES, at, at2, num, lane);
        else store_row<T, E>(rows0 + (size_t)(h - lo) * D, v);
      }
    }
  };
  part(std::integral_constant<int, 0>{});
  part(std::integral_constant<int, 1>{});
  part(std::integral_constant<int, 2>{});
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
  // A warp takes one head while there are few tokens (the card is filled by heads), and up to all the heads of its eighth when
  // there are many (the sines are then taken once per token).  32 + 16 heads of 128, us, one / all: 16 tokens 3.6 / 5.6, 400 9.2 / 8.2,
  // 1000 18.4 / 12.3, 8192 132 / 67; this rule 3.1, 7.7, 12.3, 67.  Four tokens a block took a sixth fewer instructions and a
  // third more time: fewer rows in flight.
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

// An AppendCall.  q / k / v: the first head of token 0 of each part, `s*` elements between tokens (rows may be slices of a wider
// tensor; every row must start on E * sizeof(T) bytes, E = head_dim / 32).  `quantized`: the caches are 4-bit units, else rows of T.
EXO_API int exo_kv4_append(const void* call, int bytes, cudaStream_t st) {
  AppendCall c;
  if (!unpack_call(c, call, bytes)) return -2;
  if (c.T == 0 || c.n_q + 2 * c.n_kv == 0) return 0;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return -2;
  if (c.T < 0 || c.n_q < 0 || c.n_kv < 0 || c.rot < 0 || c.rot > c.head_dim || c.rot % (c.head_dim / 16) || c.block_size <= 0 ||
      (c.quantized && c.block_size % UNIT) || c.n_slots > 0x7fffffffL || (c.axes && c.n_axes <= 0)) return -2;
  AppendParams p{c.q, c.k, c.v, c.sq, c.sk, c.sv, c.positions, c.axes, c.n_axes, c.inv_freq, c.mscale, c.n_q, c.n_kv, c.rot, c.q_out, c.kcache,
                 c.vcache, c.slots, c.n_slots, c.block_size, FastDiv(c.block_size), c.q_norm, c.k_norm, c.eps, c.T, c.v_unit, 0};
  const int head_dim = c.head_dim, dtype = c.dtype;
  const bool quantized = c.quantized;
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

// A ReadCall: rows of the cache at `slots` as T: kout / vout [rows, n_kv, D]; a slot outside the cache gives zeros.
EXO_API int exo_kv4_read(const void* call, int bytes, cudaStream_t st) {
  ReadCall c;
  if (!unpack_call(c, call, bytes)) return -2;
  const long rows = c.rows;
  const int n_kv = c.n_kv, head_dim = c.head_dim, dtype = c.dtype;
  if (rows == 0 || n_kv == 0) return 0;
  if (rows < 0 || n_kv < 0 || c.block_size <= 0 || c.block_size % UNIT || c.n_slots > 0x7fffffffL) return -2;
  // all heads of a slot by one warp where slots fill the card, else spread (8 heads of 128; us, one warp / spread: 1000 slots
  // 7.2 / 5.1, 2048 7.7 / 7.7, 4096 9.2 / 12.3, 8192 13.8 / 22.0)
  const int most = (2 * n_kv * (head_dim / 8) + 31) / 32;
  const int warps = rows >= 148 * 16 ? 1 : most;
  const long blocks = (rows * warps + 7) / 8;
  if (blocks > 0x7fffffffL) return -2;
  const FastDiv by_block(c.block_size);
  cudaError_t e;
#define READ(TT, DD)                                                                                                          \
  e = launch_pdl(kv4_read_kernel<TT, DD>, dim3((unsigned)blocks), dim3(256), 0, st, (const uint8_t*)c.kcache,                  \
                 (const uint8_t*)c.vcache, c.slots, (TT*)c.kout, (TT*)c.vout, rows, n_kv, c.block_size, by_block, c.n_slots, warps)
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
