// Attention of fp32 queries over a 4-bit KV cache, on the CUDA cores: any number of queries per sequence, any number of heads per
// key head.  (fp32 models are for checking others by: nothing here is rounded to 16 bits.)  One warp owns one query row and up to four heads that share a key head, its lanes split the head dim (two neighbouring dims and D / 64 such pairs), and
// keys are visited in order with a running maximum and sum.
#include "kv4.cuh"

namespace {

using namespace kv4;

__device__ __forceinline__ float sink_at(const void* sinks, int dtype, int h) {
  return dtype == EXO_BF16 ? __bfloat162float(((const __nv_bfloat16*)sinks)[h]) : ((const float*)sinks)[h];
}

template <int D, int GT>
__global__ void __launch_bounds__(128)
kv4_ragged_kernel(const float* __restrict__ q, const uint8_t* __restrict__ kcache, const uint8_t* __restrict__ vcache,
                  const int* __restrict__ tables, const int* __restrict__ seq_lens, const int* __restrict__ cu_q,
                  float* __restrict__ out, float scale, int T_, int B, int Hq, int Hkv, int n_blocks, int max_blocks, int block_size,
                  int window, const void* sinks, int sink_dtype) {
  constexpr int P = D / 64;                     // pairs of dims a lane holds: dims 64 i + 2 lane, + 1
  const int per = Hq / Hkv, tiles = (per + GT - 1) / GT;
  const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long t = w / (Hkv * tiles);
  if (t >= T_) return;
  const int rem = (int)(w % (Hkv * tiles)), kvh = rem / tiles, h0 = kvh * per + (rem % tiles) * GT;
  const int nh = min(GT, (kvh + 1) * per - h0);
  const int b = seq_of_row(cu_q, B, (int)t);
  float qr[GT][2 * P], acc[GT][2 * P], m[GT], l[GT];
#pragma unroll
  for (int i = 0; i < GT; i++) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < P; j++) {
      qr[i][2 * j] = qr[i][2 * j + 1] = acc[i][2 * j] = acc[i][2 * j + 1] = 0.f;
      if (i < nh) {
        const float* qp = q + ((size_t)t * Hq + h0 + i) * D + 64 * j + 2 * lane;
        qr[i][2 * j] = qp[0] * scale;
        qr[i][2 * j + 1] = qp[1] * scale;
      }
    }
  }
  int lo = 0, hi = 0;                           // keys [lo, hi) are visible
  if (b >= 0) {
    const int n = (int)min((long)seq_lens[b], (long)max_blocks * block_size);
    const int pos = seq_lens[b] - (cu_q[b + 1] - cu_q[b]) + ((int)t - cu_q[b]);
    hi = min(n, pos + 1);
    lo = window > 0 ? max(0, pos + 1 - window) : 0;
  }
  const int units = block_size / UNIT;
  for (int key = lo; key < hi; key++) {
    const int blk = min(max(tables[(size_t)b * max_blocks + key / block_size], 0), n_blocks - 1);
    const size_t u = unit_index(blk, kvh, Hkv, units, key % block_size / UNIT) * Geo<D>::BYTES;
    const int tok = key % UNIT;
    const uint8_t *ku = kcache + u, *vu = vcache + u;
    const __half *km = reinterpret_cast<const __half*>(ku + Geo<D>::CODES), *vm = reinterpret_cast<const __half*>(vu + Geo<D>::CODES);
    float kf[2 * P], vf[2 * P];
#pragma unroll
    for (int j = 0; j < P; j++) {
      const int dim = 64 * j + 2 * lane, g = dim / GROUP;
      const uint32_t kc = ku[k_byte<D>(tok, dim)], vc = vu[v_byte<D>(tok, dim)];
      const int ki = k_meta<D>(tok, g), vi = v_meta<D>(tok, g);
      const float ks = __half2float(km[ki]), kl = __half2float(km[ki + UNIT * Geo<D>::G]);
      const float vs = __half2float(vm[vi]), vl = __half2float(vm[vi + UNIT * Geo<D>::G]);
      kf[2 * j] = fmaf((float)(kc & 15), ks, kl);
      kf[2 * j + 1] = fmaf((float)(kc >> 4), ks, kl);
      vf[2 * j] = fmaf((float)(vc & 15), vs, vl);
      vf[2 * j + 1] = fmaf((float)(vc >> 4), vs, vl);
    }
#pragma unroll
    for (int i = 0; i < GT; i++) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * P; j++) s += qr[i][j] * kf[j];
      s = warp_sum(s);
      const float mn = fmaxf(m[i], s), use = mn == -INFINITY ? 0.f : mn;
      const float corr = expf(m[i] - use), pr = expf(s - use);
      l[i] = l[i] * corr + pr;
#pragma unroll
      for (int j = 0; j < 2 * P; j++) acc[i][j] = acc[i][j] * corr + pr * vf[j];
      m[i] = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < GT; i++) {
    if (i >= nh) continue;
    float lt = l[i], sc = 1.f;
    if (sinks && b >= 0) {
      const float sk = sink_at(sinks, sink_dtype, h0 + i), mn = fmaxf(m[i], sk);
      sc = m[i] == -INFINITY ? 0.f : expf(m[i] - mn);
      lt = l[i] * sc + (sk == -INFINITY ? 0.f : expf(sk - mn));
    }
    const float inv = lt == 0.f ? 0.f : sc / lt;              // a row that sees nothing is zero; NaN stays NaN
#pragma unroll
    for (int j = 0; j < P; j++) {
      float* op = out + ((size_t)t * Hq + h0 + i) * D + 64 * j + 2 * lane;
      op[0] = acc[i][2 * j] * inv;
      op[1] = acc[i][2 * j + 1] * inv;
    }
  }
}

}  // namespace

// An AttnCall with fp32 q and out.
EXO_API int exo_kv4_attn_ragged(const void* call, int bytes, cudaStream_t st) {
  AttnCall c;
  if (!unpack_call(c, call, bytes)) return -2;
  const int T_ = c.T, B = c.B, Hq = c.Hq, Hkv = c.Hkv, D = c.D, n_blocks = c.n_blocks, max_blocks = c.max_blocks, block_size = c.block_size;
  if (T_ == 0) return 0;
  if (T_ < 0 || B <= 0 || Hkv <= 0 || Hq % Hkv || block_size <= 0 || block_size % UNIT || n_blocks <= 0) return -2;
  const int per = Hq / Hkv, GT = per >= 4 ? 4 : per >= 2 ? 2 : 1;
  const long warps = (long)T_ * Hkv * ((per + GT - 1) / GT);
  const unsigned blocks = (unsigned)((warps + 3) / 4);
#define LAUNCH(DD, GG)                                                                                                         \
  kv4_ragged_kernel<DD, GG><<<blocks, 128, 0, st>>>((const float*)c.q, (const uint8_t*)c.kcache, (const uint8_t*)c.vcache, c.tables,  \
                                                    c.seq_lens, c.cu_q, (float*)c.out, c.scale, T_, B, Hq, Hkv, n_blocks, max_blocks, \
                                                    block_size, c.window, c.sinks, c.sink_dtype)
#define BY_G(DD)                   \
  if (GT == 4) LAUNCH(DD, 4);      \
  else if (GT == 2) LAUNCH(DD, 2); \
  else LAUNCH(DD, 1)
  if (D == 64) { BY_G(64); }
  else if (D == 128) { BY_G(128); }
  else if (D == 256) { BY_G(256); }
  else return -2;
#undef BY_G
#undef LAUNCH
  EXO_CHECK_LAUNCH();
  return 0;
}
