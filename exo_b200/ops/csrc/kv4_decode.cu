// Attention of single query rows over a 4-bit KV cache, split over the keys (bf16 queries).
//
// What bounds it: 10 D bytes per 16 keys and key head, each used by Hq / Hkv query heads: HBM, if the 4-bit codes become
// matrix operands cheaply enough (at 6.5 TB/s an SM receives some 37 codes a clock and can issue 128 lane instructions).
// So no code is ever turned into its value.  With a code n and a group's scale s and least value m,
//   q . k = sum_g s_g (q_g . n_g) + sum_g m_g (1 . q_g)          o = sum_j p_j (s_jg n_j + m_jg)
// * codes enter the matrix instructions as fp16 SUBNORMALS: a nibble masked out of a word at bit 0 (bit 4) is the fp16 number
//   n 2^-24 (n 2^-20), exactly, without conversion, offset or correction: one AND for two codes, one shift for eight.  The
//   factors are taken out of the queries (2^-4 of those dims that meet nibbles at bit 4) and of the sums at the end.
// * S^T = K Q^T and O^T = V^T P^T, keys (dims) as the 16 rows and query heads as the 8 columns of m16n8k16: codes are the A
//   operand, built in registers, and eight heads fill a tile.  tcgen05 would want the codes expanded to bytes or halves in
//   shared memory or TMEM, which costs the instructions that the subnormals save, for tiles of 128 rows where 8 heads are.
// * s_g of the keys multiplies the group's fp32 partial sums; s_jg of the values multiplies p_j (fp16, 2^-11: the group's P
//   operand).  m_g (1 . q_g) and p_j m_jg are one more matrix instruction each, fp16 with q's sums split in two parts.
// * P reaches the B operand's layout with movmatrix, not shared memory.
//
// fp16 holds p only within a range: p is kept relative to R = (a maximum seen so far, of which newer ones may be up to 2^8
// over) - x, where 2^x brings p and p s_jg to at most 2^15, x from the largest scale met.  A unit that breaks either bound
// (one vote a unit) moves R and rescales the sums; the common unit has no shuffle and no rescale.  Queries are scaled per
// head to 2^9..2^10 by a power of two.
//
// Work.  All (row, head group, block of one or two 16-key units per warp) are put in line, EXTRA blocks in front of each row and
// head group for what it costs beside its keys, and the line is cut into equal shares, one per CTA: ragged lengths balance to a
// block (rows of a few blocks are not cut: what a cut costs, some 2.5 us, is more than they take).  Each of a CTA's warps takes
// its units of a block, fetched by asynchronous copies into the warp's own ring (10 D bytes of keys and of values a unit: what is
// in flight per SM covers the HBM latency), runs its own softmax and meets the others once per row and head group.  Plain 16-byte cp.async, a line per lane, costs a third of the instructions that two
// bulk copies of one lane cost here (address, expect, two issues a unit), needs no barrier, and streams as fast (6.4 TB/s of
// 1280-byte units in a probe with 16 warps an SM; one warp that issues bulk copies for others: 3.3).
// A row that a CTA holds whole is finished there.  A row cut by a share's end leaves fp32 parts; the last CTA to arrive at the
// row's ticket adds them in the order of the shares (so the result does not depend on timing), in two levels where there are
// more than eight.  A second kernel for this cost 5 to 8 us a call.
//
// Measured (of 6.5 TB/s): 64 rows x 4096 keys, 8 key heads of 128 with 4 query heads each, 74 us (0.69); 32 x 2048, 30 us (0.43; some
// 8 us are launch, first loads and the joining of parts); one row x 131072 keys, 8 query heads a key head, 45 us (0.57);
// 64 x 6000 keys, 16 query heads a key head, 80 us (0.46: two tiles of heads double the instructions a unit, and 168 registers
// leave 12 warps an SM).  Half the issue slots and 40% of the ALU are used: 16 warps an SM at 128 registers hide no more.
#include "kv4.cuh"

namespace {

using namespace kv4;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int HEADROOM = 8;       // a score may pass its reference maximum by 2^8 before the sums are rescaled

struct Params {
  const __nv_bfloat16* q;         // [T, Hq, D]
  const uint8_t *kcache, *vcache;
  const int *tables, *seq_lens, *cu_q;
  __nv_bfloat16* out;
  float* parts;                   // [grid][2][NH][D] unnormalised outputs of rows cut by a share's ends: 0 the row that came
                                  // in from the share before, 1 the row that goes on in the next
  float2* part_ml;                // [grid][2][NH] (R, l)
  int* tickets;                   // [3][grid] zeros, and zeros again when the kernel ends
  const void* sinks;
  float scale_log2;
  int T, B, Hq, Hkv, n_blocks, max_blocks, units_per_block, window, sink_dtype, groups;   // groups: head groups of a key head
};

__device__ __forceinline__ float sink_log2(const Params& p, int h) {
  return (p.sink_dtype == EXO_BF16 ? __bfloat162float(((const __nv_bfloat16*)p.sinks)[h]) : ((const float*)p.sinks)[h]) * LOG2E;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                    const float* c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ bool above(uint32_t a, uint32_t b) {      // either half of a over b's
  const __half2 r = __hgt2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r) != 0;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t a) { return __half22float2(*reinterpret_cast<__half2*>(&a)); }
__device__ __forceinline__ void async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N> __device__ __forceinline__ void lds(uint32_t* v, const uint8_t* p) {      // N words
  if constexpr (N == 1) {
    v[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = u.x; v[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + 4 * i);
      v[i] = u.x; v[i + 1] = u.y; v[i + 2] = u.z; v[i + 3] = u.w;
    }
  }
}

// Keys that a query row sees, as units.
struct Row { int b, lo, hi, u0, nblk; };
// which of keys `key`, `key + 1` are seen, as a mask of a half2's halves
__device__ __forceinline__ uint32_t seen_pair(const Row& r, int key) {
  return (key >= r.lo && key < r.hi ? 0xffffu : 0u) | (key + 1 >= r.lo && key + 1 < r.hi ? 0xffff0000u : 0u);
}
template <int BLOCK> __device__ __forceinline__ Row row_of(const Params& p, int t) {
  Row r{-1, 0, 0, 0, 0};
  int first = t, q_len = 1, n = 0;
  bool one = false;                              // the plain decode step: row t is sequence t (its three numbers load together)
  if (t < p.B) {
    const int c0 = p.cu_q[t], c1 = p.cu_q[t + 1];
    n = p.seq_lens[t];
    one = c0 == t && c1 == t + 1;
  }
  r.b = t;
  if (!one) {
    r.b = seq_of_row(p.cu_q, p.B, t);
    if (r.b < 0) return r;
    first = p.cu_q[r.b];
    q_len = p.cu_q[r.b + 1] - first;
    n = p.seq_lens[r.b];
  }
  const int pos = n - q_len + (t - first);
  r.hi = (int)min((long)pos + 1, (long)p.max_blocks * p.units_per_block * UNIT);
  r.lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
  if (r.hi <= r.lo) return r;
  r.u0 = r.lo / UNIT;
  r.nblk = ((r.hi + UNIT - 1) / UNIT - r.u0 + BLOCK - 1) / BLOCK;
  return r;
}

constexpr int EXTRA = 3;          // what a row and head group costs beside its blocks (queries in, sums out), in blocks
constexpr int SMALL = 4;          // rows of so few blocks belong whole to the share in which they begin
constexpr int FAN = 8;            // parts that are added at once
constexpr uint32_t NONE = 0xffffffffu, STOP = 0xfffffffeu;

// A place in the line.  `start` is where the row and head group begins, counted from the share's begin.
template <int BLOCK> struct Cursor {
  Row r;
  int t, hh, blk, start;
  __device__ __forceinline__ bool small() const { return r.nblk <= SMALL; }
  // the block behind the last that the share of `end` holds of this row (0 or less: it holds none)
  __device__ __forceinline__ int blocks_to(int end) const { return small() ? (start < end ? r.nblk : 0) : min(r.nblk, end - start - EXTRA); }
  __device__ __forceinline__ bool next_item(const Params& p, int HH, int end) {      // false: the share ends first
    start += r.nblk + EXTRA;
    blk = 0;
    if (start >= end) return false;
    if (++hh == HH) {
      hh = 0;
      do r = row_of<BLOCK>(p, ++t); while (r.nblk == 0);          // (the line goes on, so there is one)
    }
    return blocks_to(end) > 0;
  }
};

template <int D, int NT> struct Cfg {
  static constexpr int NH = 8 * NT;                            // heads of a group
  // Two CTAs an SM.  Registers decide on the warps: a scheduler holds 4 warps of 128 registers, or 3 of 168 (sums of 256 dims, or
  // of 16 heads of 128).  Two units at a time give a warp two chains of instructions to interleave and halve what a turn of the
  // loop costs; the shared memory of 256-wide heads allows for one.
  static constexpr int WARPS = D == 256 || (D == 128 && NT == 2) ? 6 : 8;
  static constexpr int CTAS = 2;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int PAIR = D == 256 ? 1 : 2;                // units of a warp in a block
  static constexpr int BLOCK = WARPS * PAIR;                   // units of a block
  static constexpr int STAGES = D == 64 ? 3 : 2;               // (two CTAs have 113 KB of shared memory each)
  static constexpr int U = Geo<D>::BYTES;
  static constexpr int STAGE = PAIR * 2 * U;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int ODIM = 64;                              // dims that the warps exchange at a time
  static constexpr int OROW = ODIM + 4;                        // floats of a head's row: 16 bytes of padding spread the banks
  static constexpr int OBUF = WARPS * NH * OROW * 4;
  static constexpr int SMEM = RING + OBUF + WARPS * NH * 8;
};

template <int D, int NT>
__global__ void __launch_bounds__(Cfg<D, NT>::THREADS, Cfg<D, NT>::CTAS) kv4_decode_kernel(const Params p) {
  using C = Cfg<D, NT>;
  using Gm = Geo<D>;
  constexpr int G = Gm::G, PER = Gm::PER, HALVES = Gm::HALVES, U = C::U, NH = C::NH, WARPS = C::WARPS, THREADS = C::THREADS, BLOCK = C::BLOCK, PAIR = C::PAIR;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * C::STAGES * C::STAGE;
  float* obuf = reinterpret_cast<float*>(smem + C::RING);
  float2* mlbuf = reinterpret_cast<float2*>(smem + C::RING + C::OBUF);
  __shared__ Cursor<BLOCK> places[WARPS][32];
  __shared__ int arrived;
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's share of the line (the launcher has made sure that the line fits 32 bits) ----
  const int HH = p.Hkv * p.groups, per_kv = p.Hq / p.Hkv;
  const int n0 = lane < p.T ? row_of<BLOCK>(p, lane).nblk : 0;     // of the first 32 rows
  auto blocks = [&](int t0) { return t0 == 0 ? n0 : t0 + lane < p.T ? row_of<BLOCK>(p, t0 + lane).nblk : 0; };
  uint32_t total = 0;
  for (int t0 = 0; t0 < p.T; t0 += 32) {
    const int n = blocks(t0);
    total += __reduce_add_sync(0xffffffffu, n ? n + EXTRA : 0);
    // rows that see nothing belong to no share
    for (unsigned none = __ballot_sync(0xffffffffu, t0 + lane < p.T && n == 0); none; none &= none - 1) {
      const int tz = t0 + __ffs(none) - 1;
      if (tz % gridDim.x == blockIdx.x)
        for (int i = threadIdx.x; i < p.Hq * D / 8; i += THREADS)
          reinterpret_cast<uint4*>(p.out + (size_t)tz * p.Hq * D)[i] = make_uint4(0, 0, 0, 0);
    }
  }
  total *= HH;
  const uint32_t share = (total + gridDim.x - 1) / gridDim.x, begin = share * blockIdx.x;
  if (begin >= total) return;
  const int end = min(total - begin, share);                      // counted from begin, as all places below
  Cursor<BLOCK> cur;
  {
    uint32_t base = 0;
    int t0 = 0;
    for (;; t0 += 32) {
      uint32_t n = blocks(t0);
      if (n) n += EXTRA;
      const uint32_t mine = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += up;
      }
      const unsigned over = __ballot_sync(0xffffffffu, (base + n) * HH > begin);
      if (over) {
        const int w = __ffs(over) - 1;
        cur.t = t0 + w;
        base += __shfl_sync(0xffffffffu, n - mine, w);
        break;
      }
      base += __shfl_sync(0xffffffffu, n, 31);
    }
    cur.r = row_of<BLOCK>(p, cur.t);
    const uint32_t in = begin - base * HH, len = cur.r.nblk + EXTRA;
    cur.hh = in / len;
    cur.start = -(int)(in % len);
    cur.blk = max(-cur.start - EXTRA, 0);
    if (cur.small() && cur.start < 0) {
      if (!cur.next_item(p, HH, end)) return;
    } else if (cur.blocks_to(end) <= cur.blk) {
      return;                                     // the share holds no block
    }
  }

  // ---- the ring.  Units are looked up 32 blocks at a time, a block a lane, and a round before they are copied (a page number
  // that misses the caches costs as much as several blocks); the lanes' places in the line wait in shared memory.
  int copied = 0;                                 // blocks looked at
  uint32_t unit_now[PAIR], unit_next[PAIR];
  auto look = [&](int by) {                       // the units `by` blocks behind this lane's place
    Cursor<BLOCK> c = places[warp][lane];
    unit_next[0] = STOP;
    if (c.blk < 0) return;
    c.blk += by;
    while (c.blk >= c.r.nblk) {
      const int over = c.blk - c.r.nblk;
      if (!c.next_item(p, HH, end)) {
        places[warp][lane].blk = -1;
        return;
      }
      c.blk = over;
      // its queries will be wanted soon
      const __nv_bfloat16* q = p.q + ((size_t)c.t * p.Hq + (c.hh / p.groups) * per_kv + c.hh % p.groups * NH) * D;
      for (int i = warp * 64; i < min(NH, per_kv - c.hh % p.groups * NH) * D; i += WARPS * 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
    }
    if (c.blk >= c.blocks_to(end)) {
      places[warp][lane].blk = -1;
      return;
    }
    places[warp][lane] = c;
    const int* table = p.tables + (size_t)c.r.b * p.max_blocks;
    const int per = p.units_per_block, kvh = c.hh / p.groups;
#pragma unroll
    for (int k = 0; k < PAIR; k++) {
      const int u = c.r.u0 + c.blk * BLOCK + warp * PAIR + k;
      unit_next[k] = NONE;
      if (u * UNIT >= c.r.hi) continue;
      const int page = __ldg(table + (per == 1 ? u : u / per));
      unit_next[k] = (uint32_t)unit_index(min(max(page, 0), p.n_blocks - 1), kvh, p.Hkv, per, per == 1 ? 0 : u % per);
    }
  };
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
  auto fetch = [&](int st) {                      // starts the copies of this warp's next units; one group of copies a call
    while (true) {
      const int j = copied & 31;
      if (j == 0) {
#pragma unroll
        for (int k = 0; k < PAIR; k++) unit_now[k] = unit_next[k];
        look(32);
      }
      uint32_t u = __shfl_sync(0xffffffffu, unit_now[0], j);
      if (u == STOP) break;
      copied++;
      if (u == NONE) continue;
#pragma unroll
      for (int k = 0; k < PAIR; k++) {
        if (k > 0) u = __shfl_sync(0xffffffffu, unit_now[k], j);
        if (k > 0 && u == NONE) break;
        const uint8_t *ks = p.kcache + (size_t)u * U + lane * 16, *vs = p.vcache + (size_t)u * U + lane * 16;
        const uint32_t dst = ring_at + st * C::STAGE + k * 2 * U;
#pragma unroll
        for (int o = 0; o < U; o += 512)
          if (U - o >= 512 || lane * 16 < U - o) {
            async16(dst + o, ks + o);
            async16(dst + U + o, vs + o);
          }
      }
      break;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  places[warp][lane] = cur;
  look(lane);
#pragma unroll 1
  for (int i = 0; i < C::STAGES; i++) fetch(i);

  const float zero[4] = {0.f, 0.f, 0.f, 0.f};
  int st = 0;
#pragma unroll 1
  do {
    // ---- one row and head group: blocks [blk0, blk1) of it are in this share ----
    const int blk0 = cur.blk, blk1 = cur.blocks_to(end);
    const int kvh = cur.hh / p.groups, hg = cur.hh % p.groups;
    const int h0 = kvh * per_kv + hg * NH, nh = min(NH, per_kv - hg * NH);

    // queries as B operands; column = head g of each tile of 8
    uint32_t qf[NT][D / 16][2], qs[NT][2];
    float c1[NT][2];                              // bits of a score per unit of a code sum
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int h = nt * 8 + g;
      float qv[G][8], big = 0.f;
#pragma unroll
      for (int i = 0; i < G; i++) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (h < nh) w = *reinterpret_cast<const uint4*>(p.q + ((size_t)cur.t * p.Hq + h0 + h) * D + 32 * i + 8 * t4);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          qv[i][2 * j] = __uint_as_float(ww[j] << 16);
          qv[i][2 * j + 1] = __uint_as_float(ww[j] & 0xffff0000u);
          big = fmaxf(big, fmaxf(fabsf(qv[i][2 * j]), fabsf(qv[i][2 * j + 1])));
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int ex = (int)(__float_as_uint(big) >> 23) - 127;            // 2^ex <= big < 2^(ex + 1)
      const int up = min(max(9 - ex, -100), 120);
      const float f = __int_as_float((up + 127) << 23);
      float sum[G];
#pragma unroll
      for (int i = 0; i < G; i++) {
        sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          qv[i][j] *= f;
          sum[i] += qv[i][j];
        }
        qf[nt][2 * i][0] = pack_half2(qv[i][0], qv[i][4]);
        qf[nt][2 * i][1] = pack_half2(qv[i][1] * 0.0625f, qv[i][5] * 0.0625f);
        qf[nt][2 * i + 1][0] = pack_half2(qv[i][2], qv[i][6]);
        qf[nt][2 * i + 1][1] = pack_half2(qv[i][3] * 0.0625f, qv[i][7] * 0.0625f);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      }
      // the sums of a head's groups in two fp16 parts; which lane holds which: see the least values' operand below
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int i = 0; i < G; i += 2) {
        const bool mine = D == 256 ? t4 == i / 2 : D == 128 ? (t4 & 1) == i / 2 : true;
        if (mine) { a = sum[i]; b = sum[i + 1]; }
      }
      const uint32_t hi = pack_half2(a, b);
      const float2 hf = unpack_half2(hi);
      const uint32_t lo = pack_half2(a - hf.x, b - hf.y);
      if constexpr (D == 256) { qs[nt][0] = hi; qs[nt][1] = lo; }
      else if constexpr (D == 128) { qs[nt][0] = t4 < 2 ? hi : lo; qs[nt][1] = 0; }
      else { qs[nt][0] = t4 == 0 ? hi : t4 == 1 ? lo : 0; qs[nt][1] = 0; }
      // accumulator columns are heads 2 t4, 2 t4 + 1: their factor sits with lanes of g = 2 t4, 2 t4 + 1
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int e = __shfl_sync(0xffffffffu, up, (2 * t4 + c) * 4);
        c1[nt][c] = p.scale_log2 * __int_as_float((127 - e) << 23) * 16777216.f;
      }
    }

    float o[NT][D / 16][4], ob[NT][4], l[NT][2], R[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[nt][i][j] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) ob[nt][j] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; c++) l[nt][c] = R[nt][c] = 0.f;
    }
    float x = 0.f, most = -INFINITY;              // R = top - x; scores (less R) may reach most = x + HEADROOM
    uint32_t s_most = 0;                          // the largest scale that x allows for (half2, both halves)

    const int u_end = min((cur.r.hi + UNIT - 1) / UNIT, cur.r.u0 + blk1 * BLOCK);
#pragma unroll 1
    for (int u = cur.r.u0 + blk0 * BLOCK + warp * PAIR; u < u_end; u += BLOCK) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
      __syncwarp();                               // every lane's part of the stage has landed
      const uint8_t* stage = ring + st * C::STAGE;
      // some of the units' tokens are hidden (of a second unit perhaps all): they may hold anything
      const bool edge = u * UNIT < cur.r.lo || (u + PAIR) * UNIT > cur.r.hi;

      // ---- S^T = K Q^T: rows g and g + 8 of the tile are tokens g and g + 8 ----
      float s[PAIR][NT][4];
#pragma unroll
      for (int k = 0; k < PAIR; k++) {
        const uint8_t* ku = stage + k * 2 * U;
        const uint8_t *m0 = ku + Gm::CODES + 2 * G * UNIT + 2 * G * g, *m1 = m0 + 2 * G * 8;
        const int pair = D == 256 ? t4 : D == 128 ? t4 & 1 : 0;
        const uint32_t a0 = *reinterpret_cast<const uint32_t*>(m0 + 4 * pair), a1 = *reinterpret_cast<const uint32_t*>(m1 + 4 * pair);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float acc[4];
          if constexpr (D == 256) mma(acc, a0, a1, a0, a1, qs[nt][0], qs[nt][1], zero);
          else mma(acc, a0, a1, 0, 0, qs[nt][0], 0, zero);
#pragma unroll
          for (int j = 0; j < 4; j++) s[k][nt][j] = acc[j] * 5.9604644775390625e-8f;      // 2^-24: to the code sums' unit
        }
      }
#pragma unroll
      for (int hf = 0; hf < HALVES; hf++) {
        uint32_t w0[PAIR][PER], w1[PAIR][PER], f0[PAIR][PER / 2], f1[PAIR][PER / 2];
#pragma unroll
        for (int k = 0; k < PAIR; k++) {
          const uint8_t* ku = stage + k * 2 * U;
          lds<PER>(w0[k], ku + ((hf * UNIT + g) * 4 + t4) * (4 * PER));
          lds<PER>(w1[k], ku + ((hf * UNIT + g + 8) * 4 + t4) * (4 * PER));
          lds<PER / 2>(f0[k], ku + Gm::CODES + 2 * (G * g + hf * PER));
          lds<PER / 2>(f1[k], ku + Gm::CODES + 2 * (G * (g + 8) + hf * PER));
        }
#pragma unroll
        for (int i = 0; i < PER; i++)
#pragma unroll
          for (int k = 0; k < PAIR; k++) {
            const float2 fa = unpack_half2(f0[k][i / 2]), fb = unpack_half2(f1[k][i / 2]);
            const float s0 = i & 1 ? fa.y : fa.x, s1 = i & 1 ? fb.y : fb.x;
            const uint32_t y0 = w0[k][i], y1 = w1[k][i], x0 = y0 >> 8, x1 = y1 >> 8;
            const int ks = 2 * (hf * PER + i);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              float acc[4];
              mma(acc, y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u, qf[nt][ks][0], qf[nt][ks][1], zero);
              mma(acc, x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, qf[nt][ks + 1][0], qf[nt][ks + 1][1], acc);
              s[k][nt][0] = fmaf(acc[0], s0, s[k][nt][0]);
              s[k][nt][1] = fmaf(acc[1], s0, s[k][nt][1]);
              s[k][nt][2] = fmaf(acc[2], s1, s[k][nt][2]);
              s[k][nt][3] = fmaf(acc[3], s1, s[k][nt][3]);
            }
          }
      }
#pragma unroll
      for (int k = 0; k < PAIR; k++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[k][nt][j] = fmaf(s[k][nt][j], c1[nt][j & 1], -R[nt][j & 1]);
      if (edge) {
#pragma unroll
        for (int k = 0; k < PAIR; k++)
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const int key = (u + k) * UNIT + g + 4 * j;
            if (key < cur.r.lo || key >= cur.r.hi) {
#pragma unroll
              for (int nt = 0; nt < NT; nt++) s[k][nt][j] = s[k][nt][j + 1] = -INFINITY;
            }
          }
      }

      // ---- do the sums' references still hold? (the units' scales are looked at a word a lane) ----
      constexpr int SW = G * UNIT / 64 > 0 ? G * UNIT / 64 : 1;          // words of scales a lane: 1, 1, 2
      const int sw = D == 64 ? lane & 15 : lane * SW;
      uint32_t sm[PAIR][SW];
      bool over = false;
#pragma unroll
      for (int k = 0; k < PAIR; k++) {
        lds<SW>(sm[k], stage + k * 2 * U + U + Gm::CODES + 4 * sw);
        if (edge) {
          const uint32_t keep = seen_pair(cur.r, (u + k) * UNIT + sw / G * 2);
#pragma unroll
          for (int i = 0; i < SW; i++) sm[k][i] &= keep;
        }
#pragma unroll
        for (int i = 0; i < SW; i++) over |= above(sm[k][i], s_most);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < 4; j++) over |= s[k][nt][j] > most;
      }
      if (__any_sync(0xffffffffu, over)) {
        uint32_t sx = s_most;
#pragma unroll
        for (int k = 0; k < PAIR; k++)
#pragma unroll
          for (int i = 0; i < SW; i++) sx = hmax2(sx, sm[k][i]);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) sx = hmax2(sx, __shfl_xor_sync(0xffffffffu, sx, off));
        const float2 pr = unpack_half2(sx);
        // 2^e is the least power of two not below the largest scale; p reaches 2^(x + 8), p s reaches 2^(x + 8 + e): both at
        // most 2^15
        const uint32_t bits = __float_as_uint(fmaxf(pr.x, pr.y));
        const int e = max((int)(bits >> 23) - 127 + ((bits & 0x7fffffu) != 0), 0);
        const uint32_t lim = e >= 16 ? 0x7bffu : (uint32_t)(e + 15) << 10;     // fp16 of 2^e, at most its largest
        s_most = lim | lim << 16;
        const float x_new = (float)(15 - HEADROOM - e);
        const bool first = most == -INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < PAIR; k++) m = fmaxf(m, fmaxf(s[k][nt][c], s[k][nt][c + 2]));
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            // in scores less the old R: the old top is x
            const float down = (first ? m : fmaxf(m, x)) - x_new, alpha = first ? 1.f : ex2(-down);
            R[nt][c] += down;
#pragma unroll
            for (int k = 0; k < PAIR; k++) {
              s[k][nt][c] -= down;
              s[k][nt][c + 2] -= down;
            }
            l[nt][c] *= alpha;
            ob[nt][c] *= alpha;
#pragma unroll
            for (int i = 0; i < D / 16; i++) { o[nt][i][c] *= alpha; o[nt][i][c + 2] *= alpha; }
          }
        x = x_new;
        most = x_new + HEADROOM;
      }

      // ---- p, and O^T += V^T P^T; scales and least values of token pairs t4 and t4 + 4 ----
#pragma unroll
      for (int k = 0; k < PAIR; k++) {
        const uint8_t* vu = stage + k * 2 * U + U;
        uint32_t vs0[G], vs1[G], vm0 = 0, vm1 = 0, b0[NT], b1[NT];
        {
          const uint8_t* ms = vu + Gm::CODES;
          lds<G>(vs0, ms + t4 * (4 * G));
          lds<G>(vs1, ms + (t4 + 4) * (4 * G));
          if (g < G) {
            vm0 = *reinterpret_cast<const uint32_t*>(ms + 2 * G * UNIT + (t4 * G + g) * 4);
            vm1 = *reinterpret_cast<const uint32_t*>(ms + 2 * G * UNIT + ((t4 + 4) * G + g) * 4);
          }
        }
        if (edge) {
          const uint32_t k01 = seen_pair(cur.r, (u + k) * UNIT + 2 * t4), k89 = seen_pair(cur.r, (u + k) * UNIT + 2 * t4 + 8);
#pragma unroll
          for (int i = 0; i < G; i++) { vs0[i] &= k01; vs1[i] &= k89; }
          vm0 &= k01;
          vm1 &= k89;
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const float p0 = ex2(s[k][nt][0]), p1 = ex2(s[k][nt][1]), p2 = ex2(s[k][nt][2]), p3 = ex2(s[k][nt][3]);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          b0[nt] = transpose8x8(pack_half2(p0, p1));
          b1[nt] = transpose8x8(pack_half2(p2, p3));
          mma(ob[nt], vm0, 0, vm1, 0, b0[nt], b1[nt], ob[nt]);
        }
#pragma unroll
        for (int hf = 0; hf < HALVES; hf++) {
          uint32_t v[4][PER / 2];                 // this lane's dims of tokens 2 t4, 2 t4 + 1, + 8, + 9
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int place = t4 + 4 * i;
            lds<PER / 2>(v[i], vu + ((hf * UNIT + place) * 8 + v_slot<D>(place, g)) * (2 * PER));
          }
#pragma unroll
          for (int i = 0; i < PER; i++) {
            const uint32_t sel = i & 1 ? 0x7632u : 0x5410u;
            const uint32_t y = __byte_perm(v[0][i / 2], v[1][i / 2], sel), z = __byte_perm(v[2][i / 2], v[3][i / 2], sel);
            const uint32_t y8 = y >> 8, z8 = z >> 8;
            const int gi = hf * PER + i;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const uint32_t q0 = hmul2(b0[nt], vs0[gi]), q1 = hmul2(b1[nt], vs1[gi]);
              mma(o[nt][2 * gi], y & 0x000f000fu, y & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u, q0, q1, o[nt][2 * gi]);
              mma(o[nt][2 * gi + 1], y8 & 0x000f000fu, y8 & 0x00f000f0u, z8 & 0x000f000fu, z8 & 0x00f000f0u, q0, q1, o[nt][2 * gi + 1]);
            }
          }
        }
      }
      __syncwarp();                               // every lane has read the stage: it may be filled again
      fetch(st);
      if (++st == C::STAGES) st = 0;
    }

    // ---- the warps' sums become one ----
    const bool whole = blk0 == 0 && blk1 == cur.r.nblk;
    const int slot = blk0 == 0 ? 1 : 0;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], off);
        // A warp that had no unit is told by its R.  One whose every score was NaN has -inf there too, and must not be dropped.
        const float lc = l[nt][c];
        if (g == 0) mlbuf[warp * NH + nt * 8 + 2 * t4 + c] = make_float2(lc == 0.f ? -INFINITY : lc != lc ? 0.f : R[nt][c], lc);
      }
#pragma unroll
    for (int part = 0; part < D / C::ODIM; part++) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float* row = obuf + (warp * NH + nt * 8 + 2 * t4 + c) * C::OROW;
#pragma unroll
          for (int i = 0; i < C::ODIM / GROUP; i++) {
            const int gi = part * (C::ODIM / GROUP) + i;
            const float least = __shfl_sync(0xffffffffu, ob[nt][c], gi * 4 + t4);
            float4 v;
            v.x = fmaf(o[nt][2 * gi][c], 16777216.f, least);
            v.y = fmaf(o[nt][2 * gi][c + 2], 1048576.f, least);
            v.z = fmaf(o[nt][2 * gi + 1][c], 16777216.f, least);
            v.w = fmaf(o[nt][2 * gi + 1][c + 2], 1048576.f, least);
            *reinterpret_cast<float4*>(row + 32 * i + 4 * g) = v;
          }
        }
      __syncthreads();
      for (int i = threadIdx.x; i < nh * (C::ODIM / 4); i += THREADS) {
        const int h = i / (C::ODIM / 4), d4 = i % (C::ODIM / 4), dim = part * C::ODIM + 4 * d4;
        float r = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) r = fmaxf(r, mlbuf[w * NH + h].x);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
          const float2 ml = mlbuf[w * NH + h];
          const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - r);
          const float4 v = *reinterpret_cast<const float4*>(obuf + (w * NH + h) * C::OROW + 4 * d4);
          sum += f * ml.y;
          a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
        }
        if (whole) {
          if (p.sinks) sum += ex2(sink_log2(p, h0 + h) - r);
          const float inv = 1.f / sum;
          __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
          *reinterpret_cast<uint2*>(p.out + ((size_t)cur.t * p.Hq + h0 + h) * D + dim) =
              make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
        } else {
          const size_t at = ((size_t)blockIdx.x * 2 + slot) * NH + h;
          *reinterpret_cast<float4*>(p.parts + at * D + dim) = a;
          if (dim == 0) p.part_ml[at] = make_float2(r, sum);
        }
      }
      __syncthreads();
    }

    // ---- a row that shares cut: the last CTA to arrive adds the parts ----
    if (!whole) {
      const uint32_t at0 = begin + cur.start;     // of the row, in the whole line
      const int first = (int)((at0 + EXTRA) / share), last = (int)((at0 + EXTRA + cur.r.nblk - 1) / share);
      auto place = [&](int i, int h) { return ((size_t)i * 2 + (i == first ? 1 : 0)) * NH + h; };
      // parts of shares lo, lo + step, .. <= hi: to the place of the first, or (all of them) to the output.  Lane i looks after
      // the factor of the i-th part of 32; the parts' rows load while the factors do.
      auto add = [&](int lo, int hi, int step, bool to_out) {
        for (int h = warp; h < nh; h += WARPS) {
          float r = -INFINITY, sum = 0.f, a[D / 32];
#pragma unroll
          for (int j = 0; j < D / 32; j++) a[j] = 0.f;
          for (int base = lo; base <= hi; base += 32 * step) {
            const int mine = base + lane * step, cnt = min(32, (hi - base) / step + 1);
            const float2 ml = lane < cnt ? __ldcg(&p.part_ml[place(mine, h)]) : make_float2(-INFINITY, 0.f);
            const float r_new = fmaxf(r, warp_max(ml.x)), keep = r == -INFINITY ? 0.f : ex2(r - r_new);
            const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - r_new);
            sum = sum * keep + warp_sum(f * ml.y);
            r = r_new;
#pragma unroll
            for (int j = 0; j < D / 32; j++) a[j] *= keep;
#pragma unroll 8
            for (int i = 0; i < cnt; i++) {
              const float fi = __shfl_sync(0xffffffffu, f, i);
              const float* src = p.parts + place(base + i * step, h) * D + lane * 2;
#pragma unroll
              for (int j = 0; j < D / 32; j += 2) {
                const float2 v = __ldcg(reinterpret_cast<const float2*>(src + 32 * j));
                a[j] = fmaf(fi, v.x, a[j]);
                a[j + 1] = fmaf(fi, v.y, a[j + 1]);
              }
            }
          }
          __syncwarp();
          if (to_out) {
            if (p.sinks) sum += ex2(sink_log2(p, h0 + h) - r);
            const float inv = 1.f / sum;
            __nv_bfloat16* dst = p.out + ((size_t)cur.t * p.Hq + h0 + h) * D + lane * 2;
#pragma unroll
            for (int j = 0; j < D / 32; j += 2)
              *reinterpret_cast<__nv_bfloat162*>(dst + 32 * j) = __floats2bfloat162_rn(a[j] * inv, a[j + 1] * inv);
          } else {
            float* dst = p.parts + place(lo, h) * D + lane * 2;
#pragma unroll
            for (int j = 0; j < D / 32; j += 2) *reinterpret_cast<float2*>(dst + 32 * j) = make_float2(a[j], a[j + 1]);
            if (lane == 0) p.part_ml[place(lo, h)] = make_float2(r, sum);
          }
        }
      };
      auto is_last = [&](int* ticket, int n) {    // of n; what the others wrote is then visible
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          arrived = atomicAdd(ticket, 1);
          if (arrived == n - 1) *ticket = 0;
        }
        __syncthreads();
        const bool yes = arrived == n - 1;
        if (yes) __threadfence();
        __syncthreads();                          // (`arrived` is used again)
        return yes;
      };
      if (last - first < FAN) {
        if (is_last(p.tickets + first, last - first + 1)) add(first, last, 1, true);
      } else {
        const int me = blockIdx.x - first, lo = first + me / FAN * FAN, hi = min(lo + FAN - 1, last);
        if (is_last(p.tickets + gridDim.x * (lo == first ? 2 : 1) + lo, hi - lo + 1)) {
          add(lo, hi, 1, false);
          if (is_last(p.tickets + first, (last - first) / FAN + 1)) add(first, last, FAN, true);
        }
      }
    }
  } while (cur.next_item(p, HH, end));
}

int variant(int D, int per) { return D == 256 || per <= 8 ? 1 : 2; }     // tiles of 8 heads (256-wide heads: registers hold one)

template <int D, int NT> int ctas() { return 148 * Cfg<D, NT>::CTAS; }

template <int D, int NT> int launch(const Params& p, int grid, cudaStream_t st) {
  using C = Cfg<D, NT>;
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return -3;
    ready[dev] = true;
  }
  const cudaError_t e = launch_pdl(kv4_decode_kernel<D, NT>, dim3(grid), dim3(C::THREADS), C::SMEM, st, p);
  if (e != cudaSuccess) return (int)e;
  EXO_CHECK_LAUNCH();
  return 0;
}

int grid_of(int D, int NT) {
  if (D == 64) return NT == 1 ? ctas<64, 1>() : ctas<64, 2>();
  if (D == 128) return NT == 1 ? ctas<128, 1>() : ctas<128, 2>();
  return ctas<256, 1>();
}

}  // namespace

// Words of zeros that exo_kv4_decode wants as its tickets, and leaves as zeros.
EXO_API int exo_kv4_decode_tickets() { return 3 * 148 * 2; }

// Bytes of scratch that exo_kv4_decode wants (0: shape not served).
EXO_API long exo_kv4_decode_workspace(int Hq, int Hkv, int D) {
  if (Hkv <= 0 || Hq % Hkv || (D != 64 && D != 128 && D != 256)) return 0;
  const int nt = variant(D, Hq / Hkv), grid = grid_of(D, nt);
  return (long)grid * (2 * 8 * nt * (8 + 4 * D));
}

// An AttnCall, one query row at a time: q [T, Hq, D] bf16, row t of sequence b (by cu_q) sees keys up to its own position.
EXO_API int exo_kv4_decode(const void* call, int bytes, cudaStream_t st) {
  AttnCall c;
  if (!unpack_call(c, call, bytes)) return -2;
  const int T_ = c.T, B = c.B, Hq = c.Hq, Hkv = c.Hkv, D = c.D, n_blocks = c.n_blocks, max_blocks = c.max_blocks, block_size = c.block_size;
  if (T_ == 0) return 0;
  if (T_ < 0 || B <= 0 || Hkv <= 0 || Hq % Hkv || block_size <= 0 || block_size % UNIT || n_blocks <= 0) return -2;
  if ((long)n_blocks * Hkv * (block_size / UNIT) >= (long)NONE) return -2;       // units are numbered in 32 bits (5 TB of 128-wide heads)
  const int per = Hq / Hkv, nt = variant(D, per), NH = 8 * nt, grid = grid_of(D, nt);
  // the line of blocks is counted in 32 bits: at most this many, with the smallest block
  if ((long)T_ * Hkv * ((per + NH - 1) / NH) * ((long)max_blocks * (block_size / UNIT) / 6 + EXTRA + 1) >= 1L << 31) return -2;
  Params p;
  p.q = (const __nv_bfloat16*)c.q; p.kcache = (const uint8_t*)c.kcache; p.vcache = (const uint8_t*)c.vcache;
  p.tables = c.tables; p.seq_lens = c.seq_lens; p.cu_q = c.cu_q; p.out = (__nv_bfloat16*)c.out;
  p.parts = (float*)c.ws;
  p.part_ml = (float2*)((char*)c.ws + (size_t)grid * 2 * NH * D * 4);
  p.tickets = c.tickets;
  p.sinks = c.sinks; p.scale_log2 = c.scale * LOG2E; p.sink_dtype = c.sink_dtype;
  p.T = T_; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.n_blocks = n_blocks; p.max_blocks = max_blocks;
  p.units_per_block = block_size / UNIT; p.window = c.window; p.groups = (per + NH - 1) / NH;
  if (D == 64) return nt == 1 ? launch<64, 1>(p, grid, st) : launch<64, 2>(p, grid, st);
  if (D == 128) return nt == 1 ? launch<128, 1>(p, grid, st) : launch<128, 2>(p, grid, st);
  if (D == 256) return launch<256, 1>(p, grid, st);
  return -2;
}
