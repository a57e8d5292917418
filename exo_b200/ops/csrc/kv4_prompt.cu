// Attention of prompts over a 4-bit KV cache: ragged causal flash attention on the 5th-generation tensor cores.
//
// One CTA = TILES x 128 query rows of one key head x a run of its sequence's keys.  A row is (new token, head of the group), so
// the heads that share a key head share its tiles, and a chunk of a few tokens still fills one.  Keys are walked in blocks of BN:
//   * seven (256-wide heads: eight) warps turn the block's codes into fp16 operand tiles: (code | 0x6400) is the fp16 number 1024 + n (1024 + 16 n at
//     bit 4), one fma takes that off, a second makes n s + m with one rounding (fp16 holds every cached value: the format clamps
//     to its range).  Nothing is permuted into memory order: the queries are stored in the order in which a word's nibbles come
//     out (0 4 1 5 2 6 3 7), and the outputs leave in the order of the values' (two groups of 32 dims, interleaved).  The packed
//     units wait in shared memory, the next block's keys copied while this block's values are widened and the other way round.
//   * one thread issues the matrix instructions:  S_t = Q_t K^T (tile t, both K-major, 128-byte swizzle) and O_t += P_t V (P from
//     TMEM, V MN-major), in the order S_0 S_1 | PV_0 S_0' PV_1 S_1' ..: each tile's softmax runs under the other's products.
//   * one warpgroup per tile does the softmax, a row per thread, its scores in registers; P goes back as fp16 over the
//     place of S.  O is rescaled only when a row's maximum has grown by more than 2^8 since it was last taken (p then fits fp16 all
//     the same), which after the first block hardly happens.
// fp16, not bf16, throughout: queries are scaled per row by a power of two, so all three operands lose 2^-11 at most.
// What bounds it: a tile's chain (scores, softmax, product: some 2900 clocks of softmax and 1800 of matrix work and hand-over a
// block of 128 keys), of which two run side by side.  No unit is full: tensor pipe 40%, exponentials 40%, ALU 41%, issue slots 50%,
// shared memory about half.  8192 tokens, 32 heads of 128 over 8: 636 us, 865 TFLOP/s.  Tried without gain: blocks handed over by
// halves with an issuing warp a tile (664), scores read 32 columns at a time (794), a quarter of the exponentials by
// polynomial (868 with that), no maximum while a row's weights stay under 2^8 (648), two softmax warpgroups a tile,
// half of the keys each (686: TMEM puts both warps of a row on one scheduler, whose exponentials are what takes the time), one tile a CTA and two CTAs an SM for 64-wide heads (1249 us against
// 1048 for 8192 tokens), an eighth dequantising warp (17 warps: 96 registers, 1224), two score buffers or queries in TMEM for
// 256-wide heads.
// With few rows the keys are split over several CTAs, whose fp32 parts kv4_prompt_merge_kernel adds in order.
// Every wait is bounded; one that runs out records a code, and the CTA unwinds and frees its TMEM.
#include "kv4.cuh"
#include "tc_common.cuh"

int* exo_tc_err_ptr();

namespace {

using namespace kv4;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int ROWS = 128;                  // of a tile
constexpr float GROWTH = 8.f;              // bits by which a row's maximum may grow before O is rescaled

template <int D> struct Cfg {
  static constexpr int TILES = D == 256 ? 1 : 2;           // TMEM: D columns of O and BN of S (and P) a tile
  static constexpr int BN = D == 256 ? 64 : 128;           // keys of a block: two K and two V stages beside Q in shared memory
  static constexpr int SOFT = 4 * TILES, DEQ = D == 256 ? 8 : 7;          // warps: softmax, dequantising; one more issues (4 a scheduler at 128 registers)
  static constexpr int THREADS = 32 * (SOFT + DEQ + 1);
  static constexpr uint32_t HALF_Q = ROWS * 128, HALF_K = BN * 128;      // bytes of 64 dims of a tile
  static constexpr uint32_t Q_TILE = D / 64 * HALF_Q, KV_TILE = D / 64 * HALF_K;
  static constexpr uint32_t S_COL = 0, O_COL = TILES * BN, TMEM = 512;
};

template <int D> struct __align__(1024) Smem {
  using C = Cfg<D>;
  uint8_t q[C::TILES][C::Q_TILE];
  uint8_t k[2][C::KV_TILE];
  uint8_t v[2][C::KV_TILE];
  alignas(16) uint8_t packed[2][C::BN / UNIT * Geo<D>::BYTES];       // the units of a block's keys, of its values
  float row_scale[C::TILES * ROWS];
  alignas(16) uint32_t nan_any[2][16];      // by V stage and dequantising warp: a visible row of values is NaN
  uint8_t nan_key[2][C::BN];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[C::TILES], p_ready[C::TILES], pv_done[C::TILES], drained;
  uint32_t tmem_base;
  int seq, tile, q0, q_len, keys;
};

struct Params {
  const __nv_bfloat16* q;
  const uint8_t *kcache, *vcache;
  const int *tables, *seq_lens, *cu_q;
  __nv_bfloat16* out;
  float* parts;                            // [splits][T][Hq][D]
  float2* part_ml;                         // [splits][T][Hq] (reference maximum in bits, sum)
  int* err;
  const void* sinks;
  float scale;
  int T, B, Hq, Hkv, n_blocks, max_blocks, units_per_block, window, sink_dtype, splits;
};

__device__ __forceinline__ float sink_log2(const Params& p, int h) {
  return (p.sink_dtype == EXO_BF16 ? __bfloat162float(((const __nv_bfloat16*)p.sinks)[h]) : ((const float*)p.sinks)[h]) * LOG2E;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 at a time (one instruction on sm_100)
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<unsigned long long&>(a)),
      "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<unsigned long long&>(a)),
      "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ __half2 as_half2(uint32_t a) { return *reinterpret_cast<const __half2*>(&a); }
__device__ __forceinline__ uint32_t as_u32(__half2 a) { return *reinterpret_cast<const uint32_t*>(&a); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
// f16 x f16 -> fp32
constexpr uint32_t idesc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
// V tile as an MN-major B operand: keys 128 B apart, 8-key groups 1024 B apart, every 64 dims one `half` further
__device__ __forceinline__ uint64_t desc_v(uint32_t smem_addr, uint32_t half) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(half >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}

// The four half2 of a word's codes: (n0, n4), (n1, n5), (n2, n6), (n3, n7) of a halfword pair, times s plus m.
__device__ __forceinline__ uint4 widen(uint32_t w, __half2 s, __half2 m) {
  const __half2 k1024 = __float2half2_rn(1024.f), sixteenth = __float2half2_rn(0.0625f), k64 = __float2half2_rn(-64.f);
  const uint32_t h = w >> 8;
  const __half2 a = __hsub2(as_half2((w & 0x000f000fu) | 0x64006400u), k1024);
  const __half2 b = __hfma2(as_half2((w & 0x00f000f0u) | 0x64006400u), sixteenth, k64);
  const __half2 c = __hsub2(as_half2((h & 0x000f000fu) | 0x64006400u), k1024);
  const __half2 d = __hfma2(as_half2((h & 0x00f000f0u) | 0x64006400u), sixteenth, k64);
  return make_uint4(as_u32(__hfma2(a, s, m)), as_u32(__hfma2(b, s, m)), as_u32(__hfma2(c, s, m)), as_u32(__hfma2(d, s, m)));
}

template <int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, 1) kv4_prompt_kernel(const Params p) {
  using C = Cfg<D>;
  using Gm = Geo<D>;
  constexpr int TILES = C::TILES, BN = C::BN, G = Gm::G, U = Gm::BYTES;
  extern __shared__ uint8_t smem_raw[];
  Smem<D>& s = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int W_DEQ = C::SOFT, W_MMA = W_DEQ + C::DEQ;
  const int per = p.Hq / p.Hkv, kvh = blockIdx.y;

  pdl_trigger();
  if (warp == W_MMA) {
    tc::tmem_alloc(&s.tmem_base, C::TMEM);
    tc::tmem_relinquish();
    if (lane == 0) {
      for (int i = 0; i < 2; i++) {
        tc::mbar_init(&s.k_full[i], 32 * C::DEQ); tc::mbar_init(&s.k_empty[i], 1);
        tc::mbar_init(&s.v_full[i], 32 * C::DEQ); tc::mbar_init(&s.v_empty[i], 1);
      }
      for (int i = 0; i < TILES; i++) { tc::mbar_init(&s.s_full[i], 1); tc::mbar_init(&s.p_ready[i], 128); tc::mbar_init(&s.pv_done[i], 1); }
      tc::mbar_init(&s.drained, 1);
      for (int i = 0; i < 16; i++) s.nan_any[0][i] = s.nan_any[1][i] = 0;
      tc::fence_barrier_init();
    }
  }
  pdl_wait();
  if (warp == 0) {
    // the (sequence, tile of rows) of this CTA; the line of tiles is walked from its end, where causal tiles are long
    int t = gridDim.x - 1 - blockIdx.x, seq = -1;
    for (int b0 = 0; b0 < p.B && seq < 0; b0 += 32) {
      const int b = min(b0 + lane, p.B - 1), c0 = p.cu_q[b], len = p.cu_q[b + 1] - c0, keys = p.seq_lens[b];
      int n = b0 + lane < p.B ? (len * per + TILES * ROWS - 1) / (TILES * ROWS) : 0;
      const int mine = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += up;
      }
      const unsigned over = __ballot_sync(0xffffffffu, n > t);
      if (over) {
        const int w = __ffs(over) - 1;
        seq = b0 + w;
        t -= __shfl_sync(0xffffffffu, n - mine, w);
        if (lane == w) { s.q0 = c0; s.q_len = len; s.keys = keys; }
      } else {
        t -= __shfl_sync(0xffffffffu, n, 31);
      }
    }
    if (lane == 0) { s.seq = seq; s.tile = t; }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  const int seq = s.seq;
  const int behind = max(p.cu_q[p.B], 0);                      // rows behind the last sequence

  if (seq >= 0) {
    // (no offset, however wrong, leads out of q)
    const int q0 = max(s.q0, 0), q_len = s.q_len, n_rows = min(q_len, p.T - q0) * per, row0 = s.tile * TILES * ROWS;
    const int kv_len = (int)min((long)s.keys, (long)p.max_blocks * p.units_per_block * UNIT);
    const int pos0 = s.keys - q_len;                           // position of the first new token
    const int tiles = TILES == 2 && n_rows - row0 > ROWS ? 2 : 1;
    const int last_tok = (min(row0 + TILES * ROWS, n_rows) - 1) / per;
    // keys that any row of the CTA sees, in blocks from a unit's border
    const int k_end = min(kv_len, pos0 + last_tok + 1), k_beg = p.window > 0 ? max(0, pos0 + row0 / per - p.window + 1) : 0;
    const int u_first = k_beg / UNIT;
    int n_all = k_end > k_beg ? (k_end - u_first * UNIT + BN - 1) / BN : 0;
    const int share = (n_all + p.splits - 1) / p.splits, b_first = min(n_all, share * (int)blockIdx.z);
    const int n_blk = min(n_all, b_first + share) - b_first;
    const int key0 = u_first * UNIT + b_first * BN;            // of this CTA's first block

    constexpr int UNITS = BN / UNIT, LINES = U / 16, N = 32 * C::DEQ;
    const int dt = tid - 32 * W_DEQ;                           // of the dequantising threads
    const int* table = p.tables + (size_t)seq * p.max_blocks;
    const int upb = p.units_per_block, u_last = max(0, (kv_len + UNIT - 1) / UNIT - 1);
    // units of a block, copied as they are (16 bytes a thread at a time): keys while the values before them are widened, and
    // the other way round; page numbers a block earlier, a unit a lane
    auto page_at = [&](int blk) {
      const int u = min((key0 + blk * BN) / UNIT + (lane & (UNITS - 1)), u_last);
      return __ldg(table + (upb == 1 ? u : u / upb));
    };
    auto copy = [&](const uint8_t* cache, uint8_t* dst, int blk, int page) {
      const int u = min((key0 + blk * BN) / UNIT + (lane & (UNITS - 1)), u_last);
      const size_t mine = unit_index(min(max(page, 0), p.n_blocks - 1), kvh, p.Hkv, upb, upb == 1 ? 0 : u % upb) * U;
#pragma unroll
      for (int i = 0; i < (UNITS * LINES + N - 1) / N; i++) {
        const int e = i * N + dt, unit = e / LINES;
        const size_t base = __shfl_sync(0xffffffffu, mine, unit & (UNITS - 1));
        if (e < UNITS * LINES)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc::smem_u32(dst) + e * 16), "l"(cache + base + e % LINES * 16) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int page = 0;
    if (warp >= W_DEQ && warp < W_MMA && n_blk > 0) {          // the first keys are on their way while the queries are laid out
      page = page_at(0);
      copy(p.kcache, s.packed[0], 0, page);
    }

    // ---- Q: fp16, scaled per row by a power of two, dims of 8 in the order 0 4 1 5 2 6 3 7 ----
    {
      constexpr int L = D / 8, STEP = C::THREADS / L, N_STEP = (TILES * ROWS + STEP - 1) / STEP;      // lanes of a row; rows at a time
      const int c = tid % L;
      uint4 raw[N_STEP];                                       // (all on their way at once: one at a time took 3 to 7 us a CTA)
#pragma unroll
      for (int k = 0; k < N_STEP; k++) {
        const int row = row0 + tid / L + k * STEP;
        raw[k] = make_uint4(0, 0, 0, 0);
        if (row < n_rows) raw[k] = *reinterpret_cast<const uint4*>(p.q + ((size_t)(q0 + row / per) * p.Hq + kvh * per + row % per) * D + 8 * c);
      }
#pragma unroll
      for (int k = 0; k < N_STEP; k++) {
        const int i = tid / L + k * STEP;
        const uint4 w = raw[k];
        if (i >= tiles * ROWS) break;
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
        float f[8], big = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[2 * j] = __uint_as_float(ww[j] << 16);
          f[2 * j + 1] = __uint_as_float(ww[j] & 0xffff0000u);
          big = fmaxf(big, fmaxf(fabsf(f[2 * j]), fabsf(f[2 * j + 1])));
        }
        const unsigned mask = L == 32 ? 0xffffffffu : ((1u << L) - 1) << (lane / L * L);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(mask, big, o));
        const int up = min(max(9 - ((int)(__float_as_uint(big) >> 23) - 127), -100), 120);
        const float by = copysignf(__int_as_float((up + 127) << 23), p.scale);      // (scores then take |scale|)
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] *= by;
        // (never 0: a hidden score is -inf times this)
        if (c == 0) s.row_scale[i] = fmaxf(fabsf(p.scale) * LOG2E * __int_as_float((127 - up) << 23), 1.1754943508222875e-38f);
        const int tile = i / ROWS, r = i % ROWS;
        *reinterpret_cast<uint4*>(s.q[tile] + c / 8 * C::HALF_Q + r * 128 + ((c % 8) ^ (r & 7)) * 16) =
            make_uint4(pack_half2(f[0], f[4]), pack_half2(f[1], f[5]), pack_half2(f[2], f[6]), pack_half2(f[3], f[7]));
      }
    }
    tc::fence_proxy_async();
    __syncthreads();

    if (warp >= W_DEQ) {
     if (warp < W_MMA) {
      // ================= dequantising warps: K(0) V(0) K(1) V(1) .. =================
      // A job is 32 pieces of 16 bytes of codes, a piece a lane: a tile's jobs go round the warps.  The rows that share a phase of a
      // job's 16-byte stores are chosen so that the swizzle puts them in different banks.
      constexpr int JOBS = UNITS * D / 64;
      const int dw = warp - W_DEQ;
      const int part = D == 64 ? lane & 1 : lane & 3;          // piece of its row (of 128 dims)
      const int row_lo = D == 64 ? ((lane >> 1) & 1) | ((lane >> 2) & 1) << 2 | ((lane >> 3) & 1) << 1 | ((lane >> 4) & 1) << 3
                                 : ((lane >> 3) & 3) | ((lane >> 2) & 1) << 2;
      // job j: unit j / (D / 64), row + 8 * (j & 1) (64-wide: all 16 rows at once), half of 256 dims
      auto job_unit = [](int j) { return j / (D / 64); };
      auto job_row = [&](int j) { return D == 64 ? row_lo : row_lo + 8 * (j & 1); };
      auto job_half = [](int j) { return D == 256 ? (j >> 1) & 1 : 0; };
      auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); };
      auto landed = [&]() {                                    // the copy in flight, for all of these warps (which are past the tile before)
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        meet();
      };
      bool ok = true;
#pragma unroll 1
      for (int it = 0; it < n_blk; it++) {
        const int st = it & 1;
        const int page_next = it + 1 < n_blk ? page_at(it + 1) : 0;
        // ---- keys ----
        if (!tc::mbar_wait(&s.k_empty[st], ((it >> 1) & 1) ^ 1, ok ? 1u << 22 : 16)) {
          ok = false;                                          // (these warps stay together: they walk on, past short waits)
          atomicExch(p.err, tc::ERR_EMPTY_TIMEOUT);
        }
        landed();
        copy(p.vcache, s.packed[1], it, page);
#pragma unroll
        for (int i = 0; i < (JOBS + C::DEQ - 1) / C::DEQ; i++) {
          const int j = i * C::DEQ + dw, half = job_half(j), row = job_row(j), key = job_unit(j) * UNIT + row;
          if (j >= JOBS) break;
          const uint8_t* unit = s.packed[0] + job_unit(j) * U;
          const uint4 code = *reinterpret_cast<const uint4*>(unit + (D == 64 ? (row * 2 + part) * 16 : (half * UNIT * 4 + row * 4 + part) * 16));
          const uint32_t w[4] = {code.x, code.y, code.z, code.w};
          const uint8_t* meta = unit + Gm::CODES + 2 * (G * row + half * 4);
          uint32_t sc[2], ls[2];
          if (D == 64) {
            sc[0] = *reinterpret_cast<const uint32_t*>(meta);
            ls[0] = *reinterpret_cast<const uint32_t*>(meta + 2 * G * UNIT);
          } else {
            const uint2 a = *reinterpret_cast<const uint2*>(meta), b = *reinterpret_cast<const uint2*>(meta + 2 * G * UNIT);
            sc[0] = a.x; sc[1] = a.y; ls[0] = b.x; ls[1] = b.y;
          }
          uint8_t* dst = s.k[st] + half * (2 * C::HALF_K) + key * 128;
#pragma unroll
          for (int k = 0; k < 4; k++) {
            // word k: group g of its 128 (64) dims, dims 8 t .. of it
            const int g = D == 64 ? k & 1 : k, t = D == 64 ? part * 2 + (k >> 1) : part;
            const uint32_t ss = __byte_perm(sc[g >> 1], 0, g & 1 ? 0x3232u : 0x1010u), mm = __byte_perm(ls[g >> 1], 0, g & 1 ? 0x3232u : 0x1010u);
            *reinterpret_cast<uint4*>(dst + (g >> 1) * C::HALF_K + ((4 * (g & 1) + t) ^ (row & 7)) * 16) = widen(w[k], as_half2(ss), as_half2(mm));
          }
        }
        tc::fence_proxy_async();
        tc::mbar_arrive(&s.k_full[st]);
        // ---- values ----
        bool nan = false;
        if (!tc::mbar_wait(&s.v_empty[st], ((it >> 1) & 1) ^ 1, ok ? 1u << 22 : 16)) {
          ok = false;
          atomicExch(p.err, tc::ERR_EMPTY_TIMEOUT);
        }
        landed();
        if (it + 1 < n_blk) copy(p.kcache, s.packed[0], it + 1, page_next);
#pragma unroll
        for (int i = 0; i < (JOBS + C::DEQ - 1) / C::DEQ; i++) {
          const int j = i * C::DEQ + dw, half = job_half(j), place = job_row(j);
          if (j >= JOBS) break;
          const int tok = (place & 8) | (place & 3) << 1 | ((place >> 2) & 1);       // the token at this place
          const uint8_t* unit = s.packed[1] + job_unit(j) * U;
          const uint4 code = *reinterpret_cast<const uint4*>(unit + (D == 64 ? (place * 2 + part) * 16 : (half * UNIT * 4 + place * 4 + part) * 16));
          const uint32_t w[4] = {code.x, code.y, code.z, code.w};
          const uint8_t* meta = unit + Gm::CODES + 4 * ((tok >> 1) * G + half * 4);
          uint32_t s4[4], l4[4];
          if (D == 64) {
            const uint2 a = *reinterpret_cast<const uint2*>(meta), b = *reinterpret_cast<const uint2*>(meta + 2 * G * UNIT);
            s4[0] = a.x; s4[1] = a.y; l4[0] = b.x; l4[1] = b.y;
          } else {
            const uint4 a = *reinterpret_cast<const uint4*>(meta), b = *reinterpret_cast<const uint4*>(meta + 2 * G * UNIT);
            s4[0] = a.x; s4[1] = a.y; s4[2] = a.z; s4[3] = a.w; l4[0] = b.x; l4[1] = b.y; l4[2] = b.z; l4[3] = b.w;
          }
          const int key = job_unit(j) * UNIT + tok, at = key0 + it * BN + key;
          const bool seen = at >= k_beg && at < kv_len;         // what no row sees may be anything: it becomes zero
          const uint32_t pick = tok & 1 ? 0x7632u : 0x5410u;
          uint32_t ss[2], mm[2];                               // (group 2 k, group 2 k + 1) of this token
#pragma unroll
          for (int k = 0; k < (D == 64 ? 1 : 2); k++) {
            ss[k] = __byte_perm(s4[2 * k], s4[2 * k + 1], pick);
            mm[k] = __byte_perm(l4[2 * k], l4[2 * k + 1], pick);
          }
          const bool bad = seen && (mm[0] & 0x7fffu) > 0x7c00u;        // a NaN row has it in every group
          nan |= bad;
          if (!seen || bad) ss[0] = ss[1] = mm[0] = mm[1] = 0;
          if (part == 0) s.nan_key[st][key] = bad;
          uint8_t* dst = s.v[st] + half * (2 * C::HALF_K) + key * 128;
#pragma unroll
          for (int k = 0; k < 4; k++) {
            // word k: chunk slot, and which 64 dims of the half
            const int slot = D == 64 ? part * 4 + k : part * 2 + (k >> 1), b64 = D == 64 ? 0 : k & 1, c = v_slot<D>(place, slot);
            *reinterpret_cast<uint4*>(dst + b64 * C::HALF_K + (c ^ (key & 7)) * 16) = widen(w[k], as_half2(ss[b64]), as_half2(mm[b64]));
          }
        }
        const bool any = __any_sync(0xffffffffu, nan);
        if (lane == 0) s.nan_any[st][dw] = any;
        tc::fence_proxy_async();
        tc::mbar_arrive(&s.v_full[st]);
        page = page_next;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
     } else {
      // ================= issuing warp =================
      // All lanes walk together and one issues: what a matrix instruction is given then stays in uniform registers (one lane alone
      // took 118 clocks an instruction, twice what the products take).
      if (n_blk > 0) {
        constexpr uint32_t ID_S = idesc_f16(ROWS, BN), ID_O = idesc_f16(ROWS, D) | (1u << 16);
        const bool one = tc::elect_one();
        const uint64_t dq = tc::umma_desc_sw128(tc::smem_u32(s.q[0])), dk = tc::umma_desc_sw128(tc::smem_u32(s.k[0])),
                       dv = desc_v(tc::smem_u32(s.v[0]), C::HALF_K);
        auto scores = [&](int t, int it) {
          const uint64_t a = dq + (uint64_t)(t * (C::Q_TILE >> 4)), b = dk + (uint64_t)((it & 1) * (C::KV_TILE >> 4));
          const uint32_t d = tmem + C::S_COL + t * BN;
          if (one) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++)
              tc::umma_bf16(d, a + (((ks >> 2) * C::HALF_Q + (ks & 3) * 32) >> 4), b + (((ks >> 2) * C::HALF_K + (ks & 3) * 32) >> 4), ID_S, ks > 0);
            tc::umma_commit(&s.s_full[t]);
            if (t == tiles - 1) tc::umma_commit(&s.k_empty[it & 1]);
          }
          __syncwarp();
        };
        bool ok = tc::mbar_wait(&s.k_full[0], 0);
        if (ok) {
          tc::tc_fence_after();
#pragma unroll
          for (int t = 0; t < TILES; t++)
            if (t < tiles) scores(t, 0);
        }
#pragma unroll 1
        for (int it = 0; it < n_blk && ok; it++) {
          const uint64_t v = dv + (uint64_t)((it & 1) * (C::KV_TILE >> 4));
#pragma unroll
          for (int t = 0; t < TILES; t++) {
            if (t >= tiles || !ok) continue;
            ok = (t > 0 || tc::mbar_wait(&s.v_full[it & 1], (it >> 1) & 1)) && tc::mbar_wait(&s.p_ready[t], it & 1);
            if (!ok) continue;
            tc::tc_fence_after();
            if (one) {
#pragma unroll
              for (int ks = 0; ks < BN / 16; ks++)
                umma_ts(tmem + C::O_COL + t * D, tmem + C::S_COL + t * BN + ks * 8, v + (uint64_t)(ks * 2048 >> 4), ID_O, it > 0 || ks > 0);
              tc::umma_commit(&s.pv_done[t]);
              if (t == tiles - 1) tc::umma_commit(&s.v_empty[it & 1]);
            }
            __syncwarp();
            if (it + 1 < n_blk) {
              // S of the next block takes the place of P: behind the product that reads it
              ok = (t > 0 || tc::mbar_wait(&s.k_full[(it + 1) & 1], ((it + 1) >> 1) & 1)) && tc::mbar_wait(&s.pv_done[t], it & 1);
              if (!ok) continue;
              tc::tc_fence_after();
              scores(t, it + 1);
            }
          }
        }
        if (!ok) {
          if (one) {
            atomicExch(p.err, tc::ERR_FULL_TIMEOUT);
            tc::umma_commit(&s.drained);
          }
          __syncwarp();
          tc::mbar_wait(&s.drained, 0, 1u << 16);
        }
      }
     }
    } else {
      // ================= softmax warpgroup of tile t, a row per thread =================
      const int t = warp >> 2, r = tid & (ROWS - 1), row = row0 + t * ROWS + r;
      if (t < tiles) {
        const bool valid = row < n_rows;
        const int pos = pos0 + (valid ? row : n_rows - 1) / per;
        const int hi = min(kv_len, pos + 1), lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
        // keys that every row of the tile sees
        const int hi_all = min(kv_len, pos0 + (row0 + t * ROWS) / per + 1);
        const int lo_all = p.window > 0 ? pos0 + (min(row0 + (t + 1) * ROWS, n_rows) - 1) / per + 1 - p.window : 0;
        const float c = s.row_scale[t * ROWS + r];
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_col = lanes + C::S_COL + t * BN, o_col = lanes + C::O_COL + t * D;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        // a NaN row of values: zero in the tile, so that rows which do not see it stay clean; the others become NaN here
        auto look_at_values = [&](int it, int a, int b) {
          if (!tc::mbar_wait(&s.v_full[it & 1], (it >> 1) & 1)) return false;
          const uint4* any = reinterpret_cast<const uint4*>(s.nan_any[it & 1]);
          const uint4 p0 = any[0], p1 = any[1];
          if (p0.x | p0.y | p0.z | p0.w | p1.x | p1.y | p1.z | p1.w)
            for (int i = max(a, 0); i < min(b, BN); i++)
              if (s.nan_key[it & 1][i]) l = __int_as_float(0x7fc00000);
          return true;
        };
        for (int it = 0; it < n_blk; it++) {
          const int kb = key0 + it * BN, a = lo - kb, b = hi - kb;            // visible: [a, b) of the block
          // (the values are there before the scores, but for the first block's: 4% of the time went to looking at them last)
          ok = (it == 0 || look_at_values(it, a, b)) && tc::mbar_wait(&s.s_full[t], it & 1);
          if (!ok) break;
          tc::tc_fence_after();
          const bool cut = kb < lo_all || kb + BN > hi_all;
          float v[64], mx = -INFINITY;
          // 64 columns at a time, the first ones last: they stay in registers for their exponentials
          auto columns = [&](int h) {
            tc::tmem_ld32(s_col + h * 64, v);
            tc::tmem_ld32(s_col + h * 64 + 32, v + 32);
            tc::tmem_ld_wait();
            if (cut) {
#pragma unroll
              for (int k = 0; k < 2; k++) {
                const int x = min(max(a - h * 64 - k * 32, 0), 32), y = min(max(b - h * 64 - k * 32, 0), 32);     // visible: [x, y) of these 32
                const uint32_t seen = (y < 32 ? (1u << y) - 1 : ~0u) & (x < 32 ? ~0u << x : 0u);
#pragma unroll
                for (int i = 0; i < 32; i++)
                  if (!(seen >> i & 1)) v[k * 32 + i] = -INFINITY;
              }
            }
          };
#pragma unroll 1
          for (int h = BN / 64 - 1; h >= 0; h--) {
            columns(h);
            float m4[4] = {mx, v[0], v[1], v[2]};
#pragma unroll
            for (int i = 3; i + 1 < 64; i += 2) m4[(i / 2) & 3] = max3(m4[(i / 2) & 3], v[i], v[i + 1]);
            mx = max3(fmaxf(m4[0], v[63]), m4[1], fmaxf(m4[2], m4[3]));
          }
          const float m_new = fmaxf(m, mx * c);
          if (__any_sync(0xffffffffu, m_new > m + GROWTH)) {
            const float alpha = m == -INFINITY ? 1.f : ex2(m - m_new);       // (nothing summed yet: zeros, or nothing written)
            m = m_new;
            l *= alpha;
            if (it > 0) {
#pragma unroll 1
              for (int h = 0; h < D / 32; h++) {
                float o[32];
                tc::tmem_ld32(o_col + h * 32, o);
                tc::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= alpha;
                tmem_st16(o_col + h * 32, reinterpret_cast<const uint32_t*>(o));
                tmem_st16(o_col + h * 32 + 16, reinterpret_cast<const uint32_t*>(o) + 16);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.f : m;
          float2 l2 = make_float2(0.f, 0.f);
          const float2 c2 = make_float2(c, c), ref2 = make_float2(-ref, -ref);
#pragma unroll 1
          for (int h = 0; h < BN / 64; h++) {
            if (h > 0) columns(h);
#pragma unroll
            for (int k = 0; k < 2; k++) {
              uint32_t packed[16];
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float2 y = fma2(make_float2(v[k * 32 + i], v[k * 32 + i + 1]), c2, ref2), e = make_float2(ex2(y.x), ex2(y.y));
                l2 = add2(l2, e);
                packed[i >> 1] = pack_half2(e.x, e.y);
              }
              tmem_st16(s_col + h * 32 + k * 16, packed);
            }
          }
          l += l2.x + l2.y;
          if (it == 0 && !(ok = look_at_values(it, a, b))) break;
          tmem_st_wait();
          tc::tc_fence_before();
          tc::mbar_arrive(&s.p_ready[t]);
        }
        if (ok && n_blk > 0) ok = tc::mbar_wait(&s.pv_done[t], (n_blk - 1) & 1);
        tc::tc_fence_after();
        if (!ok) {
          if (lane == 0) atomicExch(p.err, tc::ERR_ACC_TIMEOUT);
        } else {
          const int head = kvh * per + (valid ? row : 0) % per;
          const size_t at = (size_t)(q0 + (valid ? row : 0) / per) * p.Hq + head;
          float inv = 1.f;
          if (p.splits > 1) {
            const size_t part = (size_t)blockIdx.z * p.T * p.Hq + at;
            if (valid) p.part_ml[part] = make_float2(m, l);
          } else {
            float sum = l;
            if (p.sinks && (l != 0.f)) sum += ex2(sink_log2(p, head) - m);
            inv = sum == 0.f ? 0.f : 1.f / sum;
          }
#pragma unroll 1
          for (int h = 0; h < D / 64; h++) {
            float o[64];
            if (n_blk > 0) {
              tc::tmem_ld32(o_col + h * 64, o);
              tc::tmem_ld32(o_col + h * 64 + 32, o + 32);
              tc::tmem_ld_wait();
            } else {
#pragma unroll
              for (int i = 0; i < 64; i++) o[i] = 0.f;
            }
            if (valid) {
              // column 2 i + e is dim 32 e + i of these 64
              if (p.splits > 1) {
                float* dst = p.parts + ((size_t)blockIdx.z * p.T * p.Hq + at) * D + h * 64;
#pragma unroll
                for (int i = 0; i < 64; i += 4) {
                  const int e = i / 32, k = 2 * (i % 32) + e;
                  *reinterpret_cast<float4*>(dst + i) = make_float4(o[k], o[k + 2], o[k + 4], o[k + 6]);
                }
              } else {
                __nv_bfloat16* dst = p.out + at * D + h * 64;
#pragma unroll
                for (int i = 0; i < 64; i += 8) {
                  const int e = i / 32, k = 2 * (i % 32) + e;
                  uint32_t w[4];
#pragma unroll
                  for (int j = 0; j < 4; j++) {
                    const __nv_bfloat162 x = __floats2bfloat162_rn(o[k + 4 * j] * inv, o[k + 4 * j + 2] * inv);
                    w[j] = *reinterpret_cast<const uint32_t*>(&x);
                  }
                  *reinterpret_cast<uint4*>(dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
                }
              }
            }
          }
        }
      }
    }
  }
  if (blockIdx.z == 0)                                         // they are zero
    for (int t = behind + blockIdx.x; t < p.T; t += gridDim.x)
      for (int i = tid; i < per * D / 8; i += C::THREADS)
        reinterpret_cast<uint4*>(p.out + ((size_t)t * p.Hq + kvh * per) * D)[i] = make_uint4(0, 0, 0, 0);
  tc::tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, C::TMEM);
  }
}

// The splits of a row become one: a warp per (row, head).
template <int D> __global__ void __launch_bounds__(256) kv4_prompt_merge_kernel(const Params p) {
  constexpr int V = D / 32;
  pdl_trigger();
  pdl_wait();
  const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5), n = (long)p.T * p.Hq;
  const int lane = threadIdx.x & 31;
  if (w >= n || w / p.Hq >= p.cu_q[p.B]) return;
  float m = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
  for (int j = 0; j < V; j++) acc[j] = 0.f;
  for (int i = 0; i < p.splits; i++) m = fmaxf(m, p.part_ml[i * n + w].x);
#pragma unroll 4
  for (int i = 0; i < p.splits; i++) {
    const float2 ml = p.part_ml[i * n + w];
    const float f = ml.x == -INFINITY ? (ml.y != ml.y ? ml.y : 0.f) : ex2(ml.x - m);
    sum += f * ml.y;
    const float* src = p.parts + (i * n + w) * D + lane * 2;
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + 32 * j);
      acc[j] = fmaf(f, v.x, acc[j]);
      acc[j + 1] = fmaf(f, v.y, acc[j + 1]);
    }
  }
  if (p.sinks && sum != 0.f) sum += ex2(sink_log2(p, (int)(w % p.Hq)) - m);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < V; j += 2)
    *reinterpret_cast<__nv_bfloat162*>(p.out + w * D + 32 * j + lane * 2) = __floats2bfloat162_rn(acc[j] * inv, acc[j + 1] * inv);
}

template <int D> long n_tiles(int T_, int B, int per) { return ((long)T_ * per + Cfg<D>::TILES * ROWS - 1) / (Cfg<D>::TILES * ROWS) + B; }

// How many CTAs share a row tile's keys.  One CTA an SM: a grid takes as many waves as it has times 148, each as long as its
// blocks and some 4 blocks' time (256-wide heads: 7) around them, and the parts are written and read once more (a block takes 2.1 to 2.8 us).  The
// least of that, with 4 blocks a split at least.  32 heads of 128 over 8, 30000 keys (us): 200 new tokens 4 splits 178, 5 splits 262,
// 8 splits 190; 400 new tokens 2 splits 331, 3 splits 429, 5 splits 285, 8 splits 340.
template <int D> int splits_of(int T_, int B, int Hq, int Hkv, long keys) {
  const long items = (n_tiles<D>(T_, B, Hq / Hkv) - (B > 1 ? B / 2 : 1)) * Hkv, blocks = (keys + Cfg<D>::BN - 1) / Cfg<D>::BN;
  int best = 1;
  double least = 1e30;
  for (int n = 1; n <= 32 && (n == 1 || (items * n <= 3 * 148 && blocks >= 4 * n)); n++) {
    const double merge = n > 1 ? (double)n * T_ * Hq * D * 8 / 1e7 : 0;        // in blocks' time, as all here
    const double t = (double)((items * n + 147) / 148) * ((blocks + n - 1) / n + (D == 256 ? 7 : 4)) + merge;
    if (t < least) { least = t; best = n; }
  }
  return best;
}

template <int D> int launch(Params& p, cudaStream_t st) {
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  const size_t smem = sizeof(Smem<D>) + 1024;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(kv4_prompt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return -3;
    ready[dev] = true;
  }
  const long tiles = n_tiles<D>(p.T, p.B, p.Hq / p.Hkv);
  if (tiles > 0x7fffffffL || p.Hkv > 65535) return -2;
  cudaError_t e = launch_pdl(kv4_prompt_kernel<D>, dim3((unsigned)tiles, p.Hkv, p.splits), dim3(Cfg<D>::THREADS), smem, st, p);
  if (e != cudaSuccess) return (int)e;
  EXO_CHECK_LAUNCH();
  if (p.splits > 1) {
    e = launch_pdl(kv4_prompt_merge_kernel<D>, dim3((unsigned)(((long)p.T * p.Hq + 7) / 8)), dim3(256), 0, st, p);
    if (e != cudaSuccess) return (int)e;
    EXO_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

// CTAs that share a row tile's keys (1: no scratch wanted); the scratch is splits * T * Hq * (D + 2) floats.
EXO_API int exo_kv4_prompt_splits(int T_, int B, int Hq, int Hkv, int D, int max_blocks, int block_size) {
  if (T_ <= 0 || B <= 0 || Hkv <= 0 || Hq % Hkv) return 1;
  const long keys = (long)max_blocks * block_size;
  return D == 64 ? splits_of<64>(T_, B, Hq, Hkv, keys) : D == 128 ? splits_of<128>(T_, B, Hq, Hkv, keys) : splits_of<256>(T_, B, Hq, Hkv, keys);
}

// An AttnCall: q, out [T, Hq, D] bf16; rows of sequence b: cu_q[b] .. cu_q[b + 1], its last at position seq_lens[b] - 1.
EXO_API int exo_kv4_prompt(const void* call, int bytes, cudaStream_t st) {
  AttnCall c;
  if (!unpack_call(c, call, bytes)) return -2;
  const int T_ = c.T, B = c.B, Hq = c.Hq, Hkv = c.Hkv, D = c.D, n_blocks = c.n_blocks, max_blocks = c.max_blocks, block_size = c.block_size;
  if (T_ == 0) return 0;
  if (T_ < 0 || B <= 0 || Hkv <= 0 || Hq % Hkv || block_size <= 0 || block_size % UNIT || n_blocks <= 0 || max_blocks <= 0 || c.splits < 1 || (c.splits > 1 && !c.ws)) return -2;
  int* err = exo_tc_err_ptr();
  if (!err) return -4;
  Params p;
  p.q = (const __nv_bfloat16*)c.q; p.kcache = (const uint8_t*)c.kcache; p.vcache = (const uint8_t*)c.vcache;
  p.tables = c.tables; p.seq_lens = c.seq_lens; p.cu_q = c.cu_q; p.out = (__nv_bfloat16*)c.out; p.err = err;
  p.parts = (float*)c.ws;
  p.part_ml = (float2*)((float*)c.ws + (size_t)c.splits * T_ * Hq * D);
  p.sinks = c.sinks; p.scale = c.scale; p.sink_dtype = c.sink_dtype;
  p.T = T_; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.n_blocks = n_blocks; p.max_blocks = max_blocks;
  p.units_per_block = block_size / UNIT; p.window = c.window; p.splits = c.splits;
  if (D == 64) return launch<64>(p, st);
  if (D == 128) return launch<128>(p, st);
  if (D == 256) return launch<256>(p, st);
  return -2;
}
