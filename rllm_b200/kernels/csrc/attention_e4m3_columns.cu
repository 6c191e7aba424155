// Paged causal attention over a cache that is kept in 8 bits (kv_e4m3.cuh) on tcgen05 with the cache's own bytes as operands, for
// sequences that bring few tokens: up to 32 rows of a kv head (a row is a (token, head of its group) pair) at a time.  Contract
// as in attention_e4m3.cu.
//
// Both products have the cache as their first operand, whose 128 rows the tensor core wants anyway, and the rows as columns:
//   S [128 keys x columns] = K Q^T (K as it lies in the pages),   O [head dims x columns] += V^T P^T (V too, read MN-major).
// So keys and values go from memory to the tensor core without passing a register: the mma.sync kernel spends most of its
// instructions on making halves of them, whatever the rows are.  kind::f8f6f4 wants the other operand in e4m3 as well, and it
// has to be worth bfloat16 and 11 bits: it is taken apart into terms, each in columns of its own, that are added up afterwards
//   Q   y = q 2^(7 - e), 2^e the row's largest power: T1 = e4m3(y), T2 = e4m3(32 (y - T1)).  Exact for a bfloat16 number down to
//       2^-13 of the row's largest, and off by 2^-22 of that at most;
//   P   W = p 2^ev over a reference of the row's own (which also makes one factor of weight and value's power): a half, then
//       T1 = e4m3(W), T2 = e4m3(32 (W - T1)), and two more in the same way: all 11 bits of a half, down to its smallest numbers,
//       2^-26 of the row's largest weight.
// (kind::f8f6f4 adds products of e4m3 with errors of 2^-21 of their absolute sum, measured over 128 of them that lay 2^17 apart.)
//
//   four warps for every eight rows, a thread a key (= TMEM lane): scores from TMEM, key's power, mask, both references, weights, terms, into shared
//               memory.  References move for all four warps at once, behind a vote a tile.  A value row that is not to be
//               read is cleared by its thread (bytes of NaN there would reach every row).
//   a warp      that allocates TMEM and issues the products; S of the tile after next follows P V of this one.
//   two warps   for K, V and their scales by asynchronous copies of 16 bytes (a tile is eight pages or more: boxes of 1 or 2 KB, and
//               scales of 16 bytes, were no faster by TMA).
// A tile is 128 lines of 128 bytes.  Heads of 64 have two keys in a line: a thread has both, S has columns of their own for the
// even keys (the lines' first 64 bytes) and the odd ones, and O too, of all 128 "dims" of a line, of which the halves that mix the
// two are left where they are (the tensor core has time).
// A cluster shares the keys of a (sequence, kv head, tile of rows); parts are merged in shared memory as in attention_e4m3.cu.
//
// What bounds it: memory for heads of 128 (64 sequences of 8,191 keys, 8 kv heads of four rows: 159 us, 6.8 TB/s of reads over two caches
// of 1.1 GB in turn; a single cold launch 6.0; the mma.sync kernel 224).  For heads of 64 a key has half the bytes and the same work for a thread (two exponentials and nine conversions for every two
// rows, seven of them at half and a quarter of the ALU's rate): 96 us, 5.7 TB/s (120), and 18 us for 24 rows of 8 sequences of 4,095 (30).
// Over few keys the way to the first tile's result, 6 us, is longer than the mma.sync kernel's.  Every sequence has clusters of one size,
// which goes by the number of sequences: one long sequence among many short ones is walked by few CTAs (63 of 500 keys and one of 32,768,
// heads of 128: 187 us, where chunks of a sequence's own length, as over the run's own type, take 89).
#include "attention_tcgen05.cuh"
#include "kv_e4m3.cuh"
#include <cooperative_groups.h>
#include <math.h>

#define EC_PRODUCERS 64
#define EC_SLACK 6.0f                // log2 of how far a weight may pass the row's reference: a vote that moves one costs a tile's time
#define EC_SHIFT 2.0f                // log2 of the weights' factor: a weight stays at or below 2^8
#define EC_SCORES 34.0f              // a score may pass its reference by 2^40: it is only for the sum of the weights, which is float32
#define EC_NONE -3.0e38f             // the reference of a row that has seen nothing
// References are whole numbers, the weights' relative to the scores': s - m is exact where it matters, however large scores are, and so is
// what a reference's move multiplies by.

template <int D, int NB, bool MANY> struct EcShape {
  static constexpr int R = 8 * NB, QN = 16 * NB;                       // rows; columns of S
  static constexpr int PC = 2 * NB, PN = 16 * PC;                      // planes of 16 of the weights' columns: two terms of eight rows each
  static constexpr int PAR = 128 / D, TN = 128 * PAR, ON = PN * PAR;   // keys a line and a tile; columns of O
  static constexpr int CTAS = NB <= 2 ? 2 : 1, THREADS = 128 * NB + 32 + EC_PRODUCERS;       // of an SM
  // Two CTAs of two stages leave 50 KB of an SM, and one of three or four as much: the next kernel's CTAs come in beside them on every
  // SM alike.  Where none fit, they gather on the SMs that are free first (a layer's two products, write and attention, 8 sequences of
  // 2,048 keys, heads of 128: 52 us with three stages, 34 with two, 37 with the mma.sync kernel).  MANY: more CTAs than have room at a
  // time keep memory busier with three (64 of 8,191: 172 -> 160 us).
  static constexpr int STAGES = MANY ? 3 : NB == 3 || (NB == 4 && D == 128) ? 4 : NB == 4 ? 3 : 2;
  static constexpr int TILE = 128 * 128, P_BYTES = ON * 128, SLOT = 2 * TN;                  // SLOT: a tile's scales
  static constexpr int COLUMNS = 2 * QN * PAR + ON;
  static constexpr int TMEM = COLUMNS <= 64 ? 64 : COLUMNS <= 128 ? 128 : COLUMNS <= 256 ? 256 : 512;
  static constexpr int SMEM = 2 * STAGES * TILE + QN * D + 2 * P_BYTES + 2 * STAGES * SLOT + 448 + R * (12 + 8 + 8 + 32 + 16);
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024 && SMEM <= 227 * 1024, "so many CTAs have room on an SM");
  static_assert(PAR * R * D * 4 <= 2 * STAGES * TILE, "the parts lie where keys and values were");
};

__device__ __forceinline__ unsigned long long ec_mul2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ unsigned ec_e4m3(unsigned halves) {          // two halves as e4m3, the low one in the low byte
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(halves));
  return r;
}
__device__ __forceinline__ unsigned long long ec_desc(const void* p, int leading, int stride, int layout) {
  return (unsigned long long)((tg_smem(p) >> 4) & 0x3FFF) | (unsigned long long)(leading >> 4) << 16 |
         (unsigned long long)(stride >> 4) << 32 | (unsigned long long)1 << 46 | (unsigned long long)layout << 61;
}
__device__ __forceinline__ void ec_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void ec_ld16(unsigned taddr, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                 "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ec_ld8(unsigned taddr, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ec_st8(unsigned taddr, const float* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]) : "memory");
}
__device__ __forceinline__ void ec_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ec_copy16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ec_copied(void* bar) {                  // this thread's arrival, when its copies have landed
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tg_smem(bar)) : "memory");
}
// the four softmax warps of eight rows
__device__ __forceinline__ void ec_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
__device__ __forceinline__ bool ec_any(int group, bool x) {
  unsigned r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r) : "r"((unsigned)x), "r"(1 + group) : "memory");
  return r != 0;
}
// The sums (or maxima; NaN is passed over) of eight numbers over a warp's lanes, each left in the lanes whose low three bits give
// `row`: lanes trade halves, nine exchanges where one number after another would take forty.
template <bool MAX> __device__ __forceinline__ float ec_fold(const float* v, int lane, int* row) {
  auto join = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i];
  int at = 0;
#pragma unroll
  for (int n = 4, d = 1; n >= 1; n /= 2, d *= 2) {
    const bool up = lane & d;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? x[i + n] : x[i], send = up ? x[i] : x[i + n];
      x[i] = join(keep, __shfl_xor_sync(0xffffffffu, send, d));
    }
    at += up ? n : 0;
  }
  x[0] = join(x[0], __shfl_xor_sync(0xffffffffu, x[0], 8));
  *row = at;
  return join(x[0], __shfl_xor_sync(0xffffffffu, x[0], 16));
}

template <int D, int NB, bool MANY>
__global__ void __launch_bounds__(EcShape<D, NB, MANY>::THREADS, EcShape<D, NB, MANY>::CTAS)
attention_e4m3_columns_kernel(const bf16* q, int q_stride, bf16* __restrict__ out, const unsigned char* kcache, const unsigned char* vcache,
                              const unsigned char* kscale, const unsigned char* vscale, const int* __restrict__ block_table, int max_blocks, const int* __restrict__ q_start,
                              const int* __restrict__ seq_lens, int seq_begin, int nq, int nkv, int page_size, int num_pages, int window,
                              float scale_log2, int q_wide, int known, int* __restrict__ err) {
  typedef EcShape<D, NB, MANY> X;
  constexpr int R = X::R, NS = X::STAGES, PAR = X::PAR, PLANE = 128 * 16, TN = X::TN, MMA = 4 * NB;      // MMA: that warp
  extern __shared__ __align__(1024) unsigned char ec_raw[];
  kv8_inputs(known, block_table, q_start, seq_lens);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, tid = threadIdx.x;
  const int C = gridDim.x, rank = blockIdx.x;              // the cluster is the grid's x
  const int kvh = blockIdx.y % nkv, s = seq_begin + blockIdx.z, g = nq / nkv;
  const int qs = q_start[s], qlen = q_start[s + 1] - qs, len = seq_lens[s];
  const int rows = qlen * g, r0 = (int)(blockIdx.y / nkv) * R;
  if (r0 >= rows || (tg_smem(ec_raw) & 1023u)) {           // (the whole cluster)
    if (r0 < rows && tid == 0) atomicOr(err, 32);
    pdl_wait();
    return;
  }
  const int pos0 = len - qlen, t_first = r0 / g, t_last = (min(r0 + R, rows) - 1) / g;
  const int hi_first = pos0 + t_first + 1, kend = (int)min((long long)pos0 + t_last + 1, (long long)max_blocks * page_size);
  const int kmin = window > 0 ? max(0, hi_first - window) : 0, lo_last = window > 0 ? max(0, pos0 + t_last + 1 - window) : 0;
  const int all_lo = kmin / TN, all = max(0, (kend + TN - 1) / TN - all_lo);
  const int tile_lo = all_lo + (int)((long long)all * rank / C), n = all_lo + (int)((long long)all * (rank + 1) / C) - tile_lo;
  unsigned char *sK = ec_raw, *sV = sK + NS * X::TILE, *sQ = sV + NS * X::TILE, *sP = sQ + X::QN * D;
  // [2 NS][keys', values'][TN] scale bytes: they come with the keys and are read until the weights are made, when the keys of NS tiles
  // on may have come
  unsigned char* sS = sP + 2 * X::P_BYTES;
  unsigned long long* bars = (unsigned long long*)(sS + 2 * NS * X::SLOT);
  unsigned long long *k_full = bars, *k_empty = bars + 8, *v_full = bars + 16, *v_empty = bars + 24;      // [NS <= 8] each
  unsigned long long *s_full = bars + 32, *p_full = bars + 34, *pv_full = bars + 36, *q_full = bars + 38;  // [2] each, q_full one
  unsigned* tmem_slot = (unsigned*)(bars + 39);
  unsigned* held = (unsigned*)(bars + 40);                 // [2 NS]: a bit for every 16 keys that were brought
  // every eight rows' factors f, and, negative, their scores' references m and, relative to m, their weights' t: [NB][3][8]
  float* info = (float*)((unsigned char*)bars + 448);
  float2* moved = (float2*)(info + 3 * R);                     // [R]: what the row's sum and its output are multiplied by
  int2* sight = (int2*)(moved + R);                        // [R]: the first key it sees, and the one behind its last
  float2* tops = (float2*)(sight + R);                     // [4][R]: the warps' largest score and weight; at the end their sums
  float* cM = (float*)(tops + 4 * R);                      // [3][R]: the CTA's references and sum
  const int* bt = block_table + (size_t)s * max_blocks;
  const int page_shift = (page_size & (page_size - 1)) == 0 ? __ffs(page_size) - 1 : -1;
  auto page_at = [&](int j) { return page_shift >= 0 ? j >> page_shift : j / page_size; };
  auto in_page = [&](int j) { return page_shift >= 0 ? j & (page_size - 1) : j % page_size; };

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init(&k_full[i], EC_PRODUCERS + 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], EC_PRODUCERS); mbar_init(&v_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4 * NB); mbar_init(&pv_full[i], 1); }
    mbar_init(q_full, 4 * NB);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tg_smem(tmem_slot)), "r"(X::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_s = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_o = tmem_s + 2 * X::QN * PAR;
  bool ok = true;

  if (warp < MMA) {
    const int group = warp >> 2, quarter = warp & 3, line = tid & 127;
    typedef unsigned long long pair;                       // two rows' numbers, for instructions that take two
    pair l[4] = {0ull, 0ull, 0ull, 0ull};
    auto notes = [&](int what, pair (&x)[4]) {             // 0: f, 1: -m, 2: -t
      *(ulonglong2*)&x[0] = *(const ulonglong2*)(info + what * 8);
      *(ulonglong2*)&x[2] = *(const ulonglong2*)(info + what * 8 + 4);
    };
    kv8_begin(known, q);
    kv8_let_in(known);
    // queries: L lanes a row, 16 numbers each
    constexpr int L = D / 16;
    {
      const int c = tid % L, r = tid / L, at = r0 + r;
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
      if (r < R && at < rows) {
        const int tok = at / g;
        const bf16* src = q + (size_t)(qs + tok) * q_stride + (size_t)(kvh * g + at - tok * g) * D + c * 16;
        if (q_wide) {
          float a[8], b[8];
          load8(src, a);
          load8(src + 8, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) { x[e] = a[e]; x[e + 8] = b[e]; }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = to_f32(src[e]);
        }
      }
      float top = 0.f, odd = 0.f;                          // odd: NaN if any number is not finite
#pragma unroll
      for (int e = 0; e < 16; ++e) { top = fmaxf(top, fabsf(x[e])); odd = fmaf(x[e], 0.f, odd); }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        odd += __shfl_xor_sync(0xffffffffu, odd, o);
      }
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);
      const float down = __uint_as_float((unsigned)(127 + 7 - e) << 23);
      if (r < R) {
        unsigned w[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y[4], z[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = x[4 * i + k] * down;
          w[0][i] = kv8_pack4(y[0], y[1], y[2], y[3]);
          kv8_floats(w[0][i], z);
          w[1][i] = kv8_pack4((y[0] - z[0]) * 32.f, (y[1] - z[1]) * 32.f, (y[2] - z[2]) * 32.f, (y[3] - z[3]) * 32.f);
        }
#pragma unroll
        for (int term = 0; term < 2; ++term) {
          const int col = (r >> 3) * 16 + term * 8 + (r & 7);
          *(uint4*)(sQ + col * D + ((D == 128 ? c ^ (col & 7) : c ^ (col >> 1 & 3)) << 4)) = make_uint4(w[term][0], w[term][1], w[term][2], w[term][3]);
        }
        if (c == 0) {
          float* note = info + (r >> 3) * 24 + (r & 7);
          note[0] = __uint_as_float((unsigned)(127 - 7 + e) << 23) * scale_log2 + odd;
          note[8] = note[16] = -EC_NONE;
          const int hi = pos0 + min(at, rows - 1) / g + 1;
          sight[r] = make_int2(window > 0 ? hi - window : 0, hi);
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    asm volatile("bar.sync 5, %0;" ::"n"(128 * NB) : "memory");         // (the rows' notes, of all warps)

    info += group * 24; moved += group * 8; sight += group * 8; tops += group * 32;
    const unsigned lane_sel = (unsigned)(quarter * 32) << 16;
    // this thread's half of O: even or odd keys' sums, and its rows' columns
    const unsigned my_o = tmem_o + lane_sel + (PAR == 2 ? (quarter >> 1) * X::PN : 0) + group * 32;
    for (int it = 0; it < n; ++it) {
      const int buf = it & 1, st = it % NS, j0 = (tile_lo + it) * TN, j = j0 + line * PAR, slot = it % (2 * NS);
      // (the tile's scores are there, so its keys and scales are, and the products issued before: the weights' place is free)
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&s_full[buf], (it >> 1) & 1, err));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      pair sc[PAR][4], ev[PAR];
      float kf[PAR];
      {
        float x[PAR][16];
#pragma unroll
        for (int u = 0; u < PAR; ++u) ec_ld16(tmem_s + (buf * PAR + u) * X::QN + group * 16 + lane_sel, x[u]);
        ec_ld_wait();
#pragma unroll
        for (int u = 0; u < PAR; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[u][i] = at_fma2(at_pack2(x[u][8 + 2 * i], x[u][9 + 2 * i]), at_pack2(1.0f / 32, 1.0f / 32), at_pack2(x[u][2 * i], x[u][2 * i + 1]));
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      const bool brought = held[slot] >> (line * PAR >> 4) & 1u;
      bool readable[PAR], all_readable = true;
#pragma unroll
      for (int u = 0; u < PAR; ++u) {
        const int kb = sS[slot * X::SLOT + line * PAR + u], vb = sS[slot * X::SLOT + TN + line * PAR + u];
        // 2^ek (255: infinity, which makes NaN of the row's zeros), NaN where the value is NaN; ev
        kf[u] = vb == KV8_NAN_SCALE ? __uint_as_float(0x7FC00000u) : __uint_as_float((unsigned)kb << 23);
        ev[u] = at_pack2((float)(vb - 127), (float)(vb - 127));
        readable[u] = brought && j + u >= kmin && j + u < kend;
        all_readable = all_readable && readable[u];
      }
      all_readable = __all_sync(0xffffffffu, all_readable);
      {
        pair f[4];
        notes(0, f);
#pragma unroll
        for (int u = 0; u < PAR; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[u][i] = ec_mul2(ec_mul2(sc[u][i], f[i]), at_pack2(kf[u], kf[u]));
      }
      if (!(j0 >= lo_last && j0 + TN <= hi_first && all_readable)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int2 s0 = sight[2 * i], s1 = sight[2 * i + 1];
#pragma unroll
          for (int u = 0; u < PAR; ++u) {
            float a, b;
            at_unpack2(sc[u][i], a, b);
            sc[u][i] = at_pack2(readable[u] && j + u >= s0.x && j + u < s0.y ? a : -INFINITY, readable[u] && j + u >= s1.x && j + u < s1.y ? b : -INFINITY);
          }
        }
      }
      float over = EC_NONE, over2 = EC_NONE;               // how far a score or a weight passes its reference
      {
        pair m[4], t[4];
        notes(1, m);
        notes(2, t);
#pragma unroll
        for (int u = 0; u < PAR; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a, b, c, d;
            const pair s = at_add2(sc[u][i], m[i]);
            at_unpack2(s, a, b);
            at_unpack2(at_add2(s, at_add2(ev[u], t[i])), c, d);
            over = at_max3(over, a, b);
            over2 = at_max3(over2, c, d);
          }
      }
      if (ec_any(group, fmaxf(over - EC_SCORES, over2) > EC_SLACK)) {
        // the rows' largest of `what(keys of a line, pair of rows)` among the keys of all four warps
        auto largest = [&](auto what, bool second) {
          float top[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            at_unpack2(what(0, i), top[2 * i], top[2 * i + 1]);
            if (PAR == 2) {
              float a, b;
              at_unpack2(what(PAR - 1, i), a, b);
              top[2 * i] = fmaxf(top[2 * i], a); top[2 * i + 1] = fmaxf(top[2 * i + 1], b);
            }
          }
          int at;
          const float x = ec_fold<true>(top, lane, &at);
          if (lane < 8) (second ? tops[quarter * 8 + at].y : tops[quarter * 8 + at].x) = x;
          ec_sync(group);
          float t = EC_NONE;
          if (line < 8)
#pragma unroll
            for (int w = 0; w < 4; ++w) t = fmaxf(t, second ? tops[w * 8 + line].y : tops[w * 8 + line].x);
          return t;
        };
        float t = largest([&](int u, int i) { return sc[u][i]; }, false);
        float2 by = make_float2(1.f, 1.f);
        float* note = info + (line & 7);
        if (line < 8 && t + note[8] - EC_SCORES > EC_SLACK) {
          const float down = -note[8] - ceilf(t);
          by.x = at_ex2(down);
          note[8] = -ceilf(t);
          note[16] -= down;                                // (the same place: the output stays as it is)
        }
        ec_sync(group);
        pair m[4];
        notes(1, m);
        t = largest([&](int u, int i) { return at_add2(at_add2(sc[u][i], m[i]), ev[u]); }, true);
        if (line < 8) {
          if (t + note[16] > EC_SLACK) { by.y = at_ex2(-note[16] - ceilf(t)); note[16] = -ceilf(t); }
          moved[line] = by;
        }
        ec_sync(group);
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = ec_mul2(l[i], at_pack2(moved[2 * i].x, moved[2 * i + 1].x));
        if (it > 0) {                                      // the product of the tile before has to be through: it writes what is rescaled
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&pv_full[buf ^ 1], ((it - 1) >> 1) & 1, err));
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            float x[8];
            ec_ld8(my_o + t * 8, x);
            ec_ld_wait();
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] *= moved[r].y;
            ec_st8(my_o + t * 8, x);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
      }
      pair m[4], t_[4];
      notes(1, m);
      notes(2, t_);
#pragma unroll
      for (int u = 0; u < PAR; ++u) {
        unsigned terms[4][4];
        const pair up = at_add2(ev[u], at_pack2(EC_SHIFT, EC_SHIFT));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float a, b, c, d;
          const pair s = at_add2(sc[u][i], m[i]);
          at_unpack2(s, a, b);
          at_unpack2(at_add2(s, at_add2(up, t_[i])), c, d);
          l[i] = at_add2(l[i], at_pack2(at_ex2(a), at_ex2(b)));
          __half2 h = __floats2half2_rn(at_ex2(c), at_ex2(d));
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            terms[t][i] = ec_e4m3(*(const unsigned*)&h);
            const unsigned b = kv8_halves((unsigned short)terms[t][i]);
            h = __hmul2(__hsub2(h, *(const __half2*)&b), __float2half2_rn(32.f));
          }
        }
        unsigned char* dst = sP + buf * X::P_BYTES + (u * X::PC + group * 2) * PLANE + line * 16;
#pragma unroll
        for (int t = 0; t < 4; t += 2)
          *(uint4*)(dst + t / 2 * PLANE) = make_uint4(
              __byte_perm(terms[t][0], terms[t][1], 0x5410), __byte_perm(terms[t][2], terms[t][3], 0x5410),
              __byte_perm(terms[t + 1][0], terms[t + 1][1], 0x5410), __byte_perm(terms[t + 1][2], terms[t + 1][3], 0x5410));
      }
      if (!all_readable && group == 0) {
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&v_full[st], (it / NS) & 1, err));
        unsigned char* v = sV + st * X::TILE + line * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (!readable[c * PAR / 8]) *(uint4*)(v + ((c ^ (line & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
    }
    if (n > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(&pv_full[(n - 1) & 1], ((n - 1) >> 1) & 1, err));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    int at;
    float sums[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) at_unpack2(l[i], sums[2 * i], sums[2 * i + 1]);
    const float sum = ec_fold<false>(sums, lane, &at);
    if (lane < 8) tops[quarter * 8 + at].x = sum;
    ec_sync(group);
    if (line < 8) {
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) all += tops[w * 8 + line].x;
      cM[group * 8 + line] = -info[8 + line];
      cM[R + group * 8 + line] = -info[16 + line];
      cM[2 * R + group * 8 + line] = all;
    }
    // O, its terms added up, as float32 rows [PAR][R][D] where keys and values were (all of them have been read)
    float* mine = (float*)ec_raw + ((PAR == 2 ? (quarter >> 1) * R : 0) + group * 8) * D + (line & (D - 1));
    float x[4][8];
    if (n > 0) {
#pragma unroll
      for (int t = 0; t < 4; ++t) ec_ld8(my_o + t * 8, x[t]);
      ec_ld_wait();
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i / 8][i % 8] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) mine[r * D] = fmaf(fmaf(fmaf(x[3][r], 1.0f / 32, x[2][r]), 1.0f / 32, x[1][r]), 1.0f / 32, x[0][r]);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  } else if (warp == MMA) {
    // ---- products ----
    kv8_begin(known);
    const unsigned id_s = (1u << 4) | (unsigned)(X::QN >> 3) << 17 | (128u >> 4) << 24;
    const unsigned id_o = (1u << 4) | 3u << 15 | (unsigned)(X::ON >> 3) << 17 | (128u >> 4) << 24;
    auto wait = [&](unsigned long long* bar, int phase) {
      const bool there = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, err));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return there;
    };
    auto scores = [&](int it) {                            // (one lane)
      const int st = it % NS;
      // K's lines have 128 bytes in a 128-byte swizzle, the queries' D bytes (heads of 64: 64-byte swizzle)
      const unsigned long long dk = ec_desc(sK + st * X::TILE, 16, 1024, 2), dq = ec_desc(sQ, 16, 8 * D, D == 128 ? 2 : 4);
#pragma unroll
      for (int u = 0; u < PAR; ++u)
#pragma unroll
        for (int k = 0; k < D / 32; ++k) ec_mma(tmem_s + ((it & 1) * PAR + u) * X::QN, dk + u * (D >> 4) + 2 * k, dq + 2 * k, id_s, k > 0);
      umma_commit(&s_full[it & 1]);
      umma_commit(&k_empty[st]);
    };
    // what the copies wrote, for the tensor core
    auto keys = [&](int it) {
      const bool there = wait(&k_full[it % NS], it / NS);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      return there;
    };
    bool go = wait(q_full, 0);
    for (int it = 0; it < 2 && it < n && go; ++it) {
      go = keys(it);
      if (go && umma_elect()) scores(it);
      __syncwarp();
    }
    for (int it = 0; it < n && go; ++it) {
      // (all that can be waited for ahead of the weights is: each wait, though over, is 150 to 250 cycles)
      const int st = it % NS;
      go = wait(&v_full[st], it / NS);
      const bool more = it + 2 < n, early = more && __all_sync(0xffffffffu, mbar_test(&k_full[(it + 2) % NS], ((it + 2) / NS) & 1));
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      go = go && wait(&p_full[it & 1], it >> 1);
      if (!go) break;
      if (umma_elect()) {
        const unsigned long long dv = ec_desc(sV + st * X::TILE, 16, 1024, 2), dp = ec_desc(sP + (it & 1) * X::P_BYTES, 128, PLANE, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) ec_mma(tmem_o, dv + k * (4096 >> 4), dp + k * (512 >> 4), id_o, it > 0 || k > 0);
        umma_commit(&pv_full[it & 1]);
        umma_commit(&v_empty[st]);
        if (early) scores(it + 2);
      }
      __syncwarp();
      if (more && !early) {
        go = keys(it + 2);
        if (go && umma_elect()) scores(it + 2);
        __syncwarp();
      }
    }
  } else {
    // ---- K, V and their scales: eight threads a line of 128 bytes, a line in eight; lane CH u + c looks up keys 16 c .. 16 c + 15
    // of the u-th of AHEAD tiles ----
    constexpr int CH = TN / 16, AHEAD = 32 / CH, LINES = D / 8;           // pieces of 16 keys a tile, tiles a lookup, lines a piece
    const int c = lane % CH, u = lane / CH, p = tid - 128 * NB - 32, c16 = p & 7, line = p >> 3;
    static_assert(EC_PRODUCERS == 64, "a step is eight lines: a thread's place in the swizzle is the same in all");
    auto pages_of = [&](int it) { return bt[min(page_at((tile_lo + it + u) * TN + c * 16), max_blocks - 1)]; };
    auto place_of = [&](int it, int page) {                // the first cache row, or -1: not to be brought
      const int j = (tile_lo + it + u) * TN + c * 16;
      const bool wanted = it + u < n && j + 16 > kmin && j < kend, there = wanted && page >= 0 && page < num_pages;
      if (wanted && !there && warp == MMA + 1) atomicOr(err, 4);
      return there ? (page * nkv + kvh) * page_size + in_page(j) : -1;
    };
    int ahead = pages_of(0), place = -1;
    kv8_begin(known, kcache, vcache, kscale, vscale);
    const unsigned to = line * 128 + ((c16 ^ line) << 4);
    auto bring = [&](const unsigned char* stage, const unsigned char* cache, int it) {
      const unsigned dst = tg_smem(stage) + to;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = __shfl_sync(0xffffffffu, place, it % AHEAD * CH + i * 8 / LINES);
        if (at >= 0) ec_copy16(dst + i * 1024, cache + (long long)at * D + (i * 8 % LINES + line) * 128 + c16 * 16);
      }
    };
    for (int it = 0; it < n && ok; ++it) {
      if (it % AHEAD == 0) {
        place = place_of(it, ahead);
        ahead = pages_of(it + AHEAD);
      }
      const int st = it % NS;
      ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], ((it / NS) & 1) ^ 1, err));
      if (!ok) break;
      bring(sK + st * X::TILE, kcache, it);
      if (warp == MMA + 1) {
        const int at = __shfl_sync(0xffffffffu, place, it % AHEAD * CH + c), slot = it % (2 * NS);
        const unsigned there = __ballot_sync(0xffffffffu, at >= 0) & ((1u << CH) - 1);
        if (u < 2 && at >= 0) ec_copy16(tg_smem(sS + slot * X::SLOT + lane * 16), (u == 0 ? kscale : vscale) + at);
        if (lane == 0) {
          held[slot] = there;
          mbar_arrive(&k_full[st]);
        }
      }
      ec_copied(&k_full[st]);
      ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ((it / NS) & 1) ^ 1, err));
      if (!ok) break;
      bring(sV + st * X::TILE, vcache, it);
      ec_copied(&v_full[st]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(X::TMEM) : "memory");

  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  if (C > 1) cluster.sync();
  for (int i = (rank * X::THREADS + tid) * 4; i < R * D; i += C * X::THREADS * 4) {
    const int r = i / D, col = i - r * D, at = r0 + r;
    if (at >= rows) break;
    float top = EC_NONE, high = -INFINITY, sum = 0.f;      // the references of the sum and, relative to it, of the weights
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float* part, float by) {
#pragma unroll
      for (int p = 0; p < PAR; ++p) {
        const float4 y = *(const float4*)(part + p * R * D + i);
        x.x = fmaf(y.x, by, x.x); x.y = fmaf(y.y, by, x.y); x.z = fmaf(y.z, by, x.z); x.w = fmaf(y.w, by, x.w);
      }
    };
    if (C == 1) {
      high = cM[R + r];
      sum = cM[2 * R + r];
      add((const float*)ec_raw, 1.f);
    } else {
      for (int c = 0; c < C; ++c) {
        const float* m = cluster.map_shared_rank(cM, c);
        kv8_join(top, high, m[r], m[R + r]);
      }
      for (int c = 0; c < C; ++c) {
        const float* m = cluster.map_shared_rank(cM, c);
        sum = fmaf(m[2 * R + r], at_ex2(m[r] - top), sum);
        add(cluster.map_shared_rank((const float*)ec_raw, c), at_ex2(m[R + r] + (m[r] - top) - high));
      }
    }
    // 2^high as two factors, for values near the small end of the range: as one it would be below the normal numbers, which ex2 makes 0
    const float by = high - EC_SHIFT, half = floorf(0.5f * by);
    const float inv = (sum == 0.f ? 0.f : 1.0f / sum) * at_ex2(half), more = at_ex2(by - half);      // NaN stays NaN
    const int tok = at / g;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * inv * more, x.y * inv * more), hi = __floats2bfloat162_rn(x.z * inv * more, x.w * inv * more);
    *(uint2*)(out + ((size_t)(qs + tok) * nq + kvh * g + at - tok * g) * D + col) = make_uint2(*(const unsigned*)&lo, *(const unsigned*)&hi);
  }
  if (C > 1) cluster.sync();                               // nobody leaves while its shared memory is being read
  kv8_end(known);
}

template <int D, int NB, bool MANY = false>
static int ec_launch(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const void* kscale, const void* vscale,
                     const int* block_table, int max_blocks, const int* q_start, const int* seq_lens, int seq_begin, int num_seqs,
                     int max_q_len, int max_keys, int nq, int nkv, int page_size, int num_pages, int window, float scale, int known, int* err,
                     cudaStream_t stream) {
  typedef EcShape<D, NB, MANY> X;
  const long long tiles = ((long long)max_q_len * (nq / nkv) + X::R - 1) / X::R, units = tiles * nkv * num_seqs;
  if (tiles * nkv > 65535 || num_seqs > 65535) return RLLM_E_UNSUPPORTED;
  if constexpr (D == 128 && NB == 1 && !MANY)
    if (units > 148 * X::CTAS)
      return ec_launch<D, NB, true>(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, seq_lens, seq_begin,
                                    num_seqs, max_q_len, max_keys, nq, nkv, page_size, num_pages, window, scale, known, err, stream);
  auto* kernel = attention_e4m3_columns_kernel<D, NB, MANY>;
  static SmemLimit limit;
  if (const int e = limit.allow(kernel, X::SMEM)) return e;
  // CTAs a unit: to fill the GPU's places, of a tile at least; clusters of eight do not fill a GPC's SMs (16 of them, a CTA an SM,
  // took two rounds)
  int C = 1;
  while (C < 8 && units * C * 2 <= (C == 4 ? 112 : 148) * X::CTAS && C * 2 * X::TN <= max_keys) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)C, (unsigned)(tiles * nkv), (unsigned)num_seqs);
  cfg.blockDim = dim3(X::THREADS);
  cfg.dynamicSmemBytes = (size_t)X::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = rllm_pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (const bf16*)q, q_stride, (bf16*)out, (const unsigned char*)kcache,
                                           (const unsigned char*)vcache, (const unsigned char*)kscale, (const unsigned char*)vscale, block_table, max_blocks, q_start, seq_lens, seq_begin, nq, nkv,
                                           page_size, num_pages, window, scale * 1.4426950408889634f,
                                           (((uintptr_t)q | ((uintptr_t)q_stride * 2)) & 15) == 0 ? 1 : 0, known, err);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return 0;
}

// Sequences seq_begin .. seq_end - 1 of bfloat16 queries, of at most max_q_len tokens each; no query sees more than max_keys
// keys; known: see kv8_inputs.  Heads of 64 or 128, pages of a multiple of 16 keys.
RLLM_EXPORT int rllm_attention_e4m3_columns(const void* q, int q_stride, void* out, const void* kcache, const void* vcache,
                                            const void* kscale, const void* vscale, const int* block_table, int max_blocks,
                                            const int* q_start, const int* seq_lens, int seq_begin, int seq_end, int max_q_len,
                                            int max_keys, int nq, int nkv, int d, int page_size, int num_pages, int window,
                                            float scale, int known, int* err, cudaStream_t stream) {
  if (max_q_len <= 0 || seq_end <= seq_begin) return 0;
  if (!q || !out || !kcache || !vcache || !kscale || !vscale || !block_table || !q_start || !seq_lens || !err || max_blocks <= 0 ||
      seq_begin < 0 || nq <= 0 || nkv <= 0 || nq % nkv || page_size <= 0 || num_pages <= 0 || window < 0 || !(scale == scale) ||
      scale > 3e38f || scale < -3e38f)
    return RLLM_E_BADARG;
  if (!(d == 64 || d == 128) || page_size % 16 || (((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)kscale | (uintptr_t)vscale | (uintptr_t)out) & 15))
    return RLLM_E_UNSUPPORTED;
  if ((long long)num_pages * nkv * page_size > 0x7fffffffLL) return RLLM_E_UNSUPPORTED;      // cache rows are counted in 32 bits
  const long long rows = (long long)max_q_len * (nq / nkv);
#define EC_LAUNCH(DD, NBB)                                                                                                             \
  return ec_launch<DD, NBB>(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, seq_lens, seq_begin,   \
                            seq_end - seq_begin, max_q_len, max_keys, nq, nkv, page_size, num_pages, window, scale, known, err, stream)
  if (d == 64) { if (rows <= 8) EC_LAUNCH(64, 1); if (rows <= 16) EC_LAUNCH(64, 2); if (rows <= 24) EC_LAUNCH(64, 3); EC_LAUNCH(64, 4); }
  if (rows <= 8) EC_LAUNCH(128, 1);
  if (rows <= 16) EC_LAUNCH(128, 2);
  if (rows <= 24) EC_LAUNCH(128, 3);
  EC_LAUNCH(128, 4);
}
