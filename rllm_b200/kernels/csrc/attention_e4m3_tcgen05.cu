// Paged causal attention over a cache that is kept in 8 bits (kv_e4m3.cuh) on tcgen05, keys and values widened inside the
// kernel: for sequences that bring up to a few tiles of 128 rows (a row is a (token, head of the kv head's group) pair), where
// widening them for all at once (attention_tcgen05.cu's DENSE form) would cost more traffic than the attention itself, and the
// mma.sync kernel (attention_e4m3.cu), which widens for 16 rows at a time, more instructions.  Contract as there.
//
// A CTA takes 128 rows of one (sequence, kv head) and a part of their keys, in tiles of 64; a cluster shares the keys.
//   warps 0-3   softmax, a thread a row (= TMEM lane): scores from TMEM, mask, running reference and sum in float32, weights as
//               halves back into TMEM; the output stays in TMEM and is rescaled when a reference moves.  Warps without a live
//               row only keep the barriers in step: a few rows cost the exponentials of 32.
//   warps 4-7   widen: copy two tiles of rows ahead into shared memory (a lane its own 16 bytes, asynchronously), and make halves of
//               them there, in the 128-byte swizzle that the products read.
//   warp 9      looks ahead: where the rows of a tile lie, their scales, the tile's largest, as factors and notes for the others
//               (done by every widening warp for itself it was a third of their time: long chains of short instructions).
//   warp 8      allocates TMEM and issues the products: S = Q K^T (128 x 64 x D), O += P V (128 x D x 64, P in TMEM, V as the
//               MN-major operand, straight from its rows).
// Halves, not bfloat16: e4m3 numbers become halves in one instruction a pair, and a weight keeps 11 bits.  Powers of two:
//   K  a row's numbers are multiplied by 2^(ek - EK + 6), EK the largest ek of the tile, and the tile's scores by 2^(EK - 6);
//   V  by 2^(ev - EV + 6), EV the tile's largest, and a weight by 2^EV over a reference of the row's weights with their values' powers,
//      beside that of its scores, as in the mma.sync kernel (both whole numbers, passed by 2^4 at most; 2^11 more, so that the halves'
//      smallest step lies at 2^-35 of the row's largest weight): the factor rides in the exponent's argument, and the sum is divided by it;
//   Q  a row by a power of two of its own, exact for bfloat16 down to 2^-27 of the row's largest.
// A factor 2^(e - E + 6) is a half's normal number, and times an e4m3 number exact, down to e = E - 20.  A tile with rows further apart
// than that ("wide": none in what a model makes) is taken key by key: what a factor lacks multiplies the key's scores, and stands in its
// weights' exponents.  So are rows whose scores are so large that a sum of them and a value's power would be rounded to whole powers.
// 8 sequences of 4,095 keys, 64 rows: heads of 64 29 us, of 128 37; 64 sequences of 8,000, 36 rows: 309 and 363.
// A token whose key or value is NaN has a NaN key and zeros for a value: rows that see it become NaN by the score, and the others'
// products stay clean.
#include "attention_tcgen05.cuh"
#include "kv_e4m3.cuh"
#include <cooperative_groups.h>

#define E8_BM 128
#define E8_BN 64
#define E8_THREADS 320
#define E8_AHEAD 8                   // tiles whose rows and factors are known at a time
#define E8_SLACK 4.0f
#define E8_SHIFT 11                  // log2 of the weights' factor: E8_SLACK + E8_SHIFT = 15
#define E8_LIFT 6                    // log2 of what keys and values are multiplied by beside: 448 2^6 is a half
#define E8_APART 20                  // log2 of how far a tile's rows may lie apart for factors that are halves
#define E8_NONE -3.0e38f             // the reference of a row that has seen nothing
#define E8_LARGE 1048576.f           // whole numbers of this size and of a few hundred more have room in a float32

// Q, the widened stages of K and of V (two each for heads of 64, one for 128: two CTAs fit one SM), two tiles of K and of V as
// they come, barriers and the tiles' notes
template <int D> constexpr int e8_stages() { return D == 64 ? 2 : 1; }
template <int D> constexpr int e8_smem_bytes() { return E8_BM * D * 2 + 2 * e8_stages<D>() * E8_BN * D * 2 + 4 * E8_BN * D + 512 + E8_AHEAD * 1024; }

// what warp 9 finds out about a tile
struct E8Tile {
  int row[E8_BN];                    // a key's cache row; -1: not to be read, or of a page that is not held
  unsigned kf[E8_BN], vf[E8_BN];     // 2^(ek - EK) and 2^(ev - EV') as pairs of halves
  int ek, ev;                        // EK and EV, scale bytes
  int wide;                          // rows lie further apart than E8_APART
  unsigned missing[2];               // a bit a key whose page is not held
  unsigned char kd[E8_BN], vd[E8_BN];      // of a wide one: EK - ek and EV - ev beyond E8_APART
};
static_assert(sizeof(E8Tile) <= 1024, "they lie behind the barriers");

// A row's references: x of its scores; y of its weights with their values' powers, relative to x; z the sum of 2^(score - x).
// They move to what is passed by more than 2^4; a weights' reference that moves changes the output so far, by what is returned.
__device__ __forceinline__ void e8_move_scores(float4& ref, float top) {
  if (top - ref.x > E8_SLACK) {
    top = ceilf(top);
    ref.z *= kv8_two_to(ref.x - top);                      // from nothing: 0, and nothing has been summed yet
    ref.y += ref.x - top;                                  // (the same place: the output stays as it is)
    ref.x = top;
  }
}
__device__ __forceinline__ float e8_move_weights(float4& ref, float top) {
  if (!(top > ref.y + E8_SLACK)) return 1.0f;
  top = ceilf(top);
  const float corr = kv8_two_to(ref.y - top);
  ref.y = top;
  return corr;
}

// A row's part of a tile key by key: the scores t_s of 64 keys, times f and what each key's factor lacks, become weights in their place
// (a function of its own, for the registers and the instructions of the tiles that need none of it: in place they cost 15 %).
// lacks: a wide tile's kd and vd, else null.  Returns the references, w: as e8_move_weights.
__device__ __noinline__ float4 e8_key_by_key(unsigned t_s, const unsigned char* lacks, float f, float ev, unsigned lo_rel, unsigned span,
                                             unsigned missing0, unsigned missing1, float4 ref) {
  float sc[32];
  auto lacks_key = [&](int j) { return lacks ? kv8_two_to(fmaxf(-(float)lacks[j], -126.f)) : 1.0f; };
  auto value_power = [&](int j) { return lacks ? ev - (float)lacks[E8_BN + j] : ev; };
  auto load = [&](int h) {
    tmem_ld32(t_s + h * 32, (unsigned*)sc);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const bool seen = (unsigned)(h * 32 + j) - lo_rel < span && !((h ? missing1 : missing0) >> j & 1u);
      sc[j] = seen ? sc[j] * f * lacks_key(h * 32 + j) : -INFINITY;
    }
  };
  float top = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    load(h);
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, sc[j]);
  }
  e8_move_scores(ref, top);
  top = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    load(h);
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, (sc[j] - ref.x) + value_power(h * 32 + j));
  }
  ref.w = e8_move_weights(ref, top);
  const float base = ref.y - (float)E8_SHIFT;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    load(h);
    unsigned pk[16];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      float w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = sc[j + e] - ref.x;
        ref.z += at_ex2(x);
        w[e] = at_ex2(x + (value_power(h * 32 + j + e) - base));
      }
      const __half2 y = __floats2half2_rn(w[0], w[1]);
      pk[j / 2] = *(const unsigned*)&y;
    }
    tmem_st16(t_s + h * 16, pk);
  }
  return ref;
}

// 2^high without the factors of weights and values, as two: it may lie below the normal numbers
__device__ __forceinline__ float e8_factors(float high, float* more) {
  const float by = fminf(fmaxf(high, -200.f), 200.f), half = floorf(by * 0.5f);
  *more = kv8_two_to(by - half);
  return kv8_two_to(half - (float)(E8_SHIFT + E8_LIFT));
}

template <int D>
__global__ void __launch_bounds__(E8_THREADS, 2)
attention_e4m3_tcgen05_kernel(const bf16* q, int q_stride, bf16* __restrict__ out, const unsigned char* __restrict__ kcache,
                              const unsigned char* __restrict__ vcache, const unsigned char* __restrict__ kscale,
                              const unsigned char* __restrict__ vscale, const int* __restrict__ block_table, int max_blocks,
                              const int* __restrict__ q_start, const int* __restrict__ seq_lens, int seq_begin, int nq, int nkv,
                              int page_size, int num_pages, int window, float scale_log2, int known, int* __restrict__ err) {
  constexpr int DP = D / 64, QPANEL = E8_BM * 128, KPANEL = E8_BN * 128, STAGE = E8_BN * D * 2, NS = e8_stages<D>();
  extern __shared__ __align__(1024) unsigned char e8_raw[];
  kv8_inputs(known, block_table, q_start, seq_lens);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int splits = gridDim.x, rank = blockIdx.x;       // the cluster is the grid's x
  const int kvh = blockIdx.y % nkv, s = seq_begin + blockIdx.z;
  const int g = nq / nkv, bq = E8_BM / g;
  const int qs = q_start[s], qlen = q_start[s + 1] - qs, len = seq_lens[s];
  const int t0 = (int)(blockIdx.y / nkv) * bq;
  if (t0 >= qlen || (tg_smem(e8_raw) & 1023u)) {          // (the whole cluster)
    if (t0 < qlen && threadIdx.x == 0) atomicOr(err, 32);
    pdl_wait();
    return;
  }
  const int ntok = min(bq, qlen - t0), live_rows = ntok * g;
  const int pos0 = len - qlen, first_pos = pos0 + t0;
  const int kend = (int)min((long long)first_pos + ntok, (long long)max_blocks * page_size);
  const int kmin = window > 0 ? max(0, first_pos - window + 1) : 0;
  const int all_lo = kmin / E8_BN, all = max(0, (kend + E8_BN - 1) / E8_BN - all_lo);
  const int tile_lo = all_lo + all * rank / splits, ntiles = all_lo + all * (rank + 1) / splits - tile_lo;
  unsigned char *sQ = e8_raw, *sK = sQ + DP * QPANEL, *sV = sK + NS * STAGE, *sRaw = sV + NS * STAGE;
  unsigned long long* bars = (unsigned long long*)(sRaw + 4 * E8_BN * D);
  unsigned long long *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;      // [2] each
  unsigned long long *s_full = bars + 8, *p_full = bars + 10, *pv_full = bars + 11;                     // s_full: [2]
  unsigned* tmem_slot = (unsigned*)(bars + 12);
  unsigned long long *t_full = bars + 16, *t_free = bars + 16 + E8_AHEAD;               // [E8_AHEAD] each
  E8Tile* tiles = (E8Tile*)((unsigned char*)bars + 512);  // [E8_AHEAD]
  const int* bt = block_table + (size_t)s * max_blocks;
  const int page_shift = (page_size & (page_size - 1)) == 0 ? __ffs(page_size) - 1 : -1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], 1); }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(p_full, 4);
    mbar_init(pv_full, 1);
    for (int i = 0; i < E8_AHEAD; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_free[i], 8); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tg_smem(tmem_slot)), "r"(256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  kv8_begin(known, q, kcache, vcache, kscale, vscale);

  // Queries as halves: a row by 2^(13 - e) with 2^e its largest's power; eight lanes a row (four for heads of 64)
  float my_factor = 0.f;
  {
    constexpr int L = D / 16;                              // lanes a row, 16 values each
    for (int base = 0; base < E8_BM; base += E8_THREADS / 32 * (32 / L)) {
      const int r = base + warp * (32 / L) + lane / L, c = lane % L;
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
      if (r < live_rows) {
        const int tl = r / g;
        const bf16* src = q + (size_t)(qs + t0 + tl) * q_stride + (size_t)(kvh * g + r - tl * g) * D + c * 16;
        float a[8], b[8];
        load8(src, a);
        load8(src + 8, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[e] = a[e]; x[e + 8] = b[e]; }
      }
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);
      const float down = __uint_as_float((unsigned)(127 + 13 - e) << 23);
      if (r < E8_BM) {
        uint4 w[2];
        __half2* h = (__half2*)w;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = __floats2half2_rn(x[2 * i] * down, x[2 * i + 1] * down);
        unsigned char* dst = sQ + (c >> 2) * QPANEL + r * 128;
        *(uint4*)(dst + ((((c & 3) * 2) ^ (r & 7)) << 4)) = w[0];
        *(uint4*)(dst + ((((c & 3) * 2 + 1) ^ (r & 7)) << 4)) = w[1];
        // the row's factor waits in the V ring for the softmax warps (they read it before the first value is widened)
        if (c == 0) ((float*)sV)[r] = __uint_as_float((unsigned)(127 - 13 - E8_LIFT + e) << 23) * scale_log2;
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp < 4) my_factor = ((float*)sV)[threadIdx.x];
  __syncthreads();
  kv8_let_in(known);                                         // behind the allocation: see pdl_launch
  const unsigned tmem_s = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_o = tmem_s + 2 * E8_BN;      // two tiles' scores: 128 + D <= 256 columns

  float4 ref = make_float4(E8_NONE, E8_NONE, 0.f, 1.f);    // see e8_move_scores
  bool ok = true;
  if (warp < 4) {
    const int r = threadIdx.x, tl = r / g;
    const bool warp_live = warp * 32 < live_rows;
    const int pos = first_pos + min(tl, ntok - 1);
    const int row_hi = min(pos + 1, kend), row_lo = window > 0 ? max(0, pos + 1 - window) : 0;
    // tiles all of whose keys every live row sees need no mask
    const int clear_lo = window > 0 ? max(0, first_pos + ntok - window) : 0, clear_hi = min(first_pos + 1, kend);
    const unsigned lane_sel = (unsigned)(warp * 32) << 16;
    for (int it = 0; it < ntiles; ++it) {
      const int j0 = (tile_lo + it) * E8_BN;
      const unsigned t_s = tmem_s + (it & 1) * E8_BN + lane_sel;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[it & 1], (it >> 1) & 1, err));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      struct { int ek, ev, wide; unsigned missing[2]; } note;
      const E8Tile& tile = tiles[it % E8_AHEAD];
      note = {tile.ek, tile.ev, tile.wide, {tile.missing[0], tile.missing[1]}};
      __syncwarp();
      if (!(warp_live && note.wide) && lane == 0) mbar_arrive(&t_free[it % E8_AHEAD]);       // (a wide one's is read to its end)
      if (!warp_live) {
        if (it > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(pv_full, (it - 1) & 1, err));
          if (!ok) break;
        }
        if (lane == 0) mbar_arrive(p_full);
        continue;
      }
      const float f = fmaxf(my_factor * kv8_power(note.ek), 1.2e-38f);     // (a masked score, -inf, times 0 would be NaN)
      const bool masked = !(j0 >= clear_lo && j0 + E8_BN <= clear_hi) || (note.missing[0] | note.missing[1]);
      const unsigned lo_rel = (unsigned)(row_lo - j0), span = (unsigned)max(row_hi - row_lo, 0);
      // the scores come from TMEM twice, 32 at a time, for their maximum and for their exponentials: all 64 at once, and the
      // weights, would not leave registers for two CTAs an SM
      float sc[32];
      auto load = [&](int h) {
        tmem_ld32(t_s + h * 32, (unsigned*)sc);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (masked) {
          const unsigned lo = lo_rel - h * 32, miss = note.missing[h];
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!((unsigned)j - lo < span) || (miss >> j & 1u)) sc[j] = -INFINITY;
        }
      };
      float mx = -INFINITY;                                // the row's largest score
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load(h);
        float mx0 = sc[0], mx1 = sc[1];
#pragma unroll
        for (int j = 2; j < 32; j += 4) {
          mx0 = at_max3(mx0, sc[j], sc[j + 1]);
          if (j + 2 < 32) mx1 = at_max3(mx1, sc[j + 2], sc[j + 3]);
        }
        mx = at_max3(mx, mx0, mx1);
      }
      mx *= f;
      float corr;                                          // what the output so far is multiplied by
      const float ev = (float)(note.ev - 127), reach = fmaxf(mx, ref.x);
      if (note.wide || __any_sync(0xffffffffu, fabsf(reach) > E8_LARGE && reach != E8_NONE)) {
        ref = e8_key_by_key(t_s, note.wide ? tiles[it % E8_AHEAD].kd : nullptr, f, ev, lo_rel, span, note.missing[0], note.missing[1], ref);
        corr = ref.w;
        __syncwarp();
        if (note.wide && lane == 0) mbar_arrive(&t_free[it % E8_AHEAD]);
      } else {
        e8_move_scores(ref, mx);
        corr = e8_move_weights(ref, (mx - ref.x) + ev);
        // weights times 2^(EV - reference + 11), in the place of the scores, and the sum without that factor.  Where it is so small that no
        // weight is above the halves' smallest, 2^-60 of the sum's, the sum keeps its bits (-1000: of a row that has seen nothing)
        const float by = fmaxf(fminf(ref.y - ev - (float)E8_SHIFT, 60.f), -1000.f), base = ref.x + by;
        const unsigned long long scale2 = at_pack2(f, f), shift2 = at_pack2(-base, -base);
        unsigned long long sum01 = at_pack2(0.f, 0.f), sum23 = sum01;
        unsigned pk[2][16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load(h);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            float x0, x1, x2, x3;
            at_unpack2(at_fma2(at_pack2(sc[j], sc[j + 1]), scale2, shift2), x0, x1);
            at_unpack2(at_fma2(at_pack2(sc[j + 2], sc[j + 3]), scale2, shift2), x2, x3);
            const float p0 = at_ex2(x0), p1 = at_ex2(x1), p2 = at_ex2(x2), p3 = at_ex2(x3);
            sum01 = at_add2(sum01, at_pack2(p0, p1));
            sum23 = at_add2(sum23, at_pack2(p2, p3));
            const __half2 h0 = __floats2half2_rn(p0, p1), h1 = __floats2half2_rn(p2, p3);
            pk[h][j / 2] = *(const unsigned*)&h0;
            pk[h][j / 2 + 1] = *(const unsigned*)&h1;
          }
          if (h == 0) tmem_st16(t_s, pk[0]);               // (columns 0 .. 15: scores that have been read; the other half's lie behind)
        }
        tmem_st16(t_s + 16, pk[1]);
        float a, b, c, d;
        at_unpack2(sum01, a, b);
        at_unpack2(sum23, c, d);
        ref.z = fmaf((a + b) + (c + d), kv8_two_to(by), ref.z);
      }
      // the product of the tile before has to be through: it wrote the output that is rescaled here
      if (it > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(pv_full, (it - 1) & 1, err));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (__any_sync(0xffffffffu, corr != 1.0f)) {
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            unsigned* v = (unsigned*)sc;
            tmem_ld32(tmem_o + lane_sel + c0, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
            tmem_st32(tmem_o + lane_sel + c0, v);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (ntiles == 0) ok = false;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(pv_full, (ntiles - 1) & 1, err));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (splits == 1) {
      float more;
      const float inv = (ref.z == 0.f ? 0.f : 1.0f / ref.z) * e8_factors(ref.y, &more);      // NaN stays NaN
      bf16* orow = out + ((size_t)(qs + t0 + tl) * nq + kvh * g + (r - tl * g)) * D;
      if (warp_live) {
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          unsigned v[32];
          if (ok) {
            tmem_ld32(tmem_o + lane_sel + c0, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          }
          if (r < live_rows) {
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(v[c + e]) * inv * more;
              store8(orow + c0 + c, y);
            }
          }
        }
      }
    } else if (warp_live) {
      // this CTA's part of the row in float32 where queries, keys and values were (all of them have been read)
      float* mine = (float*)sQ + r * (D + 4);
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        unsigned v[32];
        if (ok) {
          tmem_ld32(tmem_o + lane_sel + c0, v);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 32; c += 4)
          *(float4*)(mine + c0 + c) = make_float4(__uint_as_float(v[c]), __uint_as_float(v[c + 1]), __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
      }
      float* ml = (float*)sQ + E8_BM * (D + 4);
      ml[r] = ref.x;
      ml[E8_BM + r] = ref.y;
      ml[2 * E8_BM + r] = ref.z;
    }
  } else if (warp < 8) {
    // ---- widening ----
    // Four lanes a row and panel of 64 dims, 16 numbers each: a warp's step is 8 rows of a panel, so that a lane's place in the
    // swizzle does not change, and its two 16-byte stores meet no other's banks.  Warp w has rows 8 w .. 8 w + 7 of either half.
    const int w = warp - 4, c = lane & 3, rl = lane >> 2;
    const int even = ((2 * c) ^ rl) << 4, place = (w * 8 + rl) * 128;      // r & 7 = rl
    // A lane's 16 bytes of its rows of a tile, on their way; [tile & 1][K, V][half][panel][lane] of this warp's.  Copies go out two
    // tiles ahead, keys and values as groups of their own.
    constexpr int PART = 2 * DP * 512;                     // bytes of a tile's K (or V) of this warp
    const unsigned char* const mine = sRaw + w * 4 * PART + lane * 16;
    const unsigned raw = tg_smem(mine);
    // the cache rows of this lane's two rows of a tile
    auto rows_of = [&](int it, int (&at)[2]) {
      if (it >= ntiles) return true;
      if (!__all_sync(0xffffffffu, mbar_wait(&t_full[it % E8_AHEAD], (it / E8_AHEAD) & 1, err))) return false;
      at[0] = tiles[it % E8_AHEAD].row[w * 8 + rl];
      at[1] = tiles[it % E8_AHEAD].row[32 + w * 8 + rl];
      return true;
    };
    auto copy = [&](int it, int which, const unsigned char* cache, const int (&at)[2]) {
      if (it < ntiles) {
        const unsigned dst = raw + ((it & 1) * 2 + which) * PART;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char* src = cache + (at[h] >= 0 ? (long long)at[h] * D + c * 16 : 0);
          const int n = at[h] >= 0 ? 16 : 0;
#pragma unroll
          for (int dp = 0; dp < DP; ++dp)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (h * DP + dp) * 512), "l"(src + dp * 64), "r"(n) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // this lane's numbers of half h of a tile times `power`, into their places
    auto widen = [&](unsigned char* tile, int it, int which, int h, unsigned factor) {
      const __half2 p2 = *(const __half2*)&factor;
#pragma unroll
      for (int dp = 0; dp < DP; ++dp) {
        const uint4 x = *(const uint4*)(mine + ((it & 1) * 2 + which) * PART + (h * DP + dp) * 512);
        uint4 y[2];
        __half2* z = (__half2*)y;
        const unsigned u[8] = {kv8_halves_lo(x.x), kv8_halves_hi(x.x), kv8_halves_lo(x.y), kv8_halves_hi(x.y),
                               kv8_halves_lo(x.z), kv8_halves_hi(x.z), kv8_halves_lo(x.w), kv8_halves_hi(x.w)};
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = __hmul2(*(const __half2*)&u[i], p2);
        unsigned char* dst = tile + dp * KPANEL + h * 4096 + place;
        *(uint4*)(dst + even) = y[0];
        *(uint4*)(dst + (even ^ 16)) = y[1];
      }
    };
    // Where there is one place for widened values, they wait for the product of the tile before, and the next tile's keys are
    // widened meanwhile: K0 K1 V0 K2 V1 K3 ... (64 sequences of 8,000 keys, heads of 128: 452 -> 359 us); else K0 V0 K1 V1 ...
    // (heads of 64: 276 us, in the other order 299).  Each makes room for its copy two tiles on.
    auto keys = [&](int it, const int (&next)[2]) {
      const int st = it % NS;
      if (!__all_sync(0xffffffffu, mbar_wait(&k_empty[st], (unsigned)((it / NS) & 1) ^ 1u, err))) return false;
      const E8Tile& x = tiles[it % E8_AHEAD];
#pragma unroll
      for (int h = 0; h < 2; ++h) widen(sK + st * STAGE, it, 0, h, x.kf[h * 32 + w * 8 + rl]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[st]);
      copy(it + 2, 0, kcache, next);
      return true;
    };
    auto values = [&](int it, const int (&next)[2]) {
      const int st = it % NS;
      if (!__all_sync(0xffffffffu, mbar_wait(&v_empty[st], (unsigned)((it / NS) & 1) ^ 1u, err))) return false;
      const E8Tile& x = tiles[it % E8_AHEAD];
#pragma unroll
      for (int h = 0; h < 2; ++h) widen(sV + st * STAGE, it, 1, h, x.vf[h * 32 + w * 8 + rl]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) { mbar_arrive(&v_full[st]); mbar_arrive(&t_free[it % E8_AHEAD]); }
      copy(it + 2, 1, vcache, next);
      return true;
    };
    int a0[2] = {-1, -1}, a1[2] = {-1, -1}, a2[2] = {-1, -1}, a3[2] = {-1, -1};
    ok = rows_of(0, a0) && rows_of(1, a1);
    copy(0, 0, kcache, a0);
    copy(0, 1, vcache, a0);
    copy(1, 0, kcache, a1);
    copy(1, 1, vcache, a1);
    if constexpr (NS == 2) {
      // (every tile commits a group of keys and one of values, two tiles ahead: three lie behind the one that is waited for)
      for (int it = 0; it < ntiles && ok; ++it) {
        ok = rows_of(it + 2, a2);
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        ok = ok && keys(it, a2);
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        ok = ok && values(it, a2);
      }
    } else {
      ok = ok && rows_of(2, a2);
      asm volatile("cp.async.wait_group 3;" ::: "memory");
      if (ntiles > 0) ok = ok && keys(0, a2);
      for (int it = 0; it < ntiles && ok; ++it) {
        // the keys of tile it + 1: behind their group lie the next keys' and one of values at most (no group is left out but
        // behind the last tile's, whose values' group all of these waits then cover)
        ok = rows_of(it + 3, a3);
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        if (it + 1 < ntiles) ok = ok && keys(it + 1, a3);
        asm volatile("cp.async.wait_group 3;" ::: "memory");
        ok = ok && values(it, a2);
        a2[0] = a3[0]; a2[1] = a3[1];
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == 9) {
    // ---- looking ahead: keys lane and lane + 32 of a tile ----
    // No condition stands around a load: a value that is chosen between a load's result and a constant is waited for where it is
    // chosen.  The block table's entries are asked for two tiles ahead, scales one.
    auto page_of = [&](int it, int h) {
      const int j = max((tile_lo + it) * E8_BN + h * 32 + lane, 0);
      return bt[min(page_shift >= 0 ? j >> page_shift : j / page_size, max_blocks - 1)];
    };
    int page[2] = {page_of(0, 0), page_of(0, 1)}, row[2], kb[2], vb[2];
    unsigned miss[2], readable[2];
    auto rows_of = [&](int it) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = (tile_lo + it) * E8_BN + h * 32 + lane;
        const bool wanted = j >= kmin && j < kend, bad = wanted && (page[h] < 0 || page[h] >= num_pages), read = wanted && !bad;
        miss[h] = __ballot_sync(0xffffffffu, bad);
        readable[h] = __ballot_sync(0xffffffffu, read);
        if (miss[h] && bad) atomicOr(err, 4);
        row[h] = read ? (page[h] * nkv + kvh) * page_size + (page_shift >= 0 ? j & (page_size - 1) : j % page_size) : -1;
        kb[h] = kscale[max(row[h], 0)];
        vb[h] = vscale[max(row[h], 0)];
        page[h] = page_of(it + 1, h);
      }
    };
    auto factor = [&](int b, int top) {                    // 2^(b - top + E8_LIFT) twice, as halves
      const __half2 p = __float2half2_rn(__uint_as_float((unsigned)(127 + E8_LIFT + max(b - top, -E8_APART)) << 23));
      return *(const unsigned*)&p;
    };
    rows_of(0);
    for (int it = 0; it < ntiles; ++it) {
      int r[2] = {row[0], row[1]}, k[2] = {kb[0], kb[1]}, v[2] = {vb[0], vb[1]};
      const unsigned ms[2] = {miss[0], miss[1]}, rd[2] = {readable[0], readable[1]};
      int kt = 0, vt = 0;
      bool live[2];                                        // neither hidden from all nor NaN
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool odd = k[h] == KV8_NAN_SCALE || v[h] == KV8_NAN_SCALE, read = rd[h] >> lane & 1u;
        live[h] = read && !odd;
        if (live[h]) { kt = max(kt, k[h]); vt = max(vt, v[h]); }
        else { k[h] = read ? KV8_NAN_SCALE : 0; v[h] = 0; }
      }
      kt = __reduce_max_sync(0xffffffffu, kt);
      vt = __reduce_max_sync(0xffffffffu, vt);
      const int kd[2] = {live[0] ? max(kt - k[0] - E8_APART, 0) : 0, live[1] ? max(kt - k[1] - E8_APART, 0) : 0};
      const int vd[2] = {live[0] ? max(vt - v[0] - E8_APART, 0) : 0, live[1] ? max(vt - v[1] - E8_APART, 0) : 0};
      const bool wide = __any_sync(0xffffffffu, (kd[0] | kd[1] | vd[0] | vd[1]) != 0);
      rows_of(it + 1);
      if (!__all_sync(0xffffffffu, mbar_wait(&t_free[it % E8_AHEAD], ((it / E8_AHEAD) & 1) ^ 1, err))) break;
      E8Tile& x = tiles[it % E8_AHEAD];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x.row[h * 32 + lane] = r[h];
        x.kf[h * 32 + lane] = k[h] == KV8_NAN_SCALE ? 0x7E007E00u : factor(k[h], kt);
        x.vf[h * 32 + lane] = factor(v[h], vt);
        if (wide) { x.kd[h * 32 + lane] = (unsigned char)kd[h]; x.vd[h * 32 + lane] = (unsigned char)vd[h]; }
      }
      if (lane == 0) { x.ek = kt; x.ev = vt; x.wide = wide; x.missing[0] = ms[0]; x.missing[1] = ms[1]; }
      __syncwarp();
      if (lane == 0) mbar_arrive(&t_full[it % E8_AHEAD]);
    }
  } else {
    // ---- products ---- (float32 accumulate, halves; the whole warp walks, one lane issues: see attention_tcgen05.cu)
    const unsigned idesc_s = (1u << 4) | ((unsigned)(E8_BN >> 3) << 17) | ((unsigned)(E8_BM >> 4) << 24);
    const unsigned idesc_pv = (1u << 4) | (1u << 16) | ((unsigned)(D >> 3) << 17) | ((unsigned)(E8_BM >> 4) << 24);
    const unsigned long long dq = umma_desc(sQ);
    const int n = __shfl_sync(0xffffffffu, ntiles, 0);
    auto wait = [&](unsigned long long* bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, err)) != 0; };
    // scores of tile it into its half of the score columns, where the weights of the tile two before were
    auto scores = [&](int it) {
      const int st = it % NS, half = it & 1;
      const unsigned long long dk = umma_desc(sK + st * STAGE);
      if (!wait(&k_full[st], (it / NS) & 1)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (umma_elect()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const unsigned long long a = dq + (unsigned long long)((k >> 2) * (QPANEL >> 4) + 2 * (k & 3));
          const unsigned long long b = dk + (unsigned long long)((k >> 2) * (KPANEL >> 4) + 2 * (k & 3));
          umma_bf16(tmem_s + half * E8_BN, a, b, idesc_s, k != 0);
        }
        umma_commit(&s_full[half]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      return true;
    };
    bool go = n > 0 && scores(0) && (n < 2 || scores(1));
    for (int it = 0; it < n && go; ++it) {
      const int st = it % NS;
      go = wait(&v_full[st], (it / NS) & 1) && wait(p_full, it & 1);
      if (!go) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned long long dv = (umma_desc(sV + st * STAGE) & ~(0x3FFFull << 16)) | ((unsigned long long)(KPANEL >> 4) << 16);
      if (umma_elect()) {
#pragma unroll
        for (int kk = 0; kk < E8_BN / 16; ++kk)
          umma_bf16_tmem_a(tmem_o, tmem_s + (it & 1) * E8_BN + kk * 8, dv + (unsigned long long)(kk * (2048 >> 4)), idesc_pv, (it != 0) || (kk != 0));
        umma_commit(pv_full);
        umma_commit(&v_empty[st]);
      }
      __syncwarp();
      if (it + 2 < n) go = wait(pv_full, it & 1) && scores(it + 2);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 8) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(256) : "memory");
  }
  if (splits == 1) { kv8_end(known); return; }
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  float* part = (float*)sQ;
  float* ml = part + E8_BM * (D + 4);
  const int first = live_rows * rank / splits, last = live_rows * (rank + 1) / splits;     // this CTA's rows
  for (int i = threadIdx.x; i < (last - first) * (D / 4); i += E8_THREADS) {
    const int row = first + i / (D / 4), c = (i % (D / 4)) * 4, tok = row / g;
    float top = E8_NONE, high = -INFINITY, sum = 0.f, more;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) {
      const float* other = cluster.map_shared_rank(ml, k);
      kv8_join(top, high, other[row], other[E8_BM + row]);
    }
    for (int k = 0; k < splits; ++k) {                       // (a CTA that has seen nothing has zeros or NaN)
      const float* other = cluster.map_shared_rank(ml, k);
      const float f = kv8_two_to(other[E8_BM + row] + (other[row] - top) - high);
      const float4 y = *(const float4*)(cluster.map_shared_rank(part, k) + row * (D + 4) + c);
      x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
      sum = fmaf(other[2 * E8_BM + row], kv8_two_to(other[row] - top), sum);
    }
    const float inv = (sum == 0.f ? 0.f : 1.0f / sum) * e8_factors(high, &more);
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * inv * more, x.y * inv * more), hi = __floats2bfloat162_rn(x.z * inv * more, x.w * inv * more);
    *(uint2*)(out + ((size_t)(qs + t0 + tok) * nq + kvh * g + row - tok * g) * D + c) = make_uint2(*(const unsigned*)&lo, *(const unsigned*)&hi);
  }
  cluster.sync();                                          // nobody leaves while its shared memory is being read
  kv8_end(known);
}

template <int D>
static int e8_launch(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const void* kscale,
                     const void* vscale, const int* block_table, int max_blocks, const int* q_start, const int* seq_lens,
                     int seq_begin, int num_seqs, int max_q_len, int max_keys, int nq, int nkv, int page_size, int num_pages,
                     int window, float scale, int known, int* err, cudaStream_t stream) {
  auto* kernel = attention_e4m3_tcgen05_kernel<D>;
  static SmemLimit limit;
  if (const int e = limit.allow(kernel, e8_smem_bytes<D>())) return e;
  const int bq = E8_BM / (nq / nkv);
  const long long tiles = ((long long)max_q_len + bq - 1) / bq, units = tiles * nkv * num_seqs;
  if (tiles * nkv > 65535 || num_seqs > 65535) return RLLM_E_UNSUPPORTED;
  // CTAs that share a tile of rows: to fill two places an SM, with two tiles of keys each at least
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= 296 && splits * 2 * 2 * E8_BN <= max_keys) splits *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)splits, (unsigned)(tiles * nkv), (unsigned)num_seqs);
  cfg.blockDim = dim3(E8_THREADS);
  cfg.dynamicSmemBytes = (size_t)e8_smem_bytes<D>();
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = rllm_pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (const bf16*)q, q_stride, (bf16*)out, (const unsigned char*)kcache,
                                           (const unsigned char*)vcache, (const unsigned char*)kscale, (const unsigned char*)vscale,
                                           block_table, max_blocks, q_start, seq_lens, seq_begin, nq, nkv, page_size, num_pages, window,
                                           scale * 1.4426950408889634f, known, err);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return 0;
}

// Sequences seq_begin .. seq_end - 1 of bfloat16 queries, of at most max_q_len tokens each; no query sees more than max_keys
// keys; known: see kv8_inputs.  Heads of 64 or 128, up to 128 of them a kv head, pages of any size.
RLLM_EXPORT int rllm_attention_e4m3_tcgen05(const void* q, int q_stride, void* out, const void* kcache, const void* vcache,
                                            const void* kscale, const void* vscale, const int* block_table, int max_blocks,
                                            const int* q_start, const int* seq_lens, int seq_begin, int seq_end, int max_q_len,
                                            int max_keys, int nq, int nkv, int d, int page_size, int num_pages, int window,
                                            float scale, int known, int* err, cudaStream_t stream) {
  if (max_q_len <= 0 || seq_end <= seq_begin) return 0;
  if (!q || !out || !kcache || !vcache || !kscale || !vscale || !block_table || !q_start || !seq_lens || !err || max_blocks <= 0 ||
      seq_begin < 0 || nq <= 0 || nkv <= 0 || nq % nkv || page_size <= 0 || num_pages <= 0 || window < 0 || !(scale > 0.f) || scale > 3e38f)
    return RLLM_E_BADARG;
  if (!(d == 64 || d == 128) || nq / nkv > E8_BM || q_stride % 8 ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kcache | (uintptr_t)vcache) & 15))
    return RLLM_E_UNSUPPORTED;
  if ((long long)num_pages * nkv * page_size > 0x7fffffffLL) return RLLM_E_UNSUPPORTED;      // cache rows are counted in 32 bits
#define E8_LAUNCH(DD) return e8_launch<DD>(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, seq_lens, \
      seq_begin, seq_end - seq_begin, max_q_len, max_keys, nq, nkv, page_size, num_pages, window, scale, known, err, stream)
  if (d == 64) E8_LAUNCH(64);
  E8_LAUNCH(128);
}
