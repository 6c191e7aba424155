// Paged causal attention over a cache that is kept in 8 bits (kv_e4m3.cuh) on tcgen05, keys and values widened inside the
// kernel: for sequences that bring up to a few tiles of 128 rows (a row is a (token, head of the kv head's group) pair), where
// widening them for all at once (attention_tcgen05.cu's DENSE form) would cost more traffic than the attention itself, and the
// mma.sync kernel (attention_e4m3.cu), which widens for 16 rows at a time, more instructions.  Contract as there.
//
// A CTA takes 128 rows of one (sequence, kv head) and a part of their keys, in tiles of 64; a cluster shares the keys.
//   warps 0-3   softmax, a thread a row (= TMEM lane): scores from TMEM, mask, running reference and sum in float32, weights as
//               halves back into TMEM; the output stays in TMEM and is rescaled when a reference moves.  Warps without a live
//               row only keep the barriers in step: a few rows cost the exponentials of 32.
//   warps 4-7   widen: 16 bytes of a row a lane, two tiles ahead of their use in registers, to halves in shared memory, in the
//               128-byte swizzle that the products read.
//   warp 8      allocates TMEM and issues the products: S = Q K^T (128 x 64 x D), O += P V (128 x D x 64, P in TMEM, V as the
//               MN-major operand, straight from its rows).
// Halves, not bfloat16: e4m3 numbers become halves in one instruction a pair, and a weight keeps 11 bits.  Powers of two:
//   K  a row's numbers are multiplied by 2^(ek - EK), EK the largest ek of the tile, and the tile's scores by 2^EK: exact down to
//      2^-24 of the tile's largest power;
//   V  by 2^(ev - EV'), EV' the tile's largest, but at least 2^-30 of a running reference that moves when passed by 2^4, and the
//      tile's weights by 2^(EV' - reference), which rides in the exponent's argument; 2^7 more, as in the mma.sync kernel;
//   Q  a row by a power of two of its own, exact for bfloat16 down to 2^-27 of the row's largest.
// A token whose key or value is NaN has a NaN key and zeros for a value: rows that see it become NaN by the score, and the others'
// products stay clean.
#include "attention_tcgen05.cuh"
#include "kv_e4m3.cuh"
#include <cooperative_groups.h>

#define E8_BM 128
#define E8_BN 64
#define E8_THREADS 288
#define E8_SLACK 4.0f
#define E8_SHIFT 7

// Q, two stages of K and of V, barriers and the stages' notes
template <int D> constexpr int e8_smem_bytes() { return E8_BM * D * 2 + 4 * E8_BN * D * 2 + 512; }

// what the widening warps tell the softmax warps of a tile
struct E8Note {
  int ek;                            // EK, a scale byte
  int shift;                         // EV' - reference
  int ref;                           // the reference, a scale byte
  int drop;                          // the one before - it (0: it has not moved, or there was none)
  unsigned missing[2];               // a bit a key whose page is not held
};

template <int D>
__global__ void __launch_bounds__(E8_THREADS, 2)
attention_e4m3_tcgen05_kernel(const bf16* q, int q_stride, bf16* __restrict__ out, const unsigned char* __restrict__ kcache,
                              const unsigned char* __restrict__ vcache, const unsigned char* __restrict__ kscale,
                              const unsigned char* __restrict__ vscale, const int* __restrict__ block_table, int max_blocks,
                              const int* __restrict__ q_start, const int* __restrict__ seq_lens, int seq_begin, int nq, int nkv,
                              int page_size, int num_pages, int window, float scale_log2, int* __restrict__ err) {
  constexpr int DP = D / 64, QPANEL = E8_BM * 128, KPANEL = E8_BN * 128, STAGE = E8_BN * D * 2;
  extern __shared__ __align__(1024) unsigned char e8_raw[];
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
  const int kend = min(first_pos + ntok, max_blocks * page_size);
  const int kmin = window > 0 ? max(0, first_pos - window + 1) : 0;
  const int all_lo = kmin / E8_BN, all = max(0, (kend + E8_BN - 1) / E8_BN - all_lo);
  const int tile_lo = all_lo + all * rank / splits, ntiles = all_lo + all * (rank + 1) / splits - tile_lo;
  unsigned char *sQ = e8_raw, *sK = sQ + DP * QPANEL, *sV = sK + 2 * STAGE;
  unsigned long long* bars = (unsigned long long*)(sV + 2 * STAGE);
  unsigned long long *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;      // [2] each
  unsigned long long *s_full = bars + 8, *p_full = bars + 10, *pv_full = bars + 11;                     // s_full: [2]
  unsigned* tmem_slot = (unsigned*)(bars + 12);
  E8Note* notes = (E8Note*)(bars + 13);                  // [4]: the softmax of a tile may be two behind its widening
  const int* bt = block_table + (size_t)s * max_blocks;
  const int page_shift = (page_size & (page_size - 1)) == 0 ? __ffs(page_size) - 1 : -1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], 1); }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(p_full, 4);
    mbar_init(pv_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tg_smem(tmem_slot)), "r"(256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // where the keys lane and lane + 32 of a tile lie: their cache rows, -1 for those outside [kmin, kend) or of pages not held
  auto page_of = [&](int it, int h) {
    const int j = (tile_lo + it) * E8_BN + h * 32 + lane;
    if (it >= ntiles || j < kmin || j >= kend) return -2;                 // not read
    return bt[page_shift >= 0 ? j >> page_shift : j / page_size];
  };
  int page_next[2] = {-2, -2};
  if (warp >= 4 && warp < 8) { page_next[0] = page_of(0, 0); page_next[1] = page_of(0, 1); }
  pdl_wait_on(q, kcache, vcache, kscale, vscale);

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
        if (c == 0) ((float*)sV)[r] = __uint_as_float((unsigned)(127 - 13 + e) << 23) * scale_log2;
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp < 4) my_factor = ((float*)sV)[threadIdx.x];
  __syncthreads();
  pdl_launch();                                            // behind the allocation: see pdl_launch
  const unsigned tmem_s = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_o = tmem_s + 2 * E8_BN;      // two tiles' scores: 128 + D <= 256 columns

  float m_ref = -INFINITY, l = 0.f;
  int ref = -1000;                                         // the reference of the values' powers, a scale byte
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
      const E8Note note = notes[it & 3];
      ref = note.ref;
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
      // the scores come from TMEM twice, 32 at a time, for their maximum and for their exponentials: all 64 at once, and the
      // weights, would not leave registers for two CTAs an SM
      float sc[32];
      auto load = [&](int h) {
        tmem_ld32(t_s + h * 32, (unsigned*)sc);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (masked) {
          const unsigned lo_rel = (unsigned)(row_lo - j0 - h * 32), span = (unsigned)max(row_hi - row_lo, 0), miss = note.missing[h];
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!((unsigned)j - lo_rel < span) || (miss >> j & 1u)) sc[j] = -INFINITY;
        }
      };
      float mx = -INFINITY;
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
      const bool moves = mx > m_ref + E8_SLACK;
      float corr = 1.0f;
      if (moves) {
        corr = at_ex2(m_ref - mx);                         // from -inf: 0, and nothing has been summed yet
        m_ref = mx;
        l *= corr;
      }
      const bool dropped = note.drop != 0;
      if (dropped) corr *= note.drop < -126 ? 0.f : __uint_as_float((unsigned)(127 + note.drop) << 23);
      // the product of the tile before has to be through: it wrote the output that is rescaled here
      if (it > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(pv_full, (it - 1) & 1, err));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (__any_sync(0xffffffffu, moves || dropped)) {
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
      // weights times 2^(EV' - reference + 7), in the place of the scores, and the sum without that factor
      const float up = (float)(note.shift + E8_SHIFT), m_safe = ((m_ref == -INFINITY) ? 0.f : m_ref) - up;
      const unsigned long long scale2 = at_pack2(f, f), shift2 = at_pack2(-m_safe, -m_safe);
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
        if (h == 0) tmem_st16(t_s, pk[0]);                 // (columns 0 .. 15: scores that have been read; the other half's lie behind)
      }
      tmem_st16(t_s + 16, pk[1]);
      {
        float a, b, c, d;
        at_unpack2(sum01, a, b);
        at_unpack2(sum23, c, d);
        l = fmaf((a + b) + (c + d), at_ex2(-up), l);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (ntiles == 0) ok = false;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(pv_full, (ntiles - 1) & 1, err));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // the result, without the values' powers' reference
    const float fe = ref < 0 ? 0.f : kv8_power(ref) * (1.0f / (1 << E8_SHIFT));
    if (splits == 1) {
      const float inv = (l == 0.f ? 0.f : 1.0f / l) * fe;  // NaN stays NaN
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
              for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(v[c + e]) * inv;
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
          *(float4*)(mine + c0 + c) = make_float4(__uint_as_float(v[c]) * fe, __uint_as_float(v[c + 1]) * fe, __uint_as_float(v[c + 2]) * fe,
                                                  __uint_as_float(v[c + 3]) * fe);
      }
      float* ml = (float*)sQ + E8_BM * (D + 4);
      ml[r] = m_ref;
      ml[E8_BM + r] = l;
    }
  } else if (warp < 8) {
    // ---- widening ----
    constexpr int L = D / 16, ROWS = 32 / L, STEPS = E8_BN / (4 * ROWS);       // lanes a row, a warp's rows a step, steps a tile
    const int w = warp - 4, c = lane % L, rl = lane / L;
    // Of the next tile: rows of the cache of keys lane and lane + 32, their scales, which of them are missing.  Its numbers are asked
    // for as soon as this tile's are widened, keys and values in turn.
    int row_n[2] = {-1, -1}, kb_n[2] = {0, 0}, vb_n[2] = {0, 0};
    unsigned miss_n[2] = {0u, 0u};
    uint4 kx[STEPS], vx[STEPS];
    auto rows_of = [&](int it) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = page_next[h], j = (tile_lo + it) * E8_BN + h * 32 + lane;
        const bool bad = page != -2 && (page < 0 || page >= num_pages);
        if (bad && w == 0) atomicOr(err, 4);
        miss_n[h] = __ballot_sync(0xffffffffu, bad);
        row_n[h] = (page == -2 || bad) ? -1 : (page * nkv + kvh) * page_size + (page_shift >= 0 ? j & (page_size - 1) : j % page_size);
        kb_n[h] = row_n[h] >= 0 ? kscale[row_n[h]] : 0;
        vb_n[h] = row_n[h] >= 0 ? vscale[row_n[h]] : 0;
        page_next[h] = page_of(it + 1, h);
      }
    };
    auto fetch = [&](uint4 (&x)[STEPS], const unsigned char* cache) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int r = (i * 4 + w) * ROWS + rl;
        const int at = __shfl_sync(0xffffffffu, i * 4 * ROWS >= 32 ? row_n[1] : row_n[0], r & 31);
        x[i] = at >= 0 ? *(const uint4*)(cache + (long long)at * D + c * 16) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    // 16 numbers times 2^(b - top) into their places of a tile
    auto widen = [&](unsigned char* tile, const uint4& raw, int r, float power) {
      const __half2 p2 = __float2half2_rn(power);
      const unsigned x[4] = {raw.x, raw.y, raw.z, raw.w};
      uint4 y[2];
      __half2* h = (__half2*)y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned lo = kv8_halves_lo(x[i]), hi = kv8_halves_hi(x[i]);
        h[2 * i] = __hmul2(*(const __half2*)&lo, p2);
        h[2 * i + 1] = __hmul2(*(const __half2*)&hi, p2);
      }
      // (the two stores of neighbouring panels' lanes in turn: their banks then do not meet)
      unsigned char* dst = tile + (c >> 2) * KPANEL + r * 128;
      const int even = (((c & 3) * 2) ^ (r & 7)) << 4, odd = even ^ 16, first = (c >> 2) & 1;
      *(uint4*)(dst + (first ? odd : even)) = first ? y[1] : y[0];
      *(uint4*)(dst + (first ? even : odd)) = first ? y[0] : y[1];
    };
    auto power_at = [&](int b, int top) { return b - top < -30 ? 0.f : __uint_as_float((unsigned)(127 + b - top) << 23); };
    if (ntiles > 0) {
      rows_of(0);
      fetch(kx, kcache);
      fetch(vx, vcache);
    }
    for (int it = 0; it < ntiles && ok; ++it) {
      const int st = it & 1;
      int kb[2] = {kb_n[0], kb_n[1]}, vb[2] = {vb_n[0], vb_n[1]};
      const unsigned miss[2] = {miss_n[0], miss_n[1]};
      if (it + 1 < ntiles) rows_of(it + 1);
      int kt = 0, vt = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool odd = kb[h] == KV8_NAN_SCALE || vb[h] == KV8_NAN_SCALE;
        if (odd) { kb[h] = KV8_NAN_SCALE; vb[h] = 0; }
        else { kt = max(kt, kb[h]); vt = max(vt, vb[h]); }
      }
      kt = __reduce_max_sync(0xffffffffu, kt);
      vt = __reduce_max_sync(0xffffffffu, vt);
      // the reference of the values' powers: the same walk in every widening warp
      int drop = 0;
      if (ref < 0) ref = vt;
      else if ((float)vt > (float)ref + E8_SLACK) { drop = ref - vt; ref = vt; }
      const int eff = max(vt, ref - 30);
      ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], ((it >> 1) & 1) ^ 1, err));
      if (!ok) break;
      if (w == 0 && lane == 0) {
        E8Note* n = &notes[it & 3];
        n->ek = kt; n->shift = eff - ref; n->ref = ref; n->drop = drop; n->missing[0] = miss[0]; n->missing[1] = miss[1];
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int r = (i * 4 + w) * ROWS + rl;
        const int b = __shfl_sync(0xffffffffu, i * 4 * ROWS >= 32 ? kb[1] : kb[0], r & 31);
        widen(sK + st * STAGE, kx[i], r, b == KV8_NAN_SCALE ? __uint_as_float(0x7FC00000u) : power_at(b, kt));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[st]);
      if (it + 1 < ntiles) fetch(kx, kcache);
      ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ((it >> 1) & 1) ^ 1, err));
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int r = (i * 4 + w) * ROWS + rl;
        const int b = __shfl_sync(0xffffffffu, i * 4 * ROWS >= 32 ? vb[1] : vb[0], r & 31);
        widen(sV + st * STAGE, vx[i], r, power_at(b, eff));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
      if (it + 1 < ntiles) fetch(vx, vcache);
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
      const int st = it & 1;
      const unsigned long long dk = umma_desc(sK + st * STAGE);
      if (!wait(&k_full[st], (it >> 1) & 1)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (umma_elect()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const unsigned long long a = dq + (unsigned long long)((k >> 2) * (QPANEL >> 4) + 2 * (k & 3));
          const unsigned long long b = dk + (unsigned long long)((k >> 2) * (KPANEL >> 4) + 2 * (k & 3));
          umma_bf16(tmem_s + st * E8_BN, a, b, idesc_s, k != 0);
        }
        umma_commit(&s_full[st]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      return true;
    };
    bool go = n > 0 && scores(0) && (n < 2 || scores(1));
    for (int it = 0; it < n && go; ++it) {
      const int st = it & 1;
      go = wait(&v_full[st], (it >> 1) & 1) && wait(p_full, it & 1);
      if (!go) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned long long dv = (umma_desc(sV + st * STAGE) & ~(0x3FFFull << 16)) | ((unsigned long long)(KPANEL >> 4) << 16);
      if (umma_elect()) {
#pragma unroll
        for (int kk = 0; kk < E8_BN / 16; ++kk)
          umma_bf16_tmem_a(tmem_o, tmem_s + st * E8_BN + kk * 8, dv + (unsigned long long)(kk * (2048 >> 4)), idesc_pv, (it != 0) || (kk != 0));
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
  if (splits == 1) return;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  float* part = (float*)sQ;
  float* ml = part + E8_BM * (D + 4);
  const int first = live_rows * rank / splits, last = live_rows * (rank + 1) / splits;     // this CTA's rows
  for (int i = threadIdx.x; i < (last - first) * (D / 4); i += E8_THREADS) {
    const int row = first + i / (D / 4), c = (i % (D / 4)) * 4, tok = row / g;
    float top = -INFINITY, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) top = fmaxf(top, cluster.map_shared_rank(ml, k)[row]);
    for (int k = 0; k < splits; ++k) {
      const float* other = cluster.map_shared_rank(ml, k);
      const float f = other[row] == -INFINITY ? 1.0f : at_ex2(other[row] - top);       // (with nothing seen, zeros or NaN)
      const float4 y = *(const float4*)(cluster.map_shared_rank(part, k) + row * (D + 4) + c);
      x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
      sum = fmaf(other[E8_BM + row], f, sum);
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * inv, x.y * inv), hi = __floats2bfloat162_rn(x.z * inv, x.w * inv);
    *(uint2*)(out + ((size_t)(qs + t0 + tok) * nq + kvh * g + row - tok * g) * D + c) = make_uint2(*(const unsigned*)&lo, *(const unsigned*)&hi);
  }
  cluster.sync();                                          // nobody leaves while its shared memory is being read
}

template <int D>
static int e8_launch(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const void* kscale,
                     const void* vscale, const int* block_table, int max_blocks, const int* q_start, const int* seq_lens,
                     int seq_begin, int num_seqs, int max_q_len, int max_keys, int nq, int nkv, int page_size, int num_pages,
                     int window, float scale, int* err, cudaStream_t stream) {
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
                                           scale * 1.4426950408889634f, err);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return 0;
}

// Sequences seq_begin .. seq_end - 1 of bfloat16 queries, of at most max_q_len tokens each; no query sees more than max_keys
// keys.  Heads of 64 or 128, up to 128 of them a kv head, pages of any size.
RLLM_EXPORT int rllm_attention_e4m3_tcgen05(const void* q, int q_stride, void* out, const void* kcache, const void* vcache,
                                            const void* kscale, const void* vscale, const int* block_table, int max_blocks,
                                            const int* q_start, const int* seq_lens, int seq_begin, int seq_end, int max_q_len,
                                            int max_keys, int nq, int nkv, int d, int page_size, int num_pages, int window,
                                            float scale, int* err, cudaStream_t stream) {
  if (max_q_len <= 0 || seq_end <= seq_begin) return 0;
  if (!q || !out || !kcache || !vcache || !kscale || !vscale || !block_table || !q_start || !seq_lens || !err || max_blocks <= 0 ||
      seq_begin < 0 || nq <= 0 || nkv <= 0 || nq % nkv || page_size <= 0 || num_pages <= 0 || window < 0 || !(scale > 0.f) || scale > 3e38f)
    return RLLM_E_BADARG;
  if (!(d == 64 || d == 128) || nq / nkv > E8_BM || q_stride % 8 ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kcache | (uintptr_t)vcache) & 15))
    return RLLM_E_UNSUPPORTED;
  if ((long long)num_pages * nkv * page_size > 0x7fffffffLL) return RLLM_E_UNSUPPORTED;      // cache rows are counted in 32 bits
#define E8_LAUNCH(DD) return e8_launch<DD>(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, seq_lens, \
      seq_begin, seq_end - seq_begin, max_q_len, max_keys, nq, nkv, page_size, num_pages, window, scale, err, stream)
  if (d == 64) E8_LAUNCH(64);
  E8_LAUNCH(128);
}
