// Paged causal attention over a cache that is kept in 8 bits (kv_e4m3.cuh), for sequences that bring any number of tokens:
// the query at position p of sequence s sees the keys max(0, p - window + 1) .. p of s (window 0: all keys 0 .. p), read from
// the pages through the block table, its own among them; kv head of query head h is h / (nq / nkv).
//
//   s_j = scale 2^ek_j (q . ck_j),   out = sum_j softmax(s)_j 2^ev_j cv_j
//
// A key whose scale is NaN makes the rows that see it NaN and no others: in a row's mask it is hidden by a selection, never
// by a product with 0, and the numbers of such a row are zeros (the writer's rule), so that they are harmless as an operand.
// A page that the sequence does not hold sets bit 4 of the error word, and its keys are left out.
//
//   rows kernel   tensor cores (mma.sync m16n8k16, f16 operands): one (sequence, kv head) and up to 8 NB rows (a row is a
//                 (token, head of the group) pair) a cluster of CTAs; see below.  Few rows over few keys, float32, heads of 256.
//   simt kernel   CUDA cores, one warp a (token, head): head sizes and pages that no other takes.
// Few rows over many keys: attention_e4m3_columns.cu; more rows: attention_e4m3_tcgen05.cu; prompts: the widening kernel of
// kv_e4m3.cu and attention_tcgen05.cu's DENSE form.
#include "kv_e4m3.cuh"
#include <cooperative_groups.h>
#include <math.h>

// The sequence of the launch's token i (flat token number): the s in [seq_begin, seq_end) with q_start[s] <= i < q_start[s + 1]
__device__ __forceinline__ int e4_sequence_of(const int* __restrict__ q_start, int seq_begin, int seq_end, int i) {
  int lo = seq_begin, hi = seq_end;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (q_start[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// CUDA cores
// ---------------------------------------------------------------------------
#define E4_SIMT_WARPS 4
template <typename T>
__global__ void __launch_bounds__(32 * E4_SIMT_WARPS)
attention_e4m3_simt_kernel(const T* q, int q_stride, T* __restrict__ out, const unsigned char* __restrict__ kcache,
                           const unsigned char* __restrict__ vcache, const unsigned char* __restrict__ kscale,
                           const unsigned char* __restrict__ vscale, const int* __restrict__ block_table, int max_blocks,
                           const int* __restrict__ q_start, const int* __restrict__ seq_lens, int seq_begin, int seq_end,
                           int num_tokens, int nq, int nkv, int d, int page_size, int num_pages, int window, float scale,
                           int* __restrict__ err) {
  extern __shared__ float qs[];      // [E4_SIMT_WARPS][d]
  pdl_wait_on(q, kcache, vcache, kscale, vscale, block_table, q_start, seq_lens);
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long gw = (long long)blockIdx.x * E4_SIMT_WARPS + warp;
  if (gw >= (long long)num_tokens * nq) return;
  const int h = (int)(gw % nq);
  const int t = q_start[seq_begin] + (int)(gw / nq);
  if (t >= q_start[seq_end]) return;
  const int s = e4_sequence_of(q_start, seq_begin, seq_end, t);
  const int kvh = h / (nq / nkv);
  const int len = seq_lens[s];
  const int pos = len - (q_start[s + 1] - t);
  const int kend = pos + 1, kstart = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
  float* myq = qs + warp * d;
  const T* qrow = q + (size_t)t * q_stride + (size_t)h * d;
  for (int i = lane; i < d; i += 32) myq[i] = to_f32(qrow[i]);
  __syncwarp();
  const int* bt = block_table + (size_t)s * max_blocks;
  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) acc[r] = 0.f;
  for (int j0 = kstart & ~31; j0 < kend; j0 += 32) {
    const int j = j0 + lane;
    long long row = -1;
    if (j >= kstart && j < kend && j / page_size < max_blocks) {
      const int page = bt[j / page_size];
      if (page < 0 || page >= num_pages) atomicOr(err, 4);
      else row = ((long long)page * nkv + kvh) * page_size + j % page_size;
    }
    float score = -INFINITY;
    if (row >= 0) {
      const uint4* kp = (const uint4*)(kcache + row * d);
      float dot = 0.f;
      for (int c = 0; c < d >> 4; ++c) {
        const uint4 raw = kp[c];
        float x[16];
        kv8_floats(raw.x, x); kv8_floats(raw.y, x + 4); kv8_floats(raw.z, x + 8); kv8_floats(raw.w, x + 12);
#pragma unroll
        for (int k = 0; k < 16; ++k) dot = fmaf(x[k], myq[c * 16 + k], dot);
      }
      score = dot * scale * kv8_power(kscale[row]);
    }
    const float top = warp_max(score);
    const bool nan = __any_sync(0xffffffffu, score != score);
    const float mnew = fmaxf(m, top);
    if (mnew == -INFINITY && !nan) continue;         // nothing seen yet
    const float mref = mnew == -INFINITY ? 0.f : mnew;
    const float corr = m == -INFINITY ? 0.f : expf(m - mref);
    const float p = row < 0 ? 0.f : expf(score - mref);
    const float power = row < 0 ? 0.f : kv8_power(vscale[row]);
    const float weight = row < 0 ? 0.f : p * power;
    m = mnew;
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int r = 0; r < 8; ++r) acc[r] *= corr;
    for (int k = 0; k < 32; ++k) {
      const long long vr = __shfl_sync(0xffffffffu, row, k);
      const float w = __shfl_sync(0xffffffffu, weight, k);
      if (vr < 0) continue;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (lane + 32 * r < d) {
          const unsigned two = kv8_halves((unsigned short)vcache[vr * d + lane + 32 * r]);
          acc[r] = fmaf(w, __low2float(*(const __half2*)&two), acc[r]);
        }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;       // NaN stays NaN
  T* orow = out + ((size_t)t * nq + h) * d;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (lane + 32 * r < d) orow[lane + 32 * r] = from_f32<T>(acc[r] * inv);
}

static int e4_check(const void* q, const void* out, const void* kcache, const void* vcache, const void* kscale,
                    const void* vscale, const int* block_table, int max_blocks, const int* q_start, const int* seq_lens,
                    int seq_begin, int seq_end, int nq, int nkv, int d, int page_size, int num_pages, int window, float scale,
                    const int* err) {
  if (!q || !out || !kcache || !vcache || !kscale || !vscale || !block_table || !q_start || !seq_lens || !err || max_blocks <= 0 ||
      seq_begin < 0 || seq_end < seq_begin || nq <= 0 || nkv <= 0 || nq % nkv || d <= 0 || page_size <= 0 || num_pages <= 0 ||
      window < 0 || !(scale == scale) || scale > 3e38f || scale < -3e38f)
    return RLLM_E_BADARG;
  if (d % 16 || d > 256 || (((uintptr_t)kcache | (uintptr_t)vcache) & 15)) return RLLM_E_UNSUPPORTED;
  return 0;
}

// ---------------------------------------------------------------------------
// tensor cores, few rows a sequence and kv head
// ---------------------------------------------------------------------------
// Keys are the rows of the first product and head dims those of the second, so that query rows are the columns (8 a tile):
//   S^T [16 keys x 8 rows] = K [16 x d] Q^T,   O^T [d x 8 rows] += V^T [d x 16 keys] P^T
// (queries as rows would come in sixteens: twice the products, accumulators and exponentials for a group of 8 or fewer).
// Operands of 8 bits become halves in registers, exactly, by one instruction a pair, and come from global memory straight
// into the lanes that need them: the order of head dims in the first product and in the second one's rows is free, so a lane
// takes contiguous bytes.
//   K: lane (gid, tig) needs keys gid and gid + 8, four dims a step of 16: bytes 64 c + 16 tig .. + 15 of the row, c = 0 ..
//      d / 64 - 1, are its dims of four steps; the queries are laid out by the same rule.
//   V: it needs keys 2 tig, 2 tig + 1 and those plus 8, and d / 8 dims: bytes gid d / 8 .. of four rows; the bytes of two
//      keys are interleaved (prmt) into pairs along the keys.
//   P^T: the accumulators of S^T hold (key gid, rows 2 tig, 2 tig + 1); movmatrix turns them into (keys 2 tig, 2 tig + 1, row gid).
// Factors: a key's power of two and its row's factor multiply the score s; a value's power rides in the weight, 2^(s + ev).  A row has
// two references, m of its scores and t, relative to m, of its weights with their values' powers: the denominator sums 2^(s - m) in
// float32, and the second product takes 2^((s - m) + (ev - t + 11)) as halves (in that order: s - m is exact where it matters, however
// large scores are), so that what a row keeps of its weights does not depend on how large the
// values are that it, or another row, does not look at (with one reference of the values' powers for all rows, a row that looked
// at values 2^20 below the others' kept 12 bits, and at 2^32 below zeros).  Both move only when passed by 2^4, so that a tile costs
// one vote, and the halves stay at or below 2^15; their smallest step, 2^-24, lies at 2^-35 of the row's largest weight.  References
// are whole numbers: what they are multiplied by when they move, or when parts meet, is exact.
// Queries are put into halves after a division by a power of two of the row's own (bfloat16: exact down to 2^-27 of the
// row's largest; float32: two halves, 22 bits, and P likewise).
// What bounds it: over few keys the start (queries, the first references, merge) and the latency of one or two tiles, 5.9 us for 511
// keys of 8 heads of 64; over many the instructions, about 300 for 16 keys of 128 dims (4 KB), a third of them conversions to
// halves at half the ALU's rate: 64 sequences of 8,191 keys, 8 heads of 128, 224 us, 4.8 TB/s.
//
// A cluster of C CTAs of 4 warps shares one (sequence, kv head, tile of rows): key tiles go round over the warps of the
// cluster, partial results are merged in shared memory, first the CTA's, then, each CTA a slice, the cluster's (distributed
// shared memory): no workspace, no counters, and a captured graph needs nothing of its own.
#define E4_WARPS 4
#define E4_SLACK 4                   // log2 of how far a score, and a weight with its value's power, may pass the row's reference
#define E4_SHIFT 11                  // log2 of the weights' factor: E4_SLACK + E4_SHIFT = 15
#define E4_NONE -3.0e38f             // the reference of a row that has seen nothing: 2^(s - reference) is 0 for a masked s, and any score moves it
__device__ __forceinline__ void e4_mma(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned e4_turn(unsigned x) {        // an 8 x 8 matrix of halves across the warp, transposed
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float e4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));           // ex2(-inf) = +0
  return y;
}
__device__ __forceinline__ unsigned e4_pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const unsigned*)&h;
}
__device__ __forceinline__ float2 e4_unpack(unsigned h) { return __half22float2(*(const __half2*)&h); }
__device__ __forceinline__ unsigned e4_word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// N bytes from global to shared memory on their way; e4_copy_or_zero: zeros where the source is not to be read
template <int N> __device__ __forceinline__ void e4_copy(unsigned dst, const void* src) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
template <int N> __device__ __forceinline__ void e4_copy_or_zero(unsigned dst, const void* src, bool valid) {
  const int n = valid ? N : 0;
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(N) : "memory");
}
__device__ __forceinline__ void e4_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void e4_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// a tile of 16 keys in shared memory: K's pieces, V's, 16 + 16 scale bytes; a pair is two of them
template <int D, int NB, typename T> constexpr int e4_ctas() {  // of an SM
  if (sizeof(T) == 2 && NB == 1) return D == 64 ? 5 : D == 128 ? 4 : 2;
  return D == 64 ? (NB <= 2 ? 3 : 2) : D == 128 ? (NB == 1 ? 3 : 2) : 2;
}
template <int D> __host__ __device__ constexpr int e4_tile_bytes() { return 32 * D + 32; }

template <int D, int NB, typename T>
__global__ void __launch_bounds__(32 * E4_WARPS, e4_ctas<D, NB, T>())
attention_e4m3_rows_kernel(const T* q, int q_stride, T* __restrict__ out, const unsigned char* __restrict__ kcache,
                           const unsigned char* __restrict__ vcache, const unsigned char* __restrict__ kscale,
                           const unsigned char* __restrict__ vscale, const int* __restrict__ block_table, int max_blocks,
                           const int* __restrict__ q_start, const int* __restrict__ seq_lens, int seq_begin, int nq, int nkv,
                           int page_size, int num_pages, int window, float scale_log2, int q_wide, int known, int* __restrict__ err) {
  constexpr int R = 8 * NB, TERMS = sizeof(T) == 4 ? 2 : 1, KC = D / 64, VW = D / 32, TB = e4_tile_bytes<D>();
  extern __shared__ __align__(16) float e4_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3;
  kv8_inputs(known, block_table, q_start, seq_lens);
  const int C = gridDim.x, rank = blockIdx.x;      // the cluster is the grid's x
  const int kvh = blockIdx.y % nkv, s = seq_begin + blockIdx.z;
  const int g = nq / nkv;
  const int qs = q_start[s], qlen = q_start[s + 1] - qs, len = seq_lens[s];
  const int rows = qlen * g, r0 = blockIdx.y / nkv * R;
  if (r0 >= rows) { pdl_wait(); return; }          // the whole cluster (a CTA that exits lets the next kernel in: it waits first)
  const int pos0 = len - qlen;
  const int t_first = r0 / g, t_last = (min(r0 + R, rows) - 1) / g;
  const int hi_first = pos0 + t_first + 1, kend = (int)min((long long)pos0 + t_last + 1, (long long)max_blocks * page_size);
  const int kmin = window > 0 ? max(0, hi_first - window) : 0;
  const int lo_last = window > 0 ? max(0, pos0 + t_last + 1 - window) : 0;
  const int* bt = block_table + (size_t)s * max_blocks;
  // A warp's pairs of tiles of 16 keys: tiles t0 + i stride and the next.  Lane l holds where tile (l & 1) of pair i lies, l / 2 =
  // i % 16 (its first cache row / 16; -1: not held or behind the end): 16 pairs are looked up at a time, for a lookup a tile
  // would stand, as a second trip to memory, between a tile and its loads.
  const int page_tiles = page_size >> 4, page_shift = (page_tiles & (page_tiles - 1)) == 0 ? __ffs(page_tiles) - 1 : -1;
  // A pair of tiles is a warp's by its place in the sequence, not in the tile of rows: see e4_rows_launch.
  const int t_lo = kmin >> 4, t_hi = (kend + 15) >> 4, stride = 2 * C * E4_WARPS;
  const int t0 = 2 * ((t_lo >> 1) + ((rank * E4_WARPS + warp - (t_lo >> 1)) & (C * E4_WARPS - 1)));
  const int pairs = t_hi > t0 ? (t_hi - t0 + stride - 1) / stride : 0;
  int places0 = -1, places1 = -1;      // of the even and the odd 16s: pairs on their way may lie 16 beyond the one at hand
  bool missing = false;                // a page of the warp's is not held (from where it is looked up on)
  auto look_up = [&](int i) {
    const int t = t0 + (i + (lane >> 1)) * stride + (lane & 1);
    int place = -1;
    bool bad = false;
    if (t >= t_lo && t < t_hi) {
      const int at = page_shift >= 0 ? t >> page_shift : t / page_tiles, page = bt[at];
      bad = page < 0 || page >= num_pages;
      if (!bad) place = (page * nkv + kvh) * page_tiles + (t - at * page_tiles);
    }
    if (__any_sync(0xffffffffu, bad)) {
      missing = true;
      if (bad) atomicOr(err, 4);
    }
    if (i & 16) places1 = place; else places0 = place;
  };
  auto place_of = [&](int i, int u) { return __shfl_sync(0xffffffffu, (i & 16) ? places1 : places0, (2 * i + u) & 31); };
  look_up(0);
  kv8_begin(known, q, kcache, vcache, kscale, vscale);
  kv8_let_in(known);
  // A warp's pair lies behind the queries: for each tile [pieces][32 lanes] of 16 bytes of K, then of V, and its scales.  A lane
  // reads back what it copied itself (the scales apart), each of its accesses 16 bytes beside its neighbour's.  There is one
  // place for K and one for V: the next pair's keys are asked for when this pair's scores are made, its values behind this
  // pair's products, so that each is on its way for about half a pair's time; twice the places left room for 12 warps an SM
  // instead of 16, which is what bounds the kernel (see below).
  constexpr int VP = D == 64 ? 8 : 16, VN = D / 8 / VP;           // bytes and number of a lane's pieces of a value row
  constexpr int RING = (int)sizeof(float) * R * (D + 4);
  const unsigned char* st = (const unsigned char*)e4_smem + RING + warp * 2 * TB;
  const unsigned ring = (unsigned)__cvta_generic_to_shared(st);
  auto whole_pair = [&](int j0) { return !missing && j0 >= kmin && j0 + 32 <= kend; };
  // rows outside [kmin, kend) or not held come in as zeros: whatever lies there stays out
  auto issue_k = [&](int i) {
    if (i < pairs) {
      if ((i & 15) == 0 && i > 0) look_up(i);
      const int j0 = (t0 + i * stride) << 4;
      const bool whole = whole_pair(j0);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int place = place_of(i, u);
        const long long row = (long long)place * 16;
        const unsigned char* kp = kcache + row * D + gid * D + tig * 16;
        const unsigned dst = ring + u * TB + lane * 16, sdst = ring + u * TB + 32 * D;
        if (whole) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < KC; ++c) e4_copy<16>(dst + (r * KC + c) * 512, kp + r * 8 * D + c * 64);
          if (lane == 0) e4_copy<16>(sdst, kscale + row);
        } else {
          const int lo = kmin - j0 - 16 * u, hi = place >= 0 ? kend - j0 - 16 * u : -1000;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const bool ok = gid + 8 * r >= lo && gid + 8 * r < hi;
#pragma unroll
            for (int c = 0; c < KC; ++c) e4_copy_or_zero<16>(dst + (r * KC + c) * 512, ok ? kp + r * 8 * D + c * 64 : kcache, ok);
          }
          if (lane == 0) e4_copy_or_zero<16>(sdst, place >= 0 ? kscale + row : kscale, place >= 0);
        }
      }
    }
    e4_copy_commit();
  };
  auto issue_v = [&](int i) {
    if (i < pairs) {
      const int j0 = (t0 + i * stride) << 4;
      const bool whole = whole_pair(j0);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int place = place_of(i, u);
        const long long row = (long long)place * 16;
        const unsigned char* vp = vcache + row * D + 2 * tig * D + gid * (D / 8);
        const unsigned dst = ring + u * TB + 16 * D + lane * VP, sdst = ring + u * TB + 32 * D + 16;
        if (whole) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < VN; ++c) e4_copy<VP>(dst + (r * VN + c) * 32 * VP, vp + ((r & 1) + 8 * (r >> 1)) * D + c * VP);
          if (lane == 0) e4_copy<16>(sdst, vscale + row);
        } else {
          const int lo = kmin - j0 - 16 * u, hi = place >= 0 ? kend - j0 - 16 * u : -1000;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = (r & 1) + 8 * (r >> 1);
            const bool ok = 2 * tig + at >= lo && 2 * tig + at < hi;
#pragma unroll
            for (int c = 0; c < VN; ++c) e4_copy_or_zero<VP>(dst + (r * VN + c) * 32 * VP, ok ? vp + at * D + c * VP : vcache, ok);
          }
          if (lane == 0) e4_copy_or_zero<16>(sdst, place >= 0 ? vscale + row : vscale, place >= 0);
        }
      }
    }
    e4_copy_commit();
  };
  issue_k(0);
  issue_v(0);

  // the tile's queries, as float32 rows of D + 4
  float* sQ = e4_smem;
  constexpr int QV = sizeof(T) == 4 ? 4 : 8;         // values of 16 bytes
  for (int i = threadIdx.x * QV; i < R * D; i += 32 * E4_WARPS * QV) {
    const int r = i / D, c = i - r * D, row = r0 + r;
    float x[QV];
#pragma unroll
    for (int e = 0; e < QV; ++e) x[e] = 0.f;
    if (row < rows) {
      const int tok = row / g;
      const T* src = q + (size_t)(qs + tok) * q_stride + (size_t)(kvh * g + row - tok * g) * D + c;
      if (q_wide) {
        if constexpr (sizeof(T) == 4) { const float4 y = *(const float4*)src; x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w; }
        else load8(src, x);
      } else {
#pragma unroll
        for (int e = 0; e < QV; ++e) x[e] = to_f32(src[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < QV; e += 4) *(float4*)(sQ + r * (D + 4) + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
  }
  __syncthreads();
  unsigned qf[NB][D / 16][2 * TERMS];
  float rfc[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float* qr = sQ + (nb * 8 + gid) * (D + 4) + tig * 16;
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 x = *(const float4*)(qr + c * 64 + i);
        top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);     // top < 2^(e + 1)
    const float down = __uint_as_float((unsigned)(127 + 13 - e) << 23), up = __uint_as_float((unsigned)(127 - 13 + e) << 23) * scale_log2;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const float4 x = *(const float4*)(qr + (kk >> 2) * 64 + (kk & 3) * 4);
      const float y[4] = {x.x * down, x.y * down, x.z * down, x.w * down};
      qf[nb][kk][0] = e4_pack(y[0], y[1]);
      qf[nb][kk][1] = e4_pack(y[2], y[3]);
      if (TERMS == 2) {
        const float2 a = e4_unpack(qf[nb][kk][0]), b = e4_unpack(qf[nb][kk][1]);
        qf[nb][kk][2 * TERMS - 2] = e4_pack(y[0] - a.x, y[1] - a.y);
        qf[nb][kk][2 * TERMS - 1] = e4_pack(y[2] - b.x, y[3] - b.y);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) rfc[nb][c] = __shfl_sync(0xffffffffu, up, (2 * tig + c) * 4);
  }

  float o[NB][D / 16][4], m[NB][2], t[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = t[nb][0] = t[nb][1] = E4_NONE;
    l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
  }

  for (int i = 0; i < pairs; ++i) {
    const int j0 = (t0 + i * stride) << 4;
    const bool whole = whole_pair(j0);
    const bool clear = whole && j0 >= lo_last && j0 + 32 <= hi_first;
    e4_copy_wait<1>();                 // the keys are here; the values may be on their way
    __syncwarp();
    int kb[4];                         // scale bytes of keys gid and gid + 8 of the two tiles
#pragma unroll
    for (int x = 0; x < 4; ++x) kb[x] = st[(x >> 1) * TB + 32 * D + gid + 8 * (x & 1)];
    // the products of the two tiles in turn (each waits for the one before it of its own sum), and two sums a tile where
    // registers allow
    constexpr int SUMS = NB == 1 && TERMS == 1 ? 2 : 1;
    float sc[2][NB][4], sd[2][NB][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[u][nb][e] = sd[u][nb][e] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint4 kx[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) kx[u][r] = *(const uint4*)(st + u * TB + (r * KC + c) * 512 + lane * 16);
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const unsigned wa = e4_word(kx[u][0], w), wc = e4_word(kx[u][1], w);
          const unsigned a[4] = {kv8_halves_lo(wa), kv8_halves_lo(wc), kv8_halves_hi(wa), kv8_halves_hi(wc)};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            e4_mma(SUMS == 2 && (w & 1) ? sd[u][nb] : sc[u][nb], a, qf[nb][c * 4 + w][0], qf[nb][c * 4 + w][1]);
            if (TERMS == 2) e4_mma(sc[u][nb], a, qf[nb][c * 4 + w][2 * TERMS - 2], qf[nb][c * 4 + w][2 * TERMS - 1]);
          }
        }
    }
    __syncwarp();                      // every lane has read the keys and their scales
    issue_k(i + 1);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      // 2^ek; 255 becomes infinity, which makes NaN of the row's zeros (and 0 a zero: such rows are below 2^-118)
      const float kf = __uint_as_float((unsigned)kb[x] << 23);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float& v = sc[x >> 1][nb][2 * (x & 1) + c];
          if (SUMS == 2) v += sd[x >> 1][nb][2 * (x & 1) + c];
          v = v * rfc[nb][c] * kf;
        }
    }
    unsigned seen = 0xffffffffu;       // bit nb * 8 + u * 4 + e (32 of them for NB = 4)
    if (!clear) {
      seen = 0u;
      const bool held[2] = {place_of(i, 0) >= 0, place_of(i, 1) >= 0};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int hi = pos0 + min(r0 + nb * 8 + 2 * tig + c, rows - 1) / g + 1, lo = window > 0 ? hi - window : 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = j0 + gid + 8 * x;
            if (held[x >> 1] && j < min(hi, kend) && j >= lo) seen |= 1u << (nb * 8 + 2 * x + c);
            else sc[x >> 1][nb][2 * (x & 1) + c] = -INFINITY;
          }
        }
    }
    e4_copy_wait<1>();                 // the values are here; the next keys may be on their way
    __syncwarp();
    float ev[4];                       // log2 of a value's power, NaN where the value is (a row that was not read has some byte)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int vb = st[(x >> 1) * TB + 32 * D + 16 + gid + 8 * (x & 1)];
      ev[x] = vb == KV8_NAN_SCALE ? __uint_as_float(0x7FC00000u) : (float)(vb - 127);
    }
    bool need = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = sc[e >> 2][nb][e & 3] - m[nb][e & 1];
        need = need || s > (float)E4_SLACK || s + ev[e >> 1] > t[nb][e & 1] + (float)E4_SLACK;
      }
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float corr[2], mx[2], tx[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) mx[c] = fmaxf(fmaxf(sc[0][nb][c], sc[0][nb][c + 2]), fmaxf(sc[1][nb][c], sc[1][nb][c + 2]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
          for (int c = 0; c < 2; ++c) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], x));
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[c] = mx[c] - m[nb][c] > (float)E4_SLACK ? ceilf(mx[c]) : m[nb][c];
          const float down = m[nb][c] - mx[c];
          l[nb][c] *= kv8_two_to(down);
          t[nb][c] += down;                                // (the same place: O stays as it is)
          m[nb][c] = mx[c];
          tx[c] = fmaxf(fmaxf((sc[0][nb][c] - mx[c]) + ev[0], (sc[0][nb][c + 2] - mx[c]) + ev[1]),
                        fmaxf((sc[1][nb][c] - mx[c]) + ev[2], (sc[1][nb][c + 2] - mx[c]) + ev[3]));
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
          for (int c = 0; c < 2; ++c) tx[c] = fmaxf(tx[c], __shfl_xor_sync(0xffffffffu, tx[c], x));
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tx[c] = tx[c] > t[nb][c] + (float)E4_SLACK ? ceilf(tx[c]) : t[nb][c];
          corr[c] = kv8_two_to(t[nb][c] - tx[c]);
          t[nb][c] = tx[c];
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) { o[nb][j][0] *= corr[0]; o[nb][j][1] *= corr[1]; o[nb][j][2] *= corr[0]; o[nb][j][3] *= corr[1]; }
      }
    }
    unsigned pb[2][NB][2 * TERMS];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float s = sc[u][nb][e] - m[nb][e & 1];
          l[nb][e & 1] += e4_ex2(s);
          w[e] = e4_ex2(s + (ev[2 * u + (e >> 1)] - (t[nb][e & 1] - (float)E4_SHIFT)));
        }
        if (!clear) {                  // (a masked score plus a NaN is one)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(seen >> (nb * 8 + u * 4 + e) & 1u)) w[e] = 0.f;
        }
        const unsigned h0 = e4_pack(w[0], w[1]), h1 = e4_pack(w[2], w[3]);
        pb[u][nb][0] = e4_turn(h0);
        pb[u][nb][1] = e4_turn(h1);
        if (TERMS == 2) {
          const float2 a = e4_unpack(h0), b = e4_unpack(h1);
          pb[u][nb][2 * TERMS - 2] = e4_turn(e4_pack(w[0] - a.x, w[1] - a.y));
          pb[u][nb][2 * TERMS - 1] = e4_turn(e4_pack(w[2] - b.x, w[3] - b.y));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unsigned xv[4][VW];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (D == 64) {
          const uint2 y = *(const uint2*)(st + u * TB + 16 * D + r * 256 + lane * 8);
          xv[r][0] = y.x; xv[r][1] = y.y;
        } else {
#pragma unroll
          for (int c = 0; c < VN; ++c) {
            const uint4 y = *(const uint4*)(st + u * TB + 16 * D + (r * VN + c) * 512 + lane * 16);
            xv[r][4 * c] = y.x; xv[r][4 * c + 1] = y.y; xv[r][4 * c + 2] = y.z; xv[r][4 * c + 3] = y.w;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < VW; ++c) {
        // bytes 4 c .. 4 c + 3 of keys 2 tig and 2 tig + 1, and of the two 8 keys on, as pairs along the keys
        const unsigned a01 = __byte_perm(xv[0][c], xv[1][c], 0x5140), a23 = __byte_perm(xv[0][c], xv[1][c], 0x7362);
        const unsigned b01 = __byte_perm(xv[2][c], xv[3][c], 0x5140), b23 = __byte_perm(xv[2][c], xv[3][c], 0x7362);
        const unsigned a[2][4] = {{kv8_halves_lo(a01), kv8_halves_hi(a01), kv8_halves_lo(b01), kv8_halves_hi(b01)},
                                  {kv8_halves_lo(a23), kv8_halves_hi(a23), kv8_halves_lo(b23), kv8_halves_hi(b23)}};
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            e4_mma(o[nb][2 * c + x], a[x], pb[u][nb][0], pb[u][nb][1]);
            if (TERMS == 2) e4_mma(o[nb][2 * c + x], a[x], pb[u][nb][2 * TERMS - 2], pb[u][nb][2 * TERMS - 1]);
          }
      }
    }
    __syncwarp();                      // every lane has read the values and their scales
    issue_v(i + 1);
  }
  e4_copy_wait<0>();

  // the CTA's result: parts [warps][R][D + 4], and every warp's reference and sum of each row
  constexpr int LD = D + 4;
  float* part = e4_smem;
  float* sM = part + E4_WARPS * R * LD;              // [warps][R]
  float* sT = sM + E4_WARPS * R;
  float* sL = sT + E4_WARPS * R;
  float* cM = sL + E4_WARPS * R;                     // [R] the CTA's
  float* cT = cM + R;
  float* cL = cT + R;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], x);
  __syncthreads();                                   // the queries and all tiles have been read
  if (gid == 0) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        sM[warp * R + nb * 8 + 2 * tig + c] = m[nb][c];
        sT[warp * R + nb * 8 + 2 * tig + c] = t[nb][c];
        sL[warp * R + nb * 8 + 2 * tig + c] = l[nb][c];
      }
  }
  __syncthreads();
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nb * 8 + 2 * tig + c;
      float top = sM[r], high = sT[r];
#pragma unroll
      for (int w = 1; w < E4_WARPS; ++w) kv8_join(top, high, sM[w * R + r], sT[w * R + r]);
      const float f = kv8_two_to(t[nb][c] + (m[nb][c] - top) - high);
      float* dst = part + (warp * R + r) * LD + gid * (D / 8);
#pragma unroll
      for (int j = 0; j < D / 16; j += 2)
        *(float4*)(dst + 2 * j) = make_float4(o[nb][j][c] * f, o[nb][j][c + 2] * f, o[nb][j + 1][c] * f, o[nb][j + 1][c + 2] * f);
    }
  if (threadIdx.x < R) {
    const int r = threadIdx.x;
    float top = sM[r], high = sT[r], sum = 0.f;
#pragma unroll
    for (int w = 1; w < E4_WARPS; ++w) kv8_join(top, high, sM[w * R + r], sT[w * R + r]);
#pragma unroll
    for (int w = 0; w < E4_WARPS; ++w) sum += sL[w * R + r] * kv8_two_to(sM[w * R + r] - top);
    cM[r] = top;
    cT[r] = high;
    cL[r] = sum;
  }
  __syncthreads();
  // high: the weights' reference relative to the sum's.  2^high as two factors, for it may lie below the normal numbers
  auto store = [&](int r, int c, float4 x, float high, float sum) {
    const int row = r0 + r;
    if (row < rows) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;   // NaN stays NaN
      const float by = fminf(fmaxf(high, -200.f), 200.f), half = floorf(by * 0.5f);
      const float up = __uint_as_float((unsigned)(127 + (int)half - E4_SHIFT) << 23), more = __uint_as_float((unsigned)(127 + (int)(by - half)) << 23);
      x.x *= up; x.y *= up; x.z *= up; x.w *= up;
      const int tok = row / g;
      T* dst = out + ((size_t)(qs + tok) * nq + kvh * g + row - tok * g) * D + c;
      if constexpr (sizeof(T) == 4) {
        *(float4*)dst = make_float4(x.x * inv * more, x.y * inv * more, x.z * inv * more, x.w * inv * more);
      } else {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x * inv * more, x.y * inv * more), hi = __floats2bfloat162_rn(x.z * inv * more, x.w * inv * more);
        *(uint2*)dst = make_uint2(*(const unsigned*)&lo, *(const unsigned*)&hi);
      }
    }
  };
  for (int i = threadIdx.x * 4; i < R * D; i += 32 * E4_WARPS * 4) {
    const int r = i / D, c = i - r * D;
    float4 x = *(const float4*)(part + r * LD + c);
#pragma unroll
    for (int w = 1; w < E4_WARPS; ++w) {
      const float4 y = *(const float4*)(part + (w * R + r) * LD + c);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    if (C == 1) store(r, c, x, cT[r], cL[r]);
    else *(float4*)(part + r * LD + c) = x;
  }
  if (C == 1) { kv8_end(known); return; }
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = (rank * 32 * E4_WARPS + threadIdx.x) * 4; i < R * D; i += C * 32 * E4_WARPS * 4) {
    const int r = i / D, at = r * LD + i - r * D;
    float top = E4_NONE, high = -INFINITY, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < C; ++c) {
      const float* m_ = cluster.map_shared_rank(cM, c);              // the weights' references lie R behind, the sums 2 R
      kv8_join(top, high, m_[r], m_[R + r]);
    }
    for (int c = 0; c < C; ++c) {
      const float* m_ = cluster.map_shared_rank(cM, c);
      const float f = kv8_two_to(m_[R + r] + (m_[r] - top) - high);
      const float4 y = *(const float4*)(cluster.map_shared_rank(part, c) + at);
      x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
      sum = fmaf(m_[2 * R + r], kv8_two_to(m_[r] - top), sum);
    }
    store(r, i - r * D, x, high, sum);
  }
  cluster.sync();                                    // nobody leaves while its shared memory is being read
  kv8_end(known);
}

template <int D, int NB, typename T>
static int e4_rows_launch(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const void* kscale,
                          const void* vscale, const int* block_table, int max_blocks, const int* q_start, const int* seq_lens,
                          int seq_begin, int num_seqs, int max_q_len, int max_keys, int nq, int nkv, int page_size,
                          int num_pages, int window, float scale, int known, int* err, cudaStream_t stream) {
  constexpr int R = 8 * NB;
  auto* kernel = attention_e4m3_rows_kernel<D, NB, T>;
  const size_t stage = sizeof(float) * R * (D + 4), merge = sizeof(float) * (E4_WARPS * R * (D + 7) + 3 * R);
  const size_t rings = stage + E4_WARPS * 2 * e4_tile_bytes<D>(), smem = rings > merge ? rings : merge;
  static SmemLimit limit;
  if (const int e = limit.allow(kernel, (int)smem)) return e;
  const long long tiles = ((long long)max_q_len * (nq / nkv) + R - 1) / R, units = tiles * nkv * num_seqs;
  if (tiles * nkv > 65535 || num_seqs > 65535) return RLLM_E_UNSUPPORTED;
  // CTAs a unit: to fill the GPU's places, of 128 keys at least (a CTA costs 2 us beside its keys); where there are enough of
  // them and keys are many, several rounds of CTAs, so that the last round is short beside the rest (64 sequences of 4,000 to
  // 12,000 keys, 32/8 heads of 128: 270 us with one CTA, 252 with two, 238 with four, 242 with eight)
  // float32: the same number whatever the call.  A row's keys then go to the same warps, and their results are added up in the same
  // order, whoever else is in the step and however the prompt was cut: its result does not depend on them (nothing else of another
  // row's enters: references are the row's own, and what they are multiplied by when they move is exact)
  int C = sizeof(T) == 4 ? 4 : 1;
  while (sizeof(T) == 2 && C < 8 && ((units * C * 2 <= 592 && C * 2 * 128 <= max_keys) || (units * C * 2 <= 2368 && C * 2 * 1024 <= max_keys))) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)C, (unsigned)(tiles * nkv), (unsigned)num_seqs);
  cfg.blockDim = dim3(32 * E4_WARPS);
  cfg.dynamicSmemBytes = smem;
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (const T*)q, q_stride, (T*)out, (const unsigned char*)kcache,
                                           (const unsigned char*)vcache, (const unsigned char*)kscale, (const unsigned char*)vscale,
                                           block_table, max_blocks, q_start, seq_lens, seq_begin, nq, nkv, page_size, num_pages,
                                           window, scale * 1.4426950408889634f,
                                           (((uintptr_t)q | ((uintptr_t)q_stride * sizeof(T))) & 15) == 0 ? 1 : 0, known, err);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  RLLM_LAUNCH_CHECK();
  return 0;
}

// Sequences seq_begin .. seq_end - 1, of at most max_q_len tokens each; no query sees more than max_keys keys; known: see kv8_inputs.  Heads of 64,
// 128 or 256, pages of a multiple of 16 keys.
RLLM_EXPORT int rllm_attention_e4m3_rows(const void* q, int q_stride, void* out, const void* kcache, const void* vcache,
                                         const void* kscale, const void* vscale, int dtype, const int* block_table,
                                         int max_blocks, const int* q_start, const int* seq_lens, int seq_begin, int seq_end,
                                         int max_q_len, int max_keys, int nq, int nkv, int d, int page_size, int num_pages,
                                         int window, float scale, int known, int* err, cudaStream_t stream) {
  if (max_q_len <= 0 || seq_end <= seq_begin) return 0;
  if (const int rc = e4_check(q, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, seq_lens, seq_begin,
                              seq_end, nq, nkv, d, page_size, num_pages, window, scale, err)) return rc;
  if (page_size % 16 || !(d == 64 || d == 128 || d == 256) || (((uintptr_t)kscale | (uintptr_t)vscale | (uintptr_t)out) & 15)) return RLLM_E_UNSUPPORTED;
  if ((long long)num_pages * nkv * (page_size >> 4) > 0x7fffffffLL) return RLLM_E_UNSUPPORTED;      // tiles of 16 rows are counted in 32 bits
#define E4_ROWS(DD, NBB, TT)                                                                                                   \
  return e4_rows_launch<DD, NBB, TT>(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, \
                                          seq_lens, seq_begin, seq_end - seq_begin, max_q_len, max_keys, nq, nkv, page_size,  \
                                          num_pages, window, scale, known, err, stream)
  // tiles of as many rows as the sequences bring, where registers hold them: every tile reads all keys again
  const long long rows = (long long)max_q_len * (nq / nkv);
  if (dtype == RLLM_DT_BF16) {
    if (d == 64) { if (rows <= 8) E4_ROWS(64, 1, bf16); if (rows <= 16) E4_ROWS(64, 2, bf16); if (rows <= 24) E4_ROWS(64, 3, bf16); E4_ROWS(64, 4, bf16); }
    if (d == 128) { if (rows <= 8) E4_ROWS(128, 1, bf16); if (rows <= 16) E4_ROWS(128, 2, bf16); E4_ROWS(128, 3, bf16); }
    E4_ROWS(256, 1, bf16);
  }
  if (dtype == RLLM_DT_F32) {
    if (d == 64) { if (rows <= 8) E4_ROWS(64, 1, float); E4_ROWS(64, 2, float); }
    if (d == 128) { if (rows <= 8) E4_ROWS(128, 1, float); E4_ROWS(128, 2, float); }
    E4_ROWS(256, 1, float);
  }
  return RLLM_E_BADARG;
}

RLLM_EXPORT int rllm_attention_e4m3_simt(const void* q, int q_stride, void* out, const void* kcache, const void* vcache,
                                         const void* kscale, const void* vscale, int dtype, const int* block_table,
                                         int max_blocks, const int* q_start, const int* seq_lens, int seq_begin, int seq_end,
                                         int num_tokens, int nq, int nkv, int d, int page_size, int num_pages, int window,
                                         float scale, int* err, cudaStream_t stream) {
  if (num_tokens <= 0 || seq_end <= seq_begin) return 0;
  if (const int rc = e4_check(q, out, kcache, vcache, kscale, vscale, block_table, max_blocks, q_start, seq_lens, seq_begin,
                              seq_end, nq, nkv, d, page_size, num_pages, window, scale, err)) return rc;
  const long long warps = (long long)num_tokens * nq, blocks = (warps + E4_SIMT_WARPS - 1) / E4_SIMT_WARPS;
  if (blocks > 0x7fffffffLL) return RLLM_E_UNSUPPORTED;
  RLLM_DISPATCH_DTYPE(dtype, T,
    rllm_launch_pdl(attention_e4m3_simt_kernel<T>, dim3((unsigned)blocks), dim3(32 * E4_SIMT_WARPS), sizeof(float) * E4_SIMT_WARPS * d,
                    stream, (const T*)q, q_stride, (T*)out, (const unsigned char*)kcache, (const unsigned char*)vcache,
                    (const unsigned char*)kscale, (const unsigned char*)vscale, block_table, max_blocks, q_start, seq_lens,
                    seq_begin, seq_end, num_tokens, nq, nkv, d, page_size, num_pages, window, scale, err));
  RLLM_LAUNCH_CHECK();
  return 0;
}
