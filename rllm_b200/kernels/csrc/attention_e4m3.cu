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
//                 (token, head of the group) pair) a cluster of CTAs; see below.
//   simt kernel   CUDA cores, one warp a (token, head): head sizes and pages that the rows kernel does not take.
#include "kv_e4m3.cuh"
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
  pdl_wait_on(q, kcache, vcache, kscale, vscale);
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
