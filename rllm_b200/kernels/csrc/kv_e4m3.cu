// Writing a cache that is kept in 8 bits, and reading it back (see kv_e4m3.cuh for what a row becomes).
#include "kv_e4m3.cuh"
#include "attention_dense.h"

// ---------------------------------------------------------------------------
// write: rotation of q, rotation and quantisation of k, quantisation of v
// ---------------------------------------------------------------------------
// One block a token, one warp a row (a query, key or value head of the token); a lane holds the dims lane, lane + 32, ...
// in registers, so a row is read once.  The angles are made once for all heads.  Any head size up to 256 and any rotary_dim.
template <typename T>
__global__ void __launch_bounds__(256)
kv_e4m3_write_kernel(const T* qkv, T* q_out, long long q_stride, const int* __restrict__ positions,
                     const int* __restrict__ token_seq, const double* __restrict__ inv_freq, int rotary_dim,
                     const int* __restrict__ block_table, int max_blocks, int num_seqs, unsigned char* __restrict__ kcache,
                     unsigned char* __restrict__ vcache, unsigned char* __restrict__ kscale,
                     unsigned char* __restrict__ vscale, int nq, int nkv, int d, int page_size, int num_pages,
                     int* __restrict__ err) {
  extern __shared__ float cs[];  // cos[rd/2], sin[rd/2]
  pdl_wait_on(qkv, positions, token_seq, block_table, q_out);
  pdl_launch();
  const int t = blockIdx.x;
  const int pos = positions[t];
  const int half = rotary_dim >> 1;
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    if (sizeof(T) == 4) {            // the true 32-bit path: float64 cosine and sine, rounded once
      double s, c;
      sincos((double)pos * inv_freq[i], &s, &c);
      cs[i] = (float)c;
      cs[half + i] = (float)s;
    } else {
      rope_cos_sin(pos, inv_freq[i], &cs[i], &cs[half + i]);
    }
  }
  __syncthreads();
  const int seq = token_seq[t];
  long long slot = -1;               // row of kv head 0; a head further: page_size rows on
  if (pos >= 0 && pos / page_size < max_blocks && seq >= 0 && seq < num_seqs) {
    const int page = block_table[(size_t)seq * max_blocks + pos / page_size];
    if (page >= 0 && page < num_pages) slot = (long long)page * nkv * page_size + pos % page_size;
  }
  if (slot < 0 && threadIdx.x == 0) atomicOr(err, 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* row = qkv + (size_t)t * (nq + 2 * nkv) * d;
  const int heads = slot < 0 ? nq : nq + 2 * nkv;
  for (int h = warp; h < heads; h += blockDim.x >> 5) {
    const T* src = row + (size_t)h * d;
    const bool turned = h < nq + nkv;
    float x[8];
    float top = 0.f;
    bool odd = false;                // an infinity or a NaN
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = lane + 32 * k;
      if (i < d) {
        float v = to_f32(src[i]);
        if (turned && i < rotary_dim) {
          if (i < half) v = v * cs[i] - to_f32(src[i + half]) * cs[half + i];
          else          v = v * cs[i - half] + to_f32(src[i - half]) * cs[i];
        }
        x[k] = v;
        top = fmaxf(top, fabsf(v));
        odd = odd || !(fabsf(v) <= 3.402823466e38f);
      }
    }
    if (h < nq) {
      __syncwarp();                  // q_out may be the row itself: all of it has been read
      T* dst = q_out + (size_t)t * q_stride + (size_t)h * d;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (lane + 32 * k < d) dst[lane + 32 * k] = from_f32<T>(x[k]);
      continue;
    }
    top = warp_max(top);
    odd = __any_sync(0xffffffffu, odd);
    const int byte = odd ? KV8_NAN_SCALE : kv8_scale_byte(top);
    const float inv = odd ? 0.f : kv8_inverse(byte);
    const long long r = slot + (long long)(turned ? h - nq : h - nq - nkv) * page_size;
    unsigned char* dst = (turned ? kcache : vcache) + r * d;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < d) dst[lane + 32 * k] = odd ? (unsigned char)0 : (unsigned char)(kv8_pack2(x[k] * inv, 0.f) & 0xffu);
    if (lane == 0) (turned ? kscale : vscale)[r] = (unsigned char)byte;
  }
}

// bfloat16 heads of 32, 64, 128 or 256, rotated whole or not at all, rows on 16 bytes: D / 16 lanes a row, each with 8 dims of its
// first half and the 8 that pair with them, two 16-byte loads.  A thread's loads of KV8_ROWS rows are on their way while the block
// makes the token's angles.  Bound by memory: 6,327 tokens of 32/8 heads of 128, 143 MB, 28 us (5.1 TB/s; a warp a row: 126 us;
// two rows a thread 31, four 33 to 36, by the registers that they leave to blocks in flight).
#define KV8_ROWS 3
template <int D>
__global__ void __launch_bounds__(128, 8)
kv_e4m3_write_bf16_kernel(const bf16* qkv, bf16* q_out, long long q_stride, const int* __restrict__ positions,
                          const int* __restrict__ token_seq, const double* __restrict__ inv_freq, int rotary_dim,
                          const int* __restrict__ block_table, int max_blocks, int num_seqs, unsigned char* __restrict__ kcache,
                          unsigned char* __restrict__ vcache, unsigned char* __restrict__ kscale,
                          unsigned char* __restrict__ vscale, int nq, int nkv, int page_size, int num_pages,
                          int* __restrict__ err) {
  constexpr int L = D / 16, H = D / 2;
  __shared__ __align__(16) float cs[D];                // cosines, sines
  pdl_wait_on(qkv, positions, token_seq, block_table, q_out);
  pdl_launch();
  const int t = blockIdx.x, heads = nq + 2 * nkv, c = (threadIdx.x % L) * 8;
  const bf16* row = qkv + (size_t)t * heads * D + c;
  uint4 lo[KV8_ROWS], hi[KV8_ROWS];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < KV8_ROWS; ++k) {
      const int h = base + (threadIdx.x + k * 128) / L;
      if (h < heads) {
        lo[k] = *(const uint4*)(row + (size_t)h * D);
        hi[k] = *(const uint4*)(row + (size_t)h * D + H);
      }
    }
  };
  load(0);
  const int pos = positions[t], seq = token_seq[t];
  long long slot = -1;                                 // row of kv head 0; a head further: page_size rows on
  if (pos >= 0 && pos / page_size < max_blocks && seq >= 0 && seq < num_seqs) {
    const int page = block_table[(size_t)seq * max_blocks + pos / page_size];
    if (page >= 0 && page < num_pages) slot = (long long)page * nkv * page_size + pos % page_size;
  }
  if (slot < 0 && threadIdx.x == 0) atomicOr(err, 2);
  if (rotary_dim) {
    for (int i = threadIdx.x; i < H; i += 128) rope_cos_sin(pos, inv_freq[i], &cs[i], &cs[H + i]);
    __syncthreads();
  }
  float cx[8], sx[8];
  if (rotary_dim) { load8(cs + c, cx); load8(cs + H + c, sx); }
  for (int base = 0; base < heads; base += KV8_ROWS * 128 / L) {
    if (base) load(base);
#pragma unroll
    for (int k = 0; k < KV8_ROWS; ++k) {
      const int h = base + (threadIdx.x + k * 128) / L;
      const bool live = h < heads;
      float a[8], b[8];
      unpack8(lo[k], a);
      unpack8(hi[k], b);
      if (rotary_dim && h < nq + nkv) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = a[e], y = b[e];
          a[e] = x * cx[e] - y * sx[e];
          b[e] = y * cx[e] + x * sx[e];
        }
      }
      if (live && h < nq) {
        bf16* dst = q_out + (size_t)t * q_stride + (size_t)h * D + c;
        store8(dst, a);
        store8(dst + H, b);
      }
      // the row's largest magnitude; NaN and infinities by their bits, which are the largest of all
      unsigned top = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
#pragma unroll
      for (int x = L / 2; x > 0; x >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
      if (!live || h < nq || slot < 0) continue;
      const bool odd = top >= 0x7f800000u;
      const int byte = odd ? KV8_NAN_SCALE : kv8_scale_byte(__uint_as_float(top));
      const float inv = odd ? 0.f : kv8_inverse(byte);
      const bool value = h >= nq + nkv;
      const long long r = slot + (long long)(value ? h - nq - nkv : h - nq) * page_size;
      unsigned char* dst = (value ? vcache : kcache) + r * D + c;
      uint2 ca = make_uint2(kv8_pack4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv), kv8_pack4(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv));
      uint2 cb = make_uint2(kv8_pack4(b[0] * inv, b[1] * inv, b[2] * inv, b[3] * inv), kv8_pack4(b[4] * inv, b[5] * inv, b[6] * inv, b[7] * inv));
      if (odd) ca = cb = make_uint2(0u, 0u);
      *(uint2*)dst = ca;
      *(uint2*)(dst + H) = cb;
      if (c == 0) (value ? vscale : kscale)[r] = (unsigned char)byte;
    }
  }
}

RLLM_EXPORT int rllm_kv_e4m3_write(const void* qkv, int dtype, void* q_out, long long q_stride, const int* positions,
                                   const int* token_seq, const double* inv_freq, int rotary_dim, const int* block_table,
                                   int max_blocks, int num_seqs, void* kcache, void* vcache, void* kscale, void* vscale,
                                   int T, int nq, int nkv, int d, int page_size, int num_pages, int* err,
                                   cudaStream_t stream) {
  if (T <= 0) return 0;
  if (!qkv || !q_out || !positions || !token_seq || !block_table || !kcache || !vcache || !kscale || !vscale || !err ||
      nq <= 0 || nkv <= 0 || d <= 0 || rotary_dim < 0 || rotary_dim > d || (rotary_dim & 1) || (rotary_dim && !inv_freq) ||
      page_size <= 0 || num_pages <= 0 || max_blocks <= 0 || num_seqs <= 0 || q_stride < (long long)nq * d)
    return RLLM_E_BADARG;
  if (d % 16 || d > 256) return RLLM_E_UNSUPPORTED;
  if (dtype == RLLM_DT_BF16 && (d == 32 || d == 64 || d == 128 || d == 256) && (rotary_dim == d || rotary_dim == 0) &&
      (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)q_stride * 2) & 15) == 0 && (((uintptr_t)kcache | (uintptr_t)vcache) & 7) == 0) {
#define KV8_WRITE(DD) rllm_launch_pdl(kv_e4m3_write_bf16_kernel<DD>, dim3(T), dim3(128), (size_t)0, stream, (const bf16*)qkv, (bf16*)q_out, \
      q_stride, positions, token_seq, inv_freq, rotary_dim, block_table, max_blocks, num_seqs, (unsigned char*)kcache,                   \
      (unsigned char*)vcache, (unsigned char*)kscale, (unsigned char*)vscale, nq, nkv, page_size, num_pages, err)
    if (d == 32) KV8_WRITE(32);
    else if (d == 64) KV8_WRITE(64);
    else if (d == 128) KV8_WRITE(128);
    else KV8_WRITE(256);
    RLLM_LAUNCH_CHECK();
    return 0;
  }
  const size_t smem = (size_t)rotary_dim * sizeof(float);
  RLLM_DISPATCH_DTYPE(dtype, T_,
    rllm_launch_pdl(kv_e4m3_write_kernel<T_>, dim3(T), dim3(256), smem, stream, (const T_*)qkv, (T_*)q_out, q_stride, positions,
                    token_seq, inv_freq, rotary_dim, block_table, max_blocks, num_seqs, (unsigned char*)kcache,
                    (unsigned char*)vcache, (unsigned char*)kscale, (unsigned char*)vscale, nq, nkv, d, page_size, num_pages, err));
  RLLM_LAUNCH_CHECK();
  return 0;
}

// ---------------------------------------------------------------------------
// read: out_k[t], out_v[t] = the rows of (token_seq[t], positions[t])
// ---------------------------------------------------------------------------
// A thread takes the same 16 numbers (16 bytes) of KV8_TOKENS tokens' rows, all of them on their way at once, and writes them as
// 16 values each.
#define KV8_TOKENS 2
template <typename T>
__global__ void __launch_bounds__(256)
kv_e4m3_read_kernel(const int* __restrict__ positions, const int* __restrict__ token_seq, const int* __restrict__ block_table,
                    int max_blocks, int num_seqs, const unsigned char* __restrict__ kcache,
                    const unsigned char* __restrict__ vcache, const unsigned char* __restrict__ kscale,
                    const unsigned char* __restrict__ vscale, T* __restrict__ out_k, T* __restrict__ out_v, int T_tokens,
                    int nkv, int d, int page_size, int num_pages, int* __restrict__ err) {
  pdl_wait_on(positions, token_seq, block_table, kcache, vcache, kscale, vscale);
  pdl_launch();
  const int per_row = d >> 4, pieces = nkv * per_row;  // pieces of a token's keys; as many of its values
  const long long t0 = (long long)blockIdx.x * KV8_TOKENS;
  int page[KV8_TOKENS], at[KV8_TOKENS];
#pragma unroll
  for (int u = 0; u < KV8_TOKENS; ++u) {
    const long long t = t0 + u;
    page[u] = -1;
    at[u] = 0;
    if (t < T_tokens) {
      const int pos = positions[t], seq = token_seq[t];
      if (pos >= 0 && pos / page_size < max_blocks && seq >= 0 && seq < num_seqs) {
        page[u] = block_table[(size_t)seq * max_blocks + pos / page_size];
        at[u] = pos % page_size;
        if (page[u] >= num_pages) page[u] = -1;
      }
      if (page[u] < 0 && threadIdx.x == 0) atomicOr(err, 4);
    }
  }
  for (int x = threadIdx.x; x < 2 * pieces; x += blockDim.x) {
    const bool value = x >= pieces;
    const int c = value ? x - pieces : x, h = c / per_row, i = (c - h * per_row) << 4;
    const unsigned char *codes = value ? vcache : kcache, *scale = value ? vscale : kscale;
    uint4 raw[KV8_TOKENS];
    int byte[KV8_TOKENS];
#pragma unroll
    for (int u = 0; u < KV8_TOKENS; ++u) {
      const long long r = ((long long)page[u] * nkv + h) * page_size + at[u];
      raw[u] = page[u] >= 0 ? *(const uint4*)(codes + r * d + i) : make_uint4(0u, 0u, 0u, 0u);
      byte[u] = page[u] >= 0 ? scale[r] : 0;
    }
#pragma unroll
    for (int u = 0; u < KV8_TOKENS; ++u) {
      if (t0 + u >= T_tokens) break;
      const float power = kv8_power(byte[u]);
      float y[16];
      kv8_floats(raw[u].x, y); kv8_floats(raw[u].y, y + 4); kv8_floats(raw[u].z, y + 8); kv8_floats(raw[u].w, y + 12);
      T* dst = (value ? out_v : out_k) + (size_t)(t0 + u) * nkv * d + (size_t)h * d + i;
      float lo[8], hi[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) { lo[k] = y[k] * power; hi[k] = y[k + 8] * power; }
      if constexpr (sizeof(T) == 4) {
        *(float4*)dst = make_float4(lo[0], lo[1], lo[2], lo[3]);
        *(float4*)(dst + 4) = make_float4(lo[4], lo[5], lo[6], lo[7]);
        *(float4*)(dst + 8) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        *(float4*)(dst + 12) = make_float4(hi[4], hi[5], hi[6], hi[7]);
      } else {
        store8(dst, lo);
        store8(dst + 8, hi);
      }
    }
  }
}

RLLM_EXPORT int rllm_kv_e4m3_read(const int* positions, const int* token_seq, const int* block_table, int max_blocks,
                                  int num_seqs, const void* kcache, const void* vcache, const void* kscale,
                                  const void* vscale, void* out_k, void* out_v, int dtype, int T, int nkv, int d,
                                  int page_size, int num_pages, int* err, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (!positions || !token_seq || !block_table || !kcache || !vcache || !kscale || !vscale || !out_k || !out_v || !err ||
      nkv <= 0 || d <= 0 || page_size <= 0 || num_pages <= 0 || max_blocks <= 0 || num_seqs <= 0)
    return RLLM_E_BADARG;
  if (d % 16 || d > 256) return RLLM_E_UNSUPPORTED;
  if (((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)out_k | (uintptr_t)out_v) & 15) return RLLM_E_UNSUPPORTED;
  const int threads = 2 * nkv * (d >> 4), block = threads >= 256 ? 256 : (threads + 31) / 32 * 32;
  const unsigned grid = (unsigned)(((long long)T + KV8_TOKENS - 1) / KV8_TOKENS);
  RLLM_DISPATCH_DTYPE(dtype, T_,
    rllm_launch_pdl(kv_e4m3_read_kernel<T_>, dim3(grid), dim3(block), (size_t)0, stream, positions, token_seq, block_table,
                    max_blocks, num_seqs, (const unsigned char*)kcache, (const unsigned char*)vcache,
                    (const unsigned char*)kscale, (const unsigned char*)vscale, (T_*)out_k, (T_*)out_v, T, nkv, d, page_size,
                    num_pages, err));
  RLLM_LAUNCH_CHECK();
  return 0;
}

// ---------------------------------------------------------------------------
// widen: what the prompt attention on tcgen05 reads of a step's sequences, as dense bfloat16 tiles
// ---------------------------------------------------------------------------
// A tile of the attention is BN = 8192 / D keys; one block widens the keys and values of a (tile, kv head, sequence), once for
// all the tiles of rows that read it (widened inside the attention they would be so by every CTA: 32 times for 1,024 tokens
// and 4 heads a kv head).  The values are exact (kv_e4m3.cuh), but for the rows that are NaN: such a token's key is NaN and its
// value 0, so that the product with the probabilities stays clean for the rows that do not see it, and those that do are NaN by
// its score.  Rows behind the sequence's end, and of pages that are not held, are zeros.  28,442 keys of 8 heads of 128 (175 MB
// in and out): 36 us, 4.9 TB/s.
template <int D>
__global__ void __launch_bounds__(512)
kv_e4m3_widen_kernel(const int* __restrict__ block_table, int max_blocks, const int* __restrict__ q_start,
                     const int* __restrict__ seq_lens, int seq_begin, const unsigned char* __restrict__ kcache,
                     const unsigned char* __restrict__ vcache, const unsigned char* __restrict__ kscale,
                     const unsigned char* __restrict__ vscale, bf16* __restrict__ kdense, bf16* __restrict__ vdense,
                     unsigned* __restrict__ marks, int nkv, int page_size, int num_pages, int window, int known, int* __restrict__ err) {
  constexpr int BN = 8192 / D, PIECES = D / 16;      // BN * PIECES = 512: a thread has 16 numbers of a key and of a value
  __shared__ unsigned mark[AT_MARK];
  kv8_inputs(known, block_table, q_start, seq_lens);
  const int page_shift = (page_size & (page_size - 1)) == 0 ? __ffs(page_size) - 1 : -1;
  const int s = seq_begin + blockIdx.z, kvh = blockIdx.y;
  const int len = seq_lens[s], pos0 = len - (q_start[s + 1] - q_start[s]);
  const int lo = window > 0 ? max(0, pos0 - window + 1) : 0, tile = lo / BN + blockIdx.x;
  if (threadIdx.x < AT_MARK) mark[threadIdx.x] = 0u;
  __syncthreads();
  const bool empty = tile * BN >= len;             // (nothing reads it)
  const int r = threadIdx.x / PIECES, j = tile * BN + r, c = (threadIdx.x % PIECES) * 16;
  long long row = -1;
  if (!empty && j >= lo && j < len) {
    const int at = page_shift >= 0 ? j >> page_shift : j / page_size;
    const int page = at < max_blocks ? block_table[(size_t)s * max_blocks + at] : -1;
    if (page >= 0 && page < num_pages) {
      row = ((long long)page * nkv + kvh) * page_size + (j - at * page_size);
    } else if (c == 0) {
      atomicOr(err, 4);
      atomicOr(&mark[1 + r / 32], 1u << (r & 31));
      atomicOr(&mark[0], AT_MARK_MISSING);
    }
  }
  kv8_begin(known, kcache, vcache, kscale, vscale, kdense, vdense, marks);
  kv8_let_in(known);
  if (empty) { kv8_end(known); return; }            // (the whole block)
  const bool held = row >= 0;
  const uint4 kx = held ? *(const uint4*)(kcache + row * D + c) : make_uint4(0u, 0u, 0u, 0u);
  const uint4 vx = held ? *(const uint4*)(vcache + row * D + c) : make_uint4(0u, 0u, 0u, 0u);
  const int kb = held ? kscale[row] : 0, vb = held ? vscale[row] : 0;
  const size_t base = (((size_t)blockIdx.z * gridDim.x + blockIdx.x) * nkv + kvh) * BN * D + threadIdx.x * 16;
  const bool odd = kb == KV8_NAN_SCALE || vb == KV8_NAN_SCALE;
  if (odd) atomicOr(&mark[0], AT_MARK_NAN);
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const uint4 raw = v ? vx : kx;
    const float power = odd ? 0.f : kv8_power(v ? vb : kb), more = odd && !v ? __uint_as_float(0x7FC00000u) : 0.f;
    float x[16], a[8], b[8];
    kv8_floats(raw.x, x); kv8_floats(raw.y, x + 4); kv8_floats(raw.z, x + 8); kv8_floats(raw.w, x + 12);
#pragma unroll
    for (int k = 0; k < 8; ++k) { a[k] = fmaf(x[k], power, more); b[k] = fmaf(x[k + 8], power, more); }
    bf16* dst = (v ? vdense : kdense) + base;
    store8(dst, a);
    store8(dst + 8, b);
  }
  __syncthreads();
  if (threadIdx.x < AT_MARK) marks[(((size_t)blockIdx.z * gridDim.x + blockIdx.x) * nkv + kvh) * AT_MARK + threadIdx.x] = mark[threadIdx.x];
  kv8_end(known);
}

// Sequences seq_begin .. seq_begin + num_seqs - 1, each from the tile of its portion's oldest visible key on, dense_tiles
// tiles at most: kdense, vdense [num_seqs][dense_tiles][nkv][8192 / d][d], marks [num_seqs][dense_tiles][nkv][AT_MARK].  known: see
// kv8_inputs.
RLLM_EXPORT int rllm_kv_e4m3_widen(const int* block_table, int max_blocks, const int* q_start, const int* seq_lens, int seq_begin,
                                   int num_seqs, int dense_tiles, const void* kcache, const void* vcache, const void* kscale,
                                   const void* vscale, void* kdense, void* vdense, void* marks, int nkv, int d, int page_size,
                                   int num_pages, int window, int known, int* err, cudaStream_t stream) {
  if (num_seqs <= 0) return 0;
  if (!block_table || !q_start || !seq_lens || !kcache || !vcache || !kscale || !vscale || !kdense || !vdense || !marks || !err ||
      seq_begin < 0 || dense_tiles <= 0 || nkv <= 0 || page_size <= 0 || num_pages <= 0 || max_blocks <= 0 || window < 0)
    return RLLM_E_BADARG;
  if (!(d == 64 || d == 128) || nkv > 65535 || num_seqs > 65535 ||
      (((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)kdense | (uintptr_t)vdense) & 15))
    return RLLM_E_UNSUPPORTED;
#define KV8_WIDEN(DD) rllm_launch_pdl(kv_e4m3_widen_kernel<DD>, dim3(dense_tiles, nkv, num_seqs), dim3(512), (size_t)0, stream, block_table, \
      max_blocks, q_start, seq_lens, seq_begin, (const unsigned char*)kcache, (const unsigned char*)vcache, (const unsigned char*)kscale,  \
      (const unsigned char*)vscale, (bf16*)kdense, (bf16*)vdense, (unsigned*)marks, nkv, page_size, num_pages, window, known, err)
  if (d == 64) KV8_WIDEN(64);
  else KV8_WIDEN(128);
  RLLM_LAUNCH_CHECK();
  return 0;
}
