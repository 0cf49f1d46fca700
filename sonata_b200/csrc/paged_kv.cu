// Paged KV cache of a ragged serving batch (bf16, B200): rotary positions
// with the append to the pages, attention of one new token a stream over its
// pages, and page copies.
//
// Pools: k and v pages [num_pages, nheads_kv, page_size, head_dim] (strides
// for the page, head and token axes, the last one dense); page_table [batch,
// max_pages] int32 names the page of each block of page_size positions of a
// stream; seq_lens [batch] int32 is on the device, so a captured step serves
// growing streams.  Pages and lengths out of range are never followed: the
// kernels skip them and record SN_ERR_INVALID_ARGUMENT in the status word.
#include "common.cuh"

#include <climits>

namespace sn {
namespace {

// A page table's entry for position `pos` of stream b, or -1.
struct PageMap {
  const int* table;  // [batch, table_stride]
  int64_t table_stride;
  int max_pages, num_pages, page_size;
};
__device__ __forceinline__ int page_of(const PageMap& m, int b, int block) {
  if (block < 0 || block >= m.max_pages) return -1;
  const int pg = m.table[static_cast<int64_t>(b) * m.table_stride + block];
  return static_cast<unsigned>(pg) < static_cast<unsigned>(m.num_pages) ? pg : -1;
}
struct PoolStrides {  // elements
  int64_t page, head, tok;
};

// ---------------------------------------------------------------------------
// rotary_paged_append.  Pure data movement (a qkv row read, q / k / v
// written, a cos / sin row per position), so it is bounded by HBM for
// prompts and by latency for a decode step.
// ---------------------------------------------------------------------------
struct AppendParams {
  const __nv_bfloat16* qkv;  // [tokens, ld]
  int64_t ld;
  __nv_bfloat16* q;  // [tokens, hq, hd]
  __nv_bfloat16 *kp, *vp;
  PoolStrides ks, vs;
  PageMap map;
  const int* seq_lens;  // lengths with the new tokens
  const int* cu;        // [batch + 1] token offsets, or null: one token a stream
  const float *cos, *sin;  // [max_pos, rot / 2]
  int tokens, batch, hq, hkv, hd, rot, max_pos, interleaved;
};

// The stream of token t: the last b with cu[b] <= t (binary search).
__device__ __forceinline__ int stream_of(const int* cu, int batch, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// One thread per (token, head, element pair of the head): elements (j, j +
// rot/2) or (2j, 2j + 1) of the rotated part, two neighbours past it.
__global__ void __launch_bounds__(256) rotary_paged_append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int h2 = p.hd / 2, heads = p.hq + 2 * p.hkv;
  const int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (e >= static_cast<int64_t>(p.tokens) * heads * h2) return;
  const int j = static_cast<int>(e % h2);
  const int head = static_cast<int>((e / h2) % heads);
  const int t = static_cast<int>(e / (static_cast<int64_t>(h2) * heads));
  const int b = p.cu ? stream_of(p.cu, p.batch, t) : t;
  const int end = p.cu ? p.cu[b + 1] : t + 1;
  if (p.cu && (t < p.cu[b] || t >= end)) return;  // a token of no stream
  const int pos = p.seq_lens[b] - (end - t);
  const bool rotated = head < p.hq + p.hkv && j < p.rot / 2;
  const bool halves = rotated && !p.interleaved;
  const int i1 = halves ? j : 2 * j, i2 = halves ? j + p.rot / 2 : 2 * j + 1;
  const __nv_bfloat16* src = p.qkv + t * p.ld + static_cast<int64_t>(head) * p.hd;
  __nv_bfloat16 o1 = src[i1], o2 = src[i2];
  if (pos < 0 || pos >= p.max_pos) {
    record_status(SN_ERR_INVALID_ARGUMENT);
    return;
  }
  if (rotated) {
    const float c = p.cos[static_cast<int64_t>(pos) * (p.rot / 2) + j], s = p.sin[static_cast<int64_t>(pos) * (p.rot / 2) + j];
    const float x1 = __bfloat162float(o1), x2 = __bfloat162float(o2);
    o1 = __float2bfloat16_rn(__fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s)));
    o2 = __float2bfloat16_rn(__fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s)));
  }
  __nv_bfloat16* dst;
  if (head < p.hq) {
    dst = p.q + (static_cast<int64_t>(t) * p.hq + head) * p.hd;
  } else {
    const int pg = page_of(p.map, b, pos / p.map.page_size);
    if (pg < 0) {
      record_status(SN_ERR_INVALID_ARGUMENT);
      return;
    }
    const bool k = head < p.hq + p.hkv;
    const PoolStrides& st = k ? p.ks : p.vs;
    dst = (k ? p.kp : p.vp) + pg * st.page + (head - p.hq - (k ? 0 : p.hkv)) * st.head +
          (pos % p.map.page_size) * st.tok;
  }
  dst[i1] = o1;
  dst[i2] = o2;
}

// ---------------------------------------------------------------------------
// paged_decode_attention, o = sum_t softmax_t(scale q.k_t) v_t, one pass over
// K and V with the running maximum and sum.
//
// One CTA per (stream, query head); each of its 4 warps takes every fourth
// position, lane l holds elements l, l + 32, ... of the head.
// ---------------------------------------------------------------------------
constexpr int kMaxHeadPerLane = 8;  // head_dim <= 256

struct AttendParams {
  const __nv_bfloat16* q;  // [batch, hq, hd], strides for batch and head
  int64_t qb, qh;
  const __nv_bfloat16 *kp, *vp;
  PoolStrides ks, vs;
  PageMap map;
  const int* seq_lens;
  __nv_bfloat16* out;  // [batch, hq, hd]
  float* lse;          // [batch, hq] or null
  float scale;
  int batch, hq, hkv, hd;
};

// Length of stream b, within the page table's reach.
__device__ __forceinline__ int stream_len(const AttendParams& p, int b) {
  const int n = p.seq_lens[b];
  const int64_t cap = static_cast<int64_t>(p.map.max_pages) * p.map.page_size;
  if (n < 0 || n > cap) {
    record_status(SN_ERR_INVALID_ARGUMENT);
    return n < 0 ? 0 : static_cast<int>(cap);
  }
  return n;
}

__global__ void __launch_bounds__(128) paged_decode_rows_kernel(const AttendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float sm[4], sl[4], so[4][32 * kMaxHeadPerLane];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / p.hq, h = blockIdx.x - b * p.hq;
  const int hk = h / (p.hq / p.hkv);
  const int len = stream_len(p, b);
  float qv[kMaxHeadPerLane], o[kMaxHeadPerLane];
#pragma unroll
  for (int i = 0; i < kMaxHeadPerLane; ++i) {
    const int c = lane + 32 * i;
    qv[i] = c < p.hd ? __bfloat162float(p.q[b * p.qb + h * p.qh + c]) * p.scale : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t < len; t += 4) {
    const int pg = page_of(p.map, b, t / p.map.page_size);
    if (pg < 0) {
      record_status(SN_ERR_INVALID_ARGUMENT);
      continue;
    }
    const int at = t % p.map.page_size;
    const __nv_bfloat16* kr = p.kp + pg * p.ks.page + hk * p.ks.head + at * p.ks.tok;
    const __nv_bfloat16* vr = p.vp + pg * p.vs.page + hk * p.vs.head + at * p.vs.tok;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxHeadPerLane; ++i) {
      const int c = lane + 32 * i;
      if (c < p.hd) s = fmaf(qv[i], __bfloat162float(kr[c]), s);
    }
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    const float keep = m == mn ? 1.f : expf(m - mn), w = s == -INFINITY ? 0.f : expf(s - mn);
    m = mn;
    l = fmaf(l, keep, w);
#pragma unroll
    for (int i = 0; i < kMaxHeadPerLane; ++i) {
      const int c = lane + 32 * i;
      if (c < p.hd) o[i] = fmaf(o[i], keep, w * __bfloat162float(vr[c]));
    }
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kMaxHeadPerLane; ++i) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  const float mt = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], lt = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : expf(sm[w] - mt);
    lt = fmaf(f[w], sl[w], lt);
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  for (int c = threadIdx.x; c < p.hd; c += 128) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v = fmaf(f[w], so[w][c], v);
    p.out[(static_cast<int64_t>(b) * p.hq + h) * p.hd + c] = __float2bfloat16_rn(v * inv);
  }
  if (p.lse && threadIdx.x == 0) p.lse[static_cast<int64_t>(b) * p.hq + h] = mt + logf(lt);
}

// ---------------------------------------------------------------------------
// copy_pages: pool [outer, num_pages, page_bytes] with byte strides; page
// src[i] -> page dst[i] in every outer index.
// ---------------------------------------------------------------------------
struct CopyParams {
  char* pool;
  int64_t outer_stride, page_stride, page_bytes;
  const int *src, *dst;
  int outer, num_pages, pairs;
};
constexpr int kCopyBytes = 16384;  // bytes a CTA copies

template <typename T>
__global__ void __launch_bounds__(256) copy_pages_kernel(const CopyParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x, o = blockIdx.y;
  const int s = p.src[i], d = p.dst[i];
  if (static_cast<unsigned>(s) >= static_cast<unsigned>(p.num_pages) ||
      static_cast<unsigned>(d) >= static_cast<unsigned>(p.num_pages)) {
    record_status(SN_ERR_INVALID_ARGUMENT);
    return;
  }
  const int64_t base = blockIdx.z * static_cast<int64_t>(kCopyBytes);
  const int n = static_cast<int>(min(static_cast<int64_t>(kCopyBytes), p.page_bytes - base) / sizeof(T));
  const T* from = reinterpret_cast<const T*>(p.pool + o * p.outer_stride + s * p.page_stride + base);
  T* to = reinterpret_cast<T*>(p.pool + o * p.outer_stride + d * p.page_stride + base);
  for (int k = threadIdx.x; k < n; k += 256) to[k] = from[k];
}

inline bool pool_ok(int64_t page, int64_t head, int64_t tok, int nheads, int page_size, int hd) {
  // rows dense, axes in any order but not overlapping below the row
  return tok >= hd && head >= hd && page >= hd && nheads >= 1 && page_size >= 1;
}

}  // namespace

int tu_status_paged(bool reset, cudaStream_t st, int* out) { return read_tu_status(reset, st, out); }

}  // namespace sn

extern "C" {

int sn_rotary_paged_append(const void* qkv, int64_t ld, void* q, void* k_pages, int64_t k_page_stride,
                           int64_t k_head_stride, int64_t k_tok_stride, void* v_pages, int64_t v_page_stride,
                           int64_t v_head_stride, int64_t v_tok_stride, int num_pages, int page_size,
                           const int* page_table, int64_t table_stride, int max_pages, const int* seq_lens,
                           const int* cu_seqlens, const float* cos, const float* sin, int max_pos, int tokens,
                           int batch, int nheads, int nheads_kv, int head_dim, int rot_dim, int interleaved,
                           void* stream) {
  if (!qkv || !q || !k_pages || !v_pages || !page_table || !seq_lens || tokens < 0 || batch < 1 || nheads < 1 ||
      nheads_kv < 1 || head_dim < 2 || head_dim % 2 != 0 || rot_dim < 0 || rot_dim % 2 != 0 || rot_dim > head_dim ||
      num_pages < 1 || page_size < 1 || max_pages < 1 || table_stride < max_pages || max_pos < 1 ||
      (rot_dim > 0 && (!cos || !sin)) || (!cu_seqlens && tokens != batch))
    return SN_ERR_INVALID_ARGUMENT;
  const int64_t width = (static_cast<int64_t>(nheads) + 2 * static_cast<int64_t>(nheads_kv)) * head_dim;
  if (ld < width || !sn::pool_ok(k_page_stride, k_head_stride, k_tok_stride, nheads_kv, page_size, head_dim) ||
      !sn::pool_ok(v_page_stride, v_head_stride, v_tok_stride, nheads_kv, page_size, head_dim))
    return SN_ERR_INVALID_ARGUMENT;
  if (width > INT32_MAX) return SN_ERR_UNSUPPORTED;
  if (tokens == 0) return SN_OK;
  sn::AppendParams p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.ld = ld;
  p.q = static_cast<__nv_bfloat16*>(q);
  p.kp = static_cast<__nv_bfloat16*>(k_pages);
  p.vp = static_cast<__nv_bfloat16*>(v_pages);
  p.ks = {k_page_stride, k_head_stride, k_tok_stride};
  p.vs = {v_page_stride, v_head_stride, v_tok_stride};
  p.map = {page_table, table_stride, max_pages, num_pages, page_size};
  p.seq_lens = seq_lens;
  p.cu = cu_seqlens;
  p.cos = cos;
  p.sin = sin;
  p.tokens = tokens;
  p.batch = batch;
  p.hq = nheads;
  p.hkv = nheads_kv;
  p.hd = head_dim;
  p.rot = rot_dim;
  p.max_pos = max_pos;
  p.interleaved = interleaved ? 1 : 0;
  const int64_t blocks = (static_cast<int64_t>(tokens) * (width / 2) + 255) / 256;
  if (blocks > INT32_MAX) return SN_ERR_UNSUPPORTED;
  return sn::launch(sn::rotary_paged_append_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                    static_cast<cudaStream_t>(stream), true, p);
}

size_t sn_paged_decode_workspace_size(int batch, int nheads, int head_dim) {
  if (batch < 1 || nheads < 1 || head_dim < 1) return 0;
  return 16;
}

int sn_paged_decode_attention(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_pages,
                              int64_t k_page_stride, int64_t k_head_stride, int64_t k_tok_stride, const void* v_pages,
                              int64_t v_page_stride, int64_t v_head_stride, int64_t v_tok_stride, int num_pages,
                              int page_size, const int* page_table, int64_t table_stride, int max_pages,
                              const int* seq_lens, void* out, float* lse, float scale, int batch, int nheads,
                              int nheads_kv, int head_dim, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_pages || !v_pages || !page_table || !seq_lens || !out || !workspace || batch < 1 || nheads < 1 ||
      nheads_kv < 1 || nheads % nheads_kv != 0 || head_dim < 1 || num_pages < 1 || page_size < 1 || max_pages < 1 ||
      table_stride < max_pages || q_batch_stride < 0 || q_head_stride < 0)
    return SN_ERR_INVALID_ARGUMENT;
  if (!sn::pool_ok(k_page_stride, k_head_stride, k_tok_stride, nheads_kv, page_size, head_dim) ||
      !sn::pool_ok(v_page_stride, v_head_stride, v_tok_stride, nheads_kv, page_size, head_dim) ||
      workspace_bytes < sn_paged_decode_workspace_size(batch, nheads, head_dim))
    return SN_ERR_INVALID_ARGUMENT;
  if (head_dim > 32 * sn::kMaxHeadPerLane || static_cast<int64_t>(batch) * nheads > INT32_MAX ||
      static_cast<int64_t>(max_pages) * page_size > INT32_MAX)
    return SN_ERR_UNSUPPORTED;
  sn::AttendParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.qb = q_batch_stride;
  p.qh = q_head_stride;
  p.kp = static_cast<const __nv_bfloat16*>(k_pages);
  p.vp = static_cast<const __nv_bfloat16*>(v_pages);
  p.ks = {k_page_stride, k_head_stride, k_tok_stride};
  p.vs = {v_page_stride, v_head_stride, v_tok_stride};
  p.map = {page_table, table_stride, max_pages, num_pages, page_size};
  p.seq_lens = seq_lens;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.scale = scale;
  p.batch = batch;
  p.hq = nheads;
  p.hkv = nheads_kv;
  p.hd = head_dim;
  return sn::launch(sn::paged_decode_rows_kernel, dim3(static_cast<unsigned>(batch * nheads)), dim3(128), 0,
                    static_cast<cudaStream_t>(stream), true, p);
}

int sn_copy_pages(void* pool, int64_t outer_stride_bytes, int64_t page_stride_bytes, int64_t page_bytes, int outer,
                  int num_pages, const int* src, const int* dst, int pairs, void* stream) {
  if (!pool || (pairs > 0 && (!src || !dst)) || outer < 1 || num_pages < 1 || pairs < 0 || page_bytes < 1 ||
      page_stride_bytes < page_bytes || (outer > 1 && outer_stride_bytes < page_bytes))
    return SN_ERR_INVALID_ARGUMENT;
  if (pairs == 0) return SN_OK;
  const int64_t parts = (page_bytes + sn::kCopyBytes - 1) / sn::kCopyBytes;
  if (outer > 65535 || parts > 65535) return SN_ERR_UNSUPPORTED;
  sn::CopyParams p;
  p.pool = static_cast<char*>(pool);
  p.outer_stride = outer_stride_bytes;
  p.page_stride = page_stride_bytes;
  p.page_bytes = page_bytes;
  p.src = src;
  p.dst = dst;
  p.outer = outer;
  p.num_pages = num_pages;
  p.pairs = pairs;
  const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(outer), static_cast<unsigned>(parts));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = sn::aligned16(pool) && (outer == 1 || outer_stride_bytes % 16 == 0) &&
                    page_stride_bytes % 16 == 0 && page_bytes % 16 == 0;
  return wide ? sn::launch(sn::copy_pages_kernel<uint4>, grid, dim3(256), 0, st, true, p)
              : sn::launch(sn::copy_pages_kernel<char>, grid, dim3(256), 0, st, true, p);
}

}  // extern "C"
