// Attention to some of a paged cache's blocks (B200): the bounds of each
// page's keys, and the choice of the blocks a query attends to.  The attention
// over the chosen blocks is paged_sparse_attention (paged_kv.cu).
//
// bounds [num_pages, hkv, 2, hd] bf16: for each page and key/value head the
// elementwise least and greatest key.  For a query q and any key k of the page
//   q . k <= sum_d max(q_d least_d, q_d greatest_d),
// with equality where one key has all the extremes.
#include "paged.cuh"
#include "select.cuh"

#include <algorithm>
#include <climits>

namespace sn {
namespace {

// ---------------------------------------------------------------------------
// update_page_bounds: the bounds of each page that holds new tokens, from all
// of its keys (so pages that were begun before, copied or refilled come out
// right).  One warp a (page, head): a row is read by 16-byte pieces, as many
// rows at once as the warp has lanes for.  How many pages there are is known on
// the device only (cu[batch]), so the warps of a grid of bounded size share them.
// ---------------------------------------------------------------------------
struct BoundsParams {
  const __nv_bfloat16* kp;
  PoolStrides ks;
  PageMap map;
  const int* seq_lens;  // with the new tokens
  const int* cu;        // [batch + 1], or null: one new token a stream
  __nv_bfloat16* bounds;
  int batch, hkv, hd;
};

// Stream b's touched blocks have slots cu[b] / page + 2 b and following: n new tokens touch n / page + 2 blocks at most.
__device__ __forceinline__ int64_t first_slot(const BoundsParams& p, int b) {
  return static_cast<int64_t>(max(p.cu[b], 0)) / p.map.page_size + 2 * static_cast<int64_t>(b);
}

// Work items: (touched page, head).
__device__ __forceinline__ int64_t bounds_items(const BoundsParams& p) { return (p.cu ? first_slot(p, p.batch) : p.batch) * p.hkv; }

// The page of work item `slot` and the keys that count in it, or -1.
__device__ __forceinline__ int touched(const BoundsParams& p, int64_t slot, int& rows) {
  int b, block;
  if (!p.cu) {
    b = static_cast<int>(slot);
    const int n = length_of(p.map, p.seq_lens, b);
    if (n < 1) return -1;
    block = (n - 1) / p.map.page_size;
    rows = n - block * p.map.page_size;
  } else {
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_slot(p, mid) <= slot) lo = mid; else hi = mid - 1;
    }
    b = lo;
    const int n = length_of(p.map, p.seq_lens, b), fresh = min(p.cu[b + 1] - p.cu[b], n);
    if (fresh < 1) return -1;
    const int64_t at = (n - fresh) / p.map.page_size + (slot - first_slot(p, b));
    if (at > (n - 1) / p.map.page_size) return -1;
    block = static_cast<int>(at);
    rows = min(n - block * p.map.page_size, p.map.page_size);
  }
  const int pg = page_of(p.map, b, block);
  if (pg < 0) record_status(SN_ERR_INVALID_ARGUMENT);
  return pg;
}

__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Rows of 16-byte pieces (head_dim a multiple of 8, at most 256): L lanes a row, 32 / L rows at a time.
__global__ void __launch_bounds__(128) page_bounds_kernel(const BoundsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t items = bounds_items(p);
  for (int64_t item = blockIdx.x * int64_t{4} + (threadIdx.x >> 5); item < items; item += gridDim.x * int64_t{4}) {
    const int h = static_cast<int>(item % p.hkv);
    int rows = 0;
    const int pg = touched(p, item / p.hkv, rows);
    if (pg < 0) continue;
    const int pieces = p.hd / 8;
    int L = 1;
    while (L < pieces) L *= 2;  // a power of two, for the exchange
    const int groups = 32 / L, group = lane / L, c = lane % L;
    const __nv_bfloat16* src = p.kp + pg * p.ks.page + h * p.ks.head + 8 * c;
    uint4 lo, hi;
    lo.x = lo.y = lo.z = lo.w = 0x7f807f80u;  // infinities
    hi.x = hi.y = hi.z = hi.w = 0xff80ff80u;
    if (c < pieces) {
#pragma unroll 8
      for (int r = group; r < rows; r += groups) {
        const uint4 k = *reinterpret_cast<const uint4*>(src + r * p.ks.tok);
        lo.x = min2(lo.x, k.x), lo.y = min2(lo.y, k.y), lo.z = min2(lo.z, k.z), lo.w = min2(lo.w, k.w);
        hi.x = max2(hi.x, k.x), hi.y = max2(hi.y, k.y), hi.z = max2(hi.z, k.z), hi.w = max2(hi.w, k.w);
      }
    }
    for (int o = L; o < 32; o *= 2) {
      lo.x = min2(lo.x, __shfl_xor_sync(0xffffffffu, lo.x, o)), lo.y = min2(lo.y, __shfl_xor_sync(0xffffffffu, lo.y, o));
      lo.z = min2(lo.z, __shfl_xor_sync(0xffffffffu, lo.z, o)), lo.w = min2(lo.w, __shfl_xor_sync(0xffffffffu, lo.w, o));
      hi.x = max2(hi.x, __shfl_xor_sync(0xffffffffu, hi.x, o)), hi.y = max2(hi.y, __shfl_xor_sync(0xffffffffu, hi.y, o));
      hi.z = max2(hi.z, __shfl_xor_sync(0xffffffffu, hi.z, o)), hi.w = max2(hi.w, __shfl_xor_sync(0xffffffffu, hi.w, o));
    }
    if (group == 0 && c < pieces) {
      __nv_bfloat16* dst = p.bounds + (static_cast<int64_t>(pg) * p.hkv + h) * 2 * p.hd + 8 * c;
      *reinterpret_cast<uint4*>(dst) = lo;
      *reinterpret_cast<uint4*>(dst + p.hd) = hi;
    }
  }
}

// Any rows: a lane an element.
__global__ void __launch_bounds__(128) page_bounds_rows_kernel(const BoundsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t items = bounds_items(p);
  for (int64_t item = blockIdx.x * int64_t{4} + (threadIdx.x >> 5); item < items; item += gridDim.x * int64_t{4}) {
    const int h = static_cast<int>(item % p.hkv);
    int rows = 0;
    const int pg = touched(p, item / p.hkv, rows);
    if (pg < 0) continue;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(p.kp) + pg * p.ks.page + h * p.ks.head;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.bounds) + (static_cast<int64_t>(pg) * p.hkv + h) * 2 * p.hd;
    for (int c = lane; c < p.hd; c += 32) {
      uint32_t lo = 0x7f80u, hi = 0xff80u;
      for (int r = 0; r < rows; ++r) {
        const uint32_t k = src[r * p.ks.tok + c];
        lo = min2(lo, k);
        hi = max2(hi, k);
      }
      dst[c] = static_cast<uint16_t>(lo);
      dst[p.hd + c] = static_cast<uint16_t>(hi);
    }
  }
}

// ---------------------------------------------------------------------------
// select_blocks.  For each (stream, key/value head) the score of a block is
// the greatest over the head's query heads of sum_d max(q_d least_d, q_d
// greatest_d); the first `first` and last `last` blocks and the highest
// scores of the others are listed in ascending order, -1 behind.  The products
// of two bf16 values are exact, and they are added up in 64 bits, so the choice
// does not depend on the order of the sum.  One cluster a (stream, head), the
// scores' keys in its shared memory.
//
// Four lanes take a block: lane t the 16-byte pieces t, t + 4, ... of both rows.
// max(q l, q g) = q (q < 0 ? l : g), one 64-bit multiply-add.  A bf16 value's
// bits, moved into the upper word of a double, are that value times 2^-896,
// zeros and subnormals too; q is multiplied by 2^800 for it, which leaves the
// order as it is.  A block with a bound that is not finite ranks above all.
// ---------------------------------------------------------------------------
constexpr int kSelHeads = 4;      // query heads at a time
constexpr int kSelMost = 22528;   // blocks a CTA's shared memory holds the keys of (180 KB)

struct SelectParams {
  const __nv_bfloat16* q;
  int64_t qb, qh;
  const __nv_bfloat16* bounds;
  PageMap map;
  const int* seq_lens;
  int* blocks;  // [batch, hkv, count]
  int batch, hq, hkv, hd, count, first, last;
  int part;  // keys a CTA holds
};

// kVec: pieces of 8 elements are 16-byte loads (head_dim a multiple of 8).
template <bool kVec>
__global__ void __launch_bounds__(kSelThreads) select_blocks_kernel(const SelectParams p) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  uint64_t* const s_keys = reinterpret_cast<uint64_t*>(s_raw);                   // [part]
  uint32_t* const s_bits = reinterpret_cast<uint32_t*>(s_keys + p.part);         // [part / 32], even
  __shared__ SelectShared s_sel;
  __shared__ uint32_t s_n, s_count;
  const int pieces = (p.hd + 7) / 8;
  double* const s_q = reinterpret_cast<double*>(s_bits + (p.part / 32 + 3) / 2 * 2);  // [kSelHeads][8 pieces]
  pdl_launch_dependents();
  pdl_wait();
  uint32_t nranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nranks));
  const int C = static_cast<int>(nranks), rank = static_cast<int>(ctarank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / C, b = row / p.hkv, hk = row % p.hkv;
  if (tid == 0) s_n = length_of(p.map, p.seq_lens, b);
  cluster_bar(C);
  const int n = static_cast<int>(peer_u32(&s_n, 0));
  const int nb = static_cast<int>((static_cast<int64_t>(n) + p.map.page_size - 1) / p.map.page_size);
  int* const out = p.blocks + static_cast<int64_t>(row) * p.count;
  if (nb <= p.count) {
    for (int i = rank * kSelThreads + tid; i < p.count; i += C * kSelThreads) out[i] = i < nb ? i : -1;
    cluster_bar(C);
    return;
  }
  for (int i = rank * kSelThreads + tid; i < p.first + p.last; i += C * kSelThreads) {
    if (i < p.first) out[i] = i;
    else out[p.count - p.last + i - p.first] = nb - p.last + i - p.first;
  }
  const int need = p.count - p.first - p.last, c = nb - p.first - p.last;
  if (need == 0) {
    cluster_bar(C);
    return;
  }
  const int each = (c + C - 1) / C;
  const int i0 = min(rank * each, c), len = min(i0 + each, c) - i0;  // blocks first + i0 ..

  // ---- scores ----
  const int group = p.hq / p.hkv, t = lane & 3;
  for (int g0 = 0; g0 < group; g0 += kSelHeads) {
    const int nh = min(kSelHeads, group - g0);
    __syncthreads();
    for (int e = tid; e < kSelHeads * 8 * pieces; e += kSelThreads) {
      const int h = e / (8 * pieces), d = e - h * 8 * pieces;
      double v = 0.;
      if (h < nh && d < p.hd) v = static_cast<double>(__bfloat162float(p.q[b * p.qb + (hk * group + g0 + h) * p.qh + d])) * 0x1p800;
      s_q[e] = v;
    }
    __syncthreads();
    for (int i = warp * 8 + (lane >> 2); i < (len + 7) / 8 * 8; i += kSelWarps * 8) {
      const bool there = i < len;
      int pg = -1;
      if (there) {
        pg = page_of(p.map, b, p.first + i0 + i);
        if (pg < 0) record_status(SN_ERR_INVALID_ARGUMENT);
      }
      const __nv_bfloat16* lo = p.bounds + (static_cast<int64_t>(max(pg, 0)) * p.hkv + hk) * 2 * p.hd;
      double acc[kSelHeads] = {0., 0., 0., 0.};
      bool odd = false;  // a bound that is not finite
      for (int k = t; k < pieces; k += 4) {
        uint32_t l[4], g[4];
        if constexpr (kVec) {
          *reinterpret_cast<uint4*>(l) = *reinterpret_cast<const uint4*>(lo + 8 * k);
          *reinterpret_cast<uint4*>(g) = *reinterpret_cast<const uint4*>(lo + p.hd + 8 * k);
        } else {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(lo) + 8 * k;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int d = 8 * k + 2 * j;
            l[j] = (d < p.hd ? e[2 * j] : 0u) | (d + 1 < p.hd ? static_cast<uint32_t>(e[2 * j + 1]) << 16 : 0u);
            g[j] = (d < p.hd ? e[p.hd + 2 * j] : 0u) | (d + 1 < p.hd ? static_cast<uint32_t>(e[p.hd + 2 * j + 1]) << 16 : 0u);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t wl = j & 1 ? l[j / 2] >> 16 : l[j / 2] & 0xffffu, wg = j & 1 ? g[j / 2] >> 16 : g[j / 2] & 0xffffu;
          odd |= (wl & 0x7f80u) == 0x7f80u || (wg & 0x7f80u) == 0x7f80u;
          const int dl = static_cast<int>((wl & 0x8000u) << 16 | (wl & 0x7fffu) << 13);
          const int dg = static_cast<int>((wg & 0x8000u) << 16 | (wg & 0x7fffu) << 13);
#pragma unroll
          for (int h = 0; h < kSelHeads; ++h) {
            const double q = s_q[h * 8 * pieces + 8 * k + j];
            acc[h] = fma(q, __hiloint2double(q < 0. ? dl : dg, 0), acc[h]);
          }
        }
      }
      uint64_t best = 0;
#pragma unroll
      for (int h = 0; h < kSelHeads; ++h) {
        acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 1);
        acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2);
        if (h < nh) best = max(best, order_key(acc[h]));
      }
      odd = __ballot_sync(0xffffffffu, odd) >> (lane & 28) & 15;
      if (odd) best = ~0ull;
      if (pg < 0) best = 0;
      if (there && t == 0) s_keys[i] = g0 == 0 ? best : max(best, s_keys[i]);
    }
  }
  __syncthreads();

  // ---- the choice, in ascending order ----
  const Cutoff<uint64_t> cut = find_cutoff(s_keys, len, static_cast<uint32_t>(need), s_sel, C, rank);
  choose(s_keys, len, cut, s_bits, s_sel);
  __syncthreads();
  const int words = (len + 31) / 32, per = (words + kSelWarps - 1) / kSelWarps;
  const int w0 = min(warp * per, words), w1 = min(w0 + per, words);
  uint32_t cnt = 0;
  for (int w = w0 + lane; w < w1; w += 32) cnt += __popc(s_bits[w]);
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  if (lane == 0) s_sel.warp[warp] = cnt;
  __syncthreads();
  uint32_t at = 0, all = 0;
  for (int v = 0; v < kSelWarps; ++v) {
    if (v == warp) at = all;
    all += s_sel.warp[v];
  }
  if (tid == 0) s_count = all;
  cluster_bar(C);
  for (int r = 0; r < rank; ++r) at += peer_u32(&s_count, r);
  for (int w = w0; w < w1; ++w) {
    const uint32_t word = s_bits[w];
    if ((word >> lane) & 1) out[p.first + at + __popc(word & ((1u << lane) - 1))] = p.first + i0 + 32 * w + lane;
    at += __popc(word);
  }
  cluster_bar(C);  // nobody leaves while its count may be read
}

template <bool kVec>
int launch_select(int rows, int C, size_t smem, cudaStream_t st, const SelectParams& p) {
  if (!smem_room<select_blocks_kernel<kVec>>(210 * 1024)) return SN_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * C);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(C);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, select_blocks_kernel<kVec>, p) != cudaSuccess) {
    cudaGetLastError();
    return SN_ERR_LAUNCH;
  }
  return SN_OK;
}

}  // namespace

int tu_status_sparse(bool reset, cudaStream_t st, int* out) { return read_tu_status(reset, st, out); }

}  // namespace sn

extern "C" {

int sn_update_page_bounds(const void* k_pages, int64_t k_page_stride, int64_t k_head_stride, int64_t k_tok_stride,
                          int num_pages, int page_size, const int* page_table, int64_t table_stride, int max_pages,
                          const int* seq_lens, const int* cu_seqlens, int batch, int nheads_kv, int head_dim,
                          void* bounds, void* stream) {
  if (!k_pages || !page_table || !seq_lens || !bounds || num_pages < 1 || page_size < 1 || max_pages < 1 ||
      table_stride < max_pages || batch < 1 || nheads_kv < 1 || head_dim < 1 ||
      !sn::pool_ok(k_page_stride, k_head_stride, k_tok_stride, nheads_kv, page_size, head_dim))
    return SN_ERR_INVALID_ARGUMENT;
  if (static_cast<int64_t>(max_pages) * page_size > INT32_MAX) return SN_ERR_UNSUPPORTED;
  // no more warps than the tables have pages for, and no more CTAs than fit on the device together
  const int64_t slots = cu_seqlens ? (max_pages + int64_t{2}) * batch : batch;
  const int64_t ctas = std::min<int64_t>((slots * nheads_kv + 3) / 4, 16 * sn::sm_count());
  sn::BoundsParams p;
  p.kp = static_cast<const __nv_bfloat16*>(k_pages);
  p.ks = {k_page_stride, k_head_stride, k_tok_stride};
  p.map = {page_table, table_stride, max_pages, num_pages, page_size};
  p.seq_lens = seq_lens;
  p.cu = cu_seqlens;
  p.bounds = static_cast<__nv_bfloat16*>(bounds);
  p.batch = batch;
  p.hkv = nheads_kv;
  p.hd = head_dim;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(ctas));
  if (head_dim % 8 == 0 && head_dim <= 256 && sn::aligned16(bounds) && sn::rows16(k_pages, k_page_stride, k_head_stride, k_tok_stride))
    return sn::launch(sn::page_bounds_kernel, grid, dim3(128), 0, st, true, p);
  return sn::launch(sn::page_bounds_rows_kernel, grid, dim3(128), 0, st, true, p);
}

int sn_select_blocks(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* bounds, int num_pages,
                     int page_size, const int* page_table, int64_t table_stride, int max_pages, const int* seq_lens,
                     int batch, int nheads, int nheads_kv, int head_dim, int count, int first, int last, int* blocks,
                     void* stream) {
  if (!q || !bounds || !page_table || !seq_lens || !blocks || num_pages < 1 || page_size < 1 || max_pages < 1 ||
      table_stride < max_pages || batch < 1 || nheads < 1 || nheads_kv < 1 || nheads % nheads_kv != 0 || head_dim < 1 ||
      q_batch_stride < 0 || q_head_stride < 0 || count < 1 || first < 0 || last < 0 || first > count ||
      last > count - first)
    return SN_ERR_INVALID_ARGUMENT;
  const int64_t rows = static_cast<int64_t>(batch) * nheads_kv;
  if (head_dim > 512 || rows > INT32_MAX / sn::kClusterMost || max_pages > sn::kClusterMost * (sn::kSelMost - 1) ||
      static_cast<int64_t>(max_pages) * page_size > INT32_MAX)
    return SN_ERR_UNSUPPORTED;
  sn::SelectParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.qb = q_batch_stride;
  p.qh = q_head_stride;
  p.bounds = static_cast<const __nv_bfloat16*>(bounds);
  p.map = {page_table, table_stride, max_pages, num_pages, page_size};
  p.seq_lens = seq_lens;
  p.blocks = blocks;
  p.batch = batch;
  p.hq = nheads;
  p.hkv = nheads_kv;
  p.hd = head_dim;
  p.count = count;
  p.first = first;
  p.last = last;
  // CTAs a row: as many as the shared memory asks for, and more where there are few long rows
  int C = 1;
  while (C < sn::kClusterMost && (max_pages > C * (sn::kSelMost - 1) || (rows * C < 2 * sn::sm_count() && max_pages > 128 * C)))
    C *= 2;
  p.part = (max_pages + C - 1) / C + 1;
  const size_t smem = static_cast<size_t>(p.part) * 8 + (p.part / 32 + 3) / 2 * 2 * 4 +
                      static_cast<size_t>(sn::kSelHeads) * ((head_dim + 7) / 8 * 8) * 8;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int r = static_cast<int>(rows);
  return head_dim % 8 == 0 && sn::aligned16(bounds) ? sn::launch_select<true>(r, C, smem, st, p)
                                                    : sn::launch_select<false>(r, C, smem, st, p);
}

}  // extern "C"
