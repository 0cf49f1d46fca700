// Eviction from the paged KV cache by accumulated attention weight (B200).
//
// In every layer, stream and key/value head with n > keep positions, `keep` of
// them stay: the first `sinks`, the last `recent`, and of the others (the
// candidates) the keep - sinks - recent of the highest mass, the lowest
// positions among equal ones.  The attention does not ask for an order, so
// what already lies in front stays where it is: the places below keep - recent
// that are not kept (holes) take, in order, the chosen candidates from behind
// (movers; there are as many), and the recent positions follow in their order,
// so that the last `recent` places are the newest ones the next time too.
// mass goes with its position and is zero behind.
#include "paged.cuh"
#include "select.cuh"

#include <algorithm>
#include <climits>

namespace sn {
namespace {

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;
constexpr int kEvictCluster = 8;  // CTAs a row at most

struct EvictParams {
  char* pool;  // [layers, 2, num_pages, hkv, page_size] rows of row_bytes, dense
  int64_t layer_bytes, kv_bytes, page_bytes, head_bytes;
  int row_bytes;
  PageMap map;
  const int* seq_lens;
  float* mass;  // [layers, batch, hkv, >= capacity] by strides
  int64_t ml, mb, mh;
  int* source;  // [layers, batch, hkv, keep] or null
  int batch, hkv, keep, recent, sinks;
  int part;  // candidates a CTA's shared memory holds
};

// One cluster a (layer, stream, head).  The candidates' keys lie in the
// cluster's shared memory, consecutive parts in its CTAs, so that the choice
// (select.cuh) reads mass once; then the same memory holds the lists of holes
// and movers, and all warps of the cluster take pairs of them.  A warp's lanes
// look up 32 pairs at once and copy K and V rows by 16 bytes, eight loads in
// flight.  The recent rows may overlap their places: they are read, the
// cluster waits, they are written.
template <typename T, int NU>  // units of T in a position's two rows, 0: 2 * row_bytes / sizeof(T)
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictParams p) {
  constexpr int U = 8;  // units in flight a lane
  extern __shared__ uint32_t s_keys[];  // [part], then the bits [part / 32]
  __shared__ SelectShared<kEvictThreads> s_sel;
  __shared__ uint32_t s_n, s_count[2];
  pdl_launch_dependents();
  pdl_wait();
  uint32_t nranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nranks));
  const int C = static_cast<int>(nranks), rank = static_cast<int>(ctarank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / C;
  const int h = row % p.hkv, b = row / p.hkv % p.batch, layer = row / p.hkv / p.batch;
  if (tid == 0) s_n = length_of(p.map, p.seq_lens, b);
  cluster_bar(C);
  const int n = static_cast<int>(peer_u32(&s_n, 0));  // one reading for all of the cluster
  const int keep = p.keep, recent = p.recent, sinks = p.sinks;
  int* const source = p.source ? p.source + static_cast<int64_t>(row) * keep : nullptr;
  if (n <= keep) {
    if (source)
      for (int i = rank * kEvictThreads + tid; i < keep; i += C * kEvictThreads) source[i] = i < n ? i : -1;
    cluster_bar(C);  // nobody leaves while its n may be read
    return;
  }
  float* const mass = p.mass + layer * p.ml + b * p.mb + h * p.mh;
  const int edge = keep - recent;               // places below: sinks, then chosen candidates
  const int c = n - recent - sinks, m = edge - sinks;  // candidates, and those that stay
  uint32_t* const s_bits = s_keys + p.part;
  // this CTA's candidates: positions sinks + i0 .. sinks + i1 - 1
  const int each = ((c + C - 1) / C + 3) / 4 * 4;
  const int i0 = min(rank * each, c), i1 = min(i0 + each, c), len = i1 - i0;
  uint32_t nholes = 0, nmovers = 0;  // in this CTA
  if (m > 0) {
    for (int i = tid; i < len; i += kEvictThreads) s_keys[i] = order_key(mass[sinks + i0 + i]);
    __syncthreads();
    const Cutoff<uint32_t> cut = find_cutoff(s_keys, len, static_cast<uint32_t>(m), s_sel, C, rank);
    choose(s_keys, len, cut, s_bits, s_sel);
    __syncthreads();  // the keys are done with: the lists go over them, holes from the front, movers from the back
    const int words = (len + 31) / 32, per = (words + kEvictWarps - 1) / kEvictWarps;
    const int w0 = min(warp * per, words), w1 = min(w0 + per, words);
    auto split = [&](int w, uint32_t& hole, uint32_t& mover) {  // of word w's candidates
      const int at = sinks + i0 + 32 * w, there = min(32, len - 32 * w);
      const uint32_t valid = there < 32 ? (1u << there) - 1 : 0xffffffffu;
      const int front = min(max(edge - at, 0), 32);  // that many lie below the edge
      const uint32_t low = front < 32 ? (1u << front) - 1 : 0xffffffffu;
      hole = ~s_bits[w] & low & valid;
      mover = s_bits[w] & ~low & valid;
    };
    uint32_t nh = 0, nm = 0, hole, mover;
    for (int w = w0 + lane; w < w1; w += 32) {
      split(w, hole, mover);
      nh += __popc(hole);
      nm += __popc(mover);
    }
    nh = __reduce_add_sync(0xffffffffu, nh);
    nm = __reduce_add_sync(0xffffffffu, nm);
    if (lane == 0) {
      s_sel.warp[warp] = nh;
      s_sel.warp2[warp] = nm;
    }
    __syncthreads();
    uint32_t ah = 0, am = 0;
    for (int v = 0; v < kEvictWarps; ++v) {
      if (v == warp) {
        ah = nholes;
        am = nmovers;
      }
      nholes += s_sel.warp[v];
      nmovers += s_sel.warp2[v];
    }
    const uint32_t below = (1u << lane) - 1;
    for (int w = w0; w < w1; ++w) {
      split(w, hole, mover);
      const int at = sinks + i0 + 32 * w + lane;
      if ((hole >> lane) & 1) s_keys[ah + __popc(hole & below)] = at;
      if ((mover >> lane) & 1) s_keys[p.part - 1 - (am + __popc(mover & below))] = at;
      if (source && at < edge && 32 * w + lane < len && !((hole >> lane) & 1)) source[at] = at;
      ah += __popc(hole);
      am += __popc(mover);
    }
  }
  if (source)
    for (int i = rank * kEvictThreads + tid; i < sinks; i += C * kEvictThreads) source[i] = i;
  if (tid == 0) {
    s_count[0] = nholes;
    s_count[1] = nmovers;
  }
  cluster_bar(C);  // the lists and their lengths are there

  const int nu = NU ? NU : static_cast<int>(2 * p.row_bytes / sizeof(T));
  char* const base = p.pool + layer * p.layer_bytes + h * p.head_bytes;
  // where a position's K row is, or -1
  auto place = [&](int at) -> int64_t {
    const int blk = at / p.map.page_size, pg = page_of(p.map, b, blk);
    if (pg < 0) {
      record_status(SN_ERR_INVALID_ARGUMENT);
      return -1;
    }
    return pg * p.page_bytes + static_cast<int64_t>(at - blk * p.map.page_size) * p.row_bytes;
  };
  const int wid = warp * C + rank, warps = kEvictWarps * C;

  // ---- movers into holes ----
  int hole_at[kEvictCluster + 1], mover_at[kEvictCluster + 1];  // the CTAs' first places in the lists
  hole_at[0] = mover_at[0] = 0;
#pragma unroll
  for (int r = 0; r < kEvictCluster; ++r) {
    hole_at[r + 1] = hole_at[r] + (r < C ? static_cast<int>(peer_u32(&s_count[0], r)) : 0);
    mover_at[r + 1] = mover_at[r] + (r < C ? static_cast<int>(peer_u32(&s_count[1], r)) : 0);
  }
  const int pairs = min(hole_at[kEvictCluster], mover_at[kEvictCluster]);  // they are equal
  const int batch = min(32, (pairs + warps - 1) / warps);
  for (int first = wid * batch; first < pairs; first += warps * batch) {
    const int cnt = min(batch, pairs - first);
    int64_t from = -1, to = -1;
    if (lane < cnt) {
      const int i = first + lane;
      int rh = 0, rm = 0, oh = 0, om = 0;
#pragma unroll
      for (int r = 1; r < kEvictCluster; ++r) {
        if (i >= hole_at[r]) rh = r, oh = hole_at[r];
        if (i >= mover_at[r]) rm = r, om = mover_at[r];
      }
      const int hole = static_cast<int>(peer_u32(s_keys + (i - oh), rh));
      const int mover = static_cast<int>(peer_u32(s_keys + (p.part - 1 - (i - om)), rm));
      from = place(mover);
      to = place(hole);
      mass[hole] = mass[mover];
      if (source) source[hole] = mover;
      if (from < 0) to = -1;
    }
    const int units = cnt * nu;
    for (int u0 = 0; u0 < units; u0 += 32 * U) {
      T v[U];
      int64_t dst[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = u0 + 32 * j + lane, at = min(u / nu, cnt - 1), e = u - at * nu;
        const int64_t off = (e >= nu / 2 ? p.kv_bytes - static_cast<int64_t>(nu / 2) * sizeof(T) : 0) + static_cast<int64_t>(e) * sizeof(T);
        const int64_t f = __shfl_sync(0xffffffffu, from, at);
        dst[j] = __shfl_sync(0xffffffffu, to, at);
        if (u >= units) dst[j] = -1;
        if (dst[j] >= 0) {
          v[j] = *reinterpret_cast<const T*>(base + f + off);
          dst[j] += off;
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (dst[j] >= 0) *reinterpret_cast<T*>(base + dst[j]) = v[j];
    }
  }
  cluster_bar(C);  // the movers have left, the lists are done with

  // ---- the recent positions, one after another: n - recent + k -> edge + k ----
  const bool overlap = n - keep < recent;
  const int per = min(32, max(1, 32 * U / nu)), round = per * warps;  // rows a warp (one a lane to look up), and all, take at once
  for (int u0 = 0; u0 < nu; u0 += 32 * U) {  // (a part of the row, where a warp cannot hold a whole one)
    for (int k0 = 0; k0 < recent; k0 += round) {
      const int mine = k0 + wid * per, cnt = min(max(recent - mine, 0), per), k = mine + lane;
      int64_t from = -1, to = -1;
      float w = 0.f;
      if (lane < cnt) {
        from = place(n - recent + k);
        to = place(edge + k);
        w = mass[n - recent + k];
        if (from < 0) to = -1;
      }
      const int units = min(cnt * nu, u0 + 32 * U);
      T v[U];
      int64_t dst[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = u0 + 32 * j + lane, at = min(u / nu, max(cnt - 1, 0)), e = u - at * nu;
        const int64_t off = (e >= nu / 2 ? p.kv_bytes - static_cast<int64_t>(nu / 2) * sizeof(T) : 0) + static_cast<int64_t>(e) * sizeof(T);
        const int64_t f = __shfl_sync(0xffffffffu, from, at);
        dst[j] = __shfl_sync(0xffffffffu, to, at);
        if (u >= units) dst[j] = -1;
        if (dst[j] >= 0) {
          v[j] = *reinterpret_cast<const T*>(base + f + off);
          dst[j] += off;
        }
      }
      if (overlap) cluster_bar(C);
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (dst[j] >= 0) *reinterpret_cast<T*>(base + dst[j]) = v[j];
      if (lane < cnt && u0 == 0) {
        mass[edge + k] = w;
        if (source) source[edge + k] = n - recent + k;
      }
    }
  }
  cluster_bar(C);
  for (int i = keep + rank * kEvictThreads + tid; i < n; i += C * kEvictThreads) mass[i] = 0.f;
}

constexpr int kPartMost = 49152;  // candidates a CTA holds (200 KB)

template <typename T, int NU>
int launch_evict(int rows, int C, cudaStream_t st, const EvictParams& p) {
  const size_t smem = (static_cast<size_t>(p.part) + (p.part + 31) / 32) * sizeof(uint32_t);
  if (!smem_room<evict_kernel<T, NU>>((kPartMost + kPartMost / 32) * 4)) return SN_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * C);
  cfg.blockDim = dim3(kEvictThreads);
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
  if (cudaLaunchKernelEx(&cfg, evict_kernel<T, NU>, p) != cudaSuccess) {
    cudaGetLastError();
    return SN_ERR_LAUNCH;
  }
  return SN_OK;
}

}  // namespace

int tu_status_evict(bool reset, cudaStream_t st, int* out) { return read_tu_status(reset, st, out); }

}  // namespace sn

extern "C" int sn_evict_positions(void* pool, int layers, int num_pages, int page_size, int nheads_kv, int head_dim,
                                  const int* page_table, int64_t table_stride, int max_pages, const int* seq_lens,
                                  float* mass, int64_t mass_layer_stride, int64_t mass_batch_stride,
                                  int64_t mass_head_stride, int batch, int keep, int recent, int sinks, int* source,
                                  void* stream) {
  if (!pool || !page_table || !seq_lens || !mass || layers < 1 || num_pages < 1 || page_size < 1 || nheads_kv < 1 ||
      head_dim < 1 || max_pages < 1 || table_stride < max_pages || batch < 1 || keep < 1 || recent < 0 || sinks < 0 ||
      recent > keep || sinks > keep - recent)
    return SN_ERR_INVALID_ARGUMENT;
  const int64_t room = static_cast<int64_t>(max_pages) * page_size;
  if ((nheads_kv > 1 && mass_head_stride < room) || (batch > 1 && mass_batch_stride < room) ||
      (layers > 1 && mass_layer_stride < room))
    return SN_ERR_INVALID_ARGUMENT;
  const int64_t rows = static_cast<int64_t>(layers) * batch * nheads_kv;
  if (rows > INT32_MAX / sn::kEvictCluster || head_dim > 8192 ||
      room > static_cast<int64_t>(sn::kEvictCluster) * (sn::kPartMost - 4))
    return SN_ERR_UNSUPPORTED;
  sn::EvictParams p;
  p.pool = static_cast<char*>(pool);
  p.row_bytes = 2 * head_dim;
  p.head_bytes = static_cast<int64_t>(page_size) * p.row_bytes;
  p.page_bytes = nheads_kv * p.head_bytes;
  p.kv_bytes = num_pages * p.page_bytes;
  p.layer_bytes = 2 * p.kv_bytes;
  p.map = {page_table, table_stride, max_pages, num_pages, page_size};
  p.seq_lens = seq_lens;
  p.mass = mass;
  p.ml = mass_layer_stride;
  p.mb = mass_batch_stride;
  p.mh = mass_head_stride;
  p.source = source;
  p.batch = batch;
  p.hkv = nheads_kv;
  p.keep = keep;
  p.recent = recent;
  p.sinks = sinks;
  // CTAs a row: as many as the shared memory asks for, and more where there are few long rows
  int C = 1;
  while (C < sn::kEvictCluster && (room > static_cast<int64_t>(C) * (sn::kPartMost - 4) ||
                                  (rows * C < 2 * sn::sm_count() && room > 1024 * C)))
    C *= 2;
  p.part = static_cast<int>((room + C - 1) / C + 4);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int r = static_cast<int>(rows);
  if (sn::aligned16(pool) && p.row_bytes % 16 == 0) {
    if (head_dim == 128) return sn::launch_evict<uint4, 32>(r, C, st, p);
    if (head_dim == 64) return sn::launch_evict<uint4, 16>(r, C, st, p);
    return sn::launch_evict<uint4, 0>(r, C, st, p);
  }
  return sn::launch_evict<uint16_t, 0>(r, C, st, p);
}
