// Choice of the highest keys of a row that is spread over the shared memory
// of a thread-block cluster.  Ranks of the cluster hold consecutive parts of
// the row; among equal keys the first ones of the row are chosen.
//
// A radix descent from the top: a histogram of 11 bits in each CTA, added up
// over the cluster by every CTA for itself through distributed shared memory,
// gives the digit in which the last chosen key lies; keys above it are chosen,
// those in it go on to the next 11 bits, and it ends when all of them are
// needed.  One cluster barrier a pass, two histograms in turn.
#pragma once

#include "common.cuh"

namespace sn {
namespace {

constexpr int kDigitBits = 11, kBins = 1 << kDigitBits;

__device__ __forceinline__ uint32_t ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Barrier over the cluster of C CTAs; orders shared memory of all of them, and global memory.
__device__ __forceinline__ void cluster_bar(int C) {
  if (C == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}
// The word at `local`'s place in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* local, int rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
// The address of `local`'s place in the shared memory of CTA `rank`.
__device__ __forceinline__ uint32_t peer_at(const void* local, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  return a;
}
__device__ __forceinline__ void put_u32(uint32_t at, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void put_u64(uint32_t at, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ uint4 peer_u128(const uint4* local, int rank) {
  uint32_t a;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Keys whose order as unsigned numbers is that of the values: NaN above all, both zeros alike.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return ~0ull;
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v == 0. ? 0. : v));
  return u >> 63 ? ~u : u | (1ull << 63);
}

__device__ __forceinline__ float order_value(uint32_t key) { return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key); }

template <int T>  // threads of a CTA
struct SelectShared {
  static constexpr int kWarps = T / 32, kQuads = kBins / (4 * T);  // each thread has kQuads times four neighbouring bins
  static_assert(kQuads * 4 * T == kBins);
  uint4 hist[2][kBins / 4];
  uint32_t warp[kWarps], warp2[kWarps];
  uint32_t digit, above, here;
};

// A key is chosen when its bits from `shift` up are above `prefix`, or equal to it and fewer than `need` keys with such bits
// lie before it in the row, `before` of them in lower ranks' parts.
template <typename K>
struct Cutoff {
  K prefix;
  int shift;
  uint32_t need, before;
};

// The bin of 4 Q T in which the need-th highest of all the cluster's keys lies: to s.digit, with the number of keys in higher
// bins to s.above and that in it to s.here.  After a cluster barrier, which makes the histograms visible; all threads of all
// CTAs.  A load from a peer takes most of a microsecond, so eight peers' are in flight at once.
template <int Q, int T>
__device__ void find_bin(const uint4* hist, uint32_t need, SelectShared<T>& s, int C, int rank) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint4 t[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) t[q] = hist[Q * tid + q];
  for (int r0 = 1; r0 < C; r0 += 8) {
    uint4 o[8][Q];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r0 + r < C) {
        const int peer = rank + r0 + r < C ? rank + r0 + r : rank + r0 + r - C;
#pragma unroll
        for (int q = 0; q < Q; ++q) o[r][q] = peer_u128(hist + Q * tid + q, peer);
      }
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r0 + r < C) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          t[q].x += o[r][q].x;
          t[q].y += o[r][q].y;
          t[q].z += o[r][q].z;
          t[q].w += o[r][q].w;
        }
      }
  }
  uint32_t mine = 0;
#pragma unroll
  for (int q = 0; q < Q; ++q) mine += t[q].x + t[q].y + t[q].z + t[q].w;
  uint32_t upto = mine;  // keys in this thread's bins and those of the threads after it
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_down_sync(0xffffffffu, upto, o);
    if (lane + o < 32) upto += v;
  }
  if (lane == 0) s.warp[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 1; w < SelectShared<T>::kWarps; ++w)
    if (w > warp) upto += s.warp[w];
  if (upto >= need && upto - mine < need) {  // one thread
    uint32_t above = upto - mine, here = 0;
    int bin = -1;
#pragma unroll
    for (int q = Q - 1; q >= 0; --q) {
      const uint32_t c[4] = {t[q].w, t[q].z, t[q].y, t[q].x};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (bin >= 0) continue;
        if (above + c[j] >= need) {
          bin = 4 * (Q * tid + q) + 3 - j;
          here = c[j];
        } else {
          above += c[j];
        }
      }
    }
    s.digit = bin;
    s.above = above;
    s.here = here;
  }
  __syncthreads();
}

// The `need` highest (at least 1, at most all) of the cluster's keys; `len` of them are this CTA's.  All threads of all CTAs
// call it.
template <int T, typename K>
__device__ Cutoff<K> find_cutoff(const K* keys, int len, uint32_t need, SelectShared<T>& s, int C, int rank) {
  constexpr int Q = SelectShared<T>::kQuads;
  const int tid = threadIdx.x;
  int top = 8 * sizeof(K);
  K prefix = 0;
#pragma unroll
  for (int q = 0; q < Q; ++q) s.hist[0][Q * tid + q] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  for (int pass = 0;; ++pass) {
    uint4* const hist = s.hist[pass & 1];
    uint32_t* const bins = reinterpret_cast<uint32_t*>(hist);
    const int low = top > kDigitBits ? top - kDigitBits : 0, width = top - low;
    const uint32_t mask = (1u << width) - 1;
    for (int i = tid; i < len; i += T) {
      const K k = keys[i];
      if (top == 8 * sizeof(K) || (k >> top) == prefix) atomicAdd(bins + (static_cast<uint32_t>(k >> low) & mask), 1u);
    }
    cluster_bar(C);
#pragma unroll
    for (int q = 0; q < Q; ++q)  // everyone has read it: that was before this pass's barrier
      s.hist[(pass + 1) & 1][Q * tid + q] = make_uint4(0, 0, 0, 0);
    find_bin<Q>(hist, need, s, C, rank);
    const uint32_t digit = s.digit, here = s.here;
    need -= s.above;
    prefix = static_cast<K>(top == 8 * sizeof(K) ? 0 : prefix << width) | digit;
    top = low;
    if (here == need || low == 0) {
      Cutoff<K> cut = {prefix, low, need, 0};
      if (here != need)
        for (int r = 0; r < rank; ++r) cut.before += peer_u32(bins + digit, r);
      return cut;
    }
    // the next pass writes s after its barrier, which every thread of this CTA reaches from here
  }
}

// One bit a key, chosen or not, in bits[0 .. (len + 31) / 32): a warp takes consecutive words.  All threads call it, with a
// barrier after it before the bits are read.
template <int T, typename K>
__device__ void choose(const K* keys, int len, const Cutoff<K>& cut, uint32_t* bits, SelectShared<T>& s) {
  constexpr int kWarps = SelectShared<T>::kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int words = (len + 31) / 32, per = (words + kWarps - 1) / kWarps;
  const int w0 = min(warp * per, words), w1 = min(w0 + per, words);
  auto equal = [&](int w) {
    const int i = 32 * w + lane;
    return __ballot_sync(0xffffffffu, i < len && (keys[i] >> cut.shift) == cut.prefix);
  };
  uint32_t rank = 0;
  for (int w = w0; w < w1; ++w) rank += __popc(equal(w));
  if (lane == 0) s.warp2[warp] = rank;
  __syncthreads();
  rank = cut.before;
  for (int v = 0; v < warp; ++v) rank += s.warp2[v];
  for (int w = w0; w < w1; ++w) {
    const int i = 32 * w + lane;
    const uint32_t eq = equal(w);
    const bool is_eq = (eq >> lane) & 1;
    const bool in = i < len && ((keys[i] >> cut.shift) > cut.prefix || (is_eq && rank + __popc(eq & ((1u << lane) - 1)) < cut.need));
    const uint32_t word = __ballot_sync(0xffffffffu, in);
    if (lane == 0) bits[w] = word;
    rank += __popc(eq);
  }
}

}  // namespace
}  // namespace sn
