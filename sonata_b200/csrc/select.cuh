// Choice of the highest of a row's keys by one CTA; among equal keys the first
// ones of the row are chosen.
#pragma once

#include "common.cuh"

namespace sn {
namespace {

// Keys whose order as unsigned numbers is that of the values: NaN above all, both zeros alike.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v), size = u & 0x7fffffffu;
  const uint32_t key = static_cast<int>(u) < 0 && size != 0 ? ~u : size | 0x80000000u;
  return size > 0x7f800000u ? 0xffffffffu : key;
}
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return ~0ull;
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v == 0. ? 0. : v));
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ float order_value(uint32_t key) { return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key); }

template <int T>  // threads of the CTA
struct SelectShared {
  static constexpr int kWarps = T / 32, kBits = T > 512 ? 12 : 11, kBins = 1 << kBits;
  static constexpr int kQuads = kBins / (4 * T);  // each thread has kQuads times four neighbouring bins
  static_assert(kQuads * 4 * T == kBins);
  uint4 hist[kBins / 4];
  uint32_t warp[kWarps], warp2[kWarps];
  uint32_t digit, above, here;

  __device__ __forceinline__ uint32_t* bins() { return reinterpret_cast<uint32_t*>(hist); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int q = 0; q < kQuads; ++q) hist[kQuads * threadIdx.x + q] = make_uint4(0, 0, 0, 0);
  }
};

// The bin in which the need-th highest of all keys lies: to s.digit, with the number of keys in higher bins to s.above and
// that in it to s.here.  All threads; the histogram is complete (a barrier before), the results are there when it returns.
template <int T>
__device__ void find_bin(uint32_t need, SelectShared<T>& s) {
  constexpr int Q = SelectShared<T>::kQuads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint4 t[Q];
  uint32_t mine = 0;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    t[q] = s.hist[Q * tid + q];
    mine += t[q].x + t[q].y + t[q].z + t[q].w;
  }
  uint32_t upto = mine;  // keys in this thread's bins and those of the threads after it
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_down_sync(0xffffffffu, upto, o);
    if (lane + o < 32) upto += v;
  }
  if (lane == 0) s.warp[warp] = upto;
  __syncthreads();
  uint32_t after = lane < SelectShared<T>::kWarps && lane > warp ? s.warp[lane] : 0;
  upto += __reduce_add_sync(0xffffffffu, after);
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

// A key is chosen when its bits from `shift` up are above `prefix`, or equal to it and fewer than `need` keys with such bits
// lie before it in the row.
template <typename K>
struct Cutoff {
  K prefix;
  int shift;
  uint32_t need;
};

// The `need` highest (at least 1, at most all) of `len` keys, key(i) the i-th: a radix descent by histograms, which
// ends when all keys with the bits so far are needed.  All threads.
template <typename K, int T, typename F>
__device__ Cutoff<K> find_cutoff(F key, int len, uint32_t need, SelectShared<T>& s) {
  int top = 8 * sizeof(K);
  K prefix = 0;
  while (true) {
    __syncthreads();  // s has been read
    s.clear();
    __syncthreads();
    constexpr int kBits = SelectShared<T>::kBits;
    const int low = top > kBits ? top - kBits : 0, width = top - low;
    const uint32_t mask = (1u << width) - 1;
    for (int i = threadIdx.x; i < len; i += T) {
      const K k = key(i);
      if (top == 8 * sizeof(K) || (k >> top) == prefix) atomicAdd(s.bins() + (static_cast<uint32_t>(k >> low) & mask), 1u);
    }
    __syncthreads();
    find_bin(need, s);
    need -= s.above;
    prefix = static_cast<K>(top == 8 * sizeof(K) ? 0 : prefix << width) | s.digit;
    top = low;
    if (s.here == need || low == 0) return {prefix, low, need};
  }
}

// One bit a key, chosen or not, in bits[0 .. (len + 31) / 32): a warp takes consecutive words.  All threads call it, with a
// barrier after it before the bits are read.
template <typename K, int T, typename F>
__device__ void choose(F key, int len, const Cutoff<K>& cut, uint32_t* bits, SelectShared<T>& s) {
  constexpr int kWarps = SelectShared<T>::kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int words = (len + 31) / 32, per = (words + kWarps - 1) / kWarps;
  const int w0 = min(warp * per, words), w1 = min(w0 + per, words);
  auto at = [&](int w) { return 32 * w + lane < len ? key(32 * w + lane) >> cut.shift : K(0); };
  auto equal = [&](int w, K k) { return __ballot_sync(0xffffffffu, 32 * w + lane < len && k == cut.prefix); };
  uint32_t rank = 0;
  for (int w = w0; w < w1; ++w) rank += __popc(equal(w, at(w)));
  if (lane == 0) s.warp2[warp] = rank;
  __syncthreads();
  rank = 0;
  for (int v = 0; v < warp; ++v) rank += s.warp2[v];
  for (int w = w0; w < w1; ++w) {
    const K k = at(w);
    const uint32_t eq = equal(w, k);
    const bool in = k > cut.prefix || ((eq >> lane & 1) && rank + __popc(eq & ((1u << lane) - 1)) < cut.need);
    const uint32_t word = __ballot_sync(0xffffffffu, 32 * w + lane < len && in);
    if (lane == 0) bits[w] = word;
    rank += __popc(eq);
  }
}

}  // namespace
}  // namespace sn
