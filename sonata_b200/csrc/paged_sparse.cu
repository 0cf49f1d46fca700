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
// Bound by the chain length - table - keys: 48 streams' last pages 3.5 us, 12288
// new tokens of prompts (12.6 MB of keys) 5.3.
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
  return max(p.cu[b], 0) / p.map.page_size + 2 * static_cast<int64_t>(b);
}

// Work items: (touched page, head).
__device__ __forceinline__ int64_t bounds_items(const BoundsParams& p) { return (p.cu ? first_slot(p, p.batch) : p.batch) * p.hkv; }

// The page of work item `slot` and the keys that count in it, or -1; a warp.
__device__ __forceinline__ int touched(const BoundsParams& p, int64_t slot, int& rows) {
  int b, block;
  if (!p.cu) {
    b = static_cast<int>(slot);
    const int n = length_of(p.map, p.seq_lens, b);
    if (n < 1) return -1;
    block = (n - 1) / p.map.page_size;
    rows = n - block * p.map.page_size;
  } else {
    // the last stream that begins at or before the slot, 32 of them looked at at a time
    const int lane = threadIdx.x & 31;
    b = -1;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int some = __popc(__ballot_sync(0xffffffffu, b0 + lane < p.batch && first_slot(p, min(b0 + lane, p.batch - 1)) <= slot));
      b += some;
      if (some < 32) break;
    }
    if (b < 0) return -1;
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
      for (unsigned r0 = group; r0 < rows; r0 += 8 * groups) {  // eight loads in flight, the last row's again past the end
        uint4 k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = *reinterpret_cast<const uint4*>(src + min(r0 + j * groups, rows - 1u) * p.ks.tok);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          lo.x = min2(lo.x, k[j].x), lo.y = min2(lo.y, k[j].y), lo.z = min2(lo.z, k[j].z), lo.w = min2(lo.w, k[j].w);
          hi.x = max2(hi.x, k[j].x), hi.y = max2(hi.y, k[j].y), hi.z = max2(hi.z, k[j].z), hi.w = max2(hi.w, k[j].w);
        }
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
// the greatest over the head's query heads of
//   sum_d max(q_d least_d, q_d greatest_d) = sum_d min(q_d, 0) least_d + max(q_d, 0) greatest_d;
// the first `first` and last `last` blocks and the highest scores of the others
// are listed in ascending order, -1 behind.  The products of two bf16 values are
// exact, and scores are compared as their sums in 64 bits, which are added in
// one order wherever it is done (elements d mod 32 by rising d, then these 32 in
// pairs of neighbours): where terms span more than 53 bits and a sum rounds, the
// choice still does not depend on which step compares a block.  A block with a
// bound that is not finite ranks above all, and so do all blocks for a head with
// a query that is not.
//
// Sums of all blocks in 64 bits would be bound by the conversions and by shared
// memory (3 streams of up to 100001 positions, pages of 16: 66 us where reading
// the bounds takes 5), and all but a few of the blocks do not need them:
// * The tensor cores give every sum in 32 bits, s, and the sum of its terms'
//   absolute values, at most S over a row's blocks.  |s - score| < E = 2^-13 S +
//   2^-110: 256 terms at most go in by 16, each such sum of 17 is off by less
//   than 17 units in the 22nd bit of its largest term, 272 2^-22 S in all; and
//   products under 2^-126 may count as 0.
// * One histogram of s over their range finds the bin of the last one that would
//   be chosen.  Blocks whose s is more than 2 E above that bin are chosen, more
//   than 2 E below it are not: their scores lie on the same side of the last
//   chosen one's.  The few between get their sums in 64 bits and are ranked, by
//   comparing all of them.  (A sum's rounding in 64 bits, 2^-46 S at most, is
//   far within what is left of E.)
// * A block whose absolute sum is not finite has no s to go by: such blocks are
//   always among those between, and the bin above which blocks are chosen for
//   certain is the one that would be if they all were.
// Two launches: scores, spread evenly over the device and bound by reading the
// bounds, and choices, a CTA a row, bound by the chain of its steps.  In one
// launch, a cluster of 8 CTAs a row with the scores in shared memory, exchanges
// of a few kilobytes between the CTAs took 2 to 3 us each (22 us for the three
// streams; now 15.4, about 7 of them the scores of 31 MB of bounds, and 14.6 for
// 48 streams of up to 8000 positions).
// ---------------------------------------------------------------------------
constexpr int kFewExact = 64;        // blocks that are ranked by comparing all of them
constexpr int kChooseMost = 262144;  // blocks of a stream: three bits each in shared memory

struct SelectParams {
  const __nv_bfloat16* q;
  int64_t qb, qh;
  const __nv_bfloat16* bounds;
  PageMap map;
  const int* seq_lens;
  int* blocks;      // [batch, hkv, count]
  uint2* scores;    // [batch, hkv, max_pages]: key of s (kOddKey: none; 0: no page), sum of absolute values; of the blocks that
                    // are not first or last
  uint64_t* exact;  // the same blocks' keys of sums in 64 bits, where they are needed
  int batch, hq, hkv, hd, count, first, last;
};

constexpr uint32_t kOddKey = 0xffffffffu;

// Blocks of a stream, and those that are compared: first .. first + compared - 1.
__device__ __forceinline__ int stream_blocks(const SelectParams& p, int b, int& compared) {
  const int64_t n = length_of(p.map, p.seq_lens, b);
  const int nb = static_cast<int>((n + p.map.page_size - 1) / p.map.page_size);
  compared = nb <= p.count || p.first + p.last == p.count ? 0 : nb - p.first - p.last;
  return nb;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Scores in 32 bits.  A warp takes 16 blocks at a time, their bounds straight from memory as operands: the contraction index
// may be permuted as long as both sides agree, so lane (g, t) takes the 16-byte chunks t, t + 4, ... of blocks g and g + 8,
// and of query head g.  (Brought to a ring in shared memory by bulk copies, two tiles in flight: 48 ragged streams 16.5 us for
// 14.5, the three long ones 17.7 for 16.4.)  blockIdx.y is the row, blockIdx.x takes groups of 64 blocks, gridDim.x of them apart.
template <int HD>
__global__ void __launch_bounds__(128, 4) block_scores_kernel(const SelectParams p) {
  constexpr int KC = HD / 32;  // chunks a lane takes of a row
  pdl_wait();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  for (int row = blockIdx.y; row < p.batch * p.hkv; row += gridDim.y) {
    const int b = row / p.hkv, hk = row - b * p.hkv, group = p.hq / p.hkv;
    uint2* const out = p.scores + static_cast<int64_t>(row) * p.map.max_pages;
    const int start = blockIdx.x * 64 + (threadIdx.x >> 5) * 16, stride = gridDim.x * 64;
    auto page = [&](int i) { return page_of(p.map, b, p.first + i); };  // of the table's entries past the stream's end, too
    for (int h0 = 0; h0 < group; h0 += 8) {
      int i = start;
      int pg0 = page(i + g), pg1 = page(i + g + 8);
      int len;
      stream_blocks(p, b, len);
      uint4 qn[KC], qp[KC];  // the negative and the positive part of head g
      const __nv_bfloat16* q = p.q + b * p.qb + static_cast<int64_t>(hk * group + h0 + g) * p.qh;
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (h0 + g < group) {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(q + 8 * (t + 4 * k));
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = e[2 * j] | static_cast<uint32_t>(e[2 * j + 1]) << 16;
        }
        qn[k] = make_uint4(min2(w[0], 0), min2(w[1], 0), min2(w[2], 0), min2(w[3], 0));
        qp[k] = make_uint4(max2(w[0], 0), max2(w[1], 0), max2(w[2], 0), max2(w[3], 0));
      }
      for (; i < len; i += stride) {
        const __nv_bfloat16* r0 = p.bounds + (static_cast<int64_t>(max(pg0, 0)) * p.hkv + hk) * 2 * HD + 8 * t;
        const __nv_bfloat16* r1 = p.bounds + (static_cast<int64_t>(max(pg1, 0)) * p.hkv + hk) * 2 * HD + 8 * t;
        uint4 a0[2 * KC], a1[2 * KC];  // chunks of the least and of the greatest keys
#pragma unroll
        for (int k = 0; k < 2 * KC; ++k) {
          a0[k] = *reinterpret_cast<const uint4*>(r0 + 32 * k);
          a1[k] = *reinterpret_cast<const uint4*>(r1 + 32 * k);
        }
        const bool ok0 = pg0 >= 0, ok1 = pg1 >= 0;
        if ((i + g < len && !ok0) || (i + g + 8 < len && !ok1)) record_status(SN_ERR_INVALID_ARGUMENT);
        pg0 = page(i + stride + g);
        pg1 = page(i + stride + g + 8);
        float s[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f};
        constexpr uint32_t kAbs = 0x7fff7fffu;
#pragma unroll
        for (int k = 0; k < 2 * KC; ++k) {
          const uint4 q4 = k < KC ? qn[k % KC] : qp[k % KC], x = a0[k], y = a1[k];
          mma_bf16(s, x.x, y.x, x.y, y.y, q4.x, q4.y);
          mma_bf16(s, x.z, y.z, x.w, y.w, q4.z, q4.w);
          mma_bf16(m, x.x & kAbs, y.x & kAbs, x.y & kAbs, y.y & kAbs, q4.x & kAbs, q4.y & kAbs);
          mma_bf16(m, x.z & kAbs, y.z & kAbs, x.w & kAbs, y.w & kAbs, q4.z & kAbs, q4.w & kAbs);
        }
        // heads 2t and 2t + 1 of blocks g and g + 8; an absolute sum that is not a number is infinite
        const bool two = h0 + 2 * t + 1 < group, one = h0 + 2 * t < group;
        auto wide = [](float x) { return x < INFINITY ? x : INFINITY; };
        float v0 = one ? s[0] : -INFINITY, v1 = one ? s[2] : -INFINITY;
        float m0 = fmaxf(wide(m[0]), wide(m[1])), m1 = fmaxf(wide(m[2]), wide(m[3]));
        if (two) v0 = fmaxf(v0, s[1]), v1 = fmaxf(v1, s[3]);
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
          v0 = fmaxf(v0, __shfl_xor_sync(0xffffffffu, v0, o));
          v1 = fmaxf(v1, __shfl_xor_sync(0xffffffffu, v1, o));
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        const int at = i + g + 8 * t;
        if (t < 2 && at < len) {
          uint2 v = make_uint2(0, 0);
          if (t ? ok1 : ok0) {
            const float wide_sum = t ? m1 : m0;
            v = wide_sum < INFINITY ? make_uint2(order_key(t ? v1 : v0), __float_as_uint(wide_sum)) : make_uint2(kOddKey, 0);
          }
          if (h0 > 0) {
            const uint2 before = out[at];  // this lane's own
            v = make_uint2(max(v.x, before.x), max(v.y, before.y));
          }
          out[at] = v;
        }
      }
    }
  }
  pdl_launch_dependents();  // not before: a CTA of the choice takes half an SM or all of it (3 long streams 17.4 -> 17.1 us)
}

// The key of one block's score in 64 bits; a warp, lane l the elements l mod 32.
__device__ __forceinline__ uint64_t exact_score(const SelectParams& p, int b, int hk, int block) {
  const int lane = threadIdx.x & 31, group = p.hq / p.hkv;
  const int pg = page_of(p.map, b, block);
  if (pg < 0) return 0;
  const __nv_bfloat16* lo = p.bounds + (static_cast<int64_t>(pg) * p.hkv + hk) * 2 * p.hd;
  const __nv_bfloat16* q = p.q + b * p.qb + static_cast<int64_t>(hk) * group * p.qh;
  uint64_t best = 0;
  bool odd = false;
  for (int h0 = 0; h0 < group; h0 += 4) {  // four heads at a time: a chain of loads and shuffles each
    double sum[4] = {0., 0., 0., 0.};
#pragma unroll 4
    for (int d = lane; d < p.hd; d += 32) {
      const float l = __bfloat162float(lo[d]), g = __bfloat162float(lo[p.hd + d]);
      odd |= !(fabsf(l) < INFINITY) || !(fabsf(g) < INFINITY);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float v = __bfloat162float(q[min(h0 + h, group - 1) * p.qh + d]);
        sum[h] = fma(static_cast<double>(v), static_cast<double>(v < 0.f ? l : g), sum[h]);
      }
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
      for (int h = 0; h < 4; ++h) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      best = max(best, order_key(sum[h]));
      odd |= !(fabs(sum[h]) < INFINITY);  // of finite values none comes near
    }
  }
  return __any_sync(0xffffffffu, odd) ? ~0ull : best;
}

// The keys of scores in 64 bits of blocks first + at[k], k < many, to keys[k]: for many of them, a warp eight blocks, four lanes a
// block, kHeads query heads at a time; head_dim 64 or 128, bounds on 16 bytes, all threads.  A bf16 value's bits moved into the
// upper word of a double are that value times 2^-896, subnormal ones too, so that no conversions (16 a cycle and SM) bind; with q
// times 2^1023 more, which leaves the order as it is, the products, multiples of 2^-266 times 2^-769, are held exactly, and
// no sum of them needs a bit below what a double has.  Added in exact_score's order: lane t has the elements 8 t .. 8 t + 7 mod 32.
// Out of line, as are the few other steps that most calls do not take: what is taken runs once a CTA, and waits for its
// instructions (16 -> 19 us with all of it inline).  6251 equal blocks of a row: 303 us; 512 rows of 500: 100; 2048 rows 538, two heads
// at a time, as four would spill where a thread has 64 registers (835).
template <int T, int kHeads>
__device__ __noinline__ void exact_scores(const SelectParams& p, int b, int hk, const int* at, uint32_t many, uint64_t* keys,
                                          SelectShared<T>& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & 3, group = p.hq / p.hkv;
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q + b * p.qb + static_cast<int64_t>(hk) * group * p.qh);
  double* const s_q = reinterpret_cast<double*>(s.hist);  // [kHeads][hd], over the histogram, which is done with
  static_assert(sizeof(s.hist) >= kHeads * 128 * sizeof(double));
  auto widen = [](uint32_t u) { return __hiloint2double(static_cast<int>((u & 0x8000u) << 16 | (u & 0x7fffu) << 13), 0); };
  auto odd_bits = [](uint32_t u) { return (u & 0x7f80u) == 0x7f80u; };
  for (int h0 = 0; h0 < group; h0 += kHeads) {
    bool odd_query = false;  // its widened bits would pass for numbers
    __syncthreads();         // the histogram, or the last heads' queries, have been read
    for (int i = threadIdx.x; i < kHeads * p.hd; i += T) {
      const uint32_t v = q[min(h0 + i / p.hd, group - 1) * p.qh + i % p.hd];
      s_q[i] = widen(v) * 0x1p1023;
      odd_query |= odd_bits(v);
    }
    odd_query = __syncthreads_or(odd_query);
    for (uint32_t i = 8 * warp; i < many; i += 8 * (T / 32)) {
      const uint32_t k = i + lane / 4;
      const int pg = k < many ? page_of(p.map, b, p.first + at[k]) : -1;
      const __nv_bfloat16* lo = p.bounds + (static_cast<int64_t>(max(pg, 0)) * p.hkv + hk) * 2 * p.hd;
      double sum[kHeads][8] = {};
      bool odd = odd_query;
      for (int c = 8 * t; c < p.hd; c += 32) {
        uint32_t l[4], g[4];
        *reinterpret_cast<uint4*>(l) = *reinterpret_cast<const uint4*>(lo + c);
        *reinterpret_cast<uint4*>(g) = *reinterpret_cast<const uint4*>(lo + p.hd + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t wl = j & 1 ? l[j / 2] >> 16 : l[j / 2] & 0xffffu, wg = j & 1 ? g[j / 2] >> 16 : g[j / 2] & 0xffffu;
          odd |= odd_bits(wl) || odd_bits(wg);
          const double least = widen(wl), greatest = widen(wg);
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            const double v = s_q[h * p.hd + c + j];
            sum[h][j] = fma(v, __double2hiint(v) < 0 ? least : greatest, sum[h][j]);
          }
        }
      }
      uint64_t best = 0;
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const double* x = sum[h];
        double all = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        all += __shfl_xor_sync(0xffffffffu, all, 1);
        all += __shfl_xor_sync(0xffffffffu, all, 2);
        best = max(best, order_key(all));
      }
      if (__ballot_sync(0xffffffffu, odd) >> (lane & 28) & 15) best = ~0ull;
      if (pg < 0) best = 0;
      if (t == 0 && k < many) keys[k] = h0 > 0 ? max(best, keys[k]) : best;
    }
  }
}

// Scores in 64 bits of all blocks, a warp a block: any head_dim and alignment.
__global__ void __launch_bounds__(128) exact_scores_kernel(const SelectParams p) {
  pdl_launch_dependents();
  pdl_wait();
  for (int row = blockIdx.y; row < p.batch * p.hkv; row += gridDim.y) {
    const int b = row / p.hkv, hk = row - b * p.hkv;
    int len;
    stream_blocks(p, b, len);
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 5); i < len; i += gridDim.x * 4) {
      const uint64_t key = exact_score(p, b, hk, p.first + i);
      if ((threadIdx.x & 31) == 0) {
        p.exact[static_cast<int64_t>(row) * p.map.max_pages + i] = key;
        if (page_of(p.map, b, p.first + i) < 0) record_status(SN_ERR_INVALID_ARGUMENT);
      }
    }
  }
}

// The range and number of the scores of a row in which some blocks have none, and the number of those that have a page.
__device__ __noinline__ void regular_range(const uint2* scores, int len, uint32_t* s_range, uint32_t& least, uint32_t& most, uint32_t& scored,
                                           uint32_t& odd) {
  least = 0xffffffffu;
  most = scored = odd = 0;
  for (int i = threadIdx.x; i < len; i += blockDim.x) {
    const uint32_t key = scores[i].x;
    if (key == kOddKey) ++odd;
    if (key == 0 || key == kOddKey) continue;
    ++scored;
    least = min(least, key);
    most = max(most, key);
  }
  __syncthreads();  // s_range has been read
  if (threadIdx.x < 2) s_range[threadIdx.x] = threadIdx.x == 0 ? 0xffffffffu : 0;
  __syncthreads();
  atomicMin(&s_range[0], least);
  atomicMax(&s_range[1], most);
  atomicAdd(&s_range[3], scored);
  atomicAdd(&s_range[4], odd);
  __syncthreads();
  least = s_range[0];
  most = s_range[1];
  scored = s_range[3];
  odd = s_range[4];
}

// Bits of the `need` highest of `len` keys.
template <int T>
__device__ __noinline__ void choose_exact(const uint64_t* keys, int len, uint32_t need, uint32_t* bits, SelectShared<T>& s) {
  auto key = [&](int i) { return keys[i]; };
  const Cutoff<uint64_t> cut = find_cutoff<uint64_t>(key, len, need, s);
  choose(key, len, cut, bits, s);
}

// One CTA a row, kPerSM of them an SM; kScored: block_scores_kernel has run, else exact_scores_kernel.
template <bool kScored, int kChooseThreads, int kPerSM>
__global__ void __launch_bounds__(kChooseThreads, kPerSM) choose_blocks_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kChooseWarps = kChooseThreads / 32, kChooseHeld = kPerSM > 2 ? 4 : 16;  // keys a thread holds
  extern __shared__ uint32_t s_bits[];
  __shared__ SelectShared<kChooseThreads> s_sel;
  __shared__ uint32_t s_range[5];  // least and greatest key, S, and for regular_range
  __shared__ uint64_t s_few[kFewExact];
  __shared__ int s_few_at[kFewExact];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, b = row / p.hkv, hk = row - b * p.hkv;
  if (tid < 5) s_range[tid] = tid == 0 ? 0xffffffffu : 0;
  s_sel.clear();
  pdl_launch_dependents();
  pdl_wait();
  int* const out = p.blocks + static_cast<int64_t>(row) * p.count;
  int len;
  const int nb = stream_blocks(p, b, len), need = p.count - p.first - p.last;
  if (len == 0) {  // all of a short stream's blocks, or none but the first and the last
    for (int i = tid; i < p.count; i += kChooseThreads) out[i] = nb <= p.count ? (i < nb ? i : -1) : i < p.first ? i : nb - p.count + i;
    return;
  }
  for (int i = tid; i < p.first + p.last; i += kChooseThreads) {
    if (i < p.first) out[i] = i;
    else out[p.count - p.last + i - p.first] = nb - p.last + i - p.first;
  }
  uint2* const scores = p.scores + static_cast<int64_t>(row) * p.map.max_pages;
  uint64_t* const exact = p.exact + static_cast<int64_t>(row) * p.map.max_pages;
  const int words = (len + 31) / 32;
  uint32_t* const s_in = s_bits;            // [words] chosen
  uint32_t* const s_open = s_in + words;    // [words] to be compared in 64 bits
  uint32_t* const s_won = s_open + words;   // [words] which of those are chosen, in their order
  const int per = ((words + kChooseWarps - 1) / kChooseWarps + 31) / 32 * 32;
  const int w0 = min(warp * per, words), w1 = min(w0 + per, words);  // the words a warp counts and lists, a lane a word
  // exclusive sums over the lanes, and all of it
  auto scan = [&](uint32_t v, uint32_t& all) {
    uint32_t upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    all = __shfl_sync(0xffffffffu, upto, 31);
    return upto - v;
  };
  if constexpr (kScored) {
    // the keys of words warp, warp + 16, ...: the first of a warp stay in registers, the rest are read again
    uint32_t held[kChooseHeld];
    uint32_t least = 0xffffffffu, most = 0, S = 0;
    auto range = [&](uint2 v) {
      least = min(least, v.x);
      most = max(most, v.x);
      S = max(S, v.y);  // non-negative floats
    };
#pragma unroll
    for (int j = 0; j < kChooseHeld; ++j) {
      const int i = tid + j * kChooseThreads;
      held[j] = 0;
      if (i < len) {
        const uint2 v = scores[i];
        held[j] = v.x;
        range(v);
      }
    }
#pragma unroll 4
    for (int i = tid + kChooseHeld * kChooseThreads; i < len; i += kChooseThreads) range(scores[i]);
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    S = __reduce_max_sync(0xffffffffu, S);
    __syncthreads();
    if (lane == 0) {
      atomicMin(&s_range[0], least);
      atomicMax(&s_range[1], most);
      atomicMax(&s_range[2], S);
    }
    __syncthreads();
    least = s_range[0];
    most = s_range[1];
    uint32_t scored = len, odd = 0;  // blocks that have a score, and that have none
    if (least == 0 || most == kOddKey) regular_range(scores, len, s_range, least, most, scored, odd);
    const bool sure = static_cast<uint32_t>(need) <= scored;  // else all blocks with a score may be needed
    const uint32_t span = most - least;
    const int shift = max(0, 32 - __clz(span) - SelectShared<kChooseThreads>::kBits);
    auto count = [&](uint32_t key) {
      if (key - least <= span) atomicAdd(s_sel.bins() + ((key - least) >> shift), 1u);  // one with a score
    };
#pragma unroll
    for (int j = 0; j < kChooseHeld; ++j) count(held[j]);
#pragma unroll 4
    for (int i = tid + kChooseHeld * kChooseThreads; i < len; i += kChooseThreads) count(scores[i].x);
    __syncthreads();
    const float E2 = fmaf(__uint_as_float(s_range[2]), 0x1p-12f, 0x1p-109f);  // 2 E
    float lo = 0.f, hi = INFINITY;
    for (uint32_t want = sure ? need : 0; want > 0;) {
      find_bin(want, s_sel);
      const uint32_t first_key = least + (s_sel.digit << shift);
      if (want == static_cast<uint32_t>(need)) lo = order_value(first_key) - E2;
      if (want + odd == static_cast<uint32_t>(need)) hi = order_value(min(first_key + ((1u << shift) - 1), most)) + E2;
      want = want == static_cast<uint32_t>(need) && odd > 0 && want > odd ? want - odd : 0;
      if (want > 0) __syncthreads();  // the digit has been read
    }
    uint32_t nin = 0, nopen = 0;
    auto sort_word = [&](int i, uint32_t key) {  // of the warp's lanes' blocks i
      if (i - lane >= len) return;
      const float v = order_value(key);  // without a score, a NaN
      const uint32_t in = __ballot_sync(0xffffffffu, sure && v > hi);
      const uint32_t open = __ballot_sync(0xffffffffu, (v >= lo && v <= hi) || key == kOddKey || (!sure && i < len));
      if (lane == 0) {
        s_in[i / 32] = in;
        s_open[i / 32] = open;
      }
      nin += __popc(in);
      nopen += __popc(open);
    };
#pragma unroll
    for (int j = 0; j < kChooseHeld; ++j) sort_word(tid + j * kChooseThreads, held[j]);
    for (int i = tid + kChooseHeld * kChooseThreads; i - lane < len; i += kChooseThreads) sort_word(i, i < len ? scores[i].x : 0);
    if (lane == 0) {  // (s_sel.warp of find_bin has been read: that was before its last barrier)
      s_sel.warp[warp] = nin;
      s_sel.warp2[warp] = nopen;
    }
    __syncthreads();
    uint32_t all_in = 0, all_open = 0;
#pragma unroll
    for (int v = 0; v < kChooseWarps; ++v) {
      all_in += s_sel.warp[v];
      all_open += s_sel.warp2[v];
    }
    const uint32_t wanted = static_cast<uint32_t>(need) - all_in;
    if (all_open != wanted) {
      // the open blocks in their order, those before this warp's words first
      __syncthreads();  // s_sel.warp2 has been read
      uint32_t mine = 0;
      for (int w = w0 + lane; w < w1; w += 32) mine += __popc(s_open[w]);
      mine = __reduce_add_sync(0xffffffffu, mine);
      if (lane == 0) s_sel.warp2[warp] = mine;
      __syncthreads();
      uint32_t open_at = 0;
#pragma unroll
      for (int v = 0; v < kChooseWarps; ++v) open_at += v < warp ? s_sel.warp2[v] : 0;
      // a list of them, a lane a word, so that every warp takes as many of them; a long one over the scores, which are done with
      const bool few = all_open <= kFewExact;
      int* const at = few ? s_few_at : reinterpret_cast<int*>(scores);
      for (int w = w0; w < w1; w += 32) {
        uint32_t left = w + lane < w1 ? s_open[w + lane] : 0, all;
        for (uint32_t k = open_at + scan(__popc(left), all); left; left &= left - 1, ++k) at[k] = 32 * (w + lane) + __ffs(left) - 1;
        open_at += all;
      }
      __syncthreads();
      if (few) {
        for (uint32_t i = warp; i < all_open; i += kChooseWarps) {
          const uint64_t key = exact_score(p, b, hk, p.first + at[i]);
          if (lane == 0) s_few[i] = key;
        }
        __syncthreads();
        if (tid < all_open) {
          const uint64_t key = s_few[tid];
          uint32_t better = 0;
          for (uint32_t j = 0; j < all_open; ++j) better += s_few[j] > key || (s_few[j] == key && j < tid);
          if (better >= wanted) atomicAnd(&s_open[at[tid] / 32], ~(1u << (at[tid] & 31)));
        }
      } else {
        exact_scores<kChooseThreads, (kPerSM > 2 ? 2 : 4)>(p, b, hk, at, all_open, exact, s_sel);
        __syncthreads();
        choose_exact(exact, static_cast<int>(all_open), wanted, s_won, s_sel);
        __syncthreads();
        for (uint32_t i = tid; i < all_open; i += kChooseThreads)
          if (!(s_won[i / 32] >> (i % 32) & 1)) atomicAnd(&s_open[at[i] / 32], ~(1u << (at[i] & 31)));
      }
      __syncthreads();
    }
  } else {
    choose_exact(exact, len, static_cast<uint32_t>(need), s_in, s_sel);
    for (int w = tid; w < words; w += kChooseThreads) s_open[w] = 0;
    __syncthreads();
  }
  // ---- the list, in ascending order ----
  uint32_t mine = 0;
  for (int w = w0 + lane; w < w1; w += 32) mine += __popc(s_in[w] | s_open[w]);
  mine = __reduce_add_sync(0xffffffffu, mine);
  __syncthreads();  // s_sel.warp has been read
  if (lane == 0) s_sel.warp[warp] = mine;
  __syncthreads();
  uint32_t at = p.first;
#pragma unroll
  for (int v = 0; v < kChooseWarps; ++v) at += v < warp ? s_sel.warp[v] : 0;
  for (int w = w0; w < w1; w += 32) {
    uint32_t left = w + lane < w1 ? s_in[w + lane] | s_open[w + lane] : 0, all;
    for (uint32_t k = at + scan(__popc(left), all); left; left &= left - 1, ++k) out[k] = p.first + 32 * (w + lane) + __ffs(left) - 1;
    at += all;
  }
}

template <bool kScored, int T, int kPerSM>
int launch_choose(int rows, size_t smem, cudaStream_t st, const SelectParams& p) {
  if (!smem_room<choose_blocks_kernel<kScored, T, kPerSM>>(kChooseMost / 32 * 3 * sizeof(uint32_t))) return SN_ERR_LAUNCH;
  return launch(choose_blocks_kernel<kScored, T, kPerSM>, dim3(static_cast<unsigned>(rows)), dim3(T), smem, st, true, p);
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

size_t sn_select_blocks_workspace_size(int batch, int nheads_kv, int max_pages) {
  if (batch < 1 || nheads_kv < 1 || max_pages < 1) return 0;
  return static_cast<size_t>(batch) * nheads_kv * max_pages * (sizeof(uint64_t) + sizeof(uint2));
}

int sn_select_blocks(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* bounds, int num_pages,
                     int page_size, const int* page_table, int64_t table_stride, int max_pages, const int* seq_lens,
                     int batch, int nheads, int nheads_kv, int head_dim, int count, int first, int last, int* blocks,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !bounds || !page_table || !seq_lens || !blocks || !workspace || num_pages < 1 || page_size < 1 ||
      max_pages < 1 || table_stride < max_pages || batch < 1 || nheads < 1 || nheads_kv < 1 || nheads % nheads_kv != 0 ||
      head_dim < 1 || q_batch_stride < 0 || q_head_stride < 0 || count < 1 || first < 0 || last < 0 || first > count ||
      last > count - first || workspace_bytes < sn_select_blocks_workspace_size(batch, nheads_kv, max_pages))
    return SN_ERR_INVALID_ARGUMENT;
  if (!sn::aligned16(workspace)) return SN_ERR_MISALIGNED;
  const int64_t rows = static_cast<int64_t>(batch) * nheads_kv;
  if (rows > INT32_MAX || max_pages > sn::kChooseMost || static_cast<int64_t>(max_pages) * page_size > INT32_MAX)
    return SN_ERR_UNSUPPORTED;
  sn::SelectParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.qb = q_batch_stride;
  p.qh = q_head_stride;
  p.bounds = static_cast<const __nv_bfloat16*>(bounds);
  p.map = {page_table, table_stride, max_pages, num_pages, page_size};
  p.seq_lens = seq_lens;
  p.blocks = blocks;
  p.exact = static_cast<uint64_t*>(workspace);
  p.scores = reinterpret_cast<uint2*>(p.exact + rows * max_pages);
  p.batch = batch;
  p.hq = nheads;
  p.hkv = nheads_kv;
  p.hd = head_dim;
  p.count = count;
  p.first = first;
  p.last = last;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool scored = sn::aligned16(bounds) && (head_dim == 64 || head_dim == 128);
  const size_t smem = static_cast<size_t>((max_pages + 31) / 32) * 3 * sizeof(uint32_t);
  if (max_pages > count) {  // there may be something to compare
    // as many CTAs a row as the table has blocks for, and over all rows no more than a few for each place on the device:
    // the lengths are on the device
    const int64_t y = std::min<int64_t>(rows, 65535), per_cta = scored ? 64 : 4;
    const int64_t x = std::min<int64_t>((max_pages + per_cta - 1) / per_cta, std::max<int64_t>(1, (scored ? 4 : 16) * sn::sm_count() / y));
    const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y));
    const int rc = !scored         ? sn::launch(sn::exact_scores_kernel, grid, dim3(128), 0, st, true, p)
                   : head_dim == 64 ? sn::launch(sn::block_scores_kernel<64>, grid, dim3(128), 0, st, true, p)
                                    : sn::launch(sn::block_scores_kernel<128>, grid, dim3(128), 0, st, true, p);
    if (rc != SN_OK) return rc;
  }
  // the choice is a chain of steps: more threads a row where there are few rows (3 streams of up to 100001 positions, 12 rows:
  // 256 threads 18.9 us, 512 16.4, 1024 18.7), two CTAs an SM where there are more, and four, with fewer keys in registers,
  // where there are more than two an SM (2048 rows of 500 blocks 136 -> 120, of 125 68 -> 53; 192 rows of 500 18.4 -> 20.5)
  const int r = static_cast<int>(rows);
  if (!scored) return sn::launch_choose<false, 256, 2>(r, smem, st, p);
  return rows <= sn::sm_count()       ? sn::launch_choose<true, 512, 1>(r, smem, st, p)
         : rows <= 2 * sn::sm_count() ? sn::launch_choose<true, 256, 2>(r, smem, st, p)
                                      : sn::launch_choose<true, 256, 4>(r, smem, st, p);
}

}  // extern "C"
