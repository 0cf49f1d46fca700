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

// Two launches: the plan of each row (a CTA each: what stays, the lists of holes and movers, mass), bound by the chain of
// its steps (7 us for 2044 candidates, 21 for 29739, of which 4 the load of their masses), and the moves, bound by HBM where
// there are many (172 MB in 33 us, 5.2 TB/s); few are moved with the plan.  12 layers of a stream of 2112 positions cut by 64:
// 13.1 us (15.5 with nothing in L2), of 30011 cut to 4096: 58 us.  In one launch, a cluster a row, either the choice is shared
// out, its histograms exchanged through distributed shared memory (27 us for the former), or the other CTAs of the cluster
// wait for the one that makes it (30 us).
constexpr int kEvictMost = 1 << 19;   // candidates of a stream: two bits each in shared memory
constexpr int kEvictWords = 52992;    // of shared memory for those bits and for keys
constexpr int kEvictCopy = 1024;      // 16-byte pieces of one copy to shared memory
constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;
constexpr int kMoveCluster = 16;      // CTAs a row at most (above 8: not portable, asked for)

struct EvictParams {
  char* pool;  // [layers, 2, num_pages, hkv, page_size] rows of row_bytes, dense
  int64_t layer_bytes, kv_bytes, page_bytes, head_bytes;
  int row_bytes;
  PageMap map;
  const int* seq_lens;
  float* mass;  // [layers, batch, hkv, >= room] by strides
  int64_t ml, mb, mh;
  int* source;  // [layers, batch, hkv, keep] or null
  int2* head;   // [layers, batch, hkv]: n, pairs of a hole and a mover (-1: the rows are moved)
  int* plan;    // [layers, batch, hkv] of plan_ints: holes, movers, and the keys where shared memory does not hold them
  int64_t plan_ints;
  int most;     // pairs of a row at most, a multiple of 4
  int batch, hkv, keep, recent, sinks;
  int held;     // keys in shared memory: all candidates' or none (then they are in the plan)
  int units;    // 16-byte pieces of a position's two rows, 0: rows are not such
};

// Of max_pages * page_size = room positions: the words of shared memory for two bits each, and room to align the keys;
// whether it holds their keys as well; pairs of a hole and a mover at most, and the integers of a row's plan.
int64_t bit_words(int64_t room) { return (room + 31) / 32 * 2 + 8; }
bool keys_held(int64_t room) { return bit_words(room) + room <= kEvictWords; }
int64_t most_pairs(int64_t room, int64_t keep) { return (std::min(room / 2, keep) + 3) / 4 * 4; }
int64_t plan_size(int64_t room, int64_t keep) { return 2 * most_pairs(room, keep) + (keys_held(room) ? 0 : (room + 3) / 4 * 4 + 4); }

// Where a position's K row is in its layer and head, or -1.
__device__ __forceinline__ int64_t place(const EvictParams& p, int b, int at) {
  const int blk = at / p.map.page_size, pg = page_of(p.map, b, blk);
  if (pg < 0) {
    record_status(SN_ERR_INVALID_ARGUMENT);
    return -1;
  }
  return pg * p.page_bytes + static_cast<int64_t>(at - blk * p.map.page_size) * p.row_bytes;
}

// Few rows are moved by the CTA that has planned them, its lists in shared memory, while the other launch finds nothing to do:
// kFewUnits pieces of 16 bytes a thread at once.  A stream's 64 positions over its budget, 64 recent ones (48 rows, masses that
// the calls before have not put in order) 17.0 -> 13.4 us, 152 over it 17.5 -> 16.5; 256, which have more than kFewPieces,
// would take 18.4 where they now take 16.6.
constexpr int kFewMoves = 512, kFewPieces = 8192, kFewUnits = 8;
struct Move { int64_t from, to; };
template <int T>
__device__ __forceinline__ void move_few(const EvictParams& p, int layer, int b, int h, int n, int pairs, const int* list, Move* moves) {
  const int tid = threadIdx.x, recent = p.recent, edge = p.keep - recent, total = pairs + recent, nu = p.units;
  char* const base = p.pool + layer * p.layer_bytes + h * p.head_bytes;
  for (int i = tid; i < total; i += T) {
    const int from = i < pairs ? list[pairs + i] : n - recent + (i - pairs), to = i < pairs ? list[i] : edge + (i - pairs);
    moves[i] = {place(p, b, from), place(p, b, to)};
  }
  __syncthreads();
  // movers by as many as fit at once, the recent ones all in the last round, as their places may be those of movers and of one another
  for (int u0 = 0, end; u0 < total * nu; u0 = end) {
    end = total * nu - u0 <= kFewUnits * T ? total * nu : min(u0 + kFewUnits * T, pairs * nu);
    uint4 v[kFewUnits];
    // piece u0 + j T + this thread of the rows' ones: its offset in a row, and whether it is to be moved
    auto piece = [&](int j, Move& move, int64_t& off) {
      const int u = u0 + j * T + tid, i = u / nu, e = u - i * nu;
      if (u >= end) return false;
      move = moves[i];
      off = (e >= nu / 2 ? p.kv_bytes - nu / 2 * 16 : 0) + e * 16;
      return move.from >= 0 && move.to >= 0;
    };
    Move move;
    int64_t off;
#pragma unroll
    for (int j = 0; j < kFewUnits; ++j)
      if (piece(j, move, off)) v[j] = *reinterpret_cast<const uint4*>(base + move.from + off);
    if (end == total * nu) __syncthreads();
#pragma unroll
    for (int j = 0; j < kFewUnits; ++j)
      if (piece(j, move, off)) *reinterpret_cast<uint4*>(base + move.to + off) = v[j];
  }
}

// The plan of a row.  A histogram of the keys' upper bits (of the masses' exponents and first bits) finds the bin of the last
// one that stays.  One more pass makes two bits of each key, above that bin and in it, and everything after that is done on
// those, a lane a word of 32: histograms of what is in the bin, over its own range, until all of it stays or all of it is equal
// (then the first ones stay); the holes and movers; their lists.  A pass over the keys is bound by issue slots (30000 of them:
// 940 warp steps, 3 us), so there are two.
template <int T>
__global__ void __launch_bounds__(T, 1024 / T) evict_plan_kernel(const EvictParams p) {
  constexpr int kWarps = T / 32;
  extern __shared__ __align__(16) uint32_t s_dyn[];
  __shared__ SelectShared<T> s_sel;
  __shared__ uint32_t s_range[2];
  __shared__ __align__(8) uint64_t s_copied;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, h = row % p.hkv, b = row / p.hkv % p.batch, layer = row / p.hkv / p.batch;
  const int keep = p.keep, recent = p.recent, sinks = p.sinks, edge = keep - recent;  // places below: sinks, then candidates that stay
  if (tid == 0) {
    mbar_init(&s_copied, 1);
    fence_barrier_init();
  }
  s_sel.clear();
  __syncthreads();
  pdl_wait();
  int* const source = p.source ? p.source + static_cast<int64_t>(row) * keep : nullptr;
  int* const plan = p.plan + row * p.plan_ints;
  float* const mass = p.mass + layer * p.ml + b * p.mb + h * p.mh;
  const int n = length_of(p.map, p.seq_lens, b);
  if (n <= keep) {
    if (tid == 0) p.head[row] = make_int2(n, 0);
    if (source)
      for (int i = tid; i < keep; i += T) source[i] = i < n ? i : -1;
    return;
  }
  const int c = n - recent - sinks, m = edge - sinks, words = (c + 31) / 32;  // candidates, and those that stay
  int *const holes = plan, *const movers = plan + p.most;
  uint32_t pairs = 0;
  const int* list = nullptr;  // holes and then movers in shared memory, where they fit
  if (m > 0) {
    uint32_t* const s_in = s_dyn;            // a bit a candidate: stays
    uint32_t* const s_equal = s_in + words;  // equals the last one that stays
    const float* const value = mass + sinks;
    // whole 16 bytes, and what lies before and behind them
    const int head = min(c, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(value) & 15)) / 4 & 3)), quads = (c - head) / 4;
    const bool held = c <= p.held;
    uint32_t* const keys = (held ? s_dyn + (2 * words + 3) / 4 * 4 : reinterpret_cast<uint32_t*>(plan + 2 * p.most)) +
                           (4 - head) % 4;
    // a key's bin: its bits under the sign's, or 0 for negative ones.  Keys in the lowest bin are counted apart: it is where
    // positions without any weight lie
    constexpr int kBits = SelectShared<T>::kBits, kShift = 31 - kBits;
    constexpr uint32_t kZero = 0x80000000u;
    auto bin = [](uint32_t k) { return (max(k, kZero) - kZero) >> kShift; };
    uint32_t low = 0;
    auto take = [&](float v) {
      const uint32_t k = order_key(v), d = bin(k);
      if (d == 0) ++low;
      else atomicAdd(s_sel.bins() + d, 1u);
      return k;
    };
    const int rest = c - head - 4 * quads;
    if (tid < head) keys[tid] = take(value[tid]);
    if (tid < rest) keys[c - rest + tid] = take(value[c - rest + tid]);
    const float4* const value4 = reinterpret_cast<const float4*>(value + head);
    uint4* const keys4 = reinterpret_cast<uint4*>(keys + head);
    if (held) {  // copied past L1, of which so much shared memory leaves little: loads by the threads took 7 us for 5.5 of 30000
      if (tid == 0)
        for (int i = 0; i < quads; i += kEvictCopy) {
          const uint32_t bytes = 16 * min(kEvictCopy, quads - i);
          mbar_expect_tx(&s_copied, bytes);
          bulk_g2s(keys4 + i, value4 + i, bytes, &s_copied, l2_policy_evict_normal());
        }
      if (tid == 0) mbar_arrive(&s_copied);
      bool copied = mbar_wait_bounded(&s_copied, 0);
      if (!copied) {
        record_status(SN_ERR_TIMEOUT);
        mbar_wait_bounded(&s_copied, 0);  // once more, as the copies land in this CTA's memory
      }
      if (__syncthreads_or(!copied)) {  // nothing may be planned by masses that have not come: the row is left as it is
        if (tid == 0) p.head[row] = make_int2(n, -1);
        if (source)
          for (int i = tid; i < keep; i += T) source[i] = i;
        return;
      }
    }
#pragma unroll 4
    for (int i = tid; i < quads; i += T) {
      const float4 v = held ? *reinterpret_cast<const float4*>(keys4 + i) : value4[i];
      keys4[i] = make_uint4(take(v.x), take(v.y), take(v.z), take(v.w));
    }
    auto count_low = [&] {
      low = __reduce_add_sync(0xffffffffu, low);
      if (lane == 0 && low) atomicAdd(s_sel.bins(), low);
      __syncthreads();
    };
    count_low();
    find_bin(static_cast<uint32_t>(m), s_sel);
    uint32_t here = s_sel.here, need = m - s_sel.above;  // in the bin, and of those that stay
    {
      const uint32_t digit = s_sel.digit, from = digit == 0 ? 0 : kZero + (digit << kShift);
      const uint32_t upto = kZero + (digit << kShift) + ((1u << kShift) - 1), span = upto - from;
      auto mark = [&](int w, uint32_t k, bool in) {
        const uint32_t above = __ballot_sync(0xffffffffu, in && k > upto), equal = __ballot_sync(0xffffffffu, in && k - from <= span);
        if (lane == 0) {
          s_in[w] = above;
          s_equal[w] = equal;
        }
      };
      const int whole = c / 32;
#pragma unroll 4
      for (int w = warp; w < whole; w += kWarps) mark(w, keys[32 * w + lane], true);
      if (whole < words && warp == whole % kWarps) mark(whole, 32 * whole + lane < c ? keys[32 * whole + lane] : 0, 32 * whole + lane < c);
    }
    // ---- words: a warp has consecutive ones ----
    const int per = (words + kWarps - 1) / kWarps, w0 = min(warp * per, words), w1 = min(w0 + per, words);
    auto scan = [&](uint32_t v, uint32_t& all) {  // exclusive sums over the lanes, and all of it
      uint32_t sum = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      all = __shfl_sync(0xffffffffu, sum, 31);
      return sum - v;
    };
    __syncthreads();
    auto before = [&](const uint32_t* counts, uint32_t& all) {  // the sum over the warps before this one, and over all
      uint32_t v = lane < kWarps ? counts[lane] : 0;
      const uint32_t sum = scan(v, all);
      return __shfl_sync(0xffffffffu, sum, warp);
    };
    // the bin's keys, until all or none of them differ in whether they stay
    while (here != need) {
      if (tid < 2) s_range[tid] = tid == 0 ? 0xffffffffu : 0;
      s_sel.clear();
      __syncthreads();
      auto each = [&](auto f) {  // f(word, bit, key) of this lane's
        for (int w = w0 + lane; w < w1; w += 32)
          for (uint32_t left = s_equal[w]; left; left &= left - 1) f(w, left & (0u - left), keys[32 * w + __ffs(left) - 1]);
      };
      uint32_t lo = 0xffffffffu, hi = 0;
      each([&](int, uint32_t, uint32_t k) {
        lo = min(lo, k);
        hi = max(hi, k);
      });
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      if (lane == 0) {
        atomicMin(&s_range[0], lo);
        atomicMax(&s_range[1], hi);
      }
      __syncthreads();
      lo = s_range[0];
      hi = s_range[1];
      if (lo == hi) break;  // equal: the first ones stay
      const int shift = max(0, 32 - __clz(hi - lo) - kBits);
      low = 0;
      each([&](int, uint32_t, uint32_t k) {
        if ((k - lo) >> shift == 0) ++low;
        else atomicAdd(s_sel.bins() + ((k - lo) >> shift), 1u);
      });
      count_low();
      find_bin(need, s_sel);
      const uint32_t digit = s_sel.digit;
      here = s_sel.here;
      need -= s_sel.above;
      each([&](int w, uint32_t bit, uint32_t k) {
        const uint32_t d = (k - lo) >> shift;
        if (d > digit) s_in[w] |= bit;
        if (d != digit) s_equal[w] &= ~bit;
      });
    }
    __syncthreads();
    // the first `need` of the equal ones stay
    uint32_t mine = 0, all;
    for (int w = w0 + lane; w < w1; w += 32) mine += __popc(s_equal[w]);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) s_sel.warp[warp] = mine;
    __syncthreads();
    uint32_t at = before(s_sel.warp, all);
    // ... and what does not stay below the edge is a hole, what stays above it moves
    auto front = [&](int w) {  // the word's candidates below the edge
      const int k = min(max(edge - (sinks + 32 * w), 0), 32);
      return k < 32 ? (1u << k) - 1 : 0xffffffffu;
    };
    auto valid = [&](int w) { return c - 32 * w < 32 ? (1u << (c - 32 * w)) - 1 : 0xffffffffu; };
    mine = 0;
    uint32_t mine_holes = 0;
    for (int w = w0; w < w1; w += 32) {
      const int k = w + lane;
      uint32_t equal = k < w1 ? s_equal[k] : 0;
      const uint32_t rank = at + scan(__popc(equal), all);
      at += all;
      if (k >= w1) continue;
      const uint32_t left = rank < need ? need - rank : 0;  // of this word's
      while (static_cast<uint32_t>(__popc(equal)) > left) equal ^= 0x80000000u >> __clz(equal);
      const uint32_t in = s_in[k] | equal, low_ones = front(k), hole = ~in & low_ones & valid(k), mover = in & ~low_ones;
      s_in[k] = in;
      s_equal[k] = hole | mover;
      mine += __popc(hole | mover);
      mine_holes += __popc(hole);
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    mine_holes = __reduce_add_sync(0xffffffffu, mine_holes);
    __syncthreads();  // s_sel.warp has been read
    if (lane == 0) {
      s_sel.warp[warp] = mine;
      s_sel.warp2[warp] = mine_holes;
    }
    __syncthreads();
    at = before(s_sel.warp, all);
    before(s_sel.warp2, pairs);
    // the lists: holes come before movers, so that one running count serves both.  In shared memory over the keys, which are
    // done with, as single stores to global memory would bind (30000 candidates: 3.5 us)
    if (held) list = reinterpret_cast<const int*>(keys);
    auto put = [&](uint32_t k, int v) {
      if (held) keys[k] = v;
      else *(k < pairs ? holes + k : movers + (k - pairs)) = v;
    };
    if (per <= 8) {  // few words a warp: one after another, a lane a candidate
      for (int w = w0; w < w1; ++w) {
        const uint32_t word = s_equal[w];
        if (word >> lane & 1) put(at + __popc(word & ((1u << lane) - 1)), sinks + 32 * w + lane);
        at += __popc(word);
      }
    } else {
      for (int w = w0; w < w1; w += 32) {
        uint32_t word = w + lane < w1 ? s_equal[w + lane] : 0;
        for (uint32_t k = at + scan(__popc(word), all); word; word &= word - 1, ++k) put(k, sinks + 32 * (w + lane) - 1 + __ffs(word));
        at += all;
      }
    }
  }
  if (source)  // of what stays where it is, and for now of the holes
    for (int i = tid; i < edge; i += T) source[i] = i;
  __syncthreads();
  pdl_launch_dependents();  // not before: CTAs of the other launch would only wait, and it may have nothing to do
  // (the histogram, which is done with, holds where the rows come from and go)
  const bool few = p.units > 0 && n - keep <= T && pairs + recent <= kFewMoves &&
                   static_cast<int>(pairs + recent) * p.units <= kFewPieces && recent * p.units <= kFewUnits * T && (list || pairs == 0);
  if (tid == 0) p.head[row] = make_int2(n, few ? -1 : static_cast<int>(pairs));
  static_assert(sizeof(s_sel.hist) >= kFewMoves * sizeof(Move));
  if (few) move_few<T>(p, layer, b, h, n, static_cast<int>(pairs), list, reinterpret_cast<Move*>(s_sel.hist));
  // mass, as the rows go: movers into holes, then the recent ones, which may overlap their places (zeros behind are left to the
  // other launch, which has more threads, if there is something for it to do)
  float w[4];
  auto read_recent = [&](int k0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + j * T + tid;
      if (k < recent) w[j] = mass[n - recent + k];
    }
  };
  read_recent(0);
#pragma unroll 4
  for (uint32_t i = tid; i < pairs; i += T) {
    const int hole = list ? list[i] : holes[i], mover = list ? list[pairs + i] : movers[i];
    if (list && !few) {
      holes[i] = hole;
      movers[i] = mover;
    }
    mass[hole] = mass[mover];
    if (source) source[hole] = mover;
  }
  __syncthreads();
  if (few && keep + tid < n) mass[keep + tid] = 0.f;
  for (int k0 = 0; k0 < recent; k0 += 4 * T) {
    if (k0 > 0) {
      read_recent(k0);
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + j * T + tid;
      if (k >= recent) continue;
      mass[edge + k] = w[j];
      if (source) source[edge + k] = n - recent + k;
    }
  }
}

__device__ __forceinline__ uint32_t ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Barrier over the cluster of C CTAs, for what they read and write in global memory.
__device__ __forceinline__ void cluster_bar(int C) {
  if (C == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// One cluster a (layer, stream, head).  All its warps take pairs of holes and movers; when those have left, the recent rows go
// to their places, which movers may have lain in, and which recent rows may overlap: what the cluster holds at once is read
// before the barrier, further ones are read and written round by round.  A warp's lanes look up 32 positions at once and copy
// K and V rows by 16 bytes, eight loads in flight a lane.
template <typename T, int NU>  // units of T in a position's two rows, 0: 2 * row_bytes / sizeof(T)
__global__ void __launch_bounds__(kMoveThreads, 3) evict_move_kernel(const EvictParams p) {
  constexpr int U = 8;  // units in flight a lane
  pdl_launch_dependents();
  pdl_wait();
  uint32_t nranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nranks));
  const int C = static_cast<int>(nranks), rank = static_cast<int>(ctarank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int keep = p.keep, recent = p.recent, edge = keep - recent;
  const int64_t row = blockIdx.x / C;
  const int h = static_cast<int>(row % p.hkv), b = static_cast<int>(row / p.hkv % p.batch), layer = static_cast<int>(row / p.hkv / p.batch);
  const int* const plan = p.plan + row * p.plan_ints;
  const int2 head = p.head[row];
  const int n = head.x, pairs = head.y;
  if (n <= keep || pairs < 0) return;  // nothing to do, or done
  {  // mass behind what is kept: whole 16 bytes, and what lies before and behind them
    const int threads = kMoveThreads * C, me = rank * kMoveThreads + static_cast<int>(threadIdx.x);
    float* const tail = p.mass + layer * p.ml + b * p.mb + h * p.mh + keep;
    const int len = n - keep, before = min(len, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(tail) & 15)) / 4 & 3)), quads = (len - before) / 4;
    if (me < before) tail[me] = 0.f;
    if (me < len - before - 4 * quads) tail[before + 4 * quads + me] = 0.f;
    for (int i = me; i < quads; i += threads) reinterpret_cast<float4*>(tail + before)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int nu = NU ? NU : static_cast<int>(2 * p.row_bytes / sizeof(T));
  char* const base = p.pool + layer * p.layer_bytes + h * p.head_bytes;
  // Unit u0 + 32 j + this lane of the cnt positions that the lanes have looked up: which of them, and its offset in it.
  auto unit = [&](int u0, int j, int cnt, int& at) {
    int e;
    if constexpr (NU > 0) {  // u0 is a multiple of 32
      at = u0 / NU + j * (32 / NU) + lane / NU;
      e = lane % NU;
    } else {
      const int u = u0 + 32 * j + lane;
      at = u / nu;
      e = u - at * nu;
    }
    const bool in = at < cnt;
    at &= 31;
    constexpr int64_t size = sizeof(T);
    return in ? (e >= nu / 2 ? p.kv_bytes - nu / 2 * size : 0) + e * size : int64_t{-1};
  };
  auto load = [&](int64_t from, int64_t to, int cnt, int u0, T (&v)[U]) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      int at;
      const int64_t off = unit(u0, j, cnt, at), f = __shfl_sync(0xffffffffu, from, at), t = __shfl_sync(0xffffffffu, to, at);
      if (off >= 0 && f >= 0 && t >= 0) v[j] = *reinterpret_cast<const T*>(base + f + off);
    }
  };
  auto store = [&](int64_t from, int64_t to, int cnt, int u0, const T (&v)[U]) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      int at;
      const int64_t off = unit(u0, j, cnt, at), f = __shfl_sync(0xffffffffu, from, at), t = __shfl_sync(0xffffffffu, to, at);
      if (off >= 0 && f >= 0 && t >= 0) *reinterpret_cast<T*>(base + t + off) = v[j];
    }
  };
  const int warps = kMoveWarps * C, wid = warp * C + rank;

  // rows of the recent positions that a warp holds at once, and where this lane's first one is and goes
  const int per = min(32, max(1, 32 * U / nu)), round = per * warps;
  int64_t recent_from = -1, recent_to = -1;
  auto look_up_recent = [&](int k) {
    recent_from = recent_to = -1;
    if (lane >= per || k >= recent) return;
    recent_from = place(p, b, n - recent + k);
    recent_to = place(p, b, edge + k);
  };
  look_up_recent(wid * per + lane);
  // ---- movers into holes ----
  const int batch = min(32, (pairs + warps - 1) / warps);
  for (int first = wid * batch; first < pairs; first += warps * batch) {
    const int cnt = min(batch, pairs - first), units = cnt * nu;
    int64_t from = -1, to = -1;
    if (lane < cnt) {
      to = place(p, b, plan[first + lane]);
      from = place(p, b, plan[p.most + first + lane]);
    }
    for (int u0 = 0; u0 < units; u0 += 32 * U) {
      T v[U];
      load(from, to, cnt, u0, v);
      store(from, to, cnt, u0, v);
    }
  }
  // ---- the recent positions, n - recent + k -> edge + k ----
  const bool overlap = n - keep < recent;
  bool moved = false;  // the movers have left
  for (int u0 = 0; u0 < nu; u0 += 32 * U) {  // (a part of the row, where a warp cannot hold a whole one)
    for (int k0 = 0; k0 < recent; k0 += round) {
      const int mine = k0 + wid * per, cnt = min(max(recent - mine, 0), per);
      if (moved) look_up_recent(mine + lane);
      T v[U];
      load(recent_from, recent_to, cnt, u0, v);
      if (!moved || overlap) cluster_bar(C);
      moved = true;
      store(recent_from, recent_to, cnt, u0, v);
    }
  }
}

// The launch of the moves, in clusters of C.
struct MoveLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  MoveLaunch(int rows, int C, cudaStream_t st) {
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * C);
    cfg.blockDim = dim3(kMoveThreads);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(C);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
  MoveLaunch(const MoveLaunch&) = delete;
};

// Whether the current device takes clusters of kMoveCluster: it need not (above 8 they are not portable), and has to be asked
// before the plan is launched, which has moved the masses when the moves are.
template <typename T, int NU>
bool large_moves() {
  static signed char known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return false;
  }
  if (known[dev] == 0) {
    const MoveLaunch one(1, kMoveCluster, nullptr);
    int fit = 0;
    const bool yes = large_clusters<evict_move_kernel<T, NU>>() &&
                     cudaOccupancyMaxActiveClusters(&fit, evict_move_kernel<T, NU>, &one.cfg) == cudaSuccess && fit > 0;
    cudaGetLastError();
    known[dev] = yes ? 1 : -1;
  }
  return known[dev] > 0;
}

template <typename T, int NU>
int launch_move(int rows, int C, cudaStream_t st, const EvictParams& p) {
  const MoveLaunch l(rows, C, st);
  if (cudaLaunchKernelEx(&l.cfg, evict_move_kernel<T, NU>, p) != cudaSuccess) {
    cudaGetLastError();
    return SN_ERR_LAUNCH;
  }
  return SN_OK;
}

template <int T>
int launch_plan(int rows, size_t smem, cudaStream_t st, const EvictParams& p) {
  if (!smem_room<evict_plan_kernel<T>>(kEvictWords * 4)) return SN_ERR_LAUNCH;
  return launch(evict_plan_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(T), smem, st, true, p);
}

// Both launches; the moves by units of T, NU of them in a position's two rows (0: as row_bytes says).
template <typename T, int NU>
int evict(int r, size_t smem, cudaStream_t st, const EvictParams& p) {
  const int64_t rows = r, room = static_cast<int64_t>(p.map.max_pages) * p.map.page_size;
  // three CTAs fit on an SM, one beside a plan: all of them start at once (48 rows, 320 moved rows each, 8 CTAs a row 18.3, 7
  // 16.6); two a row at least, as not all of the streams may be cut.  Clusters of 16 where each CTA has an SM of its own (4
  // rows of 30011 positions 41 -> 33 us; 24 rows of 2112, 2.6 CTAs an SM: 16.3 -> 21)
  const int C = rows * kMoveCluster <= sm_count() && large_moves<T, NU>()
                    ? kMoveCluster
                    : static_cast<int>(std::clamp<int64_t>((3 * sm_count() - 2 * rows) / rows, 2, 8));
  // the plan's passes are shorter with more threads, its barriers longer: 48 rows of 8000 positions 26.5 us with 1024 threads a
  // row and 29.5 with 512, of 4096 both 18.9, of 2112 18.8 and 17.7 (moves included); where there are more rows than SMs, 512,
  // and where there are more than two an SM, 256, four CTAs an SM, whose moves fill the waits of one another's plans (4096 rows
  // of 2112: 191 -> 144, 768 rows 41 -> 35, 144 of them with work 18.4 -> 19.8, 480 of 9000 129 -> 125).  That holds while four
  // plans' keys fit an SM, up to some 11500 positions: of tables of 9000 768 rows take 375 us, with 512 threads 379, but of
  // 16000 and 30000 675 and 687, with 512 threads 615 and 621
  const int rc = rows > 2 * sm_count()                 ? launch_plan<256>(r, smem, st, p)
                 : rows <= sm_count() && room > 4096 ? launch_plan<1024>(r, smem, st, p)
                                                     : launch_plan<512>(r, smem, st, p);
  return rc != SN_OK ? rc : launch_move<T, NU>(r, C, st, p);
}

}  // namespace

int tu_status_evict(bool reset, cudaStream_t st, int* out) { return read_tu_status(reset, st, out); }

}  // namespace sn

extern "C" {

size_t sn_evict_workspace_size(int layers, int batch, int nheads_kv, int64_t max_positions, int keep) {
  if (layers < 1 || batch < 1 || nheads_kv < 1 || max_positions < 1 || keep < 1) return 0;
  return static_cast<size_t>(layers) * batch * nheads_kv * (sizeof(int2) + sn::plan_size(max_positions, keep) * sizeof(int)) + 16;
}

int sn_evict_positions(void* pool, int layers, int num_pages, int page_size, int nheads_kv, int head_dim,
                       const int* page_table, int64_t table_stride, int max_pages, const int* seq_lens, float* mass,
                       int64_t mass_layer_stride, int64_t mass_batch_stride, int64_t mass_head_stride, int batch,
                       int keep, int recent, int sinks, int* source, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (!pool || !page_table || !seq_lens || !mass || !workspace || layers < 1 || num_pages < 1 || page_size < 1 ||
      nheads_kv < 1 || head_dim < 1 || max_pages < 1 || table_stride < max_pages || batch < 1 || keep < 1 || recent < 0 ||
      sinks < 0 || recent > keep || sinks > keep - recent)
    return SN_ERR_INVALID_ARGUMENT;
  const int64_t room = static_cast<int64_t>(max_pages) * page_size;
  if ((nheads_kv > 1 && mass_head_stride < room) || (batch > 1 && mass_batch_stride < room) ||
      (layers > 1 && mass_layer_stride < room) ||
      workspace_bytes < sn_evict_workspace_size(layers, batch, nheads_kv, room, keep))
    return SN_ERR_INVALID_ARGUMENT;
  if (!sn::aligned16(workspace)) return SN_ERR_MISALIGNED;
  const int64_t rows = static_cast<int64_t>(layers) * batch * nheads_kv;
  if (rows > INT32_MAX / sn::kMoveCluster || head_dim > 8192 || room > sn::kEvictMost) return SN_ERR_UNSUPPORTED;
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
  p.head = static_cast<int2*>(workspace);
  p.plan = reinterpret_cast<int*>(p.head + (rows + 1) / 2 * 2);
  p.plan_ints = sn::plan_size(room, keep);
  p.most = static_cast<int>(sn::most_pairs(room, keep));
  p.batch = batch;
  p.hkv = nheads_kv;
  p.keep = keep;
  p.recent = recent;
  p.sinks = sinks;
  p.units = sn::aligned16(pool) && p.row_bytes % 16 == 0 ? 2 * p.row_bytes / 16 : 0;
  p.held = sn::keys_held(room) ? static_cast<int>(room) : 0;
  const size_t smem = static_cast<size_t>(sn::bit_words(room) + p.held) * sizeof(uint32_t);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int r = static_cast<int>(rows);
  if (p.units) {
    if (head_dim == 128) return sn::evict<uint4, 32>(r, smem, st, p);
    if (head_dim == 64) return sn::evict<uint4, 16>(r, smem, st, p);
    return sn::evict<uint4, 0>(r, smem, st, p);
  }
  return sn::evict<uint16_t, 0>(r, smem, st, p);
}

}  // extern "C"
