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
#include "tc.cuh"

#include <algorithm>
#include <climits>

namespace sn {
namespace {

// A page table: its entry for a block of page_size positions of stream b, or -1 where there is none.
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
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
struct PoolStrides {  // elements
  int64_t page, head, tok;
};

// ---------------------------------------------------------------------------
// rotary_paged_append.  Pure data movement (a qkv row read, q / k / v
// written, a cos / sin row per position), so it is bounded by HBM for
// prompts (12288 tokens of 24 heads of 128: 27.1 us, 5.8 TB/s) and by the chain
// stream - length - table - page for a decode step (48 tokens: 2.8 us).
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
  const bool rotated = head < p.hq + p.hkv && j < p.rot / 2;
  const bool halves = rotated && !p.interleaved;
  const int i1 = halves ? j : 2 * j, i2 = halves ? j + p.rot / 2 : 2 * j + 1;
  const __nv_bfloat16* src = p.qkv + t * p.ld + static_cast<int64_t>(head) * p.hd;
  __nv_bfloat16 o1 = src[i1], o2 = src[i2];
  __nv_bfloat16* const q = p.q + (static_cast<int64_t>(t) * p.hq + head) * p.hd;  // if it is a head of q
  const bool stray = p.cu && (t < p.cu[b] || t >= end);  // a token of no stream
  const int pos = p.seq_lens[b] - (end - t);
  if (stray || pos < 0 || pos >= p.max_pos) {
    if (!stray) record_status(SN_ERR_INVALID_ARGUMENT);
    if (head < p.hq) q[i1] = q[i2] = __float2bfloat16_rn(0.f);
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
    dst = q;
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

// The same by 16-byte chunks (head_dim and rot_dim multiples of 16, 16-byte
// rows).  A warp takes one token: lane u + U * phase (U = head_dim / 16 units
// a head) holds the token's 8 cos and sin values of its unit in registers and
// takes the heads phase and phase + 32 / U (blockIdx.y: the next ones; six heads
// a lane took 28.7 us for 27.1 and 3.5 for 2.8 below, fewer warps holding more).
// A unit is the two chunks whose elements pair up (8u and rot/2 + 8u of the halves
// layout) or two neighbours, so a head is read and written in whole 128-byte
// lines.  The qkv loads wait for nothing, so they cover the look-up of the
// stream, its length, the table row and the page; they are read once, so they
// are the first to leave L2 (17.7 us for 18.7 with 48 heads of half rotation).
constexpr int kAppendHeads = 2;

// A warp writes zeros to the n elements (a multiple of 16) of a q row.  Out of line: in the kernel it costs the others 4% of
// their time.
__device__ __noinline__ void zero_row(__nv_bfloat16* row, int n) {
  for (int i = 8 * (threadIdx.x & 31); i < n; i += 256) *reinterpret_cast<uint4*>(row + i) = make_uint4(0, 0, 0, 0);
}

template <bool kInterleaved>
__global__ void __launch_bounds__(128) rotary_paged_append_vec_kernel(const AppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int U = p.hd / 16, phases = 32 / U;
  const int phase = lane / U, u = lane - phase * U;
  const int heads = p.hq + 2 * p.hkv;
  const bool turned = u < p.rot / 16;
  const bool apart = !kInterleaved && turned;
  const int c1 = apart ? 8 * u : 16 * u, c2 = apart ? p.rot / 2 + 8 * u : 16 * u + 8;
  const __nv_bfloat16* src = p.qkv + t * p.ld;
  uint4 a[kAppendHeads], b[kAppendHeads];
  const int h0 = blockIdx.y * (kAppendHeads * phases) + phase;
#pragma unroll
  for (int i = 0; i < kAppendHeads; ++i) {
    const int h = h0 + i * phases;
    if (phase < phases && h < heads) {
      a[i] = __ldcs(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(h) * p.hd + c1));
      b[i] = __ldcs(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(h) * p.hd + c2));
    }
  }
  // the stream: the number of streams that end at or before t, 32 probes at a time
  int s = t, end = t + 1;
  if (p.cu) {
    int lo = 0, n = p.batch;
    while (n > 32) {
      const int step = (n + 31) / 32;
      const int at = min(lo + (lane + 1) * step, p.batch);
      lo += __popc(__ballot_sync(0xffffffffu, lane + 1 < 32 && (lane + 1) * step < n && p.cu[at] <= t)) * step;
      n = min(step, p.batch - lo);
    }
    lo += __popc(__ballot_sync(0xffffffffu, lane < n && p.cu[min(lo + lane + 1, p.batch)] <= t));
    s = min(lo, p.batch - 1);
    end = p.cu[s + 1];
    if (t < p.cu[s] || t >= end) {  // a token of no stream
      zero_row(p.q + static_cast<int64_t>(t) * p.hq * p.hd, p.hq * p.hd);
      return;
    }
  }
  const int pos = p.seq_lens[s] - (end - t);
  if (pos < 0 || pos >= p.max_pos) {
    record_status(SN_ERR_INVALID_ARGUMENT);
    zero_row(p.q + static_cast<int64_t>(t) * p.hq * p.hd, p.hq * p.hd);
    return;
  }
  const int pg = page_of(p.map, s, pos / p.map.page_size);
  if (pg < 0) record_status(SN_ERR_INVALID_ARGUMENT);
  float cs[8], sn[8];
  if (turned) {
    const float4* cr = reinterpret_cast<const float4*>(p.cos + static_cast<int64_t>(pos) * (p.rot / 2) + 8 * u);
    const float4* sr = reinterpret_cast<const float4*>(p.sin + static_cast<int64_t>(pos) * (p.rot / 2) + 8 * u);
    *reinterpret_cast<float4*>(cs) = cr[0];
    *reinterpret_cast<float4*>(cs + 4) = cr[1];
    *reinterpret_cast<float4*>(sn) = sr[0];
    *reinterpret_cast<float4*>(sn + 4) = sr[1];
  }
  const int row = pos % p.map.page_size;
#pragma unroll
  for (int i = 0; i < kAppendHeads; ++i) {
    const int h = h0 + i * phases;
    if (phase >= phases || h >= heads) continue;
    if (turned && h < p.hq + p.hkv) {
      uint32_t x[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
      auto turn = [&](float x1, float x2, int j, float& y1, float& y2) {
        y1 = __fsub_rn(__fmul_rn(x1, cs[j]), __fmul_rn(x2, sn[j]));
        y2 = __fadd_rn(__fmul_rn(x2, cs[j]), __fmul_rn(x1, sn[j]));
      };
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y1, y2, y3, y4;
        if (kInterleaved) {  // register j of each chunk is a pair
          turn(bf16lo(x[j]), bf16hi(x[j]), j, y1, y2);
          turn(bf16lo(x[4 + j]), bf16hi(x[4 + j]), 4 + j, y3, y4);
          x[j] = pack2(y1, y2);
          x[4 + j] = pack2(y3, y4);
        } else {  // elements 2j, 2j + 1 of both chunks
          turn(bf16lo(x[j]), bf16lo(x[4 + j]), 2 * j, y1, y2);
          turn(bf16hi(x[j]), bf16hi(x[4 + j]), 2 * j + 1, y3, y4);
          x[j] = pack2(y1, y3);
          x[4 + j] = pack2(y2, y4);
        }
      }
      a[i] = make_uint4(x[0], x[1], x[2], x[3]);
      b[i] = make_uint4(x[4], x[5], x[6], x[7]);
    }
    __nv_bfloat16* dst;
    if (h < p.hq) {
      dst = p.q + (static_cast<int64_t>(t) * p.hq + h) * p.hd;
    } else {
      if (pg < 0) continue;
      dst = h < p.hq + p.hkv ? p.kp + pg * p.ks.page + (h - p.hq) * p.ks.head + row * p.ks.tok
                             : p.vp + pg * p.vs.page + (h - p.hq - p.hkv) * p.vs.head + row * p.vs.tok;
    }
    *reinterpret_cast<uint4*>(dst + c1) = a[i];
    *reinterpret_cast<uint4*>(dst + c2) = b[i];
  }
}

// ---------------------------------------------------------------------------
// paged_decode_attention, o = sum_t softmax_t(scale q.k_t) v_t, one pass over
// K and V with the running maximum and sum.
//
// One CTA per (stream, query head); each of its 4 warps takes every fourth
// position, lane l holds elements l, l + 32, ... of the head.  Any head_dim up
// to 256, any strides; bounded by the chain of a position (dot product, sum over
// the warp, exponential).
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
// The tensor-core form (head_dim 64 or 128, pages of whole 16-position tiles,
// 16-byte rows).  K and V are read once and the products are small, so it is
// bounded by HBM as long as enough loads are in flight and the warps issue
// few instructions a tile; everything below serves that:
//
// * A warp works alone on tiles of 16 positions of one (stream, key/value
//   head): one lane keeps a ring of two tiles (four of 64-element heads)
//   filled by TMA, 16 KB a warp, 12 warps an SM; no barrier of more than the
//   warp in the loop.  The products are mma.m16n8k16 (tcgen05 would want 128
//   rows of a tile; the 8 columns of heads here leave the tensor pipe idle
//   either way).  Loads by every lane instead, into operand registers or by
//   cp.async, took 500 instructions a tile for 280 here (3 streams of up to
//   100001 positions: 102 and 118 us for 84; with the weights' second product
//   86.6, 5.7 TB/s of 6.4).
// * S^T = K q^T: the contraction index may be permuted as long as K and q
//   agree, so lane (g = lane / 4, t = lane % 4) takes whole 16-byte chunks t,
//   t + 4, ... of two positions, and the same chunks of q's head g.
// * O^T += V^T P^T: the lane takes one chunk (two) of four positions, pairs of
//   positions are packed by byte permutes (the output index is permuted, which
//   the store undoes); P goes from S's accumulator layout to the operand
//   layout by an 8x8 transpose (movmatrix).
// * With order(i) = 0 4 1 5 2 6 3 7, lane g takes K rows order(g) and
//   order(g) + 8 and V chunk order(g): in the 128-byte swizzle TMA writes, the
//   eight lanes of a shared-memory phase then hit eight different chunks.
// * Softmax in the exponent of 2 with a running maximum that moves only when
//   a score passes it by more than 8 (weights up to 2^8 are as exact in bf16
//   and fp32): the warp's vote replaces the reduction and the rescaling of
//   most tiles.  P goes into the product as two bf16 operands, its rounding and
//   what that left (2^-16 together, so the output's own rounding is all that
//   shows: error 0.0017 of the norm for 0.0022 with one operand, 64 ragged
//   streams 67.2 us for 66.4); the sum of weights is fp32.
// * With more than 8 heads a set, q is read from shared memory instead of held as
//   operands: there would be no registers for the second product (8 streams of
//   8000 positions, 32 query and 2 key/value heads, 38.9 us for 35.9).
// * The work of all streams is one axis of tiles, cut evenly over the grid,
//   whatever the lengths are (they are only known on the device).  A CTA's
//   warps take every sixth tile of its piece of a (stream, head) and join
//   through shared memory; a (stream, head) cut over several CTAs is joined by
//   the CTA that finishes last, in the order of the pieces, so the result does
//   not depend on which one that is.  (With the weights in one operand, 12 warps
//   in one CTA an SM: 84.5 and 67.5 us for the long and the 64 ragged streams, 4
//   warps in three: 87.8 and 64.3; six in two: 85.4 and 65.9.)
// ---------------------------------------------------------------------------
constexpr int kAttWarps = 6;
constexpr int kCutGain = 14;   // steps that a cut has to save
constexpr int kCutSteps = 2;   // and the least a CTA takes of one
constexpr int kJoinMost = 48;  // partial results that one CTA joins by itself
constexpr int kJoinGroup = 8;  // and those of a group otherwise
constexpr int kTile = 16;
constexpr int kAttHeadsMax = 16;   // heads a CTA takes together
constexpr int kAttGridMax = 640;   // partial results the workspace holds, two a CTA

struct AttendSplit {
  float* part;       // [2 * grid][kHeadsMax][HD + 2] partial sums, maxima, outputs
  unsigned* ticket;  // [2][2 * grid] arrivals of a set's pieces or groups, of a group's pieces; zero between calls
  int group, sets;   // query heads per key/value head; head sets of a stream (hkv * sets per kv head)
  int sets_per_kv, heads_per_set;
  int slots;  // CTAs that are on the device together: no more take part in a cut
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// A warp's bounded wait for a tile: true in every lane or in none, however close to the limit it lands.
__device__ __forceinline__ bool wait_tile(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
}
// One tile of K or V: [head_dim / 64][16 positions][64 elements].
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int row, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(0), "r"(row), "r"(0), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }

// Tiles a warp's ring holds (16 KB for K and V together), and a CTA's shared
// memory (the rings start on 1024 bytes, as the swizzle wants).
template <int HD>
constexpr int ring_stages() { return 2 * 128 / HD; }
template <int HD>
constexpr uint32_t stage_bytes() { return 2 * kTile * HD * 2; }
template <int HD>
constexpr uint32_t ring_bytes() { return kAttWarps * ring_stages<HD>() * stage_bytes<HD>(); }

// The pieces of one (stream, head set) joined, in their order whichever CTA does it: called by each of the n CTAs that have
// one, the mine-th, when its partial result is written.  A piece has the first of its CTA's two places, but for the first
// piece of a set that starts inside a CTA's share (skip 1).
template <int HD, int H>
__device__ __forceinline__ void join_pieces(const AttendSplit& sp, unsigned char* ring, int first, int skip, int n,
                                         int mine, int nh, __nv_bfloat16* out, float* lse) {
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPart = H * (HD + 2);
  // A set's tickets are those of its first piece's place, so that they do not depend on the call's sizes.  Many pieces are
  // joined in groups, each by its last CTA to arrive and in the place of its first piece, with that place's ticket, and
  // the groups by the last of those: about 100 pieces of 16 heads (3 streams of up to 100001 positions, one key/value
  // head) 65 -> 51 us; with 17 to 48 pieces the second round costs more than it saves (4 streams of up to 10303 positions
  // 23.4 -> 29.3 us).
  const int each = n > kJoinMost ? kJoinGroup : n;
  int from = mine / each * each, step = 1, cnt = min(each, n - from);
  bool final = each == n;
  unsigned* arrival = sp.ticket + (final ? 0 : 2 * kAttGridMax) + 2 * (first + from) + (from == 0 ? skip : 0);
  while (true) {
    __syncthreads();
    if (tid == 0) {
      __threadfence();  // the whole CTA's partial result (the barrier above) before its arrival
      const unsigned before = atomicAdd(arrival, 1u);
      s_last = before == static_cast<unsigned>(cnt - 1);
      if (s_last) *arrival = 0;  // ready for the next call
    }
    __syncthreads();
    if (!s_last) break;
    __threadfence();
    float* const pieces = sp.part + static_cast<int64_t>(2) * (first + from) * kPart;
    const int at0 = from == 0 ? skip * kPart : 0, stride = 2 * step * kPart;
    auto piece = [&](int k) { return pieces + (k == 0 ? at0 : k * stride); };
    // weights of the cnt pieces from, from + step, ...: all their maxima and sums first, then a warp a head
    float* pm = reinterpret_cast<float*>(ring);  // [cnt][nh], the piece's factor in the end
    float* pl = pm + cnt * nh;                   // [cnt][nh]
    for (int e = tid; e < cnt * nh; e += kAttWarps * 32) {
      const int k = e / nh, h = e - k * nh;
      const float* q = piece(k);
      pm[e] = __ldcg(q + h);
      pl[e] = __ldcg(q + H + h);
    }
    __syncthreads();
    for (int h = warp; h < nh; h += kAttWarps) {
      float mt = -INFINITY, lt = 0.f;
      for (int k = lane; k < cnt; k += 32) mt = fmaxf(mt, pm[k * nh + h]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      for (int k = lane; k < cnt; k += 32) {
        const float f = pm[k * nh + h] == -INFINITY ? 0.f : exp2_approx(pm[k * nh + h] - mt);
        lt = fmaf(f, pl[k * nh + h], lt);
        pm[k * nh + h] = f;
      }
      lt = warp_sum(lt);
      if (final) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        for (int k = lane; k < cnt; k += 32) pm[k * nh + h] *= inv;
        if (lse && lane == 0) lse[h] = (mt + log2f(lt)) * 0.6931471805599453f;
      } else if (lane == 0) {
        piece(0)[h] = mt;
        piece(0)[H + h] = lt;
      }
    }
    __syncthreads();
    // four elements a thread, the pieces dealt to `deals` sets of threads
    const int quads = nh * (HD / 4);
    const int deals = max(1, kAttWarps * 32 / quads);
    float4* sums = reinterpret_cast<float4*>(pm + (2 * cnt * nh + 3) / 4 * 4);  // [deals][quads]
    for (int e = tid; e < deals * quads; e += kAttWarps * 32) {
      const int d = e / quads, q4 = e - d * quads, h = q4 / (HD / 4);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int k = d; k < cnt; k += deals) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(piece(k) + 2 * H) + q4);
        const float f = pm[k * nh + h];
        v.x = fmaf(f, x.x, v.x);
        v.y = fmaf(f, x.y, v.y);
        v.z = fmaf(f, x.z, v.z);
        v.w = fmaf(f, x.w, v.w);
      }
      sums[e] = v;
    }
    __syncthreads();
    for (int e = tid; e < quads; e += kAttWarps * 32) {
      float4 v = sums[e];
      for (int d = 1; d < deals; ++d) {
        const float4 x = sums[d * quads + e];
        v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
      }
      if (final)
        *reinterpret_cast<uint2*>(out + 4 * e) =
            make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
      else
        reinterpret_cast<float4*>(piece(0) + 2 * H)[e] = v;
    }
    if (final) break;
    final = true;
    from = 0;
    step = each;
    cnt = (n + each - 1) / each;
    arrival = sp.ticket + 2 * first + skip;
  }
}

template <int HD, int NT>
__global__ void __launch_bounds__(kAttWarps * 32, 2)
    paged_decode_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                            const AttendParams p, const AttendSplit sp) {
  constexpr int KC = HD / 32;  // 16-byte K chunks a lane takes of a row
  constexpr int VC = HD / 64;  // V chunks
  constexpr int MT = HD / 16;  // 16-row tiles of O^T
  constexpr int H = 8 * NT;
  __shared__ float s_m[kAttWarps][H], s_l[kAttWarps][H];
  constexpr int S = ring_stages<HD>();
  constexpr int BOX = kTile * 128;  // bytes of one TMA box: 16 positions of 64 elements
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kAttWarps][S];
  __shared__ float s_f[kAttWarps][H], s_mt[H];
  __shared__ uint4 s_q[NT == 1 ? 1 : H * (HD / 8)];  // q of two 8-head tiles: as operands they would spill the loop's registers
  __shared__ long long s_sum[kAttWarps];
  __shared__ int s_max[kAttWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int me = blockIdx.x;
  unsigned char* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  auto s_o = [&](int w) { return reinterpret_cast<float*>(ring + w * (S * stage_bytes<HD>())); };  // [H][HD]
  if (lane == 0) {
    for (int k = 0; k < S; ++k) mbar_init(&full[warp][k], 1);
    fence_barrier_init();
  }
  const int og = (g >> 1) | ((g & 1) << 2);  // order(g)
  const uint32_t mine = smem_u32(ring) + warp * (S * stage_bytes<HD>());
  // this lane's chunks: K rows og, og + 8 and V rows t, t + 4, t + 8, t + 12 (the swizzle is of the row's low 3 bits)
  const uint32_t k_even = og * 128 + ((t ^ og) << 4), k_odd = og * 128 + (((t + 4) ^ og) << 4);
  const uint32_t v_lo = t * 128 + ((og ^ t) << 4), v_hi = (t + 4) * 128 + ((og ^ (t + 4)) << 4);
  uint32_t parity = 0;  // of each ring slot's next wait
  bool dead = false;    // a wait ran out: nothing more is loaded, what is in flight is still waited for, its tile is left out

  pdl_launch_dependents();
  if (tid == 0) {
    tc::prefetch_map(&kmap);
    tc::prefetch_map(&vmap);
  }
  pdl_wait();

  // ---- this CTA's share of all tiles: [at, stop) ----
  long long total = 0;
  int longest = 0, tiles = 0;  // up to 32 streams: tiles of stream `lane`, in every warp
  for (int b = p.batch <= 32 ? lane : tid; b < p.batch; b += kAttWarps * 32) {
    tiles = tiles_of(stream_len(p, b));
    total += tiles;
    longest = max(longest, tiles);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (p.batch > 32) {
    if (lane == 0) {
      s_sum[warp] = total;
      s_max[warp] = longest;
    }
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kAttWarps; ++w) {
      total += s_sum[w];
      longest = max(longest, s_max[w]);
    }
  }
  total *= sp.sets;
  for (int b = me; b < p.batch; b += gridDim.x) {
    const int n = p.batch <= 32 ? __shfl_sync(0xffffffffu, tiles, b) : tiles_of(stream_len(p, b));
    if (n > 0) continue;  // an empty stream: zeros
    for (int c = tid; c < p.hq * HD; c += kAttWarps * 32)
      p.out[static_cast<int64_t>(b) * p.hq * HD + c] = __float2bfloat16_rn(0.f);
    if (p.lse)
      for (int h = tid; h < p.hq; h += kAttWarps * 32) p.lse[static_cast<int64_t>(b) * p.hq + h] = -INFINITY;
  }
  // Cutting a (stream, head set) over CTAs costs its partial results, the last CTA's join and a second start in most
  // CTAs, as much as about 14 steps of a CTA's warps over their tiles.  So nothing is cut unless the longest one is that
  // much above the even share: a CTA takes one (stream, head set), or, with more of them than CTAs, those that start in
  // its share of the tiles.  Measured, cut / not: 4 streams of 2000 positions 13.5 / 20.5 us, 2 of 1500 13.9 / 14.3, 50 of
  // 931 to 1863 31.5 / 28.9, 86 of up to 906 with one key/value head 34.8 / 19.3.
  const int grid = min(static_cast<int>(gridDim.x), sp.slots);  // CTAs with a share
  const bool cut = longest - total / grid > kCutGain * kAttWarps;
  const bool single = !cut && static_cast<long long>(p.batch) * sp.sets <= gridDim.x;
  const long long share = max((total + grid - 1) / grid, cut ? static_cast<long long>(kCutSteps) * kAttWarps : 1LL);
  long long at = me * share;
  const long long stop = single ? at + 1 : me < grid ? min(at + share, total) : 0;
  if (at >= stop) return;
  int b = 0;
  long long in_b = 0;  // place of `at` within the stream's tiles, head set by head set
  if (single) {
    b = me / sp.sets;
    if (b >= p.batch) return;
    const int n = p.batch <= 32 ? __shfl_sync(0xffffffffu, tiles, b) : tiles_of(stream_len(p, b));
    if (n == 0) return;
    in_b = static_cast<long long>(me - b * sp.sets) * n;
  } else {
    long long before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {  // every warp for itself
      if (p.batch > 32) tiles = b0 + lane < p.batch ? tiles_of(stream_len(p, b0 + lane)) : 0;
      const long long n = static_cast<long long>(tiles) * sp.sets;
      long long upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned here = __ballot_sync(0xffffffffu, at - before < upto);
      if (here) {
        const int l = __ffs(here) - 1;
        b = b0 + l;
        in_b = at - before - __shfl_sync(0xffffffffu, upto - n, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (p.batch <= 32) __syncthreads();  // the ring's barriers are set up
  const float scale2 = p.scale * 1.4426950408889634f;
  const int tpp = p.map.page_size / kTile;  // tiles a page

  bool first_piece = true;
  while (at < stop) {
    const int len = stream_len(p, b);
    const int nt = tiles_of(len);
    if (nt == 0) {
      ++b;
      in_b = 0;
      continue;
    }
    const int set = static_cast<int>(in_b / nt);
    const int lo = static_cast<int>(in_b - static_cast<long long>(set) * nt);
    if (!cut && lo > 0) {  // it belongs to the CTA where it starts
      at += nt - lo;
      in_b += nt - lo;
      if (in_b == static_cast<long long>(nt) * sp.sets) {
        ++b;
        in_b = 0;
      }
      continue;
    }
    const int hi = cut ? static_cast<int>(min(static_cast<long long>(nt), lo + (stop - at))) : nt;
    const int hk = set / sp.sets_per_kv;
    const int h0 = hk * sp.group + (set - hk * sp.sets_per_kv) * sp.heads_per_set;
    const int nh = min(sp.heads_per_set, (hk + 1) * sp.group - h0);  // heads of this set

    // q, in the operand layout: head g of each 8-head tile, chunks t + 4c
    uint4 qv[NT][NT == 1 ? KC : 1];
    if constexpr (NT == 1) {
      const __nv_bfloat16* qr = p.q + b * p.qb + (h0 + g) * p.qh;
#pragma unroll
      for (int c = 0; c < KC; ++c) qv[0][c] = g < nh ? *reinterpret_cast<const uint4*>(qr + 8 * (t + 4 * c)) : make_uint4(0, 0, 0, 0);
    } else {
      for (int e = tid; e < H * (HD / 8); e += kAttWarps * 32) {
        const int h = e / (HD / 8), c = e - h * (HD / 8);
        s_q[h * (HD / 8) + (c ^ ((h & 1) << 2))] =
            h < nh ? *reinterpret_cast<const uint4*>(p.q + b * p.qb + (h0 + h) * p.qh + 8 * c) : make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
    }
    const uint32_t q_at = smem_u32(s_q) + g * (HD * 2) + t * 16;  // chunks of odd heads swapped in fours: no two in a bank
    float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
    }
    auto load_tile = [&](int row, int pg, int slot) {  // positions row .. row + 15 of page pg
      if (lane == 0) {
        unsigned char* dst = ring + warp * (S * stage_bytes<HD>()) + slot * stage_bytes<HD>();
        mbar_arrive_expect_tx(&full[warp][slot], stage_bytes<HD>());
        tma_load_5d(dst, &kmap, row, hk, pg, &full[warp][slot]);
        tma_load_5d(dst + (HD / 64) * BOX, &vmap, row, hk, pg, &full[warp][slot]);
      }
    };
    // This warp's tiles are lo + warp + kAttWarps k, k < count.  Lane l looks up the page (and the row in it) of the l-th of the
    // next 32, and of the 32 after those one batch ahead, so that no tile waits for the table.
    const int count = (hi - lo - warp + kAttWarps - 1) / kAttWarps;  // <= 0: none
    auto look_up = [&](int k, int& row) {
      row = 0;
      if (k >= count) return 0;
      const int i = lo + warp + kAttWarps * k, blk = i / tpp;
      row = (i - blk * tpp) * kTile;
      return blk < p.map.max_pages ? p.map.table[static_cast<int64_t>(b) * p.map.table_stride + blk] : -1;
    };
    int row_now, row_then, pg_now = look_up(lane, row_now), pg_then = look_up(lane + 32, row_then);
    uint32_t loaded = 0;  // slots that hold a tile
    auto load_next = [&](int k, int into) {  // tile k into ring slot `into`
      loaded &= ~(1u << into);
      if (k >= count || dead) return;
      if (k > 0 && (k & 31) == 0) {
        pg_now = pg_then;
        row_now = row_then;
        pg_then = look_up(k + 32 + lane, row_then);
      }
      const int pg = __shfl_sync(0xffffffffu, pg_now, k & 31), row = __shfl_sync(0xffffffffu, row_now, k & 31);
      if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.map.num_pages)) {
        record_status(SN_ERR_INVALID_ARGUMENT);
        return;
      }
      load_tile(row, pg, into);
      loaded |= 1u << into;
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) load_next(k, k);
    int slot = 0;
    for (int k = 0; k < count; ++k) {
      const int i = lo + warp + kAttWarps * k;
      __syncwarp();  // every lane is done with the slot of the last step
      load_next(k + S - 1, slot == 0 ? S - 1 : slot - 1);
      bool there = (loaded >> slot) & 1;  // the same in every lane, as everything that decides about loads and shuffles
      if (there) {
        there = wait_tile(&full[warp][slot], (parity >> slot) & 1);
        if (!there) {
          record_status(SN_ERR_TIMEOUT);
          dead = true;
          wait_tile(&full[warp][slot], (parity >> slot) & 1);  // once more, as its copy may land on what the ring holds next
        }
        parity ^= 1u << slot;
      }
      const uint32_t src = mine + slot * stage_bytes<HD>();
      slot = slot + 1 == S ? 0 : slot + 1;
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 4; ++k) s[n][k] = s2[n][k] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint32_t at_k = src + (c / 2) * BOX + (c & 1 ? k_odd : k_even);
        const uint4 k0 = lds16(at_k), k1 = lds16(at_k + 1024);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint4 qc;
          if constexpr (NT == 1) qc = qv[0][c];
          else qc = lds16(q_at + n * (8 * HD * 2) + ((c ^ (g & 1)) << 6));
          mma_16816(s[n], k0.x, k1.x, k0.y, k1.y, qc.x, qc.y);
          mma_16816(s2[n], k0.z, k1.z, k0.w, k1.w, qc.z, qc.w);
        }
      }
      // scores of positions og and og + 8, heads 2t and 2t + 1
      const bool inside = there && (i + 1) * kTile <= len;  // the whole tile counts
      const bool on0 = inside || (there && i * kTile + og < len), on1 = inside || (there && i * kTile + og + 8 < len);
      bool over = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          s[n][k] = on0 ? (s[n][k] + s2[n][k]) * scale2 : -INFINITY;
          s[n][2 + k] = on1 ? (s[n][2 + k] + s2[n][2 + k]) * scale2 : -INFINITY;
          over |= fmaxf(s[n][k], s[n][2 + k]) > m[n][k] + 8.f;
        }
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float v = fmaxf(s[n][k], s[n][2 + k]);
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
            const float mn = fmaxf(m[n][k], v);
            const float keep = m[n][k] == mn ? 1.f : exp2_approx(m[n][k] - mn);
            m[n][k] = mn;
            l[n][k] *= keep;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[n][j][k] *= keep;
              o[n][j][2 + k] *= keep;
            }
          }
        }
      }
      uint32_t pb[NT][2], pr[NT][2];  // P and what its rounding left
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float base = m[n][k] == -INFINITY ? 0.f : m[n][k];  // nothing but -inf so far: weights 0
          s[n][k] = exp2_approx(s[n][k] - base);
          s[n][2 + k] = exp2_approx(s[n][2 + k] - base);
          l[n][k] += s[n][k] + s[n][2 + k];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t hi = pack2(s[n][2 * k], s[n][2 * k + 1]);
          const uint32_t rest = pack2(s[n][2 * k] - bf16lo(hi), s[n][2 * k + 1] - bf16hi(hi));
          pb[n][k] = transpose_8x8(hi);
          pr[n][k] = transpose_8x8(rest);
        }
      }
      // V^T operands: row g of an O^T tile is element e0 of the head, row g + 8 element e1; rows that do not count are
      // zeroed (their weights are 0, but what is left in the page may be NaN)
      uint4 vr[VC][4];
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        const uint32_t at_v = src + (HD / 64 + c) * BOX;
        vr[c][0] = lds16(at_v + v_lo);
        vr[c][1] = lds16(at_v + v_hi);
        vr[c][2] = lds16(at_v + 1024 + v_lo);
        vr[c][3] = lds16(at_v + 1024 + v_hi);
      }
      if (!inside) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool on = there && i * kTile + t + 4 * u < len;
#pragma unroll
          for (int c = 0; c < VC; ++c) vr[c][u] = on ? vr[c][u] : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int q2 = 0; q2 < MT / 2; ++q2) {  // O^T tiles 2 q2 and 2 q2 + 1: both halves of one register
        const int c0 = HD == 64 ? 0 : 2 * (q2 / 4), c1 = HD == 64 ? 0 : c0 + 1;
        const int w0 = HD == 64 ? q2 : q2 % 4, w1 = HD == 64 ? q2 + 2 : q2 % 4;
        auto word = [](const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; };
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x7632u : 0x5410u;
          const uint32_t a0 = __byte_perm(word(vr[c0][0], w0), word(vr[c0][1], w0), sel);
          const uint32_t a1 = __byte_perm(word(vr[c1][0], w1), word(vr[c1][1], w1), sel);
          const uint32_t a2 = __byte_perm(word(vr[c0][2], w0), word(vr[c0][3], w0), sel);
          const uint32_t a3 = __byte_perm(word(vr[c1][2], w1), word(vr[c1][3], w1), sel);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(o[n][2 * q2 + half], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            mma_16816(o[n][2 * q2 + half], a0, a1, a2, a3, pr[n][0], pr[n][1]);
          }
        }
      }
    }
    __syncwarp();  // the warp's ring is idle: its outputs go over it

    // ---- join the warps ----
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = l[n][k];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) {
          s_m[warp][8 * n + 2 * t + k] = m[n][k];
          s_l[warp][8 * n + 2 * t + k] = v;
        }
        if (8 * n + 2 * t + k >= nh) continue;
        float* so = s_o(warp) + (8 * n + 2 * t + k) * HD + 8 * og;
#pragma unroll
        for (int j = 0; j < MT; j += 4) {  // O^T tile j: elements 8 og + j and, 4 (64) further on, of row g + 8
          *reinterpret_cast<float4*>(so + j) = make_float4(o[n][j][k], o[n][j + 1][k], o[n][j + 2][k], o[n][j + 3][k]);
          *reinterpret_cast<float4*>(so + j + (HD == 64 ? 4 : 64)) =
              make_float4(o[n][j][2 + k], o[n][j + 1][2 + k], o[n][j + 2][2 + k], o[n][j + 3][2 + k]);
        }
      }
    }
    __syncthreads();
    const bool whole = lo == 0 && hi == nt;
    float* part = sp.part + (static_cast<int64_t>(2) * me + (first_piece ? 0 : 1)) * (H * (HD + 2));
    if (tid < kAttWarps * H) {  // each warp's factor
      const int w = tid / H, h = tid - w * H;
      float mt = s_m[0][h];
#pragma unroll
      for (int k = 1; k < kAttWarps; ++k) mt = fmaxf(mt, s_m[k][h]);
      s_f[w][h] = s_m[w][h] == -INFINITY ? 0.f : exp2_approx(s_m[w][h] - mt);
      if (w == 0) s_mt[h] = mt;
    }
    __syncthreads();
    for (int e = tid; e < nh * (HD / 4); e += kAttWarps * 32) {  // four elements of a head
      const int h = e / (HD / 4);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float lt = 0.f;
#pragma unroll
      for (int w = 0; w < kAttWarps; ++w) {
        const float4 x = reinterpret_cast<const float4*>(s_o(w))[e];
        const float f = s_f[w][h];
        lt = fmaf(f, s_l[w][h], lt);
        v.x = fmaf(f, x.x, v.x);
        v.y = fmaf(f, x.y, v.y);
        v.z = fmaf(f, x.z, v.z);
        v.w = fmaf(f, x.w, v.w);
      }
      if (whole) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(b) * p.hq + h0) * HD + 4 * e) =
            make_uint2(pack2(v.x * inv, v.y * inv), pack2(v.z * inv, v.w * inv));
        if (p.lse && e % (HD / 4) == 0)
          p.lse[static_cast<int64_t>(b) * p.hq + h0 + h] = (s_mt[h] + log2f(lt)) * 0.6931471805599453f;
      } else {
        reinterpret_cast<float4*>(part + 2 * H)[e] = v;
        if (e % (HD / 4) == 0) {
          part[h] = s_mt[h];
          part[H + h] = lt;
        }
      }
    }
    if (!whole) {
      // the stream's set covers tiles [i0, i0 + nt) of the whole axis; its pieces are CTAs first, first + 1, ...
      const long long i0 = at - lo;
      const int first = static_cast<int>(i0 / share), n = static_cast<int>((i0 + nt - 1) / share) - first + 1;
      const int64_t row = static_cast<int64_t>(b) * p.hq + h0;
      join_pieces<HD, H>(sp, ring, first, i0 > first * share ? 1 : 0, n, me - first, nh,
                         p.out + row * HD, p.lse ? p.lse + row : nullptr);
    }
    tc::fence_proxy_async_smem();
    __syncthreads();  // the rings may be filled again
    at += hi - lo;
    in_b += hi - lo;
    first_piece = false;
    if (in_b == static_cast<long long>(nt) * sp.sets) {
      ++b;
      in_b = 0;
    }
  }
}

// ---------------------------------------------------------------------------
// copy_pages: pool [outer, num_pages, page_bytes] with byte strides; page
// src[i] -> page dst[i] in every outer index.  16 KB a CTA, in one pass: bounded
// by HBM (36000 pages of 16 KB in 178 us, 6.6 TB/s), 2.1 us for a handful.
// ---------------------------------------------------------------------------
struct CopyParams {
  char* pool;
  int64_t outer_stride, page_stride, page_bytes;
  const int *src, *dst;
  int outer, num_pages;
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

// TMA map of a pool's tiles, [head_dim / 64][16 positions][64 elements]: (element, position, 64-element part, head, page).
inline bool pool_map(CUtensorMap* map, const void* base, const PoolStrides& st, int num_pages, int heads,
                     int page_size, int hd) {
  const uint32_t parts = static_cast<uint32_t>(hd / 64);
  const uint64_t dims[5] = {64, static_cast<uint64_t>(page_size), parts, static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(num_pages)};
  const uint64_t strides[4] = {static_cast<uint64_t>(st.tok) * 2, 128, static_cast<uint64_t>(st.head) * 2,
                               static_cast<uint64_t>(st.page) * 2};
  const uint32_t box[5] = {64, kTile, parts, 1, 1};
  return tc::make_map_bf16_sw128(map, base, 5, dims, strides, box);
}

template <int HD, int NT>
int launch_decode(int grid, cudaStream_t st, const CUtensorMap& km, const CUtensorMap& vm, const AttendParams& p,
                  const AttendSplit& sp) {
  constexpr int smem = static_cast<int>(ring_bytes<HD>()) + 1024;
  if (!smem_room<paged_decode_mma_kernel<HD, NT>>(smem)) return SN_ERR_LAUNCH;
  return launch(paged_decode_mma_kernel<HD, NT>, dim3(static_cast<unsigned>(grid)), dim3(kAttWarps * 32), smem, st, true, km,
                vm, p, sp);
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto rows16 = [](const void* base, int64_t a, int64_t b, int64_t c) {
    return sn::aligned16(base) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
  };
  // 16-byte chunks throughout: 12288 tokens of 24 heads of 128 in 27.1 us (5.8 TB/s) against 168 us element by element
  if (head_dim % 16 == 0 && rot_dim % 16 == 0 && head_dim <= 512 && nheads + 2 * nheads_kv <= 65535 && rows16(qkv, ld, 0, 0) && sn::aligned16(q) &&
      rows16(k_pages, k_page_stride, k_head_stride, k_tok_stride) &&
      rows16(v_pages, v_page_stride, v_head_stride, v_tok_stride) && sn::aligned16(cos) && sn::aligned16(sin)) {
    const int warp_heads = sn::kAppendHeads * (32 / (head_dim / 16));
    const dim3 grid(static_cast<unsigned>((tokens + 3) / 4),
                    static_cast<unsigned>((nheads + 2 * nheads_kv + warp_heads - 1) / warp_heads));
    return interleaved ? sn::launch(sn::rotary_paged_append_vec_kernel<true>, grid, dim3(128), 0, st, true, p)
                       : sn::launch(sn::rotary_paged_append_vec_kernel<false>, grid, dim3(128), 0, st, true, p);
  }
  const int64_t blocks = (static_cast<int64_t>(tokens) * (width / 2) + 255) / 256;
  if (blocks > INT32_MAX) return SN_ERR_UNSUPPORTED;
  return sn::launch(sn::rotary_paged_append_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st,
                    true, p);
}

size_t sn_paged_decode_workspace_size(int batch, int nheads, int head_dim) {
  if (batch < 1 || nheads < 1 || head_dim < 1) return 0;
  // the tickets, then two partial results a CTA
  static_assert(4 * sn::kAttGridMax == SN_PAGED_DECODE_COUNTERS);
  return SN_PAGED_DECODE_COUNTERS * sizeof(unsigned) + static_cast<size_t>(2) * sn::kAttGridMax * sn::kAttHeadsMax * (head_dim + 2) * sizeof(float);
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
  if (!sn::aligned16(workspace)) return SN_ERR_MISALIGNED;
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto rows16 = [](const void* base, int64_t a, int64_t b, int64_t c) {
    return sn::aligned16(base) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
  };
  // whole tiles in a page and 16-byte rows: the tensor-core form (measured beside it: 64 ragged streams of up to 5000
  // positions 2060 -> 67 us, one stream of 257 positions 56 -> 5.8 us); anything else goes row by row
  if ((head_dim == 64 || head_dim == 128) && page_size % sn::kTile == 0 && sn::aligned16(out) &&
      rows16(q, q_batch_stride, q_head_stride, 0) && rows16(k_pages, k_page_stride, k_head_stride, k_tok_stride) &&
      rows16(v_pages, v_page_stride, v_head_stride, v_tok_stride)) {
    sn::AttendSplit sp;
    sp.group = nheads / nheads_kv;
    sp.sets_per_kv = (sp.group + sn::kAttHeadsMax - 1) / sn::kAttHeadsMax;
    sp.heads_per_set = (sp.group + sp.sets_per_kv - 1) / sp.sets_per_kv;
    sp.sets = nheads_kv * sp.sets_per_kv;
    sp.ticket = static_cast<unsigned*>(workspace);
    sp.part = reinterpret_cast<float*>(sp.ticket + SN_PAGED_DECODE_COUNTERS);
    CUtensorMap km, vm;
    if (!sn::pool_map(&km, k_pages, p.ks, num_pages, nheads_kv, page_size, head_dim) ||
        !sn::pool_map(&vm, v_pages, p.vs, num_pages, nheads_kv, page_size, head_dim))
      return SN_ERR_LAUNCH;
    const bool two = sp.heads_per_set > 8;  // an operand takes 8 heads: two of them read a group's K and V once
    // two CTAs an SM, and no more than the page tables have tiles for
    const int64_t tiles = static_cast<int64_t>(max_pages) * (page_size / sn::kTile) * batch * sp.sets;
    const int64_t most = (tiles + sn::kAttWarps - 1) / sn::kAttWarps;
    sp.slots = static_cast<int>(std::min<int64_t>(std::min(2 * sn::sm_count(), sn::kAttGridMax), most));
    // and one for every (stream, head set) where they are short (4096 at most)
    const int grid = static_cast<int>(std::max<int64_t>(sp.slots, std::min<int64_t>(static_cast<int64_t>(batch) * sp.sets, 4096)));
    if (head_dim == 64)
      return two ? sn::launch_decode<64, 2>(grid, st, km, vm, p, sp) : sn::launch_decode<64, 1>(grid, st, km, vm, p, sp);
    return two ? sn::launch_decode<128, 2>(grid, st, km, vm, p, sp) : sn::launch_decode<128, 1>(grid, st, km, vm, p, sp);
  }
  return sn::launch(sn::paged_decode_rows_kernel, dim3(static_cast<unsigned>(batch * nheads)), dim3(128), 0, st,
                    true, p);
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
  const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(outer), static_cast<unsigned>(parts));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = sn::aligned16(pool) && (outer == 1 || outer_stride_bytes % 16 == 0) &&
                    page_stride_bytes % 16 == 0 && page_bytes % 16 == 0;
  // 36000 pages of 16 KB: 179 us by 16 bytes, 983 us byte by byte
  return wide ? sn::launch(sn::copy_pages_kernel<uint4>, grid, dim3(256), 0, st, true, p)
              : sn::launch(sn::copy_pages_kernel<char>, grid, dim3(256), 0, st, true, p);
}

}  // extern "C"
