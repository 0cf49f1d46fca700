// Mamba2 over prompts (bf16 tensors, fp32 arithmetic): the causal convolution
// and the selective state space scan of ragged prompts packed along the
// token axis, from the in_proj rows [z | x B C | dt].
//
//   xBC_t = SiLU(bias + sum_k w[d, k] u_{t - W + 1 + k}[d])
//   dt_t  = softplus(dt_raw_t + dt_bias)                      per head
//   S_t   = exp(dt_t A) S_{t-1} + dt_t x_t (x) B_t            [headdim, d_state]
//   y_t   = S_t C_t + D x_t                                   (* SiLU(z_t))
//
// conv_state and ssm_state are read as each prompt's state before its first
// token and left as the state after its last one, in the layouts of the
// single-token kernels.  Prompt i holds tokens cu[i] .. cu[i + 1] - 1; the
// offsets are on the device, so every CTA finds its own prompt.  Offsets out
// of [0, tokens] or falling are clamped and recorded as
// SN_ERR_INVALID_ARGUMENT in the status word.
#include "tc.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

namespace sn {
namespace {

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

struct Prompts {
  const int* cu;  // [batch + 1], or null: one prompt of all tokens
  int batch, tokens;
};
struct PromptBlock {
  int seq;     // -1: no such block
  int start;   // first token of the prompt
  int len;     // tokens of the prompt
  int block;   // index of the block within the prompt
  int blocks;  // blocks of the prompt
};

// Tokens [s, e) of prompt b0 + lane (empty past the last), called by whole
// warps for b0 = 0, 32, ... in turn with `upto` = 0 before the first.  Offsets
// are clamped and never fall, so that prompts cannot overlap whatever the
// tensor holds; true when they had to be changed.
__device__ __forceinline__ bool prompt_bounds(const Prompts& p, int b0, int& upto, int& s, int& e) {
  const int lane = threadIdx.x & 31, b = b0 + lane;
  const bool on = b < p.batch;
  const int s0 = on && p.cu ? p.cu[b] : 0, e0 = !on ? 0 : p.cu ? p.cu[b + 1] : p.tokens;
  s = max(min(max(s0, 0), p.tokens), upto);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s = max(s, v);
  }
  e = max(min(e0, p.tokens), s);
  upto = __shfl_sync(0xffffffffu, e, 31);
  return on && (s != s0 || e != e0);
}

// The index-th block, where every prompt is cut into blocks of `rows` tokens
// (at least `least` of them, so that an empty prompt still has one where its
// state has to be handled).  Called by whole warps; every lane gets the answer.
__device__ __forceinline__ PromptBlock find_block(const Prompts& p, int rows, int least, int index) {
  const int lane = threadIdx.x & 31;
  int before = 0, last = 0;
  if (p.batch == 1 && !p.cu) {
    const int n = max((p.tokens + rows - 1) / rows, least);
    return {index < n ? 0 : -1, 0, p.tokens, index, n};
  }
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int s, e;
    if (prompt_bounds(p, b0, last, s, e)) record_status(SN_ERR_INVALID_ARGUMENT);
    const int n = b0 + lane < p.batch ? max((e - s + rows - 1) / rows, least) : 0;
    int upto = n;  // inclusive scan over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const int at = index - before;
    const unsigned here = __ballot_sync(0xffffffffu, at < upto && n > 0);
    if (here) {
      const int l = __ffs(here) - 1;
      PromptBlock r;
      r.seq = b0 + l;
      r.start = __shfl_sync(0xffffffffu, s, l);
      r.len = __shfl_sync(0xffffffffu, e, l) - r.start;
      r.blocks = __shfl_sync(0xffffffffu, n, l);
      r.block = at - (__shfl_sync(0xffffffffu, upto, l) - r.blocks);
      return r;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return {-1, 0, 0, 0, 0};
}

struct PromptParams {
  const __nv_bfloat16* zx;  // [tokens, ld]
  int64_t ld;
  __nv_bfloat16* conv_state;  // [batch, conv_dim, W]
  const __nv_bfloat16* w;     // [conv_dim, W]
  const __nv_bfloat16* bias;  // [conv_dim] or null
  __nv_bfloat16* ssm_state;   // [batch, nh, hd, ds]
  const float* A;             // [nh]
  const __nv_bfloat16* D;     // [nh] or null
  const __nv_bfloat16* dt_bias;  // [nh] or null
  __nv_bfloat16* y;           // [tokens, nh, hd]
  __nv_bfloat16* xbc;         // workspace [tokens, conv_dim]
  Prompts prompts;
  int di, gds, ds, ng, nh, hd, hpg, W, gate;
};

// Zeros in the rows of y before the first prompt and after the last (offsets clamped as above; where they fall, a row of a
// prompt may be among them, and the scan, a later launch, writes it), shared by `count` CTAs of which this is the
// index-th.  Out of line, since a call with such rows is the exception.
__device__ __noinline__ void zero_rows(__nv_bfloat16* y, int n, int before, int after, int tokens, int index, int count) {
  const int rows = before + tokens - after;
  for (int r = index; r < rows; r += count) {
    __nv_bfloat16* row = y + static_cast<int64_t>(r < before ? r : after + r - before) * n;
    for (int i = threadIdx.x; i < n; i += blockDim.x) row[i] = __float2bfloat16_rn(0.f);
  }
}
__device__ __forceinline__ void zero_outside(const PromptParams& p, int index, int count) {
  if (!p.prompts.cu) return;
  const int tokens = p.prompts.tokens;
  const int before = min(max(p.prompts.cu[0], 0), tokens), after = min(max(p.prompts.cu[p.prompts.batch], 0), tokens);
  if (before > 0 || after < tokens) zero_rows(p.y, p.di, before, after, tokens, index, count);
}

// ---------------------------------------------------------------------------
// Convolution: one thread per channel and block of kConvRows tokens.  The
// thread of a prompt's first block also moves the channel's state on (it is
// the only one that reads it).
// ---------------------------------------------------------------------------
constexpr int kConvRows = 32;
constexpr int kMaxConvWidth = 8;

__global__ void __launch_bounds__(256) prompt_conv_kernel(const PromptParams p) {
  pdl_launch_dependents();
  pdl_wait();
  zero_outside(p, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
  const PromptBlock pb = find_block(p.prompts, kConvRows, 1, blockIdx.y);
  if (pb.seq < 0) return;
  const int conv_dim = p.di + 2 * p.gds;
  const int d = blockIdx.x * 256 + threadIdx.x;
  if (d >= conv_dim) return;
  const int W = p.W;
  const __nv_bfloat16* u = p.zx + static_cast<int64_t>(pb.start) * p.ld + p.di + d;  // u[t * ld]
  __nv_bfloat16* st = p.conv_state + (static_cast<int64_t>(pb.seq) * conv_dim + d) * W;
  float w[kMaxConvWidth], h[kMaxConvWidth];  // h: the last W inputs, newest last
#pragma unroll
  for (int k = 0; k < kMaxConvWidth; ++k) w[k] = k < W ? __bfloat162float(p.w[static_cast<int64_t>(d) * W + k]) : 0.f;
  const float bias = p.bias ? __bfloat162float(p.bias[d]) : 0.f;
  const int t0 = pb.block * kConvRows, t1 = min(t0 + kConvRows, pb.len);
#pragma unroll
  for (int k = 0; k < kMaxConvWidth; ++k) {
    const int t = t0 - W + k;
    h[k] = k >= W ? 0.f : __bfloat162float(t >= 0 ? u[t * p.ld] : st[k + t0]);  // input t < 0 is state column W + t
  }
  if (t0 == 0) {  // the state after the prompt: the last W inputs
    __nv_bfloat16 moved[kMaxConvWidth];
#pragma unroll
    for (int k = 0; k < kMaxConvWidth; ++k) {
      const int t = pb.len - W + k;
      if (k < W) moved[k] = t >= 0 ? u[t * p.ld] : st[W + t];
    }
#pragma unroll
    for (int k = 0; k < kMaxConvWidth; ++k)
      if (k < W) st[k] = moved[k];
  }
  for (int t = t0; t < t1; ++t) {
    float acc = bias;
#pragma unroll
    for (int k = 0; k < kMaxConvWidth; ++k) {
      if (k < W) {
        h[k] = k + 1 < W ? h[k + 1 < kMaxConvWidth ? k + 1 : k] : __bfloat162float(u[t * p.ld]);
        acc = fmaf(h[k], w[k], acc);
      }
    }
    p.xbc[static_cast<int64_t>(pb.start + t) * conv_dim + d] = __float2bfloat16_rn(silu(acc));
  }
}

// ---------------------------------------------------------------------------
// Scan, token by token (any headdim, d_state <= 256): 16 lanes per (prompt,
// head, headdim row) hold the row's state in fp32 registers, lane l the
// elements l, l + 16, ...  Bounded by the chain of a token (1.7 us).
// ---------------------------------------------------------------------------
constexpr int kScanPerLane = 16;

__global__ void __launch_bounds__(256) prompt_scan_rows_kernel(const PromptParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int l16 = threadIdx.x & 15;
  const int64_t rows = static_cast<int64_t>(p.prompts.batch) * p.nh * p.hd;
  const int64_t row_ = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 4;
  const bool valid = row_ < rows;
  const int64_t row = valid ? row_ : 0;
  const int b = static_cast<int>(row / (static_cast<int64_t>(p.nh) * p.hd));
  const int hp = static_cast<int>(row - static_cast<int64_t>(b) * p.nh * p.hd);
  const int h = hp / p.hd, g = h / p.hpg;
  // tokens [start, end), as prompt_bounds has them: no offset below one before it
  int start = 0;
  const int e0 = p.prompts.cu ? p.prompts.cu[b + 1] : p.prompts.tokens;
  if (p.prompts.cu)
    for (int i = l16; i <= b; i += 16) start = max(start, p.prompts.cu[i]);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) start = max(start, __shfl_xor_sync(0xffffffffu, start, o));
  start = min(start, p.prompts.tokens);
  const int end = min(max(e0, start), p.prompts.tokens);
  const int conv_dim = p.di + 2 * p.gds;
  __nv_bfloat16* st = p.ssm_state + row * p.ds;
  float s[kScanPerLane];
#pragma unroll
  for (int i = 0; i < kScanPerLane; ++i) {
    const int n = l16 + 16 * i;
    s[i] = n < p.ds ? __bfloat162float(st[n]) : 0.f;
  }
  const float a = p.A[h], dtb = p.dt_bias ? __bfloat162float(p.dt_bias[h]) : 0.f;
  const float dv = p.D ? __bfloat162float(p.D[h]) : 0.f;
  const int64_t dt_at = 2 * static_cast<int64_t>(p.di) + 2 * p.gds + h;
  // the two rows of a warp may belong to prompts of different lengths: both halves run to the longer one
  const int steps = max(end - start, __shfl_xor_sync(0xffffffffu, end - start, 16));
  for (int i = 0; i < steps; ++i) {
    const bool on = start + i < end;
    const int64_t t = on ? start + i : start;
    float acc = 0.f, x = 0.f;
    if (on) {
      const __nv_bfloat16* r = p.xbc + t * conv_dim;
      x = __bfloat162float(r[hp]);
      float dt = __bfloat162float(p.zx[t * p.ld + dt_at]) + dtb;
      dt = dt <= 20.f ? log1pf(expf(dt)) : dt;
      const float decay = expf(dt * a), dtx = dt * x;
      const __nv_bfloat16* Br = r + p.di + static_cast<int64_t>(g) * p.ds;
      const __nv_bfloat16* Cr = Br + p.gds;
#pragma unroll
      for (int k = 0; k < kScanPerLane; ++k) {
        const int n = l16 + 16 * k;
        if (n < p.ds) {
          s[k] = fmaf(s[k], decay, dtx * __bfloat162float(Br[n]));
          acc = fmaf(s[k], __bfloat162float(Cr[n]), acc);
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (on && valid && l16 == 0) {
      float out = fmaf(x, dv, acc);
      if (p.gate) out *= silu(__bfloat162float(p.zx[t * p.ld + hp]));
      p.y[t * p.di + hp] = __float2bfloat16_rn(out);
    }
  }
  if (valid) {
#pragma unroll
    for (int i = 0; i < kScanPerLane; ++i) {
      const int n = l16 + 16 * i;
      if (n < p.ds) st[n] = __float2bfloat16_rn(s[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// The tensor-core form: headdim 64, d_state 128, convolution widths 2 to 4.
//
// Mathematics.  In a chunk of L = 128 tokens, with a_i = sum_{k <= i} dt_k A
// counted from the chunk's start,
//   Y = M X + diag(exp a_i) C S_in,   M_ij = (C B^T)_ij exp(a_i - a_j) dt_j  (j <= i)
//   S_out = exp(a_L) S_in + sum_j exp(a_L - a_j) dt_j B_j (x) x_j
// so a chunk is four products of 128 rows: C B^T, shared by the heads of a
// group, then C S, M X and B^T (w x) of each head; only the states go from
// chunk to chunk.  A long prompt is cut into segments of whole chunks: one
// launch finds each segment's own contribution to the state, the next joins
// those before a segment and does its outputs.
//
// Numbers.  The products are kind::f16 with fp32 accumulators.  Operands in
// fp16 (11 significant bits) instead of bf16 (8) keep their roundings below
// that of the bf16 results.  fp16 has all of its bits from 2^-14 to 2^16 only, so
// exact powers of two put the largest value of what shares one near the top:
//   x      a head's 128 tokens of a chunk, to below 2^14 (its weights in the
//          state are below 2): all bits to 2^-27 of the largest
//   B, C   a group's 128 tokens by 128 states, likewise; then a token's row of
//          C again, by up to 2^15, where its largest is below 1/8 of that
//   M      (C B^T)_ij < 2^35, dt_j below 2 by the chunk's largest, 2^-21: below
//          2^15, and about 2^5 where all are of one size.  B and dt of a score
//          may be 2^-16 together of their largest, and C 2^-15 besides, before
//          it loses bits
//   S      by a bound carried along with it, to below 2^14
// Nothing overflows; what lies further below is rounded to 2^-25 in those units
// (the rows' powers of two cost 5 us of 260 and 0.5 of 33 below).  States and
// sums stay in fp32.  Causality is a zero in M, so an infinity or NaN of a token
// reaches the earlier tokens of its own chunk too (and, through the state, all
// later ones); other prompts never share a chunk with it.  A is taken to be
// negative (it is -exp(A_log)), so that no decay exceeds 1.
//
// Layout.  The convolution writes its results as the shared-memory images the
// products read (128-byte swizzle, 128 tokens by 64 channels, 16 KB), padded
// with zero rows to whole chunks of a prompt, so a chunk's operands come in
// three bulk copies and no product sees another prompt's tokens.
//
// Measured, one prompt of 16384 tokens, 64 heads, one group (142.6 MB of rows
// and 134.2 MB of outputs, 43 us at the copy bandwidth of 6.44 TB/s): 260 us,
// of them 64 the convolution, 43 the states, 153 the outputs.  The tiles of x,
// B and C (142 MB) are written by the first and read by the other two.
// ---------------------------------------------------------------------------
constexpr int kChunk = 128;
constexpr int kTileBytes = kChunk * 128;  // 128 tokens x 64 channels of fp16
constexpr int kRowTileBytes = 2 * kTileBytes + kChunk;  // two of them and a byte for each token
constexpr int kTop = 14;                    // x, B and C as operands are below 2^14
constexpr float kMScale = 1.f / (1 << 21);  // of M: 128 2^14 2^14 2 to 2^15
constexpr float kLog2e = 1.4426950408889634f;

struct ChunkWork {  // workspace arrays; chunks are counted over all prompts
  unsigned char* x;  // [chunks][nh] tiles
  unsigned char* b;  // [chunks][ng] pairs of tiles (128 states)
  unsigned char* c;  // [chunks][ng] pairs of tiles, then the power of two of each token's row, as the exponent of a float
  float* cum;        // [chunks][nh][128] cumulative dt A / ln 2
  float* dt;         // [chunks][nh][128], 0 past the prompt's end
  float2* meta;      // [chunks][nh] largest dt; sum of dt exp(a_L - a_j)
  float* scale;      // [chunks][nh + 2 ng] power of two of each head's x, each group's B and C: value / operand
  float* state;      // [slots][nh][64][128] see prompt_scan_mma_kernel
  float* total;      // [slots][nh] sum of dt A / ln 2 over a segment
  int xblocks, blocks;  // 128-channel blocks of x; of x, B and C together
  int seg;              // chunks a segment
};

// The power of two at or below |v| (at least 2^-least); 1 for 0, infinities and NaN.
__device__ __forceinline__ float pow2_floor(float v, uint32_t least = 24) {
  const uint32_t e = (__float_as_uint(v) >> 23) & 255u;
  return e == 0 || e == 255 ? 1.f : __uint_as_float(max(e, 127u - least) << 23);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 products in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t v) { return make_float2(bf16lo(v), bf16hi(v)); }
__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / v of a power of two, exactly.
__device__ __forceinline__ float rcp_pow2(float v) { return __uint_as_float((254u << 23) - __float_as_uint(v)); }
__device__ __forceinline__ float2 silu2(float2 v) {
  const float2 z = mul2(v, splat(-kLog2e));
  return mul2(v, make_float2(rcp_approx(1.f + exp2_approx(z.x)), rcp_approx(1.f + exp2_approx(z.y))));
}

// dt and decays of 16 heads of one chunk.
constexpr int kDtHeads = 16;
__device__ __forceinline__ void prompt_dt(const PromptParams& p, const ChunkWork& wk, const PromptBlock& pb, int64_t chunk, int h0,
                                          float* s_dt) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t0 = pb.block * kChunk;
  const int r = tid >> 1, e0 = (tid & 1) * 8;  // token; the first of 8 heads
  const int64_t at = 2 * static_cast<int64_t>(p.di) + 2 * p.gds + h0 + e0;
  const __nv_bfloat16* src = p.zx + (pb.start + t0 + r) * p.ld + at;
  const bool live = t0 + r < pb.len;
  float v[8];
  if (live && h0 + e0 + 8 <= p.nh && (at & 7) == 0) {
    const uint4 u = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = bf16lo(w[k]);
      v[2 * k + 1] = bf16hi(w[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = live && h0 + e0 + k < p.nh ? __bfloat162float(src[k]) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (p.dt_bias && h0 + e0 + k < p.nh) v[k] += __bfloat162float(p.dt_bias[h0 + e0 + k]);
    v[k] = v[k] <= 20.f ? log1pf(__expf(v[k])) : v[k];
    s_dt[(e0 + k) * 129 + r] = live ? v[k] : 0.f;
  }
  __syncthreads();
  for (int h = warp; h < kDtHeads && h0 + h < p.nh; h += 8) {
    const float a2 = p.A[h0 + h] * kLog2e;
    float c[4], run = 0.f, top = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = s_dt[h * 129 + lane * 4 + k];
      run = fmaf(v[k], a2, run);
      c[k] = run;
      top = fmaxf(top, v[k]);
    }
    float upto = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    const float before = upto - run, all = __shfl_sync(0xffffffffu, upto, 31);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] += before;
      sum = fmaf(v[k], exp2_approx(all - c[k]), sum);
    }
    if (lane == 31) c[3] = all;  // the state's decay and the last token's are the same number
    sum = warp_sum(sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int64_t row = chunk * p.nh + h0 + h;
    reinterpret_cast<float4*>(wk.cum + row * kChunk)[lane] = make_float4(c[0], c[1], c[2], c[3]);
    reinterpret_cast<float4*>(wk.dt + row * kChunk)[lane] = make_float4(v[0], v[1], v[2], v[3]);
    if (lane == 0) wk.meta[row] = make_float2(top, sum);
  }
}

// Column k of 8 channels' convolution state [8][W].
template <int W>
__device__ __forceinline__ uint4 state_column(const __nv_bfloat16* st, int k) {
  uint32_t v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    v[c] = static_cast<uint32_t>(__bfloat16_as_ushort(st[2 * c * W + k])) |
           static_cast<uint32_t>(__bfloat16_as_ushort(st[(2 * c + 1) * W + k])) << 16;
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// 16 bytes from global to shared memory, or 16 zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// One 128-channel block of one chunk (blockIdx.x < blocks), or 16 heads' dt
// and decays.  The inputs come through shared memory; a thread has two
// channels of 32 tokens, a warp the 64 channels of a tile.  kMany: in one run
// of tokens and four CTAs an SM (64 registers); else in every fourth 8 tokens,
// so that few tokens are spread over the warps, and three.
// Inputs read and tiles written once (252 MB of HBM traffic for 16384 tokens,
// 39 us; the special functions of a SiLU 32 us): measured 64, issue slots 72%
// busy.  16-byte loads to registers, 8 channels of 8 tokens a thread, took 16%
// fewer instructions but 128 registers, so 15 warps an SM where there are 30 (87
// us for 62).  What only C's rows need is in every block's code and takes 2 of
// the 64; a copy of the code for C alone took more.
template <int W, bool kMany>
__global__ void __launch_bounds__(256, kMany ? 4 : 3) prompt_conv_tile_kernel(const PromptParams p, const ChunkWork wk) {
  __shared__ __align__(16) unsigned char s_rows[(kChunk + W - 1) * 256];  // tokens t0 - W + 1 ..
  __shared__ float s_max[8], s_row[2][kChunk];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blk = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  // by the CTAs of dt: all of them would take 1 us of 258 longer over 16384 tokens
  if (blk >= wk.blocks)
    zero_outside(p, blockIdx.y * (gridDim.x - wk.blocks) + blk - wk.blocks, (gridDim.x - wk.blocks) * gridDim.y);
  const PromptBlock pb = find_block(p.prompts, kChunk, 0, blockIdx.y);
  if (pb.seq < 0) return;
  const int t0 = pb.block * kChunk;
  const int64_t chunk = blockIdx.y;
  if (blk >= wk.blocks) {
    prompt_dt(p, wk, pb, chunk, (blk - wk.blocks) * kDtHeads, reinterpret_cast<float*>(s_rows));
    return;
  }
  const int d0 = blk < wk.xblocks ? blk * 128 : p.di + (blk - wk.xblocks) * 128;  // channel of the convolution
  const int wide = blk < wk.xblocks ? min(128, p.di - d0) : 128;                   // 64 or 128 of them
  const int left = pb.len - t0;                                                    // tokens from here on
  const __nv_bfloat16* u = p.zx + (static_cast<int64_t>(pb.start) + t0) * p.ld + p.di + d0;
  // first and last inputs of the prompt: 8 channels a thread of the first chunk's first 16, which are the only ones that
  // read or write these channels' state
  const bool edge = t0 == 0 && tid < 16 && tid * 8 < wide;
  __nv_bfloat16* st = p.conv_state + (static_cast<int64_t>(pb.seq) * (p.di + 2 * p.gds) + d0 + tid * 8) * W;  // [8][W]
  {
    const int c = tid & 15;
    for (int k = tid >> 4; k < kChunk + W - 1; k += 16) {
      const int t = k - (W - 1);
      const bool in = t < left && c * 8 < wide;
      if (t0 + t >= 0) copy16(smem_u32(s_rows) + k * 256 + c * 16, in ? u + t * p.ld + c * 8 : u, in);
    }
    if (edge) {  // inputs before the prompt are the state's columns 1 .. W - 1
#pragma unroll
      for (int k = 0; k < W - 1; ++k) *reinterpret_cast<uint4*>(s_rows + k * 256 + tid * 16) = state_column<W>(st, k + 1);
    }
  }
  constexpr int kNext = kMany ? 8 : 32;                             // from a thread's 8 tokens to its next
  const int half = warp & 1, r0 = (warp >> 1) * (kMany ? 32 : 8);  // tile and first tokens of the warp
  const bool on = half * 64 < wide, of_x = blk < wk.xblocks, of_c = blk >= wk.xblocks + p.ng;
  float2 w[W], bias = make_float2(0.f, 0.f);
  if (on) {
    const int d = d0 + half * 64 + 2 * lane;
    uint32_t wu[W];  // taps of d, then of d + 1
#pragma unroll
    for (int k = 0; k < W; ++k) wu[k] = reinterpret_cast<const uint32_t*>(p.w + static_cast<int64_t>(d) * W)[k];
    auto tap = [&](int e) { return e & 1 ? bf16hi(wu[e / 2]) : bf16lo(wu[e / 2]); };
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = make_float2(tap(k), tap(W + k));
    if (p.bias) bias = unpack_bf16(*reinterpret_cast<const uint32_t*>(p.bias + d));
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  float top = 0.f;
  uint32_t out[4][8];  // [8 tokens][token], fp16 over the 8 tokens' own power of two, below 2^13
  float own[4];
  if (on) {
    const unsigned char* in = s_rows + r0 * 256 + half * 128 + lane * 4;
    float2 past[W - 1];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      own[g] = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) out[g][r] = 0;
      if (r0 + kNext * g >= left) continue;
      if (!kMany || g == 0) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) past[k] = unpack_bf16(*reinterpret_cast<const uint32_t*>(in + (kNext * g + k) * 256));
      }
      float2 o[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float2 v = unpack_bf16(*reinterpret_cast<const uint32_t*>(in + (W - 1 + kNext * g + r) * 256));
        o[r] = bias;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) o[r] = fma2(past[k], w[k], o[r]);
        o[r] = silu2(fma2(v, w[W - 1], o[r]));
#pragma unroll
        for (int k = 0; k < W - 2; ++k) past[k] = past[k + 1];
        past[W - 2] = v;
      }
      if (left < kChunk) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r0 + kNext * g + r >= left) o[r] = make_float2(0.f, 0.f);
      }
      if (of_c) {  // the largest of each token, over the warp's states
        unsigned mine = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(o[r].x), fabsf(o[r].y))));
          mine = lane == r ? m : mine;
        }
        if (lane < 8) s_row[half][r0 + kNext * g + lane] = __uint_as_float(mine);
      }
      float most = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) most = fmaxf(most, fmaxf(fabsf(o[r].x), fabsf(o[r].y)));
      top = fmaxf(top, most);
      own[g] = most == 0.f ? 0.f : pow2_floor(most);
      const float2 inv = splat(most == 0.f ? 1.f : 4096.f * rcp_pow2(own[g]));
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float2 v = mul2(o[r], inv);
        out[g][r] = pack_f16(v.x, v.y);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
  // the largest of this head of x, or of the block of B or C
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (!of_x || (k & 1) == half) top = fmaxf(top, s_max[k]);
  const float sc = pow2_floor(top);
  // Rows of C far below the block's largest get a power of two of their own (`row`, of the token of this lane among the
  // warp's 32); the block's is then stored negative.  Not the others, so that chunks of even tokens, the usual ones, cost
  // the scan nothing (all rows: 262 for 258 us).
  auto quiet = [&](int t) {
    const float m = fmaxf(s_row[0][t], s_row[1][t]) * rcp_pow2(sc);
    return t < left && m > 0.f && m < 1.f / 8 ? pow2_floor(m, 15) : 1.f;
  };
  float row = 1.f;
  bool any = false;
  if (of_c) {
    const int t = r0 + kNext * (lane >> 3) + (lane & 7);
    row = quiet(t);
    if (half == 0) wk.c[(chunk * p.ng + blk - wk.xblocks - p.ng) * kRowTileBytes + 2 * kTileBytes + t] = __float_as_uint(row) >> 23;
    if (warp == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) any |= quiet(lane + 32 * k) < 1.f;
      any = __any_sync(0xffffffffu, any);
    }
  }
  if (lane == 0 && on && warp < (of_x ? 2 : 1))
    wk.scale[chunk * (p.nh + 2 * p.ng) + (of_x ? blk * 2 + half : p.nh + blk - wk.xblocks)] =
        sc * (any ? -1.f / (1 << (kTop - 1)) : 1.f / (1 << (kTop - 1)));
  if (on) {
    unsigned char* tile;
    if (of_x) {
      tile = wk.x + (chunk * p.nh + blk * 2 + half) * kTileBytes;
    } else {
      const int g = blk - wk.xblocks;
      tile = of_c ? wk.c + (chunk * p.ng + g - p.ng) * kRowTileBytes : wk.b + (chunk * p.ng + g) * 2 * kTileBytes;
      tile += half * kTileBytes;
    }
    tile += r0 * 128 + (lane & 3) * 4;
    const float up = rcp_pow2(sc) * ((1 << (kTop - 1)) / 4096.f);
    const bool rows = __any_sync(0xffffffffu, row < 1.f);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      // to the block's power of two: exact where the result has all of its bits
      float to = own[g] * up;
      if (to < 1.f / (1 << 14)) {  // of fp16's own range below 2^-24: in two steps
        to *= 1 << 12;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&out[g][r]), __float2half2_rn(1.f / (1 << 12)));
          out[g][r] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      const __half2 f = __float2half2_rn(to);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&out[g][r]), f);
        if (rows) v = __hmul2(v, __float2half2_rn(rcp_pow2(__shfl_sync(0xffffffffu, row, 8 * g + r))));
        *reinterpret_cast<uint32_t*>(tile + (kNext * g + r) * 128 + (((lane >> 2) ^ r) << 4)) =
            *reinterpret_cast<const uint32_t*>(&v);
      }
    }
  }
  if (edge) {  // the state after the prompt, its last W inputs
    uint4 col[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int t = pb.len - W + k;  // < 0: the old state's column W + t
      col[k] = t >= 0 ? *reinterpret_cast<const uint4*>(u + t * p.ld + tid * 8) : state_column<W>(st, W + t);
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const uint32_t v = c / 2 == 0 ? col[k].x : c / 2 == 1 ? col[k].y : c / 2 == 2 ? col[k].z : col[k].w;
        st[c * W + k] = __ushort_as_bfloat16(static_cast<unsigned short>(c & 1 ? v >> 16 : v & 0xFFFFu));
      }
    }
  }
}

// ---- tcgen05 pieces of this kernel ----
// Operand whose rows run along the contraction (K): 64 elements of the other
// axis a 128-byte row, 8-row groups 1024 bytes apart, the next 64 elements of
// that axis `next` bytes on.
__device__ __forceinline__ uint64_t desc_k_rows(uint32_t addr, uint32_t next) {
  uint64_t d = 0;
  d |= (static_cast<uint64_t>(addr) >> 4) & 0x3FFFull;
  d |= static_cast<uint64_t>(next >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}
// kind::f16, fp16 operands, fp32 accumulator; a_k_rows / b_k_rows: the operand is laid out as above.
constexpr uint32_t idesc_f16(int M, int N, bool a_k_rows, bool b_k_rows) {
  return (1u << 4) | (a_k_rows ? 1u << 15 : 0u) | (b_k_rows ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
// The same product with A in tensor memory (two fp16 a column).
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  uint32_t lo[16], hi[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    lo[i] = __float_as_uint(v[i]);
    hi[i] = __float_as_uint(v[16 + i]);
  }
  tmem_st16(taddr, lo);
  tmem_st16(taddr + 16, hi);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
// The power of two whose exponent is the byte at a.
__device__ __forceinline__ float lds_pow2(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
  return __uint_as_float(r << 23);
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

struct Segment {
  int seq, start, len, index, count;  // prompt, its tokens; segment of it, of how many
  int chunk0;                         // the prompt's first chunk, over all prompts
  int slot0;                          // its first state slot (prompts of several segments have one a segment)
};
__device__ __forceinline__ Segment find_segment(const Prompts& p, int seg, int index) {
  const int lane = threadIdx.x & 31;
  if (p.batch == 1) {
    const int s = min(max(p.cu ? p.cu[0] : 0, 0), p.tokens), e = max(min(p.cu ? p.cu[1] : p.tokens, p.tokens), s);
    const int n = ((e - s + kChunk - 1) / kChunk + seg - 1) / seg;
    if (index >= n) return {-1, 0, 0, 0, 0, 0, 0};
    return {0, s, e - s, index, n, 0, 0};
  }
  int before = 0, chunks = 0, slots = 0, last = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int s, e;
    prompt_bounds(p, b0, last, s, e);
    const int nc = (e - s + kChunk - 1) / kChunk;
    const int n = (nc + seg - 1) / seg, ns = n > 1 ? n : 0;
    int u = n, uc = nc, us = ns;  // inclusive scans
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, u, o), vc = __shfl_up_sync(0xffffffffu, uc, o);
      const int vs = __shfl_up_sync(0xffffffffu, us, o);
      if (lane >= o) {
        u += v;
        uc += vc;
        us += vs;
      }
    }
    const unsigned here = __ballot_sync(0xffffffffu, index - before < u && n > 0);
    if (here) {
      const int l = __ffs(here) - 1;
      Segment r;
      r.seq = b0 + l;
      r.start = __shfl_sync(0xffffffffu, s, l);
      r.len = __shfl_sync(0xffffffffu, e, l) - r.start;
      r.count = __shfl_sync(0xffffffffu, n, l);
      r.index = index - before - (__shfl_sync(0xffffffffu, u, l) - r.count);
      r.chunk0 = chunks + __shfl_sync(0xffffffffu, uc - nc, l);
      r.slot0 = slots + __shfl_sync(0xffffffffu, us - ns, l);
      return r;
    }
    before += __shfl_sync(0xffffffffu, u, 31);
    chunks += __shfl_sync(0xffffffffu, uc, 31);
    slots += __shfl_sync(0xffffffffu, us, 31);
  }
  return {-1, 0, 0, 0, 0, 0, 0};
}

constexpr int kScanThreads = 512;
// What both kernels of the scan start with: their heads (a pair within a
// group), segment and chunks, and a place on a 1024-byte boundary.
struct ScanWork {
  Segment sg;
  int g, h0, heads, c0, chunks;
};
__device__ __forceinline__ ScanWork scan_work(const PromptParams& p, const ChunkWork& wk) {
  ScanWork r;
  const int ppg = (p.hpg + 1) / 2;
  r.g = blockIdx.x / ppg;
  r.h0 = r.g * p.hpg + (blockIdx.x - r.g * ppg) * 2;
  r.heads = min(2, (r.g + 1) * p.hpg - r.h0);
  r.sg = find_segment(p.prompts, wk.seg, blockIdx.y);
  r.c0 = r.sg.index * wk.seg;
  r.chunks = min(wk.seg, (r.sg.len + kChunk - 1) / kChunk - r.c0);
  return r;
}
__device__ __forceinline__ unsigned char* aligned_smem(unsigned char* raw) {
  const uint32_t pad = (1024u - (smem_u32(raw) & 1023u)) & 1023u;
  if (pad > 384) {  // does not happen: dynamic shared memory starts on a 1024-byte boundary
    record_status(SN_ERR_MISALIGNED);
    return nullptr;
  }
  return raw + pad;
}

// ---------------------------------------------------------------------------
// The states of segments.  From the last chunk of a segment backwards every
// token's weight to the segment's end is known as it comes, so the whole
// segment is one accumulation S += B^T (w x) in tensor memory, with nothing
// to wait for between chunks: 16 warps scale x in place, a 17th copies and
// issues.  The segment's state from nothing goes to slot index + 1 of the
// prompt; the first segment's starts from the prompt's state, which itself
// goes to slot 0 (the last segment's CTAs of the next launch overwrite it).
// The last segment has nothing to do.  Measured: 43 us for 96 segments of 32
// chunks, 64 KB a chunk, 2400 cycles each; shared memory is busy for 1700 of them
// (the copies in, x scaled in place, the operands of the products).
// ---------------------------------------------------------------------------
constexpr int kStateStages = 3;
constexpr uint32_t kStateStage = 4 * kTileBytes;  // B, then x of two heads
constexpr uint32_t kStateBytes = kStateStages * kStateStage;
constexpr uint32_t kStateSmem = kStateBytes + 128 /* barriers */ + 384;

__global__ void __launch_bounds__(kScanThreads + 32, 1) prompt_states_kernel(const PromptParams p, const ChunkWork wk) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* smem = aligned_smem(smem_raw);
  if (!smem) return;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStateBytes);
  uint64_t *full = bars, *ready = bars + kStateStages, *empty = bars + 2 * kStateStages, *done = bars + 3 * kStateStages;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(done + 1);
  float *s_unit = reinterpret_cast<float*>(done + 2), *s_total = s_unit + 2;
  pdl_launch_dependents();
  pdl_wait();
  const ScanWork w = scan_work(p, wk);
  const Segment& sg = w.sg;
  if (sg.seq < 0 || sg.index + 1 >= sg.count) return;  // the same in every warp
  const int last = sg.chunk0 + w.c0 + w.chunks - 1;  // chunks go from here down
  auto load = [&](int k) {  // one thread
    const int st = k % kStateStages;
    const int64_t chunk = last - k;
    const uint32_t at = smem_u32(smem) + st * kStateStage;
    mbar_arrive_expect_tx(full + st, (2 + w.heads) * kTileBytes);
    bulk_load(at, wk.b + (chunk * p.ng + w.g) * 2 * kTileBytes, 2 * kTileBytes, full + st);
    bulk_load(at + 2 * kTileBytes, wk.x + (chunk * p.nh + w.h0) * kTileBytes, w.heads * kTileBytes, full + st);
  };
  int loaded = 0;
  if (tid == 16 * 32) {
    for (int i = 0; i < kStateStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(ready + i, 16);
      mbar_init(empty + i, 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
    for (; loaded < min(kStateStages, w.chunks); ++loaded) load(loaded);
  }
  __syncwarp();
  if (warp == 16) tc::tmem_alloc(tslot, 128);
  if (warp < w.heads) {
    // the unit of the sum: the largest of the chunks' units, decayed to the segment's end
    const int h = w.h0 + warp;
    float after = 0.f, top = 0.f;
    for (int k0 = 0; k0 < w.chunks; k0 += 32) {
      const int k = k0 + lane;
      float a = 0.f, u = 0.f;
      if (k < w.chunks) {
        const int64_t chunk = last - k, th = chunk * p.nh + h;
        a = wk.cum[th * kChunk + kChunk - 1];
        const float* sc = wk.scale + chunk * (p.nh + 2 * p.ng);
        u = sc[h] * sc[p.nh + w.g] * pow2_floor(wk.meta[th].x);
      }
      float upto = a;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      top = fmaxf(top, u * exp2_approx(after + upto - a));
      after += __shfl_sync(0xffffffffu, upto, 31);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) {
      s_unit[warp] = 2.f * pow2_floor(top, 100);  // every token's weight is below 2
      s_total[warp] = after;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tslot;
  bool dead = false;

  if (warp == 16) {
    if (lane == 0) {
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !mbar_wait_bounded(bar, parity)) {
          record_status(SN_ERR_TIMEOUT);
          dead = true;
        }
      };
      const uint32_t id = w.heads == 2 ? idesc_f16(128, 128, true, true) : idesc_f16(128, 64, true, true);
      for (int k = 0; k < w.chunks && !dead; ++k) {
        const int st = k % kStateStages;
        wait(ready + st, (k / kStateStages) & 1);
        if (dead) break;
        tc::fence_after_sync();
        const uint32_t at = smem_u32(smem) + st * kStateStage;
        const uint64_t db = desc_k_rows(at, kTileBytes), dx = desc_k_rows(at + 2 * kTileBytes, kTileBytes);
#pragma unroll
        for (int j = 0; j < 8; ++j)  // S^T += B^T (w x), of both heads
          tc::mma_bf16(tmem, db + j * 128, dx + j * 128, id, k > 0 || j > 0);
        tc::mma_commit(empty + st);
        if (k + 1 == w.chunks) tc::mma_commit(done);
        // the stage of the chunk before this one is free once its products are done: this one's run meanwhile
        if (k > 0 && loaded < w.chunks) {
          wait(empty + (k - 1) % kStateStages, ((k - 1) / kStateStages) & 1);
          if (!dead) load(loaded++);
        }
      }
      if (dead)  // copies in flight land before the CTA leaves
        for (int k = max(0, loaded - kStateStages); k < loaded; ++k)
          mbar_wait_bounded(full + k % kStateStages, (k / kStateStages) & 1);
    }
    __syncwarp();
  } else {
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!__all_sync(0xffffffffu, dead || mbar_wait_bounded(bar, parity))) {
        record_status(SN_ERR_TIMEOUT);
        dead = true;
      }
    };
    // token, head and half of its 64 elements: eight lanes that share a phase of shared memory have eight tokens' rows
    const int i = warp * 8 + (lane & 7), hh = lane >> 4, half = (lane >> 3) & 1, h = w.h0 + min(hh, w.heads - 1);
    const bool on = hh < w.heads;
    float a_i, a_end, dt, sx, sB;
    auto fetch = [&](int k) {
      const int64_t chunk = last - k, th = chunk * p.nh + h;
      a_i = wk.cum[th * kChunk + i];
      a_end = wk.cum[th * kChunk + kChunk - 1];
      dt = wk.dt[th * kChunk + i];
      const float* sc = wk.scale + chunk * (p.nh + 2 * p.ng);
      sx = sc[h];
      sB = sc[p.nh + w.g];
    };
    fetch(0);
    const float runit = rcp_pow2(s_unit[h - w.h0]);
    float after = 0.f;  // log2 of the decay from the chunk's end to the segment's
    for (int k = 0; k < w.chunks; ++k) {
      const float wj = dt * (sx * sB * runit) * exp2_approx(after + a_end - a_i);
      after += a_end;
      if (k + 1 < w.chunks) fetch(k + 1);
      const int st = k % kStateStages;
      wait(full + st, (k / kStateStages) & 1);
      if (on) {
        const uint32_t row = smem_u32(smem) + st * kStateStage + (2 + hh) * kTileBytes + i * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t at = row + (((4 * half + c) ^ (i & 7)) << 4);
          const uint4 x = lds128(at);
          const float2 m0 = mul2(unpack_f16(x.x), splat(wj)), m1 = mul2(unpack_f16(x.y), splat(wj));
          const float2 m2 = mul2(unpack_f16(x.z), splat(wj)), m3 = mul2(unpack_f16(x.w), splat(wj));
          sts128(at, pack_f16(m0.x, m0.y), pack_f16(m1.x, m1.y), pack_f16(m2.x, m2.y), pack_f16(m3.x, m3.y));
        }
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(ready + st);
      __syncwarp();
    }
    wait(done, 0);
    tc::fence_after_sync();
    // row n of S^T; warps of a head and half of its columns
    const int q = warp & 3, n = q * 32 + lane, wg = warp >> 3, hf = (warp >> 2) & 1;
    if (wg < w.heads) {
      float v[32];
      tc::tmem_ld32(tmem + 64 * wg + 32 * hf + (static_cast<uint32_t>(q * 32) << 16), v);
      const int hd = w.h0 + wg;
      const int64_t at = static_cast<int64_t>(32 * hf) * 128 + n, slot = static_cast<int64_t>(p.nh) * 64 * 128;
      float* ws = wk.state + (static_cast<int64_t>(sg.slot0) * p.nh + hd) * 64 * 128 + at;
      const float unit = s_unit[wg], decay = exp2_approx(s_total[wg]);
      const __nv_bfloat16* s0 = p.ssm_state + (static_cast<int64_t>(sg.seq) * p.nh + hd) * 64 * 128 + at;
      if (sg.index == 0) {
        float s[32];  // all loads before the first store, which might be to the same place for all the compiler knows
#pragma unroll
        for (int k = 0; k < 32; ++k) s[k] = __bfloat162float(s0[k * 128]);
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          ws[k * 128] = s[k];
          v[k] = fmaf(s[k], decay, v[k] * unit);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] *= unit;
      }
#pragma unroll
      for (int k = 0; k < 32; ++k) ws[(sg.index + 1) * slot + k * 128] = v[k];
      if (n == 0 && hf == 0) wk.total[static_cast<int64_t>(sg.slot0 + sg.index + 1) * p.nh + hd] = s_total[wg];
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 16) tc::tmem_dealloc(tmem, 128);
}

// Shared memory (from a 1024-byte boundary): the heads' state / weighted-x
// operands, then twice a stage of B, X of two heads, C and the exponents of C's
// rows, with the tokens' factors and the rest behind them where the next stage's
// boundary leaves room.
constexpr uint32_t kOperandAt = 0;
constexpr uint32_t kStageAt = 2 * kTileBytes;
constexpr uint32_t kStageX = 2 * kTileBytes, kStageC = 4 * kTileBytes, kStageRows = 6 * kTileBytes;
constexpr uint32_t kStageBytes = kStageRows + 2048;
constexpr uint32_t kAfter0 = kStageAt + kStageRows + kChunk, kAfter1 = kAfter0 + kStageBytes;
// factors of the tokens: [512 bytes] of head 0 (two), head 1, and the last of head 1 behind the second stage
constexpr uint32_t kFactorsAt = kAfter0, kFactorsLast = kAfter1;
constexpr uint32_t kEndsAt = kFactorsAt + 3 * 4 * kChunk;  // block ends of the heads, then the chunks' common factors
constexpr uint32_t kBarsAt = kEndsAt + 256;
static_assert(kBarsAt + 128 == kStageAt + kStageBytes);
constexpr uint32_t kScanSmem = kFactorsLast + 4 * kChunk + 384;
static_assert(kScanSmem <= 227 * 1024);
// Tensor memory columns: S of two heads, C B^T, M of two heads, Y of two heads.
constexpr int kServe = 4;  // the serving warp of a head's eight
constexpr uint32_t kColS = 0, kColG = 128, kColM = 256, kColY = 384;

// One segment of one pair of heads of a group (blockIdx.x: pair, blockIdx.y:
// segment): two heads, because they share B, C and C B^T and one computes while
// the other waits for its products; shared memory, tensor memory and registers
// are full then.  Warps 0-7 have the first head, 8-15 the second, a thread one row
// (token i, or state n) and half of the columns of every product: 16 warps with
// 128 registers each (a 17th for the copies would leave 96).  Of a head's warps
// the one with the first 32 rows and the later columns has no part of M (it is
// all above the diagonal), so it serves the others: it issues the products and
// copies and works out the chunk's common factors.
// Measured: 153 us for 128 segments of 32 chunks, 4.5 us (7900 cycles) a chunk
// of two heads.  It is bounded by the chain of a chunk (S to its operand, C S,
// M, w x, M X, outputs: each waits for the one before), with issue slots 41% busy
// and the tensor pipe 27%.  Longer: M X into columns of its own by way of C B^T's
// (214 us), groups of warps for the rows and for the decays (190), the outputs a
// chunk behind (205), arrivals in place of the two barriers (165).
__global__ void __launch_bounds__(kScanThreads, 1) prompt_scan_mma_kernel(const PromptParams p, const ChunkWork wk) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned char* smem = aligned_smem(smem_raw);
  if (!smem) return;
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarsAt);
  uint64_t *full = bars, *empty = bars + 2, *bar_g = bars + 4, *gfree = bars + 5, *bar_y2 = bars + 6, *bar_y = bars + 8,
           *bar_s = bars + 10;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + 12);
  pdl_launch_dependents();
  pdl_wait();
  const ScanWork w = scan_work(p, wk);
  const Segment& sg = w.sg;
  if (sg.seq < 0) return;  // the same in every warp
  const int g = w.g, h0 = w.h0, heads = w.heads, c0 = w.c0, nchunks = w.chunks;
  // the copies of a chunk's operands into its stage (one thread)
  auto load = [&](int c) {
    const uint32_t st = sbase + kStageAt + (c & 1) * kStageBytes;
    const int64_t chunk = sg.chunk0 + c0 + c;
    mbar_arrive_expect_tx(full + (c & 1), 2 * kTileBytes + heads * kTileBytes + kRowTileBytes);
    bulk_load(st, wk.b + (chunk * p.ng + g) * 2 * kTileBytes, 2 * kTileBytes, full + (c & 1));
    bulk_load(st + kStageC, wk.c + (chunk * p.ng + g) * kRowTileBytes, kRowTileBytes, full + (c & 1));
    bulk_load(st + kStageX, wk.x + (chunk * p.nh + h0) * kTileBytes, heads * kTileBytes, full + (c & 1));
  };
  int loaded = min(2, nchunks);  // chunks whose copies have been issued
  if (tid == kServe * 32) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 8 * heads);
      mbar_init(bar_y2 + i, 1);
      mbar_init(bar_y + i, 1);
      mbar_init(bar_s + i, 1);
    }
    mbar_init(bar_g, 1);
    mbar_init(gfree, 8 * heads);
    fence_barrier_init();
    for (int c = 0; c < loaded; ++c) load(c);
  }
  __syncwarp();
  const int wg = warp >> 3, half = (warp >> 2) & 1, q = warp & 3, i = q * 32 + lane, h = h0 + wg;
  const bool serving = (warp & 7) == kServe;
  // Inputs of a chunk: a token's own for every thread, the head's for the serving warp; loaded a chunk ahead.
  const int chunk0 = sg.chunk0 + c0;
  float next_a, next_dt;
  auto fetch = [&](int c) {
    const int64_t at = (static_cast<int64_t>(chunk0 + c) * p.nh + h) * kChunk + i;
    next_a = wk.cum[at];
    next_dt = wk.dt[at];
  };
  struct {
    float a_end, sx, sB, sC;
    float2 meta;
  } head;
  auto fetch_head = [&](int c) {
    const int64_t th = static_cast<int64_t>(chunk0 + c) * p.nh + h;
    const float* sc = wk.scale + static_cast<int64_t>(chunk0 + c) * (p.nh + 2 * p.ng);
    head.a_end = wk.cum[th * kChunk + kChunk - 1];
    head.meta = wk.meta[th];
    head.sx = sc[h];
    head.sB = sc[p.nh + g];
    head.sC = sc[p.nh + p.ng + g];
  };
  // The first chunk's inputs and the state before the segment (row n = i of S^T, this half's 32 columns, true values):
  // all of them on their way before anything waits
  float v0[32];
  if (wg < heads) {
    fetch(0);
    if (serving) fetch_head(0);
    const int64_t at = static_cast<int64_t>(32 * half) * 128 + i, slot = static_cast<int64_t>(p.nh) * 64 * 128;
    const __nv_bfloat16* st = p.ssm_state + (static_cast<int64_t>(sg.seq) * p.nh + h) * 64 * 128 + at;
    float* ws = wk.state + (static_cast<int64_t>(sg.slot0) * p.nh + h) * 64 * 128 + at;
    if (sg.count == 1) {
#pragma unroll
      for (int k = 0; k < 32; ++k) v0[k] = __bfloat162float(st[k * 128]);
    } else {  // slot 0, or the segments before this one joined
      const int first = min(sg.index, 1);
#pragma unroll
      for (int k = 0; k < 32; ++k) v0[k] = ws[first * slot + k * 128];
      for (int j = 2; j <= sg.index; ++j) {
        const float dec = exp2_approx(wk.total[static_cast<int64_t>(sg.slot0 + j) * p.nh + h]);
#pragma unroll
        for (int k = 0; k < 32; ++k) v0[k] = fmaf(v0[k], dec, ws[j * slot + k * 128]);
      }
    }
  }
  if (warp == 0) tc::tmem_alloc(tslot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tslot;
  bool dead = false;  // a wait ran out: no further waits but for what is in flight
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // whole warps
    if (!__all_sync(0xffffffffu, dead || mbar_wait_bounded(bar, parity))) {
      record_status(SN_ERR_TIMEOUT);
      dead = true;
    }
  };

  if (wg < heads) {
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tS = tmem + kColS + wg * 64 + 32 * half + lanes, tG = tmem + kColG + lanes,
                   tM = tmem + kColM + wg * 64 + lanes, tY = tmem + kColY + wg * 64 + 32 * half + lanes;
    const uint32_t opnd = sbase + kOperandAt + wg * kTileBytes;
    float* fj = reinterpret_cast<float*>(smem + kFactorsAt) + wg * 2 * kChunk;  // of token j within its block, see below
    float* ej = wg == 0 ? fj + kChunk : reinterpret_cast<float*>(smem + kFactorsLast);  // exp2(a_last(block) - a_j) dt_j
    float* cend = reinterpret_cast<float*>(smem + kEndsAt) + wg * 16;                   // [4]; first [8] maxima
    const uint32_t row = i * 128, sw = i & 7;
    const int bar_id = 1 + wg;
    // the chunk's common factors, two buffers: 1 / sdt, a_end, S to its operand, S to the new unit and decayed;
    // C S from its operand's unit to that of M X, M X to outputs, x' to D x
    float4* common = reinterpret_cast<float4*>(smem + kEndsAt + 128) + wg * 4;

    float unit = 1.f, bound = 0.f;  // S = unit * tensor memory; |S| <= bound
    {
#pragma unroll
      for (int k = 0; k < 32; ++k) bound = fmaxf(bound, fabsf(v0[k]));
      tmem_st32(tS, v0);
      tmem_wait_st();
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
      if (lane == 0) cend[warp & 7] = bound;
      named_bar_sync(bar_id, 256);
#pragma unroll
      for (int k = 0; k < 8; ++k) bound = fmaxf(bound, cend[k]);
    }

    const float D = serving && p.D ? __bfloat162float(p.D[h]) : 0.f;
    auto derive_head = [&](int c) {  // every scale is a power of two: products and reciprocals of them are exact
      const float sdt = pow2_floor(head.meta.x), rdt = rcp_pow2(sdt), dec = exp2_approx(head.a_end);
      const float unit_new = head.sB * head.sx * sdt, runit = rcp_pow2(head.sB) * rcp_pow2(head.sx) * rdt;
      const float sb = pow2_floor(bound, 100), sS = sb * (1.f / 8192.f);  // |S / sS| < 2^14
      if (lane == 0) {
        common[2 * (c & 1)] = make_float4(rdt, head.a_end, unit * (rcp_pow2(sb) * 8192.f), dec * (unit * runit));
        common[2 * (c & 1) + 1] = make_float4(sS * runit * kMScale, head.sC * (1.f / kMScale) * unit_new, D * head.sx, unit_new);
      }
      unit = unit_new;
      constexpr float most = static_cast<float>(1 << (2 * kTop));  // of a product of x and B
      bound = fmaf(dec, bound, unit_new * most * (head.meta.y * rdt));
    };
    struct Factors {
      float a_i, dtn;     // cumulative decay; dt / sdt as it goes into M
      float wj;           // the token's weight in the state
      float f_op, f_dec;  // as common
      float f_y;          // exp(a_i) C S, likewise
      float fy, dx;
    } f;
    float unit_last = 1.f;
    auto take = [&](int c) {
      const float4 u = common[2 * (c & 1)], w = common[2 * (c & 1) + 1];
      f.a_i = next_a;
      const float dtn = next_dt * u.x;
      f.dtn = dtn * kMScale;
      f.wj = dtn * exp2_approx(u.y - next_a);
      f.f_op = u.z;
      f.f_dec = u.w;
      f.f_y = exp2_approx(next_a) * w.x;
      f.fy = w.y;
      f.dx = w.z;
      unit_last = w.w;
    };
    // C B^T of chunk c (the second head's serving warp, if there is one), once both heads have read the last chunk's
    auto issue_g = [&](int c) {
      wait(full + (c & 1), (c >> 1) & 1);
      if (c > 0) wait(gfree, (c - 1) & 1);
      if (lane == 0 && !dead) {
        tc::fence_after_sync();
        constexpr uint32_t id = idesc_f16(128, 128, false, false);
        const uint64_t db = tc::smem_desc_sw128(smem + kStageAt + (c & 1) * kStageBytes), dc = db + kStageC / 16;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t at = ((k >> 2) * kTileBytes + (k & 3) * 32) / 16;
          tc::mma_bf16(tmem + kColG, dc + at, db + at, id, k > 0);
        }
        tc::mma_commit(bar_g);
      }
      __syncwarp();
    };
    const bool issues_g = serving && wg == heads - 1;
    if (serving) {
      derive_head(0);
      if (nchunks > 1) fetch_head(1);
    }
    named_bar_sync(bar_id, 256);
    take(0);
    if (nchunks > 1) fetch(1);
    if (issues_g) issue_g(0);
    const uint64_t d_op = desc_k_rows(opnd, 16);
    for (int c = 0; c < nchunks; ++c) {
      const unsigned stage = c & 1, ph = (c >> 1) & 1;
      const uint32_t sst = sbase + kStageAt + stage * kStageBytes;
      const uint32_t xrow = sst + kStageX + wg * kTileBytes + row;
      if (c > 0) {  // the last chunk's products are done: its stage, the operand buffer and S are free
        wait(bar_s + wg, (c - 1) & 1);
        tc::fence_after_sync();
        if (lane == 0) mbar_arrive(empty + ((c - 1) & 1));
        __syncwarp();
      }
      auto refill = [&]() {  // the next chunk's copies, into the last one's stage
        if (warp == kServe && c > 0 && c + 1 < nchunks) {
          wait(empty + ((c - 1) & 1), ((c - 1) >> 1) & 1);
          if (lane == 0 && !dead) load(c + 1);
          if (!dead) loaded = c + 2;
          __syncwarp();
        }
      };
      if (p.gate) {  // the gates' lines, on their way to L2
        const int t = (c0 + c) * kChunk + i;
        if (half == 0 && t < sg.len)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.zx + (sg.start + t) * p.ld + h * 64));
      }
      // ---- S: operand of C S, and decayed, in the new unit ----
      {
        float v[32];
        tc::tmem_ld32(tS, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 m = mul2(make_float2(v[8 * k + 2 * j], v[8 * k + 2 * j + 1]), splat(f.f_op));
            o[j] = pack_f16(m.x, m.y);
          }
          sts128(opnd + row + (((4 * half + k) ^ sw) << 4), o[0], o[1], o[2], o[3]);
        }
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 m = mul2(make_float2(v[k], v[k + 1]), splat(f.f_dec));
          v[k] = m.x;
          v[k + 1] = m.y;
        }
        tmem_st32(tS, v);
      }
      uint4 x[4];  // this half of this token's row of X
      // of the row's 32-token block: first and last token
      const float a_first = __shfl_sync(0xffffffffu, f.a_i, 0), a_last = __shfl_sync(0xffffffffu, f.a_i, 31);
      if (half == 0) {
        // within the block exp(a_i - a_j) = exp(a_i - a_first) exp(a_first - a_j) as long as the second stays far
        // from overflow; with more decay than 2^-100 in 32 tokens the exponents are subtracted first
        fj[i] = a_first - a_last < 100.f ? exp2_approx(a_first - f.a_i) * f.dtn : f.a_i - __log2f(f.dtn);
        if (lane == 31) cend[q] = f.a_i;
      } else {
        ej[i] = exp2_approx(a_last - f.a_i) * f.dtn;
      }
      __syncwarp();
      tmem_wait_st();
      tc::fence_before_sync();
      tc::fence_proxy_async_smem();
      named_bar_sync(bar_id, 256);
      if (serving) {
        wait(full + stage, ph);
        if (lane == 0 && !dead) {  // Y = C S
          tc::fence_after_sync();
          constexpr uint32_t id = idesc_f16(128, 64, false, true);
          const uint64_t dc = tc::smem_desc_sw128(smem + kStageAt + stage * kStageBytes + kStageC);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc::mma_bf16(tmem + kColY + wg * 64, dc + ((k >> 2) * kTileBytes + (k & 3) * 32) / 16, d_op + k * 128, id, k > 0);
          tc::mma_commit(bar_y2 + wg);
        }
        __syncwarp();
        refill();
        if (c + 1 < nchunks) {
          derive_head(c + 1);
          if (c + 2 < nchunks) fetch_head(c + 2);
        }
      }
      // ---- M from C B^T: blocks half and half + 2 of 32 columns ----
      wait(bar_g, c & 1);  // the chunk's operands are there too
      tc::fence_after_sync();
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = lds128(xrow + (((4 * half + k) ^ sw) << 4));
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const int jb = 2 * jj + half;
        uint32_t m[16];
        if (jb > q) {
#pragma unroll
          for (int k = 0; k < 16; ++k) m[k] = 0;
          tmem_st16(tM + 16 * jb, m);
          continue;
        }
        float v[32];
        tc::tmem_ld32(tG + 32 * jb, v);
        auto scaled = [&](const float* e, float2 r) {
          const float4* e4 = reinterpret_cast<const float4*>(e + 32 * jb);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 f4 = e4[k];
            const float2 m0 = mul2(mul2(make_float2(v[4 * k], v[4 * k + 1]), r), make_float2(f4.x, f4.y));
            const float2 m1 = mul2(mul2(make_float2(v[4 * k + 2], v[4 * k + 3]), r), make_float2(f4.z, f4.w));
            m[2 * k] = pack_f16(m0.x, m0.y);
            m[2 * k + 1] = pack_f16(m1.x, m1.y);
          }
        };
        if (jb < q) {  // an earlier block: exp(a_i - a_last) exp(a_last - a_j) dt_j, both at most 1
          scaled(ej, splat(exp2_approx(f.a_i - cend[jb])));
        } else {
          if (a_first - a_last < 100.f) {
            // v r first: r <= 1, and fj may be as large as 2^101
            scaled(fj, splat(exp2_approx(f.a_i - a_first)));
          } else {
            const float4* l4 = reinterpret_cast<const float4*>(fj + 32 * jb);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 l = l4[k];
              m[2 * k] = pack_f16(v[4 * k] * exp2_approx(f.a_i - l.x), v[4 * k + 1] * exp2_approx(f.a_i - l.y));
              m[2 * k + 1] = pack_f16(v[4 * k + 2] * exp2_approx(f.a_i - l.z), v[4 * k + 3] * exp2_approx(f.a_i - l.w));
            }
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) {  // causal: columns up to the row's own
            const uint32_t keep = 2 * k < lane ? 0xFFFFFFFFu : 2 * k == lane ? 0xFFFFu : 0u;
            m[k] &= keep;
          }
        }
        tmem_st16(tM + 16 * jb, m);
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(gfree);
      __syncwarp();
      // ---- Y = exp(a_i) C S, in the unit of M X ----
      wait(bar_y2 + wg, c & 1);
      tc::fence_after_sync();
      float v[32];
      tc::tmem_ld32(tY, v);
#pragma unroll
      for (int k = 0; k < 32; k += 2) {
        const float2 m = mul2(make_float2(v[k], v[k + 1]), splat(f.f_y));
        v[k] = m.x;
        v[k + 1] = m.y;
      }
      tmem_st32(tY, v);
      // ---- weighted x ----
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 m = mul2(unpack_f16(u[j]), splat(f.wj));
          o[j] = pack_f16(m.x, m.y);
        }
        sts128(opnd + row + (((4 * half + k) ^ sw) << 4), o[0], o[1], o[2], o[3]);
      }
      tmem_wait_st();
      tc::fence_before_sync();
      tc::fence_proxy_async_smem();
      named_bar_sync(bar_id, 256);
      if (serving) {
        if (lane == 0 && !dead) {
          tc::fence_after_sync();
          {  // Y += M X
            constexpr uint32_t id = idesc_f16(128, 64, false, true);
            const uint64_t dx = desc_k_rows(sst + kStageX + wg * kTileBytes, 16);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_f16_ts(tmem + kColY + wg * 64, tmem + kColM + wg * 64 + 8 * k, dx + k * 128, id, 1);
            tc::mma_commit(bar_y + wg);
          }
          constexpr uint32_t id = idesc_f16(128, 64, true, true);  // S += B^T (w x)
          const uint64_t db = desc_k_rows(sst, kTileBytes);
#pragma unroll
          for (int k = 0; k < 8; ++k) tc::mma_bf16(tmem + kColS + wg * 64, db + k * 128, d_op + k * 128, id, 1);
          tc::mma_commit(bar_s + wg);
        }
        __syncwarp();
        if (issues_g && c + 1 < nchunks) issue_g(c + 1);
      }
      // Outputs (and gates) go between a thread's row and whole 64-byte pieces of rows through the warp's part of the
      // chunk's X tile, which nothing reads once M X is done: lane l has 16 bytes l % 4 of rows l / 4, + 8, ...
      float fy_row = f.fy;
      if (f.fy < 0.f) fy_row *= -lds_pow2(sst + kStageRows + i);  // the chunk has rows of C with powers of two of their own
      const float2 fy = splat(fy_row), dx = splat(f.dx);
      const int tw = (c0 + c) * kChunk + q * 32 + (lane >> 2);  // the token of this lane's first piece
      const int64_t tok = sg.start + tw;
      const uint32_t stg = sst + kStageX + wg * kTileBytes + (q * 32 + (lane >> 2)) * 128;
      // 16-byte pieces are swizzled by the row's low bits reversed: eight lanes with a piece of eight rows, or with four
      // pieces of two rows, then hit eight places
      const int piece = 4 * half + (lane & 3), psw = __brev(lane >> 2) >> 29, osw = __brev(i & 7) >> 29;
      uint4 zv[4];
      if (p.gate) {
        const __nv_bfloat16* z = p.zx + tok * p.ld + h * 64 + 8 * piece;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          zv[k] = tw + 8 * k < sg.len ? *reinterpret_cast<const uint4*>(z + 8 * k * p.ld) : make_uint4(0, 0, 0, 0);
      }
      if (c + 1 < nchunks) {
        take(c + 1);
        if (c + 2 < nchunks) fetch(c + 2);
      }
      wait(bar_y + wg, c & 1);
      tc::fence_after_sync();
      if (p.gate) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sts128(stg + k * 1024 + ((piece ^ psw) << 4), zv[k].x, zv[k].y, zv[k].z, zv[k].w);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) zv[k] = lds128(xrow + (((4 * half + k) ^ osw) << 4));
        __syncwarp();
      }
      float yv[32];
      tc::tmem_ld32(tY, yv);
      tc::fence_before_sync();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, zu[4] = {zv[k].x, zv[k].y, zv[k].z, zv[k].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 y = fma2(make_float2(yv[8 * k + 2 * j], yv[8 * k + 2 * j + 1]), fy, mul2(unpack_f16(u[j]), dx));
          if (p.gate) y = mul2(y, silu2(unpack_bf16(zu[j])));
          const __nv_bfloat162 b = __floats2bfloat162_rn(y.x, y.y);
          o[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        sts128(xrow + (((4 * half + k) ^ osw) << 4), o[0], o[1], o[2], o[3]);
      }
      __syncwarp();
      __nv_bfloat16* out = p.y + (tok * p.nh + h) * 64 + 8 * piece;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 o = lds128(stg + k * 1024 + ((piece ^ psw) << 4));
        if (tw + 8 * k < sg.len) *reinterpret_cast<uint4*>(out + static_cast<int64_t>(8 * k) * p.nh * 64) = o;
      }
      tc::fence_proxy_async_smem();  // before the stage is handed back to the copies
      __syncwarp();
    }
    // ---- the state after the segment ----
    wait(bar_s + wg, (nchunks - 1) & 1);
    if (dead) mbar_wait_bounded(bar_s + wg, (nchunks - 1) & 1);
    __syncwarp();
    tc::fence_after_sync();
    if (sg.index + 1 == sg.count) {
      __nv_bfloat16* st = p.ssm_state + (static_cast<int64_t>(sg.seq) * p.nh + h) * 64 * 128 + 32 * half * 128 + i;
      float v[32];
      tc::tmem_ld32(tS, v);
#pragma unroll
      for (int k = 0; k < 32; ++k) st[k * 128] = __float2bfloat16_rn(v[k] * unit_last);
    }
  }
  if (dead && tid == kServe * 32)  // copies in flight land before the CTA leaves
    for (int c = max(0, loaded - 2); c < loaded; ++c) mbar_wait_bounded(full + (c & 1), (c >> 1) & 1);
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

// ---- host: sizes of the tensor-core form ----
struct ScanPlan {
  int64_t chunks;    // at most, over all prompts
  int64_t slots;     // state slots
  int64_t segments;  // at most
  int seg, pairs, xblocks, blocks;
  size_t x, b, c, cum, dt, meta, scale, state, total, bytes;  // offsets
};
inline bool plan_scan(int tokens, int batch, int d_inner, int ng, int d_state, int nh, ScanPlan* out) {
  if (d_state != 128 || d_inner != static_cast<int64_t>(nh) * 64) return false;
  ScanPlan r;
  // a prompt of t > 0 tokens has (t - 1) / n + 1 pieces of n, so all of them at most these many
  auto pieces = [&](int64_t n) { return batch + std::max(tokens - 1, 0) / n; };
  r.chunks = pieces(kChunk);
  const int hpg = nh / ng;
  r.pairs = ng * ((hpg + 1) / 2);
  r.xblocks = (d_inner + 127) / 128;
  r.blocks = r.xblocks + 2 * ng;
  // Chunks a segment: the least time over the SMs' waves of both launches, from what was measured (tenths of a
  // microsecond): 43 a chunk of the outputs and 110 to start and end a CTA of them, 11 and 90 for the states.
  const int sms = sm_count();
  const int64_t nc = std::max<int64_t>(1, (static_cast<int64_t>(tokens) + kChunk - 1) / kChunk);
  const int64_t each = (nc + batch - 1) / batch;  // of a prompt, if they are alike
  int64_t best = INT64_MAX;
  r.seg = static_cast<int>(each);
  for (int64_t n = 1; n <= std::min<int64_t>(each, 32); ++n) {  // segments of such a prompt
    const int64_t seg = (each + n - 1) / n;
    const int64_t waves = (batch * ((each + seg - 1) / seg) * r.pairs + sms - 1) / sms;
    const int64_t waves1 = n == 1 ? 0 : (batch * ((each + seg - 1) / seg - 1) * r.pairs + sms - 1) / sms;
    const int64_t cost = waves * (43 * seg + 110) + waves1 * (11 * seg + 90);
    if (cost < best) {
      best = cost;
      r.seg = static_cast<int>(seg);
    }
  }
  // Prompts are seldom alike: where the average one is not cut, one half as long again is not either (9 prompts of 1
  // to 2048 tokens 161 -> 148 us, 8 of 300 to 600 83 -> 77, 166 and 262 tokens with 32 heads 30 -> 28).
  if (batch > 1 && r.seg == each) r.seg = static_cast<int>((3 * each + 1) / 2);
  r.segments = pieces(static_cast<int64_t>(r.seg) * kChunk);
  r.slots = std::min(r.segments, 2 * (r.segments - batch) + 1);  // cut prompts have at least two pieces
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  const size_t nch = static_cast<size_t>(r.chunks);
  r.x = take(nch * nh * kTileBytes);
  r.b = take(nch * ng * 2 * kTileBytes);
  r.c = take(nch * ng * kRowTileBytes);
  r.cum = take(nch * nh * kChunk * 4);
  r.dt = take(nch * nh * kChunk * 4);
  r.meta = take(nch * nh * 8);
  r.scale = take(nch * (nh + 2 * ng) * 4);
  r.state = take(static_cast<size_t>(r.slots) * nh * 64 * 128 * 4);
  r.total = take(static_cast<size_t>(r.slots) * nh * 4);
  r.bytes = at;
  *out = r;
  return true;
}

}  // namespace

int tu_status_prompt(bool reset, cudaStream_t st, int* out) { return read_tu_status(reset, st, out); }

}  // namespace sn

extern "C" {

size_t sn_mamba2_prompt_workspace_size(int tokens, int batch, int d_inner, int ngroups, int d_state, int nheads) {
  if (tokens < 0 || batch < 1 || d_inner < 1 || ngroups < 1 || d_state < 1 || nheads < 1) return 0;
  size_t n = static_cast<size_t>(tokens) * (d_inner + 2 * static_cast<size_t>(ngroups) * d_state) * 2;
  sn::ScanPlan plan;
  if (nheads % ngroups == 0 && sn::plan_scan(tokens, batch, d_inner, ngroups, d_state, nheads, &plan))
    n = std::max(n, plan.bytes);
  return (n + 255) / 256 * 256 + 256;
}

int sn_mamba2_prompt(const void* zxbcdt, int64_t ld, void* conv_state, const void* conv_weight, const void* conv_bias,
                     void* ssm_state, const float* A, const void* D, const void* dt_bias, void* y,
                     const int* cu_seqlens, int batch, int tokens, int d_inner, int ngroups, int d_state, int nheads,
                     int headdim, int d_conv, int gate, void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 1 || tokens < 0 || (tokens > 0 && (!zxbcdt || !y || !workspace)) || !conv_state || !conv_weight ||
      !ssm_state || !A || d_inner < 1 || ngroups < 1 || d_state < 1 || nheads < 1 || headdim < 1 || d_conv < 1 ||
      d_conv > sn::kMaxConvWidth || (!cu_seqlens && batch != 1))
    return SN_ERR_INVALID_ARGUMENT;
  if (static_cast<int64_t>(nheads) * headdim != d_inner || nheads % ngroups != 0) return SN_ERR_INVALID_ARGUMENT;
  const int64_t gds = static_cast<int64_t>(ngroups) * d_state;
  if (ld < 2 * static_cast<int64_t>(d_inner) + 2 * gds + nheads) return SN_ERR_INVALID_ARGUMENT;
  if (tokens > 0 &&
      workspace_bytes < sn_mamba2_prompt_workspace_size(tokens, batch, d_inner, ngroups, d_state, nheads))
    return SN_ERR_INVALID_ARGUMENT;
  if (d_state > 16 * sn::kScanPerLane || d_inner + 2 * gds > INT32_MAX) return SN_ERR_UNSUPPORTED;
  if (tokens == 0) return SN_OK;
  sn::PromptParams p;
  p.zx = static_cast<const __nv_bfloat16*>(zxbcdt);
  p.ld = ld;
  p.conv_state = static_cast<__nv_bfloat16*>(conv_state);
  p.w = static_cast<const __nv_bfloat16*>(conv_weight);
  p.bias = static_cast<const __nv_bfloat16*>(conv_bias);
  p.ssm_state = static_cast<__nv_bfloat16*>(ssm_state);
  p.A = A;
  p.D = static_cast<const __nv_bfloat16*>(D);
  p.dt_bias = static_cast<const __nv_bfloat16*>(dt_bias);
  p.y = static_cast<__nv_bfloat16*>(y);
  p.xbc = reinterpret_cast<__nv_bfloat16*>((reinterpret_cast<uintptr_t>(workspace) + 255) / 256 * 256);
  p.prompts = {cu_seqlens, batch, tokens};
  p.di = d_inner;
  p.gds = static_cast<int>(gds);
  p.ds = d_state;
  p.ng = ngroups;
  p.nh = nheads;
  p.hd = headdim;
  p.hpg = nheads / ngroups;
  p.W = d_conv;
  p.gate = gate ? 1 : 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  sn::ScanPlan plan;
  const bool rows16 = sn::aligned16(zxbcdt) && ld % 8 == 0 && sn::aligned16(y) && sn::aligned16(conv_state) &&
                      sn::aligned16(conv_weight) && (!conv_bias || sn::aligned16(conv_bias));
  // 64-element heads, 128 states, 16-byte rows: the tensor-core form; anything else token by token (37 / 1021 / 16384
  // tokens of 64 heads: 14 / 33 / 260 us, token by token 66 / 1266 / 27454)
  if (d_conv >= 2 && d_conv <= 4 && rows16 &&
      sn::plan_scan(tokens, batch, d_inner, ngroups, d_state, nheads, &plan) && plan.chunks <= 65535 && plan.segments <= 65535) {
    unsigned char* base = reinterpret_cast<unsigned char*>(p.xbc);
    sn::ChunkWork wk;
    wk.x = base + plan.x;
    wk.b = base + plan.b;
    wk.c = base + plan.c;
    wk.cum = reinterpret_cast<float*>(base + plan.cum);
    wk.dt = reinterpret_cast<float*>(base + plan.dt);
    wk.meta = reinterpret_cast<float2*>(base + plan.meta);
    wk.scale = reinterpret_cast<float*>(base + plan.scale);
    wk.state = reinterpret_cast<float*>(base + plan.state);
    wk.total = reinterpret_cast<float*>(base + plan.total);
    wk.xblocks = plan.xblocks;
    wk.blocks = plan.blocks;
    wk.seg = plan.seg;
    const int conv_blocks = plan.blocks + (nheads + sn::kDtHeads - 1) / sn::kDtHeads;
    // more CTAs than three an SM hold at once: four (16384 tokens 255 us in all, with three 264, both
    // before C's rows had powers of two); else three and tokens
    // spread over the warps (37 / 1021 tokens 13.4 / 33.0 us, with four 13.9 / 34.1)
    const bool many = plan.chunks * conv_blocks > 3 * sn::sm_count();
    auto pick = [&](auto wide, auto narrow) { return many ? wide : narrow; };
    auto conv = d_conv == 4   ? pick(sn::prompt_conv_tile_kernel<4, true>, sn::prompt_conv_tile_kernel<4, false>)
                : d_conv == 3 ? pick(sn::prompt_conv_tile_kernel<3, true>, sn::prompt_conv_tile_kernel<3, false>)
                              : pick(sn::prompt_conv_tile_kernel<2, true>, sn::prompt_conv_tile_kernel<2, false>);
    int rc = sn::launch(conv, dim3(static_cast<unsigned>(conv_blocks), static_cast<unsigned>(plan.chunks)), dim3(256), 0, st,
                        true, p, wk);
    if (rc != SN_OK) return rc;
    const dim3 grid(static_cast<unsigned>(plan.pairs), static_cast<unsigned>(plan.segments));
    if (!sn::smem_room<sn::prompt_scan_mma_kernel>(sn::kScanSmem)) return SN_ERR_LAUNCH;
    if (tokens > static_cast<int64_t>(plan.seg) * sn::kChunk) {  // a prompt may have several segments
      if (!sn::smem_room<sn::prompt_states_kernel>(sn::kStateSmem)) return SN_ERR_LAUNCH;
      rc = sn::launch(sn::prompt_states_kernel, grid, dim3(sn::kScanThreads + 32), sn::kStateSmem, st, true, p, wk);
      if (rc != SN_OK) return rc;
    }
    return sn::launch(sn::prompt_scan_mma_kernel, grid, dim3(sn::kScanThreads), sn::kScanSmem, st, true, p, wk);
  }
  const int64_t rows = static_cast<int64_t>(batch) * d_inner;
  const int64_t blocks = tokens / sn::kConvRows + static_cast<int64_t>(batch);
  if (blocks > 65535 || rows > INT32_MAX / 16) return SN_ERR_UNSUPPORTED;
  const int conv_dim = d_inner + 2 * static_cast<int>(gds);
  const int rc = sn::launch(sn::prompt_conv_kernel,
                            dim3(static_cast<unsigned>((conv_dim + 255) / 256), static_cast<unsigned>(blocks)),
                            dim3(256), 0, st, true, p);
  if (rc != SN_OK) return rc;
  return sn::launch(sn::prompt_scan_rows_kernel, dim3(static_cast<unsigned>((rows + 15) / 16)), dim3(256), 0, st, true,
                    p);
}

}  // extern "C"
