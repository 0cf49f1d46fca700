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
#include "common.cuh"

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

// The index-th block, where every prompt is cut into blocks of `rows` tokens
// (at least `least` of them, so that an empty prompt still has one where its
// state has to be handled).  Called by whole warps; every lane gets the answer.
__device__ __forceinline__ PromptBlock find_block(const Prompts& p, int rows, int least, int index) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    int s = 0, e = 0, n = 0;
    if (b < p.batch) {
      const int s0 = p.cu ? p.cu[b] : 0, e0 = p.cu ? p.cu[b + 1] : p.tokens;
      s = min(max(s0, 0), p.tokens);
      e = min(max(e0, s), p.tokens);
      if (s != s0 || e != e0) record_status(SN_ERR_INVALID_ARGUMENT);
      n = max((e - s + rows - 1) / rows, least);
    }
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
// elements l, l + 16, ...
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
  const int s0 = p.prompts.cu ? p.prompts.cu[b] : 0, e0 = p.prompts.cu ? p.prompts.cu[b + 1] : p.prompts.tokens;
  const int start = min(max(s0, 0), p.prompts.tokens);
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

}  // namespace

int tu_status_prompt(bool reset, cudaStream_t st, int* out) { return read_tu_status(reset, st, out); }

}  // namespace sn

extern "C" {

size_t sn_mamba2_prompt_workspace_size(int tokens, int batch, int d_inner, int ngroups, int d_state, int nheads) {
  if (tokens < 0 || batch < 1 || d_inner < 1 || ngroups < 1 || d_state < 1 || nheads < 1) return 0;
  return (static_cast<size_t>(tokens) * (d_inner + 2 * static_cast<size_t>(ngroups) * d_state) * 2 + 255) / 256 * 256 +
         256;
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
