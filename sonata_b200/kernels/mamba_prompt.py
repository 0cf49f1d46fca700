"""Mamba2 over prompts on B200: the many-token form of the decode-step ops.

``mamba2_prompt`` takes the in_proj rows of ragged prompts through the causal
convolution and the selective state space scan, and leaves the convolution
and SSM states as ``mamba_step.mamba2_split_conv`` +
``mamba_step.selective_state_update`` would after the last token, in the same
layouts, so that decoding goes on from them (C ABI: ``sn_mamba2_prompt``).
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from ._common import call, current_handle, fast, on_stream, require_cuda, same_device

_BF16 = torch.bfloat16


def _dense(name, t, shape, dtype=_BF16):
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.shape == shape and t.is_contiguous():
        return
    require_cuda(name, t, dtype)
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} tensor, got {tuple(t.shape)}")


def _check(zxbcdt, conv_state, weight, bias, ssm_state, A, D, dt_bias, d_inner, ngroups, d_state, nheads, cu_seqlens):
    require_cuda("zxbcdt", zxbcdt, _BF16, 2)
    if zxbcdt.shape[0] > 0 and zxbcdt.stride(1) != 1:
        raise ValueError("zxbcdt must be contiguous along its last dimension")
    tokens = zxbcdt.shape[0]
    conv_dim = d_inner + 2 * ngroups * d_state
    if d_inner % nheads or nheads % ngroups:
        raise ValueError(f"d_inner {d_inner} must split into {nheads} heads, and these into {ngroups} groups")
    if zxbcdt.shape[1] < d_inner + conv_dim + nheads:
        raise ValueError(f"zxbcdt has {zxbcdt.shape[1]} columns, fewer than {d_inner + conv_dim + nheads}")
    batch = 1
    if cu_seqlens is not None:
        require_cuda("cu_seqlens", cu_seqlens, torch.int32, 1)
        if cu_seqlens.numel() < 2 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous int32 [batch + 1] tensor, batch >= 1")
        batch = cu_seqlens.numel() - 1
    width = conv_state.shape[-1]
    _dense("conv_state", conv_state, (batch, conv_dim, width))
    _dense("weight", weight, (conv_dim, width))
    _dense("ssm_state", ssm_state, (batch, nheads, d_inner // nheads, d_state))
    _dense("A", A, (nheads,), torch.float32)
    if bias is not None:
        _dense("bias", bias, (conv_dim,))
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None:
            _dense(name, t, (nheads,))
    same_device(zxbcdt=zxbcdt, conv_state=conv_state, weight=weight, bias=bias, ssm_state=ssm_state, A=A, D=D,
                dt_bias=dt_bias, cu_seqlens=cu_seqlens)
    raise ValueError("the arguments of mamba2_prompt do not fit together")


@functools.lru_cache(maxsize=256)
def _workspace_size(*sizes: int) -> int:
    return _lib.lib().sn_mamba2_prompt_workspace_size(*sizes)


def mamba2_prompt(zxbcdt: torch.Tensor, conv_state: torch.Tensor, weight: torch.Tensor, bias, ssm_state: torch.Tensor,
                  A: torch.Tensor, D, dt_bias, d_inner: int, ngroups: int, d_state: int, nheads: int,
                  cu_seqlens: torch.Tensor | None = None, gate: bool = False, stream=None) -> torch.Tensor:
    """zxbcdt [tokens, >= width]: the in_proj rows [z | x B C | dt] of all
    prompts, packed (row stride taken from the tensor); prompt i holds rows
    cu_seqlens[i] .. cu_seqlens[i+1]-1 (int32 [batch + 1] on the device;
    None: one prompt).  conv_state [batch, conv_dim, W] and ssm_state [batch,
    nheads, headdim, d_state] are each prompt's state before its first token
    and are updated in place; A fp32 [nheads] (negative), D / dt_bias bf16
    [nheads] or None, weight [conv_dim, W], bias [conv_dim] or None.  Returns
    y [tokens, nheads, headdim] = S_t C_t + D x_t, times SiLU(z_t) with gate;
    zeros in rows of no prompt."""
    if stream is None:
        r = fast().prompt(zxbcdt, conv_state, weight, bias, ssm_state, A, D, dt_bias, d_inner, ngroups, d_state, nheads,
                          cu_seqlens, gate)
        if r is not None:
            return r if type(r) is not int else _lib.check("sn_mamba2_prompt", r)
    # one expression that holds for every valid call; _check says what is wrong with the others
    dev = torch.cuda.current_device()
    conv_dim, heads = d_inner + 2 * ngroups * d_state, (nheads,)
    try:
        (tokens, columns), width = zxbcdt.shape, conv_state.shape[-1]
        batch = 1 if cu_seqlens is None else cu_seqlens.shape[0] - 1
        ok = (zxbcdt.dtype is conv_state.dtype is weight.dtype is ssm_state.dtype is _BF16 and A.dtype is torch.float32 and
              d_inner % nheads == 0 and nheads % ngroups == 0 and columns >= d_inner + conv_dim + nheads and batch >= 1 and
              conv_state.shape == (batch, conv_dim, width) and weight.shape == (conv_dim, width) and
              ssm_state.shape == (batch, nheads, d_inner // nheads, d_state) and A.shape == heads and
              (tokens == 0 or zxbcdt.stride(1) == 1) and conv_state.is_contiguous() and weight.is_contiguous() and
              ssm_state.is_contiguous() and A.is_contiguous() and
              zxbcdt.get_device() == conv_state.get_device() == weight.get_device() == ssm_state.get_device() ==
              A.get_device() == dev)
        for t, shape in ((bias, (conv_dim,)), (D, heads), (dt_bias, heads)):
            if t is not None:
                ok = ok and t.dtype is _BF16 and t.shape == shape and t.is_contiguous() and t.get_device() == dev
        if cu_seqlens is not None:
            ok = ok and (cu_seqlens.dtype is torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous() and
                         cu_seqlens.get_device() == dev)
    except (AttributeError, TypeError, ValueError, IndexError, ZeroDivisionError):
        ok = False
    if not ok:
        _check(zxbcdt, conv_state, weight, bias, ssm_state, A, D, dt_bias, d_inner, ngroups, d_state, nheads, cu_seqlens)

    def launch(st):
        y = zxbcdt.new_empty((tokens, nheads, d_inner // nheads))
        if tokens == 0:
            return y
        nbytes = _workspace_size(tokens, batch, d_inner, ngroups, d_state, nheads)
        ws = torch.empty(nbytes, device=zxbcdt.device, dtype=torch.uint8)
        call("sn_mamba2_prompt", zxbcdt.data_ptr(), zxbcdt.stride(0) if tokens > 1 else columns,
             conv_state.data_ptr(), weight.data_ptr(), None if bias is None else bias.data_ptr(), ssm_state.data_ptr(),
             A.data_ptr(), None if D is None else D.data_ptr(), None if dt_bias is None else dt_bias.data_ptr(),
             y.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr(), batch, tokens, d_inner, ngroups, d_state,
             nheads, d_inner // nheads, width, 1 if gate else 0, ws.data_ptr(), nbytes, st)
        return y

    if stream is None:
        return launch(current_handle(dev))
    with on_stream(stream) as st:
        return launch(st)
