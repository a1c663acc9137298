"""Selective state space scan over prompts and its step for single tokens.

Per head the state h is P x N, the decay one number per token:
  d_t = softplus(dt_t + dt_bias),   h_t = exp(A d_t) h_{t-1} + d_t x_t B_t^T,   y_t = (h_t C_t + D x_t) silu(z_t)
and heads of one group share B and C.  `state_space_scan` takes whole sequences (a batch of equally long ones, or a packed batch
with `cu_seqlens`), `state_space_step` one token per row together with the short convolution in front of the recurrence.  For a
prompt that convolution is `short_conv` (layer.py), whose cache the step takes over.  Forward only; everything runs in the CUDA
library on the current stream of the tensors' device.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib as L
from .gated_delta import _check_cu_seqlens, _forward_only, _launched

_TYPES16 = (torch.bfloat16, torch.float16)
MAX_STATE = 256        # largest N
MAX_TAPS = 8           # of the convolution


def _head_vector(t: Optional[torch.Tensor], H: int, name: str, dev) -> Optional[torch.Tensor]:
    if t is None:
        return None
    L.require_cuda(t)
    if tuple(t.shape) != (H,):
        raise ValueError(f"{name} must be [{H}], one value per head")
    return t.detach().to(device=dev, dtype=torch.float32).contiguous()


def _rows(t: Optional[torch.Tensor], aligned: bool = False) -> Optional[torch.Tensor]:
    """t [B, T, ...] itself where its tokens lie one distance apart and its last axis is contiguous (`aligned`: and every row of
    it begins on a 16-byte boundary), else a dense copy."""
    if t is None:
        return None
    even = t.shape[0] <= 1 or t.shape[1] <= 1 or t.stride(0) == t.shape[1] * t.stride(1)
    even = even and (t.shape[-1] <= 1 or t.stride(-1) == 1)
    if aligned:
        even = even and not any(v * t.element_size() % 16 for n, v in zip(t.shape[:-1], t.stride()) if n > 1) and t.data_ptr() % 16 == 0
    return t if even else t.clone(memory_format=torch.contiguous_format)       # (a dense one at an odd place, too)


def state_space_scan(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    dt_bias: Optional[torch.Tensor] = None,
    dt_softplus: bool = True,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.LongTensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Selective state space scan, chunkwise.

    x, z: [B,T,H,P]; dt: [B,T,H]; B, C: [B,T,G,N] with G dividing H; A, D, dt_bias: [H]; initial_state: [N_seq,H,P,N]
    (not changed); cu_seqlens: [N_seq+1] with B == 1.  Returns (y [B,T,H,P] in x's dtype, final state [N_seq,H,P,N] fp32 or
    None).  x, B, C and z are bf16 or fp16 (fp32 is refused: the products run on 16-bit operands) and may be parts of wider
    rows, as a projection's output is split (x, B and C are copied where these do not begin on 16-byte boundaries); dt may
    have a type of its own.  Any P, N up to 256, any lengths from 0 on; rows
    behind the last entry of cu_seqlens come out as zero.  D None: no skip; z None: no gate.
    A times a step is meant to be at most 0 (a decay); growth is computed too as long as e^(A sum d) over any 128 tokens is finite.
    A large step resets the state (d C.B has to stay a finite float, whatever x is: 1e30 is safe).
    The last bits of y and of the states depend on how long the whole call is (the tokens are cut into blocks), those of y also on
    whether a final state is asked for; those of two equal calls do not differ.
    Offsets on the device that fall or leave the input are reported through `check_status()`.
    """
    r = L.native.ssm_scan(x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens, bool(dt_softplus), bool(output_final_state), True) \
        if cu_seqlens is None or cu_seqlens.is_cuda else None
    if r is not None:
        return r
    _forward_only(x, dt, A, B, C, D, z, dt_bias, initial_state)
    if x.dim() != 4 or dt.dim() != 3 or B.dim() != 4 or C.shape != B.shape:
        raise ValueError("x [B,T,H,P], dt [B,T,H], B and C [B,T,G,N] expected")
    Bn, T, H, P = x.shape
    G, N = B.shape[2:]
    if tuple(dt.shape) != (Bn, T, H) or tuple(B.shape[:2]) != (Bn, T) or G == 0 or H % G or min(H, P, N) == 0:
        raise ValueError("x [B,T,H,P], dt [B,T,H], B and C [B,T,G,N] expected, with G dividing H")
    if z is not None and z.shape != x.shape:
        raise ValueError("z must have the shape of x")
    dev = L.require_cuda(x, dt, A, B, C, D, z, dt_bias, initial_state)
    if x.dtype not in _TYPES16 or any(t is not None and t.dtype != x.dtype for t in (B, C, z)):
        raise TypeError("x, B, C and z must all be bf16 or all fp16")
    L.dtype_code(dt.dtype)
    if N > MAX_STATE:
        raise NotImplementedError(f"state sizes above {MAX_STATE} are not supported")
    if cu_seqlens is not None:
        if Bn != 1:
            raise ValueError(f"The batch size is expected to be 1 rather than {Bn} when using `cu_seqlens`.")
        if cu_seqlens.dim() != 1 or len(cu_seqlens) < 2:
            raise ValueError("cu_seqlens must be a vector of at least two offsets")
        _check_cu_seqlens(cu_seqlens, T)
        cu_seqlens = cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()
    nseq = Bn if cu_seqlens is None else len(cu_seqlens) - 1
    if initial_state is not None:
        if tuple(initial_state.shape) != (nseq, H, P, N):
            raise ValueError(f"initial_state must be [{nseq},{H},{P},{N}]")
        initial_state = initial_state.to(torch.float32).contiguous()
    if Bn * T == 0:
        ht = None
        if output_final_state:
            ht = initial_state.clone() if initial_state is not None else torch.zeros(nseq, H, P, N, device=dev)
        return torch.empty(Bn, T, H, P, dtype=x.dtype, device=dev), ht
    A, D, dt_bias = (_head_vector(t, H, n, dev) for t, n in ((A, "A"), (D, "D"), (dt_bias, "dt_bias")))
    wide = P % 8 == 0 and N % 8 == 0              # rows of whole 16-byte pieces: the kernels read them as such
    with torch.no_grad():
        return _launched(L.native.ssm_scan(_rows(x, wide), _rows(dt), A, _rows(B, wide), _rows(C, wide), D, _rows(z), dt_bias, initial_state,
                                           cu_seqlens, bool(dt_softplus), bool(output_final_state), False), "lampa_ssm_scan")


def state_space_step(
    xbc: torch.Tensor,
    dt: torch.Tensor,
    conv_cache: torch.Tensor,
    state: torch.Tensor,
    conv_weight: torch.Tensor,
    conv_bias: Optional[torch.Tensor],
    A: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    dt_bias: Optional[torch.Tensor] = None,
    dt_softplus: bool = True,
    activation: Optional[str] = "silu",
) -> torch.Tensor:
    """One token per row: the short convolution and the recurrence in one launch, both states in place.

    xbc: [B, H*P + 2*G*N], a row's x, B and C before the convolution; dt: [B,H]; z: [B,H,P]; conv_cache: [B, channels, W] in
    xbc's dtype (ShortConvolution's cache: the last W inputs); conv_weight: [channels, W] or [channels, 1, W]; conv_bias:
    [channels] or None, of the weight's type or one of its own; state: [B,H,P,N] fp32.  Returns y [B,H,P] in xbc's dtype (bf16, fp16 or fp32).  The number of groups
    follows from the width of xbc.  Rows of xbc, dt and z may be parts of wider rows.
    """
    if activation not in (None, "silu", "swish"):
        raise ValueError(f"Activation `{activation}` not supported yet.")
    silu = activation is not None
    r = L.native.ssm_step(xbc, dt, conv_cache, state, conv_weight, conv_bias, A, D, z, dt_bias, bool(dt_softplus), silu, True)
    if r is not None:
        return r
    _forward_only(xbc, dt, conv_cache, state, conv_weight, conv_bias, A, D, z, dt_bias)
    if xbc.dim() != 2 or dt.dim() != 2 or state.dim() != 4 or conv_cache.dim() != 3:
        raise ValueError("xbc [B,channels], dt [B,H], conv_cache [B,channels,W], state [B,H,P,N] expected")
    Bn, ch = xbc.shape
    H, P, N = state.shape[1:]
    W = conv_cache.shape[2]
    if min(H, P, N) == 0 or ch <= H * P or (ch - H * P) % (2 * N) or H % ((ch - H * P) // (2 * N)):
        raise ValueError(f"xbc must have H*P + 2*G*N = {H}*{P} + 2*G*{N} channels with G dividing H; got {ch}")
    if tuple(dt.shape) != (Bn, H) or state.shape[0] != Bn or tuple(conv_cache.shape) != (Bn, ch, W):
        raise ValueError("xbc [B,channels], dt [B,H], conv_cache [B,channels,W], state [B,H,P,N] expected")
    if z is not None and tuple(z.shape) != (Bn, H, P):
        raise ValueError(f"z must be [{Bn},{H},{P}]")
    dev = L.require_cuda(xbc, dt, conv_cache, state, conv_weight, conv_bias, A, D, z, dt_bias)
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous fp32 tensor (it is updated in place)")
    if conv_cache.dtype != xbc.dtype or not conv_cache.is_contiguous():
        raise ValueError("conv_cache must be a contiguous tensor of xbc's dtype (it is updated in place)")
    if z is not None and z.dtype != xbc.dtype:
        raise TypeError("z must have xbc's dtype")
    for t in (xbc, dt, conv_weight):
        L.dtype_code(t.dtype)
    if N > MAX_STATE or not 2 <= W <= MAX_TAPS:
        raise NotImplementedError(f"state sizes above {MAX_STATE} and convolutions of other than 2 to {MAX_TAPS} taps are not supported")
    w, b = _conv_params(conv_weight, conv_bias, ch, W)
    if Bn == 0:
        return torch.empty(Bn, H, P, dtype=xbc.dtype, device=dev)
    last = lambda t: t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()  # noqa: E731
    A, D, dt_bias = (_head_vector(t, H, n, dev) for t, n in ((A, "A"), (D, "D"), (dt_bias, "dt_bias")))
    with torch.no_grad():
        return _launched(L.native.ssm_step(last(xbc), last(dt), conv_cache, state, w, b, A, D, last(z), dt_bias, bool(dt_softplus), silu,
                                           False), "lampa_ssm_step")


def _conv_params(weight: torch.Tensor, bias: Optional[torch.Tensor], channels: int, taps: int):
    w = weight.detach()
    if w.dim() == 3 and w.shape[1] == 1:
        w = w[:, 0]
    if tuple(w.shape) != (channels, taps):
        raise ValueError(f"the convolution's weight must be [{channels}, {taps}]")
    if bias is not None and tuple(bias.shape) != (channels,):
        raise ValueError(f"the convolution's bias must be [{channels}]")
    if bias is None:
        return w.contiguous(), None
    b = bias.detach()
    if b.dtype != w.dtype:                        # the kernels take one type for both: fp32 holds either
        w, b = w.float(), b.float()
    return w.contiguous(), b.contiguous()
