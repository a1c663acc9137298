"""Producers and consumers of the gated-delta op inside one mixer layer, host side.

Same names and argument meaning as the reference:
  ShortConvolution                       models/hattention/short_convolution.py:528-720
  compute_lambda                         models/hattention/modeling_h_gated_deltanet.py:151-166
  FusedRMSNormGated / rms_norm_gated     models/hattention/fused_norm.py:1003-1064, 858-880
plus `gate_inputs`, the three statements that turn the a/b/l projections into g, beta and lambda
(modeling_h_gated_deltanet.py:429-450) as one call, `short_conv`, the convolution of sequences that continue from a cache, and
`block_norm`, the norms before and after a block with its gate and residual scale.  Forward only; everything runs in the CUDA
library on the current stream.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import _lib as L

_LAMBDA_MODES = {"positive": 0, "bounded": 1, None: 2}


class ShortConvolution(nn.Module):
    """Depthwise causal convolution over the token axis of [B, T, D] with an optional SiLU.

    Parameters are those of the reference's nn.Conv1d subclass: `weight` [D, 1, W] and `bias` [D]
    or None.  forward(x, residual, mask, cache, output_final_state, cu_seqlens) -> (y, cache);
    a call with one token per sequence and a cache is the decode step, which updates the cache
    [N, D, W] in place.
    """

    def __init__(self, hidden_size: int, kernel_size: int, bias: bool = False, activation: Optional[str] = "silu",
                 use_fast_conv1d: Optional[bool] = True, device=None, dtype=None, **kwargs):
        super().__init__()
        if kernel_size % 2 != 0:
            raise ValueError("Kernel size must be the power of 2")
        if activation is not None:
            assert activation in ["silu", "swish"], f"Activation `{activation}` not supported yet."
        self.hidden_size = hidden_size
        self.kernel_size = (kernel_size,)
        self.activation = activation
        conv = nn.Conv1d(hidden_size, hidden_size, kernel_size, groups=hidden_size, bias=bias,
                         padding=kernel_size - 1, device=device, dtype=dtype)      # same initialisation
        self.weight = conv.weight
        self.bias = conv.bias

    @property
    def state_size(self) -> int:
        return self.hidden_size * self.kernel_size[0]

    def _params(self):
        w = self.weight.detach().reshape(self.hidden_size, self.kernel_size[0]).contiguous()
        b = None if self.bias is None else self.bias.detach().contiguous()
        return w, b

    @torch.no_grad()
    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                cache: Optional[torch.Tensor] = None, output_final_state: bool = False,
                cu_seqlens: Optional[torch.LongTensor] = None, **kwargs) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        B, T, D = x.shape
        W = self.kernel_size[0]
        N = B if cu_seqlens is None else len(cu_seqlens) - 1
        if mask is not None:
            if cu_seqlens is not None:
                raise ValueError("`mask` and `cu_seqlens` cannot be provided at the same time")
            x = x.mul_(mask.unsqueeze(-1))
        if output_final_state and cache is None:
            cache = x.new_zeros(N, D, W)
        if cache is not None and B * T == N:
            return self.step(x, residual, cache, cu_seqlens)
        dev = L.require_cuda(x, residual, cache, cu_seqlens)
        w, b = self._params()
        x = x.contiguous()
        residual = None if residual is None else residual.contiguous()
        cu = None if cu_seqlens is None else cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()
        if cache is not None and (not cache.is_contiguous() or cache.dtype != x.dtype):
            raise ValueError("cache must be a contiguous [N, D, W] tensor of x's dtype")
        y = torch.empty_like(x)
        rc = L.lib().lampa_short_conv_fwd(L.ptr(x), L.ptr(w), L.ptr(b), L.ptr(residual), L.ptr(cu),
                                          0 if cu is None else N, B, T, D, W, L.dtype_code(x.dtype),
                                          L.dtype_code(w.dtype), int(self.activation is not None), L.ptr(y),
                                          L.ptr(cache), int(cu is not None), L.stream_ptr(dev))
        L.check(rc, "lampa_short_conv_fwd")
        return y, cache

    @torch.no_grad()
    def step(self, x: torch.Tensor, residual: Optional[torch.Tensor], cache: torch.Tensor,
             cu_seqlens: Optional[torch.LongTensor] = None):
        dev = L.require_cuda(x, residual, cache)
        shape = x.shape
        N, D, W = cache.shape
        w, b = self._params()
        xf = x.reshape(N, D).contiguous()
        rf = None if residual is None else residual.reshape(N, D).contiguous()
        if not cache.is_contiguous() or cache.dtype != x.dtype:
            raise ValueError("cache must be a contiguous [N, D, W] tensor of x's dtype")
        y = torch.empty_like(xf)
        rc = L.lib().lampa_short_conv_step(L.ptr(xf), L.ptr(cache), L.ptr(w), L.ptr(b), L.ptr(rf), N, D, W,
                                           L.dtype_code(x.dtype), L.dtype_code(w.dtype),
                                           int(self.activation is not None), L.ptr(y), L.stream_ptr(dev))
        L.check(rc, "lampa_short_conv_step")
        return y.view(shape), cache


@torch.no_grad()
def gate_inputs(a: Optional[torch.Tensor], b: Optional[torch.Tensor], dl: Optional[torch.Tensor],
                A_log: Optional[torch.Tensor], dt_bias: Optional[torch.Tensor], L_param: Optional[torch.Tensor],
                lambda_mode: Optional[str] = "positive", attention_mask: Optional[torch.Tensor] = None,
                lambda_dtype: Optional[torch.dtype] = None):
    """(g, beta, l) of the hierarchical layer: a, b [B,T,H] (outputs of a_proj / b_proj), dl
    [B,T,H,L] or [B,T,H*L] (output of l_proj), A_log / dt_bias [H], L_param [H,L];
    g = -exp(A_log) softplus(a + dt_bias) in fp32, beta = sigmoid(b) in b's dtype,
    l = compute_lambda(L_param, dl, lambda_mode) in `lambda_dtype` (default: dl's dtype), each
    multiplied by attention_mask [B,T] when given.  Inputs set to None skip their output."""
    ref = a if a is not None else (b if b is not None else dl)
    dev = L.require_cuda(a, b, dl, A_log, dt_bias, L_param, attention_mask)
    Bn, T = ref.shape[:2]
    H = (a if a is not None else b).shape[2] if (a is not None or b is not None) else L_param.shape[0]
    if lambda_mode not in _LAMBDA_MODES:
        raise ValueError
    g = beta = lam = None
    nl = 0
    if a is not None:
        a = a.contiguous()
        g = torch.empty(Bn, T, H, dtype=torch.float32, device=dev)
    if b is not None:
        b = b.to(ref.dtype).contiguous()
        beta = torch.empty(Bn, T, H, dtype=b.dtype, device=dev)
    if dl is not None:
        nl = L_param.shape[-1]
        dl = dl.to(ref.dtype).reshape(Bn, T, H, nl).contiguous()
        lam = torch.empty(Bn, T, H, nl, dtype=lambda_dtype or dl.dtype, device=dev)
    f32 = lambda t: None if t is None else t.detach().to(device=dev, dtype=torch.float32).contiguous()
    A_log, dt_bias, Lw = f32(A_log), f32(dt_bias), f32(L_param)
    m = None if attention_mask is None else attention_mask[:, -T:].to(torch.float32).contiguous()
    rc = L.lib().lampa_gate_inputs(L.ptr(a), L.ptr(b), L.ptr(dl), L.ptr(A_log), L.ptr(dt_bias), L.ptr(Lw), L.ptr(m),
                                   Bn * T, H, nl, L.dtype_code(ref.dtype),
                                   L.dtype_code(beta.dtype if beta is not None else ref.dtype),
                                   L.dtype_code(lam.dtype if lam is not None else ref.dtype),
                                   _LAMBDA_MODES[lambda_mode], L.ptr(g), L.ptr(beta), L.ptr(lam), L.stream_ptr(dev))
    L.check(rc, "lampa_gate_inputs")
    return g, beta, lam


def compute_lambda(L: torch.Tensor, dl: torch.Tensor, lambda_mode: Optional[str]) -> torch.Tensor:
    """softplus(L * dl) ("positive"), exp(-exp(L) * softplus(dl)) ("bounded") or L * dl (None);
    L broadcasts as [1, 1, H, levels] against dl [B, T, H, levels]."""
    if lambda_mode not in _LAMBDA_MODES:
        raise ValueError
    Lp = L.reshape(L.shape[-2], L.shape[-1])
    return gate_inputs(None, None, dl, None, None, Lp, lambda_mode,
                       lambda_dtype=torch.promote_types(L.dtype, dl.dtype))[2]


@torch.no_grad()
def rms_norm_gated(x: torch.Tensor, g: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                   activation: str = "swish", residual: Optional[torch.Tensor] = None, prenorm: bool = False,
                   residual_in_fp32: bool = False, eps: float = 1e-6) -> torch.Tensor:
    """y = x / sqrt(mean(x^2) + eps) * weight * g * sigmoid(g) over the last axis (activation
    "sigmoid": ... * sigmoid(g)).  bias, residual and prenorm of the reference signature are not
    supported (the layer does not use them)."""
    if bias is not None or residual is not None or prenorm:
        raise NotImplementedError
    if activation not in ("swish", "silu", "sigmoid"):
        raise ValueError(f"Unsupported activation: {activation}")
    dev = L.require_cuda(x, g, weight)
    D = x.shape[-1]
    xf, gf = x.contiguous(), g.to(x.dtype).contiguous()
    w = None if weight is None else weight.detach().contiguous()
    y = torch.empty_like(xf)
    rc = L.lib().lampa_rmsnorm_gate(L.ptr(xf), L.ptr(gf), L.ptr(w), xf.numel() // D, D, L.dtype_code(x.dtype),
                                    L.dtype_code(w.dtype) if w is not None else L.LAMPA_F32, float(eps),
                                    int(activation == "sigmoid"), L.ptr(y), L.stream_ptr(dev))
    L.check(rc, "lampa_rmsnorm_gate")
    return y


@torch.no_grad()
def add_rms_norm(res: torch.Tensor, delta: Optional[torch.Tensor], weight: Optional[torch.Tensor], eps: float = 1e-6,
                 perm: Optional[torch.Tensor] = None, seg_offsets: Optional[torch.Tensor] = None, nseg: int = 1,
                 delta_at_r: bool = False, y_at_r: bool = False, out_dtype: Optional[torch.dtype] = torch.bfloat16):
    """Fused residual add + RMS norm (+ row permutation) on an fp32 residual stream `res` [rows, D],
    in place: the `RMSNorm(x, residual, prenorm=True)` of the reference's blocks
    (models/hattention/fused_norm.py:1288-1330, modeling_gated_deltaproduct.py:1169-1199) with the
    ordering layer's gather / un-gather (models/baselines/hmamba.py:428-455) folded in.

    For every j: r = perm[j] inside j's segment (r = j without perm);
    res[r] += delta[r if delta_at_r else j]; y[r if y_at_r else j] = rms_norm(res[r]) * weight.
    delta None: norm only.  out_dtype None: add only (returns None)."""
    dev = L.require_cuda(res, delta, weight, perm)
    if res.dtype != torch.float32 or not res.is_contiguous() or res.dim() != 2:
        raise ValueError("res must be a contiguous fp32 [rows, D] tensor (updated in place)")
    rows, D = res.shape
    if delta is not None:
        delta = delta.contiguous()
        if tuple(delta.shape) != (rows, D):
            raise ValueError("delta must match res")
    if perm is not None:
        perm = perm.to(torch.int64).contiguous().view(-1)
        if perm.numel() != rows:
            raise ValueError("perm must have one entry per row")
    if seg_offsets is not None:
        seg_offsets = seg_offsets.to(device=dev, dtype=torch.int64).contiguous()
        nseg = seg_offsets.numel() - 1
    w = None if weight is None else weight.detach().to(torch.float32).contiguous()
    y = None if out_dtype is None else torch.empty(rows, D, dtype=out_dtype, device=dev)
    rc = L.lib().lampa_add_rmsnorm(L.ptr(res), L.ptr(delta), L.dtype_code(delta.dtype) if delta is not None else 0,
                                   L.ptr(perm), L.ptr(seg_offsets), max(int(nseg), 1), rows, D, L.ptr(w), float(eps),
                                   int(delta_at_r), int(y_at_r), L.ptr(y), L.dtype_code(out_dtype) if y is not None else 0,
                                   L.ptr(L.status_word(dev)), L.stream_ptr(dev))
    L.check(rc, "lampa_add_rmsnorm")
    return y


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
               cache: Optional[torch.Tensor] = None, output_final_state: bool = False,
               cu_seqlens: Optional[torch.LongTensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Depthwise causal convolution over the tokens of x [B,T,D] for sequences that continue: what lies before a sequence's first
    token is what its cache [N,D,W] holds (W last inputs, as ShortConvolution keeps them; None: zeros).  With output_final_state
    the cache, or a new one, becomes the last W inputs of each sequence, in place, and is returned; that of an empty sequence
    stays.  weight: [D,W] or [D,1,W], W from 2 to 8; bias: [D], of the weight's type or one of its own; cu_seqlens: [N+1] with B == 1 (rows behind its last entry come out
    as zero).  x may be a part of wider rows.  Returns (y [B,T,D] in x's dtype, cache or None)."""
    from .gated_delta import _check_cu_seqlens, _forward_only, _launched
    from .state_space import _conv_params, _rows
    if activation not in (None, "silu", "swish"):
        raise ValueError(f"Activation `{activation}` not supported yet.")
    silu = activation is not None
    if (cache is not None or not output_final_state) and (cu_seqlens is None or cu_seqlens.is_cuda):
        r = L.native.conv_resume(x, weight, bias, cache, cu_seqlens, silu, bool(output_final_state), True)
        if r is not None:
            return r, (cache if output_final_state else None)
    _forward_only(x, weight, bias, cache)
    if x.dim() != 3 or weight.dim() < 2:
        raise ValueError("x [B,T,D] and weight [D,W] expected")
    B, T, D = x.shape
    W = weight.shape[-1]
    dev = L.require_cuda(x, weight, bias, cache)
    for t in (x, weight):
        L.dtype_code(t.dtype)
    if not 2 <= W <= 8:
        raise NotImplementedError("convolutions of other than 2 to 8 taps are not supported")
    w, b = _conv_params(weight, bias, D, W)
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError(f"The batch size is expected to be 1 rather than {B} when using `cu_seqlens`.")
        if cu_seqlens.dim() != 1 or len(cu_seqlens) < 2:
            raise ValueError("cu_seqlens must be a vector of at least two offsets")
        _check_cu_seqlens(cu_seqlens, T)
        cu_seqlens = cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()
    N = B if cu_seqlens is None else len(cu_seqlens) - 1
    if cache is not None and (tuple(cache.shape) != (N, D, W) or not cache.is_contiguous() or cache.dtype != x.dtype):
        raise ValueError(f"cache must be a contiguous [{N}, {D}, {W}] tensor of x's dtype")
    if cache is None and output_final_state:
        cache = torch.zeros(N, D, W, dtype=x.dtype, device=dev)
    if B * T * D == 0:
        return torch.empty(B, T, D, dtype=x.dtype, device=dev), (cache if output_final_state else None)
    with torch.no_grad():
        y = _launched(L.native.conv_resume(_rows(x), w, b, cache, cu_seqlens, silu, bool(output_final_state), False), "lampa_short_conv_resume")
    return y, (cache if output_final_state else None)


_GATE_ACTS = {None: 0, "sigmoid": 1, "silu": 2, "swish": 2}


def block_norm(res: torch.Tensor, delta: Optional[torch.Tensor], post_weight: Optional[torch.Tensor] = None,
               pre_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale=None,
               gate_activation: Optional[str] = None, eps: float = 1e-6, cu_seqlens: Optional[torch.LongTensor] = None,
               post_norm: bool = True, out_dtype: Optional[torch.dtype] = torch.bfloat16) -> Optional[torch.Tensor]:
    """Norms before and after a block on its fp32 residual stream `res` [rows,D], in place and in one pass:
        res += scale * act(gate) * rms_norm(delta) * post_weight        (post_norm False: delta itself)
        y = rms_norm(res) * pre_weight                                  (the next block's input, in out_dtype)
    delta [rows,D]: the block's output (None: the norm only).  gate: [rows,D], [D], or with cu_seqlens [N+1] one row [N,D] per
    sequence (a row of no sequence keeps its residual); gate_activation None, "sigmoid" or "silu".  scale: None, a number or [D].
    Weights [D] or None.  out_dtype None: no norm behind the update (returns None).  D up to 8192."""
    from .gated_delta import _check_cu_seqlens, _forward_only, _launched
    if gate_activation not in _GATE_ACTS:
        raise ValueError(f"Unsupported activation: {gate_activation}")
    act, ydt = _GATE_ACTS[gate_activation], -1 if out_dtype is None else L.dtype_code(out_dtype)
    is_tensor = isinstance(scale, torch.Tensor)
    number = scale if is_tensor else 1.0 if scale is None else float(scale)
    if cu_seqlens is None or cu_seqlens.is_cuda:
        r = L.native.block_norm(res, delta, post_weight, pre_weight, gate, number, act, float(eps), cu_seqlens, bool(post_norm), ydt, True)
        if r is not None:
            return None if r is True else r
    _forward_only(res, delta, post_weight, pre_weight, gate, scale if is_tensor else None)
    if res.dim() != 2 or res.dtype != torch.float32 or not res.is_contiguous():
        raise ValueError("res must be a contiguous fp32 [rows, D] tensor (updated in place)")
    rows, D = res.shape
    dev = L.require_cuda(res, delta, post_weight, pre_weight, gate, scale if is_tensor else None)
    if delta is None and (gate is not None or out_dtype is None):
        raise ValueError("without delta there is the norm of res only")
    if delta is not None and tuple(delta.shape) != (rows, D):
        raise ValueError("delta must match res")
    if cu_seqlens is not None and gate is None:
        raise ValueError("cu_seqlens says which sequence's gate a row takes: gate is missing")
    if D > 8192:
        raise NotImplementedError("rows of more than 8192 elements are not supported")
    vec = lambda t, n: None if t is None else _vector(t, D, n)  # noqa: E731
    post_weight, pre_weight = vec(post_weight, "post_weight"), vec(pre_weight, "pre_weight")
    if is_tensor:
        number = vec(scale, "scale")
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or len(cu_seqlens) < 2:
            raise ValueError("cu_seqlens must be a vector of at least two offsets")
        _check_cu_seqlens(cu_seqlens, rows)
        cu_seqlens = cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()
    if gate is not None:
        n = rows if cu_seqlens is None else len(cu_seqlens) - 1
        if gate.dim() == 1 or (gate.dim() == 2 and gate.shape[0] == 1):
            gate = gate.expand(n, gate.shape[-1])
        if tuple(gate.shape) != (n, D):
            raise ValueError(f"gate must be [{n}, {D}] or [{D}]")
        if gate.dtype not in (torch.float32, delta.dtype):
            L.dtype_code(gate.dtype)
            gate = gate.float()
    for t in (delta, gate):
        if t is not None:
            L.dtype_code(t.dtype)
    if rows * D == 0:
        return None if out_dtype is None else torch.empty(rows, D, dtype=out_dtype, device=dev)
    last = lambda t: t if t is None or D <= 1 or t.stride(-1) == 1 else t.contiguous()  # noqa: E731
    with torch.no_grad():
        r = _launched(L.native.block_norm(res, last(delta), post_weight, pre_weight, last(gate), number, act, float(eps), cu_seqlens,
                                          bool(post_norm), ydt, False), "lampa_block_norm")
    return None if r is True else r


def _vector(t: torch.Tensor, n: int, name: str) -> torch.Tensor:
    if tuple(t.shape) != (n,):
        raise ValueError(f"{name} must be [{n}]")
    return t.detach().to(torch.float32).contiguous()


class FusedRMSNormGated(nn.Module):
    """RMS norm over the last axis followed by a swish (or sigmoid) gate (fused_norm.py:1003-1064)."""

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, eps: float = 1e-5,
                 activation: str = "swish", device=None, dtype=None):
        super().__init__()
        if activation not in ["swish", "silu", "sigmoid"]:
            raise ValueError(f"Unsupported activation: {activation}")
        self.hidden_size = hidden_size
        self.elementwise_affine = elementwise_affine
        self.eps = eps
        self.activation = activation
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, g: torch.Tensor, residual: Optional[torch.Tensor] = None,
                prenorm: bool = False, residual_in_fp32: bool = False) -> torch.Tensor:
        return rms_norm_gated(x, g, self.weight, self.bias, self.activation, residual=residual, eps=self.eps,
                              prenorm=prenorm, residual_in_fp32=residual_in_fp32)
