"""Refusals of the state space operators, without a GPU: what the checks of arguments say, and the C entry points' own."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


def _scan(**kw):
    import lampa_b200
    a = dict(x=torch.zeros(1, 8, 4, 16, dtype=BF), dt=torch.zeros(1, 8, 4), A=torch.zeros(4), B=torch.zeros(1, 8, 2, 16, dtype=BF), C=torch.zeros(1, 8, 2, 16, dtype=BF))
    a.update(kw)
    return lampa_b200.state_space_scan(**a)


def test_scan_refusals():
    import lampa_b200
    with pytest.raises(lampa_b200.LampaError, match="CUDA tensors only"):
        _scan()
    with pytest.raises(NotImplementedError, match="forward pass only"):
        _scan(x=torch.zeros(1, 8, 4, 16, dtype=BF, requires_grad=True))
    with pytest.raises(NotImplementedError, match="forward pass only"):
        _scan(A=torch.zeros(4, requires_grad=True))
    for bad in (dict(x=torch.zeros(8, 4, 16, dtype=BF)), dict(dt=torch.zeros(1, 8, 3)), dict(B=torch.zeros(1, 8, 3, 16, dtype=BF), C=torch.zeros(1, 8, 3, 16, dtype=BF)),
                dict(C=torch.zeros(1, 8, 2, 8, dtype=BF)), dict(z=torch.zeros(1, 8, 4, 8, dtype=BF)), dict(B=torch.zeros(1, 7, 2, 16, dtype=BF), C=torch.zeros(1, 7, 2, 16, dtype=BF)),
                dict(x=torch.zeros(1, 8, 4, 0, dtype=BF))):
        with pytest.raises(ValueError):
            _scan(**bad)


def test_step_refusals():
    import lampa_b200
    a = dict(xbc=torch.zeros(2, 4 * 8 + 2 * 16, dtype=BF), dt=torch.zeros(2, 4), conv_cache=torch.zeros(2, 64, 4, dtype=BF), state=torch.zeros(2, 4, 8, 16),
             conv_weight=torch.zeros(64, 4, dtype=BF), conv_bias=None, A=torch.zeros(4))
    with pytest.raises(lampa_b200.LampaError, match="CUDA tensors only"):
        lampa_b200.state_space_step(**a)
    with pytest.raises(NotImplementedError, match="forward pass only"):
        lampa_b200.state_space_step(**dict(a, state=torch.zeros(2, 4, 8, 16, requires_grad=True)))
    for bad in (dict(xbc=torch.zeros(2, 63, dtype=BF)), dict(xbc=torch.zeros(2, 32, dtype=BF)), dict(dt=torch.zeros(2, 3)), dict(conv_cache=torch.zeros(3, 64, 4, dtype=BF)),
                dict(state=torch.zeros(3, 4, 8, 16)), dict(z=torch.zeros(2, 4, 9, dtype=BF)), dict(activation="gelu"), dict(state=torch.zeros(2, 3, 8, 16))):
        with pytest.raises(ValueError):
            lampa_b200.state_space_step(**dict(a, **bad))


def test_conv_refusals():
    import lampa_b200
    x, w = torch.zeros(1, 9, 8, dtype=BF), torch.zeros(8, 4, dtype=BF)
    with pytest.raises(lampa_b200.LampaError, match="CUDA tensors only"):
        lampa_b200.short_conv(x, w)
    with pytest.raises(NotImplementedError, match="forward pass only"):
        lampa_b200.short_conv(x, w.clone().requires_grad_())
    with pytest.raises(ValueError):
        lampa_b200.short_conv(x, w, activation="gelu")
    with pytest.raises(ValueError):
        lampa_b200.short_conv(x[0], w)


def test_norm_refusals():
    import lampa_b200
    res, delta = torch.zeros(4, 8), torch.zeros(4, 8)
    with pytest.raises(lampa_b200.LampaError, match="CUDA tensors only"):
        lampa_b200.block_norm(res, delta)
    with pytest.raises(NotImplementedError, match="forward pass only"):
        lampa_b200.block_norm(res, delta.clone().requires_grad_())
    with pytest.raises(ValueError):
        lampa_b200.block_norm(res.bfloat16(), delta)
    with pytest.raises(ValueError):
        lampa_b200.block_norm(res, delta, gate_activation="gelu")
    with pytest.raises(TypeError):
        lampa_b200.block_norm(res, delta, out_dtype=torch.float64)


def test_c_entry_points_refuse():
    from lampa_b200 import _lib
    lib, n = _lib.lib(), ctypes.c_size_t(0)
    d = lambda **kw: _lib.SsmDesc(**dict(dict(B=1, T=1000, H=4, P=64, N=64, G=1, nseq=0, dtype=0, dt_dtype=0, dt_softplus=1), **kw))  # noqa: E731
    size = lambda x: lib.lampa_ssm_workspace_bytes(ctypes.byref(x), ctypes.byref(n))  # noqa: E731
    assert size(d()) == 0
    assert size(d(T=0)) == 0 and n.value == 0
    assert size(d(G=3)) == -1 and size(d(H=0)) == -1 and size(d(B=2, nseq=3)) == -1 and size(d(dt_dtype=5)) == -1
    assert size(d(dtype=2)) == -2 and size(d(N=257)) == -2
    none = [None] * 2

    def scan(x, ws=None, nb=0, cu=None):
        return lib.lampa_ssm_scan(ctypes.byref(x), None, 0, 0, None, 0, None, None, 0, 0, None, 0, 0, None, None, 0, 0, None, None, cu, None, None, ws, nb, *none)
    assert scan(d()) == -1 and scan(d(dtype=2)) == -2 and scan(d(nseq=2)) == -1 and scan(d(T=0)) == 0
    step = lambda x, taps=4: lib.lampa_ssm_step(ctypes.byref(x), None, 0, None, 0, None, None, None, taps, 0, 1, None, None, None, 0, 0, None, None, None, None)  # noqa: E731
    assert step(d()) == -1 and step(d(N=300)) == -2 and step(d(), 9) == -2 and step(d(B=0)) == 0
    conv = lambda nt=10, W=4, nseq=1: lib.lampa_short_conv_resume(None, 8, None, None, None, nseq, nt, 8, W, 0, 0, 1, None, 0, None, None, None)  # noqa: E731
    assert conv() == -1 and conv(W=9) == -2 and conv(nt=0) == 0 and conv(nseq=0) == -1
    norm = lambda rows=4, D=8, act=0: lib.lampa_block_norm(None, None, 0, 0, None, 0, 0, act, None, 0, rows, D, None, 1, None, 1.0, None, 1e-6, None, 0, None, None)  # noqa: E731
    assert norm() == -1 and norm(rows=0) == 0 and norm(act=7) == -1
