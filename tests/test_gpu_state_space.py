"""The state space scan, its step, the convolution that continues and the block norms, against the recurrence in 64 bits.

Bounds: tests/ssm_oracle.py derives them for the scan.  The step and the norms work in fp32 (errors of a few 2^-24 per operation, the
fast exponential's 2^-21 in gates), so that their 16-bit results are off by half a step of their own and little else.
"""
import math

import pytest
import torch

from tests import ssm_oracle as oracle

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def lb():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import lampa_b200
    yield lampa_b200
    lampa_b200.check_status()


@pytest.fixture(autouse=True)
def _checked_by_the_tests(monkeypatch):
    monkeypatch.setenv("LAMPA_B200_CHECK", "0")    # the status word is read below, not inside the calls


def _near(got, ref, bound, what):
    d = (got.double() - ref).abs()
    # a value beyond the type's largest rounds to infinity of its sign, and nothing else does (65 520 and more in fp16)
    beyond = torch.isinf(got) & (got.sign() == ref.sign()) & (ref.abs() + bound >= torch.finfo(got.dtype).max)
    bad = ~(d <= bound) & ~beyond
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / bound).max()):.2f} of the bound"


def _rel(got, ref):
    return float((got.double() - ref).norm() / ref.norm().clamp_min(1e-300))


def scan_inputs(seed, B, T, H, P, G, N, dtype, z=False, D=True, h0=False, nseq=None, pitch=0, dt_dtype=None, decay=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    u = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    row = r(B, T, H * P + 2 * G * N + pitch).to(dtype)
    x, b, c = row[..., :H * P].unflatten(2, (H, P)), row[..., H * P:H * P + G * N].unflatten(2, (G, N)), row[..., H * P + G * N:H * P + 2 * G * N].unflatten(2, (G, N))
    step = torch.exp(math.log(1e-3) + u(H) * math.log(100.0))
    return dict(x=x, dt=r(B, T, H).to(dt_dtype or dtype), A=-(1 + 15 * u(H)) * decay, B=b, C=c, D=(1 + 0.1 * r(H)) if D else None,
                z=r(B, T, H, P).to(dtype) if z else None, dt_bias=step + torch.log(-torch.expm1(-step)),
                initial_state=0.3 * r(nseq or B, H, P, N) if h0 else None)


def check_scan(lb, a, cu=None, softplus=True, final=True, on_device=True):
    off = None if cu is None else torch.tensor(cu, device="cuda" if on_device else "cpu")
    y, ht = lb.state_space_scan(**a, dt_softplus=softplus, output_final_state=final, cu_seqlens=off)
    lb.check_status()
    ry, rh, ya, ha = oracle.scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], softplus, a["initial_state"], cu)
    assert y.shape == a["x"].shape and y.dtype == a["x"].dtype
    _near(y, ry, oracle.y_bound(y.dtype, ya), "y")
    if not final:
        assert ht is None
        return y, None
    assert ht.dtype == F32 and ht.shape == rh.shape
    _near(ht, rh, oracle.state_bound(ha, a["x"].shape[1]), "state")
    if float(rh.norm()) > 0:
        assert _rel(ht, rh) < 1e-6, _rel(ht, rh)
    return y, ht


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,T,H,P,G,N", [
    (1, 1, 1, 64, 1, 64), (1, 63, 2, 64, 1, 128), (2, 64, 4, 32, 2, 16), (1, 65, 3, 16, 3, 32), (3, 200, 2, 64, 1, 64),
    (1, 129, 2, 128, 2, 128), (1, 70, 2, 96, 1, 256), (1, 130, 1, 1, 1, 1), (2, 77, 3, 5, 1, 7), (1, 66, 2, 65, 1, 130), (1, 100, 2, 24, 1, 200)])
def test_scan_sizes(lb, dtype, B, T, H, P, G, N):
    check_scan(lb, scan_inputs(T + P, B, T, H, P, G, N, dtype, z=True))
    check_scan(lb, scan_inputs(T + N, B, T, H, P, G, N, dtype, D=False, h0=True))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("P,N,H,G", [(64, 128, 4, 2), (64, 64, 3, 1), (32, 16, 6, 1), (128, 64, 2, 1)])
def test_scan_over_blocks(lb, dtype, P, N, H, G):
    """Long enough for several blocks of several chunks, slow and fast decays"""
    for decay in (0.02, 1.0, 30.0):
        check_scan(lb, scan_inputs(int(decay * 10), 1, 3001, H, P, G, N, dtype, z=True, h0=True, decay=decay))


@pytest.mark.parametrize("P,N,H,G,T", [(64, 128, 4, 1, 1300), (64, 64, 6, 2, 700), (40, 72, 5, 1, 515), (136, 128, 3, 3, 260), (8, 8, 2, 1, 400), (64, 120, 1, 1, 129)])
def test_scan_kernels_agree(lb, P, N, H, G, T):
    """The tcgen05 kernels and their mma.sync twins on one input, each within its bound of the recurrence"""
    from lampa_b200 import _lib
    for pitch in (0, 8):
        a = scan_inputs(T, 2, T, H, P, G, N, BF, z=True, h0=True, pitch=pitch)
        try:
            for off in (0, 1):
                _lib.lib().lampa_debug_force_mma_sync(off)
                check_scan(lb, a)
        finally:
            _lib.lib().lampa_debug_force_mma_sync(0)
        a["z"] = torch.cat([a["z"], a["z"][..., :1]], 3)[..., :P]          # rows of z that are not 16-byte aligned
        check_scan(lb, a)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [[1], [0, 1, 63, 0, 64, 65, 200, 0], [5, 700, 0, 0, 1, 129, 1300, 2], [128, 128, 128], [0, 0, 3]])
def test_scan_packed(lb, dtype, lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    for h0 in (False, True):
        a = scan_inputs(sum(lens) + h0, 1, cu[-1], 3, 64, 1, 64, dtype, z=h0, h0=h0, nseq=len(lens))
        y, ht = check_scan(lb, a, cu)
        y2, _ = check_scan(lb, a, cu, final=False, on_device=False)
        if ht is not None and h0:
            for s, n in enumerate(lens):
                if n == 0:
                    assert torch.equal(ht[s], a["initial_state"][s])


def test_scan_of_a_sequence_does_not_see_its_neighbours(lb):
    """NaN and infinity in one packed sequence, and in the rows of another head, reach nothing else"""
    lens = [70, 300, 40, 130]
    cu = [0, 70, 370, 410, 540]
    a = scan_inputs(5, 1, 540, 2, 64, 1, 64, BF, z=True, h0=True, nseq=4)
    clean, hc = lb.state_space_scan(**a, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"))
    for what, t, p in (("x", 100, 3), ("x", 369, 0), ("dt", 200, None), ("B", 70, 5), ("C", 150, 7)):
        for bad in (math.nan, math.inf):
            b = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in a.items()}
            if what == "dt":
                b["dt"][0, t, 1] = bad
            else:
                b[what][0, t, 0, p] = bad
            y, ht = lb.state_space_scan(**b, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"))
            lb.check_status()
            for s in (0, 2, 3):
                assert torch.equal(y[0, cu[s]:cu[s + 1]], clean[0, cu[s]:cu[s + 1]]) and torch.equal(ht[s], hc[s])
            assert torch.equal(y[0, 70:t], clean[0, 70:t]), f"{what} {bad}: rows in front of it changed"
            if what == "x":                        # column p of its head from there on, nothing else
                assert not torch.isfinite(y[0, t:370, 0, p]).any() and not torch.isfinite(ht[1, 0, p]).any()
                keep = [i for i in range(64) if i != p]
                assert torch.equal(y[0, 70:370, 0][:, keep], clean[0, 70:370, 0][:, keep]) and torch.equal(y[0, 70:370, 1], clean[0, 70:370, 1])
                assert torch.equal(ht[1, 0, keep], hc[1, 0, keep])
            elif what == "dt":
                assert torch.equal(y[0, 70:370, 0], clean[0, 70:370, 0]) and not torch.isfinite(y[0, t, 1]).any() and not torch.isfinite(ht[1, 1]).any()
            elif what == "B":
                assert not torch.isfinite(y[0, t:370]).any() and not torch.isfinite(ht[1, :, :, p]).any()
            else:
                assert not torch.isfinite(y[0, t]).any() and torch.equal(y[0, t + 1:370], clean[0, t + 1:370]) and torch.equal(ht, hc)


def test_scan_plain_steps_and_their_limits(lb):
    """dt as it is: zero steps change nothing, huge ones forget everything"""
    a = scan_inputs(9, 1, 150, 2, 64, 1, 64, BF, h0=True, dt_dtype=F32)
    a["dt_bias"] = None
    a["dt"] = torch.zeros_like(a["dt"])
    y, ht = check_scan(lb, a, softplus=False)
    assert torch.equal(ht, a["initial_state"])
    a["dt"] = a["dt"] + 1e4
    check_scan(lb, a, softplus=False)
    a["dt"] = (torch.rand_like(a["dt"]) < 0.5) * 0.3          # tokens that are switched off in between
    check_scan(lb, a, softplus=False)


@pytest.mark.parametrize("pitch", [0, 8, 3])
def test_scan_reads_parts_of_wider_rows(lb, pitch):
    a = scan_inputs(3, 2, 90, 2, 64, 1, 64, BF, z=True, pitch=pitch)
    y, ht = check_scan(lb, a)
    dense = {k: (v.contiguous() if isinstance(v, torch.Tensor) else v) for k, v in a.items()}
    y2, h2 = lb.state_space_scan(**dense, output_final_state=True)
    assert torch.equal(y, y2) and torch.equal(ht, h2)
    odd = dict(a, x=a["x"].transpose(2, 3).contiguous().transpose(2, 3), dt=a["dt"].transpose(1, 2).contiguous().transpose(1, 2))
    y3, h3 = lb.state_space_scan(**odd, output_final_state=True)
    assert torch.equal(y, y3) and torch.equal(ht, h3)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_scan_of_expanded_and_single_axes(lb, dtype):
    """B and C of one group for all by a stride of zero, one x for all heads, one head or token out of many"""
    a = scan_inputs(13, 1, 300, 4, 64, 2, 64, dtype, z=True)
    a["B"], a["C"] = (a[k][:, :, :1].expand(1, 300, 2, 64) for k in ("B", "C"))
    check_scan(lb, a)
    a["x"], a["z"] = (a[k][:, :, :1].expand(1, 300, 4, 64) for k in ("x", "z"))
    check_scan(lb, a)
    a["x"] = a["x"][:, :1].expand(1, 300, 4, 64)
    check_scan(lb, a)
    a = scan_inputs(14, 1, 300, 4, 64, 2, 64, dtype, z=True, pitch=3)
    one = dict(a, x=a["x"][:, :, 1:2], dt=a["dt"][..., 1:2], z=a["z"][:, :, 1:2], B=a["B"][:, :, 1:], C=a["C"][:, :, 1:], A=a["A"][1:2], D=a["D"][1:2], dt_bias=a["dt_bias"][1:2])
    check_scan(lb, one)
    check_scan(lb, {k: (v[:, 7:8] if k in ("x", "dt", "B", "C", "z") else v) for k, v in one.items()})


@pytest.mark.parametrize("dtype", [BF, FP])
def test_scan_many_short_sequences_and_a_long_one(lb, dtype):
    lens = [3, 0, 1] * 90 + [2500] + [2] * 60
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    check_scan(lb, scan_inputs(15, 1, cu[-1], 6, 32, 1, 16, dtype, h0=True, nseq=len(lens)), cu)


@pytest.mark.parametrize("dt_dtype", [F32, FP, BF])
def test_scan_step_types(lb, dt_dtype):
    check_scan(lb, scan_inputs(4, 1, 100, 2, 64, 1, 64, BF, dt_dtype=dt_dtype))


def test_scan_continues(lb):
    """Two halves with the state carried over are the whole"""
    a = scan_inputs(6, 2, 500, 4, 64, 2, 64, BF, z=True)
    y, ht = lb.state_space_scan(**a, output_final_state=True)
    cut = lambda s: {k: (v[:, s] if k in ("x", "dt", "B", "C", "z") else v) for k, v in a.items()}  # noqa: E731
    y0, h0 = lb.state_space_scan(**cut(slice(0, 201)), output_final_state=True)
    y1, h1 = lb.state_space_scan(**dict(cut(slice(201, 500)), initial_state=h0), output_final_state=True)
    assert _rel(h1, ht.double()) < 1e-6
    _, _, ya, _ = oracle.scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"])
    _near(torch.cat([y0, y1], 1), y.double(), 2 * oracle.y_bound(BF, ya), "y")


def test_scan_nothing_to_do(lb):
    a = scan_inputs(7, 2, 4, 2, 16, 1, 16, BF, h0=True)
    none = {k: (v[:, :0] if k in ("x", "dt", "B", "C") else v) for k, v in a.items()}
    y, ht = lb.state_space_scan(**none, output_final_state=True)
    assert y.shape == (2, 0, 2, 16) and torch.equal(ht, a["initial_state"]) and ht.data_ptr() != a["initial_state"].data_ptr()


def test_scan_offsets_on_the_device_are_checked(lb):
    a = scan_inputs(8, 1, 300, 2, 64, 1, 64, BF, nseq=3)
    for cu in ([0, 100, 50, 300], [0, 100, 200, 301], [-1, 100, 200, 300], [0, 100, 400, 300], [5, 100, 200, 300], [0, -7, 200, 300]):
        lb.state_space_scan(**a, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"))
        with pytest.raises(lb.LampaError):
            lb.check_status()
    y, ht = lb.state_space_scan(**a, output_final_state=True, cu_seqlens=torch.tensor([0, 100, 100, 230], device="cuda"))
    lb.check_status()
    assert (y[0, 230:] == 0).all() and (ht[1] == 0).all()          # rows behind the last sequence


def test_scan_waits_are_bounded(lb):
    """With no polls left every wait gives up: the call ends, says so, and the next one is right"""
    from lampa_b200 import _lib
    for H, T in ((4, 1000), (48, 1500)):          # blocks of one chunk, and of several
        a = scan_inputs(12, 1, T, H, 64, 1, 128, BF, z=True, h0=True)
        want = lb.state_space_scan(**a, output_final_state=True)
        try:
            _lib.lib().lampa_debug_set_poll_budget(0)
            lb.state_space_scan(**a, output_final_state=True)
            torch.cuda.synchronize()
        finally:
            _lib.lib().lampa_debug_set_poll_budget(1 << 22)
        with pytest.raises(lb.LampaError):
            lb.check_status()
        again = lb.state_space_scan(**a, output_final_state=True)
        lb.check_status()
        assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])


def test_scan_in_a_graph_and_on_another_stream(lb):
    a = scan_inputs(10, 1, 2000, 4, 64, 1, 128, BF, z=True, h0=True)
    want = lb.state_space_scan(**a, output_final_state=True)
    again = lb.state_space_scan(**a, output_final_state=True)
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = lb.state_space_scan(**a, output_final_state=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want[0], other[0]) and torch.equal(want[1], other[1])
    x0 = a["x"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = lb.state_space_scan(**a, output_final_state=True)
    a["x"].mul_(-1)
    g.replay()
    torch.cuda.synchronize()
    neg = [t.clone() for t in held]
    direct = lb.state_space_scan(**a, output_final_state=True)
    assert torch.equal(neg[0], direct[0]) and torch.equal(neg[1], direct[1])
    a["x"].copy_(x0)
    g.replay()
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_scan_offsets_beyond_32_bits(lb):
    """x and y of 2^31 elements and more: the end of the sequence, which a fast decay keeps from what was before"""
    T, H, P, N = (1 << 31) // 1024 + 1000, 16, 64, 16
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(1, T, H, P, dtype=BF, device="cuda").normal_(generator=gen)
    b, c = (torch.empty(1, T, 1, N, dtype=BF, device="cuda").normal_(generator=gen) for _ in range(2))
    dt = torch.full((1, T, H), 0.5, dtype=BF, device="cuda")
    A = -torch.linspace(1, 4, H, device="cuda")
    y, ht = lb.state_space_scan(x, dt, A, b, c, dt_softplus=False, output_final_state=True)
    cut = T - 300
    ry, rh, ya, ha = oracle.scan(x[:, cut:], dt[:, cut:], A, b[:, cut:], c[:, cut:], softplus=False)
    _near(y[:, cut + 100:], ry[:, 100:], oracle.y_bound(BF, ya[:, 100:]), "y")
    assert _rel(ht, rh) < 1e-6
    _near(y[:, :200], oracle.scan(x[:, :200], dt[:, :200], A, b[:, :200], c[:, :200], softplus=False)[0], oracle.y_bound(BF, oracle.scan(x[:, :200], dt[:, :200], A, b[:, :200], c[:, :200], softplus=False)[2]), "y")


# ---- single tokens ---------------------------------------------------------------------------------
def step_inputs(seed, B, H, P, G, N, W, dtype, z=True, pitch=0, w_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    ch = H * P + 2 * G * N
    row = r(B, ch + H * P + H + pitch).to(dtype)
    return dict(xbc=row[:, :ch], dt=row[:, ch:ch + H], conv_cache=r(B, ch, W).to(dtype), state=r(B, H, P, N), conv_weight=(0.5 * r(ch, W)).to(w_dtype or dtype),
                conv_bias=(0.1 * r(ch)).to(w_dtype or dtype), A=-torch.rand(H, generator=gen, device="cuda") * 8, D=r(H),
                z=row[:, ch + H:ch + H + H * P].unflatten(1, (H, P)) if z else None, dt_bias=r(H) - 2)


def check_step(lb, a, activation="silu", softplus=True):
    cache, state = a["conv_cache"].clone(), a["state"].clone()
    y = lb.state_space_step(**a, activation=activation, dt_softplus=softplus)
    B, H, P, N = state.shape
    ch = a["xbc"].shape[1]
    G = (ch - H * P) // (2 * N)
    w = a["conv_weight"].reshape(ch, -1)
    v, new, _ = oracle.conv(a["xbc"][:, None], w, a["conv_bias"], activation, cache, None)
    v = v[:, 0]
    x, b, c = v[:, :H * P].unflatten(1, (H, P)), v[:, H * P:H * P + G * N].unflatten(1, (G, N)), v[:, H * P + G * N:].unflatten(1, (G, N))
    ry, rh, ya, ha = oracle.scan(x[:, None], a["dt"][:, None], a["A"], b[:, None], c[:, None], a["D"], None if a["z"] is None else a["z"][:, None],
                                 a["dt_bias"], softplus, state)
    assert torch.equal(a["conv_cache"].double(), new)
    # the convolution's result is off by a few 2^-24 of its own sum of at most 8 terms; relative to the values here 2^-18 covers it
    slack = 2.0 ** -18
    conv_slack = 2.0 ** -20 * (1 + v.abs().max())
    _near(a["state"], rh, slack * ha + conv_slack * ha.abs().max() * 0.05, "state")
    _near(y, ry[:, 0], oracle.half_step(y.dtype) * ry[:, 0].abs() + 2.0 ** -16 * ya[:, 0] + 2.0 ** -18 * ya.max() + 2.0 ** -25, "y")
    # steps as they are may be negative: a state then grows by e^g, g = A d > 0, and the roundings of dt + dt_bias and of the product, 2^-24
    # of g each, appear in it g times as large (where it decays, g e^g is below 0.4 and they are in the 1e-6)
    grow = float((a["A"].double() * oracle.step_size(a["dt"], a["dt_bias"], softplus)).max().clamp_min(0))
    assert _rel(a["state"], rh) < 1e-6 + grow * 2.0 ** -23
    return y


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("B,H,P,G,N,W", [(1, 8, 64, 1, 64, 4), (3, 6, 32, 2, 16, 4), (2, 4, 64, 1, 128, 2), (2, 2, 128, 2, 256, 8), (1, 1, 1, 1, 1, 3),
                                         (2, 3, 5, 1, 7, 4), (1, 32, 64, 1, 132, 4), (9, 4, 16, 4, 4, 5), (1, 2, 7, 1, 255, 4)])
def test_step_sizes(lb, dtype, B, H, P, G, N, W):
    check_step(lb, step_inputs(N + P, B, H, P, G, N, W, dtype))
    check_step(lb, dict(step_inputs(N, B, H, P, G, N, W, dtype, z=False, pitch=3, w_dtype=F32), D=None, conv_bias=None), activation=None, softplus=False)


@pytest.mark.parametrize("B,H,P,G,N,W,dtype", [(700, 2, 64, 2, 64, 4, BF), (40, 16, 64, 1, 128, 4, BF), (30, 16, 40, 1, 256, 3, FP), (160, 3, 5, 3, 20, 4, F32),
                                               (20, 32, 128, 1, 64, 4, BF), (19, 64, 256, 1, 16, 4, BF), (150, 2, 33, 1, 7, 4, BF)])
def test_step_many_rows(lb, B, H, P, G, N, W, dtype):
    """More clusters than the GPU holds at a time, and rows of a CTA that take several passes"""
    check_step(lb, step_inputs(B, B, H, P, G, N, W, dtype, pitch=1))


def test_steps_are_the_scan(lb):
    """conv + scan of a prompt, then steps: the same as conv + scan of all tokens, and as steps from the start"""
    H, P, G, N, W, B, T, more = 4, 64, 1, 64, 4, 2, 70, 5
    a = step_inputs(2, B, H, P, G, N, W, BF)
    gen = torch.Generator(device="cuda").manual_seed(3)
    ch = H * P + 2 * G * N
    u, dt = torch.randn(B, T + more, ch, generator=gen, device="cuda").to(BF), torch.randn(B, T + more, H, generator=gen, device="cuda").to(BF)
    par = {k: a[k] for k in ("A", "D", "dt_bias")}

    def prompt(n, cache=None, h0=None, t0=0):
        v, cache = lb.short_conv(u[:, t0:t0 + n], a["conv_weight"], a["conv_bias"], cache=cache, output_final_state=True)
        x, b, c = v[..., :H * P].unflatten(2, (H, P)), v[..., H * P:H * P + N].unflatten(2, (G, N)), v[..., H * P + N:].unflatten(2, (G, N))
        y, h = lb.state_space_scan(x, dt[:, t0:t0 + n], B=b, C=c, initial_state=h0, output_final_state=True, **par)
        return y, cache, h
    y_all, c_all, h_all = prompt(T + more)
    y, cache, h = prompt(T)
    for t in range(T, T + more):
        yt = lb.state_space_step(u[:, t], dt[:, t], cache, h, a["conv_weight"], a["conv_bias"], **par)
        assert float((yt.float() - y_all[:, t].float()).norm() / y_all[:, t].float().norm()) < 3 * 2.0 ** -8
    assert torch.equal(cache, c_all) and _rel(h, h_all.double()) < 2.0 ** -8       # (the prompt's convolution is rounded to bf16)
    y2, cache2, h2 = prompt(T - 30)
    _, cache2, h2 = prompt(30 + more, cache2, h2, T - 30)
    assert torch.equal(cache2, c_all) and _rel(h2, h_all.double()) < 1e-6


def test_step_in_a_graph(lb):
    a = step_inputs(4, 4, 8, 64, 1, 128, 4, BF)
    keep = {k: a[k].clone() for k in ("conv_cache", "state")}
    ys = [lb.state_space_step(**a) for _ in range(3)]
    end = {k: a[k].clone() for k in keep}
    for k, v in keep.items():
        a[k].copy_(v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lb.state_space_step(**a)
    torch.cuda.current_stream().wait_stream(s)
    for k, v in keep.items():
        a[k].copy_(v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lb.state_space_step(**a)
    for k, v in keep.items():
        a[k].copy_(v)
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ys[i])
    for k, v in end.items():
        assert torch.equal(a[k], v)


# ---- convolution -----------------------------------------------------------------------------------
def check_conv(lb, x, w, b, act, cache, cu, final=True, on_device=True):
    old = None if cache is None else cache.clone()
    y, new = lb.short_conv(x, w, b, act, cache=cache, output_final_state=final,
                           cu_seqlens=None if cu is None else torch.tensor(cu, device="cuda" if on_device else "cpu"))
    lb.check_status()
    ry, rc, ya = oracle.conv(x, w.reshape(x.shape[2], -1), b, act, old, cu)
    # fp32 sums of at most 9 terms, the fast exponential and division: 2^-20; the result's own rounding
    _near(y, ry, oracle.half_step(y.dtype) * ry.abs() + 2.0 ** -19 * (ya + ry.abs()) + 2.0 ** -25, "y")
    if final:
        assert torch.equal(new.double(), rc) and (cache is None or new is cache)
    else:
        assert new is None and (cache is None or torch.equal(cache, old))


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("B,T,D,W", [(1, 1, 8, 4), (2, 3, 64, 4), (1, 16, 24, 2), (3, 17, 40, 8), (1, 100, 7, 3), (2, 33, 513, 5), (1, 260, 1024, 4)])
def test_conv_sizes(lb, dtype, B, T, D, W):
    gen = torch.Generator(device="cuda").manual_seed(T + D)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    for pitch, act, bias, cached in ((0, "silu", True, True), (8, None, False, True), (3, "silu", True, False)):
        x = r(B, T, D + pitch)[..., :D]
        check_conv(lb, x, r(D, W), r(D) if bias else None, act, r(B, D, W) if cached else None, None)
        check_conv(lb, x, r(D, 1, W).float(), None, act, r(B, D, W) if cached else None, None, final=False)


@pytest.mark.parametrize("W", [2, 4, 7, 8])
@pytest.mark.parametrize("lens", [[1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1], [14, 3, 0, 15, 1, 2, 0, 0, 40], [0, 0, 5], [15, 17, 31, 1, 16], [13, 9, 2, 8, 70]])
def test_conv_packed(lb, W, lens):
    """Sequences that begin just before the end of a thread's run, shorter than the taps, and empty"""
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    gen = torch.Generator(device="cuda").manual_seed(W)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF)  # noqa: E731
    for D in (16, 5):
        check_conv(lb, r(1, cu[-1], D), r(D, W), r(D), "silu", r(len(lens), D, W), cu)
        check_conv(lb, r(1, cu[-1], D), r(D, W), r(D), "silu", None, cu, on_device=False)


def test_conv_long_and_its_caches_in_place(lb):
    """Many sequences at once, each cache read and written by the call"""
    gen = torch.Generator(device="cuda").manual_seed(0)
    lens = torch.randint(0, 60, (150,), generator=torch.Generator().manual_seed(1)).tolist()
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF)  # noqa: E731
    check_conv(lb, r(1, cu[-1], 256), r(256, 8), r(256), "silu", r(len(lens), 256, 8), cu)


def test_conv_offsets_on_the_device_are_checked(lb):
    x, w, cache = torch.randn(1, 100, 16, device="cuda", dtype=BF), torch.randn(16, 4, device="cuda", dtype=BF), torch.zeros(3, 16, 4, device="cuda", dtype=BF)
    for cu in ([0, 60, 30, 100], [0, 30, 60, 101], [-2, 30, 60, 100], [3, 30, 60, 100], [0, 300, 60, 100]):
        lb.short_conv(x, w, cache=cache, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"))
        with pytest.raises(lb.LampaError):
            lb.check_status()
    y, _ = lb.short_conv(x, w, cu_seqlens=torch.tensor([0, 30, 30, 90], device="cuda"))
    lb.check_status()
    assert (y[0, 90:] == 0).all()


# ---- norms around a block ---------------------------------------------------------------------------
def check_norm(lb, rows, D, dtype, out, seed=0, post=True, pre=True, gate="row", act=None, scale="vec", eps=1e-5, cu=None, post_norm=True, pitch=0, on_device=True, g_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(seed + rows + D)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    res, delta = r(rows, D), (2 * r(rows, D + pitch)).to(dtype)[:, :D]
    n = rows if cu is None else len(cu) - 1
    g = None if gate is None else r(n, D + pitch).to(g_dtype or dtype)[:, :D] if gate == "row" else r(D).to(g_dtype or dtype)
    sc = {"vec": r(D), "num": 0.37, None: None}[scale]
    pw, qw = (1 + 0.2 * r(D) if post else None), (1 + 0.2 * r(D) if pre else None)
    full = None if g is None else g if gate == "row" else g.expand(n, D)
    ry, rr, up = oracle.block_norm(res, delta, pw, qw, full, 1.0 if sc is None else sc, act, eps, cu, post_norm)
    got = lb.block_norm(res, delta, pw, qw, gate=g, scale=sc, gate_activation=act, eps=eps, post_norm=post_norm, out_dtype=out,
                        cu_seqlens=None if cu is None else torch.tensor(cu, device="cuda" if on_device else "cpu"))
    lb.check_status()
    # fp32: a sum of D squares (random roundings, 2^-20 for D up to 8192), square root, division, four products, the fast exponential
    _near(res, rr, 2.0 ** -20 * (rr.abs() + 2 * up) + 1e-30, "res")
    if out is None:
        assert got is None
        return
    err = 2.0 ** -19 * (ry.abs() + (rr.abs() + 2 * up) / (rr.square().mean(1, keepdim=True) + eps).sqrt() * (1 if qw is None else qw.abs()))
    _near(got, ry, oracle.half_step(out) * ry.abs() + err + 2.0 ** -25, "y")


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 4), (7, 96), (65, 128), (5, 130), (33, 1000), (9, 1024), (4, 1536), (3, 8192), (2, 4100), (2, 1537), (1, 8191)])
def test_norm_sizes(lb, dtype, rows, D):
    check_norm(lb, rows, D, dtype, dtype, act="sigmoid")
    check_norm(lb, rows, D, dtype, F32, gate=None, scale=None, post=False, pre=False)
    check_norm(lb, rows, D, dtype, BF, gate="one", act="silu", scale="num", pitch=4)
    check_norm(lb, rows, D, dtype, None, post_norm=False, pitch=1)
    check_norm(lb, rows, D, dtype, dtype, act="silu", g_dtype=F32)
    check_norm(lb, rows, D, dtype, dtype, act="silu", g_dtype=FP if dtype == BF else BF)


@pytest.mark.parametrize("D", [128, 1028, 33])
def test_norm_gates_per_sequence(lb, D):
    check_norm(lb, 300, D, BF, BF, cu=[0, 100, 100, 101, 300])
    check_norm(lb, 300, D, FP, F32, cu=[0, 100, 100, 101, 300], act="silu", on_device=False)
    check_norm(lb, 300, D, BF, BF, cu=[0, 0, 120, 250], act="sigmoid")             # rows of no sequence keep their residual


def test_norm_alone_and_many_rows(lb):
    res = torch.randn(40000, 64, device="cuda")
    keep = res.clone()
    y = lb.block_norm(res, None, out_dtype=F32)
    assert torch.equal(res, keep)
    _near(y, (keep.double() / (keep.double().square().mean(1, keepdim=True) + 1e-6).sqrt()), 1e-5, "y")
    check_norm(lb, 40001, 64, BF, BF, act="sigmoid")
    zero = torch.zeros(5, 64, device="cuda")
    assert (lb.block_norm(zero, torch.zeros(5, 64, device="cuda"), out_dtype=F32) == 0).all()


def test_norm_offsets_on_the_device_are_checked(lb):
    res, delta, gate = torch.randn(100, 32, device="cuda"), torch.randn(100, 32, device="cuda"), torch.randn(3, 32, device="cuda")
    for cu in ([0, 60, 30, 100], [0, 30, 60, 101], [-1, 30, 60, 100], [3, 30, 60, 100]):
        lb.block_norm(res, delta, gate=gate, cu_seqlens=torch.tensor(cu, device="cuda"))
        with pytest.raises(lb.LampaError):
            lb.check_status()


# ---- a block of a model ------------------------------------------------------------------------------
def test_block_together(lb):
    """LSH order, norm, projection, convolution, scan, norm, projection, norm behind the block with gate and scale, for a packed batch"""
    d, H, P, G, N, W = 96, 4, 32, 1, 64, 4
    gen = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    lens = [301, 0, 77, 500]
    cu = [0, 301, 301, 378, 878]
    off = torch.tensor(cu, device="cuda")
    n, ch = cu[-1], H * P + 2 * G * N
    x, gate = r(n, d), r(4, d).to(BF)
    w_in, w_out = (r(H * P + ch + H, d) / d ** 0.5).to(BF), (r(d, H * P) / (H * P) ** 0.5).to(BF)
    wc, bc, A, D, dtb = (0.5 * r(ch, W)).to(BF), (0.1 * r(ch)).to(BF), -(1 + 4 * torch.rand(H, generator=gen, device="cuda")), r(H), r(H) - 2
    w1, w2, w3, sc = 1 + 0.1 * r(d), 1 + 0.1 * r(d), 1 + 0.1 * r(d), 0.1 * r(d)

    res = x.clone()
    h = lb.block_norm(res, None, pre_weight=w1)
    row = h @ w_in.t()
    v, cache = lb.short_conv(row[None, :, H * P:H * P + ch], wc, bc, output_final_state=True, cu_seqlens=off)
    y, state = lb.state_space_scan(v[..., :H * P].unflatten(2, (H, P)), row[None, :, H * P + ch:], A, v[..., H * P:H * P + N].unflatten(2, (G, N)),
                                   v[..., H * P + N:].unflatten(2, (G, N)), D, row[None, :, :H * P].unflatten(2, (H, P)), dtb,
                                   output_final_state=True, cu_seqlens=off)
    o = y.view(n, H * P) @ w_out.t()
    nxt = lb.block_norm(res, o, w2, w3, gate=gate, scale=sc, gate_activation="sigmoid", cu_seqlens=off)
    lb.check_status()

    # the same in 64 bits, with the roundings to bf16 that the calls make between them
    rh, _, _ = oracle.block_norm(x, None, None, w1, None, 1.0, None, 1e-6, None, True)
    rh = rh.to(BF).double()
    rrow = (rh @ w_in.double().t()).to(BF)
    rv, rc, _ = oracle.conv(rrow[None, :, H * P:H * P + ch], wc, bc, "silu", None, cu)
    rv = rv.to(BF)
    ry, rs, _, _ = oracle.scan(rv[..., :H * P].unflatten(2, (H, P)), rrow[None, :, H * P + ch:], A, rv[..., H * P:H * P + N].unflatten(2, (G, N)),
                               rv[..., H * P + N:].unflatten(2, (G, N)), D, rrow[None, :, :H * P].unflatten(2, (H, P)), dtb, True, None, cu)
    ro = (ry.view(n, H * P).to(BF).double() @ w_out.double().t()).to(BF)
    rn, rres, _ = oracle.block_norm(x, ro, w2, w3, gate, sc, "sigmoid", 1e-6, cu, True)
    # relative to the norm of each: h, row, v, scores and y, o are rounded to bf16 (2^-8 at most, in different places: they add up as
    # squares) along the way, and a step size that moves by 2^-8 moves a whole decay: 8 half steps bound what is left
    for got, ref, k in ((cache, rc, 3), (state, rs, 8), (o, ro.double(), 8), (res, rres, 4), (nxt, rn, 4)):
        assert _rel(got, ref.double()) < k * 2.0 ** -8, (k, _rel(got, ref.double()))
