"""The state space operators where a call is allowed but out of the ordinary, against the recurrence in 64 bits with the bounds of ssm_oracle.py."""
import pytest
import torch

from tests.test_gpu_state_space import BF, F32, FP, check_conv, check_scan, check_step, lb, scan_inputs, step_inputs  # noqa: F401  (lb is a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _checked_by_the_tests(monkeypatch):
    monkeypatch.setenv("LAMPA_B200_CHECK", "0")


@pytest.fixture(params=["tcgen05", "mma.sync"])
def form(request, lb):  # noqa: F811
    from lampa_b200 import _lib
    _lib.lib().lampa_debug_force_mma_sync(int(request.param == "mma.sync"))
    yield request.param
    _lib.lib().lampa_debug_force_mma_sync(0)


# ---- scan: large steps among small ones --------------------------------------------------------------
RESETS = {"sixth": [5], "some": [5, 70, 71, 127, 128, 200, 263], "seventh": list(range(0, 300, 7)), "second": list(range(1, 300, 2))}


def reset_inputs(dtype, large, where, softplus, own, seed=21):
    """Steps of 0.001 to 0.1 with `large` at some tokens, A = -16 and -1; own: these tokens add to the state, else their x is zero"""
    a = scan_inputs(seed, 1, 300, 2, 64, 1, 64, dtype, z=True, h0=True, dt_dtype=F32)
    a["A"] = torch.tensor([-16.0, -1.0], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d = 0.001 + 0.099 * torch.rand(1, 300, 2, generator=gen, device="cuda")
    dt = torch.log(torch.expm1(d)) if softplus else d
    dt[:, RESETS[where]] = large
    a.update(dt=dt, dt_bias=None)
    if not own:
        x = a["x"].clone()
        x[:, RESETS[where]] = 0
        a["x"] = x
    return a


@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("large", [6.0, 1e3, 1e4, 1e6, 1e30])
@pytest.mark.parametrize("where", list(RESETS))
def test_scan_small_steps_behind_a_large_one(lb, form, dtype, large, where, softplus):  # noqa: F811
    """A large step resets the state; the tokens behind it in its chunk are as exact as any"""
    if dtype == FP and form == "tcgen05":
        pytest.skip("fp16 has the mma.sync form only")
    for own in (False, True):
        check_scan(lb, reset_inputs(dtype, large, where, softplus, own), softplus=softplus)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_scan_decay_beyond_the_largest_float(lb, form, dtype):  # noqa: F811
    """A d below the lowest finite float is a decay of zero, also for the tokens behind it"""
    a = reset_inputs(dtype, 1e35, "some", False, False)
    a["A"] = torch.tensor([-1e4, -2.0], device="cuda")
    a["dt"][..., 0] = torch.where(a["dt"][..., 0] < 1, a["dt"][..., 0] * 1e-3, a["dt"][..., 0])
    check_scan(lb, a, softplus=False)


# ---- scan: one of two waiting warps gives up -----------------------------------------------------------
@pytest.mark.parametrize("products,others", [(0, 1 << 16), (1, 1 << 16), (1 << 16, 0), (1 << 16, 1), (0, 1), (1, 0)])
def test_scan_one_warp_gives_up(lb, products, others):  # noqa: F811
    """The output pass ends and says so whichever of its two waiting warps runs out (test_state_space_handover.py has the model), and the next call is right"""
    from lampa_b200 import _lib
    for H, T, z in ((4, 1000, True), (48, 1500, True), (48, 1500, False)):       # blocks of one chunk, and of several
        a = scan_inputs(12, 1, T, H, 64, 1, 128, BF, z=z, h0=True)
        want = lb.state_space_scan(**a, output_final_state=True)
        try:
            assert _lib.lib().lampa_debug_set_poll_budget(others) == 0 and _lib.lib().lampa_debug_set_product_poll_budget(products) == 0
            lb.state_space_scan(**a, output_final_state=True)
            torch.cuda.synchronize()
        finally:
            _lib.lib().lampa_debug_set_poll_budget(1 << 22)
        if 0 in (products, others):
            with pytest.raises(lb.LampaError):
                lb.check_status()
        else:                                      # a single poll may wait long enough in hardware to succeed
            try:
                lb.check_status()
            except lb.LampaError:
                pass
        again = lb.state_space_scan(**a, output_final_state=True)
        lb.check_status()
        assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])


# ---- scan: what a state is kept for ----------------------------------------------------------------------
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_scan_of_a_batch_whose_sequences_are_one_block_each(lb, form, dtype, given):  # noqa: F811
    """Several chunks, no workspace: the block kernel of the tcgen05 form goes from the entering state to the final one"""
    for P, N in ((64, 128), (40, 24)):
        a = scan_inputs(41 + P, 10, 300, 32, P, 1, N, dtype, z=True, h0=given, decay=0.1)
        y, _ = check_scan(lb, a)
        assert torch.equal(y, lb.state_space_scan(**a)[0])


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_scan_of_a_packed_batch_that_one_sequence_dominates(lb, form, dtype, given):  # noqa: F811
    lens = [40] * 7 + [0, 4500, 0, 300, 1, 1000, 129, 128]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    a = scan_inputs(43, 1, cu[-1] + 5, 8, 64, 1, 64, dtype, z=True, h0=given, nseq=len(lens))
    off = torch.tensor(cu, device="cuda")
    y, ht = lb.state_space_scan(**a, output_final_state=True, cu_seqlens=off)
    assert (y[0, cu[-1]:] == 0).all()
    cut = {k: (v[:, :cu[-1]] if k in ("x", "dt", "B", "C", "z") else v) for k, v in a.items()}
    check_scan(lb, cut, cu)
    check_scan(lb, cut, cu, final=False)
    for s, n in enumerate(lens):
        if n == 0:
            assert torch.equal(ht[s], a["initial_state"][s] if given else torch.zeros_like(ht[s]))


def test_scan_of_many_prompts_takes_little_scratch(lb):  # noqa: F811
    """16 384 packed prompts of 40 tokens: what a call allocates beside y is not a state to each of them"""
    n, H, P, N = 16384, 4, 64, 64
    a = scan_inputs(44, 1, 40 * n, H, P, 1, N, BF)
    off = torch.arange(n + 1, device="cuda") * 40
    lb.state_space_scan(**a, cu_seqlens=off)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y, _ = lb.state_space_scan(**a, cu_seqlens=off)
    assert torch.cuda.max_memory_allocated() - before - 2 * y.numel() < 100 << 20        # a state each would be 1 GB
    lb.check_status()


# ---- scan: x, B and C that lie at odd places ----------------------------------------------------------
@pytest.mark.parametrize("what", ["x", "B", "C"])
def test_scan_of_dense_inputs_at_odd_places(lb, what):  # noqa: F811
    """Dense, but not on a 16-byte boundary: copied to one, so that the same kernels run"""
    a = {k: v.contiguous() if isinstance(v, torch.Tensor) else v for k, v in scan_inputs(31, 1, 400, 2, 64, 1, 64, BF).items()}
    want = lb.state_space_scan(**a, output_final_state=True)
    buf = torch.zeros(a[what].numel() + 8, dtype=BF, device="cuda")
    odd = buf[1:1 + a[what].numel()].view(a[what].shape)
    odd.copy_(a[what])
    assert odd.is_contiguous() and odd.data_ptr() % 16
    got = lb.state_space_scan(**dict(a, **{what: odd}), output_final_state=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- a convolution's bias of a type of its own ---------------------------------------------------------
@pytest.mark.parametrize("w_dtype,b_dtype", [(BF, F32), (FP, F32), (BF, FP), (FP, BF), (F32, BF)])
def test_bias_keeps_its_bits(lb, w_dtype, b_dtype):  # noqa: F811
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, w, b = r(2, 50, 24).to(F32), (0.01 * r(24, 4)).to(w_dtype), (1 + r(24).abs()).to(b_dtype)
    check_conv(lb, x, w, b, None, r(2, 24, 4), None)
    a = step_inputs(6, 3, 2, 8, 1, 8, 4, F32, w_dtype=w_dtype)
    a.update(conv_weight=a["conv_weight"] * 0.01, conv_bias=(1 + r(32).abs()).to(b_dtype))
    check_step(lb, a)


# ---- the C entry point of a scan over no tokens ----------------------------------------------------------
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("given", [False, True])
def test_scan_entry_point_of_no_tokens_has_a_final_state(lb, packed, given):  # noqa: F811
    import ctypes
    from lampa_b200 import _lib as L
    h0 = torch.randn(3, 2, 5, 7, device="cuda") if given else None
    ht = torch.full((3, 2, 5, 7), 9.0, device="cuda")
    cu = torch.zeros(4, dtype=torch.int64, device="cuda") if packed else None
    d = L.SsmDesc(B=1 if packed else 3, T=0, H=2, P=5, N=7, G=1, nseq=3 if packed else 0, dtype=0, dt_dtype=0, dt_softplus=1)
    dev = torch.device("cuda:0")
    rc = L.lib().lampa_ssm_scan(ctypes.byref(d), None, 0, 0, None, 0, None, None, 0, 0, None, 0, 0, None, None, 0, 0, None,
                                L.ptr(h0), L.ptr(cu), None, L.ptr(ht), None, 0, L.ptr(L.status_word(dev)), L.stream_ptr(dev))
    assert rc == 0
    lb.check_status()
    assert torch.equal(ht, h0 if given else torch.zeros_like(ht))
    if packed:                                     # offsets that leave the (empty) input
        cu[1] = 4
        L.check(L.lib().lampa_ssm_scan(ctypes.byref(d), None, 0, 0, None, 0, None, None, 0, 0, None, 0, 0, None, None, 0, 0, None,
                                       L.ptr(h0), L.ptr(cu), None, L.ptr(ht), None, 0, L.ptr(L.status_word(dev)), L.stream_ptr(dev)), "lampa_ssm_scan")
        with pytest.raises(lb.LampaError):
            lb.check_status()


# ---- scan: values that are not finite ---------------------------------------------------------------------
@pytest.mark.parametrize("H", [2, 256])           # blocks of one chunk, and of all of a sequence's
@pytest.mark.parametrize("dtype", [BF, FP])
def test_scan_spreads_nothing_that_is_not_finite(lb, form, dtype, H):  # noqa: F811
    """NaN and infinity spoil their sequence from their token on, an x only its column and a dt only its head, in both forms and types"""
    cu = [0, 70, 370, 410, 540]
    off = torch.tensor(cu, device="cuda")
    a = scan_inputs(51, 1, 540, H, 64, 1, 64, dtype, z=True, h0=True, nseq=4)
    clean, hc = lb.state_space_scan(**a, output_final_state=True, cu_seqlens=off)
    assert torch.isfinite(clean).all() and torch.isfinite(hc).all()
    keep = [i for i in range(64) if i != 9]
    for what, t in (("x", 100), ("x", 134), ("x", 369), ("dt", 200), ("dt", 71), ("B", 70), ("B", 260), ("C", 150), ("initial_state", 70)):
        for bad in (float("nan"), float("inf"), -float("inf")):
            if what == "dt" and bad < 0:
                continue                           # a step of zero
            b = dict(a, **{what: a[what].clone()})
            if what == "dt":
                b["dt"][0, t, 1] = bad
            elif what == "initial_state":
                b[what][1, 0, 9, 5] = bad
            else:
                b[what][0, t, 0, 9] = bad
            y, ht = lb.state_space_scan(**b, output_final_state=True, cu_seqlens=off)
            lb.check_status()
            where = f"{what} {bad} at {t}"
            for s in (0, 2, 3):
                assert torch.equal(y[0, cu[s]:cu[s + 1]], clean[0, cu[s]:cu[s + 1]]) and torch.equal(ht[s], hc[s]), where
            assert torch.equal(y[0, 70:t], clean[0, 70:t]), where
            if what in ("x", "initial_state"):
                # (a state's infinity may meet a decay that has become zero, and then is NaN as 0 * inf is in the recurrence)
                assert not torch.isfinite(y[0, t:370, 0, 9]).any() and torch.equal(y[0, 70:370, 0][:, keep], clean[0, 70:370, 0][:, keep]), where
                assert torch.equal(y[0, 70:370, 1:], clean[0, 70:370, 1:]) and torch.equal(ht[1, 0, keep], hc[1, 0, keep]) and torch.equal(ht[1, 1:], hc[1, 1:]), where
                assert not torch.isfinite(ht[1, 0, 9] if what == "x" else ht[1, 0, 9, 5]).any(), where
            elif what == "dt":
                assert not torch.isfinite(y[0, t:370, 1]).any() and not torch.isfinite(ht[1, 1]).any(), where
                others = [h for h in range(H) if h != 1]
                assert torch.equal(y[0, 70:370][:, others], clean[0, 70:370][:, others]) and torch.equal(ht[1, others], hc[1, others]), where
            elif what == "B":
                assert not torch.isfinite(y[0, t:370]).any() and not torch.isfinite(ht[1, :, :, 9]).any(), where
                assert torch.equal(ht[1][..., keep], hc[1][..., keep]), where
            else:
                assert not torch.isfinite(y[0, t]).any() and torch.equal(y[0, t + 1:370], clean[0, t + 1:370]) and torch.equal(ht, hc), where
