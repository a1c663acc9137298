"""Cases of the state space operators: the scan over whole sequences, its step for single tokens, the convolution in front of
them and the norms around the block they sit in.

  scan    state_space_scan: a prompt, an event in LSH order, a packed batch, a batch that continues from states
  step    state_space_step: convolution and recurrence of one token per stream, cache and state in place
  conv    short_conv: the convolution of a prompt that continues from a cache, which is advanced in place
  norm    block_norm: post-norm, gate, residual scale and the next block's pre-norm on an fp32 residual stream in place

A block's input projection writes one row [z | x B C | dt] per token; the convolution reads its x B C part in place and the scan
reads z and dt in place, so these inputs have the projection's row pitch.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TAPS = 4           # of the convolution
EPS = 1e-5
CHUNK = 128        # tokens per chunk of the plain form


def listed():
    return [
        # a prompt of a few tokens whose state is kept for the decode: latency
        dict(name="scan_37", kind="scan", seqs=1, tokens=37, packed=False, heads=8, p=64, n=64, groups=1, gated=False,
             initial=False, final=True, dtype="bf16"),
        # a small event, not padded, gated by z, no state kept
        dict(name="scan_6007", kind="scan", seqs=1, tokens=6007, packed=False, heads=8, p=64, n=64, groups=1, gated=True,
             initial=False, final=False, dtype="bf16"),
        # the largest event (60 000 hits padded to 61 440), a block twice as wide as its input
        dict(name="scan_61440", kind="scan", seqs=1, tokens=61440, packed=False, heads=16, p=64, n=128, groups=1, gated=True,
             initial=False, final=True, dtype="bf16"),
        # four streams that continue a chunk later, two groups of B and C
        dict(name="scan_4x2049", kind="scan", seqs=4, tokens=8196, packed=False, heads=16, p=64, n=128, groups=2, gated=False,
             initial=True, final=True, dtype="bf16"),
        # events of odd lengths packed, small heads, fp16 as the tracking configuration runs
        dict(name="scan_packed_fp16", kind="scan", seqs=7, tokens=24001, packed=True, heads=6, p=32, n=16, groups=1, gated=True,
             initial=True, final=True, dtype="fp16"),
        # one stream of single tokens: nothing but latency
        dict(name="step_b1", kind="step", batch=1, heads=8, p=64, n=64, groups=1, gated=True, dtype="bf16"),
        # five streams with odd heads
        dict(name="step_b5_fp16", kind="step", batch=5, heads=6, p=32, n=16, groups=2, gated=False, dtype="fp16"),
        # 64 streams: the states are 34 MB
        dict(name="step_b64", kind="step", batch=64, heads=16, p=64, n=128, groups=1, gated=True, dtype="bf16"),
        # convolution of a packed batch of odd lengths, each continuing from its cache
        dict(name="conv_packed_6007", kind="conv", seqs=3, tokens=6007, channels=640, pitch=1160, dtype="fp16"),
        # convolution of the largest event, in place of its projection's rows
        dict(name="conv_61440", kind="conv", seqs=1, tokens=61440, channels=1280, pitch=2320, dtype="bf16"),
        # norms around the block of one event at the model's width, gated token by token
        dict(name="norm_9001x128", kind="norm", rows=9001, width=128, seqs=1, per_seq=False, act="sigmoid", delta="bf16", out="bf16"),
        # the largest event in a wide model, one gate per event, scale per channel
        dict(name="norm_61440x1024", kind="norm", rows=61440, width=1024, seqs=5, per_seq=True, act="none", delta="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "step", "conv", "norm"])
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 40000), width=4 * _log(rng, 4, 384), seqs=rng.randint(1, 9), per_seq=rng.random() < 0.5,
                    act=rng.choice(["none", "sigmoid", "silu"]), delta=rng.choice(["bf16", "fp16", "fp32"]),
                    out=rng.choice(["bf16", "fp16", "fp32"]))
    if kind == "conv":
        channels = 8 * rng.randint(2, 160)
        return dict(kind=kind, seqs=rng.randint(1, 9), tokens=_log(rng, 40, 61440), channels=channels,
                    pitch=channels + 8 * rng.randint(0, 100), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    groups = rng.choice([1, 1, 2])
    heads = groups * _log(rng, 1, 8)
    p, n = rng.choice([16, 32, 64, 64, 96]), rng.choice([16, 32, 64, 128, 128])
    c = dict(kind=kind, heads=heads, p=p, n=n, groups=groups, gated=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "step":
        return dict(c, batch=_log(rng, 1, 64))
    seqs = rng.randint(1, 8)
    packed = rng.random() < 0.5
    tokens = _log(rng, 40, 40000)
    if not packed:
        tokens -= tokens % seqs
    return dict(c, seqs=seqs, tokens=tokens, packed=packed, initial=rng.random() < 0.5, final=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------------
def _lengths(case):
    """Lengths of the packed sequences: odd, unequal, the same for every seed; the largest is about half of all."""
    s, t = case["seqs"], case["tokens"]
    if not case.get("packed", True) or s == 1:
        return [t // s] * s
    w = [1 + (7 * i * i + 3 * i) % 11 for i in range(s)]
    cuts = [0] + [t * sum(w[:i + 1]) // sum(w) for i in range(s)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int64, device="cuda")


def _mixer(case, r, u):
    """Parameters of the recurrence: decays of 1 to 16 per unit of time, steps of 0.001 to 0.1 around which dt moves."""
    h = case["heads"]
    step = torch.exp(math.log(1e-3) + u(h) * (math.log(0.1) - math.log(1e-3)))
    return dict(A=-(1 + 15 * u(h)), D=1 + 0.1 * r(h), dt_bias=step + torch.log(-torch.expm1(-step)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    u = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    s = dict(case=case)
    if case["kind"] == "norm":
        rows, d, ns = case["rows"], case["width"], case["seqs"]
        dt = DTYPES[case["delta"]]
        lens = _lengths(dict(seqs=ns, tokens=rows))
        s.update(res=r(rows, d), delta=(2 * r(rows, d) * (0.2 + u(rows, 1))).to(dt), gate=r(ns if case["per_seq"] else rows, d).to(dt),
                 post=1 + 0.1 * r(d), pre=1 + 0.1 * r(d), scale=0.1 + 0.05 * r(d), cu=_offsets(lens) if case["per_seq"] else None,
                 lens=torch.tensor(lens, device="cuda"))
        return s
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "conv":
        t, d = case["tokens"], case["channels"]
        lens = _lengths(case)
        s.update(x=r(1, t, case["pitch"]).to(dt)[:, :, 16:16 + d] if case["pitch"] >= d + 16 else r(1, t, case["pitch"]).to(dt)[:, :, :d],
                 w=(r(d, TAPS) * 0.5).to(dt), b=(r(d) * 0.1).to(dt), cache=r(case["seqs"], d, TAPS).to(dt), cu=_offsets(lens),
                 lens=torch.tensor(lens, device="cuda"))
        return s
    h, p, n, g = case["heads"], case["p"], case["n"], case["groups"]
    s.update(_mixer(case, r, u))
    width, inner = 2 * h * p + 2 * g * n + h, h * p + 2 * g * n
    if case["kind"] == "step":
        b = case["batch"]
        row = r(b, width).to(dt)
        s.update(xbc=row[:, h * p:h * p + inner], dt=row[:, h * p + inner:], z=row[:, :h * p].unflatten(1, (h, p)) if case["gated"] else None,
                 w=(r(inner, TAPS) * 0.5).to(dt), b=(r(inner) * 0.1).to(dt), cache=r(b, inner, TAPS).to(dt), state=r(b, h, p, n) * 0.2)
        return s
    batch = 1 if case["packed"] else case["seqs"]
    t = case["tokens"] // batch
    lens = _lengths(case)
    row = r(batch, t, width).to(dt)
    xbc = F.silu(r(batch, t, inner)).to(dt)
    s.update(x=xbc[..., :h * p].unflatten(2, (h, p)), B=xbc[..., h * p:h * p + g * n].unflatten(2, (g, n)), C=xbc[..., h * p + g * n:].unflatten(2, (g, n)),
             dt=row[..., h * p + inner:], z=row[..., :h * p].unflatten(2, (h, p)) if case["gated"] else None,
             h0=r(case["seqs"], h, p, n) * 0.2 if case["initial"] else None, cu=_offsets(lens) if case["packed"] else None,
             lens=torch.tensor(lens, device="cuda"))
    return s


# ---- one pass --------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        import lampa_b200
        if kind == "scan":
            return lampa_b200.state_space_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                               initial_state=s["h0"], output_final_state=s["case"]["final"], cu_seqlens=s["cu"])
        if kind == "step":
            y = lampa_b200.state_space_step(s["xbc"], s["dt"], s["cache"], s["state"], s["w"], s["b"], s["A"], D=s["D"], z=s["z"],
                                            dt_bias=s["dt_bias"])
            return y, s["state"], s["cache"]
        if kind == "conv":
            return lampa_b200.short_conv(s["x"], s["w"], s["b"], cache=s["cache"], output_final_state=True, cu_seqlens=s["cu"])
        act = None if s["case"]["act"] == "none" else s["case"]["act"]
        y = lampa_b200.block_norm(s["res"], s["delta"], s["post"], s["pre"], gate=s["gate"], scale=s["scale"], gate_activation=act, eps=EPS,
                                  cu_seqlens=s["cu"], out_dtype=DTYPES[s["case"]["out"]])
        return y, s["res"]
    return {"scan": _scan, "step": _step, "conv": _conv, "norm": _norm}[kind](s)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _scan(s):
    """Chunks of 128 tokens that begin with their sequence: inside one the output is a masked matrix product, and the state that enters
    it is a sum over the earlier chunks of its sequence, each with the decay in between."""
    x, bm, cm, lens = s["x"].flatten(0, 1).float(), s["B"].flatten(0, 1).float(), s["C"].flatten(0, 1).float(), s["lens"]
    h, p, n = x.shape[1], x.shape[2], bm.shape[2]
    total, g = x.shape[0], bm.shape[1]
    d = _softplus(s["dt"].flatten(0, 1).float() + s["dt_bias"])
    chunks = (lens + CHUNK - 1) // CHUNK
    seq_of = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), chunks, output_size=int(_chunks(s["case"])))
    first = torch.cumsum(chunks, 0) - chunks
    within = (torch.arange(len(seq_of), device="cuda") - first[seq_of])[:, None] * CHUNK + torch.arange(CHUNK, device="cuda")
    there = within < lens[seq_of][:, None]                                               # [chunks, 128]
    row = torch.where(there, within + (torch.cumsum(lens, 0) - lens)[seq_of][:, None], 0)
    xs, bs, cs = x[row] * there[..., None, None], bm[row] * there[..., None, None], cm[row]
    ds = d[row] * there[..., None]                                                       # [c, 128, h]
    dec = torch.cumsum((ds * s["A"]).double(), 1)                                        # long sums of small steps: in 64 bits
    causal = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device="cuda").tril()
    gap = (dec[:, :, None] - dec[:, None]).masked_fill(~causal[..., None], -math.inf).float()
    score = torch.einsum("cign,cjgn->cijg", cs, bs).repeat_interleave(h // g, 3) * torch.exp(gap) * ds[:, None]
    y = torch.einsum("cijh,cjhp->cihp", score, xs)
    del score, gap
    left = torch.exp((dec[:, -1:] - dec).float()) * ds
    local = torch.einsum("cjhp,cjhn->chpn", xs * left[..., None], bs.repeat_interleave(h // g, 2))
    # entering state of chunk c: initial state decayed through the chunks before it, and their own parts
    end = torch.cumsum(dec[:, -1], 0)                                                    # [c, h], over all chunks
    before = end - dec[:, -1]
    same = (seq_of[:, None] == seq_of) & (torch.arange(len(seq_of), device="cuda")[:, None] > torch.arange(len(seq_of), device="cuda"))
    through = torch.exp((before[:, None] - end[None]).masked_fill(~same[..., None], -math.inf).float())
    enter = torch.einsum("ceh,ehpn->chpn", through, local)
    if s["h0"] is not None:
        live = lens > 0                                                                  # an empty sequence has no first chunk
        start = before[torch.where(live, first, 0)]
        enter = enter + torch.exp((before - start[seq_of]).float())[..., None, None] * s["h0"][seq_of]
    y = y + torch.exp(dec.float())[..., None] * torch.einsum("cihn,chpn->cihp", cs.repeat_interleave(h // g, 2), enter)
    out = torch.zeros(total, h, p, device="cuda")
    out[row[there]] = y[there]
    out = out + s["D"][:, None] * x
    if s["z"] is not None:
        out = out * _silu(s["z"].flatten(0, 1).float())
    out = out.to(s["x"].dtype).view(s["x"].shape)
    if not s["case"]["final"]:
        return out, None
    last = torch.cumsum(chunks, 0) - 1
    final = torch.exp(dec[last, -1].float())[..., None, None] * enter[last] + local[last]
    empty = (lens == 0)[:, None, None, None]
    return out, torch.where(empty, s["h0"] if s["h0"] is not None else torch.zeros_like(final), final)


def _chunks(case):
    return sum((n + CHUNK - 1) // CHUNK for n in _lengths(case))


def _step(s):
    h, p, n = s["state"].shape[1:]
    cache = s["cache"]
    cache.copy_(torch.cat([cache[..., 1:], s["xbc"][..., None]], -1))
    v = _silu((cache.float() * s["w"].float()).sum(-1) + s["b"].float())
    g = (v.shape[1] - h * p) // (2 * n)
    x, bm, cm = v[:, :h * p].unflatten(1, (h, p)), v[:, h * p:h * p + g * n].unflatten(1, (g, n)), v[:, h * p + g * n:].unflatten(1, (g, n))
    bm, cm = bm.repeat_interleave(h // g, 1), cm.repeat_interleave(h // g, 1)
    d = _softplus(s["dt"].float() + s["dt_bias"])
    s["state"].copy_(torch.exp(d * s["A"])[..., None, None] * s["state"] + (d[..., None] * x)[..., None] * bm[:, :, None])
    y = (s["state"] * cm[:, :, None]).sum(-1) + s["D"][:, None] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return y.to(s["xbc"].dtype), s["state"], s["cache"]


def _conv(s):
    x, lens, cache = s["x"][0], s["lens"], s["cache"]
    t, d = x.shape
    start = torch.cumsum(lens, 0) - lens
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), lens, output_size=t)
    rows = torch.cat([x, cache.transpose(1, 2).reshape(-1, d)])                          # behind the tokens: the caches' slots
    at = torch.arange(t, device="cuda")[:, None] - (TAPS - 1) + torch.arange(TAPS, device="cuda")
    local = at - start[seq][:, None]                                                     # negative: that many tokens before the sequence
    at = torch.where(local >= 0, at, t + seq[:, None] * TAPS + TAPS + local)
    y = s["b"].float() + (rows[at].float() * s["w"].float().t()).sum(1)
    end = lens[:, None] - TAPS + torch.arange(TAPS, device="cuda")
    keep = torch.where(end >= 0, start[:, None] + end, t + torch.arange(len(lens), device="cuda")[:, None] * TAPS + TAPS + end)
    cache.copy_(rows[keep].transpose(1, 2))
    return _silu(y).to(x.dtype)[None], cache


def _norm(s):
    act = {"none": lambda v: v, "sigmoid": lambda v: 1 / (1 + torch.exp(-v)), "silu": _silu}[s["case"]["act"]]
    o, res = s["delta"].float(), s["res"]
    gate = act(s["gate"].float())
    if s["cu"] is not None:
        gate = torch.repeat_interleave(gate, s["lens"], 0, output_size=res.shape[0])
    res += s["scale"] * gate * (o / torch.sqrt((o * o).mean(1, keepdim=True) + EPS) * s["post"])
    y = res / torch.sqrt((res * res).mean(1, keepdim=True) + EPS) * s["pre"]
    return y.to(DTYPES[s["case"]["out"]]), res


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        e, o = DTYPES[case["delta"]].itemsize, DTYPES[case["out"]].itemsize
        rows, d = case["rows"], case["width"]
        return {"bytes": rows * d * (8 + e + o) + (case["seqs"] if case["per_seq"] else rows) * d * e + 12 * d, "flops": 12 * rows * d}
    e = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "conv":
        return {"bytes": 2 * e * case["channels"] * (case["tokens"] + TAPS * case["seqs"]), "flops": 2 * TAPS * case["channels"] * case["tokens"]}
    h, p, n, g = case["heads"], case["p"], case["n"], case["groups"]
    if case["kind"] == "step":
        b, inner = case["batch"], h * p + 2 * g * n
        return {"bytes": b * (8 * h * p * n + e * (inner * (1 + 2 * TAPS) + h + (2 if case["gated"] else 1) * h * p)) + e * inner * (TAPS + 1),
                "flops": b * (5 * h * p * n + 2 * TAPS * inner)}
    t, states = case["tokens"], case["seqs"] * h * p * n * 4
    return {"bytes": e * t * ((3 if case["gated"] else 2) * h * p + 2 * g * n + h) + states * (case["initial"] + case["final"]),
            "flops": 4 * t * h * p * n}


# ---- the definition in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "step": _exact_step, "conv": _exact_conv, "norm": _exact_norm}[case["kind"]](case, s)


def _exact_scan(case, s):
    """Token by token, all sequences at once, as the recurrence says."""
    lens = _lengths(case)
    h, p, n, rep = case["heads"], case["p"], case["n"], case["heads"] // case["groups"]
    A, D = s["A"].double(), s["D"].double()
    x, dt = s["x"].reshape(-1, h, p).double(), s["dt"].reshape(-1, h).double()
    bm, cm = s["B"].reshape(-1, case["groups"], n).double(), s["C"].reshape(-1, case["groups"], n).double()
    d = torch.logaddexp(dt + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    a, dx = torch.exp(d * A)[..., None, None], d[..., None] * x
    state = s["h0"].double() if s["h0"] is not None else torch.zeros(len(lens), h, p, n, dtype=torch.float64, device="cuda")
    y = torch.empty_like(x)
    starts = [sum(lens[:i]) for i in range(len(lens))]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])                            # longest first: those still running are a prefix
    state = state[order].clone()
    for t in range(max(lens)):
        live = sum(lens[i] > t for i in order)
        if live == 1:
            at = starts[order[0]] + t
            i = slice(at, at + 1)
        else:
            i = torch.tensor([starts[j] + t for j in order[:live]], device="cuda")
        run_ = state[:live]
        run_.mul_(a[i]).add_(dx[i][..., None] * bm[i].repeat_interleave(rep, 1)[:, :, None])
        y[i] = torch.matmul(run_, cm[i].repeat_interleave(rep, 1)[..., None])[..., 0]
    y += D[:, None] * x
    if s["z"] is not None:
        z = s["z"].reshape(-1, h, p).double()
        y *= z * torch.sigmoid(z)
    final = torch.empty_like(state)
    final[order] = state
    return y.view(s["x"].shape), final if case["final"] else None


def _exact_step(case, s):
    h, p, n, g = case["heads"], case["p"], case["n"], case["groups"]
    taps = torch.cat([s["cache"][:, :, 1:], s["xbc"].unsqueeze(2)], 2).double()
    v = torch.einsum("bdw,dw->bd", taps, s["w"].double()) + s["b"].double()
    v = v * torch.sigmoid(v)
    x, bm, cm = torch.split(v, [h * p, g * n, g * n], 1)
    x, bm, cm = x.view(-1, g, h // g, p), bm.view(-1, g, n), cm.view(-1, g, n)
    d = torch.logaddexp(s["dt"].double() + s["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda")).view(-1, g, h // g)
    state = s["state"].double().view(-1, g, h // g, p, n) * torch.exp(d * s["A"].double().view(g, -1))[..., None, None]
    state += torch.einsum("bgh,bghp,bgn->bghpn", d, x, bm)
    y = torch.einsum("bghpn,bgn->bghp", state, cm) + s["D"].double().view(g, -1, 1) * x
    y = y.reshape(-1, h, p)
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    return y, state.reshape(s["state"].shape), taps


def _exact_conv(case, s):
    """Sequence by sequence, with the cache's slots in front of its tokens."""
    x, w, b, outs, caches, at = s["x"][0].double(), s["w"].double(), s["b"].double(), [], [], 0
    for i, n in enumerate(_lengths(case)):
        seq = torch.cat([s["cache"][i].double().t(), x[at:at + n]])                     # slots 1 .. 3 of the cache are the last three tokens
        y = F.conv1d(seq[1:].t()[None], w[:, None], b, groups=w.shape[0])[0].t()
        outs.append(y * torch.sigmoid(y))
        caches.append(seq[n:n + TAPS].t())
        at += n
    return torch.cat(outs)[None], torch.stack(caches)


def _exact_norm(case, s):
    o, res, gate = s["delta"].double(), s["res"].double(), s["gate"].double()
    gate = torch.sigmoid(gate) * (gate if case["act"] == "silu" else 1) if case["act"] != "none" else gate
    if case["per_seq"]:
        gate = torch.cat([gate[i].expand(n, -1) for i, n in enumerate(_lengths(dict(seqs=case["seqs"], tokens=case["rows"])))])
    o = o * torch.rsqrt(o.square().mean(1, keepdim=True) + EPS) * s["post"].double()
    res = res + gate * s["scale"].double() * o
    return res * torch.rsqrt(res.square().mean(1, keepdim=True) + EPS) * s["pre"].double(), res
