"""The state space operators in 64 bits, token by token, and how far a kernel may be from them.

Each function also returns the same sums taken over absolute values: an error that is a rounding of the operands, of the scores or of
a state is at most that many roundings times this sum, whatever cancels in the result itself.
"""
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def silu(v):
    return v * torch.sigmoid(v)


def step_size(dt, bias, softplus):
    d = dt.double() + (0 if bias is None else bias.double())
    return torch.logaddexp(d, torch.zeros((), dtype=torch.float64, device=d.device)) if softplus else d


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, h0=None, cu=None):
    """(y, final state, |y|-sum, |state|-sum) of x [B,T,H,P]; cu: list of offsets, or None"""
    Bn, T, H, P = x.shape
    G, N = B.shape[2:]
    dev = x.device
    spans = [(b * T, (b + 1) * T) for b in range(Bn)] if cu is None else list(zip(cu[:-1], cu[1:]))
    xf, bf, cf = x.reshape(-1, H, P).double(), B.reshape(-1, G, N).double().repeat_interleave(H // G, 1), C.reshape(-1, G, N).double().repeat_interleave(H // G, 1)
    d = step_size(dt.reshape(-1, H), dt_bias, softplus)
    a = torch.exp(d * A.double())
    Dv = torch.zeros(H, dtype=torch.float64, device=dev) if D is None else D.double()
    y, ya = torch.zeros_like(xf), torch.zeros_like(xf)
    ht = torch.zeros(len(spans), H, P, N, dtype=torch.float64, device=dev)
    ha = torch.zeros_like(ht)
    for s, (t0, t1) in enumerate(spans):
        h = torch.zeros(H, P, N, dtype=torch.float64, device=dev) if h0 is None else h0[s].double().clone()
        m = h.abs()
        for t in range(t0, t1):
            new = (d[t][:, None] * xf[t])[:, :, None] * bf[t][:, None]
            h = a[t][:, None, None] * h + new
            m = a[t][:, None, None] * m + new.abs()
            y[t] = (h * cf[t][:, None]).sum(-1) + Dv[:, None] * xf[t]
            ya[t] = (m * cf[t].abs()[:, None]).sum(-1) + (Dv[:, None] * xf[t]).abs()
        ht[s], ha[s] = h, m
    if z is not None:
        g = silu(z.reshape(-1, H, P).double())
        y, ya = y * g, ya * g.abs()
    return y.view(x.shape), ht, ya.view(x.shape), ha


def y_bound(dtype, sums):
    """bf16: one rounding of scores or state (whose sum is `sums`) and one of the result, 2^-8 each, and a twentieth for the
    fp32 arithmetic around them (exponents up to 100 off by 2^-23 each: 2^-16, products of 2^-24).  fp16: scores, state and inputs
    are two bf16 pieces (2^-16 each with the dropped product), exponents as before: 2^-13 in all, the result 2^-11 and at
    least half the smallest number, 2^-25."""
    if dtype == torch.bfloat16:
        return 2.1 * 2.0 ** -8 * sums + 1e-37
    return (2.0 ** -11 + 2.0 ** -13) * sums + 2.0 ** -25


def state_bound(sums, tokens):
    """Terms in three bf16 pieces: 2^-24.  Sums of 64 products that are rounded or cut at every one of 12 steps: 2^-23 each, 12 of
    them; one rounding per chunk of 64 tokens; exponentials of sums up to 100 whose steps and adding are good to 2^-23: 100 * 2 * 2^-23 at
    the most where the weight is e^-100, below 2^-21 where it counts (x e^-x < 0.4), 2^-20 for step, exponential and product."""
    return (16 + tokens / 64 + 8) * 2.0 ** -23 * sums + 1e-37


def conv(x, w, b, act, cache, cu):
    """(y, new cache, |y|-sum) of x [B,T,D]; cache [N,D,W] or None"""
    Bn, T, D = x.shape
    W = w.shape[1]
    spans = [(i * T, (i + 1) * T) for i in range(Bn)] if cu is None else list(zip(cu[:-1], cu[1:]))
    xf = x.reshape(-1, D).double()
    y, ya, new = torch.zeros_like(xf), torch.zeros_like(xf), []
    for s, (t0, t1) in enumerate(spans):
        old = torch.zeros(W, D, dtype=torch.float64, device=x.device) if cache is None else cache[s].double().t()
        seq = torch.cat([old, xf[t0:t1]])
        for t in range(t1 - t0):
            win = seq[t + 1:t + 1 + W]
            y[t0 + t] = (win * w.double().t()).sum(0) + (0 if b is None else b.double())
            ya[t0 + t] = (win * w.double().t()).abs().sum(0) + (0 if b is None else b.double().abs())
        new.append(seq[-W:].t())
    return (silu(y) if act else y).view(x.shape), torch.stack(new), ya.view(x.shape)


def block_norm(res, delta, post, pre, gate, scale, act, eps, cu, post_norm):
    """(y, new res, size of the update) in 64 bits; scale a number or [D]"""
    r = res.double()
    up = torch.zeros_like(r)
    if delta is not None:
        o = delta.double()
        if post_norm:
            o = o / torch.sqrt(o.square().mean(1, keepdim=True) + eps)
        if post is not None:
            o = o * post.double()
        has = torch.ones(r.shape[0], 1, dtype=torch.bool, device=r.device)
        if gate is not None:
            g = gate.double()
            g = g if act is None else torch.sigmoid(g) * (g if act == "silu" else 1)
            if cu is not None:
                full = torch.zeros_like(r)
                has[:] = False
                for s, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
                    full[a:b] = g[s]
                    has[a:b] = True
                g = full
            o = o * g
        up = torch.where(has, o * (scale.double() if isinstance(scale, torch.Tensor) else scale), 0)
    r = r + up
    y = r / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    return (y if pre is None else y * pre.double()), r, up.abs()
