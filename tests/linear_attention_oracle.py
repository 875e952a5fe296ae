"""64-bit forms of the linear-attention block's operators with bounds on the rounding of a computation in float32 sums
(torch in float64, step by step; no code of the package).

Units: U = 2^-24 is half a step of float32.  Each value comes with its size, the same sums over absolute values.

Step by step a state's entry takes three roundings a step (the fade's own, its product, the sum), each at most U of the
entry's size, which is never less than what is left of earlier sizes: after n steps at most 3 n U of its size,
2 U an addition where an accumulator may cut instead of rounding.  A product with it adds its K terms.  So steps(n, K) U
bounds every result of n steps, whatever the order of the sums.

The tensor-core path rounds q k^T times the fade, and the state as it meets q, to the tensors' type once: half a step of
it, relative.  float16 operands are first scaled by a power of two that brings the largest entry of their row into [1, 2):
smaller ones keep 2^-25 of that at least.  The products that a state is made of have operands of 22 bits or more, relative to the
largest of their block in float16: 2^-22 of that."""
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # eps / 2
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def rounding(value, kind):
    """How far rounding `value` to a type may move it."""
    return HALF_STEP[kind] * value.abs() + TINY[kind]


def _run(a, b, v, l, x, back):
    """X_t = l X_{t-1} + b_t v_t^T, out_t = X_t^T a_t over [T, H, D]; back: time runs down, X carried after its fade."""
    out = torch.zeros_like(v)
    x = x.clone()
    for t in (range(v.shape[0] - 1, -1, -1) if back else range(v.shape[0])):
        if not back:
            x = l * x
        x = x + b[t][..., :, None] * v[t][..., None, :]
        out[t] = (x * a[t][..., :, None]).sum(-2)
        if back:
            x = l * x
    return out, x


def attention(q, k, v, log_decay, s0, borders, scale, do=None, ds=None):
    """Rows [L, H, D] (k, v [L, Hk, D]) in float64; borders: (first, past) of each sequence.  {name: (value, size)}."""
    shared = q.shape[1] // k.shape[1]
    l = torch.exp(log_decay.double())[:, None, None]
    wide = lambda t: t.repeat_interleave(shared, 1)  # noqa: E731

    def passes(q, k, v, s0, do, ds):
        k, v = wide(k), wide(v)
        like = {"o": v, "dq": q, "dk": k, "dv": v}
        out = {n: torch.zeros_like(t) for n, t in like.items() if n == "o" or do is not None}
        ends = {"s": torch.zeros_like(s0), "ds0": torch.zeros_like(s0)}
        for i, (a, b) in enumerate(borders):
            z = slice(a, b)
            o, ends["s"][i] = _run(q[z], k[z], v[z], l, s0[i], False)
            out["o"][z] = scale * o
            if do is None:
                continue
            out["dq"][z] = scale * _run(do[z], v[z], k[z], l, s0[i].mT, False)[0]
            out["dv"][z], ends["ds0"][i] = _run(k[z], scale * q[z], do[z], l, ds[i], True)
            out["dk"][z] = _run(v[z], scale * do[z], q[z], l, ds[i].mT, True)[0]
        for n in ("dk", "dv"):
            if n in out:
                out[n] = out[n].unflatten(1, (-1, shared)).sum(2)
        return {**out, **(ends if do is not None else {"s": ends["s"]})}

    given = (q, k, v, s0, do, ds)
    value = passes(*given)
    scale = abs(scale)
    size = passes(*(None if t is None else t.abs() for t in given))
    return {n: (value[n], size[n]) for n in value}


def steps(n, K):
    """Units of a result of n steps over K places (and what sums over shared heads and scales add)."""
    return 6 * n + 2 * K + 32


def layer_norm(x, w, b, eps, dy=None):
    """{name: (value, bound before the rounding to the output's type)} over rows [R, C] in float64.

    mean: C additions, (C + 2) U of mean |x|; the centred value takes that and its own rounding, e_d; the variance is the
    mean of squares, off by 2 e_d |d| and (C + 4) U of itself, and half of that, relatively, is the standard deviation's
    (and 4 U for the quotient and the root).  Sums over rows: (R + 4) U of the sum of sizes."""
    C, R = x.shape[1], x.shape[0]
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True) + eps
    rstd = var.rsqrt()
    de = (C + 2) * U * x.abs().mean(1, keepdim=True) + U * d.abs()
    rel = ((2 * de * d.abs() + de * de).mean(1, keepdim=True) / var + (C + 8) * U) / 2 + 4 * U  # of rstd
    hat = d * rstd
    he = (de * rstd + hat.abs() * (rel + 2 * U)) * 1.01
    out = {"y": (hat * w + b, he * w.abs() + 2 * U * ((hat * w).abs() + b.abs()))}
    if dy is None:
        return out
    g = dy * w
    ge = U * g.abs()
    m1, m2 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    m1e = (C + 4) * U * g.abs().mean(1, keepdim=True)
    m2e = (he * g.abs() + (C + 6) * U * (g * hat).abs()).mean(1, keepdim=True)
    inner = g - m1 - hat * m2
    ie = ge + m1e + he * m2.abs() + (hat.abs() + he) * m2e + 4 * U * (g.abs() + m1.abs() + (hat * m2).abs())
    out["dx"] = (rstd * inner, rstd * (ie * 1.01 + inner.abs() * (rel + 2 * U)))
    out["dw"] = ((dy * hat).sum(0), (dy.abs() * he).sum(0) + (R + 4) * U * (dy * hat).abs().sum(0))
    out["db"] = (dy.sum(0), (R + 4) * U * dy.abs().sum(0))
    return out


def used(got, value, bound, kind):
    """The largest share of its allowed error that any element of `got` uses (to be <= 1; a NaN uses infinitely much)."""
    allowed = bound + rounding(value.abs() + bound, kind)
    if not value.numel():
        return 0.0
    share = (got.detach().double().cpu() - value.cpu()).abs() / allowed.cpu()
    return float(torch.where(share.isnan(), torch.inf, share).max())
