"""The operators of a linear-attention block, measured at the sizes that they are used at.

Reached through ``csn_b200.ops``:

* ``linear_attention(q, k, v, log_decay, s0, cu_seqlens, scale)`` -- attention without a softmax, whose memory of
  head h fades by exp(log_decay[h]) a step:
      S_t = exp(log_decay) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
  over a dense [B, T, H, D] batch or packed [L, H, D] sequences, k and v with as many heads as q or fewer (each
  shared by neighbouring heads of q), with its backward pass;
* ``linear_attention_step(q, k, v, log_decay, s, scale)`` -- the same advanced by one token, the float32 state
  [B, H, Dk, Dv] in place;
* ``layer_norm(x, weight, bias, eps)`` -- y = (x - mean) / sqrt(var + eps) weight + bias over the last axis of 16-bit
  rows of any width, with its backward pass.

``own`` chooses between the plain forms below and the framework's kernels.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "clifford-space-network_b200")
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5


def _ops():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from csn_b200 import ops
    return ops


# ------------------------------------------------------------------------- cases
def _attention(name, kind, batch, length, heads, shared, dk, dv, train, packed=False):
    return {"name": name, "op": "attention", "type": kind, "batch": batch, "length": length, "heads": heads,
            "shared": shared, "dk": dk, "dv": dv, "train": train, "packed": packed}


def _norm(name, kind, rows, channels, train, wide_weights=False):
    return {"name": name, "op": "norm", "type": kind, "rows": rows, "channels": channels, "train": train,
            "wide_weights": wide_weights}


def listed():
    return [
        # one decoding step of a small server batch: nothing but latency
        {"name": "step B8 H8 D64 bf16", "op": "step", "type": "bf16", "batch": 8, "heads": 8, "shared": 1, "dk": 64, "dv": 64},
        # one decoding step of 256 streams, the batch that the rotor generation step is measured at: the states' bytes
        {"name": "step B256 H16 D128 bf16", "op": "step", "type": "bf16", "batch": 256, "heads": 16, "shared": 1, "dk": 128, "dv": 128},
        # a few tokens of several streams at once, going on from their states (checking drafted tokens)
        _attention("attention B16 T37 H16 D64 bf16", "bf16", 16, 37, 16, 1, 64, 64, False),
        # the training step of the character model's sizes (batch 32, length 2048, width 128), float32
        _attention("attention train B32 T2048 H4 D32 fp32", "fp32", 32, 2048, 4, 1, 32, 32, True),
        # a training step of an ordinary language-model layer of width 2048
        _attention("attention train B8 T4096 H16 D128 bf16", "bf16", 8, 4096, 16, 1, 128, 128, True),
        # reading one long prompt: a single sequence and few heads, so time itself has to be split
        _attention("attention prompt B1 T65536 H8 D128 bf16", "bf16", 1, 65536, 8, 1, 128, 128, False),
        # fine-tuning on packed sequences of different lengths, three heads to a key, unequal head sizes
        _attention("attention train packed L20011 H12 Dk72 Dv104 fp16", "fp16", 37, 20011, 12, 3, 72, 104, True, packed=True),
        # the norm of a decoding step: latency
        _norm("norm R8 C2048 bf16", "bf16", 8, 2048, False),
        # the norm of an ordinary layer's training step
        _norm("norm train R32768 C2048 bf16", "bf16", 32768, 2048, True),
        # the norm of each head's output in that layer: very many short rows under one weight
        _norm("norm train R524288 C128 bf16", "bf16", 524288, 128, True),
        # an odd number of rows of an odd width, float32 weights beside 16-bit activations
        _norm("norm train R4099 C771 fp16", "fp16", 4099, 771, True, wide_weights=True),
        # wide rows
        _norm("norm train R8192 C8192 bf16", "bf16", 8192, 8192, True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def _width(rng, low, high):
    """A width: mostly a multiple of 8 as models have, sometimes any number."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "step", "norm", "norm"])
    if op == "norm":
        c = _width(rng, 32, 16384)
        return {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"]), "rows": _spread(rng, 1, min(524288, (1 << 26) // c)),
                "channels": c, "train": rng.random() < 0.7, "wide_weights": rng.random() < 0.3}
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    shared = rng.choice([1, 1, 1, 2, 3, 4])
    heads = shared * rng.choice([1, 2, 4, 5, 8])
    dk = rng.choice([32, 64, 64, 128, 128, _width(rng, 8, 128)])
    dv = dk if rng.random() < 0.7 else _width(rng, 8, 128)
    case = {"op": op, "type": kind, "heads": heads, "shared": shared, "dk": dk, "dv": dv}
    states = (1 << 26) // (heads * dk * dv)  # of a batch
    if op == "step":
        return {**case, "batch": _spread(rng, 1, min(256, states))}
    rows = (1 << 26) // (heads * max(dk, dv)) // (4 if kind == "fp32" else 1)
    if rng.random() < 0.35:
        length = _spread(rng, 16, min(65536, rows))
        batch, packed = _spread(rng, 1, max(1, min(64, states, length // 8))), True
    else:
        length = _spread(rng, 1, min(65536, rows))
        batch, packed = _spread(rng, 1, max(1, min(256, states, rows // length))), False
    return {**case, "batch": batch, "length": length, "train": rng.random() < 0.6, "packed": packed}


# ------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    typ = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=typ):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    state = {"case": dict(case)}
    if case["op"] == "norm":
        r, c = case["rows"], case["channels"]
        weights = torch.float32 if case["wide_weights"] else typ
        state["x"] = (torch.randn(r, c, generator=g, device=dev) * 2.0 + 0.5).to(typ)
        state["w"], state["b"] = normal(c, scale=0.2, dtype=torch.float32) + 1.0, normal(c, scale=0.2, dtype=torch.float32)
        state["w"], state["b"] = state["w"].to(weights), state["b"].to(weights)
        if case["train"]:
            state["dy"] = normal(r, c)
            state["leaves"] = ["x", "w", "b"]
    else:
        h, hk, dk, dv, batch = case["heads"], case["heads"] // case["shared"], case["dk"], case["dv"], case["batch"]
        if case["op"] == "step":
            lead = (batch,)
        else:
            lead = (case["length"],) if case["packed"] else (batch, case["length"])
        # one projection gives queries, keys and values side by side, as slices of its rows
        cuts = [h * dk, hk * dk, hk * dv]
        parts = normal(*lead, sum(cuts)).split(cuts, -1)
        state["q"], state["k"] = parts[0].unflatten(-1, (h, dk)), parts[1].unflatten(-1, (hk, dk))
        state["v"] = parts[2].unflatten(-1, (hk, dv))
        # the heads' memories run from 32 steps to 4096
        state["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(5.0, 12.0, h, device=dev)))
        state["s"] = normal(batch, h, dk, dv, scale=4.0, dtype=torch.float32)
        if case["op"] == "step":
            return state
        if case["packed"]:
            # a few rows stay behind the last sequence, and a sequence may be empty
            n = case["length"] - min(7, case["length"] // 8)
            ends = torch.sort(torch.randint(0, n + 1, (batch - 1,), generator=g, device=dev)).values
            border = torch.tensor([0, n], device=dev)
            state["cu"] = torch.cat([border[:1], ends, border[1:]]).to(torch.int32)
            state["borders"] = state["cu"].tolist()  # the packing program's own copy
        if case["train"]:
            state["do"], state["ds"] = normal(*lead, h, dv), normal(batch, h, dk, dv, dtype=torch.float32)
            state["leaves"] = ["q", "k", "v", "s"]
    for name in state.get("leaves", ()):
        state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------- plain forms
_BLOCK = 64


def _plain_sequences(q, k, v, log_decay, s, scale, do=None, ds=None):
    """[B, T, H, D] float32 in blocks of steps: within a block as a masked product, between blocks by the state."""
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    length, g = q.shape[2], log_decay[:, None]
    starts = list(range(0, length, _BLOCK))
    out = {"o": torch.empty(*q.shape[:3], v.shape[-1], device=q.device)}
    if do is not None:
        do = do.transpose(1, 2)
        out.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))

    def factors(n):
        at = torch.arange(n, device=q.device, dtype=torch.float32)
        gap = at[:, None] - at[None, :]
        fade = torch.exp(g[..., None] * gap.clamp(min=0.0)) * (gap >= 0.0)
        return fade, torch.exp(g * (at + 1.0))[..., None], torch.exp(g * (n - 1.0 - at))[..., None], torch.exp(g * n)[..., None]

    for a in starts:
        z = slice(a, min(a + _BLOCK, length))
        fade, since, left, whole = factors(z.stop - a)
        qb, kb, vb = q[:, :, z], k[:, :, z], v[:, :, z]
        out["o"][:, :, z] = scale * ((qb @ kb.mT * fade) @ vb + since * (qb @ s))
        if do is not None:
            db = do[:, :, z]
            out["dq"][:, :, z] = scale * ((db @ vb.mT * fade) @ kb + since * (db @ s.mT))
        s = whole * s + (kb * left).mT @ vb
    out["s"] = s
    if do is not None:
        for a in reversed(starts):
            z = slice(a, min(a + _BLOCK, length))
            fade, since, left, whole = factors(z.stop - a)
            qb, kb, vb, db = q[:, :, z], k[:, :, z], v[:, :, z], do[:, :, z]
            out["dk"][:, :, z] = scale * ((db @ vb.mT * fade).mT @ qb) + left * (vb @ ds.mT)
            out["dv"][:, :, z] = scale * ((qb @ kb.mT * fade).mT @ db) + left * (kb @ ds)
            ds = whole * ds + scale * (qb * since).mT @ db
        out["ds0"] = ds
    return {n: t.transpose(1, 2) if n in ("o", "dq", "dk", "dv") else t for n, t in out.items()}


def _plain_attention(s, case):
    typ, shared = _TYPES[case["type"]], case["shared"]
    q, k, v = (s[n].detach().float() for n in ("q", "k", "v"))
    k, v = (t.repeat_interleave(shared, -2) for t in (k, v))
    s0, scale = s["s"].detach(), case["dk"] ** -0.5
    do, ds = (s["do"].float(), s["ds"]) if case["train"] else (None, None)
    if case["packed"]:
        rows = ["o", "dq", "dk", "dv"] if case["train"] else ["o"]
        like = {"o": v, "dq": q, "dk": k, "dv": v}
        out = {n: torch.zeros(*q.shape[:2], like[n].shape[-1], device=q.device) for n in rows}
        ends = {n: torch.empty_like(s0) for n in (["s", "ds0"] if case["train"] else ["s"])}
        for i, (a, b) in enumerate(zip(s["borders"][:-1], s["borders"][1:])):
            cut = lambda t: None if t is None else t[None, a:b]  # noqa: E731
            one = _plain_sequences(cut(q), cut(k), cut(v), s["log_decay"], s0[i:i + 1], scale, cut(do),
                                   None if ds is None else ds[i:i + 1])
            for n in rows:
                out[n][a:b] = one[n][0]
            for n in ends:
                ends[n][i] = one[n][0]
        out.update(ends)
    else:
        out = _plain_sequences(q, k, v, s["log_decay"], s0, scale, do, ds)
    for n in ("dk", "dv"):
        if n in out:
            out[n] = out[n].unflatten(-2, (-1, shared)).sum(-2)
    return {n: t if n in ("s", "ds0") else t.to(typ) for n, t in out.items()}


def _plain_step(s, case):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    k, v = (t.repeat_interleave(case["shared"], 1) for t in (k, v))
    s["s"] = torch.exp(s["log_decay"])[:, None, None] * s["s"] + k[..., :, None] * v[..., None, :]
    o = case["dk"] ** -0.5 * (q[..., None, :] @ s["s"])[..., 0, :]
    return {"o": o.to(_TYPES[case["type"]]), "s": s["s"]}


def _plain_norm(s, case):
    typ = _TYPES[case["type"]]
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    hat = centred * rstd
    out = {"y": (hat * w + b).to(typ)}
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = (rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))).to(typ)
        out["dw"], out["db"] = (dy * hat).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)
    return out


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"attention": _plain_attention, "step": _plain_step, "norm": _plain_norm}[op](state, case)
    ops = _ops()
    if op == "step":
        o = ops.linear_attention_step(state["q"], state["k"], state["v"], state["log_decay"], state["s"])
        return {"o": o, "s": state["s"]}
    if op == "attention":
        o, s = ops.linear_attention(state["q"], state["k"], state["v"], state["log_decay"], s0=state["s"],
                                    cu_seqlens=state.get("cu"))
        if not case["train"]:
            return {"o": o, "s": s}
        dq, dk, dv, ds0 = torch.autograd.grad((o, s), [state[n] for n in state["leaves"]], (state["do"], state["ds"]))
        return {"o": o.detach(), "s": s.detach(), "dq": dq, "dk": dk, "dv": dv, "ds0": ds0}
    y = ops.layer_norm(state["x"], state["w"], state["b"], _EPS)
    if not case["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, [state[n] for n in state["leaves"]], state["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


# -------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "norm":
        n, c = case["rows"] * case["channels"], case["channels"]
        weights = 2 * c * (4 if case["wide_weights"] else size)
        if not case["train"]:
            return {"bytes": 2 * n * size + weights, "flops": 8 * n}
        return {"bytes": 5 * n * size + 2 * weights, "flops": 22 * n}  # x, y; x and dy again, dx
    h, hk, dk, dv = case["heads"], case["heads"] // case["shared"], case["dk"], case["dv"]
    row = (h * (dk + dv) + hk * (dk + dv)) * size  # q and o, k and v
    states, each = case["batch"] * h * dk * dv * 4, h * dk * dv
    if case["op"] == "step":
        return {"bytes": case["batch"] * row + 2 * states, "flops": 5 * case["batch"] * each}
    rows = case["length"] * (1 if case["packed"] else case["batch"])
    total = {"bytes": rows * row + 2 * states, "flops": 4 * rows * each}
    if case["train"]:  # q, k, v and do, the three gradients; the states once more, both ways, and three products with them
        total["bytes"] += rows * (2 * row - h * dv * size) + 3 * states
        total["flops"] += 10 * rows * each
    return total


# ------------------------------------------------------- the definition in 64 bits
def _exact_attention(s, case):
    """Step by step, all sequences at once: longest first, so that those still running at step t are the first n_t."""
    shared, scale = case["shared"], case["dk"] ** -0.5
    flat = lambda t: t.detach().double().flatten(0, -3)  # noqa: E731
    q, k, v = (flat(s[n]) for n in ("q", "k", "v"))
    head = torch.arange(case["heads"], device=q.device) // shared
    rows = q.shape[0]
    if case["packed"]:
        borders = s["cu"].tolist()
    else:
        borders = list(range(0, rows + 1, case["length"]))
    lens = torch.tensor([b - a for a, b in zip(borders[:-1], borders[1:])], device=q.device)
    order = torch.argsort(lens, descending=True, stable=True)
    begin = torch.tensor(borders[:-1], device=q.device)[order]
    longest = int(lens.max())
    running = (lens[order][None, :] > torch.arange(longest, device=q.device)[:, None]).sum(1).tolist() if longest else []
    fade = torch.exp(s["log_decay"].double())[:, None, None]
    state = s["s"].detach().double()[order].clone()
    back = torch.empty_like(order)
    back[order] = torch.arange(len(order), device=q.device)
    o = torch.zeros(rows, case["heads"], case["dv"], device=q.device, dtype=torch.float64)
    train = case["train"]
    if train:
        do, ds = flat(s["do"]), s["ds"].double()[order].clone()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(do)
    for t, n in enumerate(running):
        at = begin[:n] + t
        kt, vt = k[at][:, head], v[at][:, head]
        state[:n] = fade * state[:n] + kt[..., :, None] * vt[..., None, :]
        o[at] = scale * (state[:n] * q[at][..., :, None]).sum(-2)
        if train:
            dq[at] = scale * (state[:n] * do[at][..., None, :]).sum(-1)
    out = {"o": o.reshape(*s["q"].shape[:-1], case["dv"]), "s": state[back]}
    if train:
        for t in range(longest - 1, -1, -1):
            n = running[t]
            at = begin[:n] + t
            ds[:n] += scale * q[at][..., :, None] * do[at][..., None, :]
            dk[at] = (ds[:n] * v[at][:, head][..., None, :]).sum(-1)
            dv[at] = (ds[:n] * k[at][:, head][..., :, None]).sum(-2)
            ds[:n] *= fade
        gather = lambda t: t.reshape(rows, -1, shared, t.shape[-1]).sum(2)  # noqa: E731
        out.update(dq=dq.reshape(s["q"].shape), dk=gather(dk).reshape(s["k"].shape), dv=gather(dv).reshape(s["v"].shape),
                   ds0=ds[back])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attention":
            # a state's step moves about 60 bytes an entry
            longest = max(b - a for a, b in zip(s["borders"][:-1], s["borders"][1:])) if case["packed"] else case["length"]
            if longest * s["s"].numel() > 1 << 35:
                return None
            return _exact_attention(s, case)
        if case["op"] == "step":
            head = torch.arange(case["heads"], device="cuda") // case["shared"]
            k, v = s["k"].double()[:, head], s["v"].double()[:, head]
            state = torch.exp(s["log_decay"].double())[None, :, None, None] * s["s"].double() + torch.einsum("bhk,bhv->bhkv", k, v)
            return {"o": torch.einsum("bhk,bhkv->bhv", s["q"].double(), state) * case["dk"] ** -0.5, "s": state}
        x, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
        deviation = x - x.sum(-1, keepdim=True) / case["channels"]
        sigma = torch.sqrt(deviation.square().sum(-1, keepdim=True) / case["channels"] + _EPS)
        out = {"y": deviation / sigma * w + b}
        if case["train"]:
            dy, hat = s["dy"].double(), deviation / sigma
            along = torch.stack([torch.ones_like(hat), hat], -1)  # the two directions that the norm takes out
            pull = torch.einsum("rc,rcj->rj", dy * w, along) / case["channels"]
            out["dx"] = (dy * w - torch.einsum("rcj,rj->rc", along, pull)) / sigma
            out["dw"], out["db"] = torch.einsum("rc,rc->c", dy, hat), torch.einsum("rc->c", dy)
        return out
