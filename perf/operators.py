"""The operators of a gated recurrent block, measured at the sizes that they are used at.

Three operators and the single-token form of the first, all reached through ``csn_b200.ops``:

* ``gated_scan(f, x, h0, gate, cu_seqlens)`` -- the gated linear recurrence
      a_t = sigmoid(f_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t silu(gate_t)  (y_t = h_t without a gate)
  for each channel over a dense [B, T, C] batch or packed [L, C] sequences, with its backward pass;
* ``gated_step(f, x, h, gate)`` -- the same recurrence advanced by one token, the float32 state in place;
* ``silu_gated_linear(x, w_gate, w_up)`` -- y = silu(x w_gate^T) * (x w_up^T), with its backward pass;
* ``dropout_add(x, residual, p, rng)`` -- y = residual + keep x / (1 - p) with the mask drawn from
  Philox4x32-10 (Salmon et al., 2011) and never stored, with its backward pass.

``own`` chooses between the plain forms below and the framework's kernels.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "clifford-space-network_b200")
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _ops():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from csn_b200 import ops
    return ops


# ------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of a small server batch: nothing but latency
        {"name": "step B8 C512 bf16", "op": "step", "type": "bf16", "batch": 8, "channels": 512, "gate": True},
        # one decoding step of 256 streams, the batch that the rotor generation step is measured at
        {"name": "step B256 C4096 bf16", "op": "step", "type": "bf16", "batch": 256, "channels": 4096, "gate": True},
        # the training step of the character model's sizes (batch 32, length 2048, width 128), float32
        {"name": "scan train B32 T2048 C128 fp32", "op": "scan", "type": "fp32", "batch": 32, "length": 2048,
         "channels": 128, "gate": False, "train": True, "packed": False},
        # a training step of an ordinary language-model layer
        {"name": "scan train B8 T4096 C2048 bf16", "op": "scan", "type": "bf16", "batch": 8, "length": 4096,
         "channels": 2048, "gate": True, "train": True, "packed": False},
        # reading one long prompt: a single sequence, so time itself has to be split
        {"name": "scan prompt B1 T65536 C1024 bf16", "op": "scan", "type": "bf16", "batch": 1, "length": 65536,
         "channels": 1024, "gate": True, "train": False, "packed": False},
        # fine-tuning on packed sequences of different lengths with an odd width
        {"name": "scan packed L20011 C771 fp16", "op": "scan", "type": "fp16", "batch": 37, "length": 20011,
         "channels": 771, "gate": True, "train": True, "packed": True},
        # feed-forward of a few decoding streams: the weights are read once
        {"name": "ffn R4 C2048 F8192 bf16", "op": "ffn", "type": "bf16", "rows": 4, "channels": 2048, "hidden": 8192,
         "train": False},
        # a prompt of an odd number of tokens through an odd-sized layer
        {"name": "ffn R1021 C1032 F2744 fp16", "op": "ffn", "type": "fp16", "rows": 1021, "channels": 1032,
         "hidden": 2744, "train": False},
        # the training step of the character model's sizes: very many rows, narrow weights
        {"name": "ffn train R65536 C128 F256 bf16", "op": "ffn", "type": "bf16", "rows": 65536, "channels": 128,
         "hidden": 256, "train": True},
        # a training step of a large layer
        {"name": "ffn train R8192 C4096 F8192 bf16", "op": "ffn", "type": "bf16", "rows": 8192, "channels": 4096,
         "hidden": 8192, "train": True},
        # dropout on the residual path of the character model, float32
        {"name": "dropout B32 T64 C128 fp32", "op": "dropout", "type": "fp32", "rows": 2048, "channels": 128,
         "p": 0.1},
        # dropout on the residual path of an ordinary layer
        {"name": "dropout R32768 C2048 bf16", "op": "dropout", "type": "bf16", "rows": 32768, "channels": 2048,
         "p": 0.1},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width: mostly a multiple of 8 as models have, sometimes any number."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "step", "ffn", "ffn", "ffn", "dropout"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "step":
        return {"op": op, "type": kind, "batch": _spread(rng, 1, 256), "channels": _width(rng, 64, 4096),
                "gate": rng.random() < 0.7}
    if op == "scan":
        c, train = _width(rng, 64, 4096), rng.random() < 0.6
        most = (1 << 25) // c
        if rng.random() < 0.35:
            length = _spread(rng, 64, min(65536, most))
            batch, packed = _spread(rng, 1, max(1, length // 16)), True
        else:
            length = _spread(rng, 1, min(65536, most))
            batch, packed = _spread(rng, 1, max(1, min(256, most // length))), False
        return {"op": op, "type": kind, "batch": batch, "length": length, "channels": c,
                "gate": rng.random() < 0.6, "train": train, "packed": packed}
    if op == "ffn":
        c = _width(rng, 64, 4096)
        f = _width(rng, 2 * c, 4 * c)
        rows = _spread(rng, 1, min(65536, max(1, (1 << 37) // (c * f))))
        return {"op": op, "type": "fp16" if kind == "fp16" else "bf16", "rows": rows, "channels": c, "hidden": f,
                "train": rows > 64 and rng.random() < 0.6}
    c = _width(rng, 64, 4096)
    return {"op": op, "type": kind, "rows": _spread(rng, 1, min(65536, (1 << 26) // c)), "channels": c,
            "p": rng.choice([0.05, 0.1, 0.25, 0.5])}


# ------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    typ = _TYPES[case["type"]]
    c = case["channels"]

    def normal(*shape, scale=1.0, dtype=typ):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    state = {"case": dict(case)}
    if case["op"] in ("scan", "step"):
        if case["op"] == "step":
            lead = (case["batch"],)
        else:
            lead = (case["length"],) if case["packed"] else (case["batch"], case["length"])
        parts = 3 if case["gate"] else 2
        # one projection gives forget logits, input and gate side by side, as slices of its rows.  The
        # channels' biases spread the memory from a few steps to about a thousand.
        rows = normal(*lead, parts * c, dtype=torch.float32)
        rows[..., :c] += torch.linspace(0.0, 7.0, c, device=dev)
        rows = rows.to(typ)
        views = [rows[..., i * c:(i + 1) * c] for i in range(parts)]
        state["f"], state["x"] = views[0], views[1]
        state["gate"] = views[2] if case["gate"] else None
        state["h"] = normal(case["batch"], c, dtype=torch.float32)
        if case["op"] == "step":
            return state
        if case["packed"]:
            # a few rows stay behind the last sequence, and a sequence may be empty
            n = case["length"] - min(7, case["length"] // 8)
            ends = torch.sort(torch.randint(0, n + 1, (case["batch"] - 1,), generator=g, device=dev)).values
            border = torch.tensor([0, n], device=dev)
            state["cu"] = torch.cat([border[:1], ends, border[1:]]).to(torch.int32)
        if case["train"]:
            state["dy"], state["dh"] = normal(*lead, c), normal(case["batch"], c, dtype=torch.float32)
            state["leaves"] = ["f", "x", "h"] + (["gate"] if case["gate"] else [])
    elif case["op"] == "ffn":
        r, f = case["rows"], case["hidden"]
        state["x"] = normal(r, c)
        state["wg"], state["wu"] = normal(f, c, scale=c ** -0.5), normal(f, c, scale=c ** -0.5)
        if case["train"]:
            state["dy"] = normal(r, f, scale=0.01)
            state["leaves"] = ["x", "wg", "wu"]
    else:
        state["x"], state["res"] = normal(case["rows"], c), normal(case["rows"], c)
        state["dy"] = normal(case["rows"], c)
        state["rng"] = torch.randint(0, 1 << 62, (2,), generator=g, device=dev, dtype=torch.int64)
        state["leaves"] = ["x", "res"]
    for name in state.get("leaves", ()):
        state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------- plain forms
def _affine_scan(a, b):
    """h_t = a_t h_{t-1} + b_t from h = 0 along axis 1, by doubling: after a pass of step k each place
    holds the map over the last 2k steps."""
    k, n = 1, b.shape[1]
    while k < n:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        if 2 * k < n:
            a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _plain_scan(s, case):
    typ, packed = _TYPES[case["type"]], case["packed"]
    f, x, h0 = s["f"].detach().float(), s["x"].detach().float(), s["h"].detach()
    gate = s["gate"].detach().float() if case["gate"] else None
    if packed:
        f, x = f[None], x[None]
        gate = gate[None] if gate is not None else None
        rows = f.shape[1]
        cu = s["cu"].long()
        first, past = cu[:-1], cu[1:]
        some = past > first
        # a row index of `rows` is a spare row, cut off again: where an empty sequence's would go
        at_first, at_last = torch.where(some, first, rows), torch.where(some, past - 1, rows)
        pick = lambda v, at: torch.cat([v[0], torch.zeros_like(v[0, :1])], 0)[at]  # noqa: E731
        place = lambda v, at: torch.zeros(rows + 1, v.shape[-1], device=v.device).index_copy(0, at, v)[None, :rows]  # noqa: E731
        mark = lambda at: torch.zeros(rows + 1, device=f.device).index_fill(0, at, 1.0)[None, :rows, None]  # noqa: E731
        inside = (torch.arange(rows, device=f.device) < cu[-1])[None, :, None]
    else:
        some = torch.ones(case["batch"], dtype=torch.bool, device=f.device)
        at_first, at_last = 0, f.shape[1] - 1
        pick = lambda v, at: v[:, at]  # noqa: E731
        place = lambda v, at: torch.zeros_like(f).index_copy(1, torch.tensor([at], device=f.device), v[:, None])  # noqa: E731
        mark = lambda at: (torch.arange(f.shape[1], device=f.device) == at).float()[None, :, None]  # noqa: E731
        inside = torch.ones(1, 1, 1, dtype=torch.bool, device=f.device)
    a, q = torch.sigmoid(f), torch.sigmoid(-f)
    start, end = mark(at_first), mark(at_last)
    h = _affine_scan(a * (1.0 - start), q * x + a * place(h0, at_first)) * inside
    sig = torch.sigmoid(gate) if gate is not None else None
    y = h * gate * sig if gate is not None else h
    y = torch.where(inside, y, 0.0)
    h_last = torch.where(some[:, None], pick(h, at_last), h0)
    out = {"y": (y[0] if packed else y).to(typ), "h": h_last}
    if not case["train"]:
        return out
    dy, dh_last = s["dy"].float(), s["dh"]
    dy = dy[None] if packed else dy
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1) * (1.0 - start) + place(h0, at_first)
    dh = torch.where(inside, dy * gate * sig if gate is not None else dy, 0.0) + place(dh_last, at_last)
    onward = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1) * (1.0 - end)
    lam = _affine_scan(onward.flip(1), dh.flip(1)).flip(1) * inside
    grads = {"df": lam * (before - x) * a * q, "dx": lam * q}
    if gate is not None:
        grads["dgate"] = torch.where(inside, dy * h * (sig + gate * sig * torch.sigmoid(-gate)), 0.0)
    out.update({k: (v[0] if packed else v).to(typ) for k, v in grads.items()})
    out["dh0"] = torch.where(some[:, None], pick(a * lam, at_first), dh_last)
    return out


def _plain_step(s, case):
    f, x = s["f"].float(), s["x"].float()
    s["h"] = torch.sigmoid(f) * s["h"] + torch.sigmoid(-f) * x
    y = s["h"]
    if case["gate"]:
        g = s["gate"].float()
        y = y * g * torch.sigmoid(g)
    return {"y": y.to(_TYPES[case["type"]]), "h": s["h"]}


def _plain_ffn(s, case):
    typ = _TYPES[case["type"]]
    x, wg, wu = s["x"].detach().float(), s["wg"].detach().float(), s["wu"].detach().float()
    g, u = x @ wg.t(), x @ wu.t()
    sig = torch.sigmoid(g)
    out = {"y": (g * sig * u).to(typ)}
    if case["train"]:
        dy = s["dy"].float()
        dg, du = dy * u * (sig + g * sig * (1.0 - sig)), dy * g * sig
        out["dx"] = (dg @ wg + du @ wu).to(typ)
        out["dwg"], out["dwu"] = (dg.t() @ x).to(typ), (du.t() @ x).to(typ)
    return out


def _philox(group, rng):
    """Philox4x32-10 of the counters (group, offset) under the key `seed`, in 64-bit whole numbers: the
    product of two 32-bit words wraps to its exact 64 bits."""
    low = 0xFFFFFFFF
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    c0, c1 = group & low, (group >> 32) & low
    c2, c3 = rng[1] & low, (rng[1] >> 32) & low
    c2, c3 = c2.expand_as(c0), c3.expand_as(c0)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], -1)


def _plain_dropout(s, case):
    typ = _TYPES[case["type"]]
    x, res, dy = s["x"].detach(), s["res"].detach(), s["dy"]
    n = x.numel()
    words = _philox(torch.arange((n + 7) // 8, device=x.device), s["rng"])
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:n].reshape(x.shape)
    cut = round(case["p"] * 65536)
    factor = (halves >= cut).float() * (65536.0 / (65536 - cut))
    return {"y": (res.float() + x.float() * factor).to(typ), "dx": (dy.float() * factor).to(typ), "dres": dy}


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"scan": _plain_scan, "step": _plain_step, "ffn": _plain_ffn, "dropout": _plain_dropout}[op](state, case)
    ops = _ops()
    if op == "step":
        y = ops.gated_step(state["f"], state["x"], state["h"], gate=state["gate"])
        return {"y": y, "h": state["h"]}
    if op == "scan":
        y, h = ops.gated_scan(state["f"], state["x"], h0=state["h"], gate=state["gate"], cu_seqlens=state.get("cu"))
        if not case["train"]:
            return {"y": y, "h": h}
        names = {"f": "df", "x": "dx", "h": "dh0", "gate": "dgate"}
        grads = torch.autograd.grad((y, h), [state[k] for k in state["leaves"]], (state["dy"], state["dh"]))
        return {"y": y.detach(), "h": h.detach(), **{names[k]: v for k, v in zip(state["leaves"], grads)}}
    if op == "ffn":
        y = ops.silu_gated_linear(state["x"], state["wg"], state["wu"])
        if not case["train"]:
            return {"y": y}
        dx, dwg, dwu = torch.autograd.grad(y, [state[k] for k in state["leaves"]], state["dy"])
        return {"y": y.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}
    y = ops.dropout_add(state["x"], state["res"], case["p"], state["rng"])
    dx, dres = torch.autograd.grad(y, [state["x"], state["res"]], state["dy"])
    return {"y": y.detach(), "dx": dx, "dres": dres}


# -------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    c = case["channels"]
    if case["op"] == "step":
        n, k = case["batch"] * c, 3 if case["gate"] else 2
        return {"bytes": n * ((k + 1) * size + 8), "flops": n * 16}
    if case["op"] == "scan":
        states = case["batch"] * c * 4
        n = case["length"] * c * (1 if case["packed"] else case["batch"])
        k = 3 if case["gate"] else 2
        total = {"bytes": n * size * (k + 1) + 2 * states, "flops": n * 16}
        if case["train"]:  # the inputs and dy again, the gradients out
            total["bytes"] += n * size * (2 * k + 1) + 3 * states
            total["flops"] += n * 32
        return total
    if case["op"] == "ffn":
        r, f = case["rows"], case["hidden"]
        ends, weights, hidden = r * c, 2 * f * c, r * f
        if not case["train"]:
            return {"bytes": size * (ends + weights + hidden), "flops": 4 * r * f * c}
        return {"bytes": size * 2 * (ends + weights + hidden), "flops": 12 * r * f * c}
    n = case["rows"] * c  # x, residual, dy in; y and dx out (the residual's gradient is dy itself)
    return {"bytes": n * size * 5, "flops": n * 20}


# ------------------------------------------------------- the definition in 64 bits
def _sequences(s, case):
    """(first row, one past the last) of each sequence, over rows [batch * length] or packed [length]."""
    if case["packed"]:
        cu = s["cu"].tolist()
        return list(zip(cu[:-1], cu[1:]))
    t = case["length"]
    return [(b * t, (b + 1) * t) for b in range(case["batch"])]


def _exact_scan(s, case):
    c = case["channels"]
    wide = lambda v: v.detach().double().reshape(-1, c)  # noqa: E731
    f, x, h0 = wide(s["f"]), wide(s["x"]), s["h"].detach().double()
    gate = wide(s["gate"]) if case["gate"] else None
    dev, rows = f.device, f.shape[0]
    seqs = _sequences(s, case)
    lens = torch.tensor([e - b for b, e in seqs], device=dev)
    # longest sequence first, so that the sequences still running at step t are the first n_t of them
    order = torch.argsort(lens, descending=True, stable=True)
    begin = torch.tensor([b for b, _ in seqs], device=dev)[order]
    longest = int(lens.max())
    running = [int(v) for v in (lens[order][None, :] > torch.arange(longest, device=dev)[:, None]).sum(1)] if longest else []
    a = 1.0 / (1.0 + torch.exp(-f))
    q = 1.0 / (1.0 + torch.exp(f))
    h, prev = h0[order].clone(), torch.zeros_like(f)
    hs = torch.zeros_like(f)
    for t, n in enumerate(running):
        at = begin[:n] + t
        prev[at] = h[:n]
        h[:n] = a[at] * h[:n] + q[at] * x[at]
        hs[at] = h[:n]
    back = torch.empty_like(order)
    back[order] = torch.arange(len(seqs), device=dev)
    sg = 1.0 / (1.0 + torch.exp(-gate)) if gate is not None else None
    y = hs * gate * sg if gate is not None else hs
    shape = s["f"].shape
    out = {"y": y.reshape(shape), "h": h[back]}
    if case["train"]:
        dy = wide(s["dy"])
        dh = dy * gate * sg if gate is not None else dy
        df, dx, lam = torch.zeros_like(f), torch.zeros_like(f), s["dh"].double()[order].clone()
        for t in range(longest - 1, -1, -1):
            n = running[t]
            at = begin[:n] + t
            lam[:n] += dh[at]
            df[at] = lam[:n] * (prev[at] - x[at]) * a[at] * q[at]
            dx[at] = lam[:n] * q[at]
            lam[:n] *= a[at]
        out.update(df=df.reshape(shape), dx=dx.reshape(shape), dh0=lam[back])
        if gate is not None:
            covered = torch.zeros(rows, 1, device=dev, dtype=torch.float64)
            for b, e in seqs:
                covered[b:e] = 1.0
            out["dgate"] = (covered * dy * hs * sg * (1.0 + gate * (1.0 - sg))).reshape(shape)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "scan":
        with torch.no_grad():
            return _exact_scan(s, case)
    if case["op"] == "step":
        a = 1.0 / (1.0 + torch.exp(-s["f"].double()))
        h = a * s["h"].double() + (1.0 - a) * s["x"].double()
        g = s["gate"].double() if case["gate"] else None
        return {"y": h * g / (1.0 + torch.exp(-g)) if g is not None else h, "h": h}
    if case["op"] == "ffn":
        if case["rows"] * case["channels"] * case["hidden"] > 1 << 38:
            return None
        x, wg, wu = (s[k].detach().double() for k in ("x", "wg", "wu"))
        g, u = torch.einsum("rc,fc->rf", x, wg), torch.einsum("rc,fc->rf", x, wu)
        silu = g / (1.0 + torch.exp(-g))
        out = {"y": silu * u}
        if case["train"]:
            dy = s["dy"].double()
            slope = (1.0 + torch.exp(-g) * (1.0 + g)) / (1.0 + torch.exp(-g)) ** 2
            dg, du = dy * u * slope, dy * silu
            out["dx"] = torch.einsum("rf,fc->rc", dg, wg) + torch.einsum("rf,fc->rc", du, wu)
            out["dwg"], out["dwu"] = torch.einsum("rf,rc->fc", dg, x), torch.einsum("rf,rc->fc", du, x)
        return out
    # the random words once more, with numpy's unsigned whole numbers
    n = case["rows"] * case["channels"]
    seed_word, offset = (int(v) for v in s["rng"].tolist())
    group = np.arange((n + 7) // 8, dtype=np.uint64)
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = [group & mask, group >> half, np.full_like(group, offset & 0xFFFFFFFF), np.full_like(group, (offset >> 32) & 0xFFFFFFFF)]
    key = [seed_word & 0xFFFFFFFF, (seed_word >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        left, right = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(right >> half) ^ ctr[1] ^ np.uint64(key[0]), right & mask,
               (left >> half) ^ ctr[3] ^ np.uint64(key[1]), left & mask]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(ctr, -1).astype("<u4")
    cut = round(case["p"] * 65536)
    keep = torch.from_numpy((words.reshape(-1).view("<u2")[:n] >= cut).astype(np.float64)).reshape(case["rows"], -1).to(s["x"].device)
    factor = keep * 65536 / (65536 - cut)
    dy = s["dy"].double()
    return {"y": s["res"].detach().double() + s["x"].detach().double() * factor, "dx": dy * factor, "dres": dy}
