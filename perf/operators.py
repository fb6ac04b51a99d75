"""The language-model operators of this framework as they are measured.

Five operators, each in its plain form (elementary torch operations in 32 bits)
and, where `own` is true, through the framework's public Python calls:

  logprob       log probability of one given token a row, with the row's
                entropy, log-sum-exp and its most likely alternatives
  logprob_grad  the gradient of those with respect to the logits
  norm          h = alpha * residual + gate * norm(block), y = norm(h)
  norm_grad     its gradients: residual, block, both weights and the gate
  matvec4       product with 4-bit weights that have a scale for each group

Tensors are column-major, as everywhere in the framework.  "rows": the
vocabulary axis comes first and is contiguous.  "lanes": the tokens come first,
so that a row's elements are `rows` apart (a matrix whose rows are tokens).
"""
import math
import os
import sys

import torch

own = False

_DTYPE = {"float": torch.float32, "float16": torch.float16}


def _package():
    """The framework's Python package (acedia-r_b200/acediar)."""
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "acedia-r_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import acediar
    return acediar


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one step of a served model: one row of a large vocabulary with 20 alternatives, where latency counts
        dict(name="logprob_decode", op="logprob", rows=1, width=131072, layout="rows", dtype="float16", top=20,
             scale=1.0, masked=0.0),
        # scoring a batch of sequences: an odd vocabulary, a part of it masked out
        dict(name="logprob_score", op="logprob", rows=4096, width=50001, layout="rows", dtype="float", top=0,
             scale=1.0, masked=0.05),
        # the row softmax configuration's matrix (tokens first), sampled at a temperature of 1.25
        dict(name="logprob_matrix", op="logprob", rows=65536, width=4096, layout="lanes", dtype="float", top=5,
             scale=0.8, masked=0.0),
        # the gradient of a training step: log probability and entropy terms
        dict(name="logprob_grad_train", op="logprob_grad", rows=4096, width=32768, layout="rows", dtype="float16",
             scale=1.0, entropy=True),
        # the gradient on the row softmax configuration's matrix, log probability alone
        dict(name="logprob_grad_matrix", op="logprob_grad", rows=65536, width=4096, layout="lanes", dtype="float",
             scale=1.0, entropy=False),
        # a decoding step of a few sequences
        dict(name="norm_decode", op="norm", rows=8, width=4096, dtype="float16", post=True, gates=1, alpha=1.0),
        # a training batch of 16 samples of 1024 tokens, each sample with a gate of its own
        dict(name="norm_train", op="norm", rows=16384, width=4096, dtype="float16", post=True, gates=16, alpha=1.0),
        # its gradient
        dict(name="norm_grad_train", op="norm_grad", rows=16384, width=4096, dtype="float16", post=True, gates=16,
             alpha=1.0),
        # the gradient of a small odd model in 32 bits: no norm after the block, one gate for all tokens
        dict(name="norm_grad_odd", op="norm_grad", rows=5000, width=1001, dtype="float", post=False, gates=1,
             alpha=0.5),
        # a square projection for one token
        dict(name="matvec4_square", op="matvec4", out=4096, inner=4096, n=1, group=128, zeros=False, dtype="float16"),
        # a model's head over a large vocabulary for one token, zero points for each group
        dict(name="matvec4_head", op="matvec4", out=131072, inner=4096, n=1, group=64, zeros=True, dtype="float16"),
        # an odd projection for six tokens at once, activations in 32 bits
        dict(name="matvec4_odd", op="matvec4", out=10007, inner=8200, n=6, group=32, zeros=True, dtype="float"),
    ]


def _between(rng, lo, hi):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprob", "logprob_grad", "norm", "norm_grad", "matvec4"])
    dtype = rng.choice(["float", "float16"])
    if op in ("logprob", "logprob_grad"):
        width = _between(rng, 500, 200000)
        rows = _between(rng, 1, max(1, min(65536, 200_000_000 // width)))
        layout = "rows" if rows < 32 else rng.choice(["rows", "lanes"])
        case = dict(op=op, rows=rows, width=width, layout=layout, dtype=dtype, scale=rng.choice([1.0, 1.0, 0.7, 1.5]))
        if op == "logprob":
            case.update(top=rng.choice([0, 1, 5, 20]), masked=rng.choice([0.0, 0.1]))
        else:
            case.update(entropy=rng.choice([False, True]))
        return case
    if op in ("norm", "norm_grad"):
        width = _between(rng, 64, 16384)
        if rng.random() < 0.6:
            width = max(80, width // 80 * 80)
        gates = rng.choice([0, 1, 1, 4])
        per = _between(rng, 1, max(1, 60_000_000 // width // max(1, gates)))
        return dict(op=op, rows=per * max(1, gates), width=width, dtype=dtype, post=rng.choice([False, True, True]),
                    gates=gates, alpha=rng.choice([1.0, 1.0, 0.5]))
    inner = _between(rng, 256, 16384)
    if rng.random() < 0.7:
        inner = max(640, inner // 640 * 640)
    out = _between(rng, 256, max(256, min(131072, 500_000_000 // inner)))
    return dict(op=op, out=out, inner=inner, n=_between(rng, 1, 8), group=rng.choice([32, 64, 128]),
                zeros=rng.choice([False, True]), dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _logits(case, g):
    """Logits of a model: a spread of about 3, an offset for each row; stored (rows, width) or (width, rows)."""
    rows, width = case["rows"], case["width"]
    shape, other = ((rows, width), (rows, 1)) if case["layout"] == "rows" else ((width, rows), (1, rows))
    x = torch.randn(shape, device="cuda", generator=g)
    x.mul_(3.0).add_(torch.rand(other, device="cuda", generator=g) * 16 - 8)
    if case.get("masked"):
        drop = torch.rand(shape, device="cuda", generator=g) < case["masked"]
        x.masked_fill_(drop, -math.inf)
    return x.to(_DTYPE[case["dtype"]])


def _ceil(a, b):
    return -(-a // b)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    op = case["op"]
    dt = _DTYPE[case.get("dtype", "float")]
    if op in ("logprob", "logprob_grad"):
        rows, width = case["rows"], case["width"]
        s["logits"] = _logits(case, g)
        # tokens count from 1; 0 asks for none (padding), about one in sixteen where there are many rows
        t = torch.randint(1, width + 1, (rows,), device="cuda", generator=g)
        if rows >= 64:
            t = torch.where(torch.rand(rows, device="cuda", generator=g) < 1 / 16, 0, t)
        s["tokens"] = t
        if op == "logprob_grad":
            # what the forward call has returned, and the loss's gradient with respect to it
            dim = 1 if case["layout"] == "rows" else 0
            step = max(1, (1 << 26) // width)
            lse, ent = [], []
            for a in range(0, rows, step):
                x = s["logits"].narrow(1 - dim, a, min(step, rows - a)).double() * case["scale"]
                l = torch.logsumexp(x, dim)
                x -= l.unsqueeze(dim)
                lse.append(l)
                ent.append(-(x.exp() * x).sum(dim))
            s["lse"] = torch.cat(lse).float()
            s["entropy"] = torch.cat(ent).float()
            s["d_logprob"] = -(torch.rand(rows, device="cuda", generator=g) + 0.5)
            s["d_entropy"] = torch.rand(rows, device="cuda", generator=g) * 0.1 if case["entropy"] else None
    elif op in ("norm", "norm_grad"):
        rows, width, gates = case["rows"], case["width"], case["gates"]
        r = torch.randn(rows, width, device="cuda", generator=g)
        b = torch.randn(rows, width, device="cuda", generator=g) * (
            torch.rand(rows, 1, device="cuda", generator=g) * 2 + 0.2)
        s["w_pre"] = (1 + 0.1 * torch.randn(width, device="cuda", generator=g)).to(dt)
        s["w_post"] = (1 + 0.1 * torch.randn(width, device="cuda", generator=g)).to(dt) if case["post"] else None
        s["gate"] = (0.5 + 0.3 * torch.randn(gates, width, device="cuda", generator=g)).to(dt) if gates else None
        s["block"] = b.to(dt)
        if op == "norm":
            s["residual"] = r.to(dt)
        else:
            # what the forward call has returned, and the gradients with respect to it
            b = s["block"].double()
            rb = (b.square().mean(1) + 1e-6).rsqrt()
            c = b * rb[:, None] * s["w_post"].double() if case["post"] else b
            if gates:
                c = (c.view(gates, -1, width) * s["gate"].double()[:, None, :]).view(rows, width)
            h = case["alpha"] * r.double() + c
            s["rstd_block"] = rb.float() if case["post"] else None
            s["rstd_h"] = (h.square().mean(1) + 1e-6).rsqrt().float()
            s["h"] = h.to(dt)
            s["d_h"] = torch.randn(rows, width, device="cuda", generator=g).to(dt)
            s["d_y"] = torch.randn(rows, width, device="cuda", generator=g).to(dt)
    else:
        out, inner, n, group = case["out"], case["inner"], case["n"], case["group"]
        # two weights a byte along the inner axis, the even one in the low half; columns of whole 16-byte pieces
        s["weights"] = torch.randint(-128, 128, (out, 16 * _ceil(inner, 32)), device="cuda", generator=g,
                                     dtype=torch.int8)
        s["scales"] = ((torch.rand(out, _ceil(inner, group), device="cuda", generator=g) + 0.5) / 128).half()
        s["zeros"] = (torch.randint(0, 16, s["scales"].shape, device="cuda", generator=g).half()
                      if case["zeros"] else None)
        s["x"] = torch.randn(n, inner, device="cuda", generator=g).to(dt)
    if own:
        s["own"] = _handles(s)
    return s


def _handles(s):
    """The same buffers as the framework's tensors."""
    acd, case = _package(), s["case"]
    wrap = lambda t, shape, dtype: None if t is None else acd.from_torch(t, shape, dtype)  # noqa: E731
    h, dt, op = {}, case["dtype"], case["op"]
    if op in ("logprob", "logprob_grad"):
        rows, width = case["rows"], case["width"]
        shape = (width, rows) if case["layout"] == "rows" else (rows, width)
        h["logits"] = wrap(s["logits"], shape, dt)
        h["tokens"] = wrap(s["tokens"], (rows,), "int64")
        for k in ("lse", "entropy", "d_logprob", "d_entropy"):
            h[k] = wrap(s.get(k), (rows,), "float")
    elif op in ("norm", "norm_grad"):
        rows, width, gates = case["rows"], case["width"], case["gates"]
        per = rows // gates if gates else rows
        shape = (width, per, gates) if gates else (width, rows)
        for k in ("residual", "block", "h", "d_h", "d_y"):
            h[k] = wrap(s.get(k), shape, dt)
        h["w_pre"] = wrap(s["w_pre"], (width,), dt)
        h["w_post"] = wrap(s["w_post"], (width,), dt)
        h["gate"] = wrap(s["gate"], (width, 1, gates), dt)
        for k in ("rstd_h", "rstd_block"):
            h[k] = wrap(s.get(k), shape[1:], "float")
    else:
        out, inner = case["out"], case["inner"]
        h["weights"] = wrap(s["weights"], (16 * _ceil(inner, 32), out), "int8")
        h["scales"] = wrap(s["scales"], (_ceil(inner, case["group"]), out), "float16")
        h["zeros"] = wrap(s["zeros"], (_ceil(inner, case["group"]), out), "float16")
        h["x"] = wrap(s["x"], (inner, case["n"]), dt)
    return h


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


def _flat(*tensors):
    return [None if t is None else t.storage for t in tensors]


def _run_own(s):
    acd, c, h = _package(), s["case"], s["own"]
    op = c["op"]
    if op == "logprob":
        r = acd.token_logprob(h["logits"], h["tokens"], axis=1 if c["layout"] == "rows" else 2, scale=c["scale"],
                              top=c["top"])
        return _flat(r.logprob, r.entropy, r.logsumexp, r.top_index, r.top_logprob)
    if op == "logprob_grad":
        return _flat(acd.token_logprob_grad(h["logits"], h["tokens"], h["lse"], h["entropy"], h["d_logprob"],
                                            h["d_entropy"], axis=1 if c["layout"] == "rows" else 2,
                                            scale=c["scale"]))
    if op == "norm":
        r = acd.residual_norm(h["residual"], h["block"], h["w_pre"], w_post=h["w_post"], gate=h["gate"],
                              alpha=c["alpha"], eps=1e-6)
        return _flat(r.h, r.y, r.rstd_h, r.rstd_block)
    if op == "norm_grad":
        r = acd.residual_norm_grad(h["d_h"], h["d_y"], h["h"], h["block"], h["rstd_h"], h["rstd_block"], h["w_pre"],
                                   w_post=h["w_post"], gate=h["gate"], alpha=c["alpha"])
        return _flat(r.d_residual, r.d_block, r.d_w_pre, r.d_w_post, r.d_gate)
    return _flat(acd.quant4_matvec(h["weights"], h["scales"], h["x"], c["group"], zeros=h["zeros"]))


def _plain_logprob(s):
    c = s["case"]
    dim = 1 if c["layout"] == "rows" else 0
    raw = s["logits"].float()
    x = raw * c["scale"]
    m = x.amax(dim, keepdim=True)
    z = x - m
    e = z.exp()
    total = e.sum(dim, keepdim=True)
    log_total = total.log()
    # an impossible token adds nothing to the entropy (0 log 0 = 0)
    entropy = (log_total - (e * torch.where(e > 0, z, 0.0)).sum(dim, keepdim=True) / total).squeeze(dim)
    lse = (m + log_total).squeeze(dim)
    asked = s["tokens"] > 0
    at = (s["tokens"] - 1).clamp(min=0).unsqueeze(dim)
    logprob = torch.where(asked, (z.gather(dim, at) - log_total).squeeze(dim), 0.0)
    if not c["top"]:
        return [logprob, entropy, lse, None, None]
    # one whole number that orders by value and, among equal values, by the lowest index
    bits = (raw + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    shape = (1, -1) if dim == 1 else (-1, 1)
    key -= torch.arange(c["width"], device="cuda").view(shape)
    at = key.topk(c["top"], dim=dim).indices
    return [logprob, entropy, lse, (at + 1).reshape(-1), (z.gather(dim, at) - log_total).reshape(-1)]


def _plain_logprob_grad(s):
    c = s["case"]
    dim = 1 if c["layout"] == "rows" else 0
    lp = s["logits"].float() * c["scale"] - s["lse"].unsqueeze(dim)
    p = lp.exp()
    asked = s["tokens"] > 0
    g = torch.where(asked, s["d_logprob"], 0.0)
    grad = p * -g.unsqueeze(dim)
    if s["d_entropy"] is not None:
        grad -= p * s["d_entropy"].unsqueeze(dim) * (lp + s["entropy"].unsqueeze(dim))
    at = (s["tokens"] - 1).clamp(min=0).unsqueeze(dim)
    grad.scatter_add_(dim, at, g.unsqueeze(dim))
    return [(grad * c["scale"]).to(_DTYPE[c["dtype"]]).reshape(-1)]


def _plain_gated(s, b):
    """block * gate, in 32 bits, the gate of each sample over its tokens."""
    c = s["case"]
    if s["gate"] is None:
        return b
    return (b.view(c["gates"], -1, c["width"]) * s["gate"].float()[:, None, :]).view(c["rows"], c["width"])


def _plain_norm(s):
    c = s["case"]
    b = s["block"].float()
    rb = None
    if c["post"]:
        rb = (b.square().mean(1) + 1e-6).rsqrt()
        b = b * rb[:, None] * s["w_post"].float()
    h = c["alpha"] * s["residual"].float() + _plain_gated(s, b)
    rh = (h.square().mean(1) + 1e-6).rsqrt()
    y = h * rh[:, None] * s["w_pre"].float()
    dt = _DTYPE[c["dtype"]]
    return [h.to(dt).reshape(-1), y.to(dt).reshape(-1), rh, rb]


def _plain_norm_grad(s):
    c = s["case"]
    dt = _DTYPE[c["dtype"]]
    dy, hh = s["d_y"].float(), s["h"].float() * s["rstd_h"][:, None]
    u = dy * s["w_pre"].float()
    dh = s["d_h"].float() + s["rstd_h"][:, None] * (u - hh * (u * hh).mean(1, keepdim=True))
    d_w_pre = (dy * hh).sum(0)
    bh = s["block"].float()
    if c["post"]:
        bh = bh * s["rstd_block"][:, None]
    d_gate = None
    if s["gate"] is not None:
        d_gate = dh * bh
        if c["post"]:
            d_gate = d_gate * s["w_post"].float()
        d_gate = d_gate.view(c["gates"], -1, c["width"]).sum(1).reshape(-1)
    db, d_w_post = _plain_gated(s, dh), None
    if c["post"]:
        d_w_post = (db * bh).sum(0)
        v = db * s["w_post"].float()
        db = s["rstd_block"][:, None] * (v - bh * (v * bh).mean(1, keepdim=True))
    return [(c["alpha"] * dh).to(dt).reshape(-1), db.to(dt).reshape(-1), d_w_pre, d_w_post, d_gate]


def _plain_matvec4(s):
    c = s["case"]
    q = torch.stack([s["weights"] & 15, (s["weights"] >> 4) & 15], dim=2).view(c["out"], -1)[:, :c["inner"]].float()
    group = torch.arange(c["inner"], device="cuda") // c["group"]
    z = s["zeros"].float()[:, group] if s["zeros"] is not None else 8.0
    w = (q - z) * s["scales"].float()[:, group]
    return [(s["x"].float() @ w.t()).to(_DTYPE[c["dtype"]]).reshape(-1)]


_PLAIN = {"logprob": _plain_logprob, "logprob_grad": _plain_logprob_grad, "norm": _plain_norm,
          "norm_grad": _plain_norm_grad, "matvec4": _plain_matvec4}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    es = 4 if case["dtype"] == "float" else 2
    if op == "logprob":
        n = case["rows"] * case["width"]
        return {"bytes": n * es + case["rows"] * (8 + 12 + 12 * case["top"]), "flops": 6 * n}
    if op == "logprob_grad":
        n = case["rows"] * case["width"]
        return {"bytes": 2 * n * es + case["rows"] * (16 + (8 if case["entropy"] else 0)), "flops": 6 * n}
    if op in ("norm", "norm_grad"):
        n, width = case["rows"] * case["width"], case["width"]
        vectors = width * (1 + int(case["post"]) + case["gates"])
        stats = case["rows"] * 4 * (1 + int(case["post"]))
        if op == "norm":
            return {"bytes": 4 * n * es + vectors * es + stats, "flops": 10 * n}
        return {"bytes": 6 * n * es + vectors * (es + 4) + stats, "flops": 20 * n}
    out, inner, n = case["out"], case["inner"], case["n"]
    scales = out * _ceil(inner, case["group"]) * 2 * (1 + int(case["zeros"]))
    return {"bytes": out * _ceil(inner, 2) + scales + n * (inner + out) * es, "flops": 2 * out * inner * n}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "logprob":
        x = s["logits"].double()
        if case["layout"] == "lanes":
            x = x.t()
        top = None
        if case["top"]:
            top = x.topk(case["top"], dim=1).values * case["scale"]
        x = x * case["scale"]
        lse = x.logsumexp(1)
        t = s["tokens"]
        lp = x[torch.arange(case["rows"], device="cuda"), (t - 1).clamp(min=0)] - lse
        lp[t == 0] = 0
        entropy = torch.special.entr((x - lse[:, None]).exp()).sum(1)
        if top is not None:
            top = top - lse[:, None]
            top = (top if case["layout"] == "rows" else top.t()).reshape(-1)
        return [lp, entropy, lse, None, top]
    if op == "logprob_grad":
        x = s["logits"].double()
        if case["layout"] == "lanes":
            x = x.t()
        p = torch.softmax(x * case["scale"], 1)
        t = s["tokens"]
        g = s["d_logprob"].double() * (t > 0)
        out = -p * g[:, None]
        out[torch.arange(case["rows"], device="cuda"), (t - 1).clamp(min=0)] += g
        if s["d_entropy"] is not None:
            # dH/dx = -p (log p + H)
            e = torch.special.entr(p)
            out += s["d_entropy"].double()[:, None] * (e - p * e.sum(1, keepdim=True))
        out *= case["scale"]
        return [(out if case["layout"] == "rows" else out.t()).reshape(-1)]
    if op in ("norm", "norm_grad"):
        rows, width, gates = case["rows"], case["width"], case["gates"]
        b = s["block"].double()
        gate = (s["gate"].double().repeat_interleave(rows // gates, 0) if gates
                else torch.ones((), device="cuda", dtype=torch.float64))
        wpre = s["w_pre"].double()
        if op == "norm":
            rb = None
            if case["post"]:
                rb = 1 / torch.sqrt((b * b).sum(1) / width + 1e-6)
                b = b * rb[:, None] * s["w_post"].double()
            h = s["residual"].double() * case["alpha"] + b * gate
            rh = 1 / torch.sqrt((h * h).sum(1) / width + 1e-6)
            return [h.reshape(-1), (h * rh[:, None] * wpre).reshape(-1), rh, rb]
        h, dy, rh = s["h"].double(), s["d_y"].double(), s["rstd_h"].double()[:, None]
        inner = (dy * wpre * h).sum(1, keepdim=True)
        total = s["d_h"].double() + rh * dy * wpre - rh ** 3 / width * inner * h
        d_w_pre = (dy * h * rh).sum(0)
        if case["post"]:
            rb, wpost = s["rstd_block"].double()[:, None], s["w_post"].double()
            n = total * gate
            d_w_post = (n * b * rb).sum(0)
            db = rb * n * wpost - rb ** 3 / width * (n * wpost * b).sum(1, keepdim=True) * b
            b = b * rb * wpost
        else:
            db, d_w_post = total * gate, None
        d_gate = (total * b).view(gates, -1, width).sum(1).reshape(-1) if gates else None
        return [(total * case["alpha"]).reshape(-1), db.reshape(-1), d_w_pre, d_w_post, d_gate]
    out, inner, group = case["out"], case["inner"], case["group"]
    byte = s["weights"].to(torch.int16) & 255
    w = torch.empty(out, 2 * byte.shape[1], device="cuda", dtype=torch.float64)
    w[:, 0::2] = (byte % 16).double()
    w[:, 1::2] = (byte // 16).double()
    w = w[:, :inner].contiguous()
    for k in range(s["scales"].shape[1]):
        part = w[:, k * group:(k + 1) * group]
        part -= s["zeros"][:, k:k + 1].double() if s["zeros"] is not None else 8.0
        part *= s["scales"][:, k:k + 1].double()
    return [(s["x"].double() @ w.t()).reshape(-1)]
