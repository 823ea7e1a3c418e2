"""Cases for timing and checking the training-step operators of baguanet.ops.

Four operators, each in a plain form (elementary torch operations, 32 bits,
rounded once at the end) and as a user calls it from the framework:

* ``embedding``   lookup of scaled table rows; the table's gradient is summed
                  over the sorted tokens.
* ``norm``        gated sandwich norm around a block: the block's output is
                  normed, gated, scaled and added to the residual stream, and
                  the sum is normed for the next block.
* ``act8_linear`` the input of a linear layer kept in 8 bits between forward
                  and backward, and the weight gradient taken from it.
* ``act8_silu``   the gated activation ``silu(a) * b`` with its two inputs
                  kept in 8 bits for the backward pass.

A case with ``train`` true is one forward and one backward pass; the others
are forward passes as in generation, with few rows.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ---------------------------------------------------------------------------
# the cases

def listed():
    return [
        # one step of generation for eight sequences: latency only
        dict(name="emb_decode", op="embedding", vocab=50000, dim=1024, n=8,
             type="bf16", out="bf16", scale=32.0, pad=0.0, train=False),
        # a short training sequence over a small table with odd sizes, the
        # table in fp32 (master weights) and its rows in bf16
        dict(name="emb_odd_fp32", op="embedding", vocab=20011, dim=1001,
             n=2049, type="fp32", out="bf16", scale=1.0, pad=0.0, train=True),
        # one ordinary micro-batch, 8 sequences of 2048 tokens
        dict(name="emb_step", op="embedding", vocab=50000, dim=2048, n=16384,
             type="bf16", out="bf16", scale=45.25, pad=0.0, train=True),
        # a large micro-batch, a tenth of it padding, and a large table
        dict(name="emb_large", op="embedding", vocab=131072, dim=4096,
             n=65536, type="bf16", out="bf16", scale=1.0, pad=0.1, train=True),
        # generation: one token of each of four sequences through the seam
        # between two blocks
        dict(name="norm_decode", op="norm", seqs=4, length=1, dim=4096,
             type="bf16", gate="channel", train=False),
        # an adaptive gate for each sequence, odd lengths, a middling width
        dict(name="norm_adaptive", op="norm", seqs=7, length=1027, dim=1536,
             type="fp16", gate="sequence", train=True),
        # a large micro-batch of a wide model
        dict(name="norm_large", op="norm", seqs=16, length=2048, dim=8192,
             type="bf16", gate="none", train=True),
        # the first classifier layer of VGG16 at batch 256, in its own fp32
        dict(name="linear_vgg", op="act8_linear", m=256, n=4096, k=25088,
             type="fp32"),
        # odd sizes everywhere
        dict(name="linear_odd", op="act8_linear", m=2053, n=1537, k=1100,
             type="fp16"),
        # a large micro-batch through a wide layer
        dict(name="linear_large", op="act8_linear", m=16384, n=8192, k=4096,
             type="bf16"),
        # the gated activation between the layers of such a block
        dict(name="silu_odd", op="act8_silu", rows=1025, dim=1377,
             type="bf16"),
        dict(name="silu_large", op="act8_silu", rows=16384, dim=8192,
             type="bf16"),
    ]


def _span(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo),
                                                      math.log(hi))))))


def draw(rng):
    op = rng.choice(["embedding", "norm", "act8_linear", "act8_silu"])
    typ = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        if op == "embedding":
            train = rng.random() < 0.75
            c = dict(op=op, vocab=_span(rng, 1000, 131072),
                     dim=_span(rng, 64, 4096),
                     n=_span(rng, 1, 65536 if train else 256), type=typ,
                     out=rng.choice([typ, "bf16"]),
                     scale=rng.choice([1.0, 0.5, 22.625]),
                     pad=rng.choice([0.0, 0.0, 0.2]), train=train)
        elif op == "norm":
            train = rng.random() < 0.75
            c = dict(op=op, seqs=_span(rng, 1, 32),
                     length=_span(rng, 1, 4096) if train else 1,
                     dim=_span(rng, 64, 8192), type=typ,
                     gate=rng.choice(["none", "channel", "sequence", "row"]),
                     train=train)
        elif op == "act8_linear":
            c = dict(op=op, m=_span(rng, 1, 16384), n=_span(rng, 64, 8192),
                     k=_span(rng, 64, 8192), type=typ)
        else:
            c = dict(op=op, rows=_span(rng, 1, 16384),
                     dim=_span(rng, 64, 16384), type=typ)
        w, top = work(c), work(_largest(op))
        # fp32 operands cost the matrix product three times as much
        heavy = 3 if op == "act8_linear" and typ == "fp32" else 1
        if w["bytes"] <= top["bytes"] and heavy * w["flops"] <= top["flops"]:
            return c


def _largest(op):
    return max((c for c in listed() if c["op"] == op),
               key=lambda c: work(c)["flops"])


def work(case):
    op, s = case["op"], SIZE[case["type"]]
    if op == "embedding":
        v, d, n, o = case["vocab"], case["dim"], case["n"], SIZE[case["out"]]
        b = 8 * n + min(n, v) * d * s + n * d * o
        if case["train"]:
            b += n * d * o + v * d * s
        return {"bytes": b, "flops": (2 if case["train"] else 1) * n * d}
    if op == "norm":
        r, d = case["seqs"] * case["length"], case["dim"]
        return {"bytes": (8 if case["train"] else 4) * r * d * s,
                "flops": (36 if case["train"] else 10) * r * d}
    if op == "act8_linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + m * n + n * k) * s + 2 * m * k,
                "flops": 2 * m * n * k}
    r, d = case["rows"], case["dim"]
    return {"bytes": r * d * 6 * s + 4 * r * d, "flops": 25 * r * d}


# ---------------------------------------------------------------------------
# inputs

def _randn(g, shape, typ, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(TYPES[typ])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = {"case": case}
    op, typ = case["op"], case["type"]
    if op == "embedding":
        v, d, n = case["vocab"], case["dim"], case["n"]
        st["weight"] = _randn(g, (v, d), typ, 0.02)
        # words come with a frequency of about one over their rank, and the
        # table holds them in any order; a padded tail has one token
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        st["tokens"] = torch.randperm(v, generator=g, device=DEV)[rank]
        st["pad_id"] = None
        if case["pad"]:
            st["pad_id"] = 1
            st["tokens"][n - int(case["pad"] * n):] = 1
        if case["train"]:
            st["dout"] = _randn(g, (n, d), case["out"])
            st["weight"].requires_grad_()
    elif op == "norm":
        b, t, d = case["seqs"], case["length"], case["dim"]
        st["x"] = _randn(g, (b, t, d), typ, 2.0)
        st["branch"] = _randn(g, (b, t, d), typ, 0.5)
        gates = {"channel": (d,), "sequence": (b, 1, d), "row": (b, t, 1)}
        st["gate"] = (None if case["gate"] == "none"
                      else _randn(g, gates[case["gate"]], typ, 0.5))
        for name in ("post", "pre"):
            st[name] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)
        st["branch_scale"] = 0.25
        if case["train"]:
            st["dy"] = _randn(g, (b, t, d), typ)
            st["dh"] = _randn(g, (b, t, d), typ)
            for name in ("x", "branch", "gate", "post", "pre"):
                if st[name] is not None:
                    st[name].requires_grad_()
    elif op == "act8_linear":
        m, n, k = case["m"], case["n"], case["k"]
        # activations have a few channels far above the rest
        x = torch.randn((m, k), generator=g, device=DEV)
        x[:, ::97] *= 20.0
        st["x"] = x.to(TYPES[typ])
        st["dy"] = _randn(g, (m, n), typ)
    else:
        r, d = case["rows"], case["dim"]
        st["x"] = _randn(g, (r, 2 * d), typ, 2.0).requires_grad_()
        st["dout"] = _randn(g, (r, d), typ)
    return st


# ---------------------------------------------------------------------------
# one pass

def run(state):
    f = _run_own if own else _run_plain
    return f(state)


def _run_own(st):
    from baguanet import ops

    case = st["case"]
    op = case["op"]
    if op == "embedding":
        out = ops.embedding(st["weight"], st["tokens"], scale=case["scale"],
                            padding_idx=st["pad_id"],
                            out_dtype=TYPES[case["out"]])
        if not case["train"]:
            return out
        (dw,) = torch.autograd.grad(out, st["weight"], st["dout"])
        return out.detach(), dw
    if op == "norm":
        y, h = ops.gated_residual_norm(
            st["x"], st["branch"], gate=st["gate"], post_weight=st["post"],
            pre_weight=st["pre"], branch_scale=st["branch_scale"], eps=EPS)
        if not case["train"]:
            return y, h
        leaves = [st[n] for n in ("x", "branch", "post", "pre", "gate")
                  if st[n] is not None]
        grads = torch.autograd.grad((y, h), leaves, (st["dy"], st["dh"]))
        return (y.detach(), h.detach()) + tuple(grads)
    if op == "act8_linear":
        kept = ops.act8_pack(st["x"])
        return ops.act8_wgrad(st["dy"], kept)
    out = ops.silu_mul_act8(st["x"])
    (dx,) = torch.autograd.grad(out, st["x"], st["dout"])
    return out.detach(), dx


@torch.no_grad()
def _run_plain(st):
    case = st["case"]
    op, typ = case["op"], TYPES[case["type"]]
    if op == "embedding":
        out = st["weight"][st["tokens"]].float() * case["scale"]
        out = out.to(TYPES[case["out"]])
        if not case["train"]:
            return out
        dw = torch.zeros(case["vocab"], case["dim"], device=DEV)
        dw.index_add_(0, st["tokens"], st["dout"].float())
        dw *= case["scale"]
        if st["pad_id"] is not None:
            dw[st["pad_id"]] = 0.0
        return out, dw.to(typ)
    if op == "norm":
        return _plain_norm(st, typ)
    if op == "act8_linear":
        kept = _plain_act8(st["x"])
        dy = st["dy"].float()
        return (dy.t() @ kept).to(typ), dy.sum(0).to(typ)
    d = case["dim"]
    a, b = st["x"][:, :d].float(), st["x"][:, d:].float()
    out = (a / (1.0 + torch.exp(-a)) * b).to(typ)
    a, b = _plain_act8(st["x"][:, :d]), _plain_act8(st["x"][:, d:])
    s = 1.0 / (1.0 + torch.exp(-a))
    dout = st["dout"].float()
    da = dout * b * s * (1.0 + a * (1.0 - s))
    return out, torch.cat([da, dout * a * s], 1).to(typ)


def _plain_norm(st, typ):
    case, c = st["case"], st["branch_scale"]
    x, o = st["x"].float(), st["branch"].float()
    gate = None if st["gate"] is None else st["gate"].float()
    post, pre = st["post"], st["pre"]
    ro = torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS)
    no = o * ro
    u = no * post
    g = 1.0 if gate is None else gate
    y = x + c * g * u
    ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    ny = y * ry
    h = ny * pre
    if not case["train"]:
        return y.to(typ), h.to(typ)
    dy, dh = st["dy"].float(), st["dh"].float()
    t = dh * pre
    dx = dy + ry * (t - ny * (ny * t).mean(-1, keepdim=True))
    du = c * g * dx
    t = du * post
    do = ro * (t - no * (no * t).mean(-1, keepdim=True))
    out = [y.to(typ), h.to(typ), dx.to(typ), do.to(typ),
           (du * no).sum((0, 1)), (dh * ny).sum((0, 1))]
    if gate is not None:
        dg = c * dx * u
        dims = {"channel": (0, 1), "sequence": (1,), "row": (2,)}[case["gate"]]
        dg = dg.sum(dims, keepdim=case["gate"] != "channel")
        out.append(dg.to(typ))
    return tuple(out)


# an 8-bit checkpoint: groups of 32 values of a row share a power of two that
# brings the largest finite one to at most 448, and each is then an e4m3
# number; the power is held where the products stay exact in the input's type
_POWERS = {torch.float32: (-117, 120), torch.bfloat16: (-117, 120),
           torch.float16: (-15, 8)}


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _plain_act8(x):
    """The values that the 8-bit copy of x stands for, in 32 bits."""
    r, k = x.shape
    lo, hi = _POWERS[x.dtype]
    v = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(r, -1, 32)
    finite = torch.isfinite(v)
    top = torch.where(finite, v.abs(), torch.zeros_like(v)).amax(-1, True)
    m, e = torch.frexp(top)
    e = e.int() - 9 + (m > 0.875).int()
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(lo, hi)
    cap = torch.where(e == hi, 240.0, 448.0)
    q = torch.minimum(torch.maximum(v * _power(-e), -cap), cap)
    q = torch.where(finite, q, torch.full_like(q, math.nan))
    q = q.to(torch.float8_e4m3fn).float() * _power(e)
    return q.view(r, -1)[:, :k].contiguous()


# ---------------------------------------------------------------------------
# the definitions in 64 bits

@torch.no_grad()
def _exact_act8(x):
    r, k = x.shape
    lo, hi = _POWERS[x.dtype]
    out = torch.empty(r, k, dtype=torch.float64, device=x.device)
    for j in range(0, k, 4096):  # in strips of whole groups, to bound memory
        v = x[:, j:j + 4096].double()
        w = v.shape[1]
        v = torch.cat([v, v.new_zeros(r, -w % 32)], 1).reshape(r, -1, 32)
        a = torch.nan_to_num(v.abs(), nan=0.0, posinf=0.0).max(-1, True)[0]
        e = torch.ceil(torch.log2(a / 448.0))
        # log2 may be off by its last bit next to a whole number
        e = torch.where(a / torch.exp2(e) > 448.0, e + 1, e)
        e = torch.where(a / torch.exp2(e - 1) <= 448.0, e - 1, e)
        e = torch.where(a > 0, e, torch.zeros_like(e)).clamp(lo, hi)
        z = v / torch.exp2(e)
        step = torch.exp2(torch.frexp(z.abs().clamp_min(2.0 ** -6))[1]
                          .double() - 4)
        z = torch.round(z / step) * step
        cap = torch.where(e == hi, 240.0, 448.0).double()
        z = torch.where(z.abs() > cap, torch.sign(z) * cap, z)
        z = torch.where(torch.isfinite(v), z, torch.full_like(z, math.nan))
        out[:, j:j + w] = (z * torch.exp2(e)).reshape(r, -1)[:, :w]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "embedding":
        with torch.no_grad():
            w, tok = st["weight"], st["tokens"]
            out = w.index_select(0, tok).double() * case["scale"]
            if not case["train"]:
                return out
            dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
            live = (torch.ones_like(tok, dtype=torch.bool)
                    if st["pad_id"] is None else tok != st["pad_id"])
            dw.index_put_((tok[live],), st["dout"][live].double()
                          * case["scale"], accumulate=True)
            return out, dw
    if op == "norm":
        leaf = {n: (None if st[n] is None else
                    st[n].detach().double().requires_grad_(case["train"]))
                for n in ("x", "branch", "post", "pre", "gate")}

        def rms(v, w):
            return v / torch.sqrt(v.pow(2).mean(-1, True) + EPS) * w

        u = rms(leaf["branch"], leaf["post"]) * st["branch_scale"]
        y = leaf["x"] + (u if leaf["gate"] is None else u * leaf["gate"])
        h = rms(y, leaf["pre"])
        if not case["train"]:
            return y, h
        at = [v for v in leaf.values() if v is not None]
        grads = torch.autograd.grad((y, h), at, (st["dy"].double(),
                                                 st["dh"].double()))
        return (y.detach(), h.detach()) + tuple(grads)
    if op == "act8_linear":
        dy = st["dy"].double()
        return torch.mm(dy.t().contiguous(), _exact_act8(st["x"])), dy.sum(0)
    d = case["dim"]
    x = st["x"].detach()
    out = torch.empty(x.shape[0], d, dtype=torch.float64, device=DEV)
    dx = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for i in range(0, x.shape[0], 4096):
        s = slice(i, i + 4096)
        a, b = x[s, :d].double(), x[s, d:].double()
        out[s] = a * torch.sigmoid(a) * b
        a, b = _exact_act8(x[s, :d]), _exact_act8(x[s, d:])
        p, do = torch.sigmoid(a), st["dout"][s].double()
        dx[s, :d] = do * b * (p + a * p * (1 - p))
        dx[s, d:] = do * a * p
    return out, dx
