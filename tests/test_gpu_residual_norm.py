"""baguanet.ops.rms_norm and gated_residual_norm against their definition in
64 bits.

Tolerances: outputs are rounded once to their type (half a step: eps / 2 of
the value, and half of float16's smallest step of 2**-24).  Before that all is
fp32: a sum of at most 16384 terms goes through fewer than 48 additions on any
path (8 of a vector, 2 vectors, 6 lane exchanges, 16 waves), and the products
around it add fewer than 16 roundings, so C = 64 half steps of 2**-24, relative
to the sum of the magnitudes, bound each number before its last rounding.
Sums over R rows add R roundings.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
C = 64 * U


def check(got, ref, extra, what):
    d = got.dtype
    assert got.shape == ref.shape, what
    got = got.detach().double().cpu()
    tol = (ref.abs() * torch.finfo(d).eps / 2 * (1 + C) + extra * (1 + 2 ** -6)
           + 2.0 ** -25 * (d == HF) + 1e-37)
    off = (got - ref).abs()
    assert (off <= tol).all(), (what, (off / tol).max().item())


def reference(x, o, gate, post, pre, rs, bs, eps, dy, dh):
    """Values, gradients and how far each may be off before its rounding."""
    dim = x.shape[-1]
    x, o = x.double(), o.double()
    one = torch.ones((), dtype=torch.float64)
    g = one if gate is None else gate.double()
    wp = one if post is None else post.double()
    wn = one if pre is None else pre.double()
    ro = one
    if post is not None:
        ro = (o.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    no = o * ro
    u = no * wp
    y = rs * x + bs * g * u
    e_y = C * ((rs * x).abs() + (bs * g * u).abs())
    out = {"y": (y, e_y)}
    ry = (y.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    ny = y * ry
    if pre is not None:
        rel = (y.abs() * e_y).mean(-1, keepdim=True) * ry ** 2 + C
        h = ny * wn
        out["h"] = (h, (wn * ry).abs() * e_y + h.abs() * rel)
    dy = torch.zeros_like(x) if dy is None else dy.double()
    t = torch.zeros_like(x)
    if pre is not None and dh is not None:
        dh = dh.double()
        t = dh * wn
    rel = (y.abs() * e_y).mean(-1, keepdim=True) * ry ** 2
    e_ny = ry * e_y + ny.abs() * (C + rel)
    mean = (ny * t).mean(-1, keepdim=True)
    mean_abs = (ny * t).abs().mean(-1, keepdim=True)
    e_mean = (e_ny * t.abs()).mean(-1, keepdim=True) + C * mean_abs
    d = dy + ry * (t - ny * mean)
    d_abs = dy.abs() + ry * (t.abs() + ny.abs() * mean_abs)
    e_d = (C + rel) * d_abs + ry * (e_ny * mean_abs + ny.abs() * e_mean)
    out["dx"] = (rs * d, abs(rs) * e_d)
    c = bs * g * wp
    if post is None:
        out["dbranch"] = (c * d, c.abs() * (e_d + C * d_abs))
    else:
        mean = (no * c * d).mean(-1, keepdim=True)
        e_in = (e_d + C * d_abs) * c.abs()
        e_mean = (no.abs() * e_in).mean(-1, keepdim=True)
        out["dbranch"] = (ro * (c * d - no * mean),
                          ro * (e_in + no.abs() * (e_mean + C * mean.abs())))
    rows = x.numel() // dim
    flat = lambda v: v.expand_as(x).reshape(-1, dim)
    if pre is not None and dh is not None:
        p = dh * ny
        out["dpre"] = (flat(p).sum(0),
                       flat(dh.abs() * e_ny + p.abs() * (C + rows * U)).sum(0))
    if post is not None:
        p = bs * g * d * no
        e = (bs * g * no).abs() * (e_d + (C + rows * U) * d_abs)
        out["dpost"] = (flat(p).sum(0), flat(e).sum(0))
    if gate is not None:
        p = bs * d * u
        e = (bs * u).abs() * (e_d + (C + (rows + dim) * U) * d_abs)
        out["dgate"] = (p.sum_to_size(gate.shape), e.sum_to_size(gate.shape))
    return out


def case(shape, dtype=BF, gate=None, post=True, pre=True, wtype=F32,
         rs=1.0, bs=1.0, eps=1e-6, seed=0, use=("y", "h"), spread=1.0):
    from baguanet import ops

    gen = torch.Generator().manual_seed(seed)
    rand = lambda s, t: torch.randn(s, generator=gen).to(t)
    dim = shape[-1]
    x, o = rand(shape, dtype), (rand(shape, F32) * spread).to(dtype)
    g = None if gate is None else rand(gate, wtype)
    wp = (1 + 0.2 * rand((dim,), F32)).to(wtype) if post else None
    wn = (1 + 0.2 * rand((dim,), F32)).to(wtype) if pre else None
    dy = rand(shape, dtype) if "y" in use else None
    dh = rand(shape, dtype) if "h" in use and pre else None
    dev = {k: None if v is None else v.cuda().requires_grad_()
           for k, v in dict(x=x, branch=o, gate=g, post=wp, pre=wn).items()}
    y, h = ops.gated_residual_norm(
        dev["x"], dev["branch"], gate=dev["gate"], post_weight=dev["post"],
        pre_weight=dev["pre"], residual_scale=rs, branch_scale=bs, eps=eps)
    assert (h is None) == (not pre)
    outs = [(v, d.cuda()) for v, d in ((y, dy), (h, dh)) if d is not None]
    names = [k for k, v in dev.items() if v is not None]
    grads = torch.autograd.grad([v for v, _ in outs], [dev[k] for k in names],
                                [d for _, d in outs], allow_unused=True)
    got = {"y": y, **({"h": h} if pre else {}),
           **{"d" + k: v for k, v in zip(names, grads)}}
    f32 = lambda v: float(torch.tensor(v, dtype=F32))
    ref = reference(x, o, g, wp, wn, f32(rs), f32(bs), f32(eps), dy, dh)
    if dh is None and pre:
        assert got.pop("dpre") is None
    assert set(got) == set(ref)
    for k, v in ref.items():
        check(got[k], *v, what=k)


@pytest.mark.parametrize("dim", [1, 2, 7, 8, 9, 15, 64, 511, 512, 513, 1000, 1024, 1025,
                                 2048, 2049, 4096, 4100, 8192, 8193, 12289,
                                 16383, 16384])
def test_widths(dim):
    case((2, 5, dim), gate=(dim,), bs=0.5, seed=dim)
    case((2, 5, dim), dtype=F32, gate=(2, 1, dim), bs=0.5, seed=dim + 1)


@pytest.mark.parametrize("rows", [1, 2, 3, 9, 600, 4099])
@pytest.mark.parametrize("dim", [72, 2080])
def test_lengths(rows, dim):
    case((rows, dim), gate=(dim,), seed=rows)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("dim", [136, 3000])
def test_types(dtype, own, dim):
    case((3, 17, dim), dtype=dtype, wtype=dtype if own else F32,
         gate=(3, 1, dim), rs=0.7, bs=-1.3, eps=1e-5)


@pytest.mark.parametrize("gate", [
    None, (40,), (1, 1, 40), (6, 1, 40), (6, 23, 40), (6, 23, 1), (1, 23, 40),
    (23, 40), (23, 1), (6, 1, 1), (1,), (), (1, 23, 1)])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
def test_gates(gate, post, pre):
    case((6, 23, 40), gate=gate, post=post, pre=pre, bs=0.3, dtype=F32)


@pytest.mark.parametrize("shape,gate", [
    ((700, 3, 264), (700, 1, 264)),    # more groups than workgroups
    ((5, 1, 264), (5, 1, 264)),        # groups of one row
    ((3, 1000, 264), (3, 1, 264)),     # groups cut in slices
    ((2, 7, 33, 264), (2, 7, 1, 264)),
    ((1500, 264), (1500, 1)),
    ((3, 500, 2100), (3, 1, 2100)),
    ((3, 40, 9001), (3, 1, 9001)),
    ((600, 2, 9001), (600, 1, 9001)),
    ((600, 2, 65), (600, 1, 65)),
    ((600, 2, 5), (600, 1, 5)),
    ((1, 1, 264), (1, 1, 264)),
    ((1, 264), (1, 1)),
])
def test_groups(shape, gate):
    case(shape, gate=gate, bs=0.5)


@pytest.mark.parametrize("kind", ["none", "column", "group", "row", "each"])
@pytest.mark.parametrize("dim", [3, 300, 600, 787, 1024, 1999, 4000, 8000,
                                 9001])
def test_gates_of_every_width(kind, dim):
    gate = {"none": None, "column": (dim,), "group": (3, 1, dim),
            "row": (3, 37, 1), "each": (3, 37, dim)}[kind]
    case((3, 37, dim), dtype=HF if dim % 2 else BF, gate=gate, bs=0.5,
         seed=dim)


@pytest.mark.parametrize("shape,gate", [
    ((1100, 2, 787), (1100, 1, 787)), ((2, 1500, 787), (2, 1, 787)),
    ((4099, 600), (4099, 1)), ((9000, 1000), None)])
def test_rows_of_two_waves(shape, gate):
    case(shape, gate=gate, bs=0.5)


@pytest.mark.parametrize("use", [("y",), ("h",)])
@pytest.mark.parametrize("post", [True, False])
def test_one_output_used(use, post):
    case((4, 9, 520), gate=(520,), use=use, post=post)


def test_small_values_keep_eps():
    case((8, 256), dtype=F32, spread=1e-4, eps=1e-6, gate=(256,))


def test_rms_norm():
    from baguanet import ops

    for dim in (5, 768, 5000):
        for weight in (True, False):
            gen = torch.Generator().manual_seed(dim)
            x = torch.randn(11, dim, generator=gen).to(BF)
            w = torch.randn(dim, generator=gen) if weight else None
            dh = torch.randn(11, dim, generator=gen).to(BF)
            xd = x.cuda().requires_grad_()
            wd = w.cuda().requires_grad_() if weight else None
            h = ops.rms_norm(xd, wd, eps=1e-5)
            leaves = [xd] + ([wd] if weight else [])
            grads = torch.autograd.grad(h, leaves, dh.cuda())
            ref = reference(x, torch.zeros_like(x), None, None,
                            w if weight else torch.ones(dim), 1.0, 1.0,
                            float(torch.tensor(1e-5)), None, dh)
            check(h, *ref["h"], what="h")
            check(grads[0], *ref["dx"], what="dx")
            if weight:
                check(grads[1], *ref["dpre"], what="dw")


@pytest.mark.parametrize("dim", [600, 2000, 4096, 8000, 16384])
def test_each_row_is_its_own(dim):
    """With many rows for each workgroup, every row comes out as it does in a
    call of its own few: sums over rows of one workgroup do not meet."""
    from baguanet import ops

    g = torch.Generator(device="cuda").manual_seed(dim)
    rows = 6000 if dim > 8192 else 12000
    x = torch.randn(rows, dim, device="cuda", generator=g)
    x *= torch.rand(rows, 1, device="cuda", generator=g) * 100
    w = torch.rand(dim, device="cuda", generator=g)
    o = x.flip(0)
    calls = [lambda a, b: ops.rms_norm(a, w),
             lambda a, b: ops.gated_residual_norm(a, b, w, None, w)[1],
             lambda a, b: ops.gated_residual_norm(a, b, w, w, None)[0],
             lambda a, b: ops.gated_residual_norm(a, b, w, w, w)[1]]
    for call in calls:
        whole = call(x, o)
        for i in range(0, rows, 250):
            s = slice(i, i + 250)
            assert torch.equal(whole[s], call(x[s], o[s]))


def test_one_row_and_no_grad():
    from baguanet import ops

    x, o = (torch.randn(600, device="cuda", requires_grad=True)
            for _ in range(2))
    w = torch.rand(600, device="cuda", requires_grad=True)
    y, h = ops.gated_residual_norm(x, o, w, w, w, branch_scale=0.5)
    assert y.requires_grad and h.requires_grad
    with torch.no_grad():
        y1, h1 = ops.gated_residual_norm(x, o, w, w, w, branch_scale=0.5)
        assert torch.equal(y, y1) and torch.equal(h, h1)
        y1, h1 = ops.gated_residual_norm(x[None], o[None], w, w, None, 1, 0.5)
        assert h1 is None and torch.equal(y, y1[0])
        n1 = ops.rms_norm(x, w)
    assert not n1.requires_grad
    assert torch.equal(ops.rms_norm(x, w), n1)


def test_empty():
    from baguanet import ops

    for shape in ((0, 16), (3, 0)):
        x = torch.zeros(*shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        g = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y, h = ops.gated_residual_norm(x, x, g, w, w)
        assert y.shape == h.shape == x.shape
        grads = torch.autograd.grad((y.sum(), h.sum()), (x, w, g))
        assert all((v == 0).all() for v in grads)


def test_rows_do_not_mix():
    """NaN and infinities of one row stay in it; a row of zeros is fine."""
    from baguanet import ops

    x = torch.randn(6, 300, device="cuda")
    o = torch.randn(6, 300, device="cuda")
    w = torch.ones(300, device="cuda")
    y0, h0 = ops.gated_residual_norm(x, o, None, w, w)
    x[1, 7], o[2, 3] = float("nan"), float("inf")
    x[4], o[4] = 0, 0
    y, h = ops.gated_residual_norm(x, o, None, w, w)
    for r in (0, 3, 5):
        assert torch.equal(y[r], y0[r]) and torch.equal(h[r], h0[r])
    assert y[1, 7].isnan() and h[1].isnan().all()
    assert h[2].isnan().any()
    assert (y[4] == 0).all() and (h[4] == 0).all()


def test_strides():
    """Sliced, transposed and expanded inputs and gradients give what their
    dense copies give."""
    from baguanet import ops

    gen = torch.Generator().manual_seed(2)
    big = torch.randn(4, 10, 99, generator=gen).cuda()
    w = torch.rand(128, generator=gen).cuda()[::2][:61]
    pairs = [(big[..., 1:62], big[..., 30:91]),
             (big[:, ::2, :61], big[:, 1::2, 5:66]),
             (big[..., :61].transpose(0, 1), big[..., 7:68].transpose(0, 1)),
             (big[:1, :1, :61].expand(4, 10, 61), big[..., 2:63]),
             (big[..., :1].expand(4, 10, 61), big[..., 38:])]
    for x, o in pairs:
        for d in (big[..., :x.shape[-1]].reshape(-1)[:x.numel()].view(x.shape),
                  x.detach() * 0.5, o[..., :1].expand_as(o)):
            res = []
            for dense in (False, True):
                f = (lambda v: v.detach().clone(
                    memory_format=torch.contiguous_format)) if dense else (
                    lambda v: v.detach())
                # a leaf for each use: autograd's own sum of three gradients
                # of one leaf has no fixed order
                leaves = [f(v).requires_grad_() for v in (x, o, w, w, w)]
                y, h = ops.gated_residual_norm(*leaves)
                res.append((y, h) + torch.autograd.grad(
                    (y, h), leaves, (f(d), f(d))))
            assert all(torch.equal(p, q) for p, q in zip(*res))


def test_same_every_time():
    from baguanet import ops

    g = torch.Generator(device="cuda").manual_seed(1)
    t = [torch.randn(3, 900, 520, device="cuda", generator=g).to(BF)
         .requires_grad_() for _ in range(2)]
    gate = torch.randn(3, 1, 520, device="cuda", generator=g).requires_grad_()
    w = torch.rand(520, device="cuda", generator=g).requires_grad_()
    first = None
    for _ in range(4):
        y, h = ops.gated_residual_norm(*t, gate, w, w)
        out = torch.autograd.grad((y, h), (*t, gate, w), (t[0], t[1]))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_differences():
    """Gradients against differences of the definition in 64 bits."""
    from baguanet import ops

    gen = torch.Generator().manual_seed(4)
    shape, dim = (3, 5, 72), 72
    vals = [torch.randn(*s, generator=gen) for s in
            (shape, shape, (3, 1, dim), (dim,), (dim,))]
    dirs = [torch.randn(*v.shape, generator=gen) for v in vals]
    cy, ch = (torch.randn(*shape, generator=gen) for _ in range(2))
    leaves = [v.cuda().requires_grad_() for v in vals]
    y, h = ops.gated_residual_norm(*leaves, branch_scale=0.75, eps=1e-5)
    grads = torch.autograd.grad((y, h), leaves, (cy.cuda(), ch.cuda()))

    def f(s):
        x, o, g, wp, wn = (v.double() + s * d.double()
                           for v, d in zip(vals, dirs))
        n = lambda v: v / (v.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
        y = x + 0.75 * g * n(o) * wp
        return (y * cy).sum() + (n(y) * wn * ch).sum()

    # central differences of two steps cancel the h**2 term; what is left is
    # of the order of h**4 = 1e-12 and rounding of 1e-16 * |f| / h
    h1 = 1e-3
    slope = (8 * (f(h1) - f(-h1)) - (f(2 * h1) - f(-2 * h1))) / (12 * h1)
    ref = reference(*vals, 1.0, 0.75, float(torch.tensor(1e-5)), cy, ch)
    got = bound = 0.0
    for name, d, v in zip(("dx", "dbranch", "dgate", "dpost", "dpre"),
                          dirs, grads):
        r, e = ref[name]
        got = got + (v.double().cpu() * d).sum()
        bound = bound + ((e + r.abs() * U) * d.abs()).sum()
    assert (got - slope).abs() <= bound + 1e-7 * slope.abs() + 1e-7


def test_not_twice_differentiable():
    from baguanet import ops

    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(ops.rms_norm(x).sum(), x, create_graph=True)


def test_other_stream_and_graph():
    from baguanet import ops

    x, o = (torch.randn(4, 300, 1100, device="cuda").to(BF).requires_grad_()
            for _ in range(2))
    gate = torch.randn(4, 1, 1100, device="cuda").requires_grad_()
    w = torch.rand(1100, device="cuda").requires_grad_()
    dy, dh = torch.randn_like(x), torch.randn_like(x)

    def step():
        y, h = ops.gated_residual_norm(x, o, gate, w, w, branch_scale=0.1)
        return (y.detach(), h.detach()) + torch.autograd.grad(
            (y, h), (x, o, gate, w), (dy, dh))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        with torch.no_grad():
            for t in (x, o, gate, dy, dh):
                t.normal_()
            w.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape,gate", [
    ((6, 23, 40), g) for g in (
        (40,), (6, 1, 40), (6, 23, 40), (6, 23, 1), (1, 23, 40), (23, 40),
        (23, 1), (6, 1, 1), (1,), (), (1, 23, 1), (1, 1, 1))
] + [
    ((3, 5, 7, 40), g) for g in (
        (5, 1, 40), (3, 1, 7, 40), (3, 1, 7, 1), (5, 1, 1), (1, 5, 1, 1),
        (7, 1), (7, 40), (3, 1, 1, 1), (1, 5, 7, 1))
] + [
    ((2, 3, 4, 5, 24), g) for g in (
        (3, 1, 5, 1), (2, 1, 4, 1, 1), (1, 3, 1, 5, 24), (2, 1, 4, 1, 24))
] + [
    ((1, 23, 40), (23, 1)), ((40,), (1,)), ((40,), ()), ((1, 1, 1), ()),
    ((4, 0, 8), (4, 1, 1)), ((6, 0, 8), ()), ((4, 0, 8), (0, 8)),
    ((20001, 24), ()), ((2, 6000, 72), (6000, 1)), ((300, 90, 16), (90, 16)),
    ((3, 4000, 8), (3, 1, 1)), ((700, 40, 9), (700, 1, 1)),
    ((64, 65, 264), (1, 264)), ((5000, 3, 8), (3, 1)),
])
def test_repeated_gates_round_once(dtype, shape, gate):
    """A gate of two bytes that is repeated over rows or elements: its
    gradient is summed in fp32, whatever it is repeated over."""
    case(shape, gate=gate, dtype=dtype, wtype=dtype, bs=0.3, seed=len(gate))


@pytest.mark.parametrize("gate", [(), (1,), (1, 1)])
def test_repeated_gate_whose_terms_pass_its_largest(gate):
    """Two rows give 70000 and -69000, each past fp16's 65504: their sum is
    1000, exact in fp32 and fp16."""
    from baguanet import ops

    half = lambda v: torch.tensor(v, dtype=HF, device="cuda")
    x, g = half([[0.0], [0.0]]), torch.ones(gate, dtype=HF, device="cuda")
    o = half([[250.0], [250.0]])
    g.requires_grad_()
    y, _ = ops.gated_residual_norm(x, o, g)
    (dg,) = torch.autograd.grad(y, g, half([[280.0], [-276.0]]))
    assert dg.shape == g.shape and dg.item() == 1000.0


@pytest.mark.parametrize("gate", [(), (900, 1), (900, 520), (3, 1, 1)])
def test_repeated_gates_in_a_graph(gate):
    """The same in every run, and in every replay of a captured pass."""
    from baguanet import ops

    rand = lambda *s: torch.randn(s, device="cuda").to(BF)
    x, o = (rand(3, 900, 520).requires_grad_() for _ in range(2))
    g, w = rand(*gate).requires_grad_(), rand(520).requires_grad_()
    dy, dh = rand(3, 900, 520), rand(3, 900, 520)

    def step():
        y, h = ops.gated_residual_norm(x, o, g, w, w, branch_scale=0.5)
        return torch.autograd.grad((y, h), (x, o, g, w), (dy, dh))

    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))
    want = step()
    assert same(step(), want) and same(step(), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        with torch.no_grad():
            for t in (x, o, g, w, dy, dh):
                t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, step())
