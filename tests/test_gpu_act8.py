"""baguanet.ops' 8-bit activation checkpoints against their definition.

Codes are whole: pack and unpack are compared bit by bit with the definition
in 64 bits.  A weight gradient is an fp32 sum over m rows of exact products:
each addition is off by at most one step of 2**-23 (matrix instructions may
cut instead of rounding) relative to the sum of the magnitudes, and the result
is rounded once.  The gated activation is a chain of fewer than 8 fp32
operations, each off by at most one step of 2**-23, and one rounding.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
POWERS = {F32: (-117, 120), BF: (-117, 120), HF: (-15, 8)}


def kept(x):
    """The values that x is kept as, in 64 bits, from the definition."""
    lo, hi = POWERS[x.dtype]
    cols = x.shape[-1]
    v = x.detach().double().cpu().reshape(-1, cols)
    v = torch.nn.functional.pad(v, (0, -cols % 32)).reshape(v.shape[0], -1, 32)
    a = torch.where(v.isfinite(), v.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(a / 448.0)
    e = e - (m == 0.5).int()  # the smallest e with a <= 448 * 2**e
    e = torch.where(a > 0, e, 0).clamp(lo, hi)
    z = torch.ldexp(v, -e)
    step = torch.ldexp(torch.ones(()).double(),
                       torch.frexp(z.abs().clamp_min(2.0 ** -6))[1] - 4)
    z = torch.round(z / step) * step
    cap = torch.where(e == hi, 240.0, 448.0).double()
    z = torch.where(z.abs() > cap, z.sign() * cap, z)
    z = torch.where(v.isfinite(), z, math.nan)
    return torch.ldexp(z, e).reshape(v.shape[0], -1)[:, :cols].reshape(x.shape)


def same(got, want):
    want = want.to(got.dtype).double()
    return torch.equal(torch.nan_to_num(got.double().cpu(), nan=1e300),
                       torch.nan_to_num(want, nan=1e300))


def within(got, ref, extra):
    d = got.dtype
    got = got.detach().double().cpu()
    tol = (ref.abs() * torch.finfo(d).eps / 2 * (1 + 2 * U) + extra
           + 2.0 ** -25 * (d == HF) + 1e-36)
    off = (got - ref).abs()
    assert got.shape == ref.shape
    assert (off <= tol).all(), (off / tol).max().item()


def rows(shape, dtype, seed=0, wild=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if wild:  # some columns far above, some far below the rest
        x[..., ::13] *= 50.0
        x[..., 5::17] *= 1e-3
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 256),
                                   (2, 3, 1001), (300, 2048), (9, 5000)])
def test_kept_values(dtype, shape):
    from baguanet import ops

    x = rows(shape, dtype)
    k = ops.act8_pack(x.cuda())
    assert k.shape == x.shape and k.dtype == dtype
    got = ops.act8_unpack(k)
    assert got.dtype == dtype and same(got, kept(x))


@pytest.mark.parametrize("shape", [(1, 2048), (1, 2049), (2, 4096), (3, 4129),
                                   (511, 2081), (512, 2081), (4, 70000)])
def test_rows_in_pieces(shape):
    """Few long rows are cut: whole, and beside the gated activation."""
    from baguanet import ops

    x = rows(shape, BF, 7)
    assert same(ops.act8_unpack(ops.act8_pack(x.cuda())), kept(x))
    both = torch.cat([x, x.flip(-1)], -1).cuda().requires_grad_()
    out = ops.silu_mul_act8(both)
    g = torch.ones_like(out)
    (dx,) = torch.autograd.grad(out, both, g)
    for r in (0, shape[0] - 1):  # a row comes out as it does alone
        one = both.detach()[r:r + 1].clone().requires_grad_()
        few = ops.silu_mul_act8(one)
        assert torch.equal(out[r:r + 1], few)
        assert torch.equal(dx[r:r + 1],
                           torch.autograd.grad(few, one, g[r:r + 1])[0])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_every_magnitude(dtype):
    """From the smallest to the largest numbers of the type, ties among
    them."""
    from baguanet import ops

    top = 16 if dtype == HF else 128
    low = -24 if dtype == HF else -149 if dtype == F32 else -133
    parts = torch.arange(256, 512).double() / 256  # 8 bits of significand
    x = torch.cat([torch.ldexp(parts, torch.tensor(e - 1))
                   for e in range(low, top + 1)]).to(dtype)
    x = x[x.isfinite()]
    n = len(x) // 32 * 32
    alone = torch.zeros(len(x), 32, dtype=dtype)
    alone[:, 3] = x
    spread = x[torch.randperm(len(x), generator=torch.Generator())][:n]
    for t in (x[:n].view(-1, 32), -alone, spread.view(-1, 32)):
        assert same(ops.act8_unpack(ops.act8_pack(t.cuda())), kept(t))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_not_finite(dtype):
    from baguanet import ops

    x = rows((4, 70), dtype)
    x[0, 3], x[1, 40], x[2, 69] = math.nan, math.inf, -math.inf
    x[3, 32:64] = math.nan
    x[3, 64:] = torch.finfo(dtype).max
    got = ops.act8_unpack(ops.act8_pack(x.cuda()))
    assert same(got, kept(x))
    assert got.isfinite().cpu().equal(x.isfinite())


def test_zeros_and_strides():
    from baguanet import ops

    z = torch.zeros(3, 64, device="cuda", dtype=BF)
    assert (ops.act8_unpack(ops.act8_pack(z)) == 0).all()
    assert ops.act8_unpack(ops.act8_pack(z[:0])).shape == (0, 64)
    assert ops.act8_unpack(ops.act8_pack(z[:, :0])).shape == (3, 0)
    big = rows((6, 8, 200), BF).cuda()
    for x in (big[..., 7:107], big[:, ::2, :33], big.transpose(0, 2),
              big[..., :1].expand(6, 8, 50), big[:1].expand(4, 8, 200),
              big[0, 0, 3:90]):
        assert same(ops.act8_unpack(ops.act8_pack(x)), kept(x))


def wgrad(m, n, k, dtype, seed=0, dy=None):
    from baguanet import ops

    x = rows((m, k), dtype, seed)
    dy = rows((m, n), dtype, seed + 1, wild=False).cuda() if dy is None else dy
    dw, db = ops.act8_wgrad(dy, ops.act8_pack(x.cuda()))
    assert dw.dtype == db.dtype == dtype
    d, q = dy.double().cpu(), kept(x)
    within(dw, d.t() @ q, (3 * m + 8) * 2 * U * (d.abs().t() @ q.abs()))
    within(db, d.sum(0), (m + 8) * U * d.abs().sum(0))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 130, 70), (17, 8, 32), (31, 64, 65), (32, 128, 128),
    (33, 129, 257), (64, 255, 96), (100, 7, 1000), (257, 300, 260)])
def test_wgrad(dtype, m, n, k):
    wgrad(m, n, k, dtype, seed=m)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k", [(5000, 40, 72), (2048, 512, 256),
                                   (1000, 1000, 1000), (20000, 3, 5)])
def test_wgrad_long(dtype, m, n, k):
    """Few tiles and many rows: the rows are cut in slices."""
    wgrad(m, n, k, dtype)


@pytest.mark.parametrize("dtype,m,n,k", [
    (BF, 1000, 2048, 8448), (F32, 700, 2048, 8440), (BF, 1000, 8448, 2048),
    (F32, 130, 8449, 2050), (HF, 300, 4401, 4350), (BF, 600, 4352, 4352)])
def test_wgrad_of_uneven_sizes(dtype, m, n, k):
    """A few tiles more than a round of the chip's: dW is computed in parts."""
    wgrad(m, n, k, dtype, seed=n)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k", [
    (1, 3, 40), (2, 1, 33), (63, 7, 8), (64, 255, 64), (65, 257, 300),
    (129, 9, 500), (4097, 129, 40), (640, 513, 1025), (900, 4353, 4000)])
def test_wgrad_of_odd_rows(dtype, m, n, k):
    """The last value of dy lies in half of the 4 bytes that reads count."""
    wgrad(m, n, k, dtype, seed=m)
    from baguanet import ops

    # that value alone, exact, from a tensor that ends with its storage and
    # from the middle of a larger one
    for dy in (torch.zeros(m, n, dtype=dtype, device="cuda"),
               torch.full((m + 2, n + 4), 7.0, dtype=dtype,
                          device="cuda")[1:m + 1, 3:n + 3]):
        dy.zero_()
        dy[-1, -1] = 3.0
        x = rows((m, k), dtype, 3).cuda()
        dw, db = ops.act8_wgrad(dy, ops.act8_pack(x))
        want = kept(x)[-1].cuda() * 3.0
        assert torch.equal(dw[-1], want.to(dtype))
        assert (dw[:-1] == 0).all() and (db[:-1] == 0).all() and db[-1] == 3


def test_wgrad_strides():
    big = rows((200, 150), BF, 3, wild=False).cuda()
    for dy in (big[:, 3:77], big[::2, 1:], big.t(), big[:1].expand(90, 150),
               big[:, :1].expand(200, 60)):
        wgrad(dy.shape[0], dy.shape[1], 100, BF, dy=dy)


def test_wgrad_extremes():
    """fp32 gradients from the largest numbers down to the smallest."""
    from baguanet import ops

    top = torch.finfo(F32).max
    dy = torch.tensor([[top], [2.0 ** -100], [-3.3e-38], [1 / 3]]).cuda()
    x = torch.eye(4).cuda()
    dw, _ = ops.act8_wgrad(dy, ops.act8_pack(x))
    want = dy.double().cpu().t()
    # 2**-133 for what three bf16 numbers cannot hold below their smallest
    assert ((dw.double().cpu() - want).abs()
            <= want.abs() * 4 * U + 2.0 ** -126).all()
    dy[1, 0] = math.inf
    dw, db = ops.act8_wgrad(dy, ops.act8_pack(x))
    assert dw[0, 1].isinf() and db[0].isinf()


def test_wgrad_empty():
    from baguanet import ops

    for m, n, k in ((0, 3, 40), (3, 0, 40), (3, 5, 0)):
        x = torch.ones(m, k, device="cuda")
        dy = torch.ones(m, n, device="cuda")
        dw, db = ops.act8_wgrad(dy, ops.act8_pack(x))
        assert dw.shape == (n, k) and (dw == 0).all()
        assert db.shape == (n,) and (db == m).all()
        assert ops.act8_wgrad(dy, ops.act8_pack(x), bias=False)[1] is None


def test_linear_act8():
    from baguanet import ops

    for dtype in (BF, F32):
        x = rows((4, 30, 96), dtype).cuda().requires_grad_()
        w = rows((50, 96), dtype, 1, wild=False).cuda().requires_grad_()
        b = rows((50,), dtype, 2, wild=False).cuda().requires_grad_()
        dy = rows((4, 30, 50), dtype, 3, wild=False).cuda()
        y = ops.linear_act8(x, w, b)
        want = torch.nn.functional.linear(x, w, b)
        assert torch.equal(y, want)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        (want_dx,) = torch.autograd.grad(want, x, dy)
        assert torch.equal(dx, want_dx)
        want_dw, want_db = ops.act8_wgrad(dy, ops.act8_pack(x))
        assert torch.equal(dw, want_dw) and torch.equal(db, want_db)
        # each gradient alone, and without a bias
        y = ops.linear_act8(x.detach(), w)
        assert torch.equal(torch.autograd.grad(y, w, dy)[0], dw)
        y = ops.linear_act8(x.detach(), w.detach(), b)
        assert torch.equal(torch.autograd.grad(y, b, dy)[0], db)
        y = ops.linear_act8(x, w.detach())
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], dx)


def test_linear_act8_layouts():
    """Inputs and gradients that do not collapse to rows."""
    from baguanet import ops

    big = rows((6, 20, 130), BF).cuda()
    w = rows((48, 64), BF, 1, wild=False).cuda().requires_grad_()
    for x in (big[..., 3:67], big[:, :, :64].transpose(0, 1),
              big[:, ::3, 5:69], big[:1, :1, :64].expand(5, 7, 64)):
        a, b = (v.detach().requires_grad_() for v in (x, x.contiguous()))
        ya, yb = ops.linear_act8(a, w), ops.linear_act8(b, w)
        assert torch.equal(ya, yb)
        d = rows((*x.shape[:-1], 48), BF, 2, wild=False).cuda()
        for g in (d, d.transpose(0, 1).contiguous().transpose(0, 1),
                  d[..., :1].expand_as(d), d[:, :1].expand_as(d)):
            ga = torch.autograd.grad(ya, (a, w), g, retain_graph=True)
            gb = torch.autograd.grad(yb, (b, w), g.contiguous(),
                                     retain_graph=True)
            assert all(torch.equal(p, q) for p, q in zip(ga, gb))
        with torch.no_grad():
            assert torch.equal(ops.linear_act8(x, w), ya)


def test_linear_act8_of_one_row_and_under_autocast():
    from baguanet import ops

    x = rows((96,), F32).cuda().requires_grad_()
    w = rows((50, 96), F32, 1, wild=False).cuda().requires_grad_()
    b = rows((50,), F32, 2, wild=False).cuda().requires_grad_()
    dy = rows((50,), F32, 3, wild=False).cuda()
    want = torch.autograd.grad(ops.linear_act8(x, w, b), (x, w, b), dy)
    assert want[1].equal(torch.outer(dy, ops.act8_unpack(ops.act8_pack(x))))
    with torch.autocast("cuda", torch.bfloat16):
        y = ops.linear_act8(x, w, b)
        got = torch.autograd.grad(y, (x, w, b), dy)
    assert y.dtype == F32  # it computes in its arguments' type
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    with torch.no_grad():
        assert torch.equal(ops.linear_act8(x, w, b),
                           torch.nn.functional.linear(x, w, b))


def test_linear_act8_holds_codes_only():
    from baguanet import ops

    w = torch.randn(64, 4096, device="cuda", dtype=BF, requires_grad=True)
    x = torch.randn(8192, 4096, device="cuda", dtype=BF)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ops.linear_act8(x, w)
    held = torch.cuda.memory_allocated() - before - y.nbytes
    # 33 bytes for 32 values, and the allocator's rounding of two blocks
    assert held <= x.numel() * 33 / 32 + 2 * 2 ** 21
    del y


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shape", [(1, 2), (3, 14), (5, 128), (2, 7, 2002),
                                   (130, 4096), (9, 10002)])
def test_silu(dtype, shape):
    from baguanet import ops

    x = (rows(shape, dtype, wild=False).float() * 3).to(dtype)
    g = rows((*shape[:-1], shape[-1] // 2), dtype, 1, wild=False)
    xd = x.cuda().requires_grad_()
    out = ops.silu_mul_act8(xd)
    (dx,) = torch.autograd.grad(out, xd, g.cuda())
    a, b = x.double().chunk(2, -1)
    ref = a * torch.sigmoid(a) * b
    within(out, ref, 16 * U * ref.abs())
    a, b = (kept(v) for v in x.chunk(2, -1))
    s, d = torch.sigmoid(a), g.double()
    da = d * b * s * (1 + a * (1 - s))
    db = d * a * s
    da_tol = (d * b * s).abs() * (1 + a.abs()) * 16 * U
    within(dx, torch.cat([da, db], -1),
           torch.cat([da_tol, 16 * U * db.abs()], -1))


def test_silu_far_values():
    from baguanet import ops

    a = torch.tensor([-1e30, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 1e30])
    x = torch.cat([a, torch.ones(8)])[None].cuda().requires_grad_()
    out = ops.silu_mul_act8(x)
    (dx,) = torch.autograd.grad(out.sum(), x)
    assert out.isfinite().all() and dx[0, 1:].isfinite().all()
    want = a.double() * torch.sigmoid(a.double())
    within(out[0], want, 16 * U * want.abs())


def test_silu_differences():
    """Its gradient against differences of the definition in 64 bits, at the
    kept values."""
    from baguanet import ops

    x = rows((6, 80), F32, wild=False)
    v = rows((6, 80), F32, 1, wild=False).double()
    c = rows((6, 40), F32, 2, wild=False)
    xd = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(ops.silu_mul_act8(xd), xd, c.cuda())
    at = torch.cat([kept(t) for t in x.chunk(2, -1)], -1)

    def f(s):
        a, b = (at + s * v).chunk(2, -1)
        return (a * torch.sigmoid(a) * b * c).sum()

    h = 1e-3
    slope = (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)
    # 480 terms below 50, each within 17 steps of its own
    assert ((dx.double().cpu() * v).sum() - slope).abs() < 480 * 50 * 34 * U


def test_silu_strides_and_empty():
    from baguanet import ops

    big = rows((6, 8, 90), BF, wild=False).cuda()
    for x in (big[..., 3:77], big[:, ::2, :60], big[..., :80].transpose(0, 1),
              big[:1, :1, :44].expand(6, 8, 44)):
        a, b = (v.detach().requires_grad_() for v in (x, x.contiguous()))
        ya, yb = ops.silu_mul_act8(a), ops.silu_mul_act8(b)
        assert torch.equal(ya, yb)
        d = big[..., :x.shape[-1] // 2].reshape(-1)[:ya.numel()].view_as(ya)
        for g in (d, d[..., :1].expand_as(d)):
            ga = torch.autograd.grad(ya, a, g, retain_graph=True)[0]
            gb = torch.autograd.grad(yb, b, g.contiguous(),
                                     retain_graph=True)[0]
            assert torch.equal(ga, gb)
    for shape in ((0, 8), (4, 0)):
        x = torch.zeros(*shape, device="cuda", requires_grad=True)
        y = ops.silu_mul_act8(x)
        assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    with torch.no_grad():  # nothing kept, the same result
        assert torch.equal(ops.silu_mul_act8(big),
                           ops.silu_mul_act8(big.clone().requires_grad_()))


@pytest.mark.parametrize("what", ["linear", "silu"])
def test_not_twice_differentiable(what):
    from baguanet import ops

    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    y = (ops.silu_mul_act8(x) if what == "silu"
         else ops.linear_act8(x, torch.ones(2, 8, device="cuda")))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_same_every_time_streams_and_graph():
    from baguanet import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    x, dy = rand(3000, 520), rand(3000, 200)
    z, dz = rand(3000, 520).requires_grad_(), rand(3000, 260)

    def step():
        dw, db = ops.act8_wgrad(dy, ops.act8_pack(x))
        out = ops.silu_mul_act8(z)
        return dw, db, out.detach(), torch.autograd.grad(out, z, dz)[0]

    equal = lambda p, q: all(torch.equal(a, b) for a, b in zip(p, q))
    want = step()
    for _ in range(3):
        assert equal(step(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        with torch.no_grad():
            for t in (x, dy, z, dz):
                t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert equal(got, step())


@pytest.mark.parametrize("big", [1.0, 3e20, 2e37])
def test_silu_of_tails(big):
    """Where 1 / (1 + exp(-a)) itself is below fp32's smallest normal number
    and the product with b is not: the factors are multiplied apart.  exp is
    within a step of 2**-23 and enters twice, and six more operations follow."""
    from baguanet import ops

    a = -torch.arange(60, 124).float() * 0.875 - torch.rand(
        5, 64, generator=torch.Generator().manual_seed(1))
    b = (1 + torch.rand(5, 64, generator=torch.Generator().manual_seed(2)))
    x = torch.cat([a, b * big], -1)
    g = rows((5, 64), F32, 3, wild=False)
    xd = x.cuda().requires_grad_()
    out = ops.silu_mul_act8(xd)
    (dx,) = torch.autograd.grad(out, xd, g.cuda())
    a, b = x.double().chunk(2, -1)
    # half a step among the numbers below the smallest normal one is 2**-150
    def near(got, ref, rel):
        off = (got.detach().double().cpu() - ref).abs()
        assert (off <= ref.abs() * rel + 8 * 2.0 ** -150).all(), (
            off / ref.abs()).max()

    near(out, a / (1 + (-a).exp()) * b, 16 * U)
    a, b = (kept(v) for v in x.chunk(2, -1))
    s, d = 1 / (1 + (-a).exp()), g.double()
    da, db = dx.chunk(2, -1)
    near(da, d * b * s * (1 + a * (1 - s)), 24 * U)
    near(db, d * a * s, 16 * U)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_documented_error_of_kept_values(dtype):
    """At most 1/16 of the value, 2**-10 / 224 of its group's largest or, but
    for fp16, 2**-127, whichever is most.  In a group whose largest is just
    above 224 a step's half is 2**-10, and values just below it become 0."""
    from baguanet import ops

    top = torch.tensor([224.5, 225.0, 240.0, 256.0, 256.5, 300.0, 447.0, 448.0,
                        448.5, 449.0]).to(dtype).double()
    below = torch.cat([torch.tensor([0.99, 1.01, 1.49, 1.51, 2.49, 2.51, 3.0])
                       * 2.0 ** e for e in range(-12, 0)])
    g = torch.Generator().manual_seed(2)
    wide = torch.exp2(torch.rand(len(top), 60, generator=g) * 24 - 16)
    x = torch.cat([below.expand(len(top), -1), wide], 1).double()
    n = x.shape[1] // 31
    x = torch.cat([top[:, None, None].expand(-1, n, 1),
                   x[:, :n * 31].reshape(len(top), n, 31)], -1).flatten(1)
    powers = (0, -6) if dtype == HF else (0, 100, -100, -125, -135)
    for p in powers:
        v = (x * 2.0 ** p).to(dtype)
        got = ops.act8_unpack(ops.act8_pack(v.cuda())).double().cpu()
        v = v.double()
        most = v.reshape(len(v), -1, 32).amax(-1, keepdim=True)
        most = most.expand(-1, -1, 32).reshape(v.shape)
        bound = torch.maximum(v / 16, most * 2.0 ** -10 / 224)
        if dtype != HF:
            bound = bound.clamp_min(2.0 ** -127)
        assert ((got - v).abs() <= bound).all()
        if p == 0:  # values come near the second bound
            worst = ((got - v).abs() / most)[v < most / 2 ** 16].max()
            assert worst > 0.9 * 2.0 ** -10 / 224


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bias", [True, False])
def test_wgrad_of_gradients_below_the_smallest_normal(dtype, bias):
    """Gradients without loss scaling: among fp16's numbers below 2**-14 (or
    bf16's below 2**-126) a product is as exact as any other."""
    from baguanet import ops

    m, n, k = 300, 140, 96
    g = torch.Generator().manual_seed(6)
    low = torch.finfo(dtype).smallest_normal
    step = low * torch.finfo(dtype).eps
    whole = torch.randint(-20, 21, (m, n), generator=g)
    dy = (whole.double() * step).to(dtype)
    assert (dy != 0).any() and (dy.abs().double() < low).all()
    # whole numbers of at most 3 bits times 2**8 and 2**13: the products' sums
    # are exact in fp32 and come out above the smallest normal number
    x = torch.randint(-7, 8, (m, k), generator=g).float() * 2.0 ** 8
    x[:, ::3] *= 2.0 ** 5
    x = x.to(dtype)
    kept_x = ops.act8_pack(x.cuda())
    assert torch.equal(ops.act8_unpack(kept_x).cpu(), x)
    dw, db = ops.act8_wgrad(dy.cuda(), kept_x, bias=bias)
    d = dy.double()
    within_exact = lambda got, ref: torch.equal(got.cpu(), ref.to(dtype))
    assert within_exact(dw, d.t() @ x.double())
    assert not bias or within_exact(db, d.sum(0))
    dw, _ = ops.act8_wgrad(dy.float().cuda(), ops.act8_pack(x.float().cuda()))
    want = d.t() @ x.double()
    if dtype == HF:  # ordinary numbers of fp32
        assert torch.equal(dw.double().cpu(), want)


def test_wgrad_of_fp32_down_to_its_smallest():
    """Three bf16 numbers of 8 bits hold an fp32 number from 2**-110 on; below
    it what their smallest, 2**-133, cannot hold is lost: less than that for
    each value."""
    from baguanet import ops

    g = torch.Generator().manual_seed(8)
    e = torch.arange(-149, 128).double()
    dy = (torch.rand(len(e), generator=g).double() + 1) * torch.exp2(e)
    dy = torch.cat([dy.float(), -dy.float()])[:, None]
    n = len(dy)
    x = torch.eye(n)
    dw, _ = ops.act8_wgrad(dy.cuda(), ops.act8_pack(x.cuda()))
    want = dy.double().t()
    assert ((dw.double().cpu() - want).abs()
            <= want.abs() * 4 * U + 2.0 ** -133).all()


def test_linear_act8_does_not_hold_its_input():
    """What a graph keeps of a layer's input that is not kept elsewhere: the
    codes, no less and no more."""
    from baguanet import ops

    w = torch.randn(64, 4096, device="cuda", dtype=BF, requires_grad=True)
    ops.linear_act8(torch.randn(8, 4096, device="cuda", dtype=BF), w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    x = torch.randn(8192, 4096, device="cuda", dtype=BF)
    y = ops.linear_act8(x, w)
    values = x.numel()
    del x
    held = torch.cuda.memory_allocated() - before - y.nbytes
    # torch rounds each of the two blocks up to 512 bytes
    assert values * 33 / 32 <= held <= values * 33 / 32 + 2 * 512
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    del y
    assert torch.cuda.memory_allocated() - before - dw.nbytes <= 512


def test_silu_holds_codes_only():
    from baguanet import ops

    ops.silu_mul_act8(torch.randn(8, 64, device="cuda", dtype=BF,
                                  requires_grad=True))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    leaf = torch.randn(4096, 4096, device="cuda", dtype=BF, requires_grad=True)
    x = leaf * 1.0
    y = ops.silu_mul_act8(x)
    values, own = x.numel(), leaf.nbytes + y.nbytes
    del x
    held = torch.cuda.memory_allocated() - before - own
    # multiplied by a plain number: torch keeps nothing for that
    assert values * 33 / 32 <= held <= values * 33 / 32 + 4 * 512
