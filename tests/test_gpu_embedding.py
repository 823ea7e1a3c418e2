"""baguanet.ops.embedding against its definition in 64 bits.

Tolerances: the lookup is one fp32 product and one rounding; a gradient row is
an fp32 sum of its c terms (each addition is off by at most half a step of a
partial sum, which the sum of the magnitudes bounds), one product and one
rounding.  Half a step is eps / 2 of the value, 2**-24 in fp32; float16 also
has a smallest step of 2**-24.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, ref, extra):
    """|got - ref| within one rounding of got's type and `extra`."""
    d = got.dtype
    got = got.detach().double().cpu()
    tol = ref.abs() * _half(d) * (1 + 2 * U32) + extra + 2.0 ** -25 * (d == HF)
    off = (got - ref).abs()
    assert (off <= tol).all(), (off - tol).max().item()


def case(vocab, dim, n, wtype=BF, out=None, scale=1.0, pad=None, tok=None,
         index=torch.int64, seed=0):
    from baguanet import ops

    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(vocab, dim, generator=g)).to(wtype)
    if tok is None:
        tok = torch.randint(0, vocab, (n,), generator=g)
    dout = torch.randn(*tok.shape, dim, generator=g).to(out or wtype)
    wd = w.cuda().requires_grad_()
    y = ops.embedding(wd, tok.to(index).cuda(), scale=scale, padding_idx=pad,
                      out_dtype=out)
    (dw,) = torch.autograd.grad(y, wd, dout.cuda())
    assert y.dtype == (out or wtype) and dw.dtype == wtype
    assert y.shape == (*tok.shape, dim) and dw.shape == w.shape

    s = torch.tensor(scale, dtype=F32).double()
    ref = w.double()[tok] * s
    check(y, ref, ref.abs() * U32)
    flat, d = tok.reshape(-1), dout.double().reshape(-1, dim)
    if pad is not None:
        keep = flat != pad % vocab
        flat, d = flat[keep], d[keep]
    sums = torch.zeros(vocab, dim, dtype=torch.float64)
    mags = sums.clone()
    sums.index_add_(0, flat, d)
    mags.index_add_(0, flat, d.abs())
    count = torch.bincount(flat, minlength=vocab).double()[:, None]
    check(dw, sums * s, (count + 2) * U32 * mags * s.abs())
    return dw


@pytest.mark.parametrize("dim", [1, 7, 8, 64, 65, 1001, 2048, 2056])
def test_widths(dim):
    case(97, dim, 300, seed=dim)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128, 129, 1000, 4097])
def test_lengths(n):
    case(50, 24, n, wtype=F32, seed=n)


@pytest.mark.parametrize("vocab", [1, 2, 3, 1023, 1024, 70001, 1050000])
def test_tables(vocab):
    case(vocab, 8, 9000, wtype=F32, seed=vocab)


@pytest.mark.parametrize("n", [16384, 16385, 40000, 131072])
def test_long(n):
    """Past one tile of the sort, with some tokens far above the rest."""
    g = torch.Generator().manual_seed(n)
    u = torch.rand(n, generator=g)
    tok = (torch.exp(u * 8.0) - 1).long()
    case(3000, 16, n, wtype=F32, tok=tok, seed=n)


@pytest.mark.parametrize("vocab,dim,n", [
    (20000, 40, 200000), (30000, 5, 150000), (12000, 1000, 131072),
    (9000, 2056, 70000), (20000, 17, 600000)])
def test_many_runs(vocab, dim, n):
    """Tokens with frequencies over their rank: some runs of thousands and
    thousands of runs of a few."""
    g = torch.Generator().manual_seed(dim)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    tok = ((vocab + 1.0) ** u - 1.0).long().clamp_(0, vocab - 1)
    case(vocab, dim, n, tok=torch.randperm(vocab, generator=g)[tok], scale=0.5,
         pad=3, seed=n)


@pytest.mark.parametrize("wtype", [BF, HF, F32])
@pytest.mark.parametrize("out", [BF, HF, F32])
def test_types(wtype, out):
    case(211, 72, 500, wtype=wtype, out=out, scale=3.3)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("pad", [None, 0, 5, -1])
def test_padding(index, pad):
    tok = torch.randint(0, 9, (6, 50), generator=torch.Generator())
    dw = case(9, 40, 300, tok=tok, index=index, pad=pad)
    if pad is not None:
        assert (dw[pad] == 0).all()


@pytest.mark.parametrize("n", [1, 64, 65, 5000])
def test_one_token_everywhere(n):
    case(1000, 136, n, tok=torch.full((n,), 777), wtype=F32)


def test_runs_across_borders():
    """Runs that end at, before and after the borders of a sum's parts."""
    lengths = [64, 63, 1, 65, 128, 127, 129, 1, 62, 2, 300, 64, 64]
    tok = torch.cat([torch.full((c,), i) for i, c in enumerate(lengths)])
    tok = tok[torch.randperm(len(tok), generator=torch.Generator())]
    case(len(lengths), 88, len(tok), tok=tok, wtype=F32)


def test_only_padding():
    dw = case(7, 16, 100, tok=torch.full((100,), 3), pad=3)
    assert (dw == 0).all()


def test_one_token_without_dimensions():
    from baguanet import ops

    w = torch.randn(9, 40, device="cuda", requires_grad=True)
    tok = torch.tensor(4, device="cuda")
    y = ops.embedding(w, tok, scale=2.0)
    assert y.shape == (40,) and torch.equal(y, 2.0 * w[4])
    (dw,) = torch.autograd.grad(y.sum(), w)
    want = torch.zeros_like(w)
    want[4] = 2.0
    assert torch.equal(dw, want)
    with torch.no_grad():
        out = ops.embedding(w, tok[None], scale=2.0)
    assert torch.equal(out[0], y) and not out.requires_grad


def test_no_tokens():
    from baguanet import ops

    w = torch.randn(5, 16, device="cuda", requires_grad=True)
    tok = torch.zeros(0, 4, dtype=torch.int64, device="cuda")
    y = ops.embedding(w, tok)
    assert y.shape == (0, 4, 16)
    (dw,) = torch.autograd.grad(y.sum(), w)
    assert (dw == 0).all()


def test_tokens_outside_the_table():
    from baguanet import ops

    w = torch.randn(6, 20, device="cuda", requires_grad=True)
    tok = torch.tensor([0, -1, 6, 5, 2 ** 40, -2 ** 62, 5], device="cuda")
    y = ops.embedding(w, tok)
    ok = torch.tensor([0, 3, 6], device="cuda")
    assert torch.equal(y[ok], w[tok[ok]])
    assert y[[1, 2, 4, 5]].isnan().all()
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    want = torch.zeros_like(w)
    want[0], want[5] = 1, 2
    assert torch.equal(dw, want)


def test_strides():
    """A slice of a table's columns, and gradients in several layouts."""
    from baguanet import ops

    g = torch.Generator().manual_seed(3)
    big = torch.randn(30, 50, generator=g).cuda()
    tok = torch.randint(0, 30, (4, 25), generator=g).cuda()
    for w in (big[:, 3:41], big[:, :40].t().contiguous().t(),
              big[::2][:, 1:]):
        t = tok % w.shape[0]
        leaf = w.detach().requires_grad_()
        y = ops.embedding(leaf, t)
        assert torch.equal(y, leaf[t])
        d = torch.randn(*y.shape, device="cuda")
        wide = torch.randn(4, 25, w.shape[1] + 3, device="cuda")
        grads = [d, d.transpose(0, 1).contiguous().transpose(0, 1),
                 wide[..., 2:-1], d[:1, :1].expand_as(y),
                 d[0, 0, 0].expand_as(y)]
        for do in grads:
            (dw,) = torch.autograd.grad(y, leaf, do, retain_graph=True)
            want = torch.zeros(w.shape, dtype=torch.float64)
            want.index_add_(0, t.reshape(-1).cpu(),
                            do.double().cpu().reshape(-1, w.shape[1]))
            # at most 100 terms of normal deviates, each below 8
            assert (dw.double().cpu() - want).abs().max() < 102 * U32 * 800


def test_same_every_time():
    from baguanet import ops

    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(500, 256, device="cuda", generator=g, requires_grad=True)
    tok = torch.randint(0, 500, (30000,), device="cuda", generator=g)
    d = torch.randn(30000, 256, device="cuda", generator=g)
    first = None
    for _ in range(4):
        (dw,) = torch.autograd.grad(ops.embedding(w, tok), w, d)
        first = dw if first is None else first
        assert torch.equal(dw, first)


def test_differences():
    """The gradient's product with a direction is the lookup's change."""
    from baguanet import ops

    g = torch.Generator().manual_seed(5)
    w = torch.randn(40, 33, generator=g).cuda().requires_grad_()
    v = torch.randn(40, 33, generator=g).cuda()
    tok = torch.randint(0, 40, (200,), generator=g).cuda()
    c = torch.randn(200, 33, generator=g).cuda()
    y = ops.embedding(w, tok, scale=0.5)
    (dw,) = torch.autograd.grad(y, w, c)
    with torch.no_grad():
        hi = ops.embedding(w + v, tok, scale=0.5).double()
        lo = ops.embedding(w - v, tok, scale=0.5).double()
    slope = (c.double() * (hi - lo)).sum() / 2
    # the lookup is linear: what differs is fp32 rounding, at most 4 roundings
    # of numbers below 8 in each of the 200 * 33 terms, and the row sums
    bound = (c.abs().double() * 4 * 8 * U32).sum() + 40 * 33 * 60 * U32 * 64
    assert (slope - (dw.double() * v.double()).sum()).abs() < bound


def test_not_twice_differentiable():
    from baguanet import ops

    w = torch.randn(5, 8, device="cuda", requires_grad=True)
    y = ops.embedding(w, torch.tensor([1, 2], device="cuda"))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y.sum(), w, create_graph=True)


def test_other_stream():
    from baguanet import ops

    w = torch.randn(300, 64, device="cuda", requires_grad=True)
    tok = torch.randint(0, 300, (5000,), device="cuda")
    d = torch.randn(5000, 64, device="cuda")
    (want,) = torch.autograd.grad(ops.embedding(w, tok), w, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        (got,) = torch.autograd.grad(ops.embedding(w, tok), w, d)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_graph_replays():
    from baguanet import ops

    w = torch.randn(400, 72, device="cuda", requires_grad=True)
    tok = torch.randint(0, 400, (20000,), device="cuda")
    d = torch.randn(20000, 72, device="cuda")

    def step():
        y = ops.embedding(w, tok, scale=2.0, padding_idx=4)
        return y.detach(), torch.autograd.grad(y, w, d)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = step()
    for i in range(4):
        with torch.no_grad():
            w.add_(0.5)
        tok.copy_(torch.randint(0, 400 >> i, (20000,), device="cuda"))
        d.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want_y, want_dw = step()
        assert torch.equal(y, want_y) and torch.equal(dw, want_dw)
