"""The training-step operators on tensors of more than 2**31 elements.

Rows far into such a tensor have to come out bit for bit as they do in a call
of their own: an offset that is cut to 32 bits would take another row's.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _room():
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GiB of GPU memory")
    yield
    torch.cuda.empty_cache()


def _noise(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", dtype=BF, generator=g)


def test_embedding_table():
    """2**32 elements and some: lookups and gradients at its far end."""
    from baguanet import ops

    vocab, dim = (1 << 20) + 3, 4104
    w = torch.zeros(vocab, dim, device="cuda", dtype=BF)
    near = _noise(5, dim)
    rows = torch.tensor([0, 523_300, 523_301, vocab - 2, vocab - 1],
                        device="cuda")
    w[rows] = near
    w.requires_grad_()
    tok = rows[torch.arange(40, device="cuda") % 5]
    y = ops.embedding(w, tok, 2.0)
    assert torch.equal(y, ops.embedding(near, torch.arange(40, device="cuda")
                                        % 5, 2.0))
    dout = _noise(40, dim, seed=1)
    (dw,) = torch.autograd.grad(y, w, dout)
    small = near.clone().requires_grad_()
    (want,) = torch.autograd.grad(
        ops.embedding(small, torch.arange(40, device="cuda") % 5, 2.0), small,
        dout)
    assert torch.equal(dw[rows], want)
    for part in dw.split(1 << 18):  # nothing else was written
        assert int((part != 0).any(1).sum()) == int(
            ((rows >= (part.storage_offset() // dim))
             & (rows < part.storage_offset() // dim + len(part))).sum())


def test_embedding_gradient_rows():
    """Gradients of more than 2**31 elements, and the sums' parts with them."""
    from baguanet import ops

    n, dim, vocab = 530_000, 4096, 37
    g = torch.Generator(device="cuda").manual_seed(2)
    tok = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    dout = torch.zeros(n, dim, device="cuda", dtype=BF)
    # small whole numbers in a few rows: every order of summing is exact
    live = torch.tensor([0, 1, 63, 64, 400_000, 524_287, 524_288, n - 1],
                        device="cuda")
    dout[live] = torch.randint(-4, 5, (len(live), dim), device="cuda",
                               generator=g).to(BF)
    w = torch.zeros(vocab, dim, device="cuda", requires_grad=True)
    y = ops.embedding(w, tok, out_dtype=BF)
    (dw,) = torch.autograd.grad(y, w, dout)
    want = torch.zeros(vocab, dim, device="cuda")
    for i in live.tolist():
        want[tok[i]] += dout[i].float()
    assert torch.equal(dw, want)


def test_norm_rows():
    from baguanet import ops

    rows, dim = 263_000, 8192
    ends = [slice(0, 64), slice(262_100, 262_200), slice(rows - 70, rows)]
    x = _noise(rows, dim).requires_grad_()
    o = x.detach().flip(0).requires_grad_()
    w = torch.rand(dim, device="cuda")
    outs = ops.gated_residual_norm(x, o, None, w, w)
    dy = torch.roll(x.detach(), 7, 0)
    got = torch.autograd.grad(outs, (x, o), (dy, dy))
    for s in ends:
        xs = x.detach()[s].clone().requires_grad_()
        os_ = o.detach()[s].clone().requires_grad_()
        few = ops.gated_residual_norm(xs, os_, None, w, w)
        want = torch.autograd.grad(few, (xs, os_), (dy[s], dy[s]))
        for a, b in zip((*outs, *got), (*few, *want)):
            assert torch.equal(a[s], b)


def test_norm_gate_of_every_element():
    from baguanet import ops

    rows, dim = 263_000, 8192
    x = _noise(rows, dim)
    gate = torch.roll(x, 3, 0).requires_grad_()
    y, _ = ops.gated_residual_norm(x, x, gate)
    (dg,) = torch.autograd.grad(y, gate, x)
    for s in (slice(0, 9), slice(262_140, 262_150), slice(rows - 9, rows)):
        few = gate.detach()[s].clone().requires_grad_()
        ys, _ = ops.gated_residual_norm(x[s], x[s], few)
        (want,) = torch.autograd.grad(ys, few, x[s])
        assert torch.equal(y[s], ys) and torch.equal(dg[s], want)


def test_checkpoint_rows():
    from baguanet import ops

    rows, dim = 263_000, 8200
    x = _noise(rows, dim).requires_grad_()
    kept = ops.act8_pack(x)
    back = ops.act8_unpack(kept)
    out = ops.silu_mul_act8(x)
    dout = out.detach()
    (dx,) = torch.autograd.grad(out, x, dout)
    for s in (slice(0, 9), slice(261_880, 261_900), slice(rows - 9, rows)):
        xs = x.detach()[s].clone().requires_grad_()
        few = ops.act8_pack(xs)
        assert torch.equal(kept.codes[s], few.codes)
        assert torch.equal(kept.exponents[s], few.exponents)
        assert torch.equal(back[s], ops.act8_unpack(few))
        ys = ops.silu_mul_act8(xs)
        (want,) = torch.autograd.grad(ys, xs, dout[s])
        assert torch.equal(out[s], ys) and torch.equal(dx[s], want)


@pytest.mark.parametrize("m,n,k", [(263_000, 8200, 64), (263_000, 64, 8224)])
def test_wgrad_rows(m, n, k):
    """Long dy, and long codes: small whole numbers in a few rows, exact."""
    from baguanet import ops

    g = torch.Generator(device="cuda").manual_seed(3)
    dy = torch.zeros(m, n, device="cuda", dtype=BF)
    x = torch.zeros(m, k, device="cuda", dtype=BF)
    live = torch.tensor([0, 63, 64, 261_300, 262_143, 262_144, m - 1],
                        device="cuda")
    for t in (dy, x):
        t[live] = torch.randint(-4, 5, (len(live), t.shape[1]), device="cuda",
                                generator=g).to(BF)
    dw, db = ops.act8_wgrad(dy, ops.act8_pack(x))
    want = dy[live].double().t() @ x[live].double()
    assert torch.equal(dw.double(), want)
    assert torch.equal(db.double(), dy[live].double().sum(0))


def test_wgrad_result():
    from baguanet import ops

    m, n, k = 65, 70_000, 33_000
    g = torch.Generator(device="cuda").manual_seed(4)
    dy = torch.randint(-2, 3, (m, n), device="cuda", generator=g).to(BF)
    x = torch.randint(-2, 3, (m, k), device="cuda", generator=g).to(BF)
    dw, _ = ops.act8_wgrad(dy, ops.act8_pack(x), bias=False)
    for s in (slice(0, 300), slice(64_900, 65_300), slice(n - 300, n)):
        want = dy[:, s].t().float() @ x.float()
        assert torch.equal(dw[s].float(), want.to(BF).float())


@pytest.mark.parametrize("per", ["element", "row"])
def test_repeated_gate_rows(per):
    """A gate that stands for three sequences: terms past 2^31, and their sums
    as those of a few rows alone."""
    from baguanet import ops

    rows, dim = 88_000, 8200
    x = _noise(3 * rows, dim).view(3, rows, dim)
    gate = x[0, :, :dim if per == "element" else 1].clone().requires_grad_()
    y, _ = ops.gated_residual_norm(x, x, gate)
    (dg,) = torch.autograd.grad(y, gate, x)
    assert dg.shape == gate.shape
    for s in (slice(0, 9), slice(85_800, 85_810), slice(rows - 9, rows)):
        few = gate.detach()[s].clone().requires_grad_()
        ys, _ = ops.gated_residual_norm(x[:, s], x[:, s], few)
        (want,) = torch.autograd.grad(ys, few, x[:, s])
        assert torch.equal(y[:, s], ys) and torch.equal(dg[s], want)
