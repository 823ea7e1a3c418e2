"""The training-step operators together, as a language model's step uses them:
embedding, gated residual norms between blocks, blocks whose activations are
kept in 8 bits, under BucketedDDP and FusedSGD."""

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
U = 2.0 ** -24


class Block(nn.Module):
    def __init__(self, dim, hidden, dtype):
        super().__init__()
        rand = lambda *s: nn.Parameter((torch.randn(*s) * s[-1] ** -0.5)
                                       .to(dtype))
        self.up, self.down = rand(2 * hidden, dim), rand(dim, hidden)
        self.bias = nn.Parameter(torch.zeros(2 * hidden, dtype=dtype))
        self.gate = nn.Parameter(torch.ones(dim) * 0.5)
        self.post = nn.Parameter(torch.ones(dim))
        self.pre = nn.Parameter(torch.ones(dim))

    def forward(self, x, h):
        from baguanet import ops

        up = ops.linear_act8(h, self.up, self.bias)
        down = ops.linear_act8(ops.silu_mul_act8(up), self.down)
        return ops.gated_residual_norm(x, down, self.gate, self.post,
                                       self.pre, branch_scale=0.7)


class Net(nn.Module):
    def __init__(self, vocab=97, dim=136, hidden=200, blocks=3, dtype=BF):
        super().__init__()
        torch.manual_seed(0)
        self.table = nn.Parameter((torch.randn(vocab, dim) * 0.1).to(dtype))
        self.first = nn.Parameter(torch.ones(dim))
        self.blocks = nn.ModuleList(Block(dim, hidden, dtype)
                                    for _ in range(blocks))
        self.kept = {}

    def forward(self, tokens):
        from baguanet import ops

        x = ops.embedding(self.table, tokens, scale=dim_scale(self.table),
                          padding_idx=0)
        self.kept["x"] = x
        h = ops.rms_norm(x, self.first)
        for b in self.blocks:
            x, h = b(x, h)
        self.kept["h"] = h
        logits = ops.linear_act8(h, self.table)  # the table is shared
        self.kept["logits"] = logits
        return logits


def dim_scale(table):
    return float(table.shape[1]) ** 0.5


def _batch(seed, n=(4, 33)):
    g = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, 97, n, generator=g)
    tok[:, -3:] = 0  # padding
    return tok.cuda(), torch.randint(0, 97, n, generator=g).cuda()


def _loss(model, batch):
    logits = model(batch[0]).float()
    return nn.functional.cross_entropy(logits.flatten(0, -2),
                                       batch[1].flatten())


def _grads(batches, dtype=BF):
    model = Net(dtype=dtype).cuda()
    out = []
    for b in batches:
        params = list(model.parameters())
        out.append(torch.autograd.grad(_loss(model, b), params))
    return out


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_same_gradients_in_buckets(dtype):
    from baguanet.parallel import BucketedDDP

    batches = [_batch(1), _batch(2)]
    want = _grads(batches, dtype)
    model = BucketedDDP(Net(dtype=dtype).cuda(), bucket_cap_mb=0.1,
                        broadcast_params=False)
    assert len(model.buckets) > 1
    model.zero_grad()
    _loss(model, batches[0]).backward()
    model.finish_backward()
    params = list(model.module.parameters())
    for p, g in zip(params, want[0]):
        assert torch.equal(p.grad, g)
    # a second micro-batch adds up in the buckets
    _loss(model, batches[1]).backward()
    model.finish_backward()
    for p, a, b in zip(params, *want):
        # one of the two sums of the shared table's parts may come first
        both = a.double() + b.double()
        tol = torch.finfo(p.dtype).eps * (a.abs().double() + b.abs().double())
        assert ((p.grad.double() - both).abs() <= tol + 1e-30).all()


def test_steps_with_fused_sgd():
    """Three steps of the optimizer are those of its rule on the gradients,
    and the same in a second run."""
    from baguanet.optim import FusedSGD
    from baguanet.parallel import BucketedDDP

    def train():
        model = BucketedDDP(Net(dtype=torch.float32).cuda(),
                            broadcast_params=False)
        opt = FusedSGD(model.parameters(), lr=0.05, momentum=0.9)
        params = list(model.module.parameters())
        mom = [torch.zeros_like(p) for p in params]
        for i in range(3):
            model.zero_grad()
            loss = _loss(model, _batch(i))
            loss.backward()
            model.finish_backward()
            assert torch.isfinite(loss)
            before = [p.detach().clone() for p in params]
            opt.step()
            for p, old, m in zip(params, before, mom):
                m.mul_(0.9).add_(p.grad)
                # two fp32 products and sums, in one order or another
                tol = 4 * U * (old.abs() + 0.05 * 2 * m.abs())
                tol = tol + 4 * U * 0.05 * p.grad.abs()
                assert ((p - (old - 0.05 * m)).abs() <= tol).all()
        return params

    for a, b in zip(train(), train()):
        assert torch.equal(a, b)


def test_table_gradient_of_both_uses():
    """The shared table's gradient, from what passed through both operators
    that use it, in 64 bits."""
    from baguanet import ops

    model = Net(dtype=torch.float32).cuda()
    batch = _batch(5)
    loss = _loss(model, batch)
    for t in model.kept.values():
        t.retain_grad()
    loss.backward()
    x, h, logits = (model.kept[k] for k in ("x", "h", "logits"))
    dy = logits.grad.double().flatten(0, -2)
    kept = ops.act8_unpack(ops.act8_pack(h.detach())).double().flatten(0, -2)
    head, head_mag = dy.t() @ kept, dy.abs().t() @ kept.abs()
    tok = batch[0].flatten()
    live = tok != 0
    dx = x.grad.double().flatten(0, -2)[live]
    look = torch.zeros_like(head).index_add_(0, tok[live], dx)
    look_mag = torch.zeros_like(head).index_add_(0, tok[live], dx.abs())
    s = dim_scale(model.table)
    want = head + s * look
    # fp32 sums over 132 rows, three times as many in the product of a
    # gradient split in three, one step of 2**-23 each at most
    tol = (3 * 132 + 8) * 2 * U * (head_mag + s * look_mag) + 2 * U * want.abs()
    assert ((model.table.grad.double() - want).abs() <= tol).all()


def test_holds_less_memory():
    """What a block's forward pass leaves for the backward pass."""
    from baguanet import ops

    torch.manual_seed(0)
    rows, dim, hidden = 4096, 1024, 2048
    block = Block(dim, hidden, BF).cuda()
    x = torch.randn(rows, dim, device="cuda").to(BF).requires_grad_()
    h = torch.randn(rows, dim, device="cuda").to(BF).requires_grad_()

    def held(f):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = f()
        now = torch.cuda.memory_allocated() - before
        del out
        return now

    def plain():
        up = nn.functional.linear(h, block.up, block.bias)
        a, b = up.chunk(2, -1)
        down = nn.functional.linear(nn.functional.silu(a) * b, block.down)
        return ops.gated_residual_norm(x, down, block.gate, block.post,
                                       block.pre, branch_scale=0.7)

    ours, theirs = held(lambda: block(x, h)), held(plain)
    # outputs y and h and the branch: 6 bytes a column; codes of the two
    # linear inputs and the gated activation's two: 33/32 of a byte each
    most = rows * (6 * dim + 33 / 32 * (dim + hidden + 2 * hidden))
    assert ours <= most + 16 * 2 ** 21
    # plain: silu's input and result, both factors, the product: 2 bytes each
    assert theirs - ours >= rows * hidden * 2


def test_whole_step_in_a_graph():
    """Forward and backward of the whole net, captured and replayed."""
    model = Net(dtype=torch.float32).cuda()
    params = list(model.parameters())
    batch = _batch(1)

    def step():
        logits = model(batch[0])
        return torch.autograd.grad(logits, params, torch.ones_like(logits))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    model.kept.clear()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    model.kept.clear()
    for i in range(4):
        for t, s in zip(batch, _batch(10 + i)):
            t.copy_(s)
        with torch.no_grad():
            for p in params:
                p.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        model.kept.clear()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def _each_operator():
    """Every operator with a gradient, as a function of its leaves."""
    from baguanet import ops

    g = torch.Generator().manual_seed(5)

    def leaf(*shape):
        return torch.randn(*shape, generator=g).cuda().requires_grad_()

    tok = torch.tensor([[3, 1, 3], [0, 2, 3]], device="cuda")
    return [
        (lambda w: ops.embedding(w, tok, 2.0), [leaf(5, 40)]),
        (lambda x, w: ops.rms_norm(x, w), [leaf(6, 40), leaf(40)]),
        (lambda x, o, gate, post, pre: ops.gated_residual_norm(
            x, o, gate, post, pre)[1],
         [leaf(6, 40), leaf(6, 40), leaf(40), leaf(40), leaf(40)]),
        (lambda x, o, gate, post, pre: ops.gated_residual_norm(
            x, o, gate, post, pre)[0],
         [leaf(2, 3, 40), leaf(2, 3, 40), leaf(2, 1, 40), leaf(40), leaf(40)]),
        (lambda x, w, b: ops.linear_act8(x, w, b),
         [leaf(2, 3, 40), leaf(24, 40), leaf(24)]),
        (lambda x: ops.silu_mul_act8(x), [leaf(6, 80)])]


@pytest.mark.parametrize("which", range(6))
def test_each_gradient_alone(which):
    """Asked for by itself, a gradient is the one of all together."""
    f, leaves = _each_operator()[which]
    y = f(*leaves)
    dout = torch.randn_like(y)
    used = torch.autograd.grad(y, leaves, dout, retain_graph=True,
                               allow_unused=True)
    for leaf, want in zip(leaves, used):
        (got,) = torch.autograd.grad(y, leaf, dout, retain_graph=True,
                                     allow_unused=True)
        assert (got is None) == (want is None)
        assert want is None or torch.equal(got, want)
    # with only one of the leaves in the graph
    for i, want in enumerate(used):
        few = [t if i == j else t.detach() for j, t in enumerate(leaves)]
        if want is not None:
            (got,) = torch.autograd.grad(f(*few), leaves[i], dout)
            assert torch.equal(got, want)


@pytest.mark.parametrize("which", range(6))
def test_graph_is_torchs_own(which):
    """Results changed in place, recomputed blocks, hooks on what is kept,
    freed graphs: as with torch's operators."""
    from torch.utils.checkpoint import checkpoint

    f, leaves = _each_operator()[which]
    y = f(*leaves)
    dout = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dout, allow_unused=True)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dout, allow_unused=True)

    def same(y, dout=dout):
        got = torch.autograd.grad(y, leaves, dout, allow_unused=True)
        for a, b in zip(got, want):
            assert (a is None) == (b is None)
            assert a is None or torch.equal(a, b)

    same(f(*leaves).mul_(2.0), dout / 2)
    same(f(*leaves).view(-1).view(y.shape))
    same(checkpoint(f, *leaves, use_reentrant=False))
    count = []

    def to_host(t):
        count.append(t.numel())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(to_host,
                                                  lambda t: t.cuda()):
        z = f(*leaves)
    assert count
    same(z)
    for leaf in leaves:
        leaf.grad = None
    f(*leaves).backward(dout)
    for leaf, b in zip(leaves, want):
        assert (leaf.grad is None) == (b is None)
        assert b is None or torch.equal(leaf.grad, b)


def test_kept_tensors_are_guarded():
    """A kept tensor that is changed before the backward pass is noticed."""
    from baguanet import ops

    w = torch.randn(40, device="cuda", requires_grad=True)
    x = torch.randn(6, 40, device="cuda")
    y = ops.rms_norm(x, w)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_is_refused(which):
    from torch.autograd import forward_ad

    f, leaves = _each_operator()[which]
    for i, leaf in enumerate(leaves):
        with forward_ad.dual_level(), torch.no_grad():
            duals = [t.detach() for t in leaves]
            duals[i] = forward_ad.make_dual(duals[i], torch.ones_like(leaf))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*duals)


@pytest.mark.parametrize("which", range(6))
def test_gradient_as_a_negated_view(which):
    f, leaves = _each_operator()[which]
    y = f(*leaves)
    dout = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, -dout, retain_graph=True,
                               allow_unused=True)
    got = torch.autograd.grad(y, leaves, torch._neg_view(dout),
                              allow_unused=True)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", range(6))
def test_backward_in_a_recording_is_refused(which):
    from torch.fx.experimental.proxy_tensor import make_fx

    f, leaves = _each_operator()[which]
    y = f(*leaves)
    used = leaves[0]
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        make_fx(lambda d: torch.autograd.grad(y, used, d)[0])(
            torch.ones_like(y))


@pytest.mark.parametrize("which", range(6))
def test_inside_a_compiled_function(which):
    """A compiled function calls the operators as they are."""
    f, leaves = _each_operator()[which]
    y = f(*leaves)
    dout = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dout, allow_unused=True)
    z = torch.compile(lambda *a: f(*a) * 2.0, backend="eager")(*leaves)
    got = torch.autograd.grad(z, leaves, dout * 0.5, allow_unused=True)
    assert torch.equal(z, y * 2.0)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", range(6))
def test_gradient_that_only_stands_for_zeros(which):
    f, leaves = _each_operator()[which]
    y = f(*leaves)
    none = torch._efficientzerotensor(y.shape, device="cuda")
    got = torch.autograd.grad(y, leaves, none, allow_unused=True)
    assert all(v is None or (v == 0).all() for v in got)


def _through(f, leaves, unpack):
    """f of the leaves, with a hook that gives back unpack(kept tensor)."""
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(),
                                                  unpack):
        return f(*leaves)


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("unpack", [
    lambda t: t.to(BF if t.dtype == torch.float32 else torch.int16),
    lambda t: t.cpu(),
    lambda t: t.reshape(-1)[:1],
    lambda t: t[None],
    lambda t: t.to_sparse(),
])
def test_hook_that_gives_back_another_tensor(which, unpack):
    """Another type, place or size than what was kept is refused: the kernels
    would read past its end."""
    f, leaves = _each_operator()[which]
    y = _through(f, leaves, unpack)
    with pytest.raises(RuntimeError, match="kept tensor has become"):
        torch.autograd.grad(y.sum(), leaves, allow_unused=True)


@pytest.mark.parametrize("which", range(6))
def test_hook_that_gives_back_another_layout(which):
    """The same values in other strides, or away from 16 bytes."""
    f, leaves = _each_operator()[which]
    y = f(*leaves)
    dout = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dout, allow_unused=True)

    def apart(t):
        return torch.stack([t, t], -1)[..., 0]

    def shifted(t):
        flat = t.reshape(-1)
        return torch.cat([flat[:1], flat])[1:].view(t.shape)

    def turned(t):
        return t.t().contiguous().t() if t.dim() == 2 else t

    def stands_for_zeros(t):
        return torch._efficientzerotensor(t.shape, dtype=t.dtype,
                                          device=t.device)

    for unpack in (apart, shifted, turned):
        got = torch.autograd.grad(_through(f, leaves, unpack), leaves, dout,
                                  allow_unused=True)
        assert all(a is b or torch.equal(a, b) for a, b in zip(got, want))
    torch.autograd.grad(_through(f, leaves, stands_for_zeros), leaves, dout,
                        allow_unused=True)
    torch.cuda.synchronize()


def test_block_holds_its_codes_outputs_and_branch():
    """A whole block's graph to a few of the allocator's 512 bytes: neither
    the linear layers' inputs nor the activation's result are in it."""
    torch.manual_seed(0)
    rows, dim, hidden = 4096, 1024, 2048
    block = Block(dim, hidden, BF).cuda()
    x = torch.randn(rows, dim, device="cuda").to(BF).requires_grad_()
    h = torch.randn(rows, dim, device="cuda").to(BF).requires_grad_()
    block(x[:8].detach(), h[:8].detach())
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = block(x, h)
    now = torch.cuda.memory_allocated() - before
    # y, h and the branch in 2 bytes; two numbers a row of the norms; 33/32 of
    # a byte for the inputs of both layers and both halves of the activation's
    kept = rows * (6 * dim + 8 + 33 / 32 * (dim + hidden + 2 * hidden))
    assert kept <= now <= kept + 16 * 512
    del out


def test_kept_tensors_that_are_exchanged():
    """Other data under a kept tensor, which is no change in place, and a
    storage that was freed: refused, not read as what it was."""
    from baguanet import ops

    def norm():
        x, o, gate, post, pre = (torch.randn(*s, device="cuda") for s in
                                 ((6, 40), (6, 40), (40,), (40,), (40,)))
        leaves = x, o, gate, post, pre
        for t in (gate, post, pre):
            t.requires_grad_()
        return leaves, ops.gated_residual_norm(*leaves)[1]

    def exchange(f):
        def change(t):
            t.data = f(t.data)
        return change

    changes = [exchange(lambda d: d.to(BF)), exchange(lambda d: d.cpu()),
               exchange(lambda d: d[:1])]
    for i in range(5):
        for change in changes:
            leaves, h = norm()
            change(leaves[i])
            # a gradient that no longer fits its leaf may be refused before
            with pytest.raises(RuntimeError):
                torch.autograd.grad(h.sum(), leaves[4 if i != 4 else 3])
        leaves, h = norm()
        size = leaves[i].untyped_storage().size()
        leaves[i].untyped_storage().resize_(size // 2)
        with pytest.raises(RuntimeError, match="no values of its own"):
            torch.autograd.grad(h.sum(), leaves[4 if i != 4 else 3])
    # the same values in another place are as good
    leaves, h = norm()
    want = torch.autograd.grad(h.sum(), leaves[2:], retain_graph=True)
    for t in leaves:
        t.data = t.data.clone()
    got = torch.autograd.grad(h.sum(), leaves[2:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for change in changes[:2]:
        w = torch.randn(9, 40, device="cuda", requires_grad=True)
        tok = torch.tensor([3, 1, 3], device="cuda")
        y = ops.embedding(w, tok)
        tok.data = tok.to(torch.int32) if change is changes[0] else tok.cpu()
        with pytest.raises(RuntimeError, match="kept tensor has become"):
            torch.autograd.grad(y.sum(), w)
