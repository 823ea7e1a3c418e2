"""Wrong calls of the training-step operators are refused before anything
runs, the same way with and without a GPU."""

import pytest
import torch

from baguanet import ops


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


TOK = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("call,what", [
    (lambda: ops.embedding(_bf(4), TOK), r"weight must be \[vocab, dim\]"),
    (lambda: ops.embedding(torch.zeros(4, 8, dtype=torch.float64), TOK),
     "weight must be float32, bfloat16 or float16"),
    (lambda: ops.embedding(_bf(4, 8), TOK.float()), "int64 or int32"),
    (lambda: ops.embedding(_bf(4, 8), TOK, padding_idx=4), "padding_idx 4"),
    (lambda: ops.embedding(_bf(4, 8), TOK, padding_idx=-5), "padding_idx -5"),
    (lambda: ops.embedding(_bf(4, 8), TOK, out_dtype=torch.int32),
     "out_dtype"),
    (lambda: ops.embedding(_bf(4, 8), TOK), "weight must be on the GPU"),
    (lambda: ops.rms_norm(torch.zeros((), dtype=torch.float32)), "scalar"),
    (lambda: ops.rms_norm(torch.zeros(4, 8, dtype=torch.int32)), "x must be"),
    (lambda: ops.rms_norm(_bf(4, 8), _bf(9)), r"weight must be \[8\]"),
    (lambda: ops.rms_norm(_bf(4, 8), torch.zeros(8, dtype=torch.float16)),
     "float32 or of x's type"),
    (lambda: ops.rms_norm(_bf(2, 16385)), "at most 16384 columns"),
    (lambda: ops.rms_norm(_bf(4, 8), eps=-1.0), "eps"),
    (lambda: ops.rms_norm(_bf(4, 8)), "x must be on the GPU"),
    (lambda: ops.rms_norm(torch._neg_view(_bf(4, 8))), "resolve_neg"),
    (lambda: ops.embedding(torch._neg_view(_bf(4, 8)), TOK), "resolve_neg"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), _bf(4, 9)), "x's shape"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), torch.zeros(4, 8)),
     "x's type"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), _bf(4, 8), gate=_bf(3, 8)),
     "cannot be broadcast"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), _bf(4, 8),
                                     gate=_bf(1, 4, 8)),
     "cannot be broadcast"),
    (lambda: ops.gated_residual_norm(
        _bf(4, 8), _bf(4, 8), gate=torch.zeros(8, dtype=torch.float16)),
     "gate must be float32 or of x's type"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), _bf(4, 8),
                                     post_weight=_bf(7)),
     r"post_weight must be \[8\]"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), _bf(4, 8),
                                     pre_weight=_bf(1, 8)),
     r"pre_weight must be \[8\]"),
    (lambda: ops.gated_residual_norm(_bf(4, 8), _bf(4, 8)),
     "x must be on the GPU"),
    (lambda: ops.act8_pack(torch.zeros(4, 8, dtype=torch.float64)),
     "x must be"),
    (lambda: ops.act8_pack(_bf(4, 8)), "x must be on the GPU"),
    (lambda: ops.linear_act8(_bf(4, 8), _bf(5, 9)), r"\[out, 8\]"),
    (lambda: ops.linear_act8(_bf(4, 8), torch.zeros(5, 8)), "x's type"),
    (lambda: ops.linear_act8(_bf(4, 8), _bf(5, 8), _bf(4)),
     r"bias must be \[5\]"),
    (lambda: ops.linear_act8(_bf(4, 8), _bf(5, 8)), "on the GPU"),
    (lambda: ops.silu_mul_act8(_bf(4, 7)), "two halves"),
    (lambda: ops.silu_mul_act8(_bf(4, 8)), "on the GPU"),
])
def test_refused(call, what):
    with pytest.raises(RuntimeError, match=what):
        call()


def _kept(rows=4, cols=40, pitch=64, groups=2, dtype=torch.bfloat16):
    return ops.Act8(torch.zeros(rows, pitch, dtype=torch.uint8),
                    torch.zeros(rows, groups, dtype=torch.uint8),
                    torch.Size((rows, cols)), dtype)


@pytest.mark.parametrize("call,what", [
    (lambda: ops.act8_unpack(_kept(pitch=40)), "codes must be"),
    (lambda: ops.act8_unpack(_kept(groups=3)), "exponents must be"),
    (lambda: ops.act8_unpack(_kept(dtype=torch.int32)), "dtype must be"),
    (lambda: ops.act8_unpack(_kept()), "codes must be on the GPU"),
    (lambda: ops.act8_wgrad(_bf(5, 8), _kept()), "rows of the kept input"),
    (lambda: ops.act8_wgrad(_bf(2, 2, 8), _kept()), "rows of the kept input"),
    (lambda: ops.act8_wgrad(torch.zeros(4, 8), _kept()),
     "the kept input's type"),
    (lambda: ops.act8_wgrad(_bf(4, 8), _kept(pitch=96)), "codes must be"),
    (lambda: ops.act8_wgrad(_bf(4, 8), _kept()), "dy must be on the GPU"),
])
def test_kept_refused(call, what):
    with pytest.raises(RuntimeError, match=what):
        call()


RECORDED = [
    lambda x: ops.embedding(x, TOK),
    lambda x: ops.rms_norm(x),
    lambda x: ops.gated_residual_norm(x, x)[0],
    lambda x: ops.act8_pack(x).codes,
    lambda x: ops.act8_unpack(_kept()) + x.sum(),
    lambda x: ops.act8_wgrad(x, _kept(cols=8, pitch=32, groups=1))[0],
    lambda x: ops.linear_act8(x, x),
    lambda x: ops.silu_mul_act8(x),
]


@pytest.mark.parametrize("f", RECORDED)
def test_recording_refused(f):
    """A recording would hold the results' memory without what fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.ones(4, 8)
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        torch.jit.trace(f, x)
    for how in (dict(), dict(tracing_mode="fake"),
                dict(tracing_mode="symbolic"), dict(pre_dispatch=True)):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(f, **how)(x)
    with pytest.raises(RuntimeError, match="must"):
        f(x)  # outside it, the call is refused for what is wrong with it


def test_counting_modes_are_no_recording():
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            ops.rms_norm(torch.ones(4, 8))


class _Wrapper(torch.Tensor):
    """A tensor around another one, with no memory of its own, as those of
    torch.distributed.tensor are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(
            cls, inner.shape, dtype=inner.dtype, device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args, kwargs=None):
        raise RuntimeError("the operator looked into a wrapper")


def _zeros(*shape):
    return torch._efficientzerotensor(shape)


def _wrapped(*shape):
    return _Wrapper(torch.zeros(*shape))


def _byte(make, *shape):
    if make is _zeros:
        return torch._efficientzerotensor(shape, dtype=torch.uint8)
    return _Wrapper(torch.zeros(*shape, dtype=torch.uint8))


@pytest.mark.parametrize("make", [_zeros, _wrapped])
@pytest.mark.parametrize("call,name", [
    (lambda m, t: ops.embedding(m(4, 8), TOK), "weight"),
    (lambda m, t: ops.rms_norm(m(4, 8)), "x"),
    (lambda m, t: ops.rms_norm(t, m(8)), "weight"),
    (lambda m, t: ops.gated_residual_norm(t, m(4, 8)), "branch"),
    (lambda m, t: ops.gated_residual_norm(t, t, m(8)), "gate"),
    (lambda m, t: ops.gated_residual_norm(t, t, None, m(8)), "post_weight"),
    (lambda m, t: ops.gated_residual_norm(t, t, None, None, m(8)),
     "pre_weight"),
    (lambda m, t: ops.act8_pack(m(4, 8)), "x"),
    (lambda m, t: ops.act8_wgrad(m(4, 8), _kept(dtype=torch.float32)), "dy"),
    (lambda m, t: ops.act8_unpack(_kept()._replace(codes=_byte(m, 4, 64))),
     "codes"),
    (lambda m, t: ops.act8_unpack(_kept()._replace(exponents=_byte(m, 4, 2))),
     "exponents"),
    (lambda m, t: ops.linear_act8(m(4, 8), t), "x"),
    (lambda m, t: ops.linear_act8(t, m(5, 8)), "weight"),
    (lambda m, t: ops.linear_act8(t, t, m(4)), "bias"),
    (lambda m, t: ops.silu_mul_act8(m(4, 8)), "x"),
])
def test_tensors_without_memory_refused(make, call, name):
    with pytest.raises(RuntimeError, match=f"{name} holds no values"):
        call(make, torch.zeros(4, 8))


def test_tokens_without_memory_or_negated_refused():
    for tok, what in (
            (torch._efficientzerotensor((3,), dtype=torch.int64),
             "tokens holds no values"),
            (_Wrapper(TOK), "tokens holds no values"),
            (torch._neg_view(TOK), "resolve_neg")):
        with pytest.raises(RuntimeError, match=what):
            ops.embedding(_bf(4, 8), tok)


@pytest.mark.parametrize("shape", [(2 ** 31, 0), (2 ** 16, 2 ** 15, 0),
                                   (2 ** 33, 2 ** 31, 0)])
def test_unpack_of_too_many_rows_refused(shape):
    """As act8_pack: the kernels count rows in 32 bits."""
    rows = 1
    for n in shape[:-1]:
        rows = rows * n % 2 ** 64
    none = torch.empty(rows, 0, dtype=torch.uint8)
    kept = ops.Act8(none, none, torch.Size(shape), torch.float32)
    with pytest.raises(RuntimeError, match=r"at most 2\^30 rows"):
        ops.act8_unpack(kept)


def test_unpack_of_no_shape_refused():
    for shape in ((4, -40), (-4, 40), (0, -1)):
        with pytest.raises(RuntimeError, match="a shape of"):
            ops.act8_unpack(_kept()._replace(shape=shape))
    with pytest.raises(RuntimeError, match="codes must be on the GPU"):
        none = torch.empty(0, 64, dtype=torch.uint8)
        ops.act8_unpack(ops.Act8(none, none[:, :2], (2 ** 29, 0, 8, 40),
                                 torch.float32))


@pytest.mark.parametrize("rows,cols", [(2 ** 20, 2 ** 15), (2 ** 30, 2 ** 32),
                                       (7, 2 ** 33)])
def test_table_too_large_for_its_gradient_refused(rows, cols):
    """Before the lookup, not in the backward pass that cannot do it."""
    one = torch.zeros(1, 1)
    table = one.expand(rows, cols).requires_grad_()
    with pytest.raises(RuntimeError, match=r"fewer than 2\^35"):
        ops.embedding(table, TOK)
    for call in (lambda: ops.embedding(table.detach(), TOK),
                 lambda: ops.embedding(one.expand(2 ** 20, 2 ** 15 - 1)
                                       .requires_grad_(), TOK)):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            call()


def test_freed_storage_refused():
    for size in (0, 4 * 31):
        x = torch.zeros(4, 8)
        x.untyped_storage().resize_(size)
        with pytest.raises(RuntimeError, match="x holds no values"):
            ops.rms_norm(x)
    x = torch.zeros(64)
    for view in (x[32:].view(4, 8), x.as_strided((4, 8), (16, 1), 8),
                 x[:8].expand(4, 8), x[63:].expand(4, 8)):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            ops.rms_norm(view)
    view = x[32:].view(4, 8)
    x.untyped_storage().resize_(4 * 63)
    with pytest.raises(RuntimeError, match="x holds no values"):
        ops.rms_norm(view)
