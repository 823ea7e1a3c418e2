"""baguanet.ops — HIP (gfx950) kernels exposed to torch.

The extension is compiled IN-TREE (build/torch_ext) so the built .so
travels with the repo snapshot.  On a GPU machine a missing/failed
extension raises — the HIP path must never silently fall back to eager.
"""

from __future__ import annotations

import contextlib
import fcntl
import hashlib
import importlib.util
import os
import sys
from pathlib import Path
from typing import NamedTuple

import torch

from .. import REPO_ROOT

_C = None
_ERR: Exception | None = None

_ARCH = "PYTORCH_ROCM_ARCH"
_CXX_FLAGS = ["-O3"]
# packed fp32 instructions stay out of every kernel: some of their forms have
# given wrong results on this hardware
_HIP_FLAGS = ["-O3", "-Xclang", "-target-feature", "-Xclang",
              "-packed-fp32-ops"]


def _sources() -> list[Path]:
    src = REPO_ROOT / "csrc"
    return [
        src / "torch" / "ops.cc",
        src / "torch" / "train_ops.cc",
        src / "hip" / "pack_kernels.hip",
        src / "hip" / "multi_tensor.hip",
        src / "hip" / "embedding.hip",
        src / "hip" / "residual_norm.hip",
        src / "hip" / "act8.hip",
        src / "hip" / "act8_wgrad.hip",
    ]


def _import_built(lib: Path):
    spec = importlib.util.spec_from_file_location("baguanet_C", lib)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _wanted(sources: list[Path]) -> str:
    """What the built extension depends on, as a hash: its sources, compiler
    flags and architecture, and the torch and Python that load it."""
    h = hashlib.sha256()
    for part in (_CXX_FLAGS, _HIP_FLAGS, os.environ.get(_ARCH, "gfx950"),
                 torch.__version__, torch.version.git_version,
                 torch.version.hip, sys.version_info[:2]):
        h.update(repr(part).encode() + b"\0")
    headers = sorted((REPO_ROOT / "csrc" / "hip").glob("*.h"))
    for p in sources + headers:
        h.update(p.name.encode() + b"\0" + p.read_bytes() + b"\0")
    return h.hexdigest()


@contextlib.contextmanager
def _locked(build_dir: Path, how: int):
    """The build directory's lock: shared to load, exclusive to build.  It ends
    with its process.  A directory that cannot be written to needs none, and a
    file system may have none."""
    with contextlib.ExitStack() as stack:
        with contextlib.suppress(OSError):
            build_dir.mkdir(parents=True, exist_ok=True)
            file = stack.enter_context(open(build_dir / "baguanet_C.lock", "a"))
            fcntl.flock(file, how)
        yield


def build_extension(verbose: bool = False, force: bool = False):
    """Load the extension from its in-tree build dir, compiled first if there
    is none built from these sources with these flags, or always with
    ``force``."""
    global _C, _ERR
    if _C is not None and not force:
        return _C
    build_dir = REPO_ROOT / "build" / "torch_ext"
    lib = build_dir / "baguanet_C.so"
    # written after a build: a library without it may be half written
    stamp = build_dir / "baguanet_C.stamp"
    try:
        sources = _sources()
        wanted = _wanted(sources)

        def built() -> bool:
            return (lib.exists() and stamp.exists()
                    and stamp.read_text() == wanted)

        if not force:
            with _locked(build_dir, fcntl.LOCK_SH):
                if built():
                    _C = _import_built(lib)
                    return _C
        with _locked(build_dir, fcntl.LOCK_EX):
            if not force and built():  # by another process, meanwhile
                _C = _import_built(lib)
                return _C
            stamp.unlink(missing_ok=True)
            module = _compile(build_dir, sources, verbose, force)
            stamp.write_text(wanted)
            _C = module
    except Exception as e:  # pragma: no cover
        _ERR = e
        raise
    return _C


def _compile(build_dir: Path, sources: list[Path], verbose: bool,
             force: bool):
    from torch.utils import cpp_extension

    os.environ.setdefault(_ARCH, "gfx950")
    if force:
        for built in build_dir.glob("*.o"):
            built.unlink()
    return cpp_extension.load(
        name="baguanet_C",
        sources=[str(p) for p in sources],
        build_directory=str(build_dir),
        extra_cflags=_CXX_FLAGS,
        extra_cuda_cflags=_HIP_FLAGS,
        verbose=verbose,
    )


def _load():
    global _C
    if _C is None:
        build_extension()
    return _C


def copy_bytes(dst: torch.Tensor, src: torch.Tensor) -> None:
    _load().copy_bytes(dst, src)


def multi_pack(flat: torch.Tensor, tensors: list[torch.Tensor]) -> None:
    _load().multi_pack(flat, tensors)


def multi_unpack(flat: torch.Tensor, tensors: list[torch.Tensor]) -> None:
    _load().multi_unpack(flat, tensors)


def fused_sgd(params, grads, momenta, lr, momentum=0.0, weight_decay=0.0,
              nesterov=False) -> None:
    _load().fused_sgd(params, grads, momenta, lr, momentum, weight_decay,
                      nesterov)


# ---------------------------------------------------------------------------
# Training-step operators.  Each takes float32, bfloat16 or float16 tensors on
# the GPU, runs on the current stream, sums in float32 and rounds once; each
# is differentiable once, with the same result in every run.  Calls may be
# captured into a graph; a backward pass only while no eager graph of the same
# leaves is alive, as with torch's own operators.  A tracer (torch.jit.trace,
# make_fx) cannot record them and is refused; torch.compile calls them as they
# are.


def embedding(weight: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
              padding_idx: int | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * weight[tokens]``, of the shape ``[*tokens.shape, dim]``.

    ``weight`` is ``[vocab, dim]``, ``tokens`` int64 or int32 of any shape;
    the result has ``out_dtype`` (default: the weight's type).  The weight's
    gradient is dense, in the weight's type: each row is the sum over the
    token's places, in their order, times ``scale``.  The row of
    ``padding_idx`` takes no gradient.  A token outside the table gives a row
    of NaN and no gradient.
    """
    return _load().embedding(weight, tokens, scale, padding_idx, out_dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
             eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x ** 2) + eps) * weight`` over the last dimension.

    ``weight`` is ``[dim]``, float32 or of x's type; ``dim`` is at most
    16384.  This is the norm before a network's first block; those between
    blocks are part of :func:`gated_residual_norm`.
    """
    return _load().rms_norm(x, weight, eps)


def gated_residual_norm(x: torch.Tensor, branch: torch.Tensor,
                        gate: torch.Tensor | None = None,
                        post_weight: torch.Tensor | None = None,
                        pre_weight: torch.Tensor | None = None,
                        residual_scale: float = 1.0,
                        branch_scale: float = 1.0, eps: float = 1e-6,
                        ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The seam between two blocks of a network, in one pass::

        u = rms_norm(branch, post_weight)          (branch, without a weight)
        y = residual_scale * x + branch_scale * gate * u
        h = rms_norm(y, pre_weight)                (None, without a weight)

    Returns ``(y, h)``: the residual stream and the next block's input.
    ``x`` and ``branch`` have one shape and type, with at most 16384 columns.
    ``gate`` may be anything that broadcasts to x: ``[dim]`` for each column,
    ``[batch, 1, dim]`` for each sequence's columns, ``[batch, length, 1]``
    for each row, or one value for each element.  It and the weights are
    float32 or of x's type, and all of them take gradients.
    """
    return _load().gated_residual_norm(x, branch, gate, post_weight,
                                       pre_weight, residual_scale,
                                       branch_scale, eps)


class Act8(NamedTuple):
    """An activation kept in 8 bits (see :func:`act8_pack`)."""

    codes: torch.Tensor
    exponents: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype


def act8_pack(x: torch.Tensor) -> Act8:
    """An 8-bit copy of ``x``, to keep from the forward to the backward pass.

    Groups of 32 neighbours of a row share a power of two that brings the
    largest to at most 448; each value is then an e4m3 number.  A value is
    off by at most 1/16 of itself, or, if that is more, by 2**-10 / 224
    (2**-17.8) of its group's largest; float32 and bfloat16 values are off by
    up to 2**-127 whatever their group holds.  NaN and infinities are kept as
    NaN.  The copy takes 33 bytes for 32 values and no part in autograd.
    """
    codes, exponents = _load().act8_pack(x)
    return Act8(codes, exponents, x.shape, x.dtype)


def act8_unpack(kept: Act8) -> torch.Tensor:
    """The values that an 8-bit copy stands for, exact in its type."""
    return _load().act8_unpack(kept.codes, kept.exponents, list(kept.shape),
                               kept.dtype)


def act8_wgrad(dy: torch.Tensor, kept: Act8, bias: bool = True,
               ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """A linear layer's weight gradient ``dy^T x`` from the 8-bit copy of x.

    ``dy`` has the rows of ``kept`` and its type.  Returns ``(dw, db)``, with
    ``db`` the sum of dy's rows, or None without ``bias``.
    """
    return _load().act8_wgrad(dy, kept.codes, kept.exponents,
                              list(kept.shape), kept.dtype, bias)


def linear_act8(x: torch.Tensor, weight: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """``torch.nn.functional.linear`` with its input kept in 8 bits.

    The result and x's gradient are those of a linear layer; the weight's
    gradient is :func:`act8_wgrad` of the 8-bit copy, which takes the place
    of x in the memory that the graph holds.
    """
    return _load().linear_act8(x, weight, bias)


def silu_mul_act8(x: torch.Tensor) -> torch.Tensor:
    """``silu(a) * b`` for ``a, b = x.chunk(2, -1)``, kept in 8 bits.

    The result is that of x itself; its gradient is taken at the 8-bit
    copies of a and b, which are all that the graph holds.
    """
    return _load().silu_mul_act8(x)
