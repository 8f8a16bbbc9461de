"""The operators of sequence models where something stands between the caller and the kernels: tracers, compilers, tensors
without data, forward-mode derivatives."""
import pytest
import torch

from veles.simd_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(dev, seed=0):
    """Every operator as (name, function, inputs); functions take the inputs alone."""
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g).to(dev)
    w = torch.randn(24, 64, generator=g)
    q, s, z = (v.to(dev) for v in ops.quantize_int4(w, 32))
    return [
        ("gated_recurrence", lambda x, a, h: ops.gated_recurrence(x, a, h), (r(2, 37, 6), r(2, 37, 6), r(2, 6))),
        ("gated_recurrence_step", lambda x, a, h: ops.gated_recurrence_step(x, a, h.clone()), (r(3, 6), r(3, 6), r(3, 6))),
        ("gated_linear", lambda x, g, u: ops.gated_linear(x, g, u, "gelu"),
         (r(5, 40).bfloat16(), r(16, 40).bfloat16(), r(16, 40).bfloat16())),
        ("matvec_int4", lambda x: ops.matvec_int4(x, q, s, z, 32), (r(3, 64).bfloat16(),)),
    ]


NAMES = [c[0] for c in _calls("cpu")]


def _flat(out):
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", NAMES)
def test_traced_calls_keep_the_operator(dev, name):
    """torch.jit.trace records the op itself, so the traced function computes other inputs' results."""
    _, fn, args = next(c for c in _calls(dev) if c[0] == name)
    _, other_fn, other = next(c for c in _calls(dev, 7) if c[0] == name)
    traced = torch.jit.trace(fn, args, check_trace=False)
    assert f"veles::{name}" in str(traced.graph)
    for a, b in zip(_flat(traced(*other)), _flat(fn(*other))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
def test_traced_training_calls_keep_the_operator(dev):
    for name, fn, args in _calls(dev):
        if name not in ("gated_recurrence", "gated_linear"):
            continue
        leaves = [a.requires_grad_() for a in args]
        traced = torch.jit.trace(fn, leaves, check_trace=False)
        assert f"veles::{name}" in str(traced.graph)
        a, b = (torch.autograd.grad(_flat(f(*leaves))[0].float().sum(), leaves) for f in (traced, fn))
        for u, v in zip(a, b):
            assert torch.equal(u, v)


@pytest.mark.parametrize("name", NAMES)
def test_meta_tensors(name):
    """Tensors without data give results of the right shapes and types, with gradients and without."""
    _, fn, args = next(c for c in _calls("cpu") if c[0] == name)
    want = _flat(fn(*args))
    if name == "matvec_int4":
        q, s, z = (v.to("meta") for v in ops.quantize_int4(torch.randn(24, 64), 32))
        fn = lambda x: ops.matvec_int4(x, q, s, z, 32)   # noqa: E731
    metas = [a.to("meta") for a in args]
    for leaves in (metas, [m.clone().requires_grad_() for m in metas]):
        if leaves is not metas and name in ("gated_recurrence_step", "matvec_int4"):
            continue
        got = _flat(fn(*leaves))
        for a, b in zip(got, want):
            assert a.is_meta and a.shape == b.shape and a.dtype == b.dtype
    if name in ("gated_recurrence", "gated_linear"):
        for grad, leaf in zip(torch.autograd.grad(got[0].sum(), leaves), leaves):
            assert grad.is_meta and grad.shape == leaf.shape and grad.dtype == leaf.dtype
