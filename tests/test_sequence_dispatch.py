"""The operators of sequence models where something stands between the caller and the kernels: tracers, compilers, tensors
without data, forward-mode derivatives."""
import pytest
import sympy
import torch
import torch._dynamo.testing
from torch._dynamo.source import ConstantSource
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv

from veles.simd_amd import _lib, ops
from veles.simd_amd.ops.sequence import _tiles

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


def test_tile_count_is_the_librarys():
    lib = _lib.lib()
    for t in [*range(0, 700), 4095, 4096, 4097, 65536, (1 << 29) - 1, 1 << 29]:
        assert _tiles(t) == lib.vs_gated_recurrence_tiles(t)


def _symbolic_cases(length):
    """Operators on GPU tensors of one symbolic dimension, as a compiler sees them; no GPU is needed."""
    def e(*s, dtype=torch.bfloat16):
        return torch.empty(*s, dtype=dtype, device="cuda")
    op = torch.ops.veles
    x = e(2, length, 6)
    yield "recurrence", op.gated_recurrence(x, x, None, None, True)
    yield "recurrence backward", op.gated_recurrence_backward(x, x, None, e(2, (length + 127) // 128, 6, dtype=torch.float32),
                                                              x, None)
    yield "linear", op.gated_linear(e(length, 40), e(16, 40), e(16, 40), "silu", True)
    yield "linear, batched", op.gated_linear(e(2, length, 40), e(16, 40), e(16, 40), "silu", False)
    yield "linear backward", op.gated_linear_backward(e(length, 40), e(16, 40), e(16, 40),
                                                      e(length, 16, 2, dtype=torch.float32), e(length, 16), "silu", True, True)
    yield "4 bits", (op.matvec_int4(e(length, 64), e(24, 32, dtype=torch.uint8), e(24, 2), None, 32),)


@pytest.mark.parametrize("known", [True, False])
def test_symbolic_lengths_stay_symbolic(known):
    """A compiler that traces a call once for all lengths: nothing fixes the length, or asks for it where it is not known."""
    env = ShapeEnv()
    with FakeTensorMode(shape_env=env):
        if known:
            symbol = env.create_symbol(70, ConstantSource("length"), dynamic_dim=DimDynamic.DYNAMIC)
            length = env.create_symintnode(symbol, hint=70)
        else:
            length = env.create_unbacked_symint()
            torch._check(length > 1)
        for name, out in _symbolic_cases(length):
            assert any(not isinstance(n, int) for o in out for n in o.shape), name
    assert not any(isinstance(g.expr, sympy.Eq) for g in env.guards), env.guards


@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_other_lengths_do_not_compile_anew(train):
    """With gradients there are two compilations: the compiler treats dimensions of one element, here a single tile of saved
    states (up to 128 steps), apart from larger ones."""
    def block(v, a, wg, wu, q, s):
        return ops.matvec_int4(ops.gated_linear(ops.gated_recurrence(v, a)[0], wg, wu), q, s, None, 32) if not train else \
            ops.gated_linear(ops.gated_recurrence(v, a)[0], wg, wu)
    g = torch.Generator().manual_seed(0)
    wg, wu = (torch.randn(96, 64, generator=g).bfloat16().cuda().requires_grad_(train) for _ in range(2))
    q, s, _ = ops.quantize_int4(torch.randn(24, 96, generator=g).cuda(), 32, True)
    torch._dynamo.reset()
    counter = torch._dynamo.testing.CompileCounterWithBackend("aot_eager")
    fn = torch.compile(block, backend=counter, dynamic=True)
    for t in (70, 33, 130, 500, 257):
        v, a = (torch.randn(2, t, 64, generator=g).bfloat16().cuda().requires_grad_(train) for _ in range(2))
        got, want = (f(v, a, wg, wu, q, s) for f in (fn, block))
        assert torch.equal(got, want)
        if train:
            for x, y in zip(*(torch.autograd.grad(o.float().sum(), (v, a, wg, wu)) for o in (got, want))):
                assert torch.equal(x, y)
    assert counter.frame_count == (2 if train else 1)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_right_or_refused(dev, name):
    """A tangent is never dropped: the CPU definitions carry it, the kernels and torch.func refuse it."""
    _, fn, args = next(c for c in _calls(dev) if c[0] == name)
    tangent = torch.ones_like(args[0])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[0], tangent)
        if dev == "cpu":
            got = torch.autograd.forward_ad.unpack_dual(_flat(fn(dual, *args[1:]))[0]).tangent
            # a hundredth of a step each way: the second difference and the results' roundings are below 5 % of the largest
            up, down = (_flat(fn(args[0] + s * 0.01 * tangent, *args[1:]))[0].double() for s in (1, -1))
            if args[0].dtype == torch.float32:
                assert ((up - down) / 0.02 - got).abs().max() <= 0.05 * got.abs().max()
            assert got is not None and got.abs().max() > 0
        else:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(dual, *args[1:])
        fn(*args)    # no tangent among the inputs
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: fn(v, *args[1:]), (args[0],), (tangent,))


@pytest.mark.parametrize("name", NAMES)
def test_default_device_does_not_matter(name):
    """CPU tensors are computed on the CPU whatever device new tensors would get."""
    _, fn, args = next(c for c in _calls("cpu") if c[0] == name)
    want = _flat(fn(*args))
    with torch.device("meta"):
        got = _flat(fn(*args))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    if name in ("gated_recurrence", "gated_linear"):
        leaves = [a.requires_grad_() for a in args]
        up = torch.ones_like(want[0])
        want = torch.autograd.grad(_flat(fn(*leaves))[0], leaves, up)
        with torch.device("meta"):
            got = torch.autograd.grad(_flat(fn(*leaves))[0], leaves, up)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
