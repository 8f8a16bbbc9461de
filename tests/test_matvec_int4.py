"""Products with 4-bit weights (ops.matvec_int4, quantize_int4) against the definition in float64.

Tolerance of an output: the matrix cores and the group sums add in float32.  With u = 2^-24 and S = sum |x| (16 + 16) s
over the row (every term that is added: 16 + q <= 31, 16 + z <= 31), each of a term's additions rounds a partial sum of at
most S: k / 32 products of 32 terms, their groups and 8 partial sums, so at most (k / 32 + 32 + 16) u S by the worst case of
every rounding having one sign; the result is rounded once (eps / 2)."""
import pytest
import torch

from veles.simd_amd import _lib, ops
from veles.simd_amd.utils import CapturedCall

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def _inputs(m, n, k, group, dtype, dev, zeros=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    x = torch.randn(m, k, generator=g).to(dtype).to(dev)
    q = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.uint8).to(dev)
    s = ((torch.rand(n, groups, generator=g) + 0.5) * 0.02).to(dtype).to(dev)
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8).to(dev) if zeros else None
    return x, q, s, z


def _weight(q, s, z, k, group):
    w = torch.zeros(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=q.device)
    w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
    at = torch.arange(k, device=q.device) // group
    return (w[:, :k] - (8.0 if z is None else z[:, at].double())) * s[:, at].double()


def _check(y, x, q, s, z, group):
    k = x.shape[-1]
    xd = x.detach().double().reshape(-1, k)
    ref = xd @ _weight(q, s, z, k, group).t()
    at = torch.arange(k, device=x.device) // group
    size = xd.abs() @ (32.0 * s.double()[:, at]).t()
    tol = (k / 32 + 48) * U * size
    tol = tol + torch.finfo(y.dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal
    got = y.double().reshape(ref.shape)
    assert ((got - ref).abs() <= tol).all(), ((got - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128, 384])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 128), (2, 17, 127), (4, 33, 130), (5, 70, 257), (8, 64, 1024),
                                   (9, 15, 96), (16, 100, 1500), (17, 31, 640), (40, 20, 33)])
def test_values(dev, dtype, group, m, n, k):
    for zeros in (True, False):
        x, q, s, z = _inputs(m, n, k, group, dtype, dev, zeros, seed=m + n + k)
        y = ops.matvec_int4(x, q, s, z, group)
        assert y.dtype == dtype and y.shape == (m, n)
        _check(y, x, q, s, z, group)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group", [(1, 4097, 4100, 128), (3, 1001, 1500, 32), (7, 8200, 512, 64), (16, 9000, 1030, 32),
                                         (12, 8193, 384, 128), (2, 40, 17000, 32), (9, 33, 20001, 64), (4, 17, 18432, 256),
                                         (3, 13700, 4500, 64), (16, 13700, 4224, 32), (5, 27300, 5000, 128),
                                         (16, 27205, 270, 32), (1, 27200, 9000, 384), (33, 8200, 1100, 128)])
def test_larger(m, n, k, group):
    """Every shape of workgroup, waves with more steps than they keep scales for, a last group that ends early."""
    x, q, s, z = _inputs(m, n, k, group, torch.bfloat16, "cuda")
    _check(ops.matvec_int4(x, q, s, z, group), x, q, s, z, group)


@pytest.mark.parametrize("dev", DEVICES)
def test_shapes_strides_and_alignment(dev):
    """Leading dimensions, a row slice of wider weights, odd offsets of x and of the weight rows."""
    x, q, s, z = _inputs(6, 40, 300, 64, torch.bfloat16, dev)
    ref = ops.matvec_int4(x, q, s, z, 64)
    assert torch.equal(ops.matvec_int4(x.view(2, 3, 300), q, s, z, 64), ref.view(2, 3, 40))
    assert torch.equal(ops.matvec_int4(x[0], q, s, z, 64), ref[0])
    wide = torch.zeros(40, 157, dtype=torch.uint8, device=dev)
    wide[:, 3:153] = q
    assert torch.equal(ops.matvec_int4(x, wide[:, 3:153], s, z, 64), ref)
    xw = torch.full((6, 305), float("nan"), dtype=torch.bfloat16, device=dev)
    xw[:, 1:301] = x
    assert torch.equal(ops.matvec_int4(xw[:, 1:301], q, s, z, 64), ref)
    assert torch.equal(ops.matvec_int4(x.t().contiguous().t(), q, s, z, 64), ref)
    assert torch.equal(ops.matvec_int4(x, q, s.t().contiguous().t(), z.t().contiguous().t(), 64), ref)
    one = ops.matvec_int4(x[:1].expand(6, 300), q, s, z, 64)
    assert torch.equal(one, ref[:1].expand(6, 40))
    windows = x.flatten()[:350].as_strided((6, 300), (10, 1))   # rows that overlap
    assert torch.equal(ops.matvec_int4(windows, q, s, z, 64), ops.matvec_int4(windows.contiguous(), q, s, z, 64))


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_do_not_depend_on_their_neighbours(dev):
    """Row 0's bits are the same whatever the other rows hold, NaN among it."""
    x, q, s, z = _inputs(16, 64, 512, 128, torch.float16, dev)
    ref = ops.matvec_int4(x, q, s, z)
    x2 = x.clone()
    x2[1:] = float("nan")
    got = ops.matvec_int4(x2, q, s, z)
    assert torch.equal(got[0], ref[0]) and torch.isnan(got[1:]).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("m,n,k", [(0, 4, 32), (3, 0, 32), (3, 4, 0)])
def test_empty(dev, m, n, k):
    x, q, s, z = _inputs(m, n, k, 32, torch.bfloat16, dev)
    y = ops.matvec_int4(x, q, s, z, 32)
    assert y.shape == (m, n) and (y == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("k", [64, 301])
def test_quantize(dev, symmetric, k):
    """Every weight is within half a step of what is kept (a step more where a rounded scale or zero point clips it)."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(7, k, generator=g).to(dev)
    w[2] = 0.0
    w[3] = w[3].abs() + 1
    q, s, z = ops.quantize_int4(w, 64, symmetric)
    assert q.shape == (7, (k + 1) // 2) and s.dtype == torch.bfloat16 and (z is None) == symmetric
    kept = _weight(q, s, z, k, 64).cpu()
    step = s.double().cpu()[:, torch.arange(k) // 64]
    off = (kept - w.double().cpu()).abs()
    # bf16 rounds the step by up to 2^-8 of it: 15 steps (7) end up to 15 / 256 of a step short
    assert (off <= step * (1.0 + 15 / 256) + 1e-12).all() and (off <= 0.5001 * step).double().mean() > 0.9
    assert (kept[2] == 0).all()
    x = torch.randn(2, k, generator=g).bfloat16().to(dev)
    _check(ops.matvec_int4(x, q, s, z, 64), x, q, s, z, 64)


@pytest.mark.gpu
def test_weight_past_32_bit_offsets():
    """The last rows of 4.3 GB of weights."""
    n, k = (1 << 20) + 40, 8192
    gen = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(2, k, device="cuda", generator=gen).bfloat16()
    q = torch.randint(0, 256, (n, k // 2), device="cuda", dtype=torch.uint8, generator=gen)
    s = (torch.rand(n, k // 128, device="cuda", generator=gen) * 0.02).bfloat16()
    y = ops.matvec_int4(x, q, s)
    _check(y[:, -100:], x, q[-100:], s[-100:], None, 128)


@pytest.mark.gpu
def test_more_rows_than_one_grid():
    """16 x 65535 rows fill a grid dimension; the rows behind them get the bits of a small call."""
    m = 16 * 65535 + 3
    x, q, s, z = _inputs(1, 20, 64, 32, torch.bfloat16, "cuda")
    x = torch.randn(m, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).bfloat16()
    y = ops.matvec_int4(x, q, s, z, 32)
    for at in (0, 16 * 65535 - 1, 16 * 65535, m - 1):
        assert torch.equal(y[at:at + 1], ops.matvec_int4(x[at:at + 1], q, s, z, 32))


@pytest.mark.gpu
def test_stream_and_capture():
    x, q, s, z = _inputs(2, 512, 2048, 128, torch.bfloat16, "cuda")
    cap = CapturedCall(lambda v: ops.matvec_int4(v, q, s, z), x)
    for seed in range(3):
        x2 = _inputs(2, 512, 2048, 128, torch.bfloat16, "cuda", seed=seed + 5)[0]
        got = cap(x2).clone()
        assert torch.equal(got, ops.matvec_int4(x2, q, s, z))
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.matvec_int4(x, q, s, z)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, ops.matvec_int4(x, q, s, z))


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, q, s, z = _inputs(2, 8, 64, 32, torch.bfloat16, dev)
    bad = [(TypeError, (x.float(), q, s, z, 32)), (TypeError, (x.half(), q, s, z, 32)), (ValueError, (x, q.int(), s, z, 32)),
           (ValueError, (x, q, s, z, 48)), (ValueError, (x, q, s, z, 0)), (ValueError, (x, q, s, z, -128)),
           (ValueError, (x[:, :60], q, s, z, 32)), (ValueError, (x, q, s[:, :1], z, 32)), (ValueError, (x, q, s, z.int(), 32)),
           (ValueError, (x, q, s, z[:4], 32)), (ValueError, (x, q.t().contiguous().t(), s, z, 32)),
           (ValueError, (x, q[0], s, z, 32)), (ValueError, (x, q[:, :1].expand(8, 32), s, z, 32)),
           (ValueError, (x, q[:1].expand(8, 32), s, z, 32)),
           (ValueError, (x, torch.zeros(1, 64, dtype=torch.uint8, device=dev)[:, ::2], s[:1], z[:1], 32))]
    for err, args in bad:
        with pytest.raises(err):
            ops.matvec_int4(*args)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.matvec_int4(x.clone().requires_grad_(), q, s, z, 32)
    if dev == "cuda":
        with pytest.raises(ValueError, match="is on"):
            ops.matvec_int4(x, q.cpu(), s, z, 32)
    for err, args in [(ValueError, (torch.zeros(4), 32)), (ValueError, (torch.zeros(2, 4), 33)),
                      (TypeError, (torch.zeros(2, 4), 32, False, torch.float32)),
                      (ValueError, (torch.full((2, 4), float("inf")), 32))]:
        with pytest.raises(err):
            ops.quantize_int4(*args)


def test_native_refusals():
    lib = _lib.lib()
    p = torch.zeros(8).data_ptr()

    def call(dtype=5, x=p, ldx=64, ldq=32, group=32, m=1, n=1, k=64):
        return lib.vs_matvec_int4(dtype, x, ldx, p, ldq, p, None, group, m, n, k, p, None)
    for kw in (dict(dtype=0), dict(group=48), dict(group=0), dict(m=-1), dict(n=-1), dict(k=-1), dict(x=None),
               dict(m=2, ldx=63), dict(n=2, ldq=31), dict(n=1 << 40), dict(k=1 << 40), dict(m=1 << 40)):
        assert call(**kw) == 1 and b"matvec_int4" in lib.vs_last_error()


@pytest.mark.parametrize("dev", DEVICES)
def test_opcheck(dev):
    x, q, s, z = _inputs(2, 8, 64, 32, torch.bfloat16, dev)
    for args in ((x, q, s, z, 32), (x, q, s, None, 32)):
        torch.library.opcheck(torch.ops.veles.matvec_int4.default, args)


def _check_offsets(y, x, q, s, z, group):
    """The bound that holds for any weights: every rounding is of a partial sum of |x| (16 + q) s or |x| (16 + z) s."""
    k = x.shape[-1]
    xd, at = x.detach().double(), torch.arange(k, device=x.device) // group
    nibbles = torch.stack([q & 15, q >> 4], -1).flatten(1)[:, :k].double()
    zero = 8.0 if z is None else z.double()[:, at]
    scale = s.double()[:, at]
    ref = xd @ ((nibbles - zero) * scale).t()
    tol = (k / 32 + 48) * U * (xd.abs() @ ((32 + nibbles + zero) * scale).t())
    tol = tol + torch.finfo(y.dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal
    assert ((y.double() - ref).abs() <= tol).all(), ((y.double() - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,group", [(1, 40, 256, 128), (3, 33, 301, 32), (16, 64, 1030, 64), (20, 17, 640, 384)])
@pytest.mark.parametrize("kind", ["zero", "near", "far"])
def test_weights_at_and_far_from_their_zero_point(dev, dtype, m, n, k, group, kind):
    """Weights that are all 0, or one step from it, and zero points up to 255."""
    x, q, s, z = _inputs(m, n, k, group, dtype, dev, seed=21)
    if kind == "far":
        z = torch.randint(0, 256, z.shape, generator=torch.Generator().manual_seed(22), dtype=torch.uint8).to(dev)
    else:
        at = torch.arange(2 * q.shape[1], device=dev).clamp(max=k - 1) // group
        nibbles = z[:, at]
        if kind == "near":
            step = torch.randint(-1, 2, nibbles.shape, generator=torch.Generator().manual_seed(23)).to(dev)
            nibbles = (nibbles.int() + step).clamp(0, 15).to(torch.uint8)
        q = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)
    _check_offsets(ops.matvec_int4(x, q, s, z, group), x, q, s, z, group)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("most", [1e37, 1.6e38])
def test_large_finite_values(dev, most):
    """Values up to the limit that the documentation names: 2 sum |x| of a group of 128 just below 3.4e38."""
    x, q, s, z = _inputs(4, 50, 512, 128, torch.bfloat16, dev, seed=24)
    x = (x.double() / x.double().abs().view(4, 4, 128).sum(-1).max() * most).bfloat16()
    y = ops.matvec_int4(x, q, s, z, 128)
    assert torch.isfinite(y).all()
    _check_offsets(y, x, q, s, z, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(1001, 1500), (5000, 600), (9001, 520), (20000, 300), (27000, 260)])
def test_a_row_has_the_same_bits_in_every_batch(n, k):
    """Every shape of workgroup: a row alone, among 16, and among more than 16 rows."""
    x, q, s, z = _inputs(37, n, k, 64, torch.bfloat16, "cuda", seed=25)
    whole = ops.matvec_int4(x, q, s, z, 64)
    _check(whole, x, q, s, z, 64)
    for rows in (slice(0, 1), slice(3, 7), slice(5, 21), slice(36, 37)):
        assert torch.equal(ops.matvec_int4(x[rows], q, s, z, 64), whole[rows])
