"""Gated linear layer (ops.gated_linear) against the definition in float64, and a block of all sequence operators.

Tolerances.  u = 2^-24, e = eps / 2 of the 16-bit type.  A product of k terms is added in float32: any order rounds partial
sums of at most S = sum |a| |b|, so it is off by at most k u S (worst case; the exact products of 16-bit numbers fit
float32).  The activation adds 8 u of itself and passes its argument's error on with a slope of at most 1.13 (gelu; silu
1.1); h is rounded once.  In the backward pass dg = dh u act'(g) is off by its inputs' errors (slopes of act' are at most
1, 1.6 for gelu is generous), 16 u of itself for the functions, and one rounding e to the 16-bit type, and so is du; the
products then carry these errors times the other operand, their own k u S, and one rounding."""
import pytest
import torch

from veles.simd_amd import _lib, ops
from veles.simd_amd.utils import CapturedCall

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24
ACTS = ["silu", "gelu", "relu", "sigmoid"]


def _inputs(m, k, f, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype).to(dev)
    wg, wu = ((torch.randn(f, k, generator=g) * max(k, 1) ** -0.5).to(dtype).to(dev) for _ in range(2))
    dh = torch.randn(m, f, generator=g).to(dtype).to(dev)
    return x, wg, wu, dh


def _act(name, g):
    """act(g) and its slope."""
    s = 1.0 / (1.0 + torch.exp(-g))
    if name == "silu":
        return g * s, s + g * s * (1 - s)
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / (2 * torch.pi) ** 0.5
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    return s, s * (1 - s)


def _oracle(x, wg, wu, dh, act):
    e = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal
    x, wg, wu, dh = (v.detach().double().cpu() for v in (x, wg, wu, dh))
    m, k = x.shape
    f = wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = k * U * (x.abs() @ wg.abs().t()), k * U * (x.abs() @ wu.abs().t())
    a, slope = _act(act, g)
    ea = 1.2 * eg + 8 * U * a.abs()
    eslope = (1.6 * eg if act != "relu" else (g.abs() <= eg).double()) + 16 * U
    h, eh = a * u, ea * u.abs() + a.abs() * eu
    dg, du = dh * u * slope, dh * a
    edg = dh.abs() * (eu * slope.abs() + u.abs() * eslope) + 4 * U * dg.abs()
    edu = dh.abs() * ea + 4 * U * du.abs()
    edg, edu = edg + e * (dg.abs() + edg) + tiny, edu + e * (du.abs() + edu) + tiny
    d, ed, w = torch.cat([dg, du], 1), torch.cat([edg, edu], 1), torch.cat([wg, wu])
    dx, edx = d @ w, ed @ w.abs() + 2 * f * U * ((d.abs() + ed) @ w.abs())
    dw, edw = d.t() @ x, ed.t() @ x.abs() + m * U * ((d.abs() + ed).t() @ x.abs())
    return dict(h=(h, eh), dx=(dx, edx), dw_gate=(dw[:f], edw[:f]), dw_up=(dw[f:], edw[f:]))


def _close(name, got, want):
    ref, bound = want
    got_d = got.detach().double().cpu().reshape(ref.shape)
    tol = bound + torch.finfo(got.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(got.dtype).smallest_normal
    bad = ~((got_d - ref).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), ((got_d - ref).abs() / tol).max().item())


def _all(x, wg, wu, dh, act, want=None):
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
    h = ops.gated_linear(*leaves, act)
    grads = torch.autograd.grad(h, leaves, dh)
    want = want or _oracle(x.reshape(-1, x.shape[-1]), wg, wu, dh.reshape(-1, dh.shape[-1]), act)
    for name, got in zip(("h", "dx", "dw_gate", "dw_up"), (h, *grads)):
        assert got.dtype == x.dtype
        _close(name, got, want[name])
    with torch.no_grad():
        assert torch.equal(ops.gated_linear(x, wg, wu, act), h)
    return (h.detach(), *grads)


SHAPES = [(1, 1, 1), (1, 64, 16), (3, 70, 33), (16, 128, 40), (17, 33, 100), (40, 200, 31), (64, 129, 65), (65, 64, 64),
          (130, 72, 200), (129, 75, 131), (300, 136, 260)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(dev, dtype, shape):
    for act in ("silu", "gelu"):
        _all(*_inputs(*shape, dtype, dev, seed=sum(shape)), act)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [5, 100])
def test_activations(dev, act, m):
    x, wg, wu, dh = _inputs(m, 64, 48, torch.bfloat16, dev, seed=2)
    _all(x * 4, wg, wu, dh, act)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4096, 200, 2100), (4100, 1000, 2056), (2100, 2048, 5000), (70, 4096, 3000),
                                   (60, 1027, 4099), (35, 1024, 17000), (20, 512, 16000), (1000, 1024, 1030)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_tiles(shape, dtype):
    """Shapes whose forward or backward products take the large tiles, ragged in every dimension."""
    _all(*_inputs(*shape, dtype, "cuda", seed=3), "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(300, 8192, 200), (70, 5003, 33), (130, 1500, 1), (66, 130, 9001), (9000, 40, 72),
                                   (9001, 513, 65), (64, 128, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sums_in_parts(shape, dtype):
    """Few outputs and a long reduction, forward, in dx or in dw: summed in parts, which changes no result between calls."""
    args = _inputs(*shape, dtype, "cuda", seed=8)
    first = _all(*args, "gelu")
    for a, b in zip(first, _all(*args, "gelu")):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,f", [(5, 2104, 1 << 20), (70, 2104, 1 << 20), ((1 << 20) + 300, 2104, 40)])
def test_operands_past_32_bit_offsets(m, k, f):
    """The last rows and features where x, the weights or the pairs have more than 2^31 elements."""
    gen = torch.Generator("cuda").manual_seed(4)
    x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16, generator=gen)
    wg, wu = (torch.randn(f, k, device="cuda", dtype=torch.bfloat16, generator=gen).mul_(k ** -0.5) for _ in range(2))
    h = ops.gated_linear(x, wg, wu)
    x, wg, wu, h = x[-64:], wg[-64:], wu[-64:], h[-64:, -64:]
    _close("h", h, _oracle(x, wg, wu, torch.zeros_like(h), "silu")["h"])


def test_workspace_sizes():
    size = _lib.lib().vs_gated_linear_workspace
    assert size(4096, 2048, 2048, 1) == 0 and size(8, 64, 64, 0) == 0
    assert size(4096, 2048, 2048, 0) >= 2 * 2048 * (4096 + 2 * 2048)
    assert 0 < size(300, 200, 8192, 1) < size(300, 200, 8192, 0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("m", [6, 90])
def test_shapes_strides_and_alignment(dev, m):
    """Leading dimensions, odd offsets, transposed storage and broadcast rows give the values of a copy."""
    x, wg, wu, dh = _inputs(m, 64, 40, torch.bfloat16, dev, seed=4)
    ref = _all(x, wg, wu, dh, "silu")
    three = _all(x.view(2, m // 2, 64), wg, wu, dh.view(2, m // 2, 40), "silu")
    for a, b in zip(three, ref):
        assert torch.equal(a.reshape(b.shape), b)

    def shifted(v, off):
        wide = torch.full((v.shape[0], v.shape[1] + 9), float("nan"), dtype=v.dtype, device=dev)
        wide[:, off:off + v.shape[1]] = v
        return wide[:, off:off + v.shape[1]]
    for change in (lambda v: shifted(v, 1), lambda v: shifted(v, 8), lambda v: v.t().contiguous().t()):
        _all(change(x), change(wg), change(wu), change(dh), "silu")
    _all(shifted(x, 8), wg, shifted(wu, 8), dh, "silu")
    _all(x, shifted(wg, 1), wu, dh, "silu")
    _all(x, wg, wu, dh.flatten()[:5 * m + 35].as_strided((m, 40), (5, 1)), "silu")   # rows that overlap
    _all(shifted(x, 3), wg, wu, dh, "silu")
    far = torch.zeros(2 * (1 << 21) + 64, dtype=torch.bfloat16, device=dev)   # rows 2^21 elements apart
    two = far.as_strided((2, 64), (1 << 21, 1)).copy_(x[:2])
    _all(two, wg, wu, dh[:2], "silu")
    _all(far.as_strided((1, 64), (1 << 22, 1)), wg, wu, dh[:1], "silu")
    one = x[:1].expand(m, 64)
    _all(one, wg, wu, dh[:, :1].expand(m, 40), "silu")
    _all(x, wg[:1].expand(40, 64), wu, dh, "silu")


@pytest.mark.parametrize("dev", DEVICES)
def test_shared_weight_and_partial_gradients(dev):
    """One tensor as both weights gets the sum of both gradients; gradients that nobody asks for are not made."""
    x, w, _, dh = _inputs(33, 64, 24, torch.bfloat16, dev, seed=5)
    want = _oracle(x, w, w, dh, "silu")
    leaf = w.detach().requires_grad_()
    h = ops.gated_linear(x, leaf, leaf)
    got, = torch.autograd.grad(h, leaf, dh)
    e = torch.finfo(w.dtype).eps
    both = (want["dw_gate"][0] + want["dw_up"][0],
            want["dw_gate"][1] + want["dw_up"][1] + e * (want["dw_gate"][0].abs() + want["dw_up"][0].abs()))
    _close("dw", got, both)
    for k in range(3):
        args = [x, w, w.clone()]
        args[k] = args[k].detach().requires_grad_()
        got, = torch.autograd.grad(ops.gated_linear(*args), args[k], dh)
        _close("part", got, want[("dx", "dw_gate", "dw_up")[k]])


@pytest.mark.parametrize("dev", DEVICES)
def test_formula_gradient_agrees_with_differences(dev):
    """Central differences of the float64 definition against the gradients (which carry 16-bit roundings)."""
    x, wg, wu, dh = _inputs(3, 5, 4, torch.float16, dev, seed=6)
    base = [v.double().cpu() for v in (x, wg, wu)]
    d = dh.double().cpu()
    for act in ("silu", "gelu", "sigmoid"):
        def loss(xv, gv, uv):
            return (_act(act, xv @ gv.t())[0] * (xv @ uv.t()) * d).sum()
        want = _oracle(x, wg, wu, dh, act)
        leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
        grads = torch.autograd.grad(ops.gated_linear(*leaves, act), leaves, dh)
        for k, name in enumerate(("dx", "dw_gate", "dw_up")):
            diff = torch.zeros_like(base[k])
            for at in range(base[k].numel()):
                vals = []
                for sign in (1, -1):
                    moved = [v.clone() for v in base]
                    moved[k].view(-1)[at] += sign * 1e-5
                    vals.append(loss(*moved))
                diff.view(-1)[at] = (vals[0] - vals[1]) / 2e-5
            _close(name, grads[k], (diff, want[name][1] + 1e-7))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("m,k,f", [(0, 8, 8), (3, 0, 8), (3, 8, 0), (100, 0, 8), (100, 8, 0)])
def test_empty(dev, m, k, f):
    x, wg, wu, dh = _inputs(m, k, f, torch.bfloat16, dev)
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
    h = ops.gated_linear(*leaves)
    assert h.shape == (m, f) and (h == 0).all()
    for g, leaf in zip(torch.autograd.grad(h, leaves, dh), leaves):
        assert g.shape == leaf.shape and (g == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 200])
def test_not_finite_rows_stay_in_their_rows(m):
    x, wg, wu, dh = _inputs(m, 72, 64, torch.bfloat16, "cuda", seed=7)
    ref = ops.gated_linear(x, wg, wu)
    x2 = x.clone()
    x2[1] = float("nan")
    x2[2, 5] = float("inf")
    got = ops.gated_linear(x2, wg, wu)
    assert torch.isnan(ops.gated_linear(x2, wg, wu, "relu")[1]).all()
    keep = torch.ones(m, dtype=torch.bool)
    keep[1:3] = False
    assert torch.equal(got[keep], ref[keep]) and torch.isnan(got[1]).all() and not torch.isfinite(got[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(8, 96), (200, 96), (200, 75), (200, 4800), (3000, 64)])
def test_streams_captures_and_repeats(m, k):
    args = _inputs(m, k, 80, torch.bfloat16, "cuda", seed=8)

    def train(x, wg, wu, dh):
        leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
        h = ops.gated_linear(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))
    ref = train(*args)
    caps = [CapturedCall(train, *args) for _ in range(2)]
    for seed in range(3):
        other = _inputs(m, k, 80, torch.bfloat16, "cuda", seed=30 + seed)
        got = [[v.clone() for v in c(*other)] for c in caps]
        want = train(*other)
        for a, b, c in zip(*got, want):
            assert torch.equal(a, c) and torch.equal(b, c)
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = train(*args)
    b = train(*args)
    torch.cuda.current_stream().wait_stream(side)
    for u, v, w in zip(a, b, ref):
        assert torch.equal(u, w) and torch.equal(v, w)


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, wg, wu, dh = _inputs(3, 16, 8, torch.bfloat16, dev)
    bad = [(ValueError, (x, wg, wu, "tanh")), (TypeError, (x.float(), wg.float(), wu.float())), (TypeError, (x, wg, wu.half())),
           (ValueError, (x[:, :8], wg, wu)), (ValueError, (x, wg[:4], wu)), (ValueError, (x, wg[0], wu[0]))]
    for err, args in bad:
        with pytest.raises(err):
            ops.gated_linear(*args)
    if dev == "cuda":
        with pytest.raises(ValueError, match="is on"):
            ops.gated_linear(x, wg, wu.cpu())
    xr = x.clone().requires_grad_()
    g, = torch.autograd.grad(ops.gated_linear(xr, wg, wu).sum(), xr, create_graph=True)
    if g.requires_grad:
        with pytest.raises(NotImplementedError, match="second"):
            g.float().sum().backward()


def test_native_refusals():
    lib = _lib.lib()
    p = torch.zeros(8).data_ptr()

    def call(dtype=5, act=0, x=p, ldx=64, ldw=64, m=1, f=1, k=64, ws=None, size=0):
        return lib.vs_gated_linear(dtype, act, x, ldx, p, ldw, p, ldw, m, f, k, p, None, ws, size, None)
    for kw in (dict(dtype=0), dict(act=4), dict(act=-1), dict(m=-1), dict(f=-1), dict(k=-1), dict(x=None),
               dict(m=2, ldx=63), dict(f=2, ldw=63), dict(m=1 << 31), dict(f=1 << 21), dict(k=1 << 21),
               dict(ldx=1 << 21)):
        assert call(**kw) == 1 and b"gated_linear" in lib.vs_last_error()
    assert call(m=100, f=100, k=65, ldx=65, ldw=65, ws=p, size=16) == 1 and b"workspace" in lib.vs_last_error()
    assert lib.vs_gated_linear_backward(5, 0, p, 8, p, 8, p, 8, None, p, 8, 1, 1, 8, p, p, None, 0, None) == 1
    assert lib.vs_gated_linear_workspace(-1, 1, 1, 0) == 0
    assert lib.vs_gated_linear_backward(5, 0, p, 8, p, 8, p, 8, p, p, 1, 9, 1, 8, None, p, p, 16, None) == 1
    assert b"workspace" in lib.vs_last_error()
    for ldx, ldg, ldu, ldh in ((7, 8, 8, 2), (8, 7, 8, 2), (8, 8, -8, 2), (8, 8, 8, 1)):
        assert lib.vs_gated_linear_backward(5, 0, p, ldx, p, ldg, p, ldu, p, p, ldh, 9, 2, 8, p, p, None, 0, None) == 1
        assert b"leading dimension" in lib.vs_last_error()


@pytest.mark.parametrize("dev", DEVICES)
def test_opcheck(dev):
    x, wg, wu, dh = _inputs(5, 24, 16, torch.bfloat16, dev)
    pre = torch.randn(5, 16, 2, device=dev)
    torch.library.opcheck(torch.ops.veles.gated_linear_backward.default, (x, wg, wu, pre, dh, "gelu", True, True))
    for args in ((x, wg, wu, "gelu", False), (x.clone().requires_grad_(), wg.clone().requires_grad_(), wu, "silu", True)):
        torch.library.opcheck(torch.ops.veles.gated_linear.default, args)


@pytest.mark.parametrize("dev", DEVICES)
def test_block_trains_prefills_and_generates(dev):
    """The operators as a model uses them: value and gate projections, the recurrence, a gated feed-forward; its gradients
    against float64, then a ragged prefill followed by single tokens with 4-bit output weights, which has to agree with the
    same positions of a whole run (both paths round to bf16 at the same places: 4 roundings of 2^-8 of the largest value)."""
    b, t, d, f = 3, 20, 64, 96
    gen = torch.Generator().manual_seed(12)
    x = torch.randn(b, t, d, generator=gen).bfloat16().to(dev)
    ws = [(torch.randn(*s, generator=gen) * s[1] ** -0.5).bfloat16().to(dev)
          for s in ((d, d), (d, d), (f, d), (f, d), (d, f))]
    wv, wa, wg, wu, wo = ws
    down = ops.quantize_int4(wo, 32)

    def mix(x, wv, wa):
        return ops.gemm_bf16(x.reshape(-1, d), wv, False, True).bfloat16().view(x.shape), \
            (ops.gemm_bf16(x.reshape(-1, d), wa, False, True) + 1.5).bfloat16().view(x.shape)
    v, a = mix(x, wv, wa)
    leaves = [q.detach().requires_grad_() for q in (v, a, wg, wu)]
    y, final = ops.gated_recurrence(leaves[0], leaves[1])
    h = ops.gated_linear(y, leaves[2], leaves[3])
    up = torch.randn(b, t, f, generator=gen).bfloat16().to(dev)
    grads = torch.autograd.grad(h, leaves, up)
    ref = [q.detach().double().cpu().requires_grad_() for q in leaves]
    hr, rows = torch.zeros(b, d, dtype=torch.float64), []
    for s in range(t):
        i = torch.sigmoid(-ref[1][:, s])
        hr = hr + i * (ref[0][:, s] - hr)
        rows.append(hr)
    yr = torch.stack(rows, 1)
    gr, ur = yr @ ref[2].t(), yr @ ref[3].t()
    want = torch.autograd.grad(gr * torch.sigmoid(gr) * ur, ref, up.double().cpu())
    # y, dg / du, dy and the result are each rounded to bf16 on the way: 4 half steps of the norm
    for got, w in zip(grads, want):
        assert (got.double().cpu() - w).norm() <= 4 * 2.0 ** -8 * w.norm()

    with torch.no_grad():
        whole = ops.matvec_int4(ops.gated_linear(ops.gated_recurrence(v, a)[0], wg, wu), *down, 32)
        lengths = torch.tensor([12, 5, 1], device=dev)
        _, state = ops.gated_recurrence(v[:, :12], a[:, :12], None, lengths)
        for s in range(6):
            at = (torch.arange(b, device=dev), lengths + s)
            tok = ops.gated_recurrence_step(v[at], a[at], state)
            out = ops.matvec_int4(ops.gated_linear(tok, wg, wu), *down, 32)
            assert (out.float() - whole[at].float()).abs().max() <= 4 * 2.0 ** -8 * whole.float().abs().max()


def _split_oracle(x, wg, wu, dh, act):
    """The gradients in float64 and how far they may be off before they are rounded to the result's type: dg and du carry 2^-16
    (float16: 2^-22, or half of the smallest step) where they are split, the sums have twice as many terms, the rest is as
    in _oracle."""
    half = x.dtype == torch.float16
    e, tiny = (2.0 ** -22, 2.0 ** -25) if half else (2.0 ** -16, 2.0 ** -133)
    x, wg, wu, dh = (v.detach().double().cpu() for v in (x, wg, wu, dh))
    (m, k), f = x.shape, wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = k * U * (x.abs() @ wg.abs().t()), k * U * (x.abs() @ wu.abs().t())
    a, slope = _act(act, g)
    ea, eslope = 1.2 * eg + 8 * U * a.abs(), 1.6 * eg + 16 * U
    dg, du = dh * u * slope, dh * a
    edg = dh.abs() * (eu * slope.abs() + u.abs() * eslope) + 4 * U * dg.abs()
    edu = dh.abs() * ea + 4 * U * du.abs()
    d, ed, w = torch.cat([dg, du], 1), torch.cat([edg, edu], 1), torch.cat([wg, wu])
    ed = ed + e * (d.abs() + ed) + tiny
    dw, edw = d.t() @ x, ed.t() @ x.abs() + 2 * m * U * ((d.abs() + ed).t() @ x.abs())
    return dict(dx=(d @ w, ed @ w.abs() + 4 * f * U * ((d.abs() + ed) @ w.abs())), dw_gate=(dw[:f], edw[:f]),
                dw_up=(dw[f:], edw[f:]))


def _rounded_once(name, got, want):
    """What was off by `bound` before it was rounded to nearest is off by what rounding the exact value costs, and twice that."""
    ref, bound = want
    off = (got.detach().double().cpu() - ref).abs()
    tol = (ref.to(got.dtype).double() - ref).abs() + 2 * bound + 1e-12 * ref.abs()
    assert (off <= tol).all(), (name, int((off > tol).sum()), (off / tol).max().item())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,f", [(1, 8, 3), (33, 64, 24), (64, 72, 64), (65, 40, 130), (200, 33, 63), (300, 264, 257)])
def test_split_gradients_are_rounded_once(dev, dtype, m, k, f):
    """With split_gradients no rounding but the result's own is left, in rows, features and steps that end inside a tile."""
    for act in ("silu", "gelu"):
        x, wg, wu, dh = _inputs(m, k, f, dtype, dev, seed=m + k)
        leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
        h = ops.gated_linear(*leaves, act, split_gradients=True)
        want = _split_oracle(x, wg, wu, dh, act)
        for name, got in zip(("dx", "dw_gate", "dw_up"), torch.autograd.grad(h, leaves, dh)):
            _rounded_once(name, got, want[name])
        with torch.no_grad():
            assert torch.equal(ops.gated_linear(x, wg, wu, act), h)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,f", [(4100, 1000, 2056), (9001, 513, 65), (64, 128, 16384), (2100, 2048, 1000), (70, 4096, 700)])
def test_split_gradients_of_large_tiles_and_parts(m, k, f):
    """Every tile shape and sums in parts; the two halves of the reduction may lie in one part or in several."""
    x, wg, wu, dh = _inputs(m, k, f, torch.bfloat16, "cuda", seed=13)
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
    want = _split_oracle(x, wg, wu, dh, "silu")
    first = torch.autograd.grad(ops.gated_linear(*leaves, split_gradients=True), leaves, dh)
    for name, got in zip(("dx", "dw_gate", "dw_up"), first):
        _rounded_once(name, got, want[name])
    again = torch.autograd.grad(ops.gated_linear(*leaves, split_gradients=True), leaves, dh)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dev", DEVICES)
def test_split_gradients_that_are_not_finite(dev):
    """A gradient that is infinite or NaN, or rounds to infinity in float16, spreads as far as without split_gradients."""
    x, wg, wu, dh = _inputs(70, 40, 24, torch.float16, dev, seed=14)
    wu = wu * 64
    for bad in (float("nan"), float("inf"), 60000.0):
        d = dh.clone()
        d[3, 5] = bad
        got = []
        for split in (False, True):
            leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
            got.append(torch.autograd.grad(ops.gated_linear(*leaves, split_gradients=split), leaves, d))
        for a, b in zip(*got):
            assert torch.equal(torch.isfinite(a), torch.isfinite(b))


@pytest.mark.gpu
def test_split_gradients_captured_and_dispatched():
    args = _inputs(130, 72, 100, torch.bfloat16, "cuda", seed=15)

    def train(x, wg, wu, dh):
        leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
        return torch.autograd.grad(ops.gated_linear(*leaves, split_gradients=True), leaves, dh)
    cap = CapturedCall(train, *args)
    for seed in range(3):
        other = _inputs(130, 72, 100, torch.bfloat16, "cuda", seed=40 + seed)
        got = [v.clone() for v in cap(*other)]
        want = train(*other)
        leaves = [v.detach().requires_grad_() for v in other[:3]]
        op = torch.autograd.grad(torch.ops.veles.gated_linear(*leaves, "silu", True, True)[0], leaves, other[3])
        for a, b, c in zip(got, want, op):
            assert torch.equal(a, b) and torch.equal(c, b)
        torch.cuda.synchronize()


def test_split_gradients_native_refusals_and_workspace():
    lib = _lib.lib()
    p = torch.zeros(8).data_ptr()

    def call(split=1, m=1, f=1, ws=None, size=0, pre=p):
        return lib.vs_gated_linear_gradients(5, 0, split, p, 8, p, 8, p, 8, pre, p, f, m, f, 8, p, p, None, ws, size, None)
    for kw in (dict(m=1 << 30), dict(f=(1 << 19) + 1), dict(pre=None), dict(m=-1)):
        assert call(**kw) == 1 and b"gated_linear" in lib.vs_last_error()
    assert call(f=9, ws=p, size=16) == 1 and b"workspace" in lib.vs_last_error()
    size = lib.vs_gated_linear_gradients_workspace
    assert size(4096, 2048, 2048, 1, 1, 1, 1, 1) == 2 * size(4096, 2048, 2048, 0, 1, 1, 1, 1) == 2 * 4096 * 8192
    assert size(1 << 30, 64, 64, 1, 1, 1, 1, 1) == 0 and size(64, 1 << 20, 64, 1, 1, 1, 1, 1) == 0


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [9, 130])
def test_tails_of_activations(dev, act, m):
    """k = 1 with a gate weight of 1 and an up weight of 1: g = u = x exactly.  h = act(x) x and, from dh = 1, the weights'
    gradients of one row, act'(x) x x and act(x) x, to a few units of their own last place however small they are: functions of
    16 u and 1.5 |g| u for the exponential's argument (g^2 / 2 for gelu; erfc's is rounded, u g^2), 4 u for the products, then
    roundings to 16 bits: one of h, two of a gradient.  A slope's two terms are rounded apart."""
    x = torch.cat([torch.arange(-9, 20.01, 0.125), torch.tensor([1e-3, -1e-3, 40.0, -40.0])]).to(torch.bfloat16)
    for values in (x, x.flip(0)):
        for v in values.split(m):
            d = v.double()
            rows = v[:, None].to(dev)
            one = torch.ones(1, 1, dtype=torch.bfloat16, device=dev)
            h = ops.gated_linear(rows, one, one, act)
            a, slope = _act(act, d)
            if act == "gelu":
                arg = d * d
                parts = 0.5 * torch.special.erfc(-d * 0.5 ** 0.5) + d.abs() * torch.exp(-0.5 * d * d) / (2 * torch.pi) ** 0.5
            else:
                arg, parts = 1.5 * d.abs(), slope.abs()
                if act == "silu":
                    s = torch.sigmoid(d)
                    parts = s + d.abs() * s * torch.sigmoid(-d)
                if act == "sigmoid":     # s (1 - s) loses digits in the file's oracle
                    slope = parts = torch.sigmoid(d) * torch.sigmoid(-d)
            rel, e = (24 + 2 * arg) * U, 2.0 ** -8
            tiny = torch.finfo(torch.bfloat16).smallest_normal

            def near(got, ref, bound, roundings):
                tol = bound + ref.abs() * ((1 + e) ** roundings - 1) + 2 * e * bound + tiny * (1 + d.abs())
                off = (got.detach().double().cpu().flatten() - ref).abs()
                assert (off <= tol).all(), (act, d[off > tol], (off / tol).max().item())
            near(h, a * d, (a * d).abs() * rel, 1)
            # a feature for every value, one row: dw_gate = dh u act'(g) x, dw_up = dh act(g) x with x = 1
            wg = v[:, None].to(dev).clone().requires_grad_()
            wu = v[:, None].to(dev).clone().requires_grad_()
            up = torch.ones(1, len(v), dtype=torch.bfloat16, device=dev)
            dwg, dwu = torch.autograd.grad(ops.gated_linear(one, wg, wu, act), (wg, wu), up)
            near(dwg, d * slope, d.abs() * parts * rel, 2)
            near(dwu, a, a.abs() * rel, 2)


def test_workspaces_of_very_many_rows():
    """Sizes stay sizes up to the documented 2^31 rows; what no launch holds is refused, not begun."""
    lib = _lib.lib()
    size = lib.vs_gated_linear_workspace
    for m in (1 << 30, (1 << 30) + 5, (1 << 31) - 300):
        for k, f in ((1, 1), (9, 30), (1001, 500)):
            rows = 2 * m * ((k + 7) // 8 * 8)
            assert rows <= size(m, f, k, 0) <= 1.01 * rows + (1 << 30)
            assert size(m, f, k + (-k) % 8, 1) == 0
    p = torch.zeros(8).data_ptr()
    m, f, k = (1 << 31) - 300, 64, 1 << 19
    need = lib.vs_gated_linear_gradients_workspace(m, f, k, 0, 1, 1, 1, 1)
    assert lib.vs_gated_linear_gradients(5, 0, 0, p, k, p, k, p, k, p, p, f, m, f, k, p, p, p, p, need, None) == 1
    assert b"too many" in lib.vs_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("k,f", [(8, 8), (1, 1)])
def test_2_to_the_30_rows(k, f):
    """More small tiles than a launch of one workgroup each would hold, read in place and from copied rows."""
    m = (1 << 30) + 5
    rows = torch.randn(1 << 12, k, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    x = rows.repeat((m >> 12) + 1, 1)[:m]
    wg, wu = (torch.randn(f, k, generator=torch.Generator().manual_seed(s)).bfloat16().cuda() for s in (6, 7))
    h = ops.gated_linear(x, wg, wu)
    want = ops.gated_linear(rows, wg, wu)
    _close("h", want, _oracle(rows, wg, wu, torch.zeros_like(want), "silu")["h"])
    assert torch.equal(h[m >> 12 << 12:], want[:m & 4095])
    blocks = h[:m >> 12 << 12].view(-1, 1 << 12, f)
    for part in blocks.split(1 << 14):
        assert torch.equal(part, want.expand_as(part))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("m,k,f", [(33, 64, 24), (300, 40, 200), (700, 2048, 33)])
def test_gradients_are_made_one_by_one(dev, split, m, k, f):
    """Every set of gradients: those that are asked for have the bits of a call of their own, in memory of their own, and the
    backward op returns nothing for the others."""
    args = _inputs(m, k, f, torch.bfloat16, dev, seed=16)
    x, wg, wu, dh = args
    pre = torch.ops.veles.gated_linear(x, wg, wu, "silu", True)[1]
    want = _oracle(x, wg, wu, dh, "silu")
    for need in range(1, 8):
        on = [bool(need >> i & 1) for i in range(3)]
        leaves = [v.detach().requires_grad_(n) for v, n in zip(args[:3], on)]
        h = ops.gated_linear(*leaves, split_gradients=split)
        got = torch.autograd.grad(h, [v for v in leaves if v.requires_grad], dh)
        op = torch.ops.veles.gated_linear_backward(x, wg, wu, pre, dh, "silu", *on, split)
        assert [o.numel() for o in op] == [v.numel() if n else 0 for v, n in zip(args, on)]
        for name, g, o in zip([n for n, a in zip(("dx", "dw_gate", "dw_up"), on) if a], got, [o for o, a in zip(op, on) if a]):
            assert torch.equal(g, o) and g.untyped_storage().nbytes() == 2 * g.numel()
            _close(name, g, want[name])


@pytest.mark.parametrize("dev", DEVICES)
def test_second_derivatives_are_recorded_to_be_refused(dev):
    x, wg, wu, dh = _inputs(5, 16, 8, torch.bfloat16, dev)
    for i in range(3):
        leaves = [v.detach().requires_grad_(j == i) for j, v in enumerate((x, wg, wu))]
        g, = torch.autograd.grad(ops.gated_linear(*leaves).sum(), leaves[i], create_graph=True)
        assert g.requires_grad
        with pytest.raises(NotImplementedError, match="second"):
            g.float().sum().backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_split_gradients_are_refused_before_the_forward_pass(dev):
    x = torch.zeros(1, 1, dtype=torch.bfloat16, device=dev)
    w = torch.zeros((1 << 19) + 1, 1, dtype=torch.bfloat16, device=dev).requires_grad_()
    with pytest.raises(ValueError, match="split gradients"):
        ops.gated_linear(x, w, w, split_gradients=True)
    with torch.no_grad():
        assert ops.gated_linear(x, w, w, split_gradients=True).shape == (1, (1 << 19) + 1)


@pytest.mark.parametrize("dev", DEVICES)
def test_split_gradients_next_to_a_tie(dev):
    """Products dh (x w) whose rounding to float32 lies half way between two float16 numbers while the product does not: both
    numbers of a split gradient have to come from one and the same rounding.  (relu, one row, k = 1: dw_up = dh g x, where g = x w
    is exact; dh g is rounded to float32 and split, the rest is exact up to the last rounding.)"""
    g = torch.Generator().manual_seed(17)
    x = torch.tensor([[1.3310546875]], dtype=torch.float16)
    w = (torch.rand(1 << 18, generator=g) + 0.5).half()
    dh = (torch.rand(1 << 18, generator=g) + 0.5).half()
    p = dh.double() * x.double()[0, 0] * w.double()
    once = torch.from_numpy(p.numpy().astype("float16"))     # (torch goes by way of float32)
    found = once != p.float().half()
    assert 10 <= int(found.sum()) <= 400
    w, dh, p = w[found][:, None], dh[found][None], p[found][:, None]
    leaf = w.clone().to(dev).requires_grad_()
    got, = torch.autograd.grad(ops.gated_linear(x.to(dev), w.to(dev), leaf, "relu", split_gradients=True), leaf, dh.to(dev))
    ref = p * x.double()
    _rounded_once("dw_up", got, (ref, ref.abs() * (2.0 ** -24 + 2.0 ** -22) + 2.0 ** -25 * x.double()))
