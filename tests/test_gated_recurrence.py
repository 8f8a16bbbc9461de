"""Gated linear recurrence (ops.gated_recurrence, gated_recurrence_step) against the definition in float64.

Tolerances: `_oracle` carries a first-order rounding analysis along its own values.  With u = 2^-24, the share
i = 1 / (1 + exp(g)) is off by at most r = (1.5 |g| + 8) u relatively (argument scaling |g| u, log2(e) rounded, exp and
reciprocal within 1 ulp each, one addition); a step rounds h once (u |h|) and its increment by i |x - h| (r + 2 u).  These
errors decay by 1 - i per step like the state does.  A tile composes maps whose parts carry the same errors, and its steps
run a second time from the composed state: a factor 2 for each.  The parts of a map, (1 - i) s from what comes in and the
tile's own share, are rounded before they are added and may cancel, so the magnitudes that are rounded are those of the
recurrence over absolute values (hm_t = (1 - i) hm + i |x|, lm = |dy| + mm, mm = (1 - i) lm), not |h| and |l|: with one
step, dstate = (1 - i) dfinal + (1 - i) dy carries u (1 - i) (|dfinal| + |dy|), however small the sum.  The result is
rounded once to the output's type (half a step: eps / 2), values below the smallest normal number by at most its spacing."""
import pytest
import torch

from veles.simd_amd import _lib, ops
from veles.simd_amd.utils import CapturedCall

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def _inputs(b, t, d, dtype, dev, seed=0, state=True, lengths=None, shift=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, d, generator=g).to(dtype).to(dev)
    gate = (torch.randn(b, t, d, generator=g) * 1.5 + shift).to(dtype).to(dev)
    h0 = torch.randn(b, d, generator=g).to(dev) if state else None
    n = None
    if lengths == "ragged":
        n = torch.randint(0, t + 1, (b,), generator=g)
        n[0] = t
        n[-1] = 0 if b > 1 else t
        n = n.to(dev)
    return x, gate, h0, n


def _oracle(x, gate, h0, n, dy=None, dfinal=None):
    """Everything in float64 on the CPU: y, final and, with dy / dfinal, dx, dgate, dstate; and the error bounds of each."""
    x, gate = x.detach().double().cpu(), gate.detach().double().cpu()
    b, t, d = x.shape
    n = torch.full((b,), t) if n is None else n.cpu().long().clamp(0, t)
    h = torch.zeros(b, d, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    e, hm = torch.zeros_like(h), h.abs()
    y, before, eb, dm = (torch.zeros(b, t, d, dtype=torch.float64) for _ in range(4))
    ey = torch.zeros_like(y)
    share = 1.0 / (1.0 + torch.exp(gate))
    r = (1.5 * gate.abs() + 8.0) * U
    for s in range(t):
        on = (s < n)[:, None]
        before[:, s], eb[:, s] = h, e
        i = share[:, s]
        dm[:, s] = x[:, s].abs() + hm
        h = torch.where(on, h + i * (x[:, s] - h), h)
        hm = torch.where(on, (1 - i) * hm + i * x[:, s].abs(), hm)
        e = torch.where(on, (1 - i) * e + U * hm + i * dm[:, s] * (r[:, s] + 2 * U), e)
        y[:, s], ey[:, s] = torch.where(on, h, 0.0), torch.where(on, 4 * e, 0.0)
    out = dict(y=(y, ey), final=(h, 4 * e + U * hm))
    if dy is None and dfinal is None:
        return out
    dy = torch.zeros(b, t, d).double() if dy is None else dy.detach().double().cpu()
    m = torch.zeros(b, d).double() if dfinal is None else dfinal.double().cpu()
    em, mm = torch.zeros_like(m), m.abs()
    dx, dg, edx, edg = (torch.zeros(b, t, d).double() for _ in range(4))
    for s in range(t - 1, -1, -1):
        on = (s < n)[:, None]
        i, rel = share[:, s], r[:, s]
        lam, lm = dy[:, s] + m, dy[:, s].abs() + mm
        el = em + U * lm
        diff = before[:, s] - x[:, s]
        dx[:, s] = torch.where(on, i * lam, 0.0)
        dg[:, s] = torch.where(on, i * (1 - i) * lam * diff, 0.0)
        edx[:, s] = torch.where(on, 4 * i * el + i * lm * (rel + 2 * U), 0.0)
        # 1 - i is off by i r + u absolutely
        edg[:, s] = torch.where(on, 4 * i * (1 - i) * (el * diff.abs() + lam.abs() * (eb[:, s] + U * dm[:, s]))
                                + i * (lam * diff).abs() * ((1 - i) * (rel + 4 * U) + i * rel + U), 0.0)
        em = torch.where(on, (1 - i) * el + U * lm + i * lm * rel, em)
        m = torch.where(on, (1 - i) * lam, m)
        mm = torch.where(on, (1 - i) * lm, mm)
    out.update(dx=(dx, edx), dgate=(dg, edg), dstate=(m, 4 * em + U * mm))
    return out


def _close(name, got, want):
    ref, bound = want
    got_d = got.detach().double().cpu()
    tol = bound + torch.finfo(got.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(got.dtype).smallest_normal
    bad = ~((got_d - ref).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), (got_d - ref).abs().max().item(),
                           ((got_d - ref).abs() / tol).max().item())


SHAPES = [(1, 1, 1), (2, 1, 64), (3, 16, 65), (2, 17, 128), (1, 33, 130), (5, 32, 2), (2, 128, 66), (2, 129, 63),
          (3, 257, 130), (1, 1000, 257), (4, 300, 128)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [None, "ragged"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(dev, dtype, lengths, shape):
    x, gate, h0, n = _inputs(*shape, dtype, dev, seed=sum(shape), lengths=lengths)
    g = torch.Generator().manual_seed(99)
    dy, df = torch.randn(shape, generator=g).to(dtype).to(dev), torch.randn(shape[0], shape[2], generator=g).to(dev)
    leaves = [v.requires_grad_() for v in (x, gate, h0)]
    y, final = ops.gated_recurrence(x, gate, h0, n)
    grads = torch.autograd.grad((y, final), leaves, (dy, df))
    want = _oracle(x, gate, h0, n, dy, df)
    assert y.dtype == dtype and final.dtype == torch.float32
    for name, got in zip(("y", "final", "dx", "dgate", "dstate"), (y, final, *grads)):
        _close(name, got, want[name])
    with torch.no_grad():  # the same values without the saved states
        y2, f2 = ops.gated_recurrence(x, gate, h0, n)
    assert torch.equal(y2, y) and torch.equal(f2, final)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 9000, 1), (1, 6001, 70), (2, 5000, 200), (1, 4100, 512), (70001, 2, 3),
                                   (300, 40, 130), (1, 2048, 64), (3, 2049, 66), (600, 300, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_wide_and_many(shape, dtype):
    """Chains of tiles: runs that end with the sequence and one step behind, more tiles than workgroups that run at once,
    more sequences than one grid dimension of 65535, partly filled tiles."""
    x, gate, h0, n = _inputs(*shape, dtype, "cuda", seed=5, lengths="ragged")
    if shape[0] == 1:
        n = torch.tensor([shape[1] - 37], device="cuda")
    g = torch.Generator().manual_seed(98)
    dy, df = torch.randn(shape, generator=g).to(dtype).cuda(), torch.randn(shape[0], shape[2], generator=g).cuda()
    leaves = [v.requires_grad_() for v in (x, gate, h0)]
    y, final = ops.gated_recurrence(x, gate, h0, n)
    grads = torch.autograd.grad((y, final), leaves, (dy, df))
    want = _oracle(x, gate, h0, n, dy, df)
    for name, got in zip(("y", "final", "dx", "dgate", "dstate"), (y, final, *grads)):
        _close(name, got, want[name])


@pytest.mark.gpu
def test_more_tiles_than_one_grid():
    """2^21 + 5 sequences of two tiles are two launches; every sequence gets the bits of a small call."""
    b, t = (1 << 21) + 5, 129
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(b, t, 1, device="cuda", generator=g)
    gate = torch.randn(b, t, 1, device="cuda", generator=g) + 2
    y, final = ops.gated_recurrence(x, gate)
    rows = torch.tensor([0, 1, 77777, (1 << 21) - 1, 1 << 21, (1 << 21) + 4], device="cuda")
    ys, fs = ops.gated_recurrence(x[rows], gate[rows])
    assert torch.equal(y[rows], ys) and torch.equal(final[rows], fs)


@pytest.mark.parametrize("dev", DEVICES)
def test_formula_gradient_agrees_with_differences(dev):
    """The gradients against central differences of the float64 definition (step 1e-5: truncation ~1e-10)."""
    x, gate, h0, n = _inputs(2, 7, 3, torch.float32, dev, seed=11)
    n = torch.tensor([7, 4], device=dev)
    w, wf = torch.randn(2, 7, 3, dtype=torch.float64), torch.randn(2, 3, dtype=torch.float64)

    def loss(xv, gv, hv):
        h, total = hv, torch.zeros((), dtype=torch.float64)
        for s in range(7):
            on = (s < n.cpu())[:, None]
            h = torch.where(on, torch.sigmoid(gv[:, s]) * h + torch.sigmoid(-gv[:, s]) * xv[:, s], h)
            total = total + (torch.where(on, h, 0.0) * w[:, s]).sum()
        return total + (h * wf).sum()

    leaves = [v.requires_grad_() for v in (x, gate, h0)]
    y, final = ops.gated_recurrence(*leaves, n)
    got = torch.autograd.grad((y, final), leaves, (w.float().to(dev), wf.float().to(dev)))
    base = [v.detach().double().cpu() for v in leaves]
    for k, grad in enumerate(got):
        for at in range(base[k].numel()):
            vals = []
            for sign in (1, -1):
                moved = [v.clone() for v in base]
                moved[k].view(-1)[at] += sign * 1e-5
                vals.append(loss(*moved))
            diff = ((vals[0] - vals[1]) / 2e-5).item()
            assert abs(grad.reshape(-1)[at].item() - diff) <= 1e-5 * max(1.0, abs(diff))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("shape", [(3, 40, 66), (2, 500, 65), (1, 5000, 64)])
def test_padding_is_never_read(dev, shape):
    """NaN and infinities behind the sequences' ends change nothing, forward and backward; lengths outside 0..t are clamped."""
    if dev == "cpu" and shape[1] > 1000:
        pytest.skip("the chained path is the GPU's")
    b, t, d = shape
    x, gate, h0, _ = _inputs(b, t, d, torch.float32, dev, seed=3)
    n = torch.tensor([t - 3, 0, -5][:b], dtype=torch.int32, device=dev)
    dy = torch.randn(b, t, d, device=dev)
    pad = torch.arange(t, device=dev)[None, :] >= n.clamp(min=0)[:, None]

    def run(fill):
        xs = [torch.where(pad[..., None], fill, v).requires_grad_() for v in (x, gate)]
        y, final = ops.gated_recurrence(*xs, h0, n)
        return (y, final, *torch.autograd.grad((y, final), xs, (torch.where(pad[..., None], fill, dy),
                                                                torch.ones_like(final))))
    clean = run(torch.tensor(0.0, device=dev))
    for bad in (float("nan"), float("inf"), float("-inf")):
        for a, c in zip(run(torch.tensor(bad, device=dev)), clean):
            assert torch.equal(a, c)
    for v in (clean[0], clean[2], clean[3]):
        assert (v[pad] == 0).all()
    if b > 1:
        assert torch.equal(clean[1][1], h0[1])
    over = ops.gated_recurrence(x, gate, h0, torch.full((b,), 1 << 40, dtype=torch.int64, device=dev))
    assert torch.equal(over[0], ops.gated_recurrence(x, gate, h0)[0])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dev, dtype):
    """Slices at odd offsets, time-major storage, broadcast inputs, channels that are not neighbours: the values of a copy."""
    b, t, d = 3, 150, 64
    base, gbase, h0, n = _inputs(b, t, 2 * d + 3, dtype, dev, seed=8, lengths="ragged")
    h0 = h0[:, :d]
    views = [(base[..., 1:d + 1], gbase[..., 2:d + 2]), (base[..., :2 * d:2], gbase[..., 1:2 * d:2]),
             (base.transpose(0, 1).contiguous().transpose(0, 1)[..., :d], gbase[..., :d]),
             (base[:1, :, :d].expand(b, t, d), gbase[:, :1, :d].expand(b, t, d)),
             (base[:, :, :1].expand(b, t, d), gbase[..., :d])]
    for xv, gv in views:
        leaves = [xv.detach().requires_grad_(), gv.detach().requires_grad_(), h0.detach().requires_grad_()]
        copies = [v.detach().contiguous().requires_grad_() for v in leaves]
        a, c = (ops.gated_recurrence(*v, n) for v in (leaves, copies))
        up = torch.ones(1, 1, 1, dtype=dtype, device=dev).expand(b, t, d)       # as sum() gives it
        up2 = torch.ones(b, t, d, dtype=dtype, device=dev)
        ga = torch.autograd.grad(a[0], leaves, up)
        gc = torch.autograd.grad(c[0], copies, up2)
        want = _oracle(*copies, n, up2, None)
        for name, got in zip(("y", "final", "dx", "dgate", "dstate"), (*a, *ga)):
            _close(name, got, want[name])
        for name, got in zip(("y", "final", "dx", "dgate", "dstate"), (*c, *gc)):
            _close(name, got, want[name])


@pytest.mark.parametrize("dev", DEVICES)
def test_single_outputs_and_no_state(dev):
    x, gate, _, _ = _inputs(2, 50, 40, torch.float32, dev, state=False)
    x, gate = x.requires_grad_(), gate.requires_grad_()
    y, final = ops.gated_recurrence(x, gate)
    df = torch.randn_like(final)
    grads = torch.autograd.grad(final, (x, gate), df, retain_graph=True)
    want = _oracle(x, gate, None, None, None, df)
    for name, got in zip(("dx", "dgate"), grads):
        _close(name, got, want[name])
    gx, = torch.autograd.grad(y.sum(), x)
    _close("dx", gx, _oracle(x, gate, None, None, torch.ones_like(y))["dx"])


@pytest.mark.parametrize("dev", DEVICES)
def test_extreme_gates(dev):
    """A gate of +inf or 200 keeps the state exactly, -inf or -200 replaces it exactly."""
    b, t, d = 2, 40, 8
    x = torch.randn(b, t, d, device=dev)
    h0 = torch.randn(b, d, device=dev)
    for v in (float("inf"), 200.0):
        y, final = ops.gated_recurrence(x, torch.full_like(x, v), h0)
        assert torch.equal(y, h0[:, None].expand(b, t, d)) and torch.equal(final, h0)
    for v in (float("-inf"), -200.0):
        y, final = ops.gated_recurrence(x, torch.full_like(x, v), h0)
        assert (y - x).abs().max() <= 2 * U * x.abs().max() * 4
    y, _ = ops.gated_recurrence(x, torch.full_like(x, float("nan")), h0)
    assert torch.isnan(y).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("b,t,d", [(0, 5, 3), (2, 0, 3), (2, 5, 0)])
def test_empty(dev, b, t, d):
    x, gate = torch.zeros(b, t, d, device=dev, requires_grad=True), torch.zeros(b, t, d, device=dev)
    h0 = torch.randn(b, d, device=dev).requires_grad_()
    y, final = ops.gated_recurrence(x, gate, h0)
    assert y.shape == (b, t, d) and torch.equal(final, h0)
    gx, gh = torch.autograd.grad(final.sum() + y.sum(), (x, h0))
    assert gx.shape == x.shape and torch.equal(gh, torch.ones_like(h0))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,d", [(1, 1), (3, 65), (8, 2048)])
def test_step_continues_a_prefill(dev, dtype, b, d):
    """Prefill of a ragged batch, then single tokens: the steps agree with the whole sequence's oracle."""
    x, gate, h0, n = _inputs(b, 12, d, dtype, dev, seed=4, lengths="ragged")
    _, state = ops.gated_recurrence(x[:, :9], gate[:, :9], h0, n.clamp(max=9))
    at = state.data_ptr()
    m = n.clamp(max=9).cpu()
    full_x, full_g = torch.zeros(b, 12, d, dtype=dtype), torch.zeros(b, 12, d, dtype=dtype)
    for r in range(b):
        k = int(m[r])
        full_x[r, :k], full_g[r, :k] = x[r, :k].cpu(), gate[r, :k].cpu()
        full_x[r, k:k + 3], full_g[r, k:k + 3] = x[r, 9:].cpu(), gate[r, 9:].cpu()
    want_y, ey = _oracle(full_x, full_g, h0, m + 3)["y"]
    for s in range(3):
        y = ops.gated_recurrence_step(x[:, 9 + s], gate[:, 9 + s], state)
        assert state.data_ptr() == at and y.dtype == dtype
        idx = (torch.arange(b), m + s)
        _close("y", y, (want_y[idx], ey[idx]))
        _close("state", state, (want_y[idx], ey[idx]))


@pytest.mark.gpu
def test_arrays_past_32_bit_offsets():
    """2.2e9 values in one sequence: its last steps, and the gradients there, are those of a sequence of its own that begins
    2000 steps earlier (what came before has decayed: the shares are 1/2)."""
    t, d, k = (1 << 21) + 130, 1040, 2000
    x = torch.randn(1, t, d, device="cuda", dtype=torch.bfloat16, generator=torch.Generator("cuda").manual_seed(5))
    gate = torch.zeros(1, t, d, device="cuda", dtype=torch.bfloat16)
    leaves = [v.requires_grad_() for v in (x, gate)]
    y, final = ops.gated_recurrence(*leaves)
    got = [y.detach()[:, -200:].clone(), final.detach()] + [g[:, -200:].clone() for g in torch.autograd.grad(final.sum(), leaves)]
    del y
    own = [v.detach()[:, -k:].clone().requires_grad_() for v in (x, gate)]
    y, final = ops.gated_recurrence(*own)
    want = [y.detach()[:, -200:], final.detach()] + [g[:, -200:] for g in torch.autograd.grad(final.sum(), own)]
    # the same steps in other tiles: a step's 3 roundings of at most u max|h| halve with every step, so 6 u max|h| on each
    # side with max|h| < 5; then a step of the result's type where the rounding falls on different sides
    for a, b in zip(got, want):
        eps = torch.finfo(a.dtype).eps
        assert ((a.double() - b.double()).abs() <= eps * b.double().abs() + 64 * U).all()


@pytest.mark.gpu
def test_more_groups_than_one_launch():
    """2^21 + 5 sequences of two tiles take two launches; the sequences around the cut have the bits of a small call."""
    b, t = (1 << 21) + 5, 130
    gen = torch.Generator("cuda").manual_seed(6)
    x, gate = (torch.randn(b, t, 1, device="cuda", dtype=torch.bfloat16, generator=gen) for _ in range(2))
    y, final = ops.gated_recurrence(x, gate)
    for at in (0, (1 << 21) - 3, b - 6):
        ys, fs = ops.gated_recurrence(x[at:at + 6], gate[at:at + 6])
        assert torch.equal(y[at:at + 6], ys) and torch.equal(final[at:at + 6], fs)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", [9, 30, 300])
def test_infinite_states_pass_through_padding(dev, t):
    """An infinite initial state of an empty sequence, and a value that is infinite at the last step before the padding."""
    n = torch.tensor([0, 5, t - 1, 1], device=dev)
    x, gate, h0, _ = _inputs(4, t, 6, torch.float32, dev, seed=9)
    h0, x = h0.clone(), x.clone()
    h0[0, 2] = float("inf")
    for b in (1, 2, 3):
        x[b, int(n[b]) - 1, 2] = -float("inf")
    y, final = ops.gated_recurrence(x, gate, h0, n)
    assert final[0, 2] == float("inf") and (final[1:, 2] == -float("inf")).all()
    other = [0, 1, 3, 4, 5]
    assert torch.isfinite(final[:, other]).all() and torch.isfinite(y[:, :, other]).all()
    for b in range(4):
        assert (y[b, int(n[b]):] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_step_counts_as_a_write(dev):
    """A backward pass that needs the state as it was before the step refuses, as for any tensor written in place."""
    x, gate, h0, _ = _inputs(2, 3, 4, torch.float32, dev)
    h0 = h0.clone()
    w = torch.randn_like(h0).requires_grad_()
    loss = (w * h0).sum()
    ops.gated_recurrence_step(x[:, 0], gate[:, 0], h0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    with torch.inference_mode():
        s = torch.zeros(2, 4, device=dev)
        ops.gated_recurrence_step(x[:, 0], gate[:, 0], s)


@pytest.mark.gpu
def test_runs_are_bitwise_alike_and_stream_ordered():
    x, gate, h0, n = _inputs(2, 3000, 96, torch.bfloat16, "cuda", seed=6, lengths="ragged")
    ref = ops.gated_recurrence(x, gate, h0, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.gated_recurrence(x, gate, h0, n)
        x2 = a[0] * 2
        c = ops.gated_recurrence(x2, gate, h0, n)
    b2 = ops.gated_recurrence(x, gate, h0, n)         # the other stream, at the same time
    torch.cuda.current_stream().wait_stream(side)
    for v in (a, b2):
        assert torch.equal(v[0], ref[0]) and torch.equal(v[1], ref[1])
    want = ops.gated_recurrence(ref[0] * 2, gate, h0, n)
    assert torch.equal(c[0], want[0])


@pytest.mark.gpu
def test_capture_forward_backward_and_step():
    """A captured training pass and step, replayed with eager work in between (the state lives outside the graph)."""
    x, gate, h0, _ = _inputs(2, 4000, 64, torch.float32, "cuda", seed=7)
    dy = torch.randn_like(x)

    def train(x, gate, h0, dy):
        leaves = [v.detach().requires_grad_() for v in (x, gate, h0)]
        y, final = ops.gated_recurrence(*leaves)
        return (y.detach(), final.detach(), *torch.autograd.grad(y, leaves, dy))

    cap = CapturedCall(train, x, gate, h0, dy)
    cap2 = CapturedCall(train, x, gate, h0, dy)
    state = h0.clone()
    step = CapturedCall(lambda a, b: ops.gated_recurrence_step(a, b, state), x[:, 0].contiguous(), gate[:, 0].contiguous())
    for seed in range(3):
        args = [*_inputs(2, 4000, 64, torch.float32, "cuda", seed=20 + seed)[:3], torch.randn_like(x)]
        got = [v.clone() for v in cap(*args)]
        other = [v.clone() for v in cap2(*args)]
        want = train(*args)
        for a, b, c in zip(got, other, want):
            assert torch.equal(a, c) and torch.equal(b, c)
        state.copy_(args[2])
        eager = args[2].clone()
        y = step(args[0][:, 1], args[1][:, 1]).clone()
        assert torch.equal(y, ops.gated_recurrence_step(args[0][:, 1], args[1][:, 1], eager))
        assert torch.equal(state, eager)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, gate, h0, _ = _inputs(2, 5, 4, torch.float32, dev)
    bad = [
        (TypeError, (x.double(), gate.double())), (TypeError, (x, gate.half())), (TypeError, (x, gate, h0.half())),
        (ValueError, (x[0], gate[0])), (ValueError, (x, gate[:, :4])), (ValueError, (x, gate, h0[:, :3])),
        (ValueError, (x, gate, h0[:1])), (TypeError, (x, gate, h0, torch.ones(2, device=dev))),
        (ValueError, (x, gate, h0, torch.ones(3, dtype=torch.int32, device=dev))),
    ]
    for err, args in bad:
        with pytest.raises(err):
            ops.gated_recurrence(*args)
    with pytest.raises(ValueError):
        ops.gated_recurrence_step(x, gate, h0)
    with pytest.raises(ValueError):
        ops.gated_recurrence_step(x[:, 0], gate[:, 0], torch.zeros(4, 2, device=dev).t())
    with pytest.raises(TypeError):
        ops.gated_recurrence_step(x[:, 0], gate[:, 0], h0.double())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gated_recurrence_step(x[:, 0].requires_grad_(), gate[:, 0], h0)
    if dev == "cuda":
        with pytest.raises(ValueError, match="is on"):
            ops.gated_recurrence(x, gate, h0.cpu())
    xr = x.clone().requires_grad_()
    y, _ = ops.gated_recurrence(xr, gate, h0)
    g, = torch.autograd.grad(y.sum(), xr, create_graph=True)
    if g.requires_grad:
        with pytest.raises(NotImplementedError, match="second"):
            g.sum().backward()


def test_native_refusals():
    """The C entry points return an error for every bad argument, with no GPU needed."""
    lib = _lib.lib()
    one = torch.zeros(4)
    p = one.data_ptr()

    def call(dtype=0, batch=1, t=1, d=1, x=p):
        return lib.vs_gated_recurrence(dtype, x, 1, 1, p, 1, 1, None, None, 0, batch, t, d, p, p, None, None, 0, None)
    for kw in (dict(dtype=4), dict(dtype=99), dict(batch=-1), dict(t=-1), dict(d=-1), dict(x=None), dict(d=1 << 40)):
        assert call(**kw) == 1 and b"gated_recurrence" in lib.vs_last_error()
    assert lib.vs_gated_recurrence_backward(0, p, 1, 1, p, 1, 1, None, 0, None, None, 0, 0, None, 1, 1, 1, p, p, None, None,
                                            0, None) == 1
    assert lib.vs_gated_recurrence_step(0, None, 1, p, 1, p, 1, 1, p, None) == 1
    need = lib.vs_gated_recurrence_workspace(1, 5000, 64)
    assert need > 0 and lib.vs_gated_recurrence(0, p, 1, 1, p, 1, 1, None, None, 0, 1, 5000, 64, p, p, None, p, need - 1,
                                                None) == 1
    assert b"workspace" in lib.vs_last_error()
    assert lib.vs_gated_recurrence_workspace(-1, 5, 5) == 0 and lib.vs_gated_recurrence_tiles(0) == 0


OPCHECK = {
    "gated_recurrence": lambda r, dev: [
        (r(2, 9, 5).requires_grad_(), r(2, 9, 5).requires_grad_(), r(2, 5).requires_grad_(),
         torch.tensor([9, 3], device=dev), True), (r(2, 9, 5), r(2, 9, 5), None, None, False)],
    "gated_recurrence_step": lambda r, dev: [(r(3, 5), r(3, 5), r(3, 5))],
    "gated_recurrence_backward": lambda r, dev: [
        (r(2, 9, 5), r(2, 9, 5), torch.tensor([9, 3], device=dev), r(2, 1, 5), r(2, 9, 5), r(2, 5)),
        (r(2, 9, 5), r(2, 9, 5), None, r(2, 1, 5), None, r(2, 5))],
}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", sorted(OPCHECK))
def test_opcheck(name, dev):
    g = torch.Generator().manual_seed(3)
    op = getattr(torch.ops.veles, name).default
    for args in OPCHECK[name](lambda *s: torch.randn(*s, generator=g).to(dev), dev):
        torch.library.opcheck(op, args)


@pytest.mark.gpu
def test_compiled_call_traces_the_op():
    x, gate, h0, _ = _inputs(2, 70, 32, torch.float32, "cuda")
    out = torch.compile(lambda a, b, c: ops.gated_recurrence(a, b, c), backend="aot_eager")(x, gate, h0)
    ref = ops.gated_recurrence(x, gate, h0)
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


@pytest.mark.parametrize("dev", DEVICES)
def test_step_on_inputs_that_share_the_states_memory(dev):
    """x or the gate may be the state itself, a row of it for all sequences, or a stretch that begins elsewhere in it."""
    g = torch.Generator().manual_seed(15)
    buf = torch.randn(40 * 64 + 70, generator=g).to(dev)
    other = torch.randn(40, 64, generator=g).to(dev)

    def views(buf):
        state = buf[:40 * 64].view(40, 64)
        yield state, state
        yield state[3:4].expand(40, 64), state
        yield buf[65:65 + 40 * 64].view(40, 64), state
        yield buf.as_strided((40, 64), (32, 1), 5), state
        yield buf[:40 * 64 // 2].view(torch.bfloat16).view(40, 64), state
    for i in range(5):
        for swap in (False, True):
            mine, ref = buf.clone(), buf.clone()
            (x, state), (rx, rs) = list(views(mine))[i], list(views(ref))[i]
            rx = rx.clone()
            a, b = other.to(x.dtype), other.to(x.dtype)
            y = ops.gated_recurrence_step(*((a, x) if swap else (x, a)), state)
            want = ops.gated_recurrence_step(*((b, rx) if swap else (rx, b)), rs)
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(y), nan) and torch.equal(y[~nan], want[~nan])
            ok = ~torch.isnan(rs)
            assert torch.equal(state[ok], rs[ok]) and torch.equal(mine[40 * 64:], ref[40 * 64:])


def _relative_oracle(x, gate, h0, dy, dfinal):
    """As _oracle, with bounds that are relative to the shares, however small.  A step computes the smaller share s of i and
    1 - i to r relatively and rounds s (x - h) by 2 u and its result by u; i l, (1 - i) l and i (1 - i) l diff have relative
    errors of r + 2 u, r + 2 u and 2 r + 6 u besides those of l and diff."""
    x, gate, h, dy, m = (v.detach().double().cpu() for v in (x, gate, h0, dy, dfinal))
    t = x.shape[1]
    take, keep = 1.0 / (1.0 + torch.exp(gate)), 1.0 / (1.0 + torch.exp(-gate))
    r = (1.5 * gate.abs() + 8.0) * U
    e, hm = torch.zeros_like(h), h.abs()
    y, ey, before, eb, dm, dx, edx, dg, edg = (torch.zeros_like(x) for _ in range(9))
    for s in range(t):
        i, k = take[:, s], keep[:, s]
        before[:, s], eb[:, s], dm[:, s] = h, e, x[:, s].abs() + hm
        h, hm = k * h + i * x[:, s], k * hm + i * x[:, s].abs()
        e = k * e + U * hm + torch.minimum(i, k) * dm[:, s] * (r[:, s] + 2 * U)
        y[:, s], ey[:, s] = h, 4 * e
    em, mm = torch.zeros_like(m), m.abs()
    final = (h, 4 * e + U * hm)
    for s in range(t - 1, -1, -1):
        i, k, rel = take[:, s], keep[:, s], r[:, s]
        lam, lm = dy[:, s] + m, dy[:, s].abs() + mm
        el = em + U * lm
        diff = before[:, s] - x[:, s]
        dx[:, s], edx[:, s] = i * lam, 4 * i * el + i * lm * (rel + 2 * U)
        dg[:, s] = i * k * lam * diff
        edg[:, s] = 4 * i * k * (el * diff.abs() + lam.abs() * (eb[:, s] + U * dm[:, s])) + dg[:, s].abs() * (2 * rel + 6 * U)
        em, m, mm = k * el + k * lm * (rel + 2 * U), k * lam, k * lm
    return dict(y=(y, ey), final=final, dx=(dx, edx), dgate=(dg, edg), dstate=(m, 4 * em + U * mm))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,d", [(3, 1, 64), (2, 12, 66), (2, 30, 65), (2, 300, 64), (1, 1500, 66)])
def test_replaced_states_and_small_shares(dev, dtype, b, t, d):
    """Gates on both sides and values of very different sizes: a value that replaces a larger state, and the gradients through
    the share that is nearly gone, have all their digits."""
    g = torch.Generator().manual_seed(t)

    def sizes(*s):
        return torch.randn(*s, generator=g) * 10.0 ** (torch.rand(*s, generator=g) * 6 - 3)
    x, dy = (sizes(b, t, d).to(dtype).to(dev) for _ in range(2))
    gate = (torch.rand(b, t, d, generator=g) * 50 - 30).to(dtype).to(dev)
    h0, df = (1e3 * sizes(b, d).to(dev) for _ in range(2))
    leaves = [v.requires_grad_() for v in (x, gate, h0)]
    y, final = ops.gated_recurrence(*leaves)
    grads = torch.autograd.grad((y, final), leaves, (dy, df))
    want = _relative_oracle(x, gate, h0, dy, df)

    def close(name, got, want):
        # what is past float16's largest number by more than its bound and half a step rounds to infinity
        ref, bound = want
        past = ref.abs() - bound >= torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 2)
        off = got.detach().double().cpu()
        assert torch.equal(off[past], ref[past].sign() * float("inf")), name
        near = (ref.abs() + bound >= torch.finfo(got.dtype).max) & ~past
        _close(name, off[~past & ~near].to(got.dtype), (ref[~past & ~near], bound[~past & ~near]))
    for name, got in zip(("y", "final", "dx", "dgate", "dstate"), (y, final, *grads)):
        close(name, got, want[name])
    state = h0.detach().clone()
    with torch.no_grad():
        y1 = ops.gated_recurrence_step(x[:, 0], gate[:, 0], state)
    for got in (y1, state):
        close("step", got, (want["y"][0][:, 0], want["y"][1][:, 0]))


@pytest.mark.parametrize("dev", DEVICES)
def test_reset_forgets_a_large_state(dev):
    """A gate of -inf or -200 replaces a state of any finite size exactly, in y, in the final state and in a step."""
    x = torch.randn(2, 140, 6, generator=torch.Generator().manual_seed(3)).to(dev) * 1e-3
    h0 = torch.full((2, 6), 1e30, device=dev)
    for v in (float("-inf"), -200.0):
        gate = torch.full_like(x, v)
        y, final = ops.gated_recurrence(x, gate, h0)
        assert torch.equal(y, x) and torch.equal(final, x[:, -1])
        state = h0.clone()
        assert torch.equal(ops.gated_recurrence_step(x[:, 0], gate[:, 0], state), x[:, 0]) and torch.equal(state, x[:, 0])


@pytest.mark.parametrize("dev", DEVICES)
def test_second_derivatives_are_recorded_to_be_refused(dev):
    """(The gradient in the state alone of a linear loss is a constant, a product of shares: there is nothing to record.)"""
    args = _inputs(2, 5, 4, torch.float32, dev)[:3]
    for i, linear in ((0, True), (1, True), (0, False), (1, False), (2, False)):
        leaves = [v.detach().requires_grad_(j == i) for j, v in enumerate(args)]
        y = ops.gated_recurrence(*leaves)[0]
        g, = torch.autograd.grad((y if linear else y.square()).sum(), leaves[i], create_graph=True)
        assert g.requires_grad
        with pytest.raises(NotImplementedError, match="second"):
            g.sum().backward()
