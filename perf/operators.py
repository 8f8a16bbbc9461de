"""The operators of sequence models as measured cases: the gated linear recurrence (forward, training pass, single-token
step), the gated linear layer (forward, training pass, few rows) and products with 4-bit weights.

``own = False`` computes them in elementary torch operations, ``own = True`` through ``veles.simd_amd.ops``.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of each of eight sequences being generated
        dict(name="step 8x2048 bf16", op="step", b=8, d=2048, dtype="bfloat16"),
        # prompts of unequal length, padded to the longest
        dict(name="recurrence ragged 16x1000x1536 fp16", op="recurrence", b=16, t=1000, d=1536, dtype="float16",
             ragged=True, train=False),
        # one long document
        dict(name="recurrence 1x65536x1024 fp32", op="recurrence", b=1, t=65536, d=1024, dtype="float32",
             ragged=False, train=False),
        # a training step's layer
        dict(name="recurrence train 4x4096x4096 bf16", op="recurrence", b=4, t=4096, d=4096, dtype="bfloat16",
             ragged=False, train=True),
        # feed-forward of one generated token
        dict(name="gated 1x2048x6144 bf16", op="gated", m=1, k=2048, f=6144, dtype="bfloat16", act="silu", train=False),
        # feed-forward of a decoding batch
        dict(name="gated 33x4096x10240 bf16", op="gated", m=33, k=4096, f=10240, dtype="bfloat16", act="silu",
             train=False),
        # sizes that fit no tile
        dict(name="gated odd 777x1003x2741 fp16", op="gated", m=777, k=1003, f=2741, dtype="float16", act="gelu",
             train=False),
        # training step of a layer
        dict(name="gated train 4096x2048x6144 bf16", op="gated", m=4096, k=2048, f=6144, dtype="bfloat16", act="silu",
             train=True),
        # prefill of a large layer
        dict(name="gated 8192x4096x12288 bf16", op="gated", m=8192, k=4096, f=12288, dtype="bfloat16", act="silu",
             train=False),
        # one token through a projection kept in 4 bits
        dict(name="int4 1x4096x4096 g128 bf16", op="int4", m=1, n=4096, k=4096, group=128, zeros=True, dtype="bfloat16"),
        # a projection of odd sizes with a group that ends early
        dict(name="int4 odd 3x1001x1500 g32 bf16", op="int4", m=3, n=1001, k=1500, group=32, zeros=False,
             dtype="bfloat16"),
        # a decoding batch through a large projection
        dict(name="int4 16x28000x8192 g64 fp16", op="int4", m=16, n=28000, k=8192, group=64, zeros=True,
             dtype="float16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """Half of the sizes are multiples of 64 (where the range has any), the others are any number."""
    v = _log(rng, lo, hi)
    return max(64, v // 64 * 64) if rng.random() < 0.5 and v >= 64 else v


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


def draw(rng):
    most = max(_cost(c) for c in listed() if c["op"] != "step")
    while True:
        op = rng.choice(("step", "recurrence", "recurrence", "gated", "gated", "int4", "int4"))
        if op == "step":
            return dict(op=op, b=_log(rng, 1, 512), d=_size(rng, 64, 8192), dtype=rng.choice(sorted(DTYPES)))
        if op == "recurrence":
            case = dict(op=op, b=_log(rng, 1, 64), t=_log(rng, 1, 65536), d=_size(rng, 64, 8192),
                        dtype=rng.choice(sorted(DTYPES)), ragged=rng.random() < 0.4, train=rng.random() < 0.5)
            if case["b"] * case["t"] * case["d"] > 1 << 26:
                continue
        elif op == "gated":
            case = dict(op=op, m=_size(rng, 1, 8192), k=_size(rng, 64, 8192), f=_size(rng, 64, 16384),
                        dtype=rng.choice(("bfloat16", "float16")),
                        act=rng.choice(("silu", "gelu", "relu", "sigmoid")), train=rng.random() < 0.4)
        else:
            case = dict(op=op, m=_log(rng, 1, 16), n=_size(rng, 64, 28000), k=_size(rng, 64, 16384),
                        group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.7,
                        dtype=rng.choice(("bfloat16", "float16")))
            if case["n"] * case["k"] > 28000 * 8192:
                continue
        if _cost(case) <= most:
            return case


def work(case):
    if case["op"] == "step":
        n, e = case["b"] * case["d"], DTYPES[case["dtype"]].itemsize
        return dict(bytes=n * (3 * e + 8), flops=10 * n)  # value, gate in; output out; state in and out
    if case["op"] == "recurrence":
        b, n, e = case["b"], case["b"] * case["t"] * case["d"], DTYPES[case["dtype"]].itemsize
        state = 4 * b * case["d"]
        if case["train"]:  # x, gate, dy in; y, dx, dgate out; state and its gradient in and out
            return dict(bytes=6 * n * e + 4 * state, flops=25 * n)
        return dict(bytes=3 * n * e + 2 * state, flops=10 * n)
    if case["op"] == "gated":
        m, k, f = case["m"], case["k"], case["f"]
        if case["train"]:
            return dict(bytes=2 * (2 * m * k + 4 * f * k + 2 * m * f), flops=12 * m * k * f)
        return dict(bytes=2 * (m * k + 2 * f * k + m * f), flops=4 * m * k * f)
    m, n, k = case["m"], case["n"], case["k"]
    groups = -(-k // case["group"])
    return dict(bytes=n * (-(-k // 2)) + n * groups * (3 if case["zeros"] else 2) + 2 * m * (k + n), flops=2 * m * n * k)


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, scale=1.0, shift=0.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dtype or torch.float32)

    st = dict(case)
    if case["op"] == "step":
        dt = DTYPES[case["dtype"]]
        b, d = case["b"], case["d"]
        st.update(x=normal(b, d, dtype=dt), gate=normal(b, d, scale=1.5, shift=2.0, dtype=dt), state=normal(b, d))
    elif case["op"] == "recurrence":
        dt = DTYPES[case["dtype"]]
        b, t, d = case["b"], case["t"], case["d"]
        # gates around 2: a memory of ten steps, of a thousand in some channels
        st.update(x=normal(b, t, d, dtype=dt), gate=normal(b, t, d, scale=1.5, shift=2.0, dtype=dt),
                  state=normal(b, d), lengths=None)
        if case["ragged"]:
            lengths = torch.randint(0, t + 1, (b,), generator=gen, device=dev)
            lengths[0] = t
            st["lengths"] = lengths.int()
        if case["train"]:
            st.update(dy=normal(b, t, d, dtype=dt), dfinal=normal(b, d))
    elif case["op"] == "gated":
        dt = DTYPES[case["dtype"]]
        m, k, f = case["m"], case["k"], case["f"]
        st.update(x=normal(m, k, dtype=dt), w_gate=normal(f, k, scale=k ** -0.5, dtype=dt),
                  w_up=normal(f, k, scale=k ** -0.5, dtype=dt))
        if case["train"]:
            st["dh"] = normal(m, f, scale=0.125, dtype=dt)
    else:
        dt = DTYPES[case["dtype"]]
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        st["x"] = normal(m, k, dtype=dt)
        # two weights to a byte, the even column in the low half
        st["qweight"] = torch.randint(0, 256, (n, -(-k // 2)), generator=gen, device=dev, dtype=torch.uint8)
        st["scales"] = ((torch.rand(n, groups, generator=gen, device=dev) + 0.5) * (0.2 / k ** 0.5)).to(dt)
        st["zeros"] = (torch.randint(4, 12, (n, groups), generator=gen, device=dev, dtype=torch.uint8)
                       if case["zeros"] else None)
    return st


# -------------------------------------------------------------- plain form
def _scan(a, b):
    """s_t = a_t s_{t-1} + b_t over dimension 1, with s_0 = 0: composed maps of doubling reach, since a recurrence has
    no form in single torch operations."""
    t, reach = a.shape[1], 1
    while reach < t:
        b = torch.cat([b[:, :reach], torch.addcmul(b[:, reach:], a[:, reach:], b[:, :-reach])], 1)
        if 2 * reach < t:
            a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _valid(st):
    """[batch, time, 1] truth values of the steps that are no padding, or None."""
    if st["lengths"] is None:
        return None
    return (torch.arange(st["t"], device=st["x"].device) < st["lengths"][:, None])[..., None]


def _plain_recurrence(st):
    x, state = st["x"].float(), st["state"]
    i = torch.sigmoid(-st["gate"].float())
    valid = _valid(st)
    if valid is not None:
        i = torch.where(valid, i, 0.0)
    a, b = 1.0 - i, i * x
    b[:, 0] += a[:, 0] * state
    h = _scan(a, b)
    y = h if valid is None else torch.where(valid, h, 0.0)
    out = dict(y=y.to(st["x"].dtype), final=h[:, -1].contiguous())
    if st["train"]:
        dy = st["dy"].float()
        if valid is not None:
            dy = torch.where(valid, dy, 0.0)
        dy = torch.cat([dy[:, :-1], (dy[:, -1] + st["dfinal"])[:, None]], 1)
        follow = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
        lam = _scan(follow, dy.flip(1)).flip(1)
        before = torch.cat([state[:, None], h[:, :-1]], 1)
        out.update(dx=(i * lam).to(st["x"].dtype), dgate=(i * a * lam * (before - x)).to(st["x"].dtype),
                   dstate=a[:, 0] * lam[:, 0])
    return out


def _act(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    if name == "relu":
        return torch.clamp(g, min=0.0)
    return torch.sigmoid(g)


def _act_slope(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return s * (1.0 + g * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    if name == "relu":
        return (g > 0).to(g.dtype)
    s = torch.sigmoid(g)
    return s * (1.0 - s)


def _plain_gated(st):
    dt = st["x"].dtype
    x, wg, wu = st["x"].float(), st["w_gate"].float(), st["w_up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a = _act(st["act"], g)
    out = dict(h=(a * u).to(dt))
    if st["train"]:
        dh = st["dh"].float()
        dg, du = dh * u * _act_slope(st["act"], g), dh * a
        out.update(dx=(dg @ wg + du @ wu).to(dt), dw_gate=(dg.t() @ x).to(dt), dw_up=(du.t() @ x).to(dt))
    return out


def _int4_values(st, dtype):
    q = torch.stack([st["qweight"] & 15, st["qweight"] >> 4], -1).flatten(1)[:, :st["k"]].to(dtype)
    group = torch.arange(st["k"], device=q.device) // st["group"]
    zeros = 8.0 if st["zeros"] is None else st["zeros"].to(dtype)[:, group]
    return (q - zeros) * st["scales"].to(dtype)[:, group]


def _plain_step(st):
    i = torch.sigmoid(-st["gate"].float())
    st["state"] += i * (st["x"].float() - st["state"])
    return dict(y=st["state"].to(st["x"].dtype), state=st["state"])


def run(st):
    if own:
        return _own(st)
    if st["op"] == "step":
        return _plain_step(st)
    if st["op"] == "recurrence":
        return _plain_recurrence(st)
    if st["op"] == "gated":
        return _plain_gated(st)
    return (st["x"].float() @ _int4_values(st, torch.float32).t()).to(st["x"].dtype)


# ----------------------------------------------------- the framework's calls
def _own(st):
    from veles.simd_amd import ops
    if st["op"] == "step":
        return dict(y=ops.gated_recurrence_step(st["x"], st["gate"], st["state"]), state=st["state"])
    if st["op"] == "recurrence":
        if not st["train"]:
            y, final = ops.gated_recurrence(st["x"], st["gate"], st["state"], st["lengths"])
            return dict(y=y, final=final)
        x, gate, state = (st[n].detach().requires_grad_() for n in ("x", "gate", "state"))
        y, final = ops.gated_recurrence(x, gate, state, st["lengths"])
        dx, dgate, dstate = torch.autograd.grad((y, final), (x, gate, state), (st["dy"], st["dfinal"]))
        return dict(y=y.detach(), final=final.detach(), dx=dx, dgate=dgate, dstate=dstate)
    if st["op"] == "gated":
        if not st["train"]:
            return dict(h=ops.gated_linear(st["x"], st["w_gate"], st["w_up"], st["act"]))
        x, wg, wu = (st[n].detach().requires_grad_() for n in ("x", "w_gate", "w_up"))
        h = ops.gated_linear(x, wg, wu, st["act"])
        dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), st["dh"])
        return dict(h=h.detach(), dx=dx, dw_gate=dwg, dw_up=dwu)
    return ops.matvec_int4(st["x"], st["qweight"], st["scales"], st["zeros"], st["group"])


# -------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "step":
        gate, h = st["gate"].double(), st["state"].double()
        keep = 1.0 / (1.0 + torch.exp(-gate))
        h = keep * h + st["x"].double() / (1.0 + torch.exp(gate))
        return dict(y=h, state=h)
    if case["op"] == "recurrence":
        return _exact_recurrence(st)
    if case["op"] == "gated":
        return _exact_gated(st)
    k, x = case["k"], st["x"].double()
    q = torch.zeros(case["n"], 2 * st["qweight"].shape[1], dtype=torch.float64, device=x.device)
    q[:, 0::2] = torch.remainder(st["qweight"], 16).double()
    q[:, 1::2] = torch.div(st["qweight"], 16, rounding_mode="floor").double()
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=x.device)
    for j in range(st["scales"].shape[1]):  # group by group
        at = slice(j * case["group"], min(k, (j + 1) * case["group"]))
        z = 8.0 if st["zeros"] is None else st["zeros"][:, j].double()
        y += (x[:, at] @ q[:, at].t() - x[:, at].sum(1, keepdim=True) * z) * st["scales"][:, j].double()
    return y


def _exact_recurrence(st):
    """Step by step."""
    b, t, d = st["b"], st["t"], st["d"]
    dev = st["x"].device
    length = torch.full((b,), t, device=dev) if st["lengths"] is None else st["lengths"].long()
    h = st["state"].double()
    hs = torch.empty(t + 1, b, d, dtype=torch.float64, device=dev)
    hs[0] = h
    gate, x = st["gate"].transpose(0, 1).contiguous(), st["x"].transpose(0, 1).contiguous()
    for s in range(t):
        g = gate[s].double()
        new = torch.sigmoid(g) * h + torch.sigmoid(-g) * x[s].double()
        h = new if st["lengths"] is None else torch.where((s < length)[:, None], new, h)
        hs[s + 1] = h
    inside = (torch.arange(t, device=dev)[:, None] < length)[..., None]
    out = dict(y=torch.where(inside, hs[1:], 0.0).transpose(0, 1), final=h)
    if st["train"]:
        dy = st["dy"].transpose(0, 1).contiguous()
        dx = torch.zeros(t, b, d, dtype=torch.float64, device=dev)
        dgate = torch.zeros_like(dx)
        back = st["dfinal"].double()
        for s in range(t - 1, -1, -1):
            g = gate[s].double()
            lam = dy[s].double() + back
            keep, take = torch.sigmoid(g), torch.sigmoid(-g)
            dx[s], dgate[s] = take * lam, keep * take * lam * (hs[s] - x[s].double())
            back = keep * lam if st["lengths"] is None else torch.where((s < length)[:, None], keep * lam, back)
        out.update(dx=torch.where(inside, dx, 0.0).transpose(0, 1),
                   dgate=torch.where(inside, dgate, 0.0).transpose(0, 1), dstate=back)
    return out


def _exact_gated(st):
    x, w = st["x"].double(), torch.cat([st["w_gate"], st["w_up"]]).double()
    g, u = torch.matmul(w, x.t()).t().split(st["f"], 1)
    if st["act"] == "gelu":
        phi = torch.special.ndtr(g)
        a, slope = g * phi, phi + g * torch.exp(-g * g / 2.0) / (2.0 * math.pi) ** 0.5
    elif st["act"] == "relu":
        a, slope = torch.where(g > 0, g, 0.0), torch.where(g > 0, 1.0, 0.0)
    else:
        e = torch.exp(-g)
        s = 1.0 / (1.0 + e)
        a, slope = (s, s * s * e) if st["act"] == "sigmoid" else (g * s, s + g * s * s * e)
    out = dict(h=a * u)
    if st["train"]:
        dh = st["dh"].double()
        d = torch.cat([dh * u * slope, dh * a], 1)
        dw = torch.matmul(d.t(), x)
        out.update(dx=torch.matmul(d, w), dw_gate=dw[:st["f"]], dw_up=dw[st["f"]:])
    return out
