"""GPU parity of the sequence-layer operators (csrc/causal_conv.hip, state_scan_*.hip, grad_clip.hip) against the float64
restatements of sequence_ref.py.

Tolerances (sequence_ref.close): half a step of the result's type, plus a count of float32 roundings times 2^-24 of the sums
of magnitudes behind the result.  The counts, worst case, errors adding up linearly:
  convolution          W products and sums, sigmoid and product (10)                       -> 2 W + 32
    dw, db             plus 32 rows in a thread's sum and the partial rows behind it       -> + 64 + B ceil(L / 16)
  scan                 per step 5 (decay: exponent and exponential 3, product and sum 2); the error of delta (softplus: 20)
                       reaches a decay exp(-s) as 22 s <= 22 / e of it; c . h and gate 40   -> 64 + 5 L
    gradients          the same again backwards, sums over channels or rows                 -> 160 + 12 L + B + D / 16
"""

import pytest
import torch

import sequence_ref as ref
from audiofakedetect import ops

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _rnd(g, *shape, scale=1.0, dtype=torch.float32):
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def _conv_inputs(seed, dtype, b, l, d, w, bias=True, state=False, wtype=None):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    wt = t if wtype == "same" else torch.float32
    return dict(x=_rnd(g, b, l, d, dtype=t), w=_rnd(g, d, w, scale=0.5, dtype=wt), b=_rnd(g, d, dtype=wt) if bias else None,
                state=_rnd(g, b, w - 1, d, dtype=t) if state else None)


def _lengths(kind, b, l):
    if kind is None:
        return None
    some = [l, 0, 1, max(1, l // 2), max(0, l - 1), l + 5, -3, 17]
    return torch.tensor([some[i % len(some)] for i in range(b)], dtype=kind, device="cuda")


CONV = [
    # dtype, B, L, D, W, act, bias, state, lengths, taps of x's type
    ("fp32", 1, 1, 1, 2, "none", False, False, None, None),
    ("fp32", 2, 3, 4, 4, "silu", True, True, None, None),
    ("bf16", 3, 17, 8, 4, "silu", True, True, torch.int32, None),
    ("bf16", 8, 33, 24, 3, "none", True, False, torch.int64, "same"),
    ("fp16", 2, 70, 37, 5, "silu", False, True, None, "same"),
    ("fp16", 8, 131, 40, 4, "silu", True, True, torch.int32, None),
    ("fp32", 2, 129, 67, 8, "silu", True, True, torch.int32, None),
    ("fp32", 1, 200, 128, 6, "none", True, False, None, None),
    ("bf16", 2, 65, 264, 7, "silu", True, True, None, None),
    ("bf16", 1, 5, 16, 8, "silu", True, True, None, None),  # fewer rows than taps
    ("bf16", 2, 64, 513, 4, "silu", True, False, None, None),
    ("bf16", 3, 41, 5, 4, "silu", True, True, torch.int32, None),  # narrower than 16 bytes of channels
    ("fp16", 2, 33, 7, 3, "none", True, False, None, "same"),
    ("bf16", 2, 50, 4, 2, "silu", False, True, None, None),
]


@pytest.mark.parametrize("dtype, b, l, d, w, act, bias, state, lens, wtype", CONV)
def test_conv_forward_and_gradients(dtype, b, l, d, w, act, bias, state, lens, wtype):
    t = _conv_inputs(l * 7 + d, dtype, b, l, d, w, bias, state, wtype)
    lengths = _lengths(lens, b, l)
    for v in t.values():
        if v is not None:
            v.requires_grad_(True)
    y, so = ops.causal_conv(t["x"], t["w"], t["b"], act, state=t["state"], lengths=lengths, return_state=True)
    g = torch.Generator().manual_seed(5)
    dy, ds = _rnd(g, b, l, d, dtype=y.dtype), _rnd(g, b, w - 1, d, dtype=y.dtype)
    names = [k for k, v in t.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad((y, so), [t[k] for k in names], (dy, ds))))
    kw = dict(act=act, lengths=lengths, dy=dy, dstate_out=ds)
    want, bound = ref.conv(**t, **kw), ref.conv(**t, **kw, absolute=True)
    k = 2 * w + 32
    ref.close(y, want["y"], bound["y"], k, "y")
    assert torch.equal(so.cpu().double(), want["state"]), "state: a copy of rows"
    rows = 64 + b * ((l + 15) // 16)
    for name in names:
        ref.close(grads[name], want["d" + name], bound["d" + name], k + (rows if name in ("w", "b") else 0), "d" + name)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("d", [1, 37, 64])
@pytest.mark.parametrize("w", [2, 4, 8])
def test_conv_steps_continue_a_prompt(dtype, d, w):
    t = _conv_inputs(3, dtype, 3, 12, d, w, True, True)
    with torch.no_grad():
        y, so = ops.causal_conv(t["x"], t["w"], t["b"], "silu", state=t["state"], return_state=True)
        head, st = ops.causal_conv(t["x"][:, :5], t["w"], t["b"], "silu", state=t["state"], return_state=True)
        assert torch.equal(head, y[:, :5])
        spare = torch.empty_like(st)
        for i in range(5, 12):
            if i % 2:
                yi = ops.causal_conv_step(t["x"][:, i], st, t["w"], t["b"], "silu")
            else:
                yi = ops.causal_conv_step(t["x"][:, i], st, t["w"], t["b"], "silu", state_out=spare)
                st, spare = spare, st
            assert torch.equal(yi, y[:, i]), i  # the same products in the same order
        assert torch.equal(st, so)


def test_conv_padding_is_never_read():
    t = _conv_inputs(9, "bf16", 4, 40, 48, 4, True, False)
    lengths = torch.tensor([40, 0, 3, 21], device="cuda", dtype=torch.int32)
    dirty = t["x"].clone()
    for i, n in enumerate(lengths.tolist()):
        dirty[i, n:] = float("nan") if i % 2 else float("inf")
    outs = []
    for x in (t["x"], dirty):
        x = x.detach().requires_grad_(True)
        y, so = ops.causal_conv(x, t["w"].requires_grad_(True), t["b"], "silu", lengths=lengths, return_state=True)
        dy = torch.ones_like(y)
        for i, n in enumerate(lengths.tolist()):
            dy[i, n:] = float("nan")
        outs.append((y, so, *torch.autograd.grad(y, [x, t["w"]], dy)))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())
    assert not outs[0][0][1].any() and not outs[0][2][2, 3:].any()


def test_conv_strided_and_unaligned_views():
    g = torch.Generator().manual_seed(4)
    both = _rnd(g, 3, 21, 2 * 48 + 1, dtype=torch.bfloat16)
    w, b = _rnd(g, 48, 4), _rnd(g, 48)
    for x in (both[:, :, :48], both[:, :, 49:], both[:, ::2, 1:49], both[:, :, :96:2], both.transpose(0, 1)[:, :, 1:49]):
        y = ops.causal_conv(x, w, b, "silu")
        assert torch.equal(y, ops.causal_conv(x.contiguous(), w, b, "silu"))
        assert y.is_contiguous()
    one = _rnd(g, 1, 1, 48, dtype=torch.bfloat16).expand(3, 20, 48)
    assert torch.equal(ops.causal_conv(one, w, b), ops.causal_conv(one.contiguous(), w, b))
    x = both[:, :, :48].detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.causal_conv(x, w, b).float().sum(), [x])  # an expanded gradient arrives
    (want,) = torch.autograd.grad(ops.causal_conv(x, w, b), [x], torch.ones(3, 21, 48, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(dx, want)


def _scan_inputs(seed, dtype, b, l, d, n, gate=True, skip=True, bias=True, state=True):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    return dict(x=_rnd(g, b, l, d, dtype=t), dt=_rnd(g, b, l, d, scale=0.5, dtype=t),
                a=-(torch.arange(1, n + 1).float() * torch.exp(0.1 * torch.randn(d, n, generator=g))).cuda(),
                b=_rnd(g, b, l, n, dtype=t), c=_rnd(g, b, l, n, dtype=t), d=_rnd(g, d) if skip else None,
                gate=_rnd(g, b, l, d, dtype=t) if gate else None,
                dt_bias=(torch.rand(d, generator=g) * 5 - 6).cuda() if bias else None,
                state=_rnd(g, b, d, n, scale=0.3) if state else None)


SCAN = [
    # dtype, B, L, D, N, lengths, absent inputs
    ("fp32", 1, 1, 1, 1, None, ("gate", "d", "state")),
    ("fp32", 2, 2, 3, 2, None, ()),
    ("fp32", 2, 15, 64, 16, None, ()),
    ("bf16", 3, 16, 65, 16, None, ("state",)),
    ("fp16", 8, 17, 40, 16, torch.int32, ()),
    ("fp32", 8, 37, 67, 13, torch.int64, ("gate",)),
    ("bf16", 2, 33, 130, 4, None, ()),
    ("fp32", 2, 50, 20, 3, torch.int32, ("d", "dt_bias")),
    ("fp16", 2, 33, 66, 8, None, ("state",)),
    ("fp32", 3, 34, 33, 5, torch.int32, ()),
    ("bf16", 2, 35, 40, 32, None, ()),
    ("fp32", 8, 40, 35, 17, torch.int32, ()),
    ("fp32", 2, 33, 20, 64, None, ()),
    ("fp16", 3, 20, 17, 33, torch.int32, ("gate",)),
    # few rows and many blocks of tokens: the time axis is split
    ("fp32", 1, 300, 20, 16, None, ()),
    ("bf16", 2, 517, 70, 16, torch.int32, ()),
    ("fp32", 8, 400, 9, 7, torch.int32, ()),
    ("fp32", 3, 390, 5, 40, torch.int32, ()),
]


@pytest.mark.parametrize("dtype, b, l, d, n, lens, absent", SCAN)
def test_scan_forward_and_gradients(dtype, b, l, d, n, lens, absent):
    t = _scan_inputs(l * 3 + n, dtype, b, l, d, n, **{{"gate": "gate", "d": "skip", "dt_bias": "bias", "state": "state"}[k]: False
                                                  for k in absent})
    softplus = "dt_bias" not in absent
    if not softplus:
        t["dt"] = t["dt"].abs()
    lengths = _lengths(lens, b, l)
    for v in t.values():
        if v is not None:
            v.requires_grad_(True)
    y, so = ops.state_scan(**t, softplus=softplus, lengths=lengths, return_state=True)
    with torch.no_grad():
        assert torch.equal(ops.state_scan(**t, softplus=softplus, lengths=lengths), y), "with and without what training keeps"
    g = torch.Generator().manual_seed(6)
    dy, ds = _rnd(g, b, l, d, dtype=y.dtype), _rnd(g, b, d, n, scale=0.3)
    names = [k for k, v in t.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad((y, so), [t[k] for k in names], (dy, ds))))
    kw = dict(softplus=softplus, lengths=lengths, dy=dy, dstate_out=ds)
    want, bound = ref.scan(**t, **kw), ref.scan(**t, **kw, absolute=True)
    ref.close(y, want["y"], bound["y"], 64 + 5 * l, "y")
    ref.close(so, want["state"], bound["state"], 64 + 5 * l, "state")
    for name in names:
        ref.close(grads[name], want["d" + name], bound["d" + name], 160 + 12 * l + b + d / 16, "d" + name)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 4, 7, 8, 16, 24, 64])
def test_scan_steps_continue_a_prompt(dtype, n):
    t = _scan_inputs(n, dtype, 3, 9, 70, n)
    par = {k: t[k] for k in ("a", "d", "dt_bias")}
    seq = ("x", "dt", "b", "c", "gate")
    with torch.no_grad():
        y, so = ops.state_scan(**t, softplus=True, return_state=True)
        _, st = ops.state_scan(**{k: t[k][:, :4] for k in seq}, **par, softplus=True, state=t["state"], return_state=True)
        spare = torch.empty_like(st)
        for i in range(4, 9):
            one = {k: t[k][:, i] for k in seq}
            if i % 2:
                yi = ops.state_scan_step(state=st, **one, **par, softplus=True)
            else:
                yi = ops.state_scan_step(state=st, **one, **par, softplus=True, state_out=spare)
                st, spare = spare, st
            kw = dict(softplus=True)
            want = ref.scan(**{k: t[k][:, :i + 1] for k in seq}, **par, state=t["state"], **kw)
            bound = ref.scan(**{k: t[k][:, :i + 1] for k in seq}, **par, state=t["state"], **kw, absolute=True)
            ref.close(yi, want["y"][:, i], bound["y"][:, i], 64 + 5 * i, f"y at {i}")
        want, bound = ref.scan(**t, softplus=True), ref.scan(**t, softplus=True, absolute=True)
        ref.close(st, want["state"], bound["state"], 64 + 45, "state by steps")
        ref.close(so, want["state"], bound["state"], 64 + 45, "state of the prompt")


def test_scan_step_takes_unaligned_states_and_strided_rows():
    t = _scan_inputs(2, "bf16", 3, 4, 20, 16)
    flat = torch.empty(3 * 20 * 16 + 3, device="cuda")
    par = {k: t[k] for k in ("a", "d", "dt_bias")}
    one = {k: t[k][:, 2] for k in ("x", "dt", "b", "c", "gate")}  # rows of a longer sequence: batch strides
    for off in (0, 1, 2):
        st = flat[off:off + 960].view(3, 20, 16)
        st.copy_(t["state"])
        y = ops.state_scan_step(state=st, **one, **par, softplus=True)
        other = t["state"].clone()
        want = ops.state_scan_step(state=other, **{k: v.contiguous() for k, v in one.items()}, **par, softplus=True)
        assert torch.equal(y, want) and torch.equal(st, other)


@pytest.mark.parametrize("dtype, b, d, n", [("fp32", 700, 200, 16), ("bf16", 2050, 33, 13), ("fp16", 1031, 130, 32),
                                            ("bf16", 2049, 64, 8), ("fp32", 2051, 20, 64), ("fp16", 2050, 65, 4)])
def test_scan_step_of_many_rows(dtype, b, d, n):
    """Batches large enough to be taken four rows at a time, with rows left over."""
    t = _scan_inputs(b, dtype, b, 1, d, n)
    one = {k: t[k][:, 0] for k in ("x", "dt", "b", "c", "gate")}
    par = {k: t[k] for k in ("a", "d", "dt_bias")}
    st = t["state"].clone()
    y = ops.state_scan_step(state=st, **one, **par, softplus=True)
    want, bound = ref.scan(**t, softplus=True), ref.scan(**t, softplus=True, absolute=True)
    ref.close(y, want["y"][:, 0], bound["y"][:, 0], 64 + 5, "y")
    ref.close(st, want["state"], bound["state"], 64 + 5, "state")


@pytest.mark.parametrize("l, d", [(40, 48), (400, 10)])
def test_scan_padding_is_never_read(l, d):
    t = _scan_inputs(11, "bf16", 4, l, d, 16)
    lens = [l, 0, 1, l // 2 + 3]
    lengths = torch.tensor(lens, device="cuda", dtype=torch.int32)
    dirty = dict(t)
    for k in ("x", "dt", "b", "c", "gate"):
        dirty[k] = t[k].clone()
        for i, n in enumerate(lens):
            dirty[k][i, n:] = float("nan") if i % 2 else float("inf")
    outs = []
    for v in (t, dirty):
        v = {k: x.detach().requires_grad_(True) for k, x in v.items()}
        y, so = ops.state_scan(**v, softplus=True, lengths=lengths, return_state=True)
        dy = torch.ones_like(y)
        for i, n in enumerate(lens):
            dy[i, n:] = float("nan")
        outs.append((y, so, *torch.autograd.grad((y, so), list(v.values()), (dy, torch.ones_like(so)))))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())
    assert torch.equal(outs[0][1][1], t["state"][1]), "an empty sequence leaves its state"


def test_scan_decays_to_zero_and_stays_finite():
    """Steps so wide that every decay underflows, and none at all: exp(-inf) = 0 and exp(0) = 1, no NaN either way."""
    t = _scan_inputs(12, "fp32", 2, 40, 33, 16)
    for dt in (1e4, 0.0):
        v = dict(t, dt=torch.full_like(t["dt"], dt), dt_bias=None)
        v = {k: x if x is None else x.detach().requires_grad_(True) for k, x in v.items()}
        y, so = ops.state_scan(**v, return_state=True)
        grads = torch.autograd.grad(y.sum() + so.sum(), [x for x in v.values() if x is not None])
        assert all(bool(torch.isfinite(g).all()) for g in (y, so, *grads))
        want = ref.scan(**v)
        bound = ref.scan(**v, absolute=True)
        ref.close(y, want["y"], bound["y"], 64 + 200, f"dt {dt}")
        if dt == 0.0:
            assert torch.equal(so, t["state"])


def test_scan_strided_views_and_expanded_rows():
    g = torch.Generator().manual_seed(8)
    d, n, r = 40, 16, 3
    proj = _rnd(g, 2, 35, 2 * d, dtype=torch.bfloat16)            # x | gate, as one projection leaves them
    bcd = _rnd(g, 2, 35, r + 2 * n, dtype=torch.bfloat16)         # low-rank dt | b | c
    t = _scan_inputs(8, "bf16", 2, 35, d, n)
    v = dict(t, x=proj[..., :d], gate=proj[..., d:], b=bcd[..., r:r + n], c=bcd[..., r + n:], dt=t["dt"][:1, :1].expand(2, 35, d))
    y, so = ops.state_scan(**v, softplus=True, return_state=True)
    w = {k: x.contiguous() for k, x in v.items()}
    y2, so2 = ops.state_scan(**w, softplus=True, return_state=True)
    assert torch.equal(y, y2) and torch.equal(so, so2)
    swapped = proj[..., :d].transpose(0, 1).contiguous().transpose(0, 1)  # time-major memory
    assert torch.equal(ops.state_scan(**dict(v, x=swapped), softplus=True), y)
    v["x"] = v["x"].transpose(1, 2).contiguous().transpose(1, 2)  # channels not contiguous: copied
    assert torch.equal(ops.state_scan(**v, softplus=True), y)
    x = proj.detach().requires_grad_(True)
    (dp,) = torch.autograd.grad(ops.state_scan(**dict(v, x=x[..., :d], gate=x[..., d:]), softplus=True).float().sum(), [x])
    parts = {k: w[k].detach().requires_grad_(True) for k in ("x", "gate")}
    dx, dg = torch.autograd.grad(ops.state_scan(**dict(w, **parts), softplus=True).float().sum(), list(parts.values()))
    assert torch.equal(dp, torch.cat([dx, dg], -1))


def test_scan_rows_far_apart_in_memory():
    """Rows farther apart than the lanes' 32-bit offsets reach."""
    t = _scan_inputs(9, "bf16", 1, 40, 24, 4)
    want = ops.state_scan(**t, softplus=True)
    far = torch.empty(40 * ((1 << 24) + 8), dtype=torch.bfloat16, device="cuda")
    x = far.as_strided((1, 40, 24), (0, (1 << 24) + 8, 1))
    x.copy_(t["x"])
    assert torch.equal(ops.state_scan(**dict(t, x=x), softplus=True), want)
    near = far.as_strided((1, 40, 24), (0, 1 << 24, 1))
    near.copy_(t["x"])
    assert torch.equal(ops.state_scan(**dict(t, x=near), softplus=True), want)
    # ... and a gradient like that
    v = t["x"].requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.state_scan(**t, softplus=True), [v], torch.ones_like(want))
    x.fill_(1.0)
    (dx2,) = torch.autograd.grad(ops.state_scan(**t, softplus=True), [v], x)
    assert torch.equal(dx, dx2)


def test_second_derivatives_are_refused():
    t = _scan_inputs(11, "fp32", 1, 4, 6, 4)
    c = _conv_inputs(11, "fp32", 1, 4, 6, 3)
    x = t["x"].detach().requires_grad_(True)
    for y in (ops.state_scan(**dict(t, x=x), softplus=True), ops.causal_conv(x, c["w"], c["b"], "silu"),
              ops.linear(x, torch.ones(5, 6, device="cuda"), activation="silu")):
        dy = torch.ones_like(y, requires_grad=True)
        (dx,) = torch.autograd.grad(y, [x], dy, create_graph=True)
        assert torch.equal(dx, torch.autograd.grad(y, [x], dy)[0])
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()


def test_a_state_that_a_backward_pass_needs_is_not_changed_unseen():
    t = _scan_inputs(10, "fp32", 2, 5, 8, 4)
    c = _conv_inputs(10, "fp32", 2, 5, 8, 4, True, True)
    x = t["x"].detach().requires_grad_(True)
    state, cstate = t["state"].clone(), c["state"].clone()
    ys = ops.state_scan(**dict(t, x=x, state=state), softplus=True), ops.causal_conv(x, c["w"], c["b"], "silu", state=cstate)
    with torch.no_grad():
        ops.state_scan_step(t["x"][:, 0], state, t["dt"][:, 0], t["a"], t["b"][:, 0], t["c"][:, 0])
        ops.causal_conv_step(t["x"][:, 0], torch.empty_like(cstate), c["w"], state_out=cstate)
    for y in ys:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), [x])
    p = torch.ones(5, device="cuda")
    before = p._version
    ops.clip_gradients([p], 1.0)
    assert p._version > before


def test_gradients_flow_through_the_state_between_parts():
    """Two parts joined by their state have the gradients of the whole, for both operators."""
    t = _scan_inputs(13, "fp32", 2, 50, 21, 6)
    c = _conv_inputs(13, "fp32", 2, 50, 21, 4, True, True)
    v = {k: x.requires_grad_(True) for k, x in t.items()}
    seq = ("x", "dt", "b", "c", "gate")
    dy = torch.randn(2, 50, 21, generator=torch.Generator().manual_seed(1)).cuda()
    par = {k: v[k] for k in ("a", "d", "dt_bias")}
    y1, st = ops.state_scan(**{k: v[k][:, :23] for k in seq}, **par, softplus=True, state=v["state"], return_state=True)
    y2 = ops.state_scan(**{k: v[k][:, 23:] for k in seq}, **par, softplus=True, state=st)
    got = dict(zip(v, torch.autograd.grad(torch.cat([y1, y2], 1), list(v.values()), dy)))
    want, bound = ref.scan(**v, softplus=True, dy=dy), ref.scan(**v, softplus=True, dy=dy, absolute=True)
    for k in v:
        ref.close(got[k], want["d" + k], bound["d" + k], 160 + 12 * 50 + 4, "d" + k)
    u = {k: x.requires_grad_(True) for k, x in c.items()}
    y1, st = ops.causal_conv(u["x"][:, :2], u["w"], u["b"], "silu", state=u["state"], return_state=True)
    y2 = ops.causal_conv(u["x"][:, 2:], u["w"], u["b"], "silu", state=st)
    got = dict(zip(u, torch.autograd.grad(torch.cat([y1, y2], 1), list(u.values()), dy)))
    want, bound = ref.conv(**u, act="silu", dy=dy), ref.conv(**u, act="silu", dy=dy, absolute=True)
    for k in u:
        ref.close(got[k], want["d" + k], bound["d" + k], 40 + 64 + 4, "d" + k)


def test_same_bits_every_time():
    t = _scan_inputs(14, "bf16", 2, 600, 80, 16)
    v = {k: x.requires_grad_(True) for k, x in t.items()}
    c = _conv_inputs(14, "bf16", 2, 600, 80, 4)
    u = {k: c[k].requires_grad_(True) for k in ("x", "w", "b")}
    runs = []
    for _ in range(3):
        y = ops.state_scan(**v, softplus=True)
        z = ops.causal_conv(**u, activation="silu")
        runs.append([y, *torch.autograd.grad(y, list(v.values()), torch.ones_like(y)),
                     z, *torch.autograd.grad(z, list(u.values()), torch.ones_like(z))])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


@pytest.mark.parametrize("b, l, d", [(0, 5, 6), (2, 0, 6), (2, 5, 0)])
def test_empty_batches_sequences_and_channels(b, l, d):
    t = {k: x.requires_grad_(True) for k, x in _scan_inputs(1, "fp32", b, l, d, 4).items()}
    y, so = ops.state_scan(**t, softplus=True, return_state=True)
    assert y.shape == (b, l, d) and torch.equal(so, t["state"]) if l == 0 else so.shape == (b, d, 4)
    grads = torch.autograd.grad((y, so), list(t.values()), (torch.zeros_like(y), torch.ones_like(so)))
    assert all(g.shape == x.shape for g, x in zip(grads, t.values()))
    if l == 0:
        assert bool((grads[list(t).index("state")] == 1).all())
    c = {k: x.requires_grad_(True) for k, x in _conv_inputs(1, "fp32", b, l, d, 4, True, True).items()}
    y, so = ops.causal_conv(c["x"], c["w"], c["b"], state=c["state"], return_state=True)
    assert y.shape == (b, l, d) and so.shape == (b, 3, d)
    grads = torch.autograd.grad((y, so), list(c.values()), (torch.zeros_like(y), torch.ones_like(so)))
    assert all(g.shape == x.shape for g, x in zip(grads, c.values()))
    if l != 0:
        with torch.no_grad():
            assert ops.causal_conv_step(c["x"][:, 0], c["state"], c["w"], c["b"]).shape == (b, d)


def test_offsets_past_32_bits():
    """More than 2^31 elements: the rows at the far end equal a short call that starts from the state in front of them."""
    l, d, tail = 70000, 32768, 40
    x = torch.empty(1, l, d, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(0))
    g = torch.Generator().manual_seed(3)
    w, bias = _rnd(g, d, 3), _rnd(g, d)
    with torch.no_grad():
        y = ops.causal_conv(x, w, bias, "silu")
        short = ops.causal_conv(x[:, -tail:], w, bias, "silu", state=x[:, -tail - 2:-tail].contiguous())
        assert torch.equal(y[:, -tail:], short)
        del y
        a = -torch.ones(d, 1, device="cuda")
        b, c = _rnd(g, 1, l, 1, dtype=torch.bfloat16), _rnd(g, 1, l, 1, dtype=torch.bfloat16)
        y, so = ops.state_scan(x, x, a, b, c, softplus=True, return_state=True)
        # decays of at least exp(-softplus(x)): 400 tokens in front decide the state to far below a rounding
        cut = 440
        s2, _ = ops.state_scan(x[:, -cut:], x[:, -cut:], a, b[:, -cut:], c[:, -cut:], softplus=True, return_state=True)
        diff = (y[:, -tail:].float() - s2[:, -tail:].float()).abs().max()
        assert float(diff) <= 2.0 ** -7 * float(s2.float().abs().max())
        assert bool((so != 0).any())


# ---- norm and clipping -------------------------------------------------------------------------------------------------
def _grads(seed, dtypes=("fp32", "bf16", "fp16"), count=40):
    g = torch.Generator().manual_seed(seed)
    sizes = [1, 2, 3, 7, 8, 15, 63, 1000, 16383, 16384, 16385, 40000, 100003]
    return [_rnd(g, sizes[i % len(sizes)], scale=10.0 ** (-(i % 4)), dtype=TYPES[dtypes[i % len(dtypes)]]) for i in range(count)]


def _norm64(ts, kind=2.0):
    flat = torch.cat([t.detach().cpu().double().reshape(-1) for t in ts])
    return float(torch.linalg.vector_norm(flat, kind))


@pytest.mark.parametrize("count", [1, 13, 40, 128, 129, 300])
@pytest.mark.parametrize("kind", [2.0, float("inf")])
def test_global_norm(count, kind):
    ts = _grads(count, count=count)
    got, want = float(ops.global_norm(ts, kind)), _norm64(ts, kind)
    assert abs(got - want) <= 2.0 ** -23 * want  # summed in float64, rounded once (plus the reference's own)


def test_global_norm_far_values_views_and_order():
    big = torch.full((1000,), 1e30, device="cuda")      # squares beyond float32
    small = torch.full((1000,), 1e-30, device="cuda")   # squares below it
    for t in (big, small):
        assert abs(float(ops.global_norm([t])) - _norm64([t])) <= 2.0 ** -23 * _norm64([t])
    base = torch.randn(5003, generator=torch.Generator().manual_seed(0)).cuda()
    views = [base[1:], base[:5000].view(50, 100).t(), base[:5000].view(50, 100)[:, 3:50], base[::3], base[:1].expand(77),
             base.bfloat16()[3:], base.half()[1:2]]
    for v in views:
        assert abs(float(ops.global_norm([v])) - _norm64([v])) <= 2.0 ** -23 * _norm64([v])
    assert float(ops.global_norm([torch.zeros(0, device="cuda")])) == 0.0
    assert float(ops.global_norm([torch.zeros(0, device="cuda"), torch.tensor(-3.0, device="cuda")])) == 3.0
    for bad in (float("nan"), float("inf")):
        for at in (0, 700, 5002):
            t = base.clone()
            t[at] = bad
            for kind in (2.0, float("inf")):
                got = float(ops.global_norm([base, t, base], kind))
                assert got != got if bad != bad else got == bad


@pytest.mark.parametrize("count", [1, 40, 97, 300])
@pytest.mark.parametrize("share", [0.25, 1.5])
@pytest.mark.parametrize("where", ["in place", "out"])
def test_clip_gradients(count, share, where):
    ts = _grads(count + 1, count=count)
    before = [t.clone() for t in ts]
    norm = _norm64(ts)
    if where == "out":
        out = [torch.full_like(t, 7.0) for t in ts]
        got = ops.clip_gradients(ts, share * norm, out=out)
        assert all(torch.equal(a, b) for a, b in zip(ts, before)), "inputs are left alone"
    else:
        out = ts
        got = ops.clip_gradients(ts, share * norm)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    f = min(1.0, share * norm / (norm + 1e-6))
    for o, b in zip(out, before):
        if share > 1:
            assert torch.equal(o, b)
        else:
            want = b.cpu().double() * f
            ref.close(o, want, want, 2, "scaled")  # the factor (rounded to float32) and the product


def test_clip_gradients_of_views_and_odd_places():
    base = torch.randn(20000, generator=torch.Generator().manual_seed(2)).cuda()
    for make in (lambda t: [t[1:9000], t[9000:]], lambda t: [t.view(100, 200).t()], lambda t: [t.view(100, 200)[:, 3:77]],
                 lambda t: [t[::2]], lambda t: [t[:1], t[1:2], t[2:2]]):
        t = base.clone()
        views = make(t)
        want = [v.clone().double() * (0.5 * _norm64(views) / (_norm64(views) + 1e-6)) for v in views]
        rest = base.clone()
        ops.clip_gradients(views, 0.5 * _norm64(views))
        for v, w in zip(views, want):
            ref.close(v, w.cpu(), w.cpu(), 2, "view")
            v.copy_(make(rest)[[i for i, u in enumerate(views) if u is v][0]])
        assert torch.equal(t, base), "nothing outside the views was touched"
    src, dst = base[1:10001], torch.zeros(10004, device="cuda")  # source and destination differ in alignment
    for off in (0, 1, 2, 3):
        ops.clip_gradients([src], 0.5, out=[dst[off:off + 10000]])
        want = src.cpu().double() * (0.5 / (_norm64([src]) + 1e-6))
        ref.close(dst[off:off + 10000], want, want, 2, f"offset {off}")
    with pytest.raises(ValueError):
        ops.clip_gradients([base[:100], base[50:150]], 1.0)
    t = base.clone()
    t[5] = float("nan")
    ops.clip_gradients([t], 1.0)
    assert bool(torch.isnan(t).all())
    t = base.clone()
    t[5] = float("inf")
    ops.clip_gradients([t], 1.0)
    assert not t[:5].any() and not t[6:].any()


def test_norm_and_clip_past_32_bits():
    n = (1 << 31) + 12345
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[-1], t[1 << 31], t[0] = 3.0, 4.0, 12.0
    assert float(ops.global_norm([t])) == 13.0
    assert float(ops.clip_gradients([t], 6.5)) == 13.0
    assert [float(t[i]) for i in (-1, 1 << 31, 0)] == [1.5, 2.0, 6.0]


def test_fused_adam_clips_as_clip_then_step():
    shapes = [(64, 1, 3, 3), (64,), (1,), (96, 64, 3, 3), (2, 320), (2,)]
    g = torch.Generator().manual_seed(9)
    p0 = [torch.randn(s, generator=g) for s in shapes]
    mine = [torch.nn.Parameter(p.clone().cuda()) for p in p0]
    theirs = [torch.nn.Parameter(p.clone().double()) for p in p0]
    opt = ops.FusedAdam(mine, lr=1e-2, weight_decay=1e-3)
    other = torch.optim.Adam(theirs, lr=1e-2, weight_decay=1e-3)
    for step in range(4):
        opt.zero_grad()
        scale = 0.5
        for p, q in zip(mine, theirs):
            grad = torch.randn(p.shape, generator=g) * 10.0 ** (step - 2)
            p.grad, q.grad = grad.cuda(), grad.double() * scale
        norm = torch.nn.utils.clip_grad_norm_(theirs, 3.0)
        other.step()
        opt.step(grad_scale=scale, max_grad_norm=3.0)
        assert abs(float(opt.last_grad_norm) - float(norm)) <= 2.0 ** -22 * float(norm)
        for p, q in zip(mine, theirs):
            # an update is at most lr; its relative error: two dozen float32 roundings
            assert float((p.detach().cpu().double() - q.detach()).abs().max()) <= (step + 1) * 1e-2 * 2e-5 + 2.0 ** -22 * float(q.detach().abs().max())


# ---- streams and graphs ------------------------------------------------------------------------------------------------
def test_on_another_stream():
    t = _scan_inputs(20, "bf16", 2, 500, 64, 16)
    want = ops.state_scan(**t, softplus=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.state_scan(**t, softplus=True)
        n = ops.global_norm([got])
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and float(n) == float(ops.global_norm([want]))


def test_two_streams_at_once_keep_apart():
    ts = [_scan_inputs(30 + i, "bf16", 1, 800, 40, 16) for i in range(2)]
    vs = [{k: x.requires_grad_(True) for k, x in t.items()} for t in ts]

    def both(v):
        y = ops.state_scan(**v, softplus=True)
        return [y, *torch.autograd.grad(y, list(v.values()), torch.ones_like(y))]

    want = [both(v) for v in vs]
    streams = [torch.cuda.Stream() for _ in vs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = both(vs[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def _capture(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_steps_in_a_graph_replay_with_new_inputs():
    t = _scan_inputs(21, "bf16", 4, 6, 70, 16)
    c = _conv_inputs(21, "bf16", 4, 6, 70, 4, True, True)
    par = {k: t[k] for k in ("a", "d", "dt_bias")}
    seq = ("dt", "b", "c", "gate")
    live = {k: t[k][:, 0].clone() for k in seq + ("x",)}
    cst, sst = c["state"].clone(), t["state"].clone()

    def step():
        x = ops.causal_conv_step(live["x"], cst, c["w"], c["b"], "silu")
        return ops.state_scan_step(x, sst, live["dt"], par["a"], live["b"], live["c"], d=par["d"], gate=live["gate"],
                                   dt_bias=par["dt_bias"], softplus=True)

    graph, y = _capture(step)
    cst.copy_(c["state"])
    sst.copy_(t["state"])
    ec, es = c["state"].clone(), t["state"].clone()
    for i in range(6):
        for k in live:
            live[k].copy_(t[k][:, i])
        graph.replay()
        torch.cuda.synchronize()
        x = ops.causal_conv_step(t["x"][:, i], ec, c["w"], c["b"], "silu")
        want = ops.state_scan_step(x, es, t["dt"][:, i], par["a"], t["b"][:, i], t["c"][:, i], d=par["d"],
                                   gate=t["gate"][:, i], dt_bias=par["dt_bias"], softplus=True)
        assert torch.equal(y, want) and torch.equal(cst, ec) and torch.equal(sst, es), i


def test_two_training_passes_and_a_clip_in_graphs():
    """Two captured graphs, replayed in turn with eager work in between: neither disturbs the other's workspace."""
    def build(seed):
        t = {k: x.requires_grad_(True) for k, x in _scan_inputs(seed, "bf16", 1, 640, 48, 16).items()}
        c = {k: x.requires_grad_(True) for k, x in _conv_inputs(seed, "bf16", 1, 640, 48, 4).items() if x is not None}
        leaves = [*t.values(), *c.values()]
        dy = torch.ones(1, 640, 48, dtype=torch.bfloat16, device="cuda")
        outs = [torch.empty_like(x) for x in leaves]

        def run():
            y = ops.state_scan(**dict(t, x=ops.causal_conv(c["x"], c["w"], c["b"], "silu") + t["x"]), softplus=True)
            grads = torch.autograd.grad(y, leaves, dy)
            norm = ops.clip_gradients(grads, 1.0, out=outs)
            return [y.detach(), norm, *outs]

        return leaves, run

    built = [build(s) for s in (40, 41)]
    graphs = [_capture(run) for _, run in built]
    for turn in range(4):
        for (leaves, run), (graph, outs) in zip(built, graphs):
            with torch.no_grad():
                leaves[0].mul_(1.25 if turn % 2 else 0.75)
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in outs]
            for o in outs[2:]:
                o.zero_()
            want = [o.clone() for o in run()]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_prompts_in_a_graph_with_changing_lengths():
    """Ragged prompts whose time axis is split, and projections of a few and of many rows: every replay is the eager result."""
    t = _scan_inputs(43, "bf16", 3, 700, 40, 16)
    c = _conv_inputs(43, "bf16", 3, 700, 40, 4, True, True)
    g = torch.Generator().manual_seed(43)
    w, b = _rnd(g, 40, 40, scale=0.2, dtype=torch.bfloat16), _rnd(g, 40)
    lengths = torch.tensor([700, 1, 0], device="cuda")

    def run():
        h, cs = ops.causal_conv(ops.linear(c["x"], w, b), c["w"], c["b"], "silu", state=c["state"], lengths=lengths,
                                return_state=True)
        y, ss = ops.state_scan(**dict(t, x=h), softplus=True, lengths=lengths, return_state=True)
        return [y, cs, ss, ops.linear(y[:, 0], w, b, "gelu")]

    graph, outs = _capture(run)
    for turn in range(4):
        lengths.copy_(torch.tensor([[700, 1, 0], [0, 699, 128], [16, 700, 700], [5, 129, 640]][turn]))
        c["x"].mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, e) for a, e in zip(got, run())), turn
        torch.cuda.synchronize()


def test_projections_on_two_streams_at_once():
    g = torch.Generator().manual_seed(44)
    sets = [[_rnd(g, m, 264, dtype=torch.bfloat16).requires_grad_(True), _rnd(g, 130, 264, dtype=torch.bfloat16).requires_grad_(True),
             _rnd(g, 130).requires_grad_(True)] for m in (9, 2000)]

    def both(v):
        y = ops.linear(*v, "silu")
        return [y, *torch.autograd.grad(y, v, torch.ones_like(y))]

    want = [both(v) for v in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = both(sets[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---- the operators together --------------------------------------------------------------------------------------------
def _layer(t, c, x, lengths=None, states=(None, None)):
    h, cs = ops.causal_conv(x, c["w"], c["b"], "silu", state=states[0], lengths=lengths, return_state=True)
    y, ss = ops.state_scan(h, t["dt"], t["a"], t["b"], t["c"], d=t["d"], gate=t["gate"], dt_bias=t["dt_bias"], softplus=True,
                           state=states[1], lengths=lengths, return_state=True)
    return y, (cs, ss)


def test_a_training_step_of_a_sequence_head():
    """Convolution -> scan -> mean classifier -> loss -> backward -> clip inside Adam, against the formulas in float64."""
    b, l, d, n = 4, 37, 24, 16
    t = _scan_inputs(50, "fp32", b, l, d, n, state=False)
    c = _conv_inputs(50, "fp32", b, l, d, 4)
    g = torch.Generator().manual_seed(51)
    wl, bl = _rnd(g, 2, d, scale=0.3), _rnd(g, 2)
    params = {k: torch.nn.Parameter(v.clone()) for k, v in
              dict(w=c["w"], cb=c["b"], a=t["a"], d=t["d"], dt_bias=t["dt_bias"], wl=wl, bl=bl).items()}
    labels = torch.tensor([0, 1, 1, 0], device="cuda")
    lengths = torch.tensor([37, 20, 1, 36], device="cuda")
    opt = ops.FusedAdam(params.values(), lr=1e-2)
    opt.zero_grad()
    y, _ = _layer(dict(t, a=params["a"], d=params["d"], dt_bias=params["dt_bias"]), dict(w=params["w"], b=params["cb"]),
                  c["x"], lengths)
    logits = ops.linear_mean(y, params["wl"], params["bl"])
    loss = ops.CrossEntropyLoss()(logits, labels)
    loss.backward()
    got = {k: p.grad.detach().clone() for k, p in params.items()}
    opt.step(max_grad_norm=0.1)
    # the same in float64
    hc = ref.conv(c["x"], c["w"], c["b"], act="silu", lengths=lengths)["y"]
    kw = dict(softplus=True, lengths=lengths)
    y64 = ref.scan(hc, t["dt"], t["a"], t["b"], t["c"], t["d"], t["gate"], t["dt_bias"], **kw)["y"]
    wl64, bl64 = wl.cpu().double(), bl.cpu().double()
    lo = (y64 @ wl64.t() + bl64).mean(1)
    p = torch.softmax(lo, -1)
    dlo = (p - torch.nn.functional.one_hot(labels.cpu(), 2).double()) / b
    assert abs(float(loss) + float(torch.log_softmax(lo, -1)[torch.arange(b), labels.cpu()].mean())) <= 1e-5
    dy = (dlo @ wl64)[:, None, :].expand(b, l, d) / l
    gs = ref.scan(hc, t["dt"], t["a"], t["b"], t["c"], t["d"], t["gate"], t["dt_bias"], dy=dy, **kw)
    gc = ref.conv(c["x"], c["w"], c["b"], act="silu", lengths=lengths, dy=gs["dx"])
    want = dict(w=gc["dw"], cb=gc["db"], a=gs["da"], d=gs["dd"], dt_bias=gs["ddt_bias"],
                wl=dlo.t() @ y64.mean(1), bl=dlo.sum(0))
    for k, v in want.items():
        scale = float(v.abs().max())
        # chains of a few hundred float32 roundings (37 steps, twice), errors adding up: 1000 x 2^-24 of the largest value
        assert float((got[k].cpu().double() - v).abs().max()) <= 1000 * 2.0 ** -24 * scale + 1e-9, k
    norm = float(torch.sqrt(sum(v.square().sum() for v in want.values())))
    assert abs(float(opt.last_grad_norm) - norm) <= 1000 * 2.0 ** -24 * norm
    assert all(bool(torch.isfinite(p).all()) for p in params.values())


def test_a_recording_scored_as_it_arrives():
    """A ragged batch of prompts with their states, then frame by frame: what the whole recordings give."""
    b, l, d, n = 3, 30, 40, 16
    t = _scan_inputs(60, "fp32", b, l, d, n, state=False)
    c = _conv_inputs(60, "fp32", b, l, d, 4)
    starts = [12, 5, 0]
    with torch.no_grad():
        whole, _ = _layer(t, c, c["x"])
        y, (cs, ss) = _layer(t, c, c["x"], lengths=torch.tensor(starts, device="cuda"))
        for i, s in enumerate(starts):
            assert torch.equal(y[i, :s], whole[i, :s])
        for k in range(18):
            at = [s + k for s in starts]

            def rows(v):
                return torch.stack([v[i, p] for i, p in enumerate(at)])

            h = ops.causal_conv_step(rows(c["x"]), cs, c["w"], c["b"], "silu")
            yk = ops.state_scan_step(h, ss, rows(t["dt"]), t["a"], rows(t["b"]), rows(t["c"]), d=t["d"], gate=rows(t["gate"]),
                                     dt_bias=t["dt_bias"], softplus=True)
            want = rows(whole)
            # the same steps in another kernel: sums of 16 products in another order, 30 tokens of decay
            assert float((yk - want).abs().max()) <= (64 + 5 * 30) * 2.0 ** -23 * float(whole.abs().max())


# ---- projections -------------------------------------------------------------------------------------------------------
LINEAR = [
    # dtype, M, K, N, act, bias, residual
    ("fp32", 1, 1, 1, "none", None, False),
    ("fp32", 3, 5, 7, "silu", "fp32", True),
    ("fp32", 33, 64, 128, "gelu", "fp32", False),
    ("fp32", 130, 100, 257, "relu", "fp32", True),
    ("fp32", 200, 1031, 90, "silu", None, False),
    ("bf16", 1, 64, 64, "gelu", "fp32", True),
    ("bf16", 17, 8, 300, "silu", "same", False),
    ("bf16", 129, 264, 136, "none", "fp32", True),
    ("bf16", 300, 1000, 131, "gelu", "fp32", True),
    ("bf16", 5, 2048, 520, "silu", "fp32", False),   # few rows: the k axis is split
    ("bf16", 256, 4096, 128, "none", None, True),
    ("fp16", 31, 33, 65, "gelu", "same", False),
    ("fp16", 140, 513, 250, "relu", "fp32", True),
    ("fp16", 64, 72, 1000, "silu", None, False),
    ("fp16", 1000, 16, 16, "none", "same", False),
    ("bf16", 2050, 1024, 1030, "silu", "fp32", True),  # 256 x 256 tiles, ragged in both directions
    ("fp16", 4100, 520, 2056, "gelu", "fp32", False),
    ("fp32", 2000, 260, 130, "gelu", "fp32", True),
    ("bf16", 1, 2048, 2048, "silu", "fp32", True),     # few rows: whole slabs, tails inside a slab and inside a batch, splits
    ("bf16", 16, 1000, 515, "gelu", "same", False),
    ("fp16", 17, 264, 33, "none", None, True),
    ("bf16", 32, 4104, 8200, "relu", "fp32", False),   # ... 32 columns at a time
    ("fp32", 5, 36, 1, "silu", "fp32", False),
    ("fp32", 16, 9000, 40, "none", "fp32", False),
    ("fp32", 31, 2052, 2100, "gelu", None, True),      # ... 32 x 128 tiles
    ("bf16", 3330, 130, 2050, "silu", "same", True),   # 128 x 128 tiles, the gradients' k long enough to be split
    ("fp16", 1700, 1024, 2000, "gelu", "fp32", False), # 128 x 64
    ("fp32", 1700, 96, 2000, "silu", "fp32", True),
    ("bf16", 40, 36, 700, "none", "fp32", True),       # 64 x 64
    ("bf16", 33, 9001, 65, "silu", "fp32", True),      # ... split, rows copied
]


@pytest.mark.parametrize("dtype, m, k, n, act, bias, residual", LINEAR)
def test_linear_forward_and_gradients(dtype, m, k, n, act, bias, residual):
    """y: K products and sums, then 10 (erf 4 ulp of a value up to 2, slope 1.13); a partial tile per split is one of the
    sums.  In front of the products behind dx and dw, dz is rounded to the type: half a step of its magnitude, which enters
    them like any other error; b's gradient is a sum of what was not rounded."""
    g = torch.Generator().manual_seed(m + k + n)
    t = TYPES[dtype]
    v = dict(x=_rnd(g, m, k, dtype=t), w=_rnd(g, n, k, scale=k ** -0.5, dtype=t),
             b=None if bias is None else _rnd(g, n, dtype=t if bias == "same" else torch.float32),
             residual=_rnd(g, m, n, dtype=t) if residual else None)
    if act == "relu":  # no pre-activation within its rounding errors of the corner
        z = ref.linear(v["x"], v["w"], v["b"])["z"]
        near = (z.abs() < 1e-3).any(1)
        v["x"][near.cuda()] = 0
        if bias is None:
            v["x"][near.cuda()] = 0
    for x in v.values():
        if x is not None:
            x.requires_grad_(True)
    y = ops.linear(v["x"], v["w"], v["b"], act, residual=v["residual"])
    with torch.no_grad():
        assert torch.equal(ops.linear(v["x"], v["w"], v["b"], act, residual=v["residual"]), y)
    dy = _rnd(g, m, n, dtype=t)
    names = [key for key, x in v.items() if x is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [v[key] for key in names], dy)))
    want, bound = ref.linear(**v, act=act, dy=dy), ref.linear(**v, act=act, dy=dy, absolute=True)
    ref.close(y, want["y"], bound["y"], k + 10, "y")
    half = ref.HALF_STEP[t]
    dz_err = half * want["dz"].abs()
    xa, wa = v["x"].detach().cpu().double().abs(), v["w"].detach().cpu().double().abs()
    extra = {"x": dz_err @ wa, "w": dz_err.t() @ xa, "b": 0, "residual": 0}
    for name in names:
        r = dy.cpu().double() if name == "residual" else want["d" + name]
        lim = r.abs() if name == "residual" else bound["d" + name]
        e = torch.as_tensor(extra[name])
        # (close()'s bound in units of 2^-24: the rounding of dz is added to it)
        ref.close(grads[name], r, lim * (m + n + k + 20) + e * 2.0 ** 24, 1, "d" + name)


def test_linear_views_leading_axes_and_unaligned_rows():
    g = torch.Generator().manual_seed(77)
    for t in (torch.bfloat16, torch.float32):
        big, wide = _rnd(g, 4, 9, 2 * 72 + 1, dtype=t), _rnd(g, 50, 80, dtype=t)
        w, b = wide[:, 5:77], _rnd(g, 50)
        for x in (big[..., :72], big[..., 1:73], big[..., 73:], big[:, ::2, :72], big.transpose(0, 1)[..., :72],
                  big[..., :144:2]):
            res = _rnd(g, *x.shape[:-1], 2 * 50, dtype=t)[..., 50:]
            got = ops.linear(x, w, b, "silu", residual=res)
            assert torch.equal(got, ops.linear(x.contiguous(), w.contiguous(), b, "silu", residual=res.contiguous()))
            assert got.shape == (*x.shape[:-1], 50)
        one = ops.linear(big[0, 0, :72], w, b)
        assert one.shape == (50,) and torch.equal(one, ops.linear(big[:1, 0, :72], w, b)[0])
        x = big[..., :72].detach().requires_grad_(True)
        y = ops.linear(x, w, b, "gelu")
        (dx,) = torch.autograd.grad(y.float().sum(), [x])  # an expanded gradient
        (dx2,) = torch.autograd.grad(ops.linear(x, w, b, "gelu"), [x], torch.ones_like(y))
        assert torch.equal(dx, dx2)
    empty = torch.zeros(0, 72, device="cuda", requires_grad=True)
    w = torch.randn(5, 72, device="cuda", requires_grad=True)
    y = ops.linear(empty, w, torch.zeros(5, device="cuda"), "silu")
    dx, dw = torch.autograd.grad(y.sum(), [empty, w])
    assert y.shape == (0, 5) and dx.shape == (0, 72) and not dw.any()


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_linear_gradients_wanted_one_by_one(act, dtype):
    """A frozen weight, a first layer, a bias alone: the same gradients, without the others' work."""
    g = torch.Generator().manual_seed(79)
    for k in (64, 37):
        v = dict(x=_rnd(g, 70, k, dtype=TYPES[dtype]), w=_rnd(g, 48, k, dtype=TYPES[dtype]), b=_rnd(g, 48),
                 residual=_rnd(g, 70, 48, dtype=TYPES[dtype]))
        dy = _rnd(g, 70, 48, dtype=TYPES[dtype])

        def grads(names):
            t = {key: x.detach().requires_grad_(key in names) for key, x in v.items()}
            y = ops.linear(t["x"], t["w"], t["b"], act, residual=t["residual"])
            return torch.autograd.grad(y, [t[key] for key in names], dy)

        every = dict(zip(v, grads(list(v))))
        for names in (["x"], ["w"], ["b"], ["residual"], ["x", "b"], ["w", "b"], ["x", "w"]):
            assert all(torch.equal(got, every[key]) for key, got in zip(names, grads(names))), names


def test_linear_rows_do_not_leak_into_each_other():
    """A row of NaN or inf in x spoils its own row of y alone, and what lies behind a view's rows is never read."""
    g = torch.Generator().manual_seed(78)
    for t, k in ((torch.bfloat16, 100), (torch.float32, 66), (torch.float16, 128)):
        x, w = _rnd(g, 150, k, dtype=t), _rnd(g, 140, k, dtype=t)
        clean = ops.linear(x, w)
        dirty = x.clone()
        dirty[70], dirty[71] = float("nan"), float("inf")
        y = ops.linear(dirty, w)
        keep = [i for i in range(150) if i not in (70, 71)]
        assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[70]).all())
        wide = torch.full((150, k + 24), float("nan"), dtype=t, device="cuda")
        wide[:, :k] = x
        assert torch.equal(ops.linear(wide[:, :k], w), clean)
        # a column of w's gradient sums over rows: a zero gradient times an infinite input is not zero, as ever
        v = x.clone().requires_grad_(True)
        dy = torch.zeros_like(clean)
        dy[3] = 1
        (dx,) = torch.autograd.grad(ops.linear(v, w), [v], dy)
        assert not dx[:3].any() and not dx[4:].any() and dx[3].any()


def test_linear_extremes_of_fp16_keep_their_slopes():
    x = torch.tensor([[300.0], [-300.0], [2.0 ** -20], [-2.0 ** -20]], device="cuda", dtype=torch.float16, requires_grad=True)
    w = torch.tensor([[300.0], [2.0 ** -20]], device="cuda", dtype=torch.float16)
    for act in ("relu", "silu", "gelu"):
        y = ops.linear(x, w, None, act)
        (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
        assert bool(torch.isfinite(dx).all()), act
        if act == "relu":  # 90000 and 2^-40 are positive, their negatives are not
            want = torch.tensor([[300.0], [0.0], [300.0], [0.0]], device="cuda").half()
            assert torch.equal(dx, want)
    for act, want in (("relu", 0.0), ("none", float("-inf"))):
        z = ops.linear(torch.full((1, 1), float("-inf"), device="cuda"), torch.ones(1, 1, device="cuda"), None, act)
        assert float(z) == want


def test_linear_same_bits_every_time_and_in_a_graph():
    g = torch.Generator().manual_seed(79)
    x, w, b = (_rnd(g, *s, dtype=torch.bfloat16).requires_grad_(True) for s in ((70, 2048), (96, 2048), (96,)))
    dy = _rnd(g, 70, 96, dtype=torch.bfloat16)

    def run():
        y = ops.linear(x, w, b, "gelu")
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]

    first = [t.clone() for t in run()]
    assert all(torch.equal(a, c) for a, c in zip(first, run()))
    graph, outs = _capture(run)
    for turn in range(3):
        with torch.no_grad():
            x.mul_(0.5)
        want = [t.clone() for t in run()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want)), turn


def test_linear_past_32_bits():
    """Rows behind 2^31 elements of x and of y equal a shorter call's (of enough rows that its k axis is not split either:
    a split sums in another order)."""
    m, k, n = 2200000, 1000, 1000
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    w = _rnd(torch.Generator().manual_seed(2), n, k, scale=0.03, dtype=torch.bfloat16)
    y = ops.linear(x, w, None, "silu")
    assert torch.equal(y[-40000:], ops.linear(x[-40000:], w, None, "silu"))
    assert torch.equal(y[:40001], ops.linear(x[:40001], w, None, "silu"))


def _silu64(v):
    return v * torch.sigmoid(v)


def _layer64(x, p, rank, n):
    """The layer of the next test in float64 torch operations, for autograd on the CPU."""
    b, l, _ = x.shape
    d = p["conv"].shape[0]
    z = x @ p["w_in"].t() + p["b_in"]
    u, gate = z[..., :d], z[..., d:]
    taps = p["conv"].shape[1]
    full = torch.cat([torch.zeros(b, taps - 1, d, dtype=x.dtype), u], 1)
    h = _silu64(sum(full[:, j:j + l] * p["conv"][:, j] for j in range(taps)) + p["conv_b"])
    s = h @ p["w_x"].t()
    dt, bb, cc = s[..., :rank] @ p["w_dt"].t(), s[..., rank:rank + n], s[..., rank + n:]
    delta = torch.nn.functional.softplus(dt + p["dt_bias"])
    state, rows = torch.zeros(b, d, n, dtype=x.dtype), []
    for t in range(l):
        state = torch.exp(delta[:, t, :, None] * p["a"]) * state + (delta[:, t] * h[:, t])[:, :, None] * bb[:, t, None, :]
        rows.append((state * cc[:, t, None, :]).sum(-1))
    y = (torch.stack(rows, 1) + p["d"] * h) * _silu64(gate)
    return y @ p["w_out"].t() + p["b_out"] + x


def test_a_whole_state_space_layer_trains():
    """Projection in -> convolution -> projections to the scan's inputs -> scan with gate -> projection out onto the residual,
    as views of each other's results, with its loss, all gradients, and the clipped step."""
    b, l, k, d, n, rank = 3, 29, 24, 40, 16, 4
    g = torch.Generator().manual_seed(90)
    shapes = dict(w_in=(2 * d, k), b_in=(2 * d,), conv=(d, 4), conv_b=(d,), w_x=(rank + 2 * n, d), w_dt=(d, rank), a=(d, n),
                  d=(d,), dt_bias=(d,), w_out=(k, d), b_out=(k,))
    p = {name: torch.nn.Parameter(_rnd(g, *s, scale=0.3)) for name, s in shapes.items()}
    with torch.no_grad():
        p["a"].copy_(-torch.arange(1, n + 1, device="cuda").float().expand(d, n))
        p["dt_bias"].sub_(2)
    x = _rnd(g, b, l, k).requires_grad_(True)
    wl, labels = _rnd(g, 2, k, scale=0.3), torch.tensor([0, 1, 1], device="cuda")
    opt = ops.FusedAdam(p.values(), lr=1e-2)
    opt.zero_grad()
    z = ops.linear(x, p["w_in"], p["b_in"])
    u, gate = z[..., :d], z[..., d:]
    h = ops.causal_conv(u, p["conv"], p["conv_b"], "silu")
    s = ops.linear(h, p["w_x"])
    dt = ops.linear(s[..., :rank], p["w_dt"])
    y = ops.state_scan(h, dt, p["a"], s[..., rank:rank + n], s[..., rank + n:], d=p["d"], gate=gate, dt_bias=p["dt_bias"],
                       softplus=True)
    out = ops.linear(y, p["w_out"], p["b_out"], residual=x)
    loss = ops.CrossEntropyLoss()(ops.linear_mean(out, wl, torch.zeros(2, device="cuda")), labels)
    loss.backward()
    got = {name: q.grad.detach().clone() for name, q in p.items()}
    got["x"] = x.grad.clone()
    q = {name: v.detach().cpu().double().requires_grad_(True) for name, v in p.items()}
    x64 = x.detach().cpu().double().requires_grad_(True)
    out64 = _layer64(x64, q, rank, n)
    loss64 = torch.nn.functional.cross_entropy((out64 @ wl.cpu().double().t()).mean(1), labels.cpu())
    loss64.backward()
    # a chain of half a dozen operators of at most a few hundred roundings each, forward and back: 4000 x 2^-24 of the
    # largest value
    tol = 4000 * 2.0 ** -24
    assert float((out.detach().cpu().double() - out64.detach()).abs().max()) <= tol * float(out64.detach().abs().max())
    for name, v in got.items():
        want = (x64 if name == "x" else q[name]).grad
        assert float((v.cpu().double() - want).abs().max()) <= tol * float(want.abs().max()), name
    before = {name: v.detach().clone() for name, v in p.items()}
    opt.step(max_grad_norm=0.05)
    norm = float(torch.sqrt(sum(v.grad.square().sum() for v in q.values())))
    assert abs(float(opt.last_grad_norm) - norm) <= tol * norm
    assert all(not torch.equal(before[name], v) for name, v in p.items())


def test_a_whole_layer_in_bf16_one_frame_at_a_time():
    """The same layer's serving form: a prompt, then single frames through the step forms, against the whole sequence."""
    b, l, k, d, n = 4, 20, 32, 64, 16
    g = torch.Generator().manual_seed(91)
    t = torch.bfloat16
    w_in, w_x, w_out = _rnd(g, 2 * d, k, scale=0.2, dtype=t), _rnd(g, d + 2 * n, d, scale=0.2, dtype=t), _rnd(g, k, d, scale=0.2, dtype=t)
    conv, conv_b = _rnd(g, d, 4, scale=0.4), _rnd(g, d, scale=0.1)
    par = dict(a=-torch.rand(d, n, generator=g).cuda() * 4, d=_rnd(g, d), dt_bias=_rnd(g, d) - 2)
    x = _rnd(g, b, l, k, dtype=t)

    def layer(x, conv_f, scan_f):
        z = ops.linear(x, w_in)
        h = conv_f(z[..., :d])
        s = ops.linear(h, w_x)
        return ops.linear(scan_f(h, s, z[..., d:]), w_out, residual=x)

    def scan_args(h, s, gate):
        return dict(x=h, dt=s[..., :d], b=s[..., d:d + n], c=s[..., d + n:], gate=gate, softplus=True, **par)

    with torch.no_grad():
        whole = layer(x, lambda u: ops.causal_conv(u, conv, conv_b, "silu"), lambda *a: ops.state_scan(**scan_args(*a)))
        states = {}

        def conv_prompt(u):
            y, states["c"] = ops.causal_conv(u, conv, conv_b, "silu", return_state=True)
            return y

        def scan_prompt(*a):
            y, states["s"] = ops.state_scan(**scan_args(*a), return_state=True)
            return y

        layer(x[:, :11], conv_prompt, scan_prompt)
        for i in range(11, l):
            y = layer(x[:, i], lambda u: ops.causal_conv_step(u, states["c"], conv, conv_b, "silu"),
                      lambda *a: ops.state_scan_step(state=states["s"], **scan_args(*a)))
            # sums in other orders (the few rows' products split k): a bf16 step apart at most at each of four roundings
            assert float((y.float() - whole[:, i].float()).abs().max()) <= 4 * 2.0 ** -7 * float(whole.float().abs().max())


@pytest.mark.parametrize("kind", ["fused", "torch"])
def test_trainer_clips_its_gradients(kind):
    import os
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if root not in sys.path:
        sys.path.insert(0, root)
    import bench

    torch.manual_seed(0)
    args, trainer, _ = bench.build("sym5-l8", 4, False, torch.device("cuda", 0))
    trainer.train_data_loader = None
    params = [p for p in trainer.model.parameters() if p.requires_grad]
    if kind == "torch":
        trainer.optimizer = torch.optim.SGD(params, lr=1.0)
    g = torch.Generator().manual_seed(4)
    batch = {"audio": 0.1 * torch.randn(4, 1, 22050, generator=g), "label": torch.tensor([0, 1, 1, 0])}
    trainer.model.train()
    trainer._run_batch(0, batch)  # without the flag: no norm is taken
    assert kind == "torch" or trainer.optimizer.last_grad_norm is None
    args.clip_grad_norm = 1e-3
    before = [p.detach().clone() for p in params]
    trainer._run_batch(0, batch)
    if kind == "fused":
        # the arena holds the gradients as the backward left them
        want = _norm64([trainer.optimizer.flat_grad])
        assert abs(float(trainer.optimizer.last_grad_norm) - want) <= 2.0 ** -22 * want and want > 1e-3
    else:
        # plain descent at a rate of 1 moves by the clipped gradients; each parameter's difference is off by its rounding
        moved = _norm64([b - p for b, p in zip(before, params)])
        noise = 2.0 ** -23 * _norm64(before)
        assert abs(moved - 1e-3) <= 1e-3 * 1e-3 + noise


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradients_of_views_under_saved_tensor_hooks(dtype):
    """x | gate and dt | b | c as views of two projections: the gradients are the same bits whether the saved tensors stay
    where they are, go to the host and back, or come back in another layout."""
    g = torch.Generator().manual_seed(80)
    t = TYPES[dtype]
    d, n, l = 40, 16, 35
    xz, dbc = _rnd(g, 2, l, 2 * d, dtype=t).requires_grad_(True), _rnd(g, 2, l, d + 2 * n, dtype=t).requires_grad_(True)
    a, skip, bias = -_rnd(g, d, n).abs(), _rnd(g, d), _rnd(g, d)
    taps, wide = _rnd(g, d, 4, scale=0.5), _rnd(g, 24, 2 * d, dtype=t)
    leaves = [xz, dbc, *(p.requires_grad_(True) for p in (a, skip, bias, taps, wide))]
    dys = [_rnd(g, 2, l, k, dtype=t) for k in (d, d, 24)]

    def run():
        x, gate = xz.chunk(2, -1)
        dt, b, c = dbc.split([d, n, n], -1)
        ys = (ops.state_scan(x, dt, a, b, c, d=skip, gate=gate, dt_bias=bias, softplus=True),
              ops.causal_conv(x, taps, None, "silu"), ops.linear(gate, wide[:, 8:8 + d], None, "gelu"))
        return lambda: torch.autograd.grad(ys, leaves, dys)

    want = run()()

    def turned(v):
        return v.transpose(-1, -2).contiguous().transpose(-1, -2) if v.dim() > 1 else v.clone()

    for hooks in (torch.autograd.graph.save_on_cpu(pin_memory=True),
                  torch.autograd.graph.saved_tensors_hooks(lambda v: v.clone(memory_format=torch.contiguous_format), lambda v: v),
                  torch.autograd.graph.saved_tensors_hooks(turned, lambda v: v)):
        with hooks:
            backward = run()
        got = backward()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), hooks


def test_scan_rows_at_the_edge_of_the_lanes_offsets():
    """fp32 rows exactly 2^24 elements apart, where 16 rows fill the 32-bit offsets, as inputs and as a gradient; and a single
    frame whose row stride is beyond them and never used."""
    t = _scan_inputs(81, "fp32", 1, 40, 24, 4)
    v = t["x"].detach().requires_grad_(True)
    want = ops.state_scan(**dict(t, x=v), softplus=True)
    (dx,) = torch.autograd.grad(want, [v], torch.ones_like(want))
    edge = torch.empty(40 << 24, device="cuda").as_strided((1, 40, 24), (0, 1 << 24, 1))
    edge.copy_(t["x"])
    x = edge.detach().requires_grad_(True)
    y = ops.state_scan(**dict(t, x=x), softplus=True)
    assert torch.equal(y, want)
    ones = torch.empty(40 << 24, device="cuda").as_strided((1, 40, 24), (0, 1 << 24, 1)).fill_(1.0)
    (dx2,) = torch.autograd.grad(y, [x], ones)
    assert torch.equal(dx, dx2)
    first = {k: u[:, :1] if u.dim() == 3 and k != "state" else u for k, u in t.items()}
    far = torch.empty((1 << 25) + 24, device="cuda").as_strided((1, 1, 24), (24, 1 << 25, 1))
    far.copy_(first["x"])
    x = far.detach().requires_grad_(True)
    y = ops.state_scan(**dict(first, x=x), softplus=True)
    assert torch.equal(y, want[:, :1])
    (dx2,) = torch.autograd.grad(y, [x], torch.ones_like(far))
    u = first["x"].detach().clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.state_scan(**dict(first, x=u), softplus=True), [u], torch.ones_like(y))
    assert torch.equal(dx, dx2)


@pytest.mark.parametrize("batch", [1, 256])  # the time axis in four segments, and in one piece
def test_scan_decays_that_leave_the_range_over_a_segment(batch):
    """Over 128 tokens a decay leaves float32's range in both directions while the states stay inside it: zeros that would
    grow by 2^184 stay zeros, a state of 1e30 that fades by 2^-160 is still there.  The count of the roundings is that of any
    scan of this length."""
    l, d, n = 512, 8, 4
    g = torch.Generator().manual_seed(82)
    t = dict(x=torch.zeros(1, l, d), dt=torch.ones(1, l, d), a=torch.ones(d, n), b=torch.rand(1, l, n, generator=g) + 0.5,
             c=torch.rand(1, l, n, generator=g) + 0.5)
    t["x"][:, 500:] = torch.randn(1, 12, d, generator=g)
    dy = torch.zeros(1, l, d)
    dy[:, :12] = torch.randn(1, 12, d, generator=g)

    def check(t, dy, names, **kw):
        v = {k: (u.expand(batch, *u.shape[1:]) if u.dim() == 3 else u).cuda().requires_grad_(True) for k, u in t.items()}
        y = ops.state_scan(**v, **kw)
        got = dict(zip(names, torch.autograd.grad(y, [v[k] for k in names], dy.expand(batch, l, d).cuda())))
        want, bound = ref.scan(**t, dy=dy, **kw), ref.scan(**t, dy=dy, absolute=True, **kw)
        for i in {0, batch - 1}:
            ref.close(y[i:i + 1], want["y"], bound["y"], 64 + 5 * l, "y")
            for k in names:
                ref.close(got[k][i:i + 1], want["d" + k], bound["d" + k], 160 + 12 * l + 1, "d" + k)
        return y

    check(t, dy, ["x", "dt", "b", "c"])
    fade = dict(t, x=torch.zeros(1, l, d), dt=torch.full((1, l, d), 0.87), a=-torch.ones(d, n),
                state=1e30 * (1 + torch.rand(1, d, n, generator=g)))
    dy = torch.zeros(1, l, d)
    dy[:, 140] = 1e20
    y = check(fade, dy, ["c", "state"])
    y = y.detach()[0, 140]
    assert 1e-25 < float(y.min()) and float(y.max()) < 1e-15
    late = torch.zeros(1, l, d)
    late[:, 300] = 1e30  # 2^100, 2^-117 by the time it has crossed the segment in front of its own
    check(fade, late, ["x"])


def test_clip_gradients_out_may_be_a_gradient_with_gaps():
    """`out` in place where an entry is the gradient itself, gaps or not, beside entries that are not."""
    base = torch.randn(50, 7, generator=torch.Generator().manual_seed(3)).cuda()
    for view in (lambda t: t[:, :3], lambda t: t[::2], lambda t: t.t()[1:4], lambda t: t):
        t, other = base.clone(), torch.randn(33, generator=torch.Generator().manual_seed(4)).cuda()
        kept, far = other.clone(), torch.zeros(33, device="cuda")
        g = view(t)
        want = t.clone()
        version = g._version
        norm = ops.clip_gradients([view(want), kept.clone()], 0.5)
        got = ops.clip_gradients([g, other], 0.5, out=[g, far])
        assert torch.equal(got, norm) and torch.equal(t, want) and torch.equal(other, kept) and g._version > version
        factor = 0.5 / (float(norm) + 1e-6)
        ref.close(far, kept.cpu().double() * factor, kept.cpu().double(), 4, "beside it")


def test_timing_classes_add_like_to_like():
    """"sequence" sums bytes, "linear" flops (issued: with the tiles' padding) and the bytes of its tensors."""
    from audiofakedetect import _native

    x = torch.ones(1, 70, 40, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w, taps = torch.ones(30, 40, device="cuda", dtype=torch.bfloat16).requires_grad_(True), torch.ones(40, 4, device="cuda")
    few = torch.ones(9, 40, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    _native.timing_reset()
    _native.timing_enable(True)
    try:
        with torch.no_grad():
            ops.causal_conv(x, taps)
            ops.linear(few, w)
        y = ops.linear(x, w, None, "silu")
        torch.autograd.grad(y, [x, w], torch.ones_like(y))
        torch.cuda.synchronize()
        seq, lin = _native.timing_collect("sequence"), _native.timing_collect("linear")
    finally:
        _native.timing_enable(False)
        _native.timing_reset()
    assert seq["launches"] == 1 and seq["work"] == seq["bytes"] == 2 * 2 * 70 * 40 and seq["issued"] == 0
    assert lin["launches"] == 3 and lin["work"] == 2.0 * 30 * 40 * (9 + 3 * 70)
    # 16 x 32 x 64 for the few rows; 64 x 64 tiles forward and for dx, 128 x 64 x 64; dw has few rows again, 32 x 48 x 128
    assert lin["issued"] == 2.0 * (16 * 32 * 64 + 2 * 128 * 64 * 64 + 32 * 48 * 128)
    xs, ws, ys = 70 * 40, 30 * 40, 70 * 30
    assert lin["bytes"] == 2.0 * (9 * 40 + ws + 9 * 30) + 2.0 * (xs + ws + ys) + 4.0 * ys + 2.0 * (ys + 2 * (xs + ws)) + 4.0 * ys


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_gelu_tails_are_right_to_the_types_last_bit(dtype):
    """GELU of a negative z is z times a tail that falls to 1e-32 over the range: relative to that value the result is off by
    its rounding, half a step, and by what float32 leaves in front of it -- 2e-6 (fit and polynomial), and the exponent's three
    roundings, 1.5 z^2 2^-24.  The slope is a difference of two such terms, Phi + z pdf, and its error is theirs."""
    t = TYPES[dtype]
    z = torch.cat([torch.linspace(-12, 9, 4001), torch.linspace(-6, -3, 3000)]).to(t)
    x = z[:, None].cuda().requires_grad_(True)
    w = torch.ones(1, 1, dtype=t, device="cuda")
    y = ops.linear(x, w, None, "gelu")
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    z = z.double()[:, None]
    cdf, pdf = 0.5 * torch.erfc(-z * 0.5 ** 0.5), torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
    inexact = 2e-6 + 1.5 * z * z * 2.0 ** -24
    least = 2.0 ** -25 if dtype == "fp16" else 0.0  # half of the smallest number
    half = ref.HALF_STEP[t]
    for got, want, terms in ((y, z * cdf, (z * cdf).abs()), (dx, cdf + z * pdf, cdf + (z * pdf).abs())):
        tol = half * want.abs() + inexact * terms * (1 + half) + least
        over = (got.detach().cpu().double() - want).abs() - tol
        i = int(over.argmax())
        assert float(over.max()) <= 0, (float(z[i]), float(got[i]), float(want[i]))
    assert dtype == "fp16" or bool(y[:100].detach().any())


def test_parameter_gradients_of_more_columns_than_a_launch_holds():
    """2^28 columns of partial sums and more: 1024 threads for each 64 of them would be 2^32.  One row: every gradient is a
    single product, the same bits as torch's."""
    d = (1 << 28) // 3 + 101
    g = torch.Generator("cuda").manual_seed(83)
    x, dy = (torch.empty(1, 1, d, device="cuda").normal_(generator=g) for _ in range(2))
    w = torch.ones(d, 2, device="cuda", requires_grad=True)
    b = torch.zeros(d, device="cuda", requires_grad=True)
    y = ops.causal_conv(x, w, b)
    assert torch.equal(y.detach(), x)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    assert torch.equal(db, dy[0, 0]) and torch.equal(dw[:, 1], (dy * x)[0, 0]) and not dw[:, 0].any()


@pytest.mark.parametrize("dtype, m, k, n, act, bias, residual", [
    ("bf16", 32, 4104, 8200, "relu", "fp32", False),  # few rows, 32 columns at a time: whole slabs, a k tail, a column tail
    ("bf16", 19, 4104, 8200, "silu", "same", True),
    ("fp16", 32, 2048, 8192, "none", None, False),
    ("fp16", 25, 1000, 16421, "gelu", "fp32", True),  # ... k not split, rows copied
    ("fp16", 140, 513, 250, "relu", "fp32", True),
    ("fp32", 130, 100, 257, "relu", "fp32", True),
])
def test_linear_on_inputs_as_they_are(dtype, m, k, n, act, bias, residual):
    """As test_linear_forward_and_gradients, of x as it is drawn: where z is within its rounding errors of relu's corner, the
    gradient that comes in is zero instead.  (y is continuous there.)  Tolerances are those of that test."""
    g = torch.Generator().manual_seed(m + k + n)
    t = TYPES[dtype]
    v = dict(x=_rnd(g, m, k, dtype=t), w=_rnd(g, n, k, scale=k ** -0.5, dtype=t),
             b=None if bias is None else _rnd(g, n, dtype=t if bias == "same" else torch.float32),
             residual=_rnd(g, m, n, dtype=t) if residual else None)
    dy = _rnd(g, m, n, dtype=t)
    if act == "relu":
        near = ref.linear(v["x"], v["w"], v["b"])["z"].abs() < 1e-3
        assert float(near.double().mean()) < 0.01
        dy[near.cuda()] = 0
    for x in v.values():
        if x is not None:
            x.requires_grad_(True)
    y = ops.linear(v["x"], v["w"], v["b"], act, residual=v["residual"])
    with torch.no_grad():
        assert torch.equal(ops.linear(v["x"], v["w"], v["b"], act, residual=v["residual"]), y)
    names = [key for key, x in v.items() if x is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [v[key] for key in names], dy)))
    want, bound = ref.linear(**v, act=act, dy=dy), ref.linear(**v, act=act, dy=dy, absolute=True)
    ref.close(y, want["y"], bound["y"], k + 10, "y")
    dz_err = ref.HALF_STEP[t] * want["dz"].abs()
    xa, wa = v["x"].detach().cpu().double().abs(), v["w"].detach().cpu().double().abs()
    extra = {"x": dz_err @ wa, "w": dz_err.t() @ xa, "b": 0}
    for name in names:
        if name == "residual":
            assert torch.equal(grads[name], dy)
        else:
            e = torch.as_tensor(extra[name])
            ref.close(grads[name], want["d" + name], bound["d" + name] * (m + n + k + 20) + e * 2.0 ** 24, 1, "d" + name)


@pytest.mark.parametrize("l, d", [(13, 5), (400, 70)])  # in one piece, and in time segments
def test_scan_of_states_that_forget_at_once(l, d):
    """a = -inf (minus the exponential of a large logarithm): every token clears the state, as with any finite a far below.
    Padding and the lanes behind the last channel, which hold their state by a step of zero, stay what they are."""
    t = _scan_inputs(84, "fp32", 2, l, d, 6)
    lengths = torch.tensor([l - 3, l], device="cuda")
    far = dict(t, a=t["a"].clone())
    far["a"][0, 1], far["a"][d - 1] = -1e30, -1e30
    outs = []
    for a in (far["a"], torch.where(far["a"] < -1e29, torch.full_like(far["a"], -float("inf")), far["a"])):
        v = {k: u.detach().requires_grad_(True) for k, u in dict(far, a=a).items()}
        y, state = ops.state_scan(**v, softplus=True, lengths=lengths, return_state=True)
        grads = torch.autograd.grad([y, state], list(v.values()), [torch.ones_like(y), torch.ones_like(state)])
        outs.append([y.detach(), state.detach(), *grads])
    for got, want in zip(*outs):
        assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


def test_conv_padding_has_zero_gradients_whatever_the_taps_are():
    t = _conv_inputs(85, "bf16", 3, 50, 24, 4)
    lengths = torch.tensor([50, 33, 0], device="cuda")
    x, w = t["x"].requires_grad_(True), t["w"].clone()
    w[3, 1], w[7, 0] = float("inf"), float("nan")
    dy = torch.ones(3, 50, 24, device="cuda", dtype=torch.bfloat16)
    (dx,) = torch.autograd.grad(ops.causal_conv(x, w, t["b"], lengths=lengths), [x], dy)
    assert not dx[1, 33:].any() and not dx[2].any()
    (want,) = torch.autograd.grad(ops.causal_conv(x, t["w"], t["b"], lengths=lengths), [x], dy)
    keep = [i for i in range(24) if i not in (3, 7)]
    assert torch.equal(dx[..., keep], want[..., keep])
