"""Argument checks of the sequence-layer entry points (no GPU needed: every refusal comes before the first launch)."""

import pytest
import torch

from audiofakedetect import _native, ops


def _conv(**kw):
    args = dict(x=torch.zeros(2, 5, 6), w=torch.zeros(6, 4), b=torch.zeros(6))
    args.update(kw)
    return args


def _scan(**kw):
    args = dict(x=torch.zeros(2, 5, 6), dt=torch.zeros(2, 5, 6), a=torch.zeros(6, 4), b=torch.zeros(2, 5, 4),
                c=torch.zeros(2, 5, 4))
    args.update(kw)
    return args


@pytest.mark.parametrize("kw, err", [
    (dict(x=torch.zeros(5, 6)), ValueError),
    (dict(x=torch.zeros(2, 5, 6, dtype=torch.float64)), TypeError),
    (dict(x=[1.0]), TypeError),
    (dict(w=torch.zeros(7, 4)), ValueError),
    (dict(w=torch.zeros(6, 1)), ValueError),
    (dict(w=torch.zeros(6, 9)), ValueError),
    (dict(w=torch.zeros(6, 4, dtype=torch.bfloat16), b=None), TypeError),  # neither float32 nor the type of x
    (dict(w=None), TypeError),
    (dict(b=torch.zeros(5)), ValueError),
    (dict(b=torch.zeros(6, dtype=torch.float16)), TypeError),
    (dict(activation="gelu"), ValueError),
    (dict(state=torch.zeros(2, 4, 6)), ValueError),
    (dict(state=torch.zeros(2, 3, 6, dtype=torch.bfloat16)), TypeError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(lengths=torch.zeros(2)), TypeError),
    (dict(lengths=[1, 2]), TypeError),
    (dict(), RuntimeError),  # fine, but on the CPU
])
def test_causal_conv_refuses(kw, err):
    with pytest.raises(err):
        ops.causal_conv(**_conv(**kw))


@pytest.mark.parametrize("kw, err", [
    (dict(x=torch.zeros(2, 5, 6)), ValueError),
    (dict(state=None), TypeError),
    (dict(state=torch.zeros(2, 2, 6)), ValueError),
    (dict(state=torch.zeros(2, 6, 3).transpose(1, 2)), ValueError),
    (dict(state_out=torch.zeros(2, 4, 6)), ValueError),
    (dict(x=torch.zeros(2, 6, requires_grad=True)), RuntimeError),
    (dict(), RuntimeError),
])
def test_causal_conv_step_refuses(kw, err):
    args = dict(x=torch.zeros(2, 6), state=torch.zeros(2, 3, 6), w=torch.zeros(6, 4))
    args.update(kw)
    with pytest.raises(err):
        ops.causal_conv_step(**args)


@pytest.mark.parametrize("kw, err", [
    (dict(dt=torch.zeros(2, 5, 7)), ValueError),
    (dict(dt=None), TypeError),
    (dict(dt=torch.zeros(2, 5, 6, dtype=torch.bfloat16)), TypeError),
    (dict(a=torch.zeros(5, 4)), ValueError),
    (dict(a=torch.zeros(6, 0), b=torch.zeros(2, 5, 0), c=torch.zeros(2, 5, 0)), ValueError),
    (dict(a=torch.zeros(6, 65), b=torch.zeros(2, 5, 65), c=torch.zeros(2, 5, 65)), ValueError),
    (dict(a=torch.zeros(6, 4, dtype=torch.bfloat16)), TypeError),
    (dict(b=torch.zeros(2, 5, 3)), ValueError),
    (dict(c=torch.zeros(2, 4, 4)), ValueError),
    (dict(d=torch.zeros(7)), ValueError),
    (dict(gate=torch.zeros(2, 5, 5)), ValueError),
    (dict(dt_bias=torch.zeros(6, dtype=torch.float16)), TypeError),
    (dict(state=torch.zeros(2, 6, 5)), ValueError),
    (dict(state=torch.zeros(2, 6, 4, dtype=torch.bfloat16)), TypeError),
    (dict(lengths=torch.zeros((2, 1), dtype=torch.int64)), ValueError),
    (dict(), RuntimeError),
])
def test_state_scan_refuses(kw, err):
    with pytest.raises(err):
        ops.state_scan(**_scan(**kw))


def test_state_scan_step_refuses():
    def args(**kw):
        a = dict(x=torch.zeros(2, 6), state=torch.zeros(2, 6, 4), dt=torch.zeros(2, 6), a=torch.zeros(6, 4),
                 b=torch.zeros(2, 4), c=torch.zeros(2, 4))
        a.update(kw)
        return a

    flat = torch.zeros(2 * 6 * 4 + 4)
    for kw, err in ((dict(state=None), TypeError), (dict(b=torch.zeros(2, 5)), ValueError),
                    (dict(state=torch.zeros(2, 4, 6).transpose(1, 2)), ValueError),
                    (dict(state=flat[:48].view(2, 6, 4), state_out=flat[4:].view(2, 6, 4)), ValueError),  # overlap
                    (dict(a=torch.zeros(6, 4, requires_grad=True)), RuntimeError), (dict(), RuntimeError)):
        with pytest.raises(err):
            ops.state_scan_step(**args(**kw))


def test_global_norm_and_clip_refuse():
    z = torch.zeros(8)
    for bad in ([z, None], [z.double()], [z.to_sparse()], [torch.zeros(8, dtype=torch.int32)]):
        with pytest.raises(TypeError):
            ops.global_norm(bad)
    with pytest.raises(ValueError):
        ops.global_norm([z], norm_type=1.0)
    with pytest.raises(RuntimeError):
        ops.global_norm([z])
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, out=[]),
               dict(max_norm=1.0, out=[torch.zeros(7)])):
        with pytest.raises(ValueError):
            ops.clip_gradients([z], **kw)
    with pytest.raises(TypeError):
        ops.clip_gradients([z], 1.0, out=[torch.zeros(8, dtype=torch.float16)])
    with pytest.raises(ValueError):  # elements that share memory
        ops.clip_gradients([torch.zeros(1).expand(8)], 1.0)
    assert float(ops.global_norm([])) == 0.0 and float(ops.clip_gradients([], 1.0)) == 0.0


def test_clip_refuses_tensors_that_overlap():
    flat = torch.zeros(32)
    a, b, c, o1, o2 = flat[:16], flat[16:], flat[8:24], torch.zeros(16), torch.zeros(16)

    def check(src, dst):
        ops._check_disjoint([t.data_ptr() for t in src], [t.data_ptr() for t in dst], [4 * t.numel() for t in src])

    check([a, b], [a, b])       # in place, side by side
    check([a], [o1])
    check([a, a], [o1, o2])     # read twice, written apart
    check([a[:0], a], [c[:0], a])
    for src, dst in (([a, a], [a, a]), ([a, c], [a, c]), ([a], [c]), ([a, b], [b, a]), ([a, c], [o1, c]), ([a, b], [o1, o1])):
        with pytest.raises(ValueError):
            check(src, dst)


def test_workspace_sizes_are_those_of_the_layout():
    lib = _native.load()
    # forward with enough rows: no time segments, no workspace; few rows and a long axis: segment states
    assert lib.afd_state_scan_workspace_bytes(128, 101, 1024, 16, 0) == 0
    assert lib.afd_state_scan_workspace_bytes(1, 16384, 1024, 16, 0) > 0
    assert lib.afd_state_scan_workspace_bytes(0, 1, 1, 1, 0) == 0
    assert lib.afd_state_scan_checkpoint_floats(2, 17, 5, 3) == 2 * 3 * 5 * 4
    assert lib.afd_causal_conv_backward_workspace_bytes(2, 65, 6, 4) == 2 * 5 * 6 * 5 * 4  # five tiles of 16 rows


def test_c_entries_refuse_bad_sizes():
    lib = _native.load()
    import ctypes

    one = ctypes.c_void_p(16)  # never dereferenced: the sizes are refused first
    strides = (_native.c_l * 12)()
    assert lib.afd_causal_conv_forward(one, 1, 1, one, None, 1, None, None, one, None, 1, 1, 1, 9, 0, 0, None) == -1
    assert b"9 (2..8)" in lib.afd_last_error()
    assert lib.afd_causal_conv_forward(one, 1, 1, one, None, 1, None, None, one, None, 0, 1, 1, 4, 0, 0, None) == -1
    assert lib.afd_causal_conv_backward(one, 1, 1, one, None, 1, None, None, one, 1, 1, None, one, one, None, None, 1, 1, 1,
                                        4, 0, 0, None, 0, None) == -4
    assert lib.afd_state_scan_forward(one, one, one, one, None, strides, one, None, None, None, None, one, None, None, 1, 1,
                                      1, 65, 1, 0, None, 0, None) == -1
    assert lib.afd_state_scan_forward(one, one, one, one, None, strides, one, None, None, None, None, one, None, None, 1,
                                      16384, 64, 16, 1, 0, None, 0, None) == -4
    assert lib.afd_state_scan_forward(one, one, one, one, None, strides, one, None, None, None, None, one, None, None, 1, 1,
                                      1, 1, 1, 7, None, 0, None) == -1
    assert lib.afd_global_norm(None, None, None, 1, 0, 1.0, 1.0, one, None, 0, None) == -1
    assert lib.afd_global_norm(None, None, None, 0, 0, 1.0, 1.0, one, None, 0, None) == -4
    assert lib.afd_adam_step_clipped(one, one, one, one, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None) == -1


def test_trainer_flag():
    import argparse

    from audiofakedetect.utils import add_default_parser_args

    parser = add_default_parser_args(argparse.ArgumentParser())
    assert parser.parse_args([]).clip_grad_norm is None
    assert parser.parse_args(["--clip-grad-norm", "0.5"]).clip_grad_norm == 0.5


# ---- the float64 restatements the GPU tests compare with: their gradients against differences ---------------------------
def _differences(f, t, dy, eps=1e-6):
    """d <dy, f> / dt by central differences, element by element."""
    out = torch.zeros_like(t)
    flat, o = t.view(-1), out.view(-1)
    for i in range(flat.numel()):
        keep = float(flat[i])
        flat[i] = keep + eps
        hi = float((f() * dy).sum())
        flat[i] = keep - eps
        lo = float((f() * dy).sum())
        flat[i] = keep
        o[i] = (hi - lo) / (2 * eps)
    return out


@pytest.mark.parametrize("act", ["none", "silu"])
def test_reference_conv_gradients_are_the_differences(act):
    import sequence_ref as ref

    g = torch.Generator().manual_seed(1)
    t = dict(x=torch.randn(2, 5, 3, generator=g).double(), w=torch.randn(3, 3, generator=g).double(),
             b=torch.randn(3, generator=g).double(), state=torch.randn(2, 2, 3, generator=g).double())
    dy = torch.randn(2, 5, 3, generator=g).double()
    lengths = torch.tensor([5, 1])
    got = ref.conv(**t, act=act, lengths=lengths, dy=dy)
    for name in t:
        diff = _differences(lambda: ref.conv(**t, act=act, lengths=lengths)["y"], t[name], dy)
        assert (got["d" + name] - diff).abs().max() < 1e-7, name
    ds = torch.randn(2, 2, 3, generator=g).double()
    got = ref.conv(**t, act=act, lengths=lengths, dy=torch.zeros_like(dy), dstate_out=ds)
    for name in ("x", "state"):
        diff = _differences(lambda: ref.conv(**t, act=act, lengths=lengths)["state"], t[name], ds)
        assert (got["d" + name] - diff).abs().max() < 1e-7, name


def test_reference_scan_gradients_are_the_differences():
    import sequence_ref as ref

    g = torch.Generator().manual_seed(2)

    def rnd(*s):
        return torch.randn(*s, generator=g).double()

    t = dict(x=rnd(2, 4, 3), dt=rnd(2, 4, 3), a=-rnd(3, 2).abs(), b=rnd(2, 4, 2), c=rnd(2, 4, 2), d=rnd(3), gate=rnd(2, 4, 3),
             dt_bias=rnd(3), state=rnd(2, 3, 2))
    dy, ds = rnd(2, 4, 3), rnd(2, 3, 2)
    lengths = torch.tensor([4, 2])
    got = ref.scan(**t, softplus=True, lengths=lengths, dy=dy)
    late = ref.scan(**t, softplus=True, lengths=lengths, dy=torch.zeros_like(dy), dstate_out=ds)
    for name in t:
        diff = _differences(lambda: ref.scan(**t, softplus=True, lengths=lengths)["y"], t[name], dy)
        assert (got["d" + name] - diff).abs().max() < 1e-7, name
        diff = _differences(lambda: ref.scan(**t, softplus=True, lengths=lengths)["state"], t[name], ds)
        assert (late["d" + name] - diff).abs().max() < 1e-7, name


@pytest.mark.parametrize("kw, err", [
    (dict(x=torch.zeros(3, 5)), ValueError),
    (dict(x=torch.tensor(1.0)), ValueError),
    (dict(x=torch.zeros(3, 4, dtype=torch.float64)), TypeError),
    (dict(x=None), TypeError),
    (dict(w=torch.zeros(6, 4, dtype=torch.bfloat16)), TypeError),
    (dict(w=torch.zeros(4)), ValueError),
    (dict(w=torch.zeros(0, 4)), ValueError),
    (dict(x=torch.zeros(3, 0), w=torch.zeros(6, 0)), ValueError),
    (dict(b=torch.zeros(5)), ValueError),
    (dict(b=torch.zeros(6, dtype=torch.float16)), TypeError),
    (dict(residual=torch.zeros(2, 6)), ValueError),
    (dict(residual=torch.zeros(3, 6, dtype=torch.float16)), TypeError),
    (dict(activation="tanh"), ValueError),
    (dict(), RuntimeError),
])
def test_linear_refuses(kw, err):
    args = dict(x=torch.zeros(3, 4), w=torch.zeros(6, 4))
    args.update(kw)
    with pytest.raises(err):
        ops.linear(**args)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_reference_linear_gradients_are_the_differences(act):
    import sequence_ref as ref

    g = torch.Generator().manual_seed(3)
    t = dict(x=torch.randn(4, 3, generator=g).double(), w=torch.randn(5, 3, generator=g).double(),
             b=torch.randn(5, generator=g).double())
    dy = torch.randn(4, 5, generator=g).double()
    got = ref.linear(**t, act=act, dy=dy)
    for name in t:
        diff = _differences(lambda: ref.linear(**t, act=act)["y"], t[name], dy)
        assert (got["d" + name] - diff).abs().max() < 1e-7, name


def test_linear_c_entries_refuse():
    import ctypes

    lib = _native.load()
    one = ctypes.c_void_p(16)
    size = lib.afd_linear_workspace_bytes
    assert size(one, 4, one, 4, 0, 4, 4, 0) == 0 and size(one, 4, one, 4, 4, 4, 4, 9) == 0
    assert size(one, 64, one, 64, 4096, 4096, 64, 0) == 0               # read as they are
    assert size(one, 65, one, 64, 4096, 4096, 64, 0) == 4096 * 64 * 4   # x's rows leave the 16-byte grid: copied
    assert size(one, 64, ctypes.c_void_p(20), 64, 4096, 4096, 64, 0) == 4096 * 64 * 4
    assert lib.afd_linear_forward(one, 4, one, 4, None, 0, None, 0, one, None, 4, 4, 4, 7, 0, None, 0, None) == -1
    assert lib.afd_linear_forward(one, 4, one, 4, None, 0, None, 0, one, None, 4, 1 << 20, 4, 0, 0, None, 0, None) == -3
    assert lib.afd_linear_forward(one, 3, one, 3, None, 0, None, 0, one, None, 4, 4, 3, 0, 0, None, 0, None) == -4
    assert lib.afd_linear_backward(one, 4, one, 4, None, one, 4, one, one, None, 0, 4, 4, 4, 2, 0, None, 0, None) == -1
    assert lib.afd_linear_backward(one, 4, one, 4, one, one, 4, one, one, None, 0, 4, 4, 4, 2, 0, None, 0, None) == -4
    assert lib.afd_linear_backward(one, 4, one, 4, None, one, 4, one, one, None, 0, 9000000, 4, 4, 0, 0, one, 0, None) == -3


def test_linear_refuses_more_rows_than_its_backward_takes():
    x = torch.zeros(1, 8).expand(8_000_001, 8)
    w = torch.zeros(4, 8, requires_grad=True)
    with pytest.raises(ValueError, match="8000001 rows"):
        ops.linear(x, w)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        ops.linear(x, w)


def test_c_entries_refuse_more_workgroups_than_a_launch_holds():
    import ctypes

    lib = _native.load()
    one = ctypes.c_void_p(16)
    strides = (_native.c_l * 12)()
    most = 0xffffff  # workgroups of 256 threads
    assert lib.afd_state_scan_step(one, one, one, one, None, strides, one, None, None, one, one, one, most + 1, 64, 16, 1, 0,
                                   None) == -3
    assert lib.afd_state_scan_forward(one, one, one, one, None, strides, one, None, None, None, None, one, None, None,
                                      most + 1, 2, 64, 16, 1, 0, None, 0, None) == -3
    assert lib.afd_state_scan_step(one, one, one, one, None, strides, one, None, None, one, one, one, 1, 0x3fffffff // 66 + 1,
                                   64, 1, 0, None) == -3
    assert lib.afd_causal_conv_step(one, 1, one, None, 1, one, one, one, 0x7fffffff, 8, 4, 0, 0, None) == -3
    assert lib.afd_linear_forward(one, 4, one, 4, None, 0, None, 0, one, None, 0x7fffff00, 80, 4, 0, 0, None, 0, None) == -3


# ---- what the entry points hand to the library, with the launches stubbed out -------------------------------------------
class _Launches:
    """The library with its sizes answered and its launches noted down: (entry, arguments)."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        if name.endswith(("_bytes", "_floats")):
            return getattr(self.lib, name)

        def note(*args):
            self.calls.append((name, args))
            return 0

        return note


class _NoDevice:
    def __init__(self, t):
        pass

    def __enter__(self):
        return 0

    def __exit__(self, *exc):
        pass


@pytest.fixture
def launches(monkeypatch):
    stub = _Launches(_native.load())
    monkeypatch.setattr(ops, "_lib", lambda: stub)
    monkeypatch.setattr(ops, "_OnDevice", _NoDevice)
    monkeypatch.setattr(ops, "_seq_gpu", lambda what, x: None)
    return stub


def _turned(t):
    """The same values with the last two axes the other way round in memory."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.clone()


@pytest.mark.parametrize("store", [lambda t: t.contiguous() if not t.is_contiguous() else t.clone(), _turned])
def test_backward_takes_the_layout_of_what_saved_tensor_hooks_give_back(launches, store):
    """A hook that stores the saved tensors elsewhere may give them back in another layout: the pointers and the strides of a
    launch have to belong together."""
    given = {}

    def unpack(t):
        given[t.data_ptr()] = t
        return t

    xz = torch.randn(2, 5, 16, requires_grad=True)
    bcd = torch.randn(2, 5, 14, requires_grad=True)
    x, gate = xz.chunk(2, -1)
    dt, b, c = bcd.split([8, 3, 3], -1)
    wide = torch.randn(6, 16)
    with torch.autograd.graph.saved_tensors_hooks(store, unpack):
        scanned = ops.state_scan(x, dt, torch.zeros(8, 3), b, c, gate=gate)
        conved = ops.causal_conv(x, torch.zeros(8, 4), torch.zeros(8), "silu", state=torch.zeros(2, 3, 8))
        linear = ops.linear(x, wide[:, 4:12], None, "silu")

    def rows(ptr, shape, strides, name):
        """Whatever lies at `ptr` with these strides is one of the tensors given back, or a copy of its rows."""
        t = given.get(ptr)
        assert t is None or (t.stride(-1) == 1 and t.stride()[:len(strides)] == tuple(strides)), (name, t.stride(), strides)
        if t is None:  # a copy: rows one behind the other
            assert strides[-1] == shape[-1], (name, strides)

    keep = []  # (copies made for a launch stay alive through their gradients; addresses are looked at right behind it)
    launches.calls.clear()
    keep.append(torch.autograd.grad(scanned.sum(), [xz, bcd], retain_graph=True))
    (name, args), = [k for k in launches.calls if k[0] == "afd_state_scan_backward"]
    strides = list(args[6])
    for i, (what, shape) in enumerate((("x", x.shape), ("dt", dt.shape), ("b", b.shape), ("c", c.shape), ("gate", gate.shape))):
        rows(args[i], shape, strides[2 * i:2 * i + 2], what)
    assert args[7] not in given or given[args[7]].is_contiguous()
    launches.calls.clear()
    keep.append(torch.autograd.grad(conved.sum(), [xz], retain_graph=True))
    (name, args), = [k for k in launches.calls if k[0] == "afd_causal_conv_backward"]
    rows(args[0], x.shape, args[1:3], "x")
    for i in (3, 6):
        assert args[i] not in given or given[args[i]].is_contiguous(), i
    launches.calls.clear()
    keep.append(torch.autograd.grad(linear.sum(), [xz]))
    (name, args), = [k for k in launches.calls if k[0] == "afd_linear_backward"]
    rows(args[0], (10, 8), [args[1]], "x")
    rows(args[2], (6, 8), [args[3]], "w")


def _calls_of_every_entry():
    """name -> (call, tensors): the tensor arguments of each entry point by name, all fit for it."""
    z = torch.zeros
    seq = dict(x=z(2, 5, 6), dt=z(2, 5, 6), a=z(6, 4), b=z(2, 5, 4), c=z(2, 5, 4), d=z(6), gate=z(2, 5, 6), dt_bias=z(6),
               state=z(2, 6, 4))
    one = {k: t[:, 0] if t.dim() == 3 and k != "state" else t for k, t in seq.items()}
    return {
        "causal_conv": (ops.causal_conv, dict(x=z(2, 5, 6), w=z(6, 4), b=z(6), state=z(2, 3, 6))),
        "causal_conv_step": (ops.causal_conv_step, dict(x=z(2, 6), state=z(2, 3, 6), w=z(6, 4), b=z(6), state_out=z(2, 3, 6))),
        "state_scan": (ops.state_scan, seq),
        "state_scan_step": (ops.state_scan_step, dict(one, state_out=z(2, 6, 4))),
        "linear": (ops.linear, dict(x=z(2, 3, 4), w=z(6, 4), b=z(6), residual=z(2, 3, 6))),
        "global_norm": (lambda **t: ops.global_norm(list(t.values())), dict(p=z(3), q=z(2, 8)[:, ::2])),
        "clip_gradients": (lambda p, q, o: ops.clip_gradients([p, q], 1.0, out=[p, o]), dict(p=z(3), q=z(4), o=z(4))),
    }


@pytest.mark.parametrize("entry", sorted(_calls_of_every_entry()))
def test_forward_mode_tangents_are_refused(launches, entry):
    """No entry point has a forward-mode derivative: a tangent is refused by name, not dropped."""
    from torch.autograd import forward_ad

    call, tensors = _calls_of_every_entry()[entry]
    with forward_ad.dual_level():
        call(**tensors)  # nothing carries a tangent: an ordinary call
        for name, t in tensors.items():
            with pytest.raises(NotImplementedError, match="forward"):
                call(**dict(tensors, **{name: forward_ad.make_dual(t, torch.ones_like(t))}))
    call(**tensors)


def test_global_norm_refuses_to_leave_the_graph_unseen(launches):
    """The norm has no backward pass: of tensors that require grad it is taken under no_grad, or not at all."""
    p = torch.ones(4, requires_grad=True)
    for tensors in ([p], [torch.zeros(3), p * 2]):
        with pytest.raises(RuntimeError, match="no_grad"):
            ops.global_norm(tensors)
        with torch.no_grad():
            assert not ops.global_norm(tensors).requires_grad
    ops.global_norm([p.detach()])


def test_scan_rows_at_the_edge_of_the_lanes_offsets(launches):
    """Rows 2^24 elements apart are read as they are, farther ones are copied, and a single row's stride does not count."""
    lib, t = _native.load(), torch.zeros
    small = dict(dt=t(1, 2, 8), a=t(8, 3), b=t(1, 2, 3), c=t(1, 2, 3))
    for far, seen in ((1 << 24, 1 << 24), ((1 << 24) + 1, 8)):
        x = torch.empty(far + 8).as_strided((1, 2, 8), (0, far, 1))
        launches.calls.clear()
        ops.state_scan(x, **small)
        (name, args), = launches.calls
        assert args[5][1] == seen and (args[0] == x.data_ptr()) == (seen == far)
    one = {k: v[:, :1] if v.dim() == 3 else v for k, v in small.items()}
    x = torch.empty((1 << 25) + 8).as_strided((1, 1, 8), (8, 1 << 25, 1))  # one frame of a time-major batch
    launches.calls.clear()
    ops.state_scan(x, **one)
    (name, args), = launches.calls
    assert args[0] == x.data_ptr() and args[5][1] <= 1 << 24
    # the library draws the line where the binding does, for every type (-4: the next check, a missing workspace)
    import ctypes

    p = ctypes.c_void_p(16)
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        for stride, rc in ((1 << 24, -4), ((1 << 24) * 4 // size + 1, -3)):
            st = (_native.c_l * 12)(*([0, stride] * 6))
            assert lib.afd_state_scan_forward(p, p, p, p, None, st, p, None, None, None, None, p, None, None, 1, 16384, 64, 16,
                                              1, dtype, None, 0, None) == rc, (dtype, stride)
            assert lib.afd_state_scan_backward(p, p, p, p, None, p, st, p, None, None, None, p, None, p, p, p, p, None, p, None,
                                               None, None, 1, 16384, 64, 16, 1, dtype, None, 0, None) == rc, (dtype, stride)


def test_clip_out_in_place_with_gaps(launches):
    base = torch.arange(24.0).view(4, 6)
    g = base[:, :3]
    ops.clip_gradients([g], 1.0, out=[g])  # (the launches are noted, not run: a factor of one)
    assert [name for name, _ in launches.calls] == ["afd_global_norm", "afd_multi_scale"]
    assert torch.equal(base, torch.arange(24.0).view(4, 6))
    ops.clip_gradients([g, torch.zeros(4, 3)], 1.0, out=[base[:, :3], torch.zeros(4, 3)])  # another view of the same elements
    with pytest.raises(ValueError, match="share memory"):
        wide = torch.zeros(4, 1).expand(4, 3)
        ops.clip_gradients([wide], 1.0, out=[wide])
    with pytest.raises(ValueError, match="overlap"):  # the other gradient would be written over with what is copied back
        ops.clip_gradients([g, torch.zeros(6)], 1.0, out=[g, base[1]])
    for other in (base[:, 3:], torch.zeros(4, 6)[:, 3:]):
        with pytest.raises(ValueError, match="gaps"):
            ops.clip_gradients([g], 1.0, out=[other])
    with pytest.raises(ValueError, match="gaps"):
        ops.clip_gradients([torch.zeros(4, 3)], 1.0, out=[base[:, 3:]])
