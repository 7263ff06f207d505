"""What the recurrent operators outside the trunk refuse, on the host and before anything is launched; their 64-bit implementations;
their operators' shapes."""

import ctypes as C

import pytest
import torch

from oracle import sequence_oracle as O


def _conv(**over):
    import boost_and_broadside_b200 as bnb

    a = dict(x=torch.zeros(3, 2, 8), weight=torch.zeros(8, 4))
    a.update(over)
    return bnb.causal_conv(a.pop("x"), a.pop("weight"), **a)


def _scan(**over):
    import boost_and_broadside_b200 as bnb

    a = dict(u=torch.zeros(3, 2, 8), delta=torch.zeros(3, 2, 8), A=torch.zeros(8, 4), B=torch.zeros(3, 2, 4), C=torch.zeros(3, 2, 4))
    a.update(over)
    first = [a.pop(k) for k in ("u", "delta", "A", "B", "C")]
    return bnb.selective_scan(*first, **a)


def test_there_is_no_cpu_path():
    import boost_and_broadside_b200 as bnb

    with pytest.raises(RuntimeError, match="no CPU path"):
        _conv()
    with pytest.raises(RuntimeError, match="no CPU path"):
        _scan()
    with pytest.raises(RuntimeError, match="no CPU path"):
        bnb.causal_conv_step(torch.zeros(2, 8), torch.zeros(2, 3, 8), torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        bnb.selective_step(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(2, 4), torch.zeros(2, 4), None, torch.zeros(2, 8, 4))


def test_arguments_are_refused_before_the_library():
    import boost_and_broadside_b200 as bnb

    with pytest.raises(ValueError, match="activation"):
        _conv(activation="gelu")
    with pytest.raises(RuntimeError, match="B must have"):
        _scan(B=torch.zeros(3, 4))
    with pytest.raises(NotImplementedError, match="forward-only"):
        bnb.causal_conv_step(torch.zeros(2, 8, requires_grad=True), torch.zeros(2, 3, 8), torch.zeros(8, 4))
    with pytest.raises(NotImplementedError, match="forward-only"):
        bnb.selective_step(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(8, 4, requires_grad=True), torch.zeros(2, 4), torch.zeros(2, 4), None,
                           torch.zeros(2, 8, 4))


class View(C.Structure):
    _fields_ = [("data", C.c_void_p), ("step", C.c_int64), ("row", C.c_int64), ("group", C.c_int64)]


class Conv(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("steps", "rows", "width", "taps", "element", "activation")] + [("x", View), ("y", View)] + [
        (n, C.c_void_p) for n in ("weight", "bias", "state_in", "state_out", "done", "lengths", "reset")]


class Scan(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("steps", "rows", "width", "states", "groups", "element", "softplus")] + [
        (n, View) for n in ("u", "delta", "z", "b", "c", "y")] + [
        (n, C.c_void_p) for n in ("a", "d", "delta_bias", "state_in", "state_out", "done", "lengths", "reset", "kept")]


def test_c_entry_points_check_their_arguments():
    from boost_and_broadside_b200 import _capi

    lib = _capi.lib
    fake = 0x1000
    v = View(fake, 16, 8, 0)

    def conv(**over):
        a = Conv(3, 2, 8, 4, 0, 0, v, v, fake, None, None, 2 * fake, None, None, None)
        for k, x in over.items():
            setattr(a, k, x)
        return lib.bnb_causal_conv_fwd(C.byref(a), None)

    assert conv(taps=5) == 3 and conv(taps=1) == 3
    assert conv(element=3) == 5 and conv(activation=2) == 5 and conv(steps=-1) == 5
    assert conv(weight=None) == 1 and conv(state_out=None) == 1
    assert conv(state_in=2 * fake) == 5                        # in place for several steps
    assert conv(rows=0, weight=None) == 0                      # nothing to do
    assert lib.bnb_causal_conv_fwd(None, None) == 1
    a = Conv(3, 2, 8, 4, 0, 0, v, v, fake, None, None, 2 * fake, None, None, None)
    assert lib.bnb_causal_conv_bwd(C.byref(a), None, None, 0, None) == 1
    assert lib.bnb_causal_conv_bwd_scratch_bytes(C.byref(a)) > 0

    def scan(fn="bnb_selective_scan_fwd", **over):
        q = Scan(3, 2, 8, 4, 1, 0, 0, v, v, View(), v, v, v, fake, None, None, None, 2 * fake, None, None, None, None)
        for k, x in over.items():
            setattr(q, k, x)
        return lib.bnb_selective_scan_fwd(C.byref(q), None, 0, None) if fn == "bnb_selective_scan_fwd" else lib.bnb_selective_step(C.byref(q), None)

    assert scan(states=65) == 3 and scan(states=0) == 3
    assert scan(groups=3) == 5 and scan(groups=0) == 5 and scan(element=7) == 5
    assert scan(a=None) == 1 and scan(state_out=None) == 1 and scan(state_in=fake + 4) == 2
    assert scan(state_in=2 * fake) == 5 and scan(reset=fake) == 5
    assert scan(rows=0) == 0 and scan(width=0) == 0
    assert scan("bnb_selective_step") == 5                     # three steps
    assert scan("bnb_selective_step", steps=1, done=fake) == 5
    long = Scan(4096, 1, 64, 16, 1, 0, 0, v, v, View(), v, v, v, fake, None, None, None, 2 * fake, None, None, None, None)
    need = lib.bnb_selective_scan_scratch_bytes(C.byref(long))
    assert need > 0 and lib.bnb_selective_scan_fwd(C.byref(long), fake, need - 1, None) == 6
    assert lib.bnb_selective_scan_bwd(C.byref(long), None, None, 0, None) == 1


class Gated(C.Structure):
    _fields_ = [("rows", C.c_int64)] + [(n, C.c_int32) for n in ("width", "hidden", "element", "weight_element", "activation")] + [
        ("x", C.c_void_p), ("x_row", C.c_int64)] + [(n, C.c_void_p) for n in ("gate_w", "up_w", "down_w", "y", "kept")]


class GatedGrads(C.Structure):
    _fields_ = [("dy", C.c_void_p), ("dy_row", C.c_int64)] + [(n, C.c_void_p) for n in ("dx", "dgate_w", "dup_w", "ddown_w")]


def test_gated_block_checks_its_arguments():
    import boost_and_broadside_b200 as bnb
    from boost_and_broadside_b200 import _capi

    x, w = torch.zeros(3, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        bnb.gated_mlp(x, w, w, w.t())
    with pytest.raises(ValueError, match="activation"):
        bnb.gated_mlp(x, w, w, w.t(), activation="relu")
    lib, fake = _capi.lib, 0x1000

    def call(**over):
        c = Gated(100, 64, 128, 1, 1, 2, fake, 64, fake, fake, fake, fake, None)
        for k, v in over.items():
            setattr(c, k, v)
        return c

    fwd = lambda **over: lib.bnb_gated_block_fwd(C.byref(call(**over)), over.pop("scratch", None), 0, None)  # noqa: E731
    assert fwd(width=0) == 3 and fwd(hidden=0) == 3 and fwd(weight_element=2) == 3
    assert fwd(activation=0) == 5 and fwd(element=3) == 5 and fwd(rows=-1) == 5
    assert fwd(gate_w=None) == 1 and fwd(x=None) == 1 and fwd(y=None) == 1
    assert fwd(y=fake + 4) == 2 and fwd() == 6
    assert fwd(rows=0) == 0
    c = call()
    assert lib.bnb_gated_block_scratch_bytes(C.byref(c), 0) >= 100 * 128 * 2
    assert lib.bnb_gated_block_scratch_bytes(C.byref(c), 1) > lib.bnb_gated_block_scratch_bytes(C.byref(c), 0)
    assert lib.bnb_gated_block_kept_bytes(C.byref(c)) == 0                                        # narrow: computed once more
    assert lib.bnb_gated_block_kept_bytes(C.byref(call(width=600))) == 2 * 128 * 128 * 4          # whole blocks of 32 x 32
    g = GatedGrads(fake, 64, fake, fake, None, fake)
    assert lib.bnb_gated_block_bwd(C.byref(call(kept=fake)), C.byref(g), None, 0, None) == 1     # half of the gate's pair
    g = GatedGrads(fake, 64, fake, fake, fake, fake)
    assert lib.bnb_gated_block_bwd(C.byref(call(width=600)), C.byref(g), None, 0, None) == 1     # nothing kept
    assert lib.bnb_gated_block_bwd(C.byref(call(kept=fake)), C.byref(g), None, 0, None) == 6


def test_split_sequences_join():
    """The 64-bit implementations themselves: a sequence in two calls, episode ends and lengths included, is the sequence in one."""
    g = torch.Generator().manual_seed(0)
    T, R, W, N = 9, 4, 6, 3
    x, w = torch.randn(T, R, W, generator=g), torch.randn(W, 4, generator=g)
    done = torch.rand(T, R, generator=g) < 0.3
    done[4] = False
    y, st = O.causal_conv(x, w, done=done, activation="silu")
    y1, s1 = O.causal_conv(x[:5], w, done=done[:5], activation="silu")
    y2, s2 = O.causal_conv(x[5:], w, state=s1, done=done[5:], activation="silu")
    assert torch.allclose(torch.cat([y1, y2]), y) and torch.allclose(s2, st)
    u, d = torch.randn(T, R, W, generator=g), torch.rand(T, R, W, generator=g)
    A, B, C_ = -torch.rand(W, N, generator=g), torch.randn(T, R, 1, N, generator=g), torch.randn(T, R, 1, N, generator=g)
    y, h = O.selective_scan(u, d, A, B, C_, done=done)
    y1, h1 = O.selective_scan(u[:5], d[:5], A, B[:5], C_[:5], done=done[:5])
    y2, h2 = O.selective_scan(u[5:], d[5:], A, B[5:], C_[5:], state=h1, done=done[5:])
    assert torch.allclose(torch.cat([y1, y2]), y) and torch.allclose(h2, h)
    n = torch.tensor([9, 0, 5, 1])
    y3, h3 = O.selective_scan(u, d, A, B, C_, done=done, lengths=n)
    assert torch.allclose(h3[2], h1[2]) and not y3[5:, 2].any() and not h3[1].any() and torch.allclose(y3[:5, 2], y[:5, 2])


def test_operators_have_shape_only_fakes():
    import boost_and_broadside_b200  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.bnb_b200
    with FakeTensorMode():
        x, w = torch.empty(5, 3, 8, device="cuda", dtype=torch.bfloat16), torch.empty(8, 4, device="cuda")
        y, st = ops.causal_conv(x, w, None, None, None, None, 1)
        assert y.shape == x.shape and y.dtype == x.dtype and st.shape == (3, 3, 8) and st.dtype == torch.float32
        A, B = torch.empty(8, 11, device="cuda"), torch.empty(5, 3, 2, 11, device="cuda", dtype=torch.bfloat16)
        y, st, kept = ops.selective_scan(x, x, A, B, B, None, None, None, None, None, None, True, True)
        assert y.shape == x.shape and st.shape == (3, 8, 11) and kept.numel() == 1 * 3 * 8 * 16
        assert ops.selective_scan(x, x, A, B, B, None, None, None, None, None, None, True, False)[2].numel() == 0
        y, kept = ops.gated_mlp(x, torch.empty(20, 8, device="cuda"), torch.empty(20, 8, device="cuda"), torch.empty(8, 20, device="cuda"), 2, True)
        assert y.shape == x.shape and kept.numel() == 0
        assert ops.selective_step(x[0], x[0], A, B[0], B[0], None, st, None, None, None, True).shape == (3, 8)
