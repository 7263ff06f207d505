"""What the operators of an update's end refuse, on the host and before anything is launched; their operators' shapes."""

import ctypes as C

import pytest
import torch


def _policy(**over):
    import boost_and_broadside_b200 as bnb

    a = dict(logits=torch.zeros(4, 12), actions=torch.zeros(4, 3, dtype=torch.int64), old=torch.zeros(4), adv=torch.zeros(4), sizes=(3, 7, 2))
    a.update(over)
    return bnb.policy_loss(a.pop("logits"), a.pop("actions"), a.pop("old"), a.pop("adv"), **a)


def test_policy_loss_has_no_cpu_path_and_checks_its_numbers():
    with pytest.raises(RuntimeError, match="no CPU path"):
        _policy()
    for clip in (-0.1, (0.2, -1.0), float("nan")):
        with pytest.raises(ValueError, match="clip"):
            _policy(clip=clip)
    with pytest.raises(ValueError, match="sizes"):
        _policy(sizes=())
    for name, over in (("old_logprob", dict(old=torch.zeros(4, requires_grad=True))), ("advantages", dict(adv=torch.zeros(4, requires_grad=True))),
                       ("ref_logprob", dict(ref_logprob=torch.zeros(4, requires_grad=True))), ("weights", dict(weights=torch.ones(4, requires_grad=True)))):
        with pytest.raises(NotImplementedError, match=name):
            _policy(**over)


class Policy(C.Structure):
    _fields_ = [("rows", C.c_int64), ("element", C.c_int32), ("n_slices", C.c_int32), ("sizes", C.c_int32 * 16), ("logits", C.c_void_p),
                ("logits_row", C.c_int64)] + [(n, C.c_void_p) for n in ("actions", "old", "adv", "ref", "weights", "mask")] + [
                    (n, C.c_float) for n in ("low", "high", "kl", "entropy")] + [(n, C.c_void_p) for n in ("loss", "stats", "logprob", "kept", "dlogits")]


def test_policy_entry_points_check_their_arguments():
    from boost_and_broadside_b200 import _capi

    lib, fake = _capi.lib, 0x1000

    def call(**over):
        c = Policy(100, 1, 3, (C.c_int32 * 16)(3, 7, 2), fake, 12, fake, fake, fake, None, None, None, 0.2, 0.2, 0.0, 0.0, fake, fake, fake, fake)
        for k, v in over.items():
            setattr(c, k, v)
        return c

    fwd = lambda scratch=None, bytes_=0, **over: lib.bnb_policy_loss_fwd(C.byref(call(**over)), scratch, bytes_, None)  # noqa: E731
    assert fwd() == 6 and fwd(scratch=fake + 4, bytes_=1 << 20) == 2
    assert fwd(n_slices=0) == 3 and fwd(n_slices=17) == 3 and fwd(sizes=(C.c_int32 * 16)(3, 0, 2)) == 3
    assert fwd(sizes=(C.c_int32 * 16)(1 << 28, 7, 2)) == 3
    assert fwd(rows=-1) == 5 and fwd(element=3) == 5 and fwd(low=-0.1) == 5 and fwd(high=float("nan")) == 5
    assert fwd(weights=fake, mask=fake) == 5
    for name in ("logits", "actions", "old", "adv", "loss", "stats", "logprob", "kept"):
        assert fwd(**{name: None}) == 1, name
    assert lib.bnb_policy_loss_fwd(None, None, 0, None) == 1
    assert fwd(scratch=fake, bytes_=1 << 20, dlogits=fake) == 5                                   # narrow slices: no gradients in a forward
    wide = (C.c_int32 * 16)(300, 2, 900)
    takes = lambda **over: lib.bnb_policy_loss_takes_gradients(C.byref(call(**over)))  # noqa: E731
    assert [takes(sizes=wide, element=e) for e in (0, 1, 2)] == [1, 1, 0] and takes() == 0 and takes(n_slices=0) == 0
    assert fwd(scratch=fake, bytes_=1 << 20, dlogits=fake + 8, sizes=wide) == 2 and fwd(scratch=fake, bytes_=1 << 20, dlogits=fake, sizes=wide, element=2) == 5
    bwd = lambda dloss, out, **over: lib.bnb_policy_loss_bwd(C.byref(call(**over)), dloss, out, 0, None)  # noqa: E731
    assert bwd(None, fake) == 1 and bwd(fake, None) == 1 and bwd(fake, fake + 2) == 2 and bwd(fake, fake, n_slices=99) == 3
    assert bwd(None, None, rows=0, logits=None) == 0
    assert lib.bnb_policy_loss_kept_bytes(C.byref(call())) == 4 * (4 + 100 * 8)
    assert lib.bnb_policy_loss_scratch_bytes(C.byref(call())) > 0


def test_operators_have_shape_only_fakes():
    import boost_and_broadside_b200  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.bnb_b200
    with FakeTensorMode():
        z = torch.empty(5, 3, 12, device="cuda", dtype=torch.bfloat16)
        a, v = torch.empty(5, 3, 3, device="cuda", dtype=torch.int64), torch.empty(5, 3, device="cuda")
        loss, l, stats, kept = ops.policy_loss(z, a, v, v, None, None, [3, 7, 2], 0.2, 0.2, 0.0, 0.0)
        assert loss.shape == () and loss.dtype == torch.float32 and l.shape == (5, 3) and stats.shape == (4,) and kept.numel() == 4 + 15 * 8
        y, kept_z = ops.linear(z, torch.empty(20, 12, device="cuda"), None, None, 2, True)
        assert y.shape == (5, 3, 20) and y.dtype == z.dtype and kept_z.numel() == 32 * 32 * 2
        assert ops.linear(z.float(), torch.empty(20, 12, device="cuda"), None, None, 2, True)[1].numel() == 4 * 32 * 32
        assert ops.policy_loss_backward(z, a, v, v, None, None, [3, 7, 2], 0.2, 0.2, 0.0, 0.0, kept, loss).shape == z.shape


class AdamTensor(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("p", "g", "m", "v", "m_scale", "v_scale", "step")] + [("n", C.c_int64), ("position", C.c_int64), ("element", C.c_int32)]


class AdamCall(C.Structure):
    _fields_ = [("state_bits", C.c_int32), ("seed", C.c_uint32), ("lr", C.c_float), ("lr_device", C.c_void_p), ("beta1", C.c_double), ("beta2", C.c_double)] + [
        (n, C.c_float) for n in ("eps", "weight_decay", "max_norm")] + [("norm_parts", C.c_void_p), ("n_norm_parts", C.c_int32), ("norm", C.c_void_p), ("control", C.c_void_p)]


def test_adamw_entry_points_check_their_arguments():
    from boost_and_broadside_b200 import _capi

    lib, fake = _capi.lib, 0x1000

    def step(tensor=None, **over):
        t = AdamTensor(fake, fake, fake, fake, None, None, fake, 10, 0, 0)
        for k, v in (tensor or {}).items():
            setattr(t, k, v)
        c = AdamCall(32, 0, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 0.0, None, 0, None, fake)
        for k, v in over.items():
            setattr(c, k, v)
        return lib.bnb_adamw_step(C.byref(t), 1, C.byref(c), None)

    assert step(state_bits=16) == 5 and step(beta1=1.0) == 5 and step(beta2=-0.1) == 5 and step(eps=float("nan")) == 5
    assert step(control=None) == 1 and step(norm_parts=fake) == 5 and step(norm_parts=fake, n_norm_parts=3, max_norm=-1.0) == 5
    assert step(state_bits=8) == 1                            # scales missing
    for name in ("p", "g", "m", "v", "step"):
        assert step(tensor={name: None}) == 1, name
    assert step(tensor={"n": -1}) == 5 and step(tensor={"element": 3}) == 5
    c = AdamCall(32, 0, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 0.0, None, 0, None, fake)
    assert lib.bnb_adamw_step(None, 1, C.byref(c), None) == 1 and lib.bnb_adamw_step(None, -1, C.byref(c), None) == 5
    assert lib.bnb_adamw_step(None, 0, C.byref(c), None) == 0 and lib.bnb_adamw_step(None, 0, None, None) == 1
    assert lib.bnb_grad_norm(None, 0, None, None) == 1


def test_adamw_checks_its_numbers():
    import boost_and_broadside_b200 as bnb

    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(max_norm=-1.0), dict(state_bits=16),
                dict(lr=torch.zeros(2))):
        with pytest.raises(ValueError, match="AdamW"):
            bnb.AdamW([p], **bad)
    with pytest.raises(ValueError, match="float64"):
        bnb.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    opt = bnb.AdamW([p])
    opt.step()                                                # no gradient, nothing to do
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2))], lr=-1.0))
    assert len(opt.param_groups) == 1
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()


def test_random_bits_are_even_and_of_their_own():
    """The 20 bits behind a rounding at random: means, neighbours, steps and seeds, within five standard errors."""
    from oracle import update_oracle as O

    n = 1 << 18
    at = torch.arange(n)
    a = O.noise(at, 3, 7).double() / 2 ** 20
    for other in (O.noise(at, 3, 8), O.noise(at, 4, 7), O.noise(at + 256, 3, 7), O.noise(at + 1, 3, 7), O.noise(at + (1 << 32), 3, 7)):
        b = other.double() / 2 ** 20
        assert abs(float(b.mean()) - 0.5) <= 5 * (1 / 12 / n) ** 0.5
        assert abs(float(((a - 0.5) * (b - 0.5)).mean())) <= 5 / 12 / n ** 0.5


class Linear(C.Structure):
    _fields_ = [("rows", C.c_int64)] + [(n, C.c_int32) for n in ("width", "out", "element", "weight_element", "bias_element", "activation")] + [
        ("x", C.c_void_p), ("x_row", C.c_int64), ("weight", C.c_void_p), ("bias", C.c_void_p), ("residual", C.c_void_p), ("residual_row", C.c_int64),
        ("y", C.c_void_p), ("kept", C.c_void_p)]


class LinearGrads(C.Structure):
    _fields_ = [("dy", C.c_void_p), ("dy_row", C.c_int64)] + [(n, C.c_void_p) for n in ("dx", "dweight", "dbias")]


def test_linear_checks_its_arguments():
    import boost_and_broadside_b200 as bnb
    from boost_and_broadside_b200 import _capi

    x, w = torch.zeros(3, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        bnb.linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        bnb.linear(x, w, activation="relu")
    lib, fake = _capi.lib, 0x1000

    def call(**over):
        c = Linear(100, 64, 128, 1, 1, 1, 2, fake, 64, fake, fake, None, 0, fake, None)
        for k, v in over.items():
            setattr(c, k, v)
        return c

    fwd = lambda **over: lib.bnb_linear_fwd(C.byref(call(**over)), None, 0, None)  # noqa: E731
    assert fwd(width=0) == 3 and fwd(out=0) == 3 and fwd(weight_element=2) == 3 and fwd(bias_element=2) == 3
    assert fwd(activation=3) == 5 and fwd(element=3) == 5 and fwd(rows=-1) == 5
    assert fwd(weight=None) == 1 and fwd(x=None) == 1 and fwd(y=None) == 1
    assert fwd(y=fake + 4) == 2 and fwd() == 6 and fwd(rows=0) == 0
    kept = lambda **over: lib.bnb_linear_kept_bytes(C.byref(call(**over)))  # noqa: E731
    assert kept(activation=0) == 0 and kept() == 128 * 128 * 2 and kept(bias=None, bias_element=0) == 128 * 128 * 2   # slopes in 16 bits
    for over in (dict(bias_element=0), dict(element=2, weight_element=2, bias_element=2), dict(element=0, weight_element=0, bias_element=0)):
        assert kept(**over) == 128 * 128 * 4                                  # z in float32
    assert lib.bnb_linear_scratch_bytes(C.byref(call()), 1) > lib.bnb_linear_scratch_bytes(C.byref(call()), 0)
    bwd = lambda g, **over: lib.bnb_linear_bwd(C.byref(call(**over)), C.byref(g) if g else None, None, 0, None)  # noqa: E731
    assert bwd(None) == 1 and bwd(LinearGrads(None, 128, fake, fake, fake)) == 1
    assert bwd(LinearGrads(fake, 128, fake, fake, fake), width=600) == 1     # nothing kept
    assert bwd(LinearGrads(fake, 128, fake + 8, fake, fake), kept=fake) == 2 and bwd(LinearGrads(fake, 128, fake, fake, fake), kept=fake) == 6
