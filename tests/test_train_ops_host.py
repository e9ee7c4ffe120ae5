"""Refusals of the training operators (no GPU needed: arguments are checked before anything touches a device)."""

import math

import pytest
import torch

import tcmi as tc
from tcmi import _lib, linalg, torchnn


def test_newton_schulz_refusals():
    x = torch.zeros(4, 5)
    for bad in (torch.zeros(4), 3.0):
        with pytest.raises(ValueError):
            linalg.newton_schulz(bad)
    for steps in (0, -1, _lib.NS_MAX_STEPS + 1, 2.5, True):
        with pytest.raises(ValueError, match="steps"):
            linalg.newton_schulz(x, steps=steps)
    for coef in ((1.0, 2.0), ((1.5, -0.5, 0.0),) * 4, (1.0, math.nan, 0.0), ((1.0, 2.0),) * 5):
        with pytest.raises(ValueError, match="coefficients"):
            linalg.newton_schulz(x, steps=5, coefficients=coef)
    for eps in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            linalg.newton_schulz(x, eps=eps)
    for dt in (torch.float64, torch.complex128, torch.int32):
        with pytest.raises(TypeError):
            linalg.newton_schulz(x.to(dt))
    with pytest.raises(_lib.TcmiError, match="GPU"):
        linalg.newton_schulz(x)


def test_abi_refuses_before_a_launch():
    lib = _lib.lib()
    co = linalg._host_doubles(linalg.NS_COEFFICIENTS * 5)
    p = 1 << 20
    args = (p, 400, 1, 160000, p, 400, 400, 1, 5, co, 1e-7, 1, None, 0, p, 1 << 40, _lib.TCMI_F32, None)

    def changed(**kw):
        a = list(args)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return lib.tcmi_newton_schulz(*a)

    assert changed(_0=None) == -1 and changed(_4=None) == -1 and changed(_14=None) == -1
    assert changed(_5=0) == -1 and changed(_7=65536) == -1 and changed(_8=17) == -1 and changed(_16=_lib.TCMI_C128) == -1
    assert changed(_15=16) == -1 and b"workspace" in lib.tcmi_last_error()
    assert changed(_14=p + 8) == -1 and b"aligned" in lib.tcmi_last_error()
    assert changed(_9=linalg._host_doubles((30.0, 0.0, 0.0) * 5)) == -1 and b"past 64" in lib.tcmi_last_error()
    assert lib.tcmi_ns_work_bytes(4, 4, 1, 5, 1, _lib.TCMI_F32, 9) == -1
    assert lib.tcmi_lce_work_bytes(None, 4, None, 4, 0, 4, 4, _lib.TCMI_F32, 0) == -1
    assert lib.tcmi_linear_cross_entropy(p, 3, p, 4, None, p, -100, 2, 4, 4, p, p, None, None, 0, 0, p, 1 << 40, _lib.TCMI_F32, None) == -1
    assert lib.tcmi_linear_cross_entropy_grad(p, 4, p, 4, None, p, -100, 2, 4, 4, p, p, 0, None, None, None, None, p, 1 << 40,
                                              _lib.TCMI_F32, None) == -1


def test_linear_cross_entropy_refusals():
    f = torchnn.linear_cross_entropy
    h, w, y = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="reduction"):
        f(h, w, y, reduction="max")
    with pytest.raises(ValueError, match="weight"):
        f(h, torch.zeros(5, 3), y)
    with pytest.raises(ValueError, match="target"):
        f(h, w, y[:2])
    with pytest.raises(ValueError, match="bias"):
        f(h, w, y, bias=torch.zeros(4))
    with pytest.raises(ValueError, match="one class"):
        f(h, torch.zeros(0, 4), y)
    with pytest.raises(TypeError, match="weight"):
        f(h, w.half(), y)
    with pytest.raises(TypeError, match="int64"):
        f(h, w, y.int())
    with pytest.raises(TypeError):
        f(h.double(), w.double(), y)
    with pytest.raises(TypeError, match="real"):
        f(h.to(torch.complex64), w.to(torch.complex64), y)
    with pytest.raises(_lib.TcmiError, match="GPU"):
        f(h, w, y)
    with pytest.raises(ValueError, match="reduction"):
        torchnn.LinearCrossEntropy(4, 5, reduction="max")


def test_muon_refusals():
    p, g, v = torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(3, 4)
    f = torchnn.muon_step
    with pytest.raises(ValueError, match="axes"):
        f(p[0], g[0], v[0])
    with pytest.raises(ValueError, match="shape"):
        f(p, g[:2], v)
    with pytest.raises(TypeError, match="grad"):
        f(p, g.half(), v)
    with pytest.raises(TypeError, match="float32"):
        f(p.half(), g.half(), v.half())
    with pytest.raises(TypeError):
        f(p.double(), g.double(), v)
    with pytest.raises(TypeError, match="real"):
        f(p.to(torch.complex64), g.to(torch.complex64), v)
    with pytest.raises(ValueError, match="adjust"):
        f(p, g, v, adjust_lr_fn="other")
    with pytest.raises(ValueError, match="momentum"):
        f(p, g, v, momentum=1.0)
    with pytest.raises(ValueError, match="share"):
        f(torch.zeros(1, 4).expand(3, 4), g, v)
    with pytest.raises(_lib.TcmiError, match="GPU"):
        f(p, g, v)
    w = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="axes"):
        torchnn.Muon([w])
    with pytest.raises(ValueError):
        torchnn.Muon([torch.nn.Parameter(p)], lr=-1.0)


def test_muon_state_survives_a_checkpoint():
    """The momentum stays float32 for 16-bit parameters (torch casts loaded state to the parameter's dtype)."""
    w = torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.bfloat16))
    a = torchnn.Muon([w])
    a.state[w]["momentum_buffer"] = torch.full((3, 4), 1.0 + 2.0 ** -20)
    b = torchnn.Muon([w])
    b.load_state_dict(a.state_dict())
    got = b.state[w]["momentum_buffer"]
    assert got.dtype == torch.float32 and bool((got == 1.0 + 2.0 ** -20).all())


def test_muon_step_gets_its_own_options_only(monkeypatch):
    """a learning-rate scheduler leaves keys of its own in the parameter groups"""
    w = torch.nn.Parameter(torch.zeros(3, 4))
    opt = torchnn.Muon([w], lr=0.5, ns_steps=3)
    sched = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.1)
    seen = []
    monkeypatch.setattr(torchnn, "muon_step", lambda p, g, v, **kw: seen.append((v.dtype, kw)))
    w.grad = torch.ones(3, 4)
    opt.step()
    sched.step()
    opt.step()
    assert [kw["lr"] for _, kw in seen] == [0.5, 0.05] and all(kw["ns_steps"] == 3 and "initial_lr" not in kw for _, kw in seen)
    assert seen[0][0] == torch.float32


def test_shared_memory_and_long_sides_are_refused():
    p = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="share memory"):
        torchnn.muon_step(p, torch.zeros(3, 4), p)
    lib = _lib.lib()
    f32 = _lib.TCMI_F32
    assert lib.tcmi_ns_work_bytes(8, 1 << 24, 1, 5, 1, f32, 0) > 0            # few rows: any length
    assert lib.tcmi_ns_work_bytes(200, 1 << 21, 1, 5, 1, f32, 0) > 0
    assert lib.tcmi_ns_work_bytes(200, (1 << 21) + 1, 1, 5, 1, f32, 0) == -1  # 32-bit offsets of a product's rows
    assert lib.tcmi_ns_work_bytes(200, (1 << 21) + 1, 1, 5, 0, _lib.TCMI_BF16, 0) > 0
    assert lib.tcmi_lce_work_bytes(None, 64, None, 64, (1 << 21) + 1, 64, 100, f32, 0) == -1
    assert lib.tcmi_lce_work_bytes(None, 64, None, 64, 1 << 21, 64, 100, f32, 0) > 0


def test_newton_schulz_form_goes_by_the_steps_growth():
    """Two passes keep a polynomial of G G^H apart from G; past 2^18 (ten steps of the default) the iterated form needs its room,
    and a row longer than that form takes is refused."""
    lib = _lib.lib()
    f32 = _lib.TCMI_F32

    def room(rows, cols, steps, what, co=linalg.NS_COEFFICIENTS):
        return lib.tcmi_ns_work_bytes_coef(rows, cols, 1, steps, linalg._host_doubles(co * steps), 1, f32, what)

    for what in (_lib.NS_WORK, _lib.NS_WORK_SAVING, _lib.NS_SAVED, _lib.NS_WORK_GRAD):
        assert 0 < room(8, 2000, 10, what) < room(8, 2000, 11, what)
        assert room(8, 2000, 16, what, (1.5, -0.5, 0.0)) < room(8, 2000, 11, what)
        assert lib.tcmi_ns_work_bytes(8, 2000, 1, 5, 1, f32, what) >= max(room(8, 2000, 5, what), room(8, 2000, 5, what, (8.0, -2.0, 0.1)))
        assert room(8, 1 << 24, 10, what) > 0 and room(8, 1 << 24, 11, what) == -1
    assert room(24, 28, 5, 9) == -1


def test_forward_mode_tangents_are_refused():
    """the kernels know no tangent: without a refusal it would vanish and the derivative be zero"""
    from torch.autograd import forward_ad

    x, t = torch.ones(3, 4), torch.ones(3, 4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            linalg._tracked(dual)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            linalg._tracked(x, None, dual)
        for k in range(3):
            args = [torch.zeros(3, 4) for _ in range(3)]
            args[k] = forward_ad.make_dual(args[k], t)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torchnn.muon_step(*args)
        assert not linalg._tracked(x, 3.0)
    assert not linalg._tracked(x)


def test_muon_refuses_views_that_negate():
    z = torch.zeros(3, 4, dtype=torch.complex64).conj().imag
    assert z.is_neg()
    for args in ((z, torch.zeros(3, 4), torch.zeros(3, 4)), (torch.zeros(3, 4), torch.zeros(3, 4), z)):
        with pytest.raises(ValueError, match="negates"):
            torchnn.muon_step(*args)
