"""The training operators on the GPU against plain 64-bit formulas.

Tolerances (2-norms, derived from the number formats, not from runs):

* newton_schulz.  A step multiplies an error by at most max |p'| = 3.45 (p the default polynomial on [0, 1.2]).  A two-piece
  product is off by 2^-22 of the operands' norms for each of the three products of a step plus the f32 carry: 4 units, so
  float32 stays within 4 * 2^-22 * (3.45^0 + ... + 3.45^4) = 2e-4.  float16 adds half its step, 2^-11; bfloat16 half its step,
  2^-8, and one-piece operands at 2^-11 for three operands in five steps, which meet the directions of large singular
  values only, |p'| <= 2.2 there: 15 * 2.2 * 2^-11 = 1.6e-2.
* its gradient: the same units (8 a step: six two-piece products and the carries), five steps, relative to what the
  cotangent could have grown to: 40 * 2^-22 * 3.45^5 |dY| / |D_0|.
* linear_cross_entropy: a logit is off by (2^-21 + D 2^-24) sum |h||w| in f32, by D 2^-24 sum |h||w| from 16-bit operands (their
  products are exact).  P then is off by twice that of the probability plus 2^-21 (two pieces) or 2^-11 (one f16 piece) of itself
  plus half of f16's smallest step under its scale (_ce64), the sums by sqrt(K) 2^-22; a gradient is held to that times
  |P| |w| (|P|^T |h|) plus half a step of the type it is returned in.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
DEFAULT = ((A, B, C),) * 5
# half a step of a type with s significant bits: neighbours are 2^(1 - s) apart relative to the lower end of a binade
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.complex64: 2.0 ** -24}


def _rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    wide = torch.complex64 if dtype == torch.complex64 else torch.float32
    return torch.randn(*shape, generator=g, dtype=wide).to(dtype)


def _ns64(x, coef=DEFAULT, eps=1e-7):
    """the definition, on the CPU in 64 bits"""
    x = x.to(torch.complex128 if x.is_complex() else torch.float64)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    for a, b, c in coef:
        s = x @ x.mH
        x = a * x + (b * s + c * s @ s) @ x
    return x.mT if tall else x


def _rel(got, want):
    got = got.detach().cpu().to(want.dtype)
    return float(torch.linalg.vector_norm(got - want) / torch.linalg.vector_norm(want))


def _ns_tol(dtype, steps=5):
    f32 = 4 * 2.0 ** -22 * sum(3.45 ** k for k in range(steps))
    return f32 + HALF_STEP[dtype] + (3 * steps * 2.2 * 2.0 ** -11 if dtype == torch.bfloat16 else 0.0)


SHAPES = [(1, 1), (1, 7), (9, 1), (3, 3), (24, 28), (63, 65), (64, 64), (65, 130), (130, 65), (128, 256), (200, 129), (129, 511),
          (1, 3000), (7, 1500), (2000, 16), (40, 900), (33, 1100), (64, 777)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.complex64]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_newton_schulz(shape, dtype):
    from tcmi import linalg

    x = _rand(1, 2, *shape, dtype=dtype)
    got = linalg.newton_schulz(x.cuda())
    assert got.dtype == dtype and got.shape == x.shape
    assert _rel(got, _ns64(x)) < _ns_tol(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_newton_schulz_strides_and_batches(dtype):
    from tcmi import linalg

    base = _rand(2, 3, 2, 80, 50, dtype=dtype)
    dev = base.cuda()
    for f in (lambda t: t.mT, lambda t: t[:, :, ::2, 1::3], lambda t: t[1:, 0], lambda t: t[:, :, :1].expand(3, 2, 40, 50),
              lambda t: t.transpose(0, 2), lambda t: t[0, 0]):
        x, want = f(dev), _ns64(f(base))
        assert _rel(linalg.newton_schulz(x), want) < _ns_tol(dtype)
    if dtype == torch.complex64:
        assert _rel(linalg.newton_schulz(dev.mH), _ns64(base.mH)) < _ns_tol(dtype)


@pytest.mark.parametrize("dtype,shape", [
    (torch.bfloat16, (700, 900)), (torch.bfloat16, (2300, 2100)), (torch.bfloat16, (3900, 4100)), (torch.bfloat16, (3, 70, 5000)),
    (torch.float32, (1500, 1601)), (torch.float32, (8, 500, 300)), (torch.float32, (96, 4124)), (torch.float16, (1030, 260)),
    (torch.complex64, (20, 130, 250)), (torch.complex64, (40, 3000))])
def test_newton_schulz_larger(dtype, shape):
    """sizes at which every tile shape, the split products and the two passes are chosen; the 64-bit formula on the GPU"""
    from tcmi import linalg

    x = _rand(98, *shape, dtype=dtype).cuda()
    want = _ns64(x)
    got = linalg.newton_schulz(x)
    assert float((got.to(want.dtype) - want).norm() / want.norm()) < _ns_tol(dtype)
    if dtype != torch.bfloat16 or shape[-1] < 1000:
        dy = _rand(99, *shape, dtype=dtype).cuda()
        leaf = x.clone().requires_grad_()
        (g,) = torch.autograd.grad(linalg.newton_schulz(leaf), leaf, dy)
        ref = _ns_grad64(x, dy)
        for a, b, c, d in ((x, dy, g, ref),) if x.dim() == 2 else zip(x, dy, g, ref):
            assert _rel(c, d.cpu()) < _ns_grad_tol(a, b, d, dtype)


def test_newton_schulz_past_32_bits():
    """more than 2^31 elements: the last matrix of a batch"""
    from tcmi import linalg

    x = torch.empty(41, 60, 900001, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(33)
    for i in range(41):
        x[i].normal_(generator=g)
    got = linalg.newton_schulz(x)
    for i in (0, 40):
        want = _ns64(x[i])
        assert float((got[i].double() - want).norm() / want.norm()) < _ns_tol(torch.float32)
        assert float((got[i, -1, -1000:].double() - want[-1, -1000:]).norm() / want[-1, -1000:].norm()) < _ns_tol(torch.float32)


def test_newton_schulz_low_rank_and_graded():
    """directions 1e-2 .. 1e-4 of the largest: the ones five steps amplify by up to 485"""
    from tcmi import linalg

    for seed, x in enumerate((_rand(3, 200, 8) @ _rand(4, 8, 300) + 0.03 * _rand(5, 200, 300),
                              _rand(6, 150, 150) * torch.logspace(0, -3, 150))):
        for dtype in (torch.float32, torch.bfloat16):
            y = x.to(dtype)
            assert _rel(linalg.newton_schulz(y.cuda()), _ns64(y)) < _ns_tol(dtype), (seed, dtype)


def test_newton_schulz_converges_to_the_polar_factor():
    from tcmi import linalg

    u, _, vh = torch.linalg.svd(_rand(7, 90, 60, dtype=torch.complex64).to(torch.complex128), full_matrices=False)
    x = ((u * torch.linspace(0.5, 1.5, 60)) @ vh).to(torch.complex64)
    q = linalg.newton_schulz(x.cuda(), steps=16, coefficients=(1.5, -0.5, 0.0))
    # |p'| <= 1.5 and falls to 0 at the fixed point; 16 steps of at most 4 units each, grown 1.5^12 times before that
    assert _rel(q, u @ vh) < 16 * 4 * 2.0 ** -22 * 1.5 ** 12 / 10
    per_step = [(A, B, C)] * 3 + [(1.5, -0.5, 0.0)] * 2
    assert _rel(linalg.newton_schulz(x.cuda(), coefficients=per_step), _ns64(x, per_step)) < _ns_tol(torch.complex64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.complex64])
@pytest.mark.parametrize("shape", [(20, 30), (10, 1500), (150, 140)])
def test_newton_schulz_special_values(shape, dtype):
    from tcmi import linalg

    x = _rand(8, 4, *shape, dtype=dtype)
    x[1] = 0
    x[2, 3, 5] = math.nan
    x[3, 0, 0] = math.inf
    got = linalg.newton_schulz(x.cuda()).cpu()
    assert _rel(got[0], _ns64(x[0])) < _ns_tol(dtype)
    assert bool((got[1] == 0).all())
    assert bool(torch.isnan(torch.view_as_real(got) if dtype == torch.complex64 else got)[2:].all())
    for scale in (1e30, 1e-25):                           # squares outside float32
        y = (_rand(9, *shape, dtype=dtype).to(torch.complex64 if dtype == torch.complex64 else torch.float32) * scale).to(dtype)
        want = _ns64(y, eps=0.0)
        assert _rel(linalg.newton_schulz(y.cuda(), eps=0.0), want) < _ns_tol(dtype)
    for empty in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        assert linalg.newton_schulz(torch.zeros(empty, dtype=dtype, device="cuda")).shape == empty


def _ns_grad64(x, dy, coef=DEFAULT, eps=1e-7):
    x = x.to(torch.complex128 if x.is_complex() else torch.float64).requires_grad_()
    return torch.autograd.grad(_ns64(x, coef, eps), x, dy.to(x.dtype))[0]


def _ns_grad_tol(x, dy, want, dtype, eps=1e-7):
    n = torch.linalg.vector_norm(x.to(want.dtype)) + eps
    return float(40 * 2.0 ** -22 * 3.45 ** 5 * torch.linalg.vector_norm(dy.to(want.dtype)) / (torch.linalg.vector_norm(want) * n)) + HALF_STEP[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (24, 28), (64, 64), (130, 65), (129, 200),
                                   (1, 3000), (7, 1500), (2000, 16), (31, 700), (1100, 40)])
def test_newton_schulz_grad(shape, dtype):
    from tcmi import linalg

    for k in range(2):
        x, dy = _rand(10 + k, *shape, dtype=dtype), _rand(20 + k, *shape, dtype=dtype)
        leaf = x.cuda().requires_grad_()
        out = linalg.newton_schulz(leaf)
        assert _rel(out, _ns64(x)) < _ns_tol(dtype)
        (got,) = torch.autograd.grad(out, leaf, dy.cuda())
        want = _ns_grad64(x, dy)
        if shape == (1, 1) or 1 in shape:
            # X is g / |g| and p only rescales it: the radial part cancels; what is left is held to |dY| / |g|
            scale = 3.45 ** 5 * torch.linalg.vector_norm(dy.to(want.dtype)) / torch.linalg.vector_norm(x.to(want.dtype))
            assert float(torch.linalg.vector_norm(got.cpu().to(want.dtype) - want)) < float(scale) * (40 * 2.0 ** -22 + HALF_STEP[dtype])
        else:
            assert _rel(got, want) < _ns_grad_tol(x, dy, want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(8, 120), (8, 121), (240, 7), (13, 241), (17, 239), (16, 256), (32, 240), (241, 32), (60, 242)])
def test_newton_schulz_where_its_forms_meet(shape, dtype):
    """short sides around the number of columns at which one workgroup gives way to two passes, and both sides of every
    number of tiles a wave holds"""
    from tcmi import linalg

    x, dy = _rand(30, 3, *shape, dtype=dtype), _rand(31, 3, *shape, dtype=dtype)
    plain = linalg.newton_schulz(x.cuda())
    leaf = x.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf)
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    for k in range(3):
        want = _ns64(x[k])
        assert _rel(plain[k], want) < _ns_tol(dtype) and _rel(out[k], want) < _ns_tol(dtype)
        want = _ns_grad64(x[k], dy[k])
        assert _rel(got[k], want) < _ns_grad_tol(x[k], dy[k], want, dtype)


@pytest.mark.parametrize("power", [-100, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.complex64])
@pytest.mark.parametrize("shape", [(20, 30), (10, 1500), (150, 140), (160, 128)])
def test_newton_schulz_does_not_depend_on_the_scale(shape, dtype, power):
    """without eps a factor 2^k leaves the result alone and divides the gradient, far from where squares overflow"""
    from tcmi import linalg

    x, dy = _rand(32, *shape, dtype=dtype), _rand(33, *shape, dtype=dtype)
    leaf = (x * 2.0 ** power).cuda().requires_grad_()
    out = linalg.newton_schulz(leaf, eps=0.0)
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    want, grad = _ns64(x, eps=0.0), _ns_grad64(x, dy, eps=0.0)
    assert _rel(out, want) < _ns_tol(dtype) and _rel(linalg.newton_schulz(leaf.detach(), eps=0.0), want) < _ns_tol(dtype)
    assert _rel(got * 2.0 ** power, grad) < _ns_grad_tol(x, dy, grad, dtype, eps=0.0)
    # a tiny and a large cotangent
    for far in (-100, 60):
        leaf = x.cuda().requires_grad_()
        (got,) = torch.autograd.grad(linalg.newton_schulz(leaf, eps=0.0), leaf, (dy * 2.0 ** far).cuda())
        assert _rel(got * 2.0 ** -far, grad) < _ns_grad_tol(x, dy, grad, dtype, eps=0.0)


@pytest.mark.parametrize("coef", [((8.0, -22.0, 16.0),) + ((3.2, -1.408, 0.16384),) * 3, ((1.5, -0.5, 0.0),) * 6, (DEFAULT[0],)])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (150, 140)), (torch.complex64, (80, 96)), (torch.complex64, (70, 90)), (torch.float32, (200, 333))])
def test_newton_schulz_grad_with_other_coefficients(dtype, shape, coef):
    """steps that can lengthen a derivative a lot, ones that cannot, a single one; sides with and without padding"""
    from tcmi import linalg

    x, dy = _rand(34, 2, *shape, dtype=dtype), _rand(35, 2, *shape, dtype=dtype)
    leaf = x.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf, len(coef), coef if len(coef) > 1 else coef[0])
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    grow, top = 1.0, 1.0
    for a, b, c in coef:                               # the steps' largest slopes where singular values can lie
        t = np.linspace(0, 1.02 * top, 1000)
        grow *= max(1.0, np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4).max())
        top = np.abs(a * t + b * t ** 3 + c * t ** 5).max()
    for k in range(2):
        want = _ns64(x[k], coef)
        # the units of the default's tolerance, every step's error times what the steps behind it can make of it
        assert _rel(out[k], want) < 4 * 2.0 ** -22 * len(coef) * grow + HALF_STEP[dtype]
        n = torch.linalg.matrix_norm(x[k].to(want.dtype))
        want = _ns_grad64(x[k], dy[k], coef)
        tol = 8 * len(coef) * 2.0 ** -22 * grow * torch.linalg.vector_norm(dy[k].to(want.dtype)) / (torch.linalg.vector_norm(want) * n)
        assert _rel(got[k], want) < float(tol) + HALF_STEP[dtype]


@pytest.mark.parametrize("batch,rows,cols", [(1, 64, 96), (1, 128, 128), (5, 192, 208), (1, 320, 256), (1, 256, 257), (40, 128, 256), (1, 600, 576)])
def test_newton_schulz_complex_where_tiles_end_at_the_half(batch, rows, cols):
    """short sides of whole tiles (the second real part is not computed), of 64 but not of 128, split products and whole ones"""
    from tcmi import linalg

    x, dy = _rand(36, batch, rows, cols, dtype=torch.complex64), _rand(37, batch, rows, cols, dtype=torch.complex64)
    leaf = x.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf)
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    for k in {0, batch // 2, batch - 1}:
        want = _ns64(x[k])
        assert _rel(out[k], want) < _ns_tol(torch.complex64)
        want = _ns_grad64(x[k], dy[k])
        assert _rel(got[k], want) < _ns_grad_tol(x[k], dy[k], want, torch.complex64)


def test_newton_schulz_grad_against_differences():
    """and at an isometry, where the gradient of an SVD does not exist"""
    from tcmi import linalg

    q, _ = torch.linalg.qr(_rand(30, 40, 20, dtype=torch.complex64).to(torch.complex128))
    dy, step = _rand(31, 40, 20, dtype=torch.complex64).to(torch.complex128), _rand(32, 40, 20, dtype=torch.complex64).to(torch.complex128)
    x = q.to(torch.complex64)
    leaf = x.cuda().requires_grad_()
    (got,) = torch.autograd.grad(linalg.newton_schulz(leaf), leaf, dy.to(torch.complex64).cuda())
    f = lambda t: float((_ns64(x.to(torch.complex128) + t * step) * dy.conj()).real.sum())  # noqa: E731
    h = 1e-5
    fd = (f(h) - f(-h)) / (2 * h)
    mine = float((got.cpu().to(torch.complex128) * step.conj()).real.sum())
    want = _ns_grad64(x, dy)
    slack = _ns_grad_tol(x, dy, want, torch.complex64) * float(torch.linalg.vector_norm(want) * torch.linalg.vector_norm(step))
    assert abs(mine - fd) < slack + 1e-6 * abs(fd)


def test_newton_schulz_in_the_backend_transforms():
    import tcmi as tc
    from tcmi import linalg

    x, w = _rand(33, 3, 20, 12), _rand(34, 20, 12)
    wd = w.cuda()

    def energy(m):
        return (linalg.newton_schulz(m) * wd).sum()

    v, g = tc.backend.value_and_grad(energy)(x[0].cuda())
    want = _ns_grad64(x[0], w)
    assert _rel(g, want) < _ns_grad_tol(x[0], w, want, torch.float32)
    vs, gs = tc.backend.vectorized_value_and_grad(energy)(x.cuda())
    for i in range(3):
        want = _ns_grad64(x[i], w)
        assert _rel(gs[i], want) < _ns_grad_tol(x[i], w, want, torch.float32)
        assert abs(float(vs[i]) - float((_ns64(x[i]) * w.double()).sum())) < _ns_tol(torch.float32) * 20 * 12
    outs = tc.backend.vmap(linalg.newton_schulz)(x.cuda())
    assert _rel(outs, _ns64(x)) < _ns_tol(torch.float32)
    # many cotangents of one matrix
    leaf = x[0].cuda().requires_grad_()
    cot = _rand(35, 4, 20, 12)
    with pytest.raises(RuntimeError):                     # outside torch.func there is no batching rule: refused, not wrong
        torch.autograd.grad(linalg.newton_schulz(leaf), leaf, cot.cuda(), is_grads_batched=True)
    _, pull = torch.func.vjp(linalg.newton_schulz, x[0].cuda())
    many = torch.func.vmap(lambda c: pull(c)[0])(cot.cuda())
    for i in range(4):
        want = _ns_grad64(x[0], cot[i])
        assert _rel(many[i], want) < _ns_grad_tol(x[0], cot[i], want, torch.float32)
    out = linalg.newton_schulz(leaf)
    (g,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="once"):
        g.sum().backward()


# ------------------------------------------------------------------------------------------------------ cross entropy
def _ce64(h, w, y, b, ignore, reduction, dloss=None):
    """losses, lse, and the gradients with |P| |w|, |P|^T |h| next to them, in 64 bits on the CPU"""
    h, w = h.double(), w.double()
    z = h @ w.T + (0 if b is None else b.double())
    keep = y != ignore
    z = torch.where(keep[:, None], z, 0.0)
    yy = torch.where(keep, y, 0)
    lse = torch.logsumexp(z, 1)
    rows = torch.where(keep, lse - z.gather(1, yy[:, None]).squeeze(1), 0.0)
    n = keep.sum()
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n}[reduction]
    d = torch.ones_like(rows) if dloss is None else dloss.double() * torch.ones_like(rows)
    r = torch.where(keep, d / n if reduction == "mean" else d, 0.0)
    p = torch.exp(z - lse[:, None])
    # What the relative errors of P multiply: the probability itself where P = p - 1 is small against it (a logit off by e
    # moves p - 1 by e p), and 2^-18, which times the smallest of them, 2^-21, is the 2^-39 that half of f16's smallest step,
    # 2^-25, under the scale 2^14 may cost any entry.
    q = p + 2.0 ** -18
    p[torch.arange(len(y)), yy] -= 1.0
    q = torch.maximum(q, p.abs()) * r.abs()[:, None]
    p = p * r[:, None]
    hz = torch.where(keep[:, None], h, 0.0)
    return loss, (p @ w, p.T @ hz, p.sum(0)), (q @ w.abs(), q.T @ hz.abs(), q.sum(0))


def _ce_tols(h, w, dtype):
    D = h.shape[1]
    top = float((torch.nan_to_num(h.double()).abs() @ w.double().abs().T).max())
    logit = ((2.0 ** -21 if dtype == torch.float32 else 0.0) + D * 2.0 ** -24) * top
    piece = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    return logit, 2 * logit + piece


def _check_ce(h, w, y, b, dtype, reduction="mean", ignore=-100, dloss=None, keep_grads=(True, True, True)):
    from tcmi import torchnn

    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (h, w, b)]
    loss = torchnn.linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2], ignore_index=ignore, reduction=reduction)
    want, grads, sizes = _ce64(h, w, y, b, ignore, reduction, dloss)
    logit, rel = _ce_tols(h, w, dtype)
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    n = 1 if reduction != "sum" else len(y)
    assert float((loss.detach().cpu().double() - want).abs().max()) <= n * (2 * logit + 2.0 ** -21) + 2.0 ** -22 * float(want.abs().max())
    # without gradients the same kernels answer, but up to 16 rows, which have their own
    plain = torchnn.linear_cross_entropy(h.cuda(), w.cuda(), y.cuda(), None if b is None else b.cuda(), ignore_index=ignore, reduction=reduction)
    if len(y) > 16:
        assert torch.equal(plain, loss.detach())
    assert float((plain.cpu().double() - want).abs().max()) <= n * (2 * logit + 2.0 ** -21) + 2.0 ** -22 * float(want.abs().max())
    live = [t for t in leaves if t is not None]
    got = torch.autograd.grad(loss, live, None if dloss is None else dloss.cuda())
    K = max(w.shape[0], h.shape[0])
    for g, ref, size in zip(got, [x for x, t in zip(grads, leaves) if t is not None], [x for x, t in zip(sizes, leaves) if t is not None]):
        assert g.dtype == dtype and g.shape == ref.shape
        tiny = 2.0 ** -25 * math.sqrt(ref.numel()) if dtype == torch.float16 else 0.0        # f16's smallest step
        slack = (rel + math.sqrt(K) * 2.0 ** -22) * float(torch.linalg.vector_norm(size)) + HALF_STEP[dtype] * float(torch.linalg.vector_norm(ref))
        assert float(torch.linalg.vector_norm(g.cpu().double() - ref)) <= slack + tiny
    return loss, got


def _ce_inputs(seed, T, D, V, dtype, bias=True):
    h, w = _rand(seed, T, D).to(dtype), (_rand(seed + 1, V, D) / math.sqrt(D)).to(dtype)
    y = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed + 2))
    h[::5] += (3 * math.sqrt(D)) * w[y[::5]]
    b = (0.3 * _rand(seed + 3, V)).to(dtype) if bias else None
    return h, w, y, b


CE_SIZES = [(1, 1, 1), (1, 3, 2), (1, 700, 3001), (16, 257, 130), (17, 257, 130), (9, 96, 140000), (5, 28, 4096), (64, 64, 128), (129, 100, 257), (33, 192, 1000), (300, 64, 129), (257, 320, 3001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", CE_SIZES)
def test_linear_cross_entropy(size, dtype):
    _check_ce(*_ce_inputs(40, *size, dtype), dtype)
    _check_ce(*_ce_inputs(50, *size, dtype, bias=False), dtype, reduction="sum")
    h, w, y, b = _ce_inputs(60, *size, dtype)
    _check_ce(h, w, y, b, dtype, reduction="none", dloss=_rand(61, size[0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_cross_entropy_ignored_rows(dtype):
    from tcmi import torchnn

    h, w, y, b = _ce_inputs(70, 70, 40, 300, dtype)
    y[1::3] = -100
    h[1] = math.nan
    h[4] = math.inf
    loss, got = _check_ce(h, w, y, b, dtype)
    assert bool((got[0][y.cuda() == -100] == 0).all())
    _check_ce(h, w, y, b, dtype, reduction="none", dloss=_rand(71, 70))
    y2 = y.clone()
    y2[y == -100] = 7
    y2[y == 5] = 6
    _check_ce(torch.nan_to_num(h, 0.0, 0.0, 0.0), w, y2, b, dtype, ignore=7)           # an ignored class that exists
    # nothing left: 0 / 0, and no gradient
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    loss = torchnn.linear_cross_entropy(hd, wd, torch.full_like(y, -100).cuda())
    assert math.isnan(float(loss))
    for g in torch.autograd.grad(loss, (hd, wd)):
        assert bool((g == 0).all())
    loss = torchnn.linear_cross_entropy(hd, wd, torch.full_like(y, -100).cuda(), reduction="sum")
    assert float(loss.detach()) == 0.0


def test_linear_cross_entropy_special_values():
    from tcmi import torchnn

    h, w, y, b = _ce_inputs(80, 40, 30, 500, torch.float32)
    # masked classes, whole tiles of them included
    b[:290] = -math.inf
    y = 290 + y % 210
    loss, got = _check_ce(h, w, y, b, torch.float32)
    assert bool((got[1][:290] == 0).all()) and bool((got[2][:290] == 0).all())
    b[:] = torch.finfo(torch.float32).min
    b[300:] = 0.0
    y = 300 + y % 200
    _check_ce(h, w, y, b, torch.float32)
    # targets outside the classes: NaN there, the others as they were
    rows = torchnn.linear_cross_entropy(h.cuda(), w.cuda(), y.cuda(), reduction="none")
    bad = y.clone()
    bad[3], bad[9] = 500, -1
    rows2 = torchnn.linear_cross_entropy(h.cuda(), w.cuda(), bad.cuda(), reduction="none")
    mask = torch.zeros(40, dtype=torch.bool, device="cuda")
    mask[[3, 9]] = True
    assert bool(torch.isnan(rows2[mask]).all()) and torch.equal(rows2[~mask], rows[~mask])
    # a NaN feature that counts: its row is NaN, the others are not
    h2 = h.clone()
    h2[5, 2] = math.nan
    rows3 = torchnn.linear_cross_entropy(h2.cuda(), w.cuda(), y.cuda(), reduction="none")
    assert bool(torch.isnan(rows3[5])) and torch.equal(rows3[torch.arange(40) != 5], rows[torch.arange(40) != 5])
    # no rows
    for red, want in (("mean", math.nan), ("sum", 0.0)):
        leaf = torch.zeros(0, 30, device="cuda", requires_grad=True)
        wd = w.cuda().requires_grad_()
        loss = torchnn.linear_cross_entropy(leaf, wd, y[:0].cuda(), reduction=red)
        assert (math.isnan(float(loss)) if math.isnan(want) else float(loss) == want)
        gh, gw = torch.autograd.grad(loss, (leaf, wd))
        assert gh.shape == (0, 30) and bool((gw == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_cross_entropy_layouts(dtype):
    """rows apart, unaligned, transposed and broadcast operands; more than one leading axis; frozen operands"""
    from tcmi import torchnn

    wide_h, wide_w = _rand(90, 50, 200).to(dtype), _rand(91, 300, 200).to(dtype)
    y = torch.randint(0, 300, (50,), generator=torch.Generator().manual_seed(92))
    for cut in (lambda t: t[:, :128], lambda t: t[:, 1:129], lambda t: t[:, 3:67], lambda t: t[::2, :64] if len(t) == 50 else t[:, :64]):
        h, w = cut(wide_h), cut(wide_w) * 0.1
        yy = y[:len(h)]
        want = _ce64(h, w, yy, None, -100, "mean")[0]
        hd, wd = cut(wide_h.cuda()), (cut(wide_w.cuda()) * 0.1)
        got = torchnn.linear_cross_entropy(hd, wd, yy.cuda())
        logit, _ = _ce_tols(h, w, dtype)
        assert abs(float(got) - float(want)) < 2 * logit + 2.0 ** -21 * (1 + float(want))
    h, w, y, b = _ce_inputs(93, 24, 32, 77, dtype)
    one = torchnn.linear_cross_entropy(h.cuda(), w.cuda(), y.cuda(), b.cuda(), reduction="none")
    many = torchnn.linear_cross_entropy(h.cuda().reshape(2, 3, 4, 32), w.cuda(), y.cuda().reshape(2, 3, 4), b.cuda(), reduction="none")
    assert torch.equal(many.reshape(-1), one)
    turned = torchnn.linear_cross_entropy(h.cuda().t().contiguous().t(), w.cuda().t().contiguous().t(), y.cuda(), b.cuda(), reduction="none")
    assert torch.equal(turned, one)
    # a broadcast row: autograd sums its gradient
    leaf = h[:1].cuda().requires_grad_()
    loss = torchnn.linear_cross_entropy(leaf.expand(24, 32), w.cuda(), y.cuda(), b.cuda(), reduction="sum")
    (g,) = torch.autograd.grad(loss, leaf)
    _, (dh, _, _), (sh, _, _) = _ce64(h[:1].expand(24, 32), w, y, b, -100, "sum")
    _, rel = _ce_tols(h, w, dtype)
    assert float((g.cpu().double() - dh.sum(0, keepdim=True)).norm()) < 24 * (rel + HALF_STEP[dtype] + 2.0 ** -18) * float(sh.norm())
    # only one of the three wanted
    for k in range(3):
        ts = [t.cuda() for t in (h, w, b)]
        ts[k].requires_grad_()
        loss = torchnn.linear_cross_entropy(ts[0], ts[1], y.cuda(), ts[2])
        (g,) = torch.autograd.grad(loss, ts[k])
        assert g.shape == ts[k].shape
        alls = [t.cuda().requires_grad_() for t in (h, w, b)]
        ref = torch.autograd.grad(torchnn.linear_cross_entropy(alls[0], alls[1], y.cuda(), alls[2]), alls)[k]
        if k < 2:
            assert torch.equal(g, ref)
        else:
            # The bias's gradient alone is summed by another kernel than with the weight's.  Either route: T products off by
            # 2^-22 (the row factor in two pieces, or whole) and T f32 additions, 2^-24 each, of the terms |P r|; then one
            # rounding to the type returned.
            size = _ce64(h, w, y, b, -100, "mean")[2][2]
            slack = 2 * (2.0 ** -22 + len(y) * 2.0 ** -24) * size + 2 * HALF_STEP[dtype] * ref.cpu().double().abs()
            assert bool(((g - ref).cpu().double().abs() <= slack).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_cross_entropy_one_row_or_class_of_an_expanded_operand(dtype):
    """one row cut from an expanded tensor carries stride 0, whether it is the input or the weight"""
    from tcmi import torchnn

    h, w, y, _ = _ce_inputs(94, 1, 64, 300, dtype, bias=False)
    for grads in (False, True):
        hd, wd = h.cuda().requires_grad_(grads), w.cuda().requires_grad_(grads)
        want = torchnn.linear_cross_entropy(hd, wd, y.cuda())
        row = hd[0].expand(4, 64)[:1]
        assert row.stride(0) == 0
        got = torchnn.linear_cross_entropy(row, wd, y.cuda())
        assert torch.equal(got, want)
        if grads:
            for a, e in zip(torch.autograd.grad(got, (hd, wd)), torch.autograd.grad(want, (hd, wd))):
                assert torch.equal(a, e)
        # one class: the loss is log 1 and no gradient is left
        only = wd[0].expand(4, 64)[:1]
        loss = torchnn.linear_cross_entropy(hd, only, torch.zeros(1, dtype=torch.int64, device="cuda"))
        assert float(loss) == 0.0
        if grads:
            for a in torch.autograd.grad(loss, (hd, wd)):
                assert bool((a == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_cross_entropy_infinities_do_not_pass_for_numbers(dtype):
    """a weight of -inf makes every gradient that it could enter NaN, never a number at a lost scale; so does a NaN loss factor"""
    from tcmi import torchnn

    h, w, y, b = _ce_inputs(95, 40, 30, 300, dtype)
    h[:, 3] = h[:, 3].abs() + 0.5
    w[5, 3] = -math.inf
    y[y == 5] = 6
    hd, wd, bd = (t.cuda().requires_grad_() for t in (h, w, b))
    (dh,) = torch.autograd.grad(torchnn.linear_cross_entropy(hd, wd, y.cuda(), bd), hd)
    assert bool(torch.isnan(dh).all())
    for reduction, dloss in (("mean", torch.tensor(math.nan)), ("none", torch.full((40,), math.nan))):
        hd, wd, bd = (t.cuda().requires_grad_() for t in (h, w.nan_to_num(neginf=0.0), b))
        loss = torchnn.linear_cross_entropy(hd, wd, y.cuda(), bd, reduction=reduction)
        for g in torch.autograd.grad(loss, (hd, wd, bd), dloss.cuda()):
            assert bool(torch.isnan(g).all())


def test_linear_cross_entropy_in_pieces():
    """enough rows that the classes are gone through in several pieces"""
    from tcmi import torchnn

    h, w, y, b = _ce_inputs(95, 70000, 16, 4500, torch.float32)
    hd, wd, bd = (t.cuda().requires_grad_() for t in (h, w, b))
    loss = torchnn.linear_cross_entropy(hd, wd, y.cuda(), bd)
    got = torch.autograd.grad(loss, (hd, wd, bd))
    parts = [_ce64(h[i:i + 10000], w, y[i:i + 10000], b, -100, "sum") for i in range(0, 70000, 10000)]
    want = sum(float(p[0]) for p in parts) / 70000
    logit, rel = _ce_tols(h[:2000], w, torch.float32)
    assert abs(float(loss) - want) < 2 * logit + 2.0 ** -21 * (1 + want)
    refs = (torch.cat([p[1][0] for p in parts]), sum(p[1][1] for p in parts), sum(p[1][2] for p in parts))
    sizes = (torch.cat([p[2][0] for p in parts]), sum(p[2][1] for p in parts), sum(p[2][2] for p in parts))
    for g, r, s in zip(got, refs, sizes):
        assert float((g.cpu().double() * 70000 - r).norm()) < (rel + math.sqrt(70000) * 2.0 ** -22) * float(s.norm())


@pytest.mark.parametrize("dtype,size", [
    (torch.bfloat16, (2000, 300, 9000)), (torch.float32, (2000, 300, 9000)), (torch.float16, (700, 128, 40000)),
    (torch.bfloat16, (4100, 640, 33001)), (torch.float32, (130, 65, 70000)), (torch.bfloat16, (2, 1111, 20000))])
def test_linear_cross_entropy_larger(dtype, size):
    """sizes at which every tile shape and the split products are chosen; the 64-bit formula on the GPU"""
    from tcmi import torchnn

    h, w, y, b = (t.cuda() for t in _ce_inputs(96, *size, dtype))
    y[::11] = -100
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = torchnn.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="sum")
    got = torch.autograd.grad(loss, leaves)
    want, grads, sizes = _ce64(h, w, y, b, -100, "sum")
    logit, rel = _ce_tols(h[:512], w, dtype)
    assert abs(float(loss.detach()) - float(want)) <= len(y) * (2 * logit + 2.0 ** -21) + 2.0 ** -22 * float(want)
    for g, ref, sz in zip(got, grads, sizes):
        slack = (rel + math.sqrt(max(size[0], size[2])) * 2.0 ** -22) * float(sz.norm()) + HALF_STEP[dtype] * float(ref.norm())
        assert float((g.double() - ref).norm()) <= slack


def test_linear_cross_entropy_past_32_bits():
    """more than 2^31 weight elements: the last classes are read and written where they lie"""
    from tcmi import torchnn

    T, D, V = 5, 16384, 131272
    g = torch.Generator(device="cuda").manual_seed(97)
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    for i in range(0, V, 8192):
        w[i:i + 8192] = torch.randn(min(8192, V - i), D, device="cuda", generator=g) / 128
    h = torch.randn(T, D, device="cuda", generator=g).bfloat16()
    y = torch.tensor([V - 1, 0, V - 130, 65536, V - 2], device="cuda")
    z = torch.cat([h.double() @ w[i:i + 8192].double().T for i in range(0, V, 8192)], 1)
    want = torch.logsumexp(z, 1) - z.gather(1, y[:, None]).squeeze(1)
    w.requires_grad_()
    rows = torchnn.linear_cross_entropy(h, w, y, reduction="none")
    top = float((h.double().abs() @ w[:8192].detach().double().abs().T).max()) * 1.5
    assert float((rows.detach().double() - want).abs().max()) <= 2 * D * 2.0 ** -24 * top + 2.0 ** -21
    (dw,) = torch.autograd.grad(rows.sum(), w)
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    p[torch.arange(T), y] -= 1.0
    for rng in (slice(0, 64), slice(V - 200, V)):
        ref, size = p[:, rng].T @ h.double(), p[:, rng].abs().T @ h.double().abs()
        slack = (4 * D * 2.0 ** -24 * top + 2.0 ** -11 + 2.0 ** -20) * float(size.norm()) + 2.0 ** -8 * float(ref.norm())
        assert float((dw[rng].double() - ref).norm()) <= slack


# -------------------------------------------------------------------------------------------------------------- muon
def _muon64(p, g, v, lr, wd, mu, nesterov, r, coef=DEFAULT, eps=1e-7):
    p, g, v = p.double(), g.double(), v.double()
    v = mu * v + (1 - mu) * g
    u = (1 - mu) * g + mu * v if nesterov else v
    return (1 - lr * wd) * p - lr * r * _ns64(u, coef, eps), v, _ns64(u, coef, eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(24, 28), (1, 5), (9, 2000), (1500, 60), (200, 70), (70, 200), (3, 40, 30), (2, 2, 130, 64)])
def test_muon_step(shape, dtype):
    from tcmi import torchnn

    for k, (nesterov, adjust) in enumerate(((True, None), (False, "match_rms_adamw"))):
        p, g, v = (0.1 * _rand(100 + k, *shape)).to(dtype), _rand(110 + k, *shape).to(dtype), _rand(120 + k, *shape)
        m, n = shape[-2:]
        r = math.sqrt(max(1.0, m / n)) if adjust is None else 0.2 * math.sqrt(max(m, n))
        want, wv, o = _muon64(p, g, v, 0.02, 0.1, 0.9, nesterov, r)
        pd, gd, vd = p.cuda(), g.cuda(), v.cuda()
        torchnn.muon_step(pd, gd, vd, lr=0.02, weight_decay=0.1, momentum=0.9, nesterov=nesterov, adjust_lr_fn=adjust)
        assert torch.equal(gd.cpu(), g)
        assert float((vd.cpu().double() - wv).norm()) <= 2.0 ** -22 * float(wv.norm())
        slack = 0.02 * r * _ns_tol(dtype) * float(o.norm()) + (HALF_STEP[dtype] + 2.0 ** -23) * float(want.norm())
        assert float((pd.cpu().double() - want).norm()) <= slack


def test_muon_strides():
    from tcmi import torchnn

    p, g, v = 0.1 * _rand(130, 50, 40), _rand(131, 40, 50), _rand(132, 100, 40)
    want, wv, o = _muon64(p, g.t(), v[::2], 0.02, 0.1, 0.95, True, math.sqrt(50 / 40))
    big = torch.zeros(50, 80, device="cuda")
    pd = big[:, ::2]
    pd.copy_(p)
    vd = v.cuda()
    torchnn.muon_step(pd, g.cuda().t(), vd[::2], lr=0.02)
    assert float((pd.cpu().double() - want).norm()) <= 0.02 * math.sqrt(50 / 40) * _ns_tol(torch.float32) * float(o.norm()) + 2.0 ** -22 * float(want.norm())
    assert bool((big[:, 1::2] == 0).all()) and torch.equal(vd[1::2].cpu(), v[1::2])
    assert float((vd[::2].cpu().double() - wv).norm()) <= 2.0 ** -22 * float(wv.norm())


def test_muon_is_not_captured_before_its_first_step(monkeypatch):
    """a captured first step would clear the momentum on every replay: refused (the capture is only pretended here)"""
    from tcmi import torchnn

    p = torch.nn.Parameter(_rand(133, 8, 6).cuda())
    p.grad = _rand(134, 8, 6).cuda()
    opt = torchnn.Muon([p])
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="before the capture"):
            opt.step()
    assert not opt.state[p]
    opt.step()
    p.grad = _rand(135, 8, 6).cuda()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for rep in range(3):
        twin = torch.nn.Parameter(p.detach().clone())
        twin.grad = p.grad.clone()
        other = torchnn.Muon([twin])
        other.state[twin]["momentum_buffer"] = opt.state[p]["momentum_buffer"].clone()
        other.step()
        graph.replay()
        assert torch.equal(p, twin) and torch.equal(opt.state[p]["momentum_buffer"], other.state[twin]["momentum_buffer"])


# ---------------------------------------------------------------------------------------- graphs, streams, together
def test_captured_and_replayed():
    """each operator in a graph, replayed with new inputs between eager calls; two graphs alive at once"""
    from tcmi import linalg, torchnn

    xs = [_rand(140 + k, 70, 90).cuda() for k in range(4)]
    h, w, y, b = (t.cuda() for t in _ce_inputs(150, 60, 64, 200, torch.float32))
    w2, b2 = w.clone(), b.clone()

    def make():
        x, hh = xs[0].clone().requires_grad_(), h.clone().requires_grad_()
        ww = w.clone().requires_grad_()
        p, v = xs[1].clone(), xs[2].clone()

        def work():
            o = linalg.newton_schulz(x)
            (gx,) = torch.autograd.grad(o, x, xs[3])
            loss = torchnn.linear_cross_entropy(hh, ww, y, b)
            gh, gw = torch.autograd.grad(loss, (hh, ww))
            torchnn.muon_step(p, gx, v, lr=0.01)
            return o.detach(), gx, loss.detach(), gh, gw

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work()
        return graph, x, hh, ww, p, v, outs

    graphs = [make(), make()]
    for rep in range(3):
        for graph, x, hh, ww, p, v, outs in graphs:
            with torch.no_grad():
                x.copy_(xs[rep] * (1 + rep))
                hh.copy_(h * (1 + 0.1 * rep))
                p.copy_(xs[1])
                v.copy_(xs[2])
            graph.replay()
            x2, hh2, ww2 = (t.detach().clone().requires_grad_() for t in (x, hh, ww))
            o = linalg.newton_schulz(x2)
            (gx,) = torch.autograd.grad(o, x2, xs[3])
            loss = torchnn.linear_cross_entropy(hh2, ww2, y, b)
            gh, gw = torch.autograd.grad(loss, (hh2, ww2))
            p2, v2 = xs[1].clone(), xs[2].clone()
            torchnn.muon_step(p2, gx, v2, lr=0.01)
            for a, e in zip(outs + (p, v), (o.detach(), gx, loss.detach(), gh, gw, p2, v2)):
                assert torch.equal(a, e)
        torch.cuda.synchronize()


def test_repeatable_and_on_another_stream():
    from tcmi import linalg, torchnn

    x = _rand(160, 300, 200).cuda().requires_grad_()
    dy = _rand(161, 300, 200).cuda()
    h, w, y, b = (t.cuda() for t in _ce_inputs(162, 200, 64, 1000, torch.bfloat16))
    h.requires_grad_(), w.requires_grad_()

    def work():
        o = linalg.newton_schulz(x)
        loss = torchnn.linear_cross_entropy(h, w, y, b)
        return (o.detach(), torch.autograd.grad(o, x, dy)[0], loss.detach()) + torch.autograd.grad(loss, (h, w))

    first = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        for a, e in zip(g, first):
            assert torch.equal(a, e)


def test_quantumnet_head_and_muon_together():
    """a training step of a hybrid model: circuit features -> head over bitstrings -> loss -> gradients -> updates, against
    the same step in 64 bits from the features' own gradients; then a few steps run"""
    import tcmi as tc
    from tcmi import torchnn

    tc.set_dtype("complex64")
    n, layers, batch = 5, 2, 16

    def features(x, weights):
        c = tc.Circuit(n)
        for i in range(n):
            c.rx(i, theta=x[i])
        for j in range(layers):
            for i in range(n - 1):
                c.cnot(i, i + 1)
            for i in range(n):
                c.rx(i, theta=weights[2 * j, i])
                c.ry(i, theta=weights[2 * j + 1, i])
        return tc.backend.real(tc.backend.stack([c.expectation_ps(z=[i]) for i in range(n)]))

    torch.manual_seed(3)
    net = torchnn.QuantumNet(features, weights_shape=[2 * layers, n]).cuda()
    head = torchnn.LinearCrossEntropy(n, 2 ** n).cuda()
    x = torch.rand(batch, n, device="cuda")
    c = tc.Circuit(n)
    for i in range(n):
        c.ry(i, theta=0.4 * (i + 1))
    y = torch.as_tensor(np.asarray(tc.backend.numpy(c.sample(batch=batch, allow_state=True, format="sample_int")))).long().cuda()
    muon = torchnn.Muon([net.q_weights[0], head.weight], lr=0.05)
    sgd = torch.optim.SGD([head.bias], lr=0.1)
    before = [p.detach().cpu().clone() for p in (net.q_weights[0], head.weight)]
    feat = net(x)
    feat.retain_grad()
    loss = head(feat, y)
    loss.backward()
    want, (dh, dw, db), (sh, sw, sb) = _ce64(feat.detach().cpu(), before[1], y.cpu(), head.bias.detach().cpu(), -100, "mean")
    logit, rel = _ce_tols(feat.detach().cpu(), before[1], torch.float32)
    assert abs(float(loss) - float(want)) < 2 * logit + 2.0 ** -20
    for g, r, s in ((feat.grad, dh, sh), (head.weight.grad, dw, sw), (head.bias.grad, db, sb)):
        assert float((g.cpu().double() - r).norm()) < (rel + 2.0 ** -18) * float(s.norm())
    grads = [p.grad.detach().cpu().clone() for p in (net.q_weights[0], head.weight)]
    muon.step()
    sgd.step()
    for p, b0, g in zip((net.q_weights[0], head.weight), before, grads):
        m, k = g.shape
        want_p, want_v, o = _muon64(b0, g, torch.zeros_like(g), 0.05, 0.1, 0.95, True, math.sqrt(max(1.0, m / k)))
        slack = 0.05 * math.sqrt(max(1.0, m / k)) * _ns_tol(torch.float32) * float(o.norm()) + 2.0 ** -22 * float(want_p.norm())
        assert float((p.detach().cpu().double() - want_p).norm()) <= slack
        assert float((muon.state[p]["momentum_buffer"].cpu().double() - want_v).norm()) <= 2.0 ** -22 * float(want_v.norm())
    for _ in range(3):
        muon.zero_grad(), sgd.zero_grad()
        loss = head(net(x), y)
        loss.backward()
        muon.step(), sgd.step()
        assert math.isfinite(float(loss))
