"""The training operators on the GPU over the rest of their range: many steps, low rank, features and probabilities of every
size.  Against plain 64-bit formulas; tolerances are derived at each test from the number formats."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
DEFAULT = (A, B, C)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.complex64: 2.0 ** -24}


def _rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    wide = torch.complex64 if dtype == torch.complex64 else torch.float32
    return torch.randn(*shape, generator=g, dtype=wide).to(dtype)


def _rel(got, want):
    got = got.detach().cpu().to(want.dtype)
    return float(torch.linalg.vector_norm(got - want) / torch.linalg.vector_norm(want))


# ----------------------------------------------------------------------------------------- Newton-Schulz, many steps
def _step64(x, coef):
    a, b, c = coef
    s = x @ x.mH
    return a * x + (b * s + c * s @ s) @ x


def _ns64(x, coefs, eps=1e-7):
    x = x.to(torch.complex128 if x.is_complex() else torch.float64)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    for coef in coefs:
        x = _step64(x, coef)
    return x.mT if tall else x


def _twice(seed, m, n, dtype):
    """every row occurs twice"""
    return torch.cat([_rand(seed, m // 2, n, dtype=dtype)] * 2)


def _amplified(x, coefs):
    """what a relative error made in each step can have grown to at the end, from perturbations of the iterates that leave
    equal rows equal (as equal arithmetic does), times 4 for directions worse than random ones; relative to the result"""
    x = x.to(torch.complex128 if x.is_complex() else torch.float64)
    x = x / torch.linalg.matrix_norm(x)
    its = [x]
    for coef in coefs:
        its.append(_step64(its[-1], coef))
    total = 0.0
    for k in range(len(coefs)):
        d = _twice(1000 + k, *x.shape, dtype=torch.float32).to(x.dtype)
        d = d * (1e-7 * torch.linalg.matrix_norm(its[k]) / torch.linalg.matrix_norm(d))
        y = its[k] + d
        for coef in coefs[k:]:
            y = _step64(y, coef)
        total += float((y - its[-1]).norm() / its[-1].norm()) / 1e-7
    return 4.0 * total


def _two_passes(x, coefs, rank):
    """Two passes in f32 while the steps multiply no direction by more than 600: M's entries and X_0 are rounded, 3 * 2^-24
    times that factor g times sqrt(rows) against a result of at least 0.7 sqrt(rank).  In f64 (up to 2^18) the same with 2^-53,
    and the rounding of A_0, which grows by g^2."""
    g = math.prod(max(abs(c[0]), 1.0) for c in coefs)
    return 3 * (2.0 ** -24 if g <= 600 else 2.0 ** -53 * g) * g * math.sqrt(min(x.shape) / rank) / 0.7 if g <= 2.0 ** 18 else 0.0


def _many_tol(x, coefs, dtype, rank):
    """two passes, or 4 units of 2^-22 a step where X is iterated; and the rounding to the type returned"""
    return _two_passes(x, coefs, rank) + 4 * 2.0 ** -22 * _amplified(x, coefs) + HALF_STEP[dtype]


@pytest.mark.parametrize("steps", [1, 2, 5, 6, 8, 10, 11, 16])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (8, 1000)), (torch.float32, (32, 1000)), (torch.float32, (60, 1000)),
                                         (torch.float32, (24, 28)), (torch.complex64, (16, 900))])
def test_newton_schulz_many_steps_of_rows_that_occur_twice(shape, dtype, steps):
    """a direction that G does not have gets a factor a a step in every polynomial of G G^H, and must stay empty all the same"""
    from tcmi import linalg

    x = _twice(200, *shape, dtype=dtype)
    coefs = [DEFAULT] * steps
    want, tol = _ns64(x, coefs), _many_tol(x, coefs, dtype, min(shape) // 2)
    assert _rel(linalg.newton_schulz(x.cuda(), steps), want) < tol
    assert _rel(linalg.newton_schulz(x.mT.cuda(), steps), want.mT) < tol
    leaf = x.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf, steps)
    assert _rel(out, want) < tol
    # The gradient: 8 units of 2^-22 a step, against a cotangent that may grow by a a step where G has nothing.
    dy = _rand(201, *shape, dtype=dtype)
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    ref = x.to(want.dtype).requires_grad_()
    (grad,) = torch.autograd.grad(_ns64(ref, coefs), ref, dy.to(want.dtype))
    size = torch.linalg.vector_norm(dy.to(want.dtype)) * max(A ** steps, 1.0) / torch.linalg.vector_norm(x.to(want.dtype))
    assert float(torch.linalg.vector_norm(got.cpu().to(want.dtype) - grad)) < float(size) * (8 * steps * 2.0 ** -22 + HALF_STEP[dtype])


@pytest.mark.parametrize("rank", [1, 4])
@pytest.mark.parametrize("steps", [5, 8, 10, 12, 16])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (8, 1000)), (torch.float32, (32, 1000)), (torch.float32, (1000, 60)),
                                         (torch.bfloat16, (32, 1000)), (torch.complex64, (16, 900)), (torch.float32, (70, 500))])
def test_newton_schulz_many_steps_of_low_rank(shape, dtype, steps, rank):
    """What the rounding of G's entries adds to its rank grows as in any arithmetic; no singular value may pass the bound that
    the polynomial keeps them under (max p on [0, 1.21] is 1.2025, and 1.005 of that where operands have 11 bits), and the
    directions that G has keep theirs."""
    from tcmi import linalg, torchnn

    m, n = shape
    wide = torch.complex64 if dtype == torch.complex64 else torch.float32
    x = (_rand(210, m, rank, dtype=wide) @ _rand(211, rank, n, dtype=wide)).to(dtype)
    for out in (linalg.newton_schulz(x.cuda(), steps), linalg.newton_schulz(x.cuda().requires_grad_(), steps).detach()):
        out = out.cpu().to(torch.complex128 if out.is_complex() else torch.float64)
        assert float(torch.linalg.matrix_norm(out, 2)) < 1.2025 * 1.005 + 1.2 * HALF_STEP[dtype] * math.sqrt(min(m, n))
    if dtype == torch.float32:
        p, v = torch.zeros(m, n, device="cuda"), torch.zeros(m, n, device="cuda")
        torchnn.muon_step(p, x.cuda(), v, lr=1.0, weight_decay=0.0, ns_steps=steps)
        r = math.sqrt(max(1.0, m / n))
        assert float(torch.linalg.matrix_norm(p.cpu().double(), 2)) / r < 1.2025 * 1.005
        if steps <= 10 and min(m, n) <= 64:               # up to here the two passes answer as 64 bits do
            assert _rel(linalg.newton_schulz(x.cuda(), steps), _ns64(x, [DEFAULT] * steps)) < _two_passes(x, [DEFAULT] * steps, rank) + 2.0 ** -23


@pytest.mark.parametrize("steps", [5, 6, 8, 10, 16])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (128, 200)), (torch.float32, (130, 260)), (torch.float32, (400, 450)),
                                         (torch.complex64, (70, 90)), (torch.complex64, (128, 192)), (torch.float16, (144, 150))])
def test_newton_schulz_many_steps_of_equal_rows_in_different_tiles(shape, dtype, steps):
    """the products' sums are the same for equal rows wherever they lie, so the direction between them stays empty"""
    from tcmi import linalg

    x = _twice(202, *shape, dtype=dtype)
    want = _ns64(x, [DEFAULT] * steps)
    tol = 4 * 2.0 ** -22 * _amplified(x, [DEFAULT] * steps) + HALF_STEP[dtype]
    for y, z in ((x, want), (x.mT, want.mT)):
        assert _rel(linalg.newton_schulz(y.cuda(), steps), z) < tol
        assert _rel(linalg.newton_schulz(y.cuda().requires_grad_(), steps), z) < tol


STEEP = tuple((8.0, -22.0 / t ** 2, 16.0 / t ** 4) for t in (1.0, 2.479, 6.145, 15.233))        # tops of the steps before, 8^4 = 4096


@pytest.mark.parametrize("dtype,shape", [(torch.float32, (20, 700)), (torch.float32, (700, 6)), (torch.float32, (60, 500)), (torch.complex64, (16, 600))])
def test_newton_schulz_few_steep_steps(shape, dtype):
    """four steps that multiply an empty direction by 4096: f64 sums of the two passes (the form goes by the factor)"""
    from tcmi import linalg

    m, n = min(shape), max(shape)
    x = _twice(220, m, n, dtype=dtype)
    want = _ns64(x, STEEP)
    x, want = (x.mT, want.mT) if shape[0] > shape[1] else (x, want)
    assert _rel(linalg.newton_schulz(x.cuda(), 4, STEEP), want) < _many_tol(x if shape[0] < shape[1] else x.mT, STEEP, dtype, m // 2)


COEFS = [(DEFAULT,), ((1.5, -0.5, 0.0),) * 6, (DEFAULT,) * 3 + ((1.5, -0.5, 0.0),) * 2, (DEFAULT,) * 7, STEEP[:1] + ((3.2, -1.408, 0.16384),) * 3]


@pytest.mark.parametrize("coef", COEFS)
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (24, 28)), (torch.float32, (8, 900)), (torch.float32, (31, 700)),
                                         (torch.float32, (60, 300)), (torch.bfloat16, (40, 260)), (torch.float16, (300, 20)),
                                         (torch.complex64, (12, 20)), (torch.complex64, (16, 250)), (torch.complex64, (200, 14))])
def test_newton_schulz_small_and_thin_with_other_coefficients(dtype, shape, coef):
    """one workgroup and two passes: single steps, triples per step, more than five of them, steep ones"""
    from tcmi import linalg

    x, dy = _rand(230, 2, *shape, dtype=dtype), _rand(231, 2, *shape, dtype=dtype)
    steps, co = len(coef), coef if len(set(coef)) > 1 else coef[0]
    leaf = x.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf, steps, co)
    plain = linalg.newton_schulz(x.cuda(), steps, co)
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    grow, top = 1.0, 1.0
    for a, b, c in coef:                                  # the steps' largest slopes where singular values can lie
        t = torch.linspace(0, 1.02 * top, 1000, dtype=torch.float64)
        grow *= max(1.0, float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max()))
        top = float((a * t + b * t ** 3 + c * t ** 5).abs().max())
    for k in range(2):
        ref = x[k].to(torch.complex128 if dtype == torch.complex64 else torch.float64).requires_grad_()
        want = _ns64(ref, coef)
        (grad,) = torch.autograd.grad(want, ref, dy[k].to(ref.dtype))
        # 4 (gradient: 8) units of 2^-22 a step, each times what the steps behind it can make of it
        assert _rel(out[k], want.detach()) < 4 * 2.0 ** -22 * steps * grow + HALF_STEP[dtype]
        if dtype != torch.bfloat16:
            assert _rel(plain[k], want.detach()) < 4 * 2.0 ** -22 * steps * grow + HALF_STEP[dtype]
        size = torch.linalg.vector_norm(dy[k].to(ref.dtype)) / torch.linalg.matrix_norm(x[k].to(ref.dtype))
        assert float(torch.linalg.vector_norm(got[k].cpu().to(ref.dtype) - grad)) < float(size) * 8 * steps * 2.0 ** -22 * grow + HALF_STEP[dtype] * float(grad.norm())


# ------------------------------------------------------------------------------------ cross entropy over its range
def _head(seed, T, D, V, dtype, bias=True):
    h, w = _rand(seed, T, D).to(dtype), (_rand(seed + 1, V, D) / math.sqrt(D)).to(dtype)
    y = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed + 2))
    return h, w, y, (0.3 * _rand(seed + 3, V)).to(dtype) if bias else None


def _grads(h, w, y, b, reduction="mean", dloss=None):
    from tcmi import torchnn

    leaves = [t.cuda().requires_grad_() for t in (h, w, b) if t is not None]
    loss = torchnn.linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2] if b is not None else None, reduction=reduction)
    return torch.autograd.grad(loss, leaves, None if dloss is None else dloss.cuda())


@pytest.mark.parametrize("power", [-60, -30, 30, 60])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype,size", [(torch.float32, (64, 32, 128)), (torch.bfloat16, (64, 32, 128)), (torch.float32, (300, 100, 1000)),
                                        (torch.bfloat16, (200, 64, 500))])
def test_head_gradients_do_not_depend_on_the_size_of_the_features(size, dtype, bias, power):
    """h 2^k against w 2^-k has the same logits: dw goes with 2^k, dh with 2^-k and db stays, bit by bit"""
    h, w, y, b = _head(300, *size, dtype, bias)
    one = _grads(h, w, y, b)
    two = _grads(h * 2.0 ** power, w * 2.0 ** -power, y, b)
    assert torch.equal(two[0] * 2.0 ** power, one[0]) and torch.equal(two[1] * 2.0 ** -power, one[1])
    if bias:
        assert torch.equal(two[2], one[2])


def _head64(h, w, y, b, scale=None):
    """P with its row factors in 64 bits, on the inputs' device: mean over the rows, or `scale` per row"""
    z = h.double() @ w.double().T + (0 if b is None else b.double())
    p = torch.softmax(z, 1)
    p[torch.arange(len(y)), y] = -torch.where(torch.nn.functional.one_hot(y, z.shape[1]).bool(), 0.0, p).sum(1)
    r = (torch.full((len(y),), 1.0 / len(y)) if scale is None else scale).to(z)
    return z, p * r[:, None]


def _check_every_class(h, w, y, b, dtype, dloss=None):
    """Each class's row of dw (and entry of db) against its own size.  P[t][v] is off by twice its logit's error (two pieces
    per operand: 2^-22 of sum |h||w|, and the sum's sqrt(D) 2^-24; half a step of the logit and of the row's log sum), 2^-22 a unit
    of exp's argument, and 2^-21 (f32: two pieces and the factor) or 2^-11 (one f16 piece); the target's entry by 2^-23 of 1
    where the log sum's rounding meets 1 - p; an entry by 2^-24 of its class's largest; the sum over rows by sqrt(T) 2^-22."""
    from tcmi import torchnn

    leaves = [t.cuda().requires_grad_() for t in (h, w, b) if t is not None]
    loss = torchnn.linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2] if b is not None else None, reduction="mean" if dloss is None else "none")
    got = torch.autograd.grad(loss, leaves, None if dloss is None else dloss.cuda())
    h, w, y, b = (t if t is None else t.cuda() for t in (h, w, y, b))
    z, pr = _head64(h, w, y, b, None if dloss is None else dloss.cuda())
    T, D = h.shape
    top = float((h.double().abs() @ w.double().abs().T).max())
    lse = torch.logsumexp(z, 1, keepdim=True)
    logit = (2.0 ** -22 + math.sqrt(D) * 2.0 ** -24) * top + 2.0 ** -24 * (z.abs() + lse.abs())
    rel = 2 * logit + 2.0 ** -22 * (z - lse).abs() + (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11) + math.sqrt(T) * 2.0 ** -22
    r = (torch.full((T,), 1.0 / T) if dloss is None else dloss).cuda().double().abs()
    err = pr.abs() * rel
    rows = torch.arange(T)
    err[rows, y] += r * (2.0 ** -23 + 2 * logit[rows, y])
    err += 2.0 ** -24 * pr.abs().amax(0, keepdim=True)
    half = HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    ref = pr.T @ h.double()
    slack = torch.linalg.vector_norm(err.T @ h.double().abs(), dim=1) + half * torch.linalg.vector_norm(ref, dim=1) + tiny * math.sqrt(D)
    off = torch.linalg.vector_norm(got[1].double() - ref, dim=1)
    assert bool((off <= slack).all()), float((off / slack).max())
    if b is not None:
        ref = pr.sum(0)
        assert bool(((got[2].double() - ref).abs() <= err.sum(0) + half * ref.abs() + tiny).all())
    return got, pr


FALL = (0, 3, 10, 16, 20, 24, 28, 32, 36, 40, 50, 70, 90)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(1, 24, 650), (70, 40, 650), (300, 64, 1300), (200, 520, 2600)])
def test_head_gradients_of_improbable_classes(size, dtype):
    """classes of probability 2^-3 to 2^-90 in every row, each held to its own size"""
    h, w, y, b = _head(310, *size, dtype)
    b = (b.float() - math.log(2.0) * torch.tensor(FALL).float().repeat(size[2] // len(FALL))).to(dtype)
    y = y // len(FALL) * len(FALL)                        # targets among the probable ones
    got, pr = _check_every_class(h, w, y, b, dtype)
    if dtype != torch.float16:
        assert bool((got[1] != 0).any(1).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [40, 129, 300, 1000])
def test_head_gradients_of_classes_that_few_rows_know(T, dtype):
    """a class is probable in some rows and at 2^-30 .. 2^-60 in the others, in the same and in other groups of rows"""
    D, V = 40, 700
    h, w, y, b = _head(320, T, D, V, dtype)
    for k, rows in enumerate((slice(0, 20), slice(0, None, 64), slice(T // 2, None), slice(T - 1, None))):
        h[:, k] = 0.0
        h[rows, k] = 1.0
        w[:, k] = -24.0
        w[torch.arange(k, V, 5), k] = 8.0
    _check_every_class(h, w, y, b, dtype)
    g = torch.Generator().manual_seed(321)
    _check_every_class(h, w, y, b, dtype, dloss=torch.randn(T, generator=g))


def test_head_gradients_of_a_million_equal_classes():
    h, w, y, _ = _head(330, 40, 16, 1 << 20, torch.float32, bias=False)
    _check_every_class(h * 0.25, w * 0.25, y, None, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_gradients_of_certain_rows(dtype):
    """rows whose loss is 1e-9 to 1e-13: the other classes' gradients against their own size"""
    h, w, y, _ = _head(340, 96, 64, 500, dtype, bias=False)
    h = (h.float() * 0.3 + torch.linspace(26.0, 34.0, 96)[:, None] * w[y].float()).to(dtype)
    _check_every_class(h, w, y, None, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [-20, -36, -60, 40])
def test_head_gradients_with_row_factors_of_every_size(dtype, power):
    """rows 64 .. with a factor of 2^power; classes that only they know, and classes that only the others know"""
    h, w, y, b = _head(350, 128, 40, 300, dtype)
    h[:, :2] = 0.0
    h[:64, 0], h[64:, 1] = 1.0, 1.0
    w[:, :2] = 4.0
    w[::3, 0], w[1::3, 1] = -40.0, -40.0
    y[:64], y[64:] = 1 + y[:64] // 3 * 3, y[64:] // 3 * 3
    g = torch.Generator().manual_seed(351)
    d = torch.randn(128, generator=g)
    d[64:] *= 2.0 ** power
    d[5] = d[70] = 0.0
    _check_every_class(h, w, y, b, dtype, dloss=d)


@pytest.mark.parametrize("factor", [1.0, 1.0 / 1371, 0.7])
def test_head_gradients_round_the_probability_and_not_the_features(factor):
    """one float16 row: dw[v][d] = P_v r h_d is off by one piece of P r (2^-11), by the rounding to float16 (2^-11) and by the
    logit (2^-24 sum |h||w| (1 + sqrt(D)), twice), element by element; no factor touches h"""
    h, w, y, _ = _head(360, 1, 200, 900, torch.float16, bias=False)
    got = _grads(h, w, y, None, "none", torch.tensor([factor]))[1].cpu().double()
    z, pr = _head64(h, w, y, None, torch.tensor([factor]))
    want = pr.T @ h.double()
    top = float((h.double().abs() @ w.double().abs().T).max())
    rel = (1 + 2.0 ** -11) ** 2 - 1 + 4 * (1 + math.sqrt(200)) * 2.0 ** -24 * top + 2.0 ** -21 * float((z - torch.logsumexp(z, 1, keepdim=True)).abs().max())
    assert bool(((got - want).abs() <= rel * want.abs() + 2.0 ** -25).all())


def test_head_gradients_of_a_row_without_a_share():
    """a loss factor of zero leaves a row out of every gradient, whatever it holds"""
    h, w, y, b = _head(370, 50, 32, 200, torch.float32)
    d = _rand(371, 50)
    d[7] = d[20] = 0.0
    bad = h.clone()
    bad[7, 3], bad[20] = math.nan, math.inf
    one, two = _grads(h, w, y, b, "none", d), _grads(bad, w, y, b, "none", d)
    keep = torch.arange(50) != 7
    keep[20] = False
    assert torch.equal(one[0][keep], two[0][keep]) and bool((two[0][~keep] == 0).all())
    assert torch.equal(one[1], two[1]) and torch.equal(one[2], two[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(70, 40, 300), (1, 5, 7), (130, 300, 260), (40, 1030, 600), (200, 33, 5000)])
def test_head_gradients_of_features_of_every_size(size, dtype):
    """Features from 2^-60 to 1 of the largest, each column of dw and dh against its own size: columns are held under their own
    powers of two.  The slack: _check_every_class's, and for dh 2^-39 a class where P lies far below 1."""
    T, D, V = size
    h, w, y, b = _head(380, T, D, V, dtype)
    g = torch.Generator().manual_seed(381)
    h = h * torch.exp2(-torch.randint(0, 61, (D,), generator=g).float()).to(dtype)
    w = w * torch.exp2(-torch.randint(0, 61, (D,), generator=g).float()).to(dtype)
    if D > 4:
        h[:, 3] = 0.0
        w[:, 4] = 0.0
    got = [t.double() for t in _grads(h, w, y, b)]
    h, w, y, b = (t.cuda() for t in (h, w, y, b))
    z, pr = _head64(h, w, y, b)
    top = float((h.double().abs() @ w.double().abs().T).max())
    lse = torch.logsumexp(z, 1, keepdim=True)
    logit = (2.0 ** -22 + math.sqrt(D) * 2.0 ** -24) * top + 2.0 ** -24 * (z.abs() + lse.abs())
    err = pr.abs() * (2 * logit + 2.0 ** -22 * (z - lse).abs() + (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11) + math.sqrt(max(T, V)) * 2.0 ** -22)
    rows = torch.arange(T)
    err[rows, y] += (2.0 ** -23 + 2 * logit[rows, y]) / T
    for k, (mine, ref, slack) in enumerate(((got[1], pr.T @ h.double(), (err + 2.0 ** -24 * pr.abs().amax(0)).T @ h.double().abs()),
                                            (got[0], pr @ w.double(), (err + 2.0 ** -39 / T) @ w.double().abs()))):
        off, size = torch.linalg.vector_norm(mine - ref, dim=0), torch.linalg.vector_norm(slack, dim=0) + HALF_STEP[dtype] * torch.linalg.vector_norm(ref, dim=0)
        assert bool((off <= size).all()), (k, float((off / size).max()))


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    from tcmi import linalg, torchnn

    h, w, y, b = (t.cuda() for t in _head(390, 20, 8, 30, torch.float32))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: linalg.newton_schulz(dual(h)), lambda: torchnn.linear_cross_entropy(dual(h), w, y),
                     lambda: torchnn.linear_cross_entropy(h, dual(w), y), lambda: torchnn.linear_cross_entropy(h, w, y, dual(b)),
                     lambda: linalg.matmul(dual(h), dual(w).mT)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert bool(torch.isfinite(linalg.newton_schulz(h)).all())
    for f in (lambda t: linalg.newton_schulz(t), lambda t: torchnn.linear_cross_entropy(t, w, y)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (h,), (h,))


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_head_with_views_that_negate(reduction):
    """the imaginary part of a conjugate keeps its sign in the view and not in memory: as cotangent, feature, weight, bias"""
    from tcmi import torchnn

    T = 1 if reduction == "none" else 12
    h, w, y, b = (t.cuda() for t in _head(400, T, 8, 30, torch.float32))
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = torchnn.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction=reduction)
    plain = torch.autograd.grad(loss.sum(), leaves, retain_graph=True)
    # Re(conj(i loss) (1 + 2i)) = 2 loss: the cotangent arrives as the imaginary part of a conjugate
    twice = (torch.complex(torch.zeros_like(loss), loss).conj() * (1 + 2j)).real.sum()
    for a, e in zip(torch.autograd.grad(twice, leaves), plain):
        assert torch.equal(a, 2 * e)
    base = torchnn.linear_cross_entropy(h, w, y, b, reduction=reduction)
    for k in range(3):
        args = [h, w, b]
        args[k] = torch._neg_view(-args[k])
        assert args[k].is_neg()
        assert torch.equal(torchnn.linear_cross_entropy(args[0], args[1], y, args[2], reduction=reduction), base)
        args[k].requires_grad_()
        mine = torchnn.linear_cross_entropy(args[0], args[1], y, args[2], reduction=reduction)
        assert torch.equal(mine.detach(), loss.detach())
        assert torch.equal(torch.autograd.grad(mine.sum(), args[k])[0], plain[k])


# ------------------------------------------------- float32 stays float32: against the same formula evaluated in float32
@pytest.mark.parametrize("size", [(16, 257, 130), (17, 257, 130), (64, 64, 128), (129, 100, 257), (33, 192, 1000), (300, 64, 129),
                                  (257, 320, 3001), (2000, 300, 9000), (130, 65, 70000), (1021, 28, 16384), (4100, 640, 3300), (600, 4096, 90)])
def test_head_gradients_are_as_near_as_float32(size):
    """Two-piece products are off by 3 * 2^-22 of their operands at most, where one piece would be by 2.5e-4: the distance to 64
    bits stays within that and four times what the formula in float32 is off by."""
    h, w, y, b = _head(410, *size, torch.float32)
    h[::5] += (3 * math.sqrt(size[1])) * w[y[::5]]
    got = _grads(h, w, y, b)
    h, w, y, b = (t.cuda() for t in (h, w, y, b))
    exact, plain = [], []
    for out, up in ((exact, torch.float64), (plain, torch.float32)):
        x, v = h.to(up), w.to(up)
        p = torch.softmax(x @ v.T + b.to(up), 1)
        p[torch.arange(len(y)), y] -= 1
        p /= len(y)
        out += [p @ v, p.T @ x, p.sum(0)]
    for mine, want, f32 in zip(got, exact, plain):
        n = torch.linalg.vector_norm(want)
        off, usual = float(torch.linalg.vector_norm(mine.double() - want) / n), float(torch.linalg.vector_norm(f32.double() - want) / n)
        assert off <= 4 * usual + 3 * 2.0 ** -22, (off, usual)


@pytest.mark.parametrize("dtype,shape", [(torch.float32, (24, 28)), (torch.float32, (31, 700)), (torch.float32, (130, 65)), (torch.float32, (129, 200)),
                                         (torch.float32, (500, 300)), (torch.float32, (700, 900)), (torch.float32, (1030, 1100)),
                                         (torch.complex64, (14, 100)), (torch.complex64, (80, 96)), (torch.complex64, (256, 128)), (torch.complex64, (333, 300))])
def test_newton_schulz_is_as_near_as_float32(shape, dtype):
    """the result and its gradient, five steps: 20 (40) units of 2^-22, and four times what float32 is off by"""
    from tcmi import linalg

    x, dy = _rand(420, *shape, dtype=dtype).cuda(), _rand(421, *shape, dtype=dtype).cuda()
    leaf = x.clone().requires_grad_()
    out = linalg.newton_schulz(leaf)
    (grad,) = torch.autograd.grad(out, leaf, dy)
    refs = []
    for up in ((torch.complex128, torch.complex64) if x.is_complex() else (torch.float64, torch.float32)):
        z = x.to(up).requires_grad_()
        v = z.mT if shape[0] > shape[1] else z
        v = v / (torch.linalg.matrix_norm(v) + 1e-7)
        for _ in range(5):
            s = v @ v.mH
            v = A * v + (B * s + C * (s @ s)) @ v
        v = v.mT if shape[0] > shape[1] else v
        refs.append((v.detach(), torch.autograd.grad(v, z, dy.to(up))[0]))
    for k, mine in enumerate((out.detach(), grad)):
        want, f32 = refs[0][k], refs[1][k]
        n = torch.linalg.vector_norm(want)
        off, usual = float(torch.linalg.vector_norm(mine.to(want.dtype) - want) / n), float(torch.linalg.vector_norm(f32.to(want.dtype) - want) / n)
        assert off <= 4 * usual + 20 * (k + 1) * 2.0 ** -22, (k, off, usual)


# -------------------------------------------------------------------------------------- the head in torch.func's transforms
def test_head_in_the_backend_transforms():
    """vmap over inputs with a shared head, over heads, over everything; value_and_grad, gradients of sums, create_graph refused"""
    import tcmi as tc
    from tcmi import torchnn

    T, D, V = 14, 20, 70
    hs, ws = torch.stack([_rand(430 + k, T, D) for k in range(3)]).cuda(), torch.stack([_rand(440 + k, V, D) / 4 for k in range(3)]).cuda()
    bs = _rand(450, 3, V).cuda()
    ys = torch.randint(0, V, (3, T), generator=torch.Generator().manual_seed(451)).cuda()
    ys[1, 4] = -100

    def one(h, w, y, b, reduction="mean"):
        return torchnn.linear_cross_entropy(h, w, y, b, reduction=reduction)

    def eager(k, j, i, reduction="mean", cot=None):
        leaves = [t.detach().clone().requires_grad_() for t in (hs[k], ws[j], bs[j])]
        loss = one(leaves[0], leaves[1], ys[i], leaves[2], reduction)
        return loss.detach(), torch.autograd.grad(loss, leaves, torch.ones_like(loss) if cot is None else cot)

    for reduction in ("mean", "sum", "none"):
        out = torch.func.vmap(lambda h, w, y, b: one(h, w, y, b, reduction))(hs, ws, ys, bs)
        shared = torch.func.vmap(lambda h, y: one(h, ws[0], y, bs[0], reduction))(hs, ys)
        heads = torch.func.vmap(lambda w, b: one(hs[0], w, ys[0], b, reduction))(ws, bs)
        for k in range(3):
            assert torch.equal(out[k], eager(k, k, k, reduction)[0]) and torch.equal(shared[k], eager(k, 0, k, reduction)[0])
            assert torch.equal(heads[k], eager(0, k, 0, reduction)[0])
    v, g = tc.backend.value_and_grad(lambda h, w, b: one(h, w, ys[0], b), argnums=(0, 1, 2))(hs[0], ws[0], bs[0])
    want, grads = eager(0, 0, 0)
    assert torch.equal(v, want) and all(torch.equal(a, e) for a, e in zip(g, grads))
    # per-sample gradients of a shared head
    per = torch.func.vmap(torch.func.grad(lambda w, b, h, y: one(h, w, y, b), argnums=(0, 1)), in_dims=(None, None, 0, 0))(ws[0], bs[0], hs, ys)
    for k in range(3):
        _, (_, dw, db) = eager(k, 0, k)
        assert torch.equal(per[0][k], dw) and torch.equal(per[1][k], db)
    # many cotangents of one loss per row
    _, pull = torch.func.vjp(lambda h, w: one(h, w, ys[1], bs[1], "none"), hs[1], ws[1])
    cot = _rand(452, 4, T).cuda()
    dh, dw = torch.func.vmap(pull)(cot)
    for k in range(4):
        _, (eh, ew, _) = eager(1, 1, 1, "none", cot[k])
        assert torch.equal(dh[k], eh) and torch.equal(dw[k], ew)
    # without a gradient, above the rows of the kernel for few
    big = _rand(453, 2, 40, D).cuda()
    yb = torch.randint(0, V, (2, 40), generator=torch.Generator().manual_seed(454)).cuda()
    out = tc.backend.vmap(lambda h, y: one(h, ws[0], y, bs[0]), vectorized_argnums=(0, 1))(big, yb)
    for k in range(2):
        assert torch.equal(out[k], one(big[k], ws[0], yb[k], bs[0]))
    leaf = hs[0].clone().requires_grad_()
    (g,) = torch.autograd.grad(one(leaf, ws[0], ys[0], bs[0]), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="once"):
        g.sum().backward()


@pytest.mark.parametrize("power", [-145, -135, 118, 126])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (20, 30)), (torch.float32, (10, 1500)), (torch.float32, (150, 140)), (torch.float32, (160, 128)),
                                         (torch.bfloat16, (150, 140)), (torch.complex64, (10, 14)), (torch.complex64, (90, 100)), (torch.complex64, (100, 96))])
def test_newton_schulz_at_the_ends_of_float32(dtype, shape, power):
    """entries down to the smallest numbers and up to the largest, where the norm or its inverse is no float32: without eps the
    result is that of the same entries in the middle of the range"""
    from tcmi import linalg

    if dtype == torch.bfloat16:                           # its smallest step: below it k 2^power is another matrix
        power = max(power, -133)
    # a few bits each, so that no entry rounds at the lower end; 1 to 2.25 at the upper
    k = torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(460)).float()
    x = (k if power < 0 else torch.sign(k + 0.5) * (1 + k.abs() / 8)).to(dtype)
    if dtype == torch.complex64:
        x = torch.complex(x.real, torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(461)).float() / (1 if power < 0 else 16))
    far = torch.ldexp(torch.view_as_real(x) if x.is_complex() else x.float(), torch.tensor(power if power < 0 else power - 1))
    far = (torch.view_as_complex(far) if x.is_complex() else far).to(dtype)
    assert bool((far.abs() > 0).any()) and bool(torch.isfinite(torch.view_as_real(far) if x.is_complex() else far).all())
    leaf = far.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf, eps=0.0)
    near = x.cuda().requires_grad_()
    ref = linalg.newton_schulz(near, eps=0.0)
    # the same sums and products up to powers of two; the factor's mantissa may round once more
    assert _rel(out, ref.detach().cpu()) < 2.0 ** -20 + HALF_STEP[dtype]
    assert _rel(linalg.newton_schulz(far.cuda(), eps=0.0), linalg.newton_schulz(x.cuda(), eps=0.0).cpu()) < 2.0 ** -20 + HALF_STEP[dtype]
    # a cotangent that keeps the gradient in range
    dy = _rand(462, *shape, dtype=dtype).cuda()
    back = -20 if power < 0 else 20
    (got,) = torch.autograd.grad(out, leaf, dy * 2.0 ** (back + (-40 if power < 0 else 40)))
    (want,) = torch.autograd.grad(ref, near, dy * 2.0 ** (back + (-40 if power < 0 else 40)))
    p = power if power < 0 else power - 1
    got, want = (torch.view_as_real(t) if t.is_complex() else t for t in (got.cpu(), want.cpu()))
    assert _rel(torch.ldexp(got.double(), torch.tensor(p)), want.double()) < 2.0 ** -18 + HALF_STEP[dtype]


@pytest.mark.parametrize("T", [1, 30, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_head_of_rows_that_are_nearly_certain(T, dtype):
    """Rows with 1 - p of 1e-3 to 1e-6 at logits of 50 to 70.  The sum of exponentials is 1 and a little, off by a few of its
    rounding, 2^-24 (eight are allowed), and that is all that is lost of 1 - p besides the logits' own error; 2^-24 of the log
    sum, 64, would be more than 1e-6."""
    from tcmi import torchnn

    D, V = 100, 2000
    for k in range(3):
        h, w, y, _ = _head(470 + 10 * k, T, D, V, dtype, bias=False)
        wy = w[y].float()
        h = (torch.linspace(16.0, 23.0, T)[:, None] * wy / wy.square().sum(1, keepdim=True)).to(dtype)
        leaves = [t.cuda().requires_grad_() for t in (h, w, torch.full((V,), 40.0).to(dtype))]
        loss = torchnn.linear_cross_entropy(leaves[0], leaves[1], y.cuda(), leaves[2], reduction="none")
        dh, dw, db = (t.double() for t in torch.autograd.grad(loss.sum(), leaves))
        h, w, y = h.cuda(), w.cuda(), y.cuda()
        z, pr = _head64(h, w, y, leaves[2].detach(), torch.ones(T))
        rows = torch.arange(T)
        little = -pr[rows, y]
        assert 1e-8 < float(little.min()) and float(little.max()) < 1e-2
        top = float((h.double().abs() @ w.double().abs().T).max())
        logit = (2.0 ** -22 + math.sqrt(D) * 2.0 ** -24) * top + 2.0 ** -24 * 70
        rel = 2 * logit + 8 * 2.0 ** -24 / little + 2.0 ** -22 * 30 + (2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11)
        want = -torch.log1p(-little)
        assert bool(((loss.detach().double() - want).abs() <= little * (2 * logit) + 8 * 2.0 ** -24 + 2.0 ** -23 * want).all())
        err = pr.abs() * rel[:, None]
        for mine, ref, slack in ((dh, pr @ w.double(), (err + 2.0 ** -39) @ w.double().abs()),
                                 (dw, pr.T @ h.double(), (err + 2.0 ** -24 * pr.abs().amax(0)).T @ h.double().abs()), (db, pr.sum(0), err.sum(0))):
            tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
            assert bool(((mine - ref).abs() <= slack + HALF_STEP[dtype] * ref.abs() + tiny).all())


@pytest.mark.parametrize("steps", [1, 3, 8, 16])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (24, 28)), (torch.float32, (9, 2000)), (torch.float32, (1500, 60)), (torch.bfloat16, (40, 900)),
                                         (torch.float16, (3, 20, 700)), (torch.float32, (2, 100, 90))])
def test_muon_with_other_numbers_of_steps(shape, dtype, steps):
    """every form of the orthogonalisation under the optimiser step; the tolerance: 4 units of 2^-22 a step times what the steps
    can make of them (from the slopes on the singular values that these matrices have), and the rounding of param"""
    from tcmi import torchnn

    p, g, v = (0.1 * _rand(480, *shape)).to(dtype), _rand(481, *shape).to(dtype), _rand(482, *shape)
    pd, vd = p.cuda(), v.cuda()
    torchnn.muon_step(pd, g.cuda(), vd, lr=0.02, weight_decay=0.1, momentum=0.9, ns_steps=steps)
    wv = 0.9 * v.double() + 0.1 * g.double()
    u = 0.1 * g.double() + 0.9 * wv
    m, n = shape[-2:]
    o = _ns64(u, [DEFAULT] * steps)
    rate = 0.02 * math.sqrt(max(1.0, m / n))
    want = (1 - 0.02 * 0.1) * p.double() - rate * o
    assert float((vd.cpu().double() - wv).norm()) <= 2.0 ** -22 * float(wv.norm())
    s = torch.linalg.svdvals(u / torch.linalg.matrix_norm(u)[..., None, None]).reshape(-1)
    grow, total = torch.ones_like(s), torch.ones_like(s)
    for _ in range(steps):
        grow = grow * (A + 3 * B * s ** 2 + 5 * C * s ** 4).abs().clamp_min(1.0)
        total = total + grow
        s = A * s + B * s ** 3 + C * s ** 5
    one_piece = 3 * steps * 2.2 * 2.0 ** -11 if dtype == torch.bfloat16 else 0.0
    tol = min(4 * 2.0 ** -22 * float(total.max()), 1.0) + one_piece
    half = HALF_STEP[dtype]
    assert float((pd.cpu().double() - want).norm()) <= rate * tol * float(o.norm()) + (half + 2.0 ** -23) * float(want.norm())


@pytest.mark.parametrize("steps", [11, 16])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (1, 3000)), (torch.float32, (5000, 3)), (torch.float32, (3, 8, 5000)), (torch.float16, (33, 2000)),
                                         (torch.bfloat16, (16, 4500)), (torch.complex64, (1, 2100)), (torch.complex64, (2, 11, 3000)), (torch.float32, (2, 5, 900))])
def test_newton_schulz_iterated_for_few_rows(dtype, shape, steps):
    """short sides whose steps are too many for two passes: any number of rows, in the result and its gradient.  4 (8) units of
    2^-22 a step times what the steps behind it make of them at these singular values; one-piece operands 2^-11 alike"""
    from tcmi import linalg

    x, dy = _rand(490, *shape, dtype=dtype), _rand(491, *shape, dtype=dtype)
    coefs = [DEFAULT] * steps
    leaf = x.cuda().requires_grad_()
    out = linalg.newton_schulz(leaf, steps)
    (got,) = torch.autograd.grad(out, leaf, dy.cuda())
    plain = linalg.newton_schulz(x.cuda(), steps)
    ref = x.to(torch.complex128 if x.is_complex() else torch.float64).requires_grad_()
    want = _ns64(ref, coefs)
    (grad,) = torch.autograd.grad(want, ref, dy.to(ref.dtype))
    want, r = want.detach(), ref.detach()
    n = torch.linalg.matrix_norm(r)[..., None, None]
    s = torch.linalg.svdvals(r / n).reshape(-1)
    slopes = []
    for _ in range(steps):
        slopes.append((A + 3 * B * s ** 2 + 5 * C * s ** 4).abs())
        s = A * s + B * s ** 3 + C * s ** 5
    behind, total = torch.ones_like(s), torch.ones_like(s)
    for slope in reversed(slopes):
        behind = behind * slope.clamp_min(1.0)
        total = total + behind
    unit = float(total.max()) * 4 * 2.0 ** -22
    half = HALF_STEP[dtype]
    assert _rel(out, want) < unit + half
    assert _rel(plain, want) < unit + half + (float(total.max()) * 3 * 2.0 ** -11 if dtype == torch.bfloat16 else 0.0)
    size = float((torch.linalg.vector_norm(dy.to(ref.dtype)) / n.min()).abs()) * A ** steps
    assert float(torch.linalg.vector_norm(got.cpu().to(ref.dtype) - grad)) < size * 8 * steps * 2.0 ** -22 + half * float(grad.norm())
