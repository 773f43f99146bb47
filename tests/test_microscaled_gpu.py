"""GPU parity of the microscaled operators against their definition in 64 bits (``oracle/mx_oracle.py``).

Codes and scale bytes are equal to the oracle's.  Bounds of the products, element by element, with S = |A| |B| (the
product of magnitudes), u the unit roundoff of the storage type (2^-11 fp16, 2^-8 bf16, 2^-24 fp32):

* the stored operand f(x^) is rounded once: S u; where f is a 16-bit MUFU form, tanh.approx adds a relative 2^-10.9
  (sigmoid, silu 2^-20; gelu through tanh at most 0.5 |x| 2^-10.9);
* fp32 sums of n products: S n 2^-23 (accumulators may truncate, which doubles the unit roundoff);
* the result is rounded once: u |result|; 16-bit results below the smallest normal number: half of the smallest
  subnormal;
* the slope f' in its MUFU form is off by at most 2 * 2^-10.9 (tanh), 2^-18 (sigmoid, silu), and for gelu, whose
  derivative holds x (1 - t^2), by (0.5 + |x| g(x)) 2^-10.9 with g the inner derivative.
"""
import math

import pytest
import torch

from oracle import ipc_oracle as O
from oracle import mx_oracle as X

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF = [torch.float16, torch.bfloat16]
ALL = HALF + [torch.float32]
NAME = {torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
MUFU = 2.0 ** -10.9
ACTS = ["relu", "tanh", "sigmoid", "silu", "gelu", "identity"]


def _mx():
    from lich_b200 import microscaled as mx
    return mx


def _rand(shape, seed, scale=1.0, dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dt)


def _states(D, B, seed, dt):
    """Rows of very different size, a row of zeros, tiny and (in fp32, bf16) very large rows."""
    x = torch.randn(D, B, generator=torch.Generator().manual_seed(seed))
    x *= torch.exp2(torch.randint(-6, 7, (D, 1), generator=torch.Generator().manual_seed(seed + 1)).float())
    x[D // 2] = 0
    x[0, ::2] = 0
    if D > 3:
        x[1] *= 2.0 ** -20 if dt is torch.float16 else 2.0 ** -120
        if dt is not torch.float16:
            x[2] *= 2.0 ** 110
    return x.to(dt)


def _ckpt(x):
    c, s = X.store8(x)
    return c.to(DEV), s.to(DEV)


def _act_err(act, x, dt):
    """Bound of |f_device(x) - f(x)| before rounding, for 16-bit storage (fp32 uses CUDA's own functions, 4 ulp)."""
    y = O.act_forward(act, x).abs()
    if act in ("relu", "identity"):
        return torch.zeros_like(y)
    if dt is torch.float32:
        return 2.0 ** -21 * y + (2.0 ** -21 * x.abs() if act == "gelu" else 0)
    if act == "tanh":
        return MUFU * y
    if act == "gelu":
        return 0.5 * x.abs() * MUFU + 2.0 ** -20 * y
    return 2.0 ** -20 * (y + 2.0 ** -20)


def _slope_err(act, x, dt):
    if act in ("relu", "identity"):
        return torch.zeros_like(x)
    g = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)
    if dt is torch.float32:
        return 2.0 ** -20 * (1 + x.abs() * (g if act == "gelu" else 1))
    if act == "tanh":
        return torch.full_like(x, 2 * MUFU)
    if act == "gelu":
        return (0.5 + x.abs() * g) * MUFU + 2.0 ** -20
    return 2.0 ** -18 * (1 + x.abs())


def _within(got, ref, tol):
    got = got.double().cpu()
    assert got.shape == ref.shape
    over = (got - ref).abs() - tol
    assert not torch.isnan(got).any()
    assert (over <= 0).all(), f"{int((over > 0).sum())} of {over.numel()} over by up to {over.max():.3e}"


# ----------------------------------------------------------------------------------------------- 8-bit checkpoint
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("D,B", [(1, 1), (4, 31), (5, 32), (33, 33), (10, 128), (70, 264), (784, 128), (100, 777)])
def test_store_and_restore(D, B, dt):
    mx = _mx()
    x = _states(D, B, 3, dt)
    c, s = mx.empty_checkpoint(D, B, device=DEV)
    c.fill_(77), s.fill_(77)
    mx.build_checkpoint(D, B, NAME[dt])(x.to(DEV), c, s)
    rc, rs = X.store8(x)
    assert torch.equal(c.cpu(), rc) and torch.equal(s.cpu(), rs)
    xhat = X.load8(rc, rs, B)
    assert ((xhat - x.double()).abs() <= torch.exp2(rs.double() - 128).repeat_interleave(32, 0)[:B].t()).all()
    for act in ACTS:
        out = torch.full((D, B), 9.0, device=DEV, dtype=dt)
        mx.build_checkpoint_restore(D, B, act, NAME[dt])(c, s, out)
        ref = O.act_forward(act, xhat)
        ref = torch.where(ref.abs() > torch.finfo(dt).max, ref.sign() * float("inf"), ref)
        big = torch.isinf(ref) | (ref.abs() > torch.finfo(dt).max * (1 - U[dt]))  # rounds to the largest, or over it
        got = out.cpu().double()
        assert (got[big].abs() >= torch.finfo(dt).max).all()
        got[big], ref[big] = 0, 0
        _within(got, ref, _act_err(act, xhat, dt) * (~big) + U[dt] * ref.abs() * (1 + 2.0 ** -9) + TINY[dt])


@pytest.mark.parametrize("dt", ALL)
def test_store_blocks_that_are_not_finite(dt):
    mx = _mx()
    x = torch.ones(3, 70, dtype=dt)
    x[0, 3], x[1, 40], x[2, 69] = float("nan"), float("inf"), -float("inf")
    c, s = mx.empty_checkpoint(3, 70, device=DEV)
    mx.build_checkpoint(3, 70, NAME[dt])(x.to(DEV), c, s)
    rc, rs = X.store8(x)
    assert torch.equal(c.cpu(), rc) and torch.equal(s.cpu(), rs)
    out = torch.zeros(3, 70, device=DEV, dtype=dt)
    mx.build_checkpoint_restore(3, 70, "identity", NAME[dt])(c, s, out)
    assert torch.equal(out.isnan().cpu(), X.load8(rc, rs, 70).isnan())


def test_store_takes_tensors_that_start_between_vectors():
    mx = _mx()
    flat = _rand((1 + 6 * 64,), 5, dt=torch.bfloat16).to(DEV)
    x = flat[1:].view(6, 64)  # contiguous, two bytes past a 16-byte boundary
    c, s = mx.empty_checkpoint(6, 64, device=DEV)
    mx.build_checkpoint(6, 64, "bfloat16")(x, c, s)
    rc, rs = X.store8(x.cpu())
    assert torch.equal(c.cpu(), rc) and torch.equal(s.cpu(), rs)
    out = torch.zeros(1 + 6 * 64, device=DEV, dtype=torch.bfloat16)
    mx.build_checkpoint_restore(6, 64, "relu", "bfloat16")(c, s, out[1:].view(6, 64))
    assert torch.equal(out[1:].cpu().double().view(6, 64), X.load8(rc, rs, 64).clamp(min=0)) and out[0] == 0


# ----------------------------------------------------------------------------------- products with a checkpoint
SIZES = [(1, 1, 1), (10, 64, 1), (64, 784, 128), (10, 65, 17), (5, 8, 33), (128, 256, 256), (136, 264, 520),
         (100, 129, 777), (72, 1000, 96), (256, 512, 1024), (48, 40, 2048), (384, 512, 264)]


def _delta_case(M, K, B, dt, act, seed=0):
    e = _rand((M, B), seed, 0.3, dt)
    x = _rand((K, B), seed + 1, 1.5, dt)
    c, s = _ckpt(x)
    xhat = X.load8(c.cpu(), s.cpu(), B)
    a = O.act_forward(act, xhat)
    u = U[dt]
    S = e.double().abs() @ a.abs().t()
    err = (e.double().abs() @ (_act_err(act, xhat, dt) + u * a.abs() + TINY[dt]).t()) * (1 + 2.0 ** -8)
    return e, c, s, e.double() @ a.t(), err + S * B * 2.0 ** -23


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("M,K,B", SIZES)
def test_weight_delta(M, K, B, dt):
    mx = _mx()
    act = ACTS[(M + K + B) % 6]
    e, c, s, ref, err = _delta_case(M, K, B, dt, act)
    alpha = 1.0 / B
    dw = torch.full((M, K), 7.0, device=DEV)
    k = mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], alpha)
    k(dw, e.to(DEV), c, s)
    _within(dw, alpha * ref, alpha * err + 2.0 ** -23 * alpha * ref.abs())
    first = dw.clone()
    k(dw, e.to(DEV), c, s, accumulate=True)
    _within(dw, 2 * alpha * ref, 2 * alpha * err + 2.0 ** -22 * 2 * alpha * ref.abs())
    k(dw, e.to(DEV), c, s)
    assert torch.equal(dw, first)  # nothing left over from a call before
    if dt is not torch.float32:
        g = torch.full((M, K), 7.0, device=DEV, dtype=dt)
        mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], alpha, NAME[dt])(g, e.to(DEV), c, s)
        _within(g, alpha * ref, (alpha * err) * (1 + U[dt]) + U[dt] * alpha * ref.abs() + TINY[dt])


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("M,K,B", SIZES)
def test_weight_update(M, K, B, dt):
    mx = _mx()
    act = ACTS[(M + 2 * K + B) % 6]
    e, c, s, ref, err = _delta_case(M, K, B, dt, act, 10)
    w0 = _rand((M, K), 12, 0.05, dt)
    w = w0.to(DEV)
    mx.build_weight_update_checkpoint(M, K, B, act, NAME[dt], 0.01)(w, e.to(DEV), c, s)
    want = w0.double() + 0.01 * ref
    _within(w, want, (0.01 * err) * (1 + U[dt]) + (U[dt] + 2.0 ** -22) * (want.abs() + 0.01 * ref.abs()) + TINY[dt])


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("M,K,B", SIZES)
@pytest.mark.parametrize("act", ACTS)
def test_error_backward(M, K, B, dt, act):
    mx = _mx()
    w, e = _rand((M, K), 1, K ** -0.5, dt), _rand((M, B), 2, 0.3, dt)
    c, s = _ckpt(_rand((K, B), 3, 1.5, dt))
    xhat = X.load8(c.cpu(), s.cpu(), B)
    up = torch.full((K, B), 7.0, device=DEV, dtype=dt)
    mx.build_error_backward_checkpoint(M, K, B, act, NAME[dt])(w.to(DEV), e.to(DEV), c, s, up)
    acc = w.double().t() @ e.double()
    S = w.double().abs().t() @ e.double().abs()
    ref = X.backward(w, e, xhat, act)
    slope = X.slope(act, xhat).abs()
    tol = _slope_err(act, xhat, dt) * (acc.abs() + S * M * 2.0 ** -23) + slope * S * M * 2.0 ** -23
    _within(up, ref, tol * (1 + U[dt]) + (U[dt] + 2.0 ** -23) * ref.abs() + TINY[dt])


def test_gradient_against_differences():
    """The error sent up is the derivative of the layer's energy with respect to the states the checkpoint holds:
    d/dx_j sum_i e_i (W f(x))_i, by central differences in 64 bits."""
    mx = _mx()
    M, K, B = 20, 24, 40
    w, e = _rand((M, K), 4, 0.3), _rand((M, B), 5, 0.5)
    c, s = _ckpt(_rand((K, B), 6, 1.0))
    xhat = X.load8(c.cpu(), s.cpu(), B)
    for act in ("tanh", "sigmoid", "silu", "gelu"):
        up = torch.empty(K, B, device=DEV)
        mx.build_error_backward_checkpoint(M, K, B, act, "float32")(w.to(DEV), e.to(DEV), c, s, up)
        dw = torch.empty(M, K, device=DEV)
        mx.build_weight_delta_checkpoint(M, K, B, act, "float32", 1.0)(dw, e.to(DEV), c, s)

        def energy(ww, xx):
            return (e.double() * (ww @ O.act_forward(act, xx))).sum()

        h = 2.0 ** -17  # truncation h^2 |f'''| / 6 < 2^-34, rounding 2^-53 |energy| / h < 2^-28
        for k, b in ((0, 0), (7, 13), (23, 39)):
            d = torch.zeros(K, B, dtype=torch.float64)
            d[k, b] = h
            num = (energy(w.double(), xhat + d) - energy(w.double(), xhat - d)) / (2 * h)
            assert abs(num - up[k, b].double().cpu()) < 2.0 ** -16
            d = torch.zeros(M, K, dtype=torch.float64)
            d[k % M, k] = h
            num = (energy(w.double() + d, xhat) - energy(w.double() - d, xhat)) / (2 * h)
            assert abs(num - dw[k % M, k].double().cpu()) < 2.0 ** -14


def test_products_mark_states_that_were_not_finite():
    mx = _mx()
    M, K, B = 128, 256, 256
    x = _rand((K, B), 1, 1.0, torch.bfloat16)
    x[5, 40] = float("nan")
    c, s = _ckpt(x)
    w, e = _rand((M, K), 2, 0.1, torch.bfloat16).to(DEV), _rand((M, B), 3, 0.1, torch.bfloat16).to(DEV)
    up = torch.zeros(K, B, device=DEV, dtype=torch.bfloat16)
    mx.build_error_backward_checkpoint(M, K, B, "tanh", "bfloat16")(w, e, c, s, up)
    want = torch.zeros(K, B, dtype=torch.bool)
    want[5, 32:64] = True
    assert torch.equal(up.isnan().cpu(), want)
    dw = torch.zeros(M, K, device=DEV)
    mx.build_weight_delta_checkpoint(M, K, B, "tanh", "bfloat16", 1.0)(dw, e, c, s)
    assert dw[:, 5].isnan().all() and not dw[:, :5].isnan().any() and not dw[:, 6:].isnan().any()


def test_empty_and_other_streams():
    mx = _mx()
    c, s = mx.empty_checkpoint(8, 0, device=DEV)
    dw = torch.full((4, 8), 3.0, device=DEV)
    mx.build_weight_delta_checkpoint(4, 8, 0, "tanh", "float16", 1.0)(
        dw, torch.empty(4, 0, device=DEV, dtype=torch.float16), c, s)
    assert not dw.any()  # an empty batch: no gradient
    e, c, s, ref, err = _delta_case(128, 256, 512, torch.bfloat16, "tanh")
    k = mx.build_weight_delta_checkpoint(128, 256, 512, "tanh", "bfloat16", 1.0)
    outs = []
    ed = e.to(DEV)
    torch.cuda.synchronize()
    for _ in range(3):  # one workspace a stream: calls on several streams at once do not meet
        st = torch.cuda.Stream(DEV)
        with torch.cuda.stream(st):
            dw = torch.empty(128, 256, device=DEV)
            k(dw, ed, c, s)
            outs.append(dw)
    torch.cuda.synchronize()
    for dw in outs:
        _within(dw, ref, err + 2.0 ** -23 * ref.abs())


# ----------------------------------------------------------------------------------------------- 4-bit operands
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 784), (3, 31), (130, 33), (128, 128), (65, 300), (300, 777), (17, 1024)])
def test_quantize_and_restore(R, K, turned, dt):
    mx = _mx()
    x = _states(K, R, 8, dt) if turned else _states(K, R, 8, dt).t().contiguous()
    for act in ("identity", "relu"):
        q, sc = mx.empty_mxfp4(R, K, device=DEV)
        q.fill_(77), sc.fill_(77)
        mx.build_mxfp4_quantize(R, K, act, NAME[dt], turned)(x.to(DEV), q, sc)
        v = O.act_forward(act, x.double())
        val, rq, rsc = X.quant4(v.t().contiguous() if turned else v)
        assert torch.equal(sc.cpu(), rsc)  # padding rows and blocks too
        out = torch.full((R, K), 9.0, device=DEV)
        mx.build_mxfp4_restore(R, K, "float32")(q, sc, out)
        assert torch.equal(out.cpu().double(), val)
        differ = (q.cpu() != rq)  # a zero's sign bit may differ and stands for the same
        assert ((q.cpu()[differ] & 0x77) == (rq[differ] & 0x77)).all()
        for odt in HALF:
            o = torch.full((R, K), 9.0, device=DEV, dtype=odt)
            mx.build_mxfp4_restore(R, K, NAME[odt])(q, sc, o)
            assert torch.equal(o.cpu(), val.to(odt))


def test_quantize_of_other_activations():
    """f(x) in 32 bits is off by a few ulp, so a code can only differ where f(x) is that near to a rounding boundary:
    every value is one of the two neighbours of f(x) on its grid."""
    mx = _mx()
    R, K = 40, 200
    x = _rand((K, R), 9, 1.5)
    for act in ("tanh", "sigmoid", "silu", "gelu"):
        q, sc = mx.empty_mxfp4(R, K, device=DEV)
        mx.build_mxfp4_quantize(R, K, act, "float32", True)(x.to(DEV), q, sc)
        out = torch.empty(R, K, device=DEV)
        mx.build_mxfp4_restore(R, K, "float32")(q, sc, out)
        v = O.act_forward(act, x.double()).t().contiguous()
        val, _, _ = X.quant4(v)
        same = out.cpu().double() == val
        assert same.double().mean() > 1 - 2.0 ** -10
        lo, hi = X.quant4(v * (1 - 2.0 ** -19))[0], X.quant4(v * (1 + 2.0 ** -19))[0]
        o = out.cpu().double()
        assert ((o == lo) | (o == hi) | same).all()


def test_quantize_blocks_that_are_not_finite():
    mx = _mx()
    for turned in (False, True):
        x = _rand((40, 200), 3, 1.0, torch.bfloat16)
        x[7, 50], x[8, 199], x[39, 0] = float("nan"), float("inf"), -float("inf")
        q, sc = mx.empty_mxfp4(40, 200, device=DEV)
        mx.build_mxfp4_quantize(40, 200, "identity", "bfloat16", turned)((x.t().contiguous() if turned else x).to(DEV), q, sc)
        val, _, rsc = X.quant4(x)
        assert torch.equal(sc.cpu(), rsc)
        out = torch.zeros(40, 200, device=DEV)
        mx.build_mxfp4_restore(40, 200, "float32")(q, sc, out)
        assert torch.equal(out.isnan().cpu(), val.isnan())


FSIZES = [(1, 1, 1), (10, 64, 1), (1024, 1024, 1), (64, 784, 7), (129, 300, 16), (128, 128, 17), (10, 1024, 33),
          (1000, 777, 300), (256, 256, 256), (130, 2000, 129), (300, 513, 520), (64, 40, 1000), (512, 1024, 264)]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("M,K,B", FSIZES)
def test_forward(M, K, B, dt):
    mx = _mx()
    w, wq, wsc = X.quant4(_rand((M, K), 1, K ** -0.5))
    a, aq, asc = X.quant4(_rand((B, K), 2, 1.0))
    out = torch.full((M, B), 9.0, device=DEV, dtype=dt)
    mx.build_mxfp4_forward(M, K, B, NAME[dt])(wq.to(DEV), wsc.to(DEV), aq.to(DEV), asc.to(DEV), out)
    ref = w @ a.t()
    _within(out, ref, (w.abs() @ a.abs().t()) * K * 2.0 ** -23 + U[dt] * ref.abs() * (1 + 2.0 ** -8) + TINY[dt])


@pytest.mark.parametrize("M,K,B", [(64, 256, 1), (256, 512, 256)])
def test_forward_marks_what_was_not_finite(M, K, B):
    mx = _mx()
    w, a = _rand((M, K), 1), _rand((B, K), 2)
    w[3, 100] = float("nan")
    _, wq, wsc = X.quant4(w)
    _, aq, asc = X.quant4(a)
    out = torch.zeros(M, B, device=DEV)
    mx.build_mxfp4_forward(M, K, B, "float32")(wq.to(DEV), wsc.to(DEV), aq.to(DEV), asc.to(DEV), out)
    bad = out.isnan().cpu()
    assert bad[3].all() and bad.sum() == B


@pytest.mark.parametrize("backend", ["simt", "tcgen05"])
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("M,K,B", SIZES + [(33, 31, 95), (130, 259, 1029), (200, 136, 4099), (257, 513, 130)])
def test_products_of_any_size_on_either_kernel(M, K, B, dt, backend):
    """Both kernels take every shape: odd strides go through copied operands and a lane-per-column epilogue on one, tails
    of tiles, splits of the reduction on the other."""
    from lich_b200 import _native as N
    from lich_b200.tilelang_kernels import KernelConfig
    mx = _mx()
    cfg = KernelConfig(backend=backend)
    act = ACTS[(M + K + 2 * B) % 6]
    e, c, s, ref, err = _delta_case(M, K, B, dt, act, 20)
    alpha = 1.0 / B
    ed = e.to(DEV)
    g = torch.full((M, K), 7.0, device=DEV, dtype=dt)
    mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], alpha, NAME[dt], cfg)(g, ed, c, s)
    _within(g, alpha * ref, (alpha * err) * (1 + U[dt]) + U[dt] * alpha * ref.abs() + TINY[dt])
    dw = torch.full((M, K), 7.0, device=DEV)
    k = mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], alpha, "float32", cfg)
    k(dw, ed, c, s)
    k(dw, ed, c, s, accumulate=True)
    _within(dw, 2 * alpha * ref, 2 * alpha * err + 2.0 ** -22 * 2 * alpha * ref.abs())
    w0 = _rand((M, K), 22, 0.05, dt)
    w = w0.to(DEV)
    mx.build_weight_update_checkpoint(M, K, B, act, NAME[dt], 0.01, cfg)(w, ed, c, s)
    want = w0.double() + 0.01 * ref
    _within(w, want, (0.01 * err) * (1 + U[dt]) + (U[dt] + 2.0 ** -22) * (want.abs() + 0.01 * ref.abs()) + TINY[dt])
    xhat = X.load8(c.cpu(), s.cpu(), B)
    up = torch.full((K, B), 7.0, device=DEV, dtype=dt)
    mx.build_error_backward_checkpoint(M, K, B, act, NAME[dt], cfg)(w0.to(DEV), ed, c, s, up)
    acc = w0.double().t() @ e.double()
    S = w0.double().abs().t() @ e.double().abs()
    rb = X.backward(w0, e, xhat, act)
    tol = _slope_err(act, xhat, dt) * (acc.abs() + S * M * 2.0 ** -23) + X.slope(act, xhat).abs() * S * M * 2.0 ** -23
    _within(up, rb, tol * (1 + U[dt]) + (U[dt] + 2.0 ** -23) * rb.abs() + TINY[dt])
    assert N.device_status() == 0


def test_products_on_views_that_start_between_vectors():
    """Contiguous tensors two bytes past a 16-byte boundary, at sizes that take the tensor-core kernel otherwise."""
    mx = _mx()
    M, K, B, dt = 512, 1024, 2048, torch.bfloat16
    e, c, s, ref, err = _delta_case(M, K, B, dt, "tanh", 30)

    def off(t):
        flat = torch.zeros(t.numel() + 1, device=DEV, dtype=t.dtype)
        flat[1:] = t.reshape(-1).to(DEV)
        return flat[1:].view(t.shape)

    alpha = 1.0 / B
    for name in ("bfloat16", "float32"):
        out = off(torch.full((M, K), 7.0, dtype=getattr(torch, name)))
        mx.build_weight_delta_checkpoint(M, K, B, "tanh", "bfloat16", alpha, name)(out, e.to(DEV), c, s)
        u = U[out.dtype] + 2.0 ** -23
        _within(out, alpha * ref, (alpha * err) * (1 + u) + u * alpha * ref.abs() + TINY[out.dtype])
        out = torch.full((M, K), 7.0, dtype=getattr(torch, name), device=DEV)
        mx.build_weight_delta_checkpoint(M, K, B, "tanh", "bfloat16", alpha, name)(out, off(e), c, s)
        _within(out, alpha * ref, (alpha * err) * (1 + u) + u * alpha * ref.abs() + TINY[out.dtype])
    w0 = _rand((M, K), 32, 0.05, dt)
    want = w0.double() + 0.01 * ref
    w = off(w0)
    mx.build_weight_update_checkpoint(M, K, B, "tanh", "bfloat16", 0.01)(w, e.to(DEV), c, s)
    _within(w, want, (0.01 * err) * (1 + U[dt]) + (U[dt] + 2.0 ** -22) * (want.abs() + 0.01 * ref.abs()) + TINY[dt])
    xhat = X.load8(c.cpu(), s.cpu(), B)
    acc, S = w0.double().t() @ e.double(), w0.double().abs().t() @ e.double().abs()
    rb = X.backward(w0, e, xhat, "tanh")
    tol = _slope_err("tanh", xhat, dt) * (acc.abs() + S * M * 2.0 ** -23) + X.slope("tanh", xhat).abs() * S * M * 2.0 ** -23
    for ww, ee, shift in ((off(w0), e.to(DEV), False), (w0.to(DEV), off(e), False), (w0.to(DEV), e.to(DEV), True)):
        up = torch.full((K, B), 7.0, dtype=dt, device=DEV)
        up = off(up) if shift else up
        mx.build_error_backward_checkpoint(M, K, B, "tanh", "bfloat16")(ww, ee, c, s, up)
        _within(up, rb, tol * (1 + U[dt]) + (U[dt] + 2.0 ** -23) * rb.abs() + TINY[dt])


@pytest.mark.parametrize("M,K,B", [(1024, 1024, 2048), (2304, 2304, 4096), (1000, 1021, 4500), (512, 640, 4096),
                                   (2048, 4096, 4160)])
def test_delta_with_a_halved_last_round(M, K, B):
    """Shapes whose last round of tiles fills half the GPU or less: its tiles are halved along the batch.  Checked on samples of the rows against 64 bits, and bit for bit against another run."""
    from lich_b200 import _native as N
    mx = _mx()
    dt = torch.bfloat16
    e, x = _rand((M, B), 1, 0.3, dt), _rand((K, B), 2, 1.5, dt)
    c, s = mx.empty_checkpoint(K, B, device=DEV)
    mx.build_checkpoint(K, B, "bfloat16")(x.to(DEV), c, s)
    xhat = X.load8(c.cpu(), s.cpu(), B)
    a = torch.tanh(xhat)
    rows = torch.arange(0, M, max(1, M // 61))
    er, ed = e[rows].double(), e.to(DEV)
    ref, S = er @ a.t(), er.abs() @ a.abs().t()
    err = (er.abs() @ (MUFU * a.abs() + U[dt] * a.abs() + TINY[dt]).t()) * (1 + 2.0 ** -8) + S * B * 2.0 ** -23
    for name in ("float32", "bfloat16"):
        k = mx.build_weight_delta_checkpoint(M, K, B, "tanh", "bfloat16", 1.0, name)
        outs = []
        for _ in range(3):
            out = torch.full((M, K), 7.0, device=DEV, dtype=getattr(torch, name))
            k(out, ed, c, s)
            outs.append(out)
        u = U[out.dtype] + 2.0 ** -23
        _within(outs[0][rows.to(DEV)], ref, err * (1 + u) + u * ref.abs())
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    w0 = _rand((M, K), 3, 0.05, dt)
    w = w0.to(DEV)
    mx.build_weight_update_checkpoint(M, K, B, "tanh", "bfloat16", 0.01)(w, ed, c, s)
    want = w0[rows].double() + 0.01 * ref
    _within(w[rows.to(DEV)], want, (0.01 * err) * (1 + U[dt]) + (U[dt] + 2.0 ** -22) * (want.abs() + 0.01 * ref.abs()))
    assert N.device_status() == 0


@pytest.mark.parametrize("B", [3, 16, 200])
def test_forward_over_the_range_of_the_scales(B):
    """Features 2^110 and 2^-120 times the others' size, and weights that undo a factor of 2^100: every block is scaled by
    its own two powers of two, so the bound is that of equal sizes."""
    mx = _mx()
    M, K = 150, 512
    for wf, af in ((1.0, 1.0), (2.0 ** -100, 2.0 ** 100), (2.0 ** 100, 2.0 ** -100)):
        w = _rand((M, K), 1, K ** -0.5) * wf
        x = torch.randn(K, B, generator=torch.Generator().manual_seed(2)) * af
        if af == 1.0:
            x[32:64] *= 2.0 ** 110
            x[64:96] *= 2.0 ** -120
            w[5:40, 32:64] = 0  # rows without the large features
        wv, wq, wsc = X.quant4(w)
        av, aq, asc = X.quant4(x.t().contiguous())
        out = torch.full((M, B), 9.0, device=DEV)
        mx.build_mxfp4_forward(M, K, B, "float32")(wq.to(DEV), wsc.to(DEV), aq.to(DEV), asc.to(DEV), out)
        ref = wv @ av.t()
        _within(out, ref, (wv.abs() @ av.abs().t()) * K * 2.0 ** -23 + U[torch.float32] * ref.abs() + TINY[torch.float32])


def test_call_layer_takes_parameters_and_keywords():
    """A parameter is not a plain tensor and a keyword no plain call: both go through the Python operator."""
    mx = _mx()
    M, K, B = 40, 50, 60
    e, c, s, ref, err = _delta_case(M, K, B, torch.float32, "tanh")
    k = mx.build_weight_delta_checkpoint(M, K, B, "tanh", "float32", 1.0)
    dw = torch.zeros(M, K, device=DEV)
    k(dw, e.to(DEV), c, s)
    again = torch.zeros(M, K, device=DEV)
    k(again, torch.nn.Parameter(e.to(DEV), requires_grad=False), c, s)
    assert torch.equal(dw, again)
    k(again, e=e.to(DEV), codes=c, scales=s, accumulate=True)
    _within(again, 2 * ref, 2 * err + 2.0 ** -22 * 2 * ref.abs())
    with pytest.raises(ValueError):
        k(dw.half(), e.to(DEV), c, s)
    with pytest.raises(ValueError):
        k(dw, e, c, s)  # one tensor on the CPU


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("M,K,B", [(640, 640, 8), (651, 641, 3), (1000, 520, 1), (300, 2001, 15), (2000, 264, 4),
                                   (1999, 331, 2), (4096, 136, 1), (77, 5203, 5)])
def test_products_of_a_few_samples(M, K, B, dt):
    """Single samples and handfuls at sizes that take the fp32 kernels: whole and ragged rows, a reduction that is split
    over a cluster, every mode."""
    mx = _mx()
    act = ACTS[(M + K + B) % 6]
    e, c, s, ref, err = _delta_case(M, K, B, dt, act, 40)
    ed, alpha = e.to(DEV), 0.5
    dw = torch.full((M, K), 7.0, device=DEV)
    k = mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], alpha)
    k(dw, ed, c, s)
    _within(dw, alpha * ref, alpha * err + 2.0 ** -23 * alpha * ref.abs())
    k(dw, ed, c, s, accumulate=True)
    _within(dw, 2 * alpha * ref, 2 * alpha * err + 2.0 ** -22 * 2 * alpha * ref.abs())
    if dt is not torch.float32:
        g = torch.full((M, K), 7.0, device=DEV, dtype=dt)
        mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], alpha, NAME[dt])(g, ed, c, s)
        _within(g, alpha * ref, (alpha * err) * (1 + U[dt]) + U[dt] * alpha * ref.abs() + TINY[dt])
    w0 = _rand((M, K), 42, 0.05, dt)
    w = w0.to(DEV)
    mx.build_weight_update_checkpoint(M, K, B, act, NAME[dt], 0.01)(w, ed, c, s)
    want = w0.double() + 0.01 * ref
    _within(w, want, (0.01 * err) * (1 + U[dt]) + (U[dt] + 2.0 ** -22) * (want.abs() + 0.01 * ref.abs()) + TINY[dt])
    xhat = X.load8(c.cpu(), s.cpu(), B)
    acc, S = w0.double().t() @ e.double(), w0.double().abs().t() @ e.double().abs()
    rb = X.backward(w0, e, xhat, act)
    tol = _slope_err(act, xhat, dt) * (acc.abs() + S * M * 2.0 ** -23) + X.slope(act, xhat).abs() * S * M * 2.0 ** -23
    outs = []
    for shift in (0, 1):  # W on and off a boundary of two elements
        flat = torch.zeros(M * K + 1, device=DEV, dtype=dt)
        flat[shift:shift + M * K] = w0.reshape(-1).to(DEV)
        up = torch.full((K, B), 7.0, device=DEV, dtype=dt)
        mx.build_error_backward_checkpoint(M, K, B, act, NAME[dt])(flat[shift:shift + M * K].view(M, K), ed, c, s, up)
        _within(up, rb, tol * (1 + U[dt]) + (U[dt] + 2.0 ** -23) * rb.abs() + TINY[dt])
        outs.append(up)
    again = torch.full((K, B), 7.0, device=DEV, dtype=dt)
    mx.build_error_backward_checkpoint(M, K, B, act, NAME[dt])(w0.to(DEV), ed, c, s, again)
    assert torch.equal(again, outs[0])


@pytest.mark.parametrize("M,K,B", [(2048, 2048, 100), (700, 1004, 612), (900, 902, 514), (1001, 903, 501)])
def test_products_of_large_ragged_rows(M, K, B):
    """Rows on boundaries of 8, 4 and 2 bytes at sizes that take the tensor cores by themselves."""
    mx = _mx()
    dt = torch.bfloat16
    e, c, s, ref, err = _delta_case(M, K, B, dt, "silu", 50)
    ed, alpha = e.to(DEV), 1.0 / B
    for name in ("float32", "bfloat16"):
        out = torch.full((M, K), 7.0, device=DEV, dtype=getattr(torch, name))
        mx.build_weight_delta_checkpoint(M, K, B, "silu", "bfloat16", alpha, name)(out, ed, c, s)
        u = U[out.dtype] + 2.0 ** -23
        _within(out, alpha * ref, (alpha * err) * (1 + u) + u * alpha * ref.abs() + TINY[out.dtype])
    w0 = _rand((M, K), 52, 0.05, dt)
    xhat = X.load8(c.cpu(), s.cpu(), B)
    acc, S = w0.double().t() @ e.double(), w0.double().abs().t() @ e.double().abs()
    rb = X.backward(w0, e, xhat, "silu")
    tol = _slope_err("silu", xhat, dt) * (acc.abs() + S * M * 2.0 ** -23) + X.slope("silu", xhat).abs() * S * M * 2.0 ** -23
    up = torch.full((K, B), 7.0, device=DEV, dtype=dt)
    mx.build_error_backward_checkpoint(M, K, B, "silu", "bfloat16")(w0.to(DEV), ed, c, s, up)
    _within(up, rb, tol * (1 + U[dt]) + (U[dt] + 2.0 ** -23) * rb.abs() + TINY[dt])
    wv, wq, wsc = X.quant4(_rand((M, K), 53, K ** -0.5))
    av, aq, asc = X.quant4(_rand((B, K), 54))
    for odt in ALL:
        out = torch.full((M, B), 9.0, device=DEV, dtype=odt)
        mx.build_mxfp4_forward(M, K, B, NAME[odt])(wq.to(DEV), wsc.to(DEV), aq.to(DEV), asc.to(DEV), out)
        r4 = wv @ av.t()
        _within(out, r4, (wv.abs() @ av.abs().t()) * K * 2.0 ** -23 + U[odt] * r4.abs() * (1 + 2.0 ** -8) + TINY[odt])


def test_tensors_without_an_address_are_refused():
    """Under torch.vmap a tensor passes for a plain one and throws when asked for its address; a sparse one has no strides."""
    mx = _mx()
    c, s = mx.empty_checkpoint(4, 40, device=DEV)
    k = mx.build_checkpoint(4, 40, "float16")
    x = torch.zeros(3, 4, 40, device=DEV, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda t: k(t, c, s))(x)
    with pytest.raises(ValueError, match="not a dense tensor"):
        k(x[0].to_sparse(), c, s)
    k(x[0], c, s)
    assert not c.any()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("D,B", [(33, 96), (20, 131)])
def test_every_f_keeps_a_block_that_was_not_finite(D, B, dt):
    """A NaN or an infinity leaves a block of NaNs: f of it is NaN, relu's too, and a quantised f(x) is marked where f(x)
    itself is not finite."""
    mx = _mx()
    x = _rand((D, B), 60, 1.0, dt)
    x[3, 5], x[4, 40], x[5, 70] = float("nan"), float("inf"), -float("inf")
    c, s = mx.empty_checkpoint(D, B, device=DEV)
    mx.build_checkpoint(D, B, NAME[dt])(x.to(DEV), c, s)
    marked = X.load8(c.cpu(), s.cpu(), B).isnan()
    assert marked.sum() == 96
    for act in ACTS:
        out = torch.zeros(D, B, device=DEV, dtype=dt)
        mx.build_checkpoint_restore(D, B, act, NAME[dt])(c, s, out)
        assert torch.equal(out.cpu().isnan(), marked)
        for turned in (False, True):
            R, K = (B, D) if turned else (D, B)
            q, sc = mx.empty_mxfp4(R, K, device=DEV)
            mx.build_mxfp4_quantize(R, K, act, NAME[dt], turned)(x.to(DEV), q, sc)
            back = torch.zeros(R, K, device=DEV)
            mx.build_mxfp4_restore(R, K, "float32")(q, sc, back)
            v = O.act_forward(act, x.double())
            v = torch.where(x.isneginf(), torch.full_like(v, 0.0 if act != "identity" else -math.inf), v)  # (the limit)
            if act in ("silu", "gelu"):
                v[5, 70] = float("nan")  # -inf times 0, as f is computed
            if act == "tanh":
                v[5, 70] = -1.0
            want = X.quant4(v.t().contiguous() if turned else v)[0].isnan()
            assert torch.equal(back.cpu().isnan(), want)


NSIZES = [("auto", 20, 30, 3), ("auto", 700, 648, 4), ("simt", 40, 72, 200), ("simt", 33, 65, 97), ("tcgen05", 136, 264, 520),
          ("tcgen05", 130, 259, 517), ("tcgen05", 256, 512, 4608)]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("backend,M,K,B", NSIZES)
def test_products_mark_states_that_were_not_finite_on_every_kernel(backend, M, K, B, act, dt):
    """One state that overflowed marks its block in the error sent up (where f' depends on the state) and its feature in
    the weights' gradient, and nothing else."""
    from lich_b200.tilelang_kernels import KernelConfig
    if dt is torch.float32:
        backend = "auto" if backend == "tcgen05" else backend
    mx = _mx()
    cfg = KernelConfig(backend=backend)
    x = _rand((K, B), 61, 1.0, dt)
    x[5, B - 1] = float("inf")
    c, s = _ckpt(x)
    bad = X.load8(c.cpu(), s.cpu(), B).isnan()
    assert bad.any()
    w, e = _rand((M, K), 62, 0.1, dt), _rand((M, B), 63, 0.1, dt)
    up = torch.zeros(K, B, device=DEV, dtype=dt)
    mx.build_error_backward_checkpoint(M, K, B, act, NAME[dt], cfg)(w.to(DEV), e.to(DEV), c, s, up)
    assert torch.equal(up.cpu().isnan(), bad & (act != "identity"))
    want = torch.zeros(M, K, dtype=torch.bool)
    want[:, 5] = True
    for name in {"float32", NAME[dt]}:
        dw = torch.zeros(M, K, device=DEV, dtype=getattr(torch, name))
        mx.build_weight_delta_checkpoint(M, K, B, act, NAME[dt], 1.0, name, cfg)(dw, e.to(DEV), c, s)
        assert torch.equal(dw.cpu().isnan(), want)
    wd = w.to(DEV)
    mx.build_weight_update_checkpoint(M, K, B, act, NAME[dt], 0.5, cfg)(wd, e.to(DEV), c, s)
    assert torch.equal(wd.cpu().isnan(), want)


@pytest.mark.parametrize("K", [64, 512, 2000])
@pytest.mark.parametrize("B", [3, 16, 200])
def test_forward_of_scales_that_undo_one_another(B, K):
    """Weights of 2^124 times activations of 2^-124 and the other way round: a block's sum of codes is up to 1152 and
    overflows if it meets the large scale first."""
    mx = _mx()
    M = 150
    for wf, af in ((124, -124), (-124, 124), (124, -140), (-120, 110)):
        wv, wq, wsc = X.quant4(torch.exp2(torch.tensor(float(wf))) * _rand((M, K), 70))
        av, aq, asc = X.quant4((_rand((B, K), 71).double() * 2.0 ** af).float())
        out = torch.full((M, B), 9.0, device=DEV)
        mx.build_mxfp4_forward(M, K, B, "float32")(wq.to(DEV), wsc.to(DEV), aq.to(DEV), asc.to(DEV), out)
        ref = wv @ av.t()
        _within(out, ref, (wv.abs() @ av.abs().t()) * K * 2.0 ** -23 + U[torch.float32] * ref.abs() + TINY[torch.float32])


# Slopes of saturated states, and gelu of negative ones, relative to their own size.  With z the exponential e^-|2x| (tanh),
# e^-|x| (sigmoid, silu) or e^-|2u| (gelu, u its inner polynomial) and r = 1 / (1 + z), every term is a product of z, r and
# numbers of the size of x: ex2.approx is off by 2^-22, rcp.approx by 2^-23, and the exponent, of size a, by a few
# roundings of 2^-24 (gelu's u by four): 2^-19 (1 + a) in 16-bit storage, 2^-20 (1 + a) in fp32; exponentials below
# 2^-126 may be 0.
def _stable(act, x):
    """(f, f', sum of the magnitudes of the terms of f', the exponent a) in 64 bits without cancellation."""
    u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    a = {"tanh": 2 * x.abs(), "sigmoid": x.abs(), "silu": x.abs(), "gelu": 2 * u.abs()}[act]
    z = torch.exp(-a)
    r = 1 / (1 + z)
    s = torch.where(x >= 0, r, z * r)
    if act == "tanh":
        return torch.tanh(x), 4 * z * r * r, 4 * z * r * r, a
    if act == "sigmoid":
        return s, z * r * r, z * r * r, a
    t = x * z * r * r * (1 if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x))
    return x * s, s + t, s + t.abs(), a


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("act", ["tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("backend,M,K,B", [("auto", 24, 40, 3), ("simt", 40, 72, 200), ("tcgen05", 136, 264, 520)])
def test_slopes_of_saturated_states(backend, M, K, B, act, dt):
    from lich_b200.tilelang_kernels import KernelConfig
    if dt is torch.float32 and backend == "tcgen05":
        backend = "auto"
    mx = _mx()
    x = _rand((K, B), 80)
    x = (torch.sign(x) * (4 + 4 * torch.rand(K, B, generator=torch.Generator().manual_seed(81)))).to(dt)
    c, s = _ckpt(x)
    xhat = X.load8(c.cpu(), s.cpu(), B)
    w, e = _rand((M, K), 82, 0.5, dt), _rand((M, B), 83, 1.0, dt)
    up = torch.zeros(K, B, device=DEV, dtype=dt)
    mx.build_error_backward_checkpoint(M, K, B, act, NAME[dt], KernelConfig(backend=backend))(w.to(DEV), e.to(DEV), c, s, up)
    _, slope, size, a = _stable(act, xhat)
    acc, S = w.double().t() @ e.double(), w.double().abs().t() @ e.double().abs()
    ref = slope * acc
    rel = (2.0 ** -20 if dt is torch.float32 else 2.0 ** -19) * (1 + a)
    tol = (size * rel + 2.0 ** -125) * (acc.abs() + S * M * 2.0 ** -23) + slope.abs() * S * M * 2.0 ** -23
    _within(up, ref, tol * (1 + U[dt]) + (U[dt] + 2.0 ** -23) * ref.abs() + TINY[dt])


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("B", [64, 67])
def test_gelu_of_negative_states(B, dt):
    mx = _mx()
    D = 40
    x = (6 * (2 * torch.rand(D, B, generator=torch.Generator().manual_seed(90)) - 1)).to(dt)
    c, s = _ckpt(x)
    xhat = X.load8(c.cpu(), s.cpu(), B)
    out = torch.zeros(D, B, device=DEV, dtype=dt)
    mx.build_checkpoint_restore(D, B, "gelu", NAME[dt])(c, s, out)
    f, _, _, a = _stable("gelu", xhat)
    rel = (2.0 ** -20 if dt is torch.float32 else 2.0 ** -19) * (1 + a)
    _within(out, f, (rel * f.abs() + 2.0 ** -125) * (1 + U[dt]) + U[dt] * f.abs() + TINY[dt])


@pytest.mark.parametrize("act", ["tanh", "sigmoid", "silu", "gelu"])
def test_slopes_of_very_large_states(act):
    """bf16 and fp32 states far beyond where f saturates, whose squares and cubes overflow: the slope is 1 or 0."""
    mx = _mx()
    for dt in (torch.bfloat16, torch.float32):
        x = torch.tensor([1e20, -1e20, 3e13, -3e13, 1e30, -1e30, 200.0, -200.0], dtype=dt).repeat_interleave(32)[None]
        c, s = _ckpt(x)
        w, e = torch.ones(1, 1, dtype=dt, device=DEV), torch.ones(1, 256, dtype=dt, device=DEV)
        up = torch.full((1, 256), 9.0, device=DEV, dtype=dt)
        mx.build_error_backward_checkpoint(1, 1, 256, act, NAME[dt])(w, e, c, s, up)
        want = (x > 0).float() if act in ("silu", "gelu") else torch.zeros(1, 256)
        assert torch.equal(up.cpu().float(), want)


def test_forward_leaves_the_sms_it_is_told_to():
    """Under a cap of 4 CTAs the 64 tiles take 16 rounds instead of one; the result is the same."""
    from lich_b200 import _native as N
    mx = _mx()
    M = K = B = 1024
    _, wq, wsc = X.quant4(_rand((M, K), 100))
    _, aq, asc = X.quant4(_rand((B, K), 101))
    args = [t.to(DEV) for t in (wq, wsc, aq, asc)]
    k = mx.build_mxfp4_forward(M, K, B, "bfloat16")
    outs, times = [], []
    try:
        for cap in (0, 4):
            N.set_max_ctas(cap)
            out = torch.empty(M, B, device=DEV, dtype=torch.bfloat16)
            k(*args, out)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()  # (200 calls one after another: the host would take longer than the GPU)
            with torch.cuda.graph(g):
                for _ in range(200):
                    k(*args, out)
            g.replay()
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            g.replay()
            b.record()
            torch.cuda.synchronize()
            outs.append(out)
            times.append(a.elapsed_time(b))
    finally:
        N.set_max_ctas(0)
    assert torch.equal(*outs)
    assert times[1] > 3 * times[0]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,B", [(40, 72, 200), (33, 65, 97), (20, 30, 3)])
def test_largest_half_precision_states(M, K, B, act):
    """65504 reads back as 64 * 2^10, which fp16 does not hold: where f(x^) is kept in two parts or in fp32 the products stay
    finite, and the bounds are the usual ones."""
    from lich_b200.tilelang_kernels import KernelConfig
    mx = _mx()
    dt = torch.float16
    x = _rand((K, B), 110, 1.0, dt)
    x[3] = 65504
    x[4, ::2] = -65504
    c, s = _ckpt(x)
    xhat = X.load8(c.cpu(), s.cpu(), B)
    assert xhat.max() == 65536
    e = _rand((M, B), 111, 0.01, dt)
    a = O.act_forward(act, xhat)
    ref, S = e.double() @ a.t(), e.double().abs() @ a.abs().t()
    err = (e.double().abs() @ (_act_err(act, xhat, dt) + U[dt] * a.abs() + TINY[dt]).t()) * (1 + 2.0 ** -8) + S * B * 2.0 ** -23
    dw = torch.zeros(M, K, device=DEV)
    backend = "auto" if B <= 4 else "simt"
    mx.build_weight_delta_checkpoint(M, K, B, act, "float16", 1.0, "float32", KernelConfig(backend=backend))(dw, e.to(DEV), c, s)
    _within(dw, ref, err + 2.0 ** -23 * ref.abs())


@pytest.mark.parametrize("threads", [False, True])
@pytest.mark.parametrize("M,K,B", [(256, 512, 4096), (130, 259, 1029)])
def test_streams_with_workspaces_do_not_meet(M, K, B, threads):
    """One operator whose calls need a workspace, on three streams at once with inputs of their own, from one thread or one
    each: what each stream computes is what it computes alone."""
    import threading

    from lich_b200.tilelang_kernels import KernelConfig
    mx = _mx()
    cfg = KernelConfig(backend="tcgen05")
    k = mx.build_weight_delta_checkpoint(M, K, B, "silu", "bfloat16", 1.0, "float32", cfg)
    kb = mx.build_error_backward_checkpoint(M, K, B, "silu", "bfloat16", cfg)
    assert k.workspace_bytes() > 0 and (kb.workspace_bytes() > 0) == (B % 8 != 0)
    w = _rand((M, K), 120, 0.1, torch.bfloat16).to(DEV)
    given = [(_rand((M, B), 121 + i, 0.3, torch.bfloat16).to(DEV), *_ckpt(_rand((K, B), 131 + i, 1.5, torch.bfloat16)))
             for i in range(3)]

    def run(e, c, s, dw, up):
        k(dw, e, c, s)
        kb(w, e, c, s, up)

    def empty():
        return torch.empty(M, K, device=DEV), torch.empty(K, B, device=DEV, dtype=torch.bfloat16)

    alone = [empty() for _ in given]
    for g, o in zip(given, alone):
        run(*g, *o)
        torch.cuda.synchronize()
    e, c, s = given[0]
    a = O.act_forward("silu", X.load8(c.cpu(), s.cpu(), B))
    S = e.cpu().double().abs() @ a.abs().t()
    _within(alone[0][0], e.cpu().double() @ a.t(), S * (2.0 ** -8 + B * 2.0 ** -23))
    streams = [torch.cuda.Stream(DEV) for _ in given]
    outs = [[empty() for _ in range(20)] for _ in given]
    torch.cuda.synchronize()

    def work(i, n):
        with torch.cuda.stream(streams[i]):
            for o in outs[i][n:n + 1] if n is not None else outs[i]:
                run(*given[i], *o)

    if threads:
        ts = [threading.Thread(target=work, args=(i, None)) for i in range(3)]
        [t.start() for t in ts]
        [t.join() for t in ts]
    else:
        for n in range(20):
            for i in range(3):
                work(i, n)
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        for dw, up in got:
            assert torch.equal(dw, want[0]) and torch.equal(up, want[1])
