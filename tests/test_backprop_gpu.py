"""Backpropagation with 8-bit checkpoints and the 4-bit predictor: the microscaled operators used together."""
import gc

import pytest
import torch

from oracle import ipc_oracle as O
from oracle import mx_oracle as X

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _model(dims, dt, act="tanh", alpha=1e-3):
    from lich_b200.trainer import IPCConfig, TileLangIPC
    return TileLangIPC(IPCConfig(dims=dims, alpha=alpha, activation=act, dtype=dt), device=DEV, seed=3)


def _batch(dims, B, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(dims[-1], B, generator=g).to(dt)
    y = torch.zeros(dims[0], B, dtype=dt)
    y[torch.randint(0, dims[0], (B,), generator=g), torch.arange(B)] = 1
    return x, y


@pytest.mark.parametrize("dims,B", [((10, 64, 64, 784), 128), ((7, 33, 65, 50), 31), ((5, 20), 16),
                                    ((16, 512, 520, 256), 520)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_step_is_backpropagation_through_the_checkpoints(dims, B, dt):
    """Every stage of a step against its definition in 64 bits, from the stage before as the device holds it."""
    from lich_b200.backprop import CheckpointedBackprop
    m = _model(dims, dt)
    bp = CheckpointedBackprop(m)
    x, y = _batch(dims, B, dt)
    w0 = [w.clone() for w in m.w]
    e0 = bp.train_step(x.to(DEV), y.to(DEV))
    _, e, ck = bp._prepare(B)
    assert e0 is e[0] and m.steps_done == 1
    rc, rs = X.store8(x)
    assert torch.equal(ck[m.L][0].cpu(), rc) and torch.equal(ck[m.L][1].cpu(), rs)
    # A checkpoint is within half a step (2^s / 2) of the device's states; those are within `off` of the 64-bit forward
    # sweep: its own roundings (operand, f in MUFU form, result, sums), and the layer above's passed on (|f'| <= 1).
    h, off, hat = x.double(), torch.zeros(dims[-1], B, dtype=torch.float64), {}
    for l in range(m.L, 0, -1):
        hat[l] = X.load8(ck[l][0].cpu(), ck[l][1].cpu(), B)
        step = torch.exp2(ck[l][1].cpu().double() - 127).repeat_interleave(32, 0)[:B].t()
        assert ((hat[l] - h).abs() <= step / 2 + off).all()
        w = w0[l - 1].cpu().double()
        f = torch.tanh(h)
        off = w.abs() @ off + (4 * U[dt] + 2.0 ** -10 * (dt != torch.float32) + 2.0 ** -16) * (w.abs() @ f.abs())
        h = w @ f
    for l in range(m.L):
        el, w = e[l].cpu().double(), w0[l].cpu().double()
        a = O.act_forward("tanh", hat[l + 1])
        slack = (2 * U[dt] + 2.0 ** -10 * (dt != torch.float32) + 2.0 ** -20)
        S = el.abs() @ a.abs().t()
        want = w + m.cfg.alpha * (el @ a.t())
        assert ((m.w[l].cpu().double() - want).abs()
                <= m.cfg.alpha * S * slack + 2 * U[dt] * want.abs() + 2.0 ** -25).all()
        if l + 1 < m.L:
            ref = X.backward(w0[l].cpu(), e[l].cpu(), hat[l + 1], "tanh")
            S = w.abs().t() @ el.abs()
            assert ((e[l + 1].cpu().double() - ref).abs() <= S * (2.0 ** -9 * (dt != torch.float32) + 2.0 ** -18)
                    + 2 * U[dt] * ref.abs() + 2.0 ** -25).all()


def test_gradient_is_close_to_plain_backpropagation():
    """Against autograd without checkpoints: an 8-bit state is off by at most 1/127 of its block's largest, half a step
    of a block whose largest is at least 63.5 steps; tanh does not grow that, so the relative error of a layer's delta
    stays below a few times 1/127."""
    from lich_b200.backprop import CheckpointedBackprop
    dims, B = (10, 96, 80, 120), 256
    m = _model(dims, torch.float32, alpha=1.0)
    x, y = _batch(dims, B, torch.float32)
    ws = [w.detach().cpu().double().requires_grad_() for w in m.w]
    h = x.double()
    for l in range(m.L - 1, -1, -1):
        h = ws[l] @ torch.tanh(h)
    (0.5 * ((y.double() - h) ** 2).sum()).backward()
    w0 = [w.clone() for w in m.w]
    CheckpointedBackprop(m).train_step(x.to(DEV), y.to(DEV))
    for l in range(m.L):
        got = (m.w[l] - w0[l]).cpu().double()
        assert (got + ws[l].grad).norm() <= 4 / 127 * ws[l].grad.norm()


def test_training_lowers_the_energy_and_four_bits_answer_alike():
    from lich_b200 import backprop as B
    res = B.main(["--dims", "10,256,256,784", "--batch", "128", "--steps", "200", "--alpha", "2e-4"])
    assert res["accuracy_16bit"] > 0.9
    assert res["accuracy_4bit"] > res["accuracy_16bit"] - 0.1
    assert res["checkpoint_bytes"] == (256 + 256 + 784) * (128 + 4)


def test_predictor_follows_refresh_and_refuses():
    from lich_b200.backprop import CheckpointedBackprop, Mxfp4Predictor
    dims, B, dt = (10, 128, 192), 40, torch.bfloat16
    m = _model(dims, dt, "relu")
    x, _ = _batch(dims, B, dt)
    p = Mxfp4Predictor(m)

    def want():
        h = x.double()
        for l in range(m.L - 1, -1, -1):
            a = X.quant4(O.act_forward("relu", h).t().contiguous())[0]
            w = X.quant4(m.w[l].cpu())[0]
            h = (w @ a.t()).to(dt).double()
        return h

    def close(got, ref):
        # a state rounded the other way moves a code of the next layer by a step at most, a sixth of its block's largest
        return (got.cpu().double() - ref).abs().max() <= 0.02 * ref.abs().max()

    first = p.predict(x.to(DEV))
    assert close(first, want())
    m.w[0].mul_(2)
    assert torch.equal(p.predict(x.to(DEV)), first)  # the layout of before
    p.refresh()
    assert close(p.predict(x.to(DEV)), want())
    with pytest.raises(ValueError):
        p.predict(x[:-1].to(DEV))
    with pytest.raises(ValueError):
        p.evaluate(x.to(DEV), torch.zeros(B + 1))
    with pytest.raises(ValueError):
        CheckpointedBackprop(m).train_step(x.to(DEV), x.to(DEV))
    from lich_b200.trainer import IPCConfig, TileLangIPC
    adam = TileLangIPC(IPCConfig(dims=dims, dtype=dt, optimizer="adamw"), device=DEV)
    with pytest.raises(ValueError):
        CheckpointedBackprop(adam)


def test_a_step_holds_what_it_says():
    """Wide layers, whose products need a copy of the states in 16 bits: one for all of them, and the errors of layers 1 and
    2 where the forward sweep's buffers were.  Nothing is left in the operators' own workspaces."""
    from lich_b200 import microscaled as mx
    from lich_b200.backprop import CheckpointedBackprop
    dims, B, dt = (10, 512, 512, 512, 784), 4104, torch.bfloat16
    m = _model(dims, dt, alpha=1e-4)
    x, y = (t.to(DEV) for t in _batch(dims, B, dt))
    bp = CheckpointedBackprop(m)
    torch.cuda.synchronize()

    def requested():  # (what is allocated depends on the blocks that earlier tests have left)
        return torch.cuda.memory_stats(DEV)["requested_bytes.all.current"]

    for build in (mx.build_weight_update_checkpoint, mx.build_error_backward_checkpoint):
        build.cache_clear()  # (else the step's operators may push out older ones, whose workspaces go with them)
    gc.collect()
    before = requested()
    bp.train_step(x, y)
    held = requested() - before
    states = sum(dims[1:]) * B
    assert bp.checkpoint_bytes(B) == sum(dims[1:]) * (4128 + 129)
    # checkpoints; two state buffers and the errors of layers 0 and 3; a workspace that the widest f(x^) is the most of
    most = bp.checkpoint_bytes(B) + 2 * B * (2 * 512 + 512 + 10) + 2 * B * 784 + (17 << 20)
    assert bp.held_bytes(B) <= most
    assert not any(s.bytes for k, s in mx._scratch.items() if B in k)
    assert held == bp.held_bytes(B)
    bp.train_step(x, y)
    assert requested() - before == held
    assert states * 2 > bp.checkpoint_bytes(B)
    k = mx.build_weight_update_checkpoint(512, 784, B, "tanh", "bfloat16", 1e-4)
    args = (torch.zeros(512, 784, device=DEV, dtype=dt), torch.zeros(512, B, device=DEV, dtype=dt),
            *mx.empty_checkpoint(784, B, device=DEV))
    for ws in (torch.empty(k.workspace_bytes() - 1, device=DEV, dtype=torch.uint8), torch.empty(1 << 30, dtype=torch.uint8),
               torch.empty(k.workspace_bytes() + 1, device=DEV, dtype=torch.uint8)[1:], 5):
        with pytest.raises(ValueError, match="workspace"):
            k(*args, workspace=ws)
    with pytest.raises(ValueError):
        bp.train_step(x, y.cpu())


def test_a_changing_rate_changes_the_step():
    from dataclasses import replace

    from lich_b200.backprop import CheckpointedBackprop
    dims, B, dt = (10, 64, 784), 128, torch.float32
    x, y = (t.to(DEV) for t in _batch(dims, B, dt))
    moved = []
    for alpha in (1e-3, 2e-3):
        m = _model(dims, dt, alpha=1e-3)
        bp = CheckpointedBackprop(m)
        w0 = m.w[0].clone()
        m.cfg = replace(m.cfg, alpha=alpha)
        bp.train_step(x, y)
        moved.append((m.w[0] - w0).double())
    assert (moved[1] - 2 * moved[0]).abs().max() <= 2.0 ** -20 * m.w[0].abs().max()
