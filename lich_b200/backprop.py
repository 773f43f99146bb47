"""Backpropagation with 8-bit checkpoints on a ``TileLangIPC`` model's weights, and its answers in 4 bits.

The baseline that incremental predictive coding is compared with, on the same network (``h[l] = W[l] f(h[l+1])``, ``h[L]``
the input), the same energy ``|y - h[0]|^2 / 2`` and the same sign: a step is ``W[l] += alpha * E[l] f(h[l+1])^T`` with
``E[0] = y - h[0]`` and ``E[l+1] = f'(h[l+1]) * (W[l]^T E[l])``.  From one sweep to the other a layer's states are kept as a
microscaled 8-bit checkpoint alone (8.25 bits a state instead of 16).  Beside the checkpoints a step holds two buffers of
the widest hidden layer, in which the forward sweep alternates and the errors of layers 1 and 2 then lie, the errors of
the other layers, and one workspace of the widest layer's states in 16 bits for all products (``held_bytes``).

    bp = CheckpointedBackprop(model)          # model: TileLangIPC; its weights are trained in place
    bp.train_step(x, y)                       # x [d_L, B], y [d_0, B]
    quick = Mxfp4Predictor(model)             # weights laid out in 4 bits once
    logits = quick.predict(x); correct = quick.evaluate(x, labels)
    # python -m lich_b200.backprop --dims 10,256,256,784 --steps 300

The reference has neither (it trains by predictive coding only and predicts in fp16, ``trainer.py:828-833``).
"""
from __future__ import annotations

import argparse

import torch

from . import _native as N
from . import microscaled as mx
from .tilelang_kernels import build_forward, build_prediction_error
from .trainer import IPCConfig, TileLangIPC, one_hot


class CheckpointedBackprop:
    """Backpropagation steps on ``model.w`` that keep the states as 8-bit checkpoints."""

    def __init__(self, model: TileLangIPC):
        if model.fused_optimizer:
            raise ValueError("CheckpointedBackprop applies W += alpha E f(h)^T; the model asks for another optimizer")
        self.model = model
        self._buffers: dict = {}
        self._layers: tuple = (None, None)
        self._space: dict = {}

    def _layer(self, l: int, B: int):
        """Layer ``l``'s operators: ``W[l] f(h[l+1])`` (the lowest layer: the output's error from it), the error's way up
        (None above the last), the weight update; and for each the keyword that gives it this object's workspace, where it
        needs one."""
        m, d, act, dt = self.model, self.model.cfg.dims, self.model.cfg.activation, self.model.dtype_name
        kind, build = ("forward", build_forward) if l else ("prediction", build_prediction_error)
        fwd = build(d[l], d[l + 1], B, act, dt, m._kernel_config(kind, d[l], d[l + 1], B))
        up = mx.build_error_backward_checkpoint(d[l], d[l + 1], B, act, dt) if l + 1 < m.L else None
        update = mx.build_weight_update_checkpoint(d[l], d[l + 1], B, act, dt, float(m.cfg.alpha))
        need = (fwd.workspace_bytes(m.device), 0 if up is None else up.workspace_bytes(), update.workspace_bytes())
        return (fwd, up, update), need

    def _plan(self, B: int) -> list:
        """``_layer`` of every layer (those of the last batch size and factor are kept)."""
        c = self.model.cfg
        key = (B, float(c.alpha), c.activation)
        if self._layers[0] != key:
            with torch.cuda.device(self.model.device):
                self._layers = (key, [self._layer(l, B) for l in range(self.model.L)])
        return self._layers[1]

    def _sizes(self, B: int) -> tuple[int, int]:
        """Elements of a state buffer, and bytes of the workspace, for a batch of ``B``."""
        return max(self.model.cfg.dims[1:-1], default=0) * B, max(max(need) for _, need in self._plan(B))

    def _prepare(self, B: int):
        """Buffers for a batch of ``B``: the two state buffers, the errors, the checkpoints (and the workspace, ``_space[B]``)."""
        buf = self._buffers.get(B)
        if buf is None:
            m, d = self.model, self.model.cfg.dims
            n, ws = self._sizes(B)
            flat = [torch.empty(n, device=m.device, dtype=m.cfg.dtype) for _ in range(2)]
            # the state buffers are free again when the first error goes up
            e = [flat[l - 1][:d[l] * B].view(d[l], B) if l in (1, 2) else
                 torch.empty((d[l], B), device=m.device, dtype=m.cfg.dtype) for l in range(m.L)]
            ck = [None] + [mx.empty_checkpoint(d[l], B, device=m.device) for l in range(1, m.L + 1)]
            # one that another batch size has, if it is large enough; a smaller one stays with its batch size, since a
            # captured graph may hold its address
            self._space[B] = next((t for t in self._space.values() if t.numel() >= ws), None)
            if self._space[B] is None:
                self._space[B] = torch.empty(ws, device=m.device, dtype=torch.uint8)
            buf = self._buffers[B] = (flat, e, ck)
        return buf

    def checkpoint_bytes(self, B: int) -> int:
        """Bytes of the checkpoints of a batch of ``B``: what is kept of the states between the two sweeps."""
        shapes = [s for d in self.model.cfg.dims[1:] for s in mx.checkpoint_shapes(d, B)]
        return sum(a * b for a, b in shapes)

    def held_bytes(self, B: int) -> int:
        """Bytes this object holds for a batch of ``B``: checkpoints, state buffers, errors and the workspace."""
        d, size = self.model.cfg.dims, self.model.cfg.dtype.itemsize
        n, ws = self._sizes(B)
        return self.checkpoint_bytes(B) + ws + size * (2 * n + B * sum(d[l] for l in range(self.model.L) if l not in (1, 2)))

    @torch.no_grad()
    def train_step(self, x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        """One step on a batch; returns ``E[0] = y - h[0]`` of before the update (a buffer of this object)."""
        m, cfg, d = self.model, self.model.cfg, self.model.cfg.dims
        if x.ndim != 2 or x.shape[0] != d[-1] or tuple(y.shape) != (d[0], x.shape[1]):
            raise ValueError(f"expected x [{d[-1]}, B] and y [{d[0]}, B], got {tuple(x.shape)} and {tuple(y.shape)}")
        B = int(x.shape[1])
        flat, e, ck = self._prepare(B)
        # per layer: the operators, and each one's workspace (those that need none take the shorter call)
        layers = [(ops, [{"workspace": self._space[B]} if n else {} for n in need]) for ops, need in self._plan(B)]
        h = x.to(cfg.dtype).contiguous()
        for l in range(m.L, 0, -1):  # keep h[l], then h[l-1] = W[l-1] f(h[l]) (the lowest layer: its error instead)
            mx.build_checkpoint(d[l], B, m.dtype_name)(h, *ck[l])
            (fwd, _, _), (ws, _, _) = layers[l - 1]
            if l > 1:
                out = flat[l % 2][:d[l - 1] * B].view(d[l - 1], B)
                fwd(h, m.w[l - 1], out, **ws)
                h = out
            else:
                fwd(h, m.w[0], y.to(cfg.dtype).contiguous(), e[0], **ws)
        for l, ((_, up, update), (_, ws_up, ws)) in enumerate(layers):
            if up is not None:  # the error goes up through the weights of before the update
                up(m.w[l], e[l], *ck[l + 1], e[l + 1], **ws_up)
            update(m.w[l], e[l], *ck[l + 1], **ws)
        m.steps_done += 1
        return e[0]


class Mxfp4Predictor:
    """``TileLangIPC.predict`` with weights and activations in 4 bits.  ``refresh()`` after the weights change."""

    def __init__(self, model: TileLangIPC):
        self.model = model
        d = model.cfg.dims
        self._w = [mx.empty_mxfp4(d[l], d[l + 1], device=model.device) for l in range(model.L)]
        self._buffers: dict = {}
        self.refresh()

    @torch.no_grad()
    def refresh(self) -> None:
        """Lay the model's present weights out in 4 bits."""
        m, d = self.model, self.model.cfg.dims
        for l in range(m.L):
            mx.build_mxfp4_quantize(d[l], d[l + 1], "identity", m.dtype_name)(m.w[l], *self._w[l])

    @torch.no_grad()
    def predict(self, x_input: torch.Tensor) -> torch.Tensor:
        """``h = W4[l] f(h)4`` for ``l = L-1..0``; returns ``[d_0, B]``."""
        m, cfg = self.model, self.model.cfg
        d, dt = cfg.dims, m.dtype_name
        h = x_input.to(cfg.dtype).contiguous()
        if h.ndim != 2 or h.shape[0] != d[-1]:
            raise ValueError("input features do not match dims[-1]")
        B = int(h.shape[1])
        bufs = self._buffers.get(B)
        if bufs is None:
            bufs = self._buffers[B] = [mx.empty_mxfp4(B, d[l + 1], device=m.device) for l in range(m.L)]
        for l in reversed(range(m.L)):
            mx.build_mxfp4_quantize(B, d[l + 1], cfg.activation, dt, True)(h, *bufs[l])
            out = torch.empty((d[l], B), device=m.device, dtype=cfg.dtype)
            mx.build_mxfp4_forward(d[l], d[l + 1], B, dt)(*self._w[l], *bufs[l], out)
            h = out
        return h

    @torch.no_grad()
    def evaluate(self, x_input: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """Correct predictions of a batch, counted on the device (``TileLangIPC.evaluate``)."""
        m = self.model
        B = int(x_input.shape[1])
        if labels.numel() != B:
            raise ValueError("labels must have one entry per batch column")
        logits = self.predict(x_input)
        cnt = torch.zeros(1, dtype=torch.int32, device=m.device)
        lab = labels.to(m.device, torch.int64).contiguous()
        N.check(N.load().ipc_count_correct(logits.data_ptr(), int(m.cfg.dims[0]), B, lab.data_ptr(), cnt.data_ptr(),
                                           N.dtype_code(m.cfg.dtype), N.stream_handle(m.device)))
        return cnt


def clustered(dims, B: int, *, seed: int, device, dtype, noise: float = 0.3):
    """A batch that can be learned: one random prototype in [0, 1] per class plus noise."""
    g = torch.Generator(device=device).manual_seed(12345)
    proto = torch.rand((dims[-1], dims[0]), generator=g, device=device)
    g.manual_seed(int(seed))
    labels = torch.randint(0, dims[0], (B,), generator=g, device=device)
    x = proto[:, labels] + noise * torch.randn((dims[-1], B), generator=g, device=device)
    return x.to(dtype), one_hot(labels, dims[0], dtype=dtype), labels


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dims", default="10,256,256,784")
    ap.add_argument("--batch", type=int, default=128)
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--alpha", type=float, default=1e-4)
    ap.add_argument("--activation", default="tanh")
    ap.add_argument("--dtype", default="bfloat16", choices=["float16", "bfloat16", "float32"])
    a = ap.parse_args(argv)
    dims, dev = tuple(int(v) for v in a.dims.split(",")), torch.device("cuda", torch.cuda.current_device())
    dt = N.torch_dtype(a.dtype)
    model = TileLangIPC(IPCConfig(dims=dims, alpha=a.alpha, activation=a.activation, dtype=dt), device=dev)
    bp = CheckpointedBackprop(model)
    for step in range(a.steps):
        x, y, _ = clustered(dims, a.batch, seed=step, device=dev, dtype=dt)
        e0 = bp.train_step(x, y)
        if step in (0, a.steps - 1):
            print(f"step {step}: energy {float((e0.float() ** 2).sum(0).mean()) / 2:.4f}")
    x, _, labels = clustered(dims, 1000, seed=10 ** 6, device=dev, dtype=dt)
    res = {"accuracy_16bit": model.accuracy(x, labels),
           "accuracy_4bit": int(Mxfp4Predictor(model).evaluate(x, labels).item()) / 1000,
           "checkpoint_bytes": bp.checkpoint_bytes(a.batch)}
    print(res)
    return res


if __name__ == "__main__":
    main()
