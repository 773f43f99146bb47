"""The C++ call layer of the microscaled operators (``csrc/mx_call.cpp``) on the CPU: the file itself, with its device
queries turned to the host (``mx_call_host.cpp``), around Python operators and C entries of the tests' own."""
import contextlib
import ctypes
import gc
import importlib.machinery
import importlib.util
import os
import subprocess
import sys
import sysconfig
import threading
import time
import weakref
from pathlib import Path

import pytest
import torch

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def call_path(tmp_path_factory):
    from lich_b200 import build
    so = tmp_path_factory.mktemp("mx_call") / "_mx_call.so"
    inc, libs = Path(torch.__file__).parent / "include", Path(torch.__file__).parent / "lib"
    cuda = Path(build.nvcc()).resolve().parents[1] / "include"
    subprocess.run([os.environ.get("CXX", "g++"), "-O0", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    "-I", sysconfig.get_paths()["include"], "-isystem", str(inc), "-isystem",
                    str(inc / "torch" / "csrc" / "api" / "include"), "-isystem", str(cuda),
                    str(HERE / "mx_call_host.cpp"), "-o", str(so), f"-L{libs}", f"-Wl,-rpath,{libs}",
                    "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"], check=True)
    return so


def _load(path):
    loader = importlib.machinery.ExtensionFileLoader("_mx_call", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_mx_call", loader))
    loader.exec_module(module)
    return module.Call


@pytest.fixture(scope="module")
def Call(call_path):
    return _load(call_path)


# the C entry of a weight product: (mode, out, e, codes, scales, M, K, B, scale, flags, act, dtype, algo, ws, bytes, stream)
ENTRY = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_int, *[ctypes.c_void_p] * 4, *[ctypes.c_int] * 3, ctypes.c_float,
                         *[ctypes.c_int] * 4, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p)


def _weight_call(Call, entry, workspace):
    """A weight product of 2 x 3 from 32 samples whose Python operator gives out ``workspace(device, stream)``."""
    class Op:
        def _workspace(self, device, stream):
            return workspace(device, stream)

        def _failed(self, rc):
            raise RuntimeError(f"entry returned {rc}")

        def __call__(self, *args, **kw):
            raise ValueError("handed back")

    f32 = torch.float32
    spec = [(torch.Size((2, 3)), f32), (torch.Size((2, 32)), f32), (torch.Size((3, 32)), torch.int8),
            (torch.Size((1, 3)), torch.uint8)]
    call = Call(Op(), 2, ctypes.cast(entry, ctypes.c_void_p).value, spec, (3, 2, 3, 32, 0, 0, 0), 1.0)
    return call, tuple(torch.zeros(s, dtype=d) for s, d in spec)


def test_threads_on_two_streams_keep_to_their_own_workspaces(Call):
    """One operator is shared by all threads.  Each has its own stream here, and each stream its workspace; while a thread
    is in the C entry's call without the interpreter lock, another one takes its turn."""
    seen, owner = [], {}

    @ENTRY
    def entry(mode, out, e, codes, scales, M, K, B, scale, flags, act, dtype, algo, ws, n, stream):
        seen.append((ws, n, stream))
        return 0

    def workspace(device, stream):
        buf = owner.setdefault(stream, torch.empty(64 * (1 + len(owner)), dtype=torch.uint8))
        return buf.data_ptr(), buf.numel()

    call, args = _weight_call(Call, entry, workspace)
    gate = threading.Barrier(2)

    def run():
        gate.wait()
        for _ in range(40):
            call(*args)

    threads = [threading.Thread(target=run) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(seen) == 80 and len(owner) == 2
    for ws, n, stream in seen:
        assert (ws, n) == (owner[stream].data_ptr(), owner[stream].numel())


ABORTS = """
import sys
sys.path[:0] = {path!r}
import torch
from test_mx_call_cpu import ENTRY, _load, _weight_call

@ENTRY
def entry(*args):
    return 0

call, args = _weight_call(_load({so!r}), entry, lambda device, stream: (None, 0))
assert call(*args) is None
out, e, codes, scales = args
batched = torch.zeros(5, 2, 32)
for case in (lambda: torch.vmap(lambda t: call(out, t, codes, scales))(batched),   # no storage of its own
             lambda: torch.func.grad(lambda t: (call(out, t, codes, scales), t.sum())[1])(e),
             lambda: call(out, e.to_sparse(), codes, scales)):                   # no dense layout to ask for
    try:
        case()
    except ValueError as exc:
        assert "handed back" in str(exc), exc
        print("refused")
"""


def test_what_throws_in_the_call_goes_to_the_operator(call_path):
    """Tensors under torch.vmap or torch.func have the type and the shape that the call asks for and throw when asked for
    their address, sparse ones when asked for their layout.  In a process of its own: an exception that leaves a C
    function ends it."""
    code = ABORTS.format(path=[str(HERE), str(HERE.parent)], so=str(call_path))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["refused"] * 3


class _Owner:
    pass


def test_the_call_holds_the_workspace_that_it_remembers(Call):
    """The address is used for every later call on the stream, so what owns the memory has to live as long, whatever the
    operator's own table holds by then."""
    seen, owners = [], []

    @ENTRY
    def entry(mode, out, e, codes, scales, M, K, B, scale, flags, act, dtype, algo, ws, n, stream):
        seen.append(ws)
        return 0

    def workspace(device, stream):
        owner = _Owner()
        owners.append(weakref.ref(owner))
        return 4096, 64, owner

    call, args = _weight_call(Call, entry, workspace)
    call(*args)
    assert owners[0]() is not None
    call(*args)
    assert len(owners) == 1 and seen == [4096, 4096]
    t = threading.Thread(target=call, args=args)  # another stream: the first one's memory is let go
    t.start(), t.join()
    assert len(owners) == 2 and owners[0]() is None and owners[1]() is not None
    del call
    assert owners[1]() is None


def _no_gpu(monkeypatch, made):
    """Workspaces of ``lich_b200.microscaled`` in CPU memory; making one takes its time and lets other threads run."""
    from lich_b200 import microscaled as mx
    real = torch.empty

    def empty(n, **kw):
        time.sleep(0.05)
        made.append(real(n, dtype=torch.uint8))
        return made[-1]

    def ws_bytes(self, n):
        n._obj.value = self.M * 256
        return 0

    monkeypatch.setattr(mx.torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(mx.torch, "empty", empty)
    monkeypatch.setattr(mx.CheckpointWeightKernel, "_ws_bytes", ws_bytes)
    return mx


def test_threads_that_meet_at_the_first_call_get_one_workspace(monkeypatch):
    made, got = [], []
    mx = _no_gpu(monkeypatch, made)
    k = mx.build_weight_delta_checkpoint(11, 13, 64, "tanh", "bfloat16", 0.125)
    gate = threading.Barrier(4)

    def first():
        gate.wait()
        got.append(k._workspace(0, 7))

    threads = [threading.Thread(target=first) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(made) == 1 and len({g[0] for g in got}) == 1 and got[0][1] == 11 * 256
    assert got[0][0] == made[0].data_ptr()
    assert k._workspace(0, 8)[0] != got[0][0] and len(made) == 2  # another stream


def test_operators_that_differ_in_the_factor_share_a_workspace(monkeypatch):
    """alpha is an argument of the launch: a schedule that changes it every step makes operators, not workspaces, and the
    memory goes when the last operator of its shape does."""
    made = []
    mx = _no_gpu(monkeypatch, made)
    ops = [mx.CheckpointWeightKernel(0, 17, 19, 64, "tanh", "bfloat16", 0.1 / (1 + i), torch.bfloat16, mx.KernelConfig())
           for i in range(5)]
    assert len({op._workspace(0, 7)[0] for op in ops}) == 1 and len(made) == 1
    other = mx.CheckpointWeightKernel(0, 23, 19, 64, "tanh", "bfloat16", 0.1, torch.bfloat16, mx.KernelConfig())
    assert other._workspace(0, 7)[0] != ops[0]._workspace(0, 7)[0] and len(made) == 2
    held = len(mx._scratch)
    op, ops = ops[-1], None
    assert op._workspace(0, 7)[0] == made[0].data_ptr() and len(mx._scratch) == held
    op = None
    gc.collect()
    assert len(mx._scratch) == held - 1
