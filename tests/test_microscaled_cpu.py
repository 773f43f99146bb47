"""Microscaled operators without a GPU: the formats' oracle, shapes, and every refusal that precedes a launch."""
import ctypes

import pytest
import torch

from oracle import mx_oracle as X


def test_oracle_formats_by_hand():
    x = torch.zeros(2, 33)
    x[0, 0], x[0, 1], x[0, 2] = 127.0, -126.5, 0.5  # step 1: 127 fits, -126.5 ties to -126, 0.5 ties to 0
    x[1, 32] = 128.0                                # step 2: 128 = 64 * 2
    codes, scales = X.store8(x)
    assert codes.shape == (2, 64) and scales.shape == (2, 2)
    assert codes[0, :3].tolist() == [127, -126, 0] and scales[0, 0] == 127
    assert codes[1, 32] == 64 and scales[1, 1] == 128 and scales[0, 1] == 0
    v = torch.tensor([[6.0, 5.0, -2.5, 0.25, 0.75, 1.25, 1.75, 3.5, 0.26, -0.1]])
    val, code, sc = X.quant4(v)
    assert val[0].tolist() == [6.0, 4.0, -2.0, 0.0, 1.0, 1.0, 2.0, 4.0, 0.5, 0.0]
    assert sc[0, 0, 0, 0, 0] == 127 and code.shape == (1, 64) and sc.shape == (1, 1, 32, 4, 4)
    assert int(code[0, 0]) == 7 + 16 * 6 and int(code[0, 1]) == 12 + 16 * 0
    val, _, sc = X.quant4(torch.tensor([[6.01, 1.0]]))  # above 6: the step doubles, 6.01 -> 3 * 2
    assert sc[0, 0, 0, 0, 0] == 128 and val[0].tolist() == [6.0, 1.0]


def test_oracle_marks_blocks_that_are_not_finite():
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = torch.ones(1, 64)
        x[0, 5] = bad
        codes, scales = X.store8(x)
        assert scales[0, 0] == 255 and not codes[0, :32].any() and scales[1, 0] != 255
        back = X.load8(codes, scales, 64)
        assert back[0, :32].isnan().all() and (back[0, 32:] == 1).all()
        assert X.quant4(x)[0][0, :32].isnan().all()


def test_shapes():
    from lich_b200 import microscaled as mx
    assert mx.checkpoint_shapes(10, 33) == ((10, 64), (2, 10))
    assert mx.checkpoint_shapes(10, 0) == ((10, 0), (0, 10))
    assert mx.mxfp4_shapes(129, 129) == ((129, 128), (2, 2, 32, 4, 4))
    c, s = mx.empty_checkpoint(3, 40, device="cpu")
    assert c.dtype == torch.int8 and s.dtype == torch.uint8 and c.shape == (3, 64) and s.shape == (2, 3)


def test_builders_refuse():
    from lich_b200 import microscaled as mx
    with pytest.raises(ValueError):
        mx.build_checkpoint(4, 4, "int8")
    with pytest.raises(ValueError):
        mx.build_checkpoint(-1, 4, "float16")
    with pytest.raises(ValueError):
        mx.build_checkpoint_restore(4, 4, "swish", "float16")
    with pytest.raises(ValueError):
        mx.build_weight_delta_checkpoint(4, 4, 4, "tanh", "float16", 1.0, "bfloat16")
    with pytest.raises(ValueError):
        mx.build_mxfp4_quantize(4, 4, "nope", "float16")
    assert mx.build_mxfp4_forward(4, 4, 4, "float16") is mx.build_mxfp4_forward(4, 4, 4, "float16")
    assert "mxfp4_forward" in mx.build_mxfp4_forward(4, 4, 4, "float16").get_kernel_source()


def test_kernels_refuse_tensors_before_any_launch():
    from lich_b200 import microscaled as mx
    x = torch.zeros(4, 40, dtype=torch.float16)
    c, s = mx.empty_checkpoint(4, 40, device="cpu")
    k = mx.build_checkpoint(4, 40, "float16")
    for args in ((x, c, s),                      # not on a GPU
                 (x.float(), c, s),              # another dtype
                 (x[:, :39], c, s),              # another shape
                 (x, c.to(torch.uint8), s), (x, c, s.t()), (x, c, None)):
        with pytest.raises(ValueError):
            k(*args)
    w = torch.zeros(4, 4, dtype=torch.float16)
    cc, ss = mx.empty_checkpoint(4, 4, device="cpu")
    with pytest.raises(ValueError):
        mx.build_weight_update_checkpoint(4, 4, 4, "tanh", "float16", 0.1)(w, w, cc, ss)
    with pytest.raises(ValueError):
        mx.build_error_backward_checkpoint(4, 4, 4, "tanh", "float16")(w, w, cc, ss, w)


def test_abi_refuses_bad_arguments():
    from lich_b200 import _native as N
    lib = N.load()
    A = N.IPC_ERR_ARG
    assert lib.ipc_mx8_store(None, None, None, -1, 4, 1, None) == A
    assert lib.ipc_mx8_store(None, None, None, 4, 4, 9, None) == A
    assert lib.ipc_mx8_restore(None, None, None, 4, 4, 77, 1, None) == A
    assert lib.ipc_mx8_weight(3, None, None, None, None, 4, 4, 4, 1.0, 0, 99, 1, 0, None, 0, None) == A
    assert lib.ipc_mx8_backward(None, None, None, None, None, 4, 4, -4, 0, 1, 0, None, 0, None) == A
    assert lib.ipc_mxfp4_quantize(None, None, None, 4, -4, 0, 0, 1, None) == A
    assert lib.ipc_mxfp4_restore(None, None, None, 4, 4, 5, None) == A
    assert lib.ipc_mxfp4_forward(None, None, None, None, None, 4, 4, -1, 1, None) == A
    n = ctypes.c_size_t(0)
    assert lib.ipc_mx8_weight_ws_bytes(3, -1, 4, 4, 1, 0, ctypes.byref(n)) == A


def test_the_call_layer_hands_everything_unusual_to_the_operator():
    from lich_b200 import microscaled as mx
    k = mx.build_checkpoint(4, 40, "float16")
    assert k.kind == "checkpoint" and (k.D, k.B) == (4, 40)  # attributes are the operator's
    with pytest.raises(AttributeError):
        k.nothing
    x = torch.zeros(4, 40, dtype=torch.float16)
    c, s = mx.empty_checkpoint(4, 40, device="cpu")
    with pytest.raises(TypeError):
        k(x, c)
    with pytest.raises(TypeError):
        k(x, c, s, s)
    with pytest.raises(ValueError, match="not a CUDA tensor"):
        k(x, codes=c, scales=s)
    with pytest.raises(ValueError, match="argument 0 is not a tensor"):
        k(1, c, s)
    with pytest.raises(ValueError):
        mx._Call(object(), 0, 0, [], (), 0.0)
    assert mx.build_mxfp4_forward(4, 5, 6, dtype="float16") is mx.build_mxfp4_forward(4, 5, 6, dtype="float16")


def test_sizes_beyond_31_bits_are_refused():
    """The C entries take 32-bit sizes: a larger one would be cut to its low bits and a part of the tensor worked on."""
    from lich_b200 import _native as N
    from lich_b200 import microscaled as mx
    for n in (2 ** 32 + 32, 2 ** 31, 2 ** 31 - 1):
        for build in (lambda: mx.build_checkpoint(1, n, "float16"), lambda: mx.build_checkpoint(n, 1, "float16"),
                      lambda: mx.build_checkpoint_restore(1, n, "tanh", "float16"),
                      lambda: mx.build_weight_update_checkpoint(1, 1, n, "tanh", "float16", 0.1),
                      lambda: mx.build_weight_delta_checkpoint(n, 1, 1, "tanh", "float16", 0.1),
                      lambda: mx.build_error_backward_checkpoint(1, n, 1, "tanh", "float16"),
                      lambda: mx.build_mxfp4_quantize(1, n, "tanh", "float16"),
                      lambda: mx.build_mxfp4_restore(n, 1, "float16"), lambda: mx.build_mxfp4_forward(1, 1, n, "float16")):
            with pytest.raises(ValueError, match="size"):
                build()
    lib, big, A = N.load(), 2 ** 31 - 1, N.IPC_ERR_ARG
    assert lib.ipc_mx8_store(None, None, None, 4, big, 1, None) == A
    assert lib.ipc_mx8_restore(None, None, None, big, 4, 0, 1, None) == A
    assert lib.ipc_mx8_weight(3, None, None, None, None, 4, big, 4, 1.0, 0, 0, 1, 0, None, 0, None) == A
    assert lib.ipc_mx8_backward(None, None, None, None, None, 4, 4, big, 0, 1, 0, None, 0, None) == A
    assert lib.ipc_mxfp4_quantize(None, None, None, 4, big, 0, 0, 1, None) == A
    assert lib.ipc_mxfp4_restore(None, None, None, big, 4, 1, None) == A
    assert lib.ipc_mxfp4_forward(None, None, None, None, None, 4, big, 4, 1, None) == A
    n = ctypes.c_size_t(0)
    assert lib.ipc_mx8_weight_ws_bytes(3, 4, 4, big, 1, 0, ctypes.byref(n)) == A
    assert lib.ipc_mx8_backward_ws_bytes(big, 4, 4, 1, 0, ctypes.byref(n)) == A


def test_configs_that_a_checkpoint_product_cannot_follow_are_refused():
    """"outer" has no kernel that reads checkpoints, and fp32 storage none on the tensor cores; tile, split and CTA overrides
    would be dropped."""
    from lich_b200 import microscaled as mx
    from lich_b200.tilelang_kernels import KernelConfig
    for build in (lambda dt, cfg: mx.build_weight_update_checkpoint(8, 8, 8, "tanh", dt, 0.1, cfg),
                  lambda dt, cfg: mx.build_weight_delta_checkpoint(8, 8, 8, "tanh", dt, 0.1, "float32", cfg),
                  lambda dt, cfg: mx.build_error_backward_checkpoint(8, 8, 8, "tanh", dt, cfg)):
        for backend in ("auto", "simt", "generic", "tcgen05"):
            build("bfloat16", KernelConfig(backend=backend))
        build("float32", KernelConfig(64, 128, 16, 128, 2, True, 8, False))  # the reference's tile fields mean nothing here
        for dt, cfg in (("bfloat16", KernelConfig(backend="outer")), ("float32", KernelConfig(backend="tcgen05")),
                        ("bfloat16", KernelConfig(tc_bn=128)), ("bfloat16", KernelConfig(tc_splits=2)),
                        ("bfloat16", KernelConfig(tc_raster=4)), ("bfloat16", KernelConfig(tc_max_ctas=64)),
                        ("bfloat16", KernelConfig(tc_pair=1)), ("bfloat16", KernelConfig(backend="nothing"))):
            with pytest.raises(ValueError):
                build(dt, cfg)
