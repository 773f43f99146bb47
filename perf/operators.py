"""The microscaled operators as workloads: what each is given, the call a user makes, and what it computes.

Five operators work on layers stored in blocks of 32 numbers that share one power of two:

``checkpoint``  the states of a layer, ``x [D, B]``, kept in 8 bits for the backward pass and read back as ``f(x^)``;
``delta``       the weight gradient ``dW = alpha * E @ f(x^)^T`` from such a checkpoint;
``backward``    the error of the layer above, ``E_up = f'(x^) * (W^T @ E)``, from such a checkpoint;
``quantize``    weights or activations in 4 bits, in blocks along the features that a product sums over;
``forward``     the product of two such operands, ``out = W4 @ A4``.

Formats.  A block of numbers v with the largest magnitude m is stored as a byte s + 127 and codes c, v ~ c * 2^s.
8 bits: s is the smallest integer with m <= 127 * 2^s, c = round-to-nearest-even(v / 2^s).  4 bits (sign, two
bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6): s is the smallest integer with m <= 6 * 2^s, c the
nearest of these numbers, ties to the even code.  A block of zeros has s = -127.

Layouts.  Checkpoint: codes int8 ``[D, 32 * ceil(B / 32)]``, scale bytes ``[ceil(B / 32), D]``.  4-bit operand of R rows
and K columns: codes uint8 ``[R, Kp / 2]`` with ``Kp = 128 * ceil(K / 128)``, the column of lower index in the lower half
of a byte; scale bytes ``[ceil(R / 128), Kp / 128, 32, 4, 4]``, that of row r and block j at
``[r / 128, j / 4, r % 32, r % 128 / 32, j % 4]``.  Padding is zero in both.
"""
import math

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the 4-bit codes 0..7


def listed():
    return [
        # the input states of the 784-64-... classifiers at their batch of 128: a latency case
        dict(name="checkpoint-784x128", op="checkpoint", D=784, B=128, act="relu", dtype="float16"),
        # one wide layer's states in a large batch: bound by memory
        dict(name="checkpoint-4096x8192", op="checkpoint", D=4096, B=8192, act="tanh", dtype="bfloat16"),
        # the input layer's gradient of the small classifiers
        dict(name="delta-64x784x128", op="delta", M=64, K=784, B=128, act="tanh", dtype="float16", out="float16"),
        # an odd layer and a last, ragged batch; the gradient kept in 32 bits to be summed over further batches
        dict(name="delta-1000x1021x777", op="delta", M=1000, K=1021, B=777, act="relu", dtype="bfloat16", out="float32"),
        # a hidden layer of the wide network
        dict(name="delta-4096x4096x8192", op="delta", M=4096, K=4096, B=8192, act="tanh", dtype="bfloat16",
             out="bfloat16"),
        # a hidden layer of the small classifiers
        dict(name="backward-64x64x128", op="backward", M=64, K=64, B=128, act="sigmoid", dtype="float16"),
        # a hidden layer of the wide network
        dict(name="backward-4096x4096x8192", op="backward", M=4096, K=4096, B=8192, act="tanh", dtype="bfloat16"),
        # weights laid out for answering, from the 32-bit master copy of an odd layer
        dict(name="quantize-weights-1000x777", op="quantize", R=1000, K=777, turned=False, act="identity",
             dtype="float32"),
        # a large batch's activations on their way into a wide layer
        dict(name="quantize-states-8192x4096", op="quantize", R=8192, K=4096, turned=True, act="relu",
             dtype="bfloat16"),
        # one sample through a layer of width 1024: a latency case, bound by reading the weights
        dict(name="forward-1024x1024x1", op="forward", M=1024, K=1024, B=1, dtype="float16"),
        # an odd layer, a ragged batch
        dict(name="forward-1000x777x300", op="forward", M=1000, K=777, B=300, dtype="bfloat16"),
        # a large batch through a wide layer: bound by the tensor cores
        dict(name="forward-4096x4096x8192", op="forward", M=4096, K=4096, B=8192, dtype="bfloat16"),
    ]


def draw(rng):
    def size(lo, hi):  # spread over the logarithm; one in three is rounded to what networks are built in
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, n - n % 64 if n >= 128 and rng.random() < 0.33 else n))

    op = rng.choice(["checkpoint", "delta", "backward", "quantize", "forward"])
    half = rng.choice(["float16", "bfloat16"])
    act = rng.choice(["relu", "tanh", "sigmoid", "silu", "gelu"])
    if op == "checkpoint":
        return dict(op=op, D=size(10, 4096), B=size(1, 8192), act=act, dtype=half)
    if op == "delta":
        if rng.random() < 0.3:  # in 32 bits with the activation that rounds nothing
            return dict(op=op, M=size(10, 4096), K=size(10, 4096), B=size(1, 4096), act="relu", dtype=half,
                        out="float32")
        return dict(op=op, M=size(10, 4096), K=size(10, 4096), B=size(1, 8192), act=act, dtype=half, out=half)
    if op == "backward":
        return dict(op=op, M=size(10, 4096), K=size(10, 4096), B=size(1, 8192), act=act, dtype=half)
    if op == "quantize":
        return dict(op=op, R=size(1, 8192), K=size(10, 4096), turned=rng.random() < 0.6,
                    act=rng.choice(["identity", "relu"]), dtype=rng.choice(["float16", "bfloat16", "float32"]))
    return dict(op=op, M=size(10, 4096), K=size(10, 4096), B=size(1, 8192), dtype=half)


# ------------------------------------------------------------------ the formats, in elementary operations
def _power(n):
    """2^n in 32 bits for whole n in [-127, 127]."""
    normal = ((n + 127).clamp(min=1) << 23).to(torch.int32).view(torch.float32)
    return torch.where(n > -127, normal, torch.full_like(normal, 2.0 ** -127))


def _exponent(m, top, top_exp):
    """The smallest s in [-127, 127] with m <= top * 2^top_exp * 2^s, top in [0.5, 1): from m's own exponent."""
    frac, exp = torch.frexp(m)
    s = exp.to(torch.int64) - top_exp + (frac > top)
    return torch.where(m > 0, s, torch.full_like(s, -127)).clamp(-127, 127)


def _store8(x):
    D, B = x.shape
    nb = -(-B // 32)
    v = torch.zeros(D, nb * 32, device=x.device, dtype=torch.float32)
    v[:, :B] = x
    v = v.view(D, nb, 32)
    s = _exponent(v.abs().amax(-1), 127 / 128, 7)
    codes = torch.round(v * _power(-s)[..., None])
    return codes.to(torch.int8).view(D, nb * 32), (s + 127).to(torch.uint8).t().contiguous()


def _load8(codes, scales, B):
    D = codes.shape[0]
    step = _power(scales.t().to(torch.int64) - 127)
    return (codes.view(D, -1, 32).float() * step[..., None]).view(D, -1)[:, :B]


def _store4(v):
    """Codes and scale bytes of ``v [R, K]`` in 32 bits, in an operand's layout."""
    R, K = v.shape
    kp, rp = -(-K // 128) * 128, -(-R // 128) * 128
    w = torch.zeros(R, kp, device=v.device, dtype=torch.float32)
    w[:, :K] = v
    w = w.view(R, kp // 32, 32)
    s = _exponent(w.abs().amax(-1), 0.75, 3)
    u = (w * _power(-s)[..., None]).abs()
    u = torch.where(u < 2, torch.round(u * 2) / 2, torch.where(u < 4, torch.round(u), torch.round(u / 2) * 2))
    code = torch.where(u <= 2, u * 2, torch.where(u <= 4, u + 2, u / 2 + 4)).to(torch.uint8)
    code = (code + 8 * (w < 0).to(torch.uint8)).view(R, kp // 2, 2)
    full = torch.zeros(rp, kp // 32, device=v.device, dtype=torch.uint8)
    full[:R] = (s + 127).to(torch.uint8)
    scales = full.view(rp // 128, 4, 32, kp // 128, 4).permute(0, 3, 2, 1, 4).contiguous()
    return code[..., 0] + 16 * code[..., 1], scales


def _load4(codes, scales, K):
    R = codes.shape[0]
    nib = torch.stack((codes & 15, codes >> 4), -1).view(R, -1).to(torch.int64)
    c = nib & 7
    mag = torch.where(c <= 4, c / 2, torch.where(c == 7, 6, c - 2).float())
    val = torch.where(nib >= 8, -mag, mag)
    s = scales.permute(0, 3, 2, 1, 4).reshape(-1, scales.shape[1] * 4)[:R].to(torch.int64) - 127
    return (val.view(R, -1, 32) * _power(s)[..., None]).view(R, -1)[:, :K]


def _f(act, x):
    if act == "relu":
        return x.clamp(min=0)
    if act == "tanh":
        return torch.tanh(x)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x


def _df(act, x):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "tanh":
        return 1 - torch.tanh(x) ** 2
    if act == "sigmoid":
        y = 1 / (1 + torch.exp(-x))
        return y * (1 - y)
    if act == "silu":
        y = 1 / (1 + torch.exp(-x))
        return y * (1 + x * (1 - y))
    if act == "gelu":
        t = torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * x * x)
    return torch.ones_like(x)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def spread(rows, cols):  # rows (features) differ in size by a factor of sixteen or so, as trained ones do
        return normal(rows, cols) * torch.exp2(2 * torch.randn(rows, 1, generator=g, device=dev).clamp(-2, 2) - 1)

    s = dict(case)
    if case["op"] == "checkpoint":
        D, B = case["D"], case["B"]
        s["x"] = spread(D, B).to(dt)
        s["codes"] = torch.empty(D, -(-B // 32) * 32, device=dev, dtype=torch.int8)
        s["scales"] = torch.empty(-(-B // 32), D, device=dev, dtype=torch.uint8)
        s["values"] = torch.empty(D, B, device=dev, dtype=dt)
    elif case["op"] == "delta":
        M, K, B = case["M"], case["K"], case["B"]
        s["e"] = (0.3 * normal(M, B)).to(dt)
        s["codes"], s["scales"] = _store8(spread(K, B).to(dt))
        s["dw"] = torch.empty(M, K, device=dev, dtype=_DTYPES[case["out"]])
        s["alpha"] = 1.0 / B  # the mean over the batch
    elif case["op"] == "backward":
        M, K, B = case["M"], case["K"], case["B"]
        s["w"] = (normal(M, K) / math.sqrt(K)).to(dt)
        s["e"] = (0.3 * normal(M, B)).to(dt)
        s["codes"], s["scales"] = _store8(spread(K, B).to(dt))
        s["e_up"] = torch.empty(K, B, device=dev, dtype=dt)
    elif case["op"] == "quantize":
        R, K = case["R"], case["K"]
        # activations come feature-major, [K, R], with R samples; weights as [R, K]
        s["x"] = spread(K, R).to(dt) if case["turned"] else (normal(R, K) / math.sqrt(K)).to(dt)
        kp = -(-K // 128) * 128
        s["codes"] = torch.empty(R, kp // 2, device=dev, dtype=torch.uint8)
        s["scales"] = torch.empty(-(-R // 128), kp // 128, 32, 4, 4, device=dev, dtype=torch.uint8)
        s["values"] = torch.empty(R, K, device=dev, dtype=torch.bfloat16)
    else:
        M, K, B = case["M"], case["K"], case["B"]
        s["w"], s["w_scales"] = _store4((normal(M, K) / math.sqrt(K)).to(dt).float())
        s["a"], s["a_scales"] = _store4(spread(K, B).to(dt).float().clamp(min=0).t())
        s["out"] = torch.empty(M, B, device=dev, dtype=dt)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from lich_b200 import microscaled as mx

    op, dt = s["op"], s["dtype"]
    if op == "checkpoint":
        D, B = s["D"], s["B"]
        mx.build_checkpoint(D, B, dt)(s["x"], s["codes"], s["scales"])
        mx.build_checkpoint_restore(D, B, s["act"], dt)(s["codes"], s["scales"], s["values"])
        return s["values"]
    if op == "delta":
        mx.build_weight_delta_checkpoint(s["M"], s["K"], s["B"], s["act"], dt, s["alpha"], s["out"])(
            s["dw"], s["e"], s["codes"], s["scales"])
        return s["dw"]
    if op == "backward":
        mx.build_error_backward_checkpoint(s["M"], s["K"], s["B"], s["act"], dt)(
            s["w"], s["e"], s["codes"], s["scales"], s["e_up"])
        return s["e_up"]
    if op == "quantize":
        mx.build_mxfp4_quantize(s["R"], s["K"], s["act"], dt, s["turned"])(s["x"], s["codes"], s["scales"])
        mx.build_mxfp4_restore(s["R"], s["K"], "bfloat16")(s["codes"], s["scales"], s["values"])
        return s["values"]
    mx.build_mxfp4_forward(s["M"], s["K"], s["B"], dt)(s["w"], s["w_scales"], s["a"], s["a_scales"], s["out"])
    return s["out"]


def _run_plain(s):
    op, dt = s["op"], _DTYPES[s["dtype"]]
    if op == "checkpoint":
        codes, scales = _store8(s["x"])
        return _f(s["act"], _load8(codes, scales, s["B"])).to(dt)
    if op == "delta":
        a = _f(s["act"], _load8(s["codes"], s["scales"], s["B"]))
        return (s["alpha"] * (s["e"].float() @ a.t())).to(_DTYPES[s["out"]])
    if op == "backward":
        x = _load8(s["codes"], s["scales"], s["B"])
        return (_df(s["act"], x) * (s["w"].float().t() @ s["e"].float())).to(dt)
    if op == "quantize":
        v = _f(s["act"], s["x"].float())
        codes, scales = _store4(v.t() if s["turned"] else v)
        return _load4(codes, scales, s["K"]).to(torch.bfloat16)
    return (_load4(s["w"], s["w_scales"], s["K"]) @ _load4(s["a"], s["a_scales"], s["K"]).t()).to(dt)


def work(case):
    if case["op"] == "checkpoint":  # x in, the checkpoint out, the values out
        D, B, e = case["D"], case["B"], 2
        return {"bytes": D * B * (2 * e + 1 + 1 / 32), "flops": 0}
    if case["op"] == "quantize":
        R, K, e = case["R"], case["K"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": R * K * (e + 0.5 + 1 / 32 + 2), "flops": 0}
    M, K, B = case["M"], case["K"], case["B"]
    if case["op"] == "delta":
        o = 4 if case["out"] == "float32" else 2
        return {"bytes": 2 * M * B + K * B * (1 + 1 / 32) + o * M * K, "flops": 2 * M * K * B}
    if case["op"] == "backward":
        return {"bytes": 2 * M * K + 2 * M * B + K * B * (1 + 1 / 32) + 2 * K * B, "flops": 2 * M * K * B}
    return {"bytes": (M * K + K * B) * (0.5 + 1 / 32) + 2 * M * B, "flops": 2 * M * K * B}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def block_step(m, top):  # the smallest power of two p with m <= top * p, from 2^-127 up
        frac, exp = torch.frexp(m / top)
        n = torch.where(frac == 0.5, exp - 1, exp).double()
        return torch.exp2(torch.where(m > 0, n, torch.full_like(n, -127.0)).clamp(-127, 127))

    def blocks(v):
        pad = (-v.shape[1]) % 32
        return torch.nn.functional.pad(v, (0, pad)).view(v.shape[0], -1, 32)

    def read8():
        p = torch.exp2(s["scales"].double() - 127).t()
        return (s["codes"].double().view(p.shape[0], -1, 32) * p[..., None]).flatten(1)[:, :case["B"]]

    def read4(codes, scales):
        grid = torch.tensor(list(_GRID) + [-v for v in _GRID], device=codes.device, dtype=torch.float64)
        R, kp = codes.shape[0], 2 * codes.shape[1]
        k = torch.arange(kp, device=codes.device)
        r = torch.arange(R, device=codes.device)[:, None]
        c = (codes[:, k // 2].to(torch.int64) >> (4 * (k % 2))) & 15
        j = (k // 32)[None, :]
        b = scales[r // 128, j // 4, r % 32, r % 128 // 32, j % 4]
        return (grid[c] * torch.exp2(b.double() - 127))[:, :case["K"]]

    def act(x):
        y = {"relu": lambda: torch.relu(x), "tanh": lambda: torch.tanh(x), "sigmoid": lambda: torch.sigmoid(x),
             "silu": lambda: x * torch.sigmoid(x), "identity": lambda: x,
             "gelu": lambda: torch.nn.functional.gelu(x, approximate="tanh")}
        return y[case["act"]]()

    if op == "checkpoint":
        v = blocks(s["x"].double())
        p = block_step(v.abs().amax(-1), 127.0)[..., None]
        return act((torch.round(v / p) * p).flatten(1)[:, :case["B"]])
    if op == "quantize":
        v = act(s["x"].double())
        v = blocks(v.t().contiguous() if case["turned"] else v)
        p = block_step(v.abs().amax(-1), 6.0)[..., None]
        u = (v / p).abs()
        mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=v.device, dtype=torch.float64)
        lo, hi = torch.bucketize(u, mids), torch.bucketize(u, mids, right=True)
        idx = torch.where(lo % 2 == 0, lo, hi)  # equal but on a tie, where one of the two is even
        grid = torch.tensor(_GRID, device=v.device, dtype=torch.float64)
        return (torch.sign(v) * grid[idx] * p).flatten(1)[:, :case["K"]]
    if op == "delta":
        return s["alpha"] * (s["e"].double() @ act(read8()).t())
    if op == "backward":
        x = read8().requires_grad_()
        slope, = torch.autograd.grad(act(x).sum(), x)
        return slope * (s["w"].double().t() @ s["e"].double())
    return read4(s["w"], s["w_scales"]) @ read4(s["a"], s["a_scales"]).t()
