"""The dense gated feed-forward block and the microscaled 4-bit format (MXFP4), as cases that can
be timed and compared.

The operators stand beside the sparse layer of `cases.py`: the dense layers and the shared expert of
the same models are gated feed-forward blocks, y = (act(x Wg^T) * (x Wu^T)) Wd^T, on the layer's
weight layouts (w13 [2I, H]: gate rows, then up rows; w2 [H, I]), and MXFP4 is how the weights of
either are kept at a quarter of their size: 32 consecutive values of a row share a scale 2^s (a byte,
s + 127), each value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (4 bits, the even one in the
low half of its byte).

A case is a dict with "op" and that operator's sizes:
  ffn         T, H, I, dtype, act    the block's forward pass
  ffn_train   T, H, I, dtype, act    forward and backward: output, gradients of x and both weights
  ffn_mxfp4   T, H, I, act           the forward pass on MXFP4 weights, bf16 tokens
  roundtrip   R, K, dtype            quantisation of R rows of K values and the values they stand for
  linear      M, N, K                bf16 rows times MXFP4 weights
  linear_both M, N, K                MXFP4 rows times MXFP4 weights
The dtype is "bf16" or "f32": inputs and outputs.
"""
import torch

own = False

SIGMA_W = 0.02
BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _ffn(T, H, I, dtype="bf16", act="silu", op="ffn"):
    return dict(op=op, T=T, H=H, I=I, dtype=dtype, act=act)


def listed():
    named = [
        # one sequence being decoded: a dense block as wide as eight experts, weights read once
        ("ffn_decode_1", _ffn(1, 2048, 6144)),
        # the layer of the first test anyone runs: launch latency only
        ("ffn_tiny_f32", _ffn(16, 256, 128, dtype="f32")),
        # a chunk of a prompt through a shared expert of ragged width, with the other activation
        ("ffn_chunk_ragged", _ffn(333, 1344, 736, act="gelu_tanh")),
        # a long prompt through the large model's dense block
        ("ffn_prefill_8192", _ffn(8192, 4096, 12288)),
        # a training step of the dense block
        ("ffn_train_4096", _ffn(4096, 2048, 6144, op="ffn_train")),
        # a training step in the reference's dtype, an odd number of tokens
        ("ffn_train_f32_1001", _ffn(1001, 2048, 768, dtype="f32", op="ffn_train")),
        # a decode batch through the large model's block, its weights in 4 bits
        ("ffn_mxfp4_decode_16", dict(op="ffn_mxfp4", T=16, H=4096, I=12288, act="silu")),
        # the rows of a decode batch: launch latency
        ("roundtrip_rows_f32", dict(op="roundtrip", R=64, K=4096, dtype="f32")),
        # a model's weights being converted
        ("roundtrip_weights", dict(op="roundtrip", R=24576, K=4096, dtype="bf16")),
        # a handful of sequences through one 4-bit projection
        ("linear_decode_5", dict(op="linear", M=5, N=4096, K=12288)),
        # a prompt through a 4-bit projection
        ("linear_prefill_2048", dict(op="linear", M=2048, N=8192, K=4096)),
        # the same with the rows in 4 bits too
        ("linear_both_4096", dict(op="linear_both", M=4096, N=8192, K=4096)),
    ]
    return [dict(name=name, **case) for name, case in named]


# No drawn case costs more than the largest listed one of its operator.
_MOST_FLOPS = {"ffn": 2.47e12, "ffn_train": 9.2e11, "ffn_train_f32": 2.8e10, "ffn_f32": 2.0e11,
               "ffn_mxfp4": 1.2e12, "linear": 2.7e11, "linear_both": 2.7e11}
_MOST_VALUES = 24576 * 4096


def _log_int(rng, lo, hi, of=1):
    """A multiple of `of` in lo..hi, spread over its logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return max(-(-lo // of), min(hi // of, int(round(v / of)))) * of


def draw(rng):
    while True:
        op = rng.choice(["ffn", "ffn", "ffn_train", "ffn_train", "ffn_mxfp4", "roundtrip", "linear", "linear", "linear_both"])
        if op == "roundtrip":
            case = dict(op=op, R=_log_int(rng, 1, 24576), K=_log_int(rng, 32, 16384, 32), dtype=rng.choice(["bf16", "bf16", "f32"]))
            if case["R"] * case["K"] <= _MOST_VALUES // (1 if case["dtype"] == "bf16" else 2):
                return case
        elif op in ("linear", "linear_both"):
            # few rows (decode) and many (prompts), any number of them and of weight rows
            M = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 64, 8192)
            case = dict(op=op, M=M, N=_log_int(rng, 128, 16384), K=_log_int(rng, 128, 16384, 32))
            if work(case)["flops"] <= _MOST_FLOPS[op] and case["N"] * case["K"] <= _MOST_VALUES:
                return case
        else:
            of = 32 if op == "ffn_mxfp4" else 8
            T = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 64, 8192)
            case = dict(op=op, T=T, H=_log_int(rng, 128, 4096, of), I=_log_int(rng, 64, 12288, of),
                        act=rng.choice(["silu", "silu", "gelu_tanh"]))
            kind = op
            if op != "ffn_mxfp4":
                case["dtype"] = rng.choice(["bf16", "bf16", "bf16", "f32"])
                kind += "_f32" if case["dtype"] == "f32" else ""
            if work(case)["flops"] <= _MOST_FLOPS[kind]:
                return case


def _dtype(case):
    return torch.float32 if case.get("dtype") == "f32" else torch.bfloat16


def prepare(case, seed):
    dev, dt = torch.device("cuda:0"), _dtype(case)
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def normal(sigma, *shape, dtype=dt):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, sigma, generator=gen)

    state = dict(op=case["op"], act=case.get("act"))
    if case["op"] in ("ffn", "ffn_train", "ffn_mxfp4"):
        T, H, I = case["T"], case["H"], case["I"]
        state.update(x=normal(1.0, T, H), w13=normal(SIGMA_W, 2 * I, H), w2=normal(SIGMA_W, H, I))
        if case["op"] == "ffn_train":
            state["dy"] = normal(1e-2, T, H)
            state["leaves"] = [state[k].requires_grad_() for k in ("x", "w13", "w2")]
        if case["op"] == "ffn_mxfp4":
            state["w13"], state["w2"] = _encode(state["w13"]), _encode(state["w2"])
    elif case["op"] == "roundtrip":
        # rows of different sizes, and in every row some columns far larger than the others
        x = normal(1.0, case["R"], case["K"], dtype=torch.float32)
        x *= torch.exp(normal(1.0, case["R"], 1, dtype=torch.float32))
        x *= torch.where(normal(1.0, 1, case["K"], dtype=torch.float32) > 2.0, 20.0, 1.0)
        state["x"] = x.to(dt)
    else:
        state["w"] = _encode(normal(SIGMA_W, case["N"], case["K"]))
        state["x"] = normal(1.0, case["M"], case["K"])
        if case["op"] == "linear_both":
            state["x"] = _encode(state["x"])
    return state


# ------------------------------------------------------------------ plain forms
def _encode(w):
    """(codes uint8 [R, K/2], scales uint8 [R, K/32]) of w [R, K]: s = floor(log2(largest of the
    block)) - 2, values to the nearest of the grid, ties to the even code."""
    v = w.detach().float().reshape(w.shape[0], -1, BLOCK)
    s = (torch.frexp(v.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    a = torch.ldexp(v, -s[..., None])
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = code + torch.signbit(a).to(torch.uint8) * 8
    code = code.reshape(w.shape)
    return (code[:, 0::2] + code[:, 1::2] * 16).contiguous(), (s + 127).to(torch.uint8)


def _decode(codes, scales):
    """float32 values of codes and scales."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float32, device=codes.device)
    at = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1, BLOCK)
    v = torch.ldexp(grid[at.long()], scales.to(torch.int32)[..., None] - 127)
    return v.reshape(codes.shape[0], -1)


def _act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _act_slope(g, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    t = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * g * g)


def _block(x, w13, w2, act):
    """(output, gate and up products, h), all float32."""
    g, u = (x @ w13.t()).chunk(2, -1)
    h = _act(g, act) * u
    return h @ w2.t(), g, u, h


def _run_plain(state):
    op, x = state["op"], state["x"]
    if op == "roundtrip":
        return _decode(*_encode(x)).to(x.dtype)
    if op == "linear":
        return (x.float() @ _decode(*state["w"]).t()).to(x.dtype)
    if op == "linear_both":
        return (_decode(*x) @ _decode(*state["w"]).t()).to(torch.bfloat16)
    if op == "ffn_mxfp4":
        return _block(x.float(), _decode(*state["w13"]), _decode(*state["w2"]), state["act"])[0].to(x.dtype)
    with torch.no_grad():
        xf, w13, w2 = x.float(), state["w13"].float(), state["w2"].float()
        y, g, u, h = _block(xf, w13, w2, state["act"])
        if op == "ffn":
            return y.to(x.dtype)
        dy = state["dy"].float()
        dh = dy @ w2
        dgu = torch.cat((dh * u * _act_slope(g, state["act"]), dh * _act(g, state["act"])), -1)
        return dict(y=y.to(x.dtype), dx=(dgu @ w13).to(x.dtype), dw13=(dgu.t() @ xf).to(x.dtype),
                    dw2=(dy.t() @ h).to(x.dtype))


def _run_own(state):
    from flash_distributed_moe_amd import flashFfnOp as ops

    op, x = state["op"], state["x"]
    if op == "roundtrip":
        return ops.dequantize_mxfp4(ops.quantize_mxfp4(x), x.dtype)
    if op == "linear":
        return ops.mxfp4_linear(x, ops.Mxfp4(*state["w"]))
    if op == "linear_both":
        return ops.mxfp4_linear(ops.Mxfp4(*x), ops.Mxfp4(*state["w"]))
    if op == "ffn_mxfp4":
        return ops.gated_ffn(x, ops.Mxfp4(*state["w13"]), ops.Mxfp4(*state["w2"]), activation=state["act"])
    y = ops.gated_ffn(x, state["w13"], state["w2"], activation=state["act"])
    if op == "ffn":
        return y
    dx, dw13, dw2 = torch.autograd.grad(y, state["leaves"], state["dy"])
    return dict(y=y.detach(), dx=dx, dw13=dw13, dw2=dw2)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """Every input read once and every output written once (weights in 4 bits with a byte for 32 of
    them: 17 bytes a block); a training step reads x, the weights and the output's gradient and
    writes the output and three gradients. The products of the definition are the operations."""
    size = 4 if case.get("dtype") == "f32" else 2
    op = case["op"]
    if op == "roundtrip":
        n = case["R"] * case["K"]
        return {"bytes": 2.0 * n * size + 2.0 * n * 17 / 32, "flops": 0.0}
    if op in ("linear", "linear_both"):
        M, N, K = case["M"], case["N"], case["K"]
        rows = M * K * (2 if op == "linear" else 17 / 32)
        return {"bytes": N * K * 17 / 32 + rows + M * N * 2.0, "flops": 2.0 * M * N * K}
    T, H, I = case["T"], case["H"], case["I"]
    if op == "ffn_mxfp4":
        return {"bytes": 3.0 * H * I * 17 / 32 + 2 * T * H * 2, "flops": 6.0 * T * H * I}
    if op == "ffn":
        return {"bytes": (3.0 * H * I + 2 * T * H) * size, "flops": 6.0 * T * H * I}
    return {"bytes": (2 * 3.0 * H * I + 4 * T * H) * size, "flops": 18.0 * T * H * I}


# ------------------------------------------------------------------ the definition, in 64 bits
_VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _exact_values(codes, scales):
    """float64 [R, K]: (-1)^sign * grid * 2^(byte - 127), a block a column of 32 values."""
    low, high = codes.long() % 16, codes.long() // 16
    both = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.long, device=codes.device)
    both[:, ::2], both[:, 1::2] = low, high
    v = _VALUES.to(codes.device)[both % 8] * (1 - 2 * (both // 8)).double()
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(BLOCK, dim=1)


def _exact_roundtrip(x):
    """Of the grid's values at the block's scale the nearest one; of two as near the one at an even place."""
    v = x.detach().double().reshape(-1, BLOCK)
    most = v.abs().max(dim=1, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(most)) - 2.0)
    grid = _VALUES.to(x.device)
    place = torch.tensor([0.0, 1e-12, 0.0, 1e-12, 0.0, 1e-12, 0.0, 1e-12], dtype=torch.float64, device=x.device)
    out = torch.empty_like(v)
    for lo in range(0, v.shape[0], 1 << 18):  # eight distances a value
        part = v[lo:lo + (1 << 18)] / scale[lo:lo + (1 << 18)]
        far = (part.abs()[..., None] - grid).abs() + place
        out[lo:lo + (1 << 18)] = grid[far.argmin(-1)] * torch.where(part < 0, -1.0, 1.0)
    return torch.where(most > 0, out * scale, torch.zeros_like(out)).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    op = state["op"]
    if op == "roundtrip":
        return _exact_roundtrip(state["x"])
    x = _exact_values(*state["x"]) if op == "linear_both" else state["x"].detach().double()
    if op in ("linear", "linear_both"):
        return torch.matmul(x, _exact_values(*state["w"]).T)
    w13, w2 = (_exact_values(*state[k]) if op == "ffn_mxfp4" else state[k].detach().double() for k in ("w13", "w2"))
    I = w2.shape[1]
    gate, up = torch.matmul(x, w13[:I].T), torch.matmul(x, w13[I:].T)
    if state["act"] == "silu":
        sig = torch.special.expit(gate)
        a, slope = gate * sig, sig + gate * sig * (1 - sig)
    else:
        c = (2.0 / torch.pi) ** 0.5
        t = torch.tanh(c * gate * (1 + 0.044715 * gate ** 2))
        a, slope = gate * (1 + t) / 2, (1 + t) / 2 + gate / 2 * (1 - t ** 2) * c * (1 + 3 * 0.044715 * gate ** 2)
    y = torch.matmul(a * up, w2.T)
    if op != "ffn_train":
        return y
    dy = state["dy"].double()
    dh = torch.matmul(dy, w2)
    dgate, dup = dh * up * slope, dh * a
    return dict(y=y, dx=torch.matmul(dgate, w13[:I]) + torch.matmul(dup, w13[I:]),
                dw13=torch.cat((torch.matmul(dgate.T, x), torch.matmul(dup.T, x))), dw2=torch.matmul(dy.T, a * up))
