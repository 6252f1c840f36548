"""MXFP4 conversion, bit for bit against its definition, products with such weights against float64, and
the dense block on them."""
import pytest
import torch

from flash_distributed_moe_amd import synth
from tests import ffn_case

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from flash_distributed_moe_amd import flashFfnOp

    return flashFfnOp


def normal(*shape, sigma=1.0, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(2000 + seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, sigma, generator=gen)


def same(q, x):
    codes, scales = ffn_case.mx_encode(x)
    assert torch.equal(q.scales, scales)
    known = (scales != 255).repeat_interleave(16, -1)  # the codes of a block of NaN say nothing
    assert torch.equal(q.codes[known], codes[known])


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 32), (64, 4096), (257, 160), (2, 7, 64), (1000, 2048), (32,)])
def test_conversion(ops, shape, dtype):
    x = normal(*shape, dtype=torch.float32) * torch.exp(3 * normal(*shape[:-1], 1, dtype=torch.float32, seed=1))
    x = x.to(DTYPES[dtype])
    q = ops.quantize_mxfp4(x)
    assert q.codes.shape == (*shape[:-1], shape[-1] // 2) and q.scales.shape == (*shape[:-1], shape[-1] // 32)
    same(q, x)
    for dt in DTYPES.values():
        back = ops.dequantize_mxfp4(q, dt)
        assert back.dtype == dt and torch.equal(back.double(), ffn_case.mx_values(q.codes, q.scales))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_ties_ends_and_special_values(ops, dtype):
    """Every tie of the grid, the values next to it, zeros of both signs, the ends of the exponents, and
    blocks with infinities and NaN (which become all NaN), each beside ordinary blocks."""
    dt = DTYPES[dtype]
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    near = torch.cat((mid, mid * (1 + 2.0 ** -6), mid * (1 - 2.0 ** -6), torch.tensor([0.0, -0.0, 6.0, 7.5, 4.0], device="cuda")))
    block = torch.cat((near, -near[:6]))
    assert block.numel() == 32
    rows = [block * 2.0 ** e for e in (0, 1, -1, 60, -60, -100, -118, -120, -122, 124)]
    for e in (-126, -130, -133):  # values below the smallest normal number
        rows.append(block.sign() * 2.0 ** e)
    rows += [torch.zeros(32, device="cuda"), -torch.zeros(32, device="cuda")]
    for v in (float("inf"), float("-inf"), float("nan")):
        bad = block.clone()
        bad[17] = v
        rows.append(bad)
    rows.append(torch.full((32,), torch.finfo(dt).max, device="cuda", dtype=dt).float())
    rows.append(torch.full((32,), torch.finfo(dt).tiny, device="cuda", dtype=dt).float())
    x = torch.stack([torch.cat((r, block)) for r in rows]).to(dt)
    q = ops.quantize_mxfp4(x)
    same(q, x)
    values = ops.dequantize_mxfp4(q, dt)
    bad = ~torch.isfinite(x).reshape(len(rows), 2, 32).all(-1)
    assert torch.equal(torch.isnan(values).reshape(len(rows), 2, 32).all(-1), bad) and int(bad.sum()) == 3
    assert torch.equal(torch.isnan(values).reshape(len(rows), 2, 32).any(-1), bad)


def test_every_code_under_every_scale(ops):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(256, 1)  # 512 values a row, all 256 bytes
    scales = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None].repeat(1, 16)
    want = ffn_case.mx_values(codes, scales)
    for dt in DTYPES.values():
        got = ops.dequantize_mxfp4(ops.Mxfp4(codes, scales), dt)
        # beyond the largest float (scales 253 and 254) the value is an infinity
        expect = want.float().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert torch.equal(got.double()[fine], expect[fine])


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_conversion_of_rows_apart(ops, dtype):
    wide = normal(19, 192, dtype=DTYPES[dtype], seed=3)
    for view in (wide[:, 64:128], wide[::2, :96], wide[:, 3:99], wide.t()[:, :0].reshape(192, 0).new_zeros(0, 64), wide[:0]):
        q, p = ops.quantize_mxfp4(view), ops.quantize_mxfp4(view.contiguous().clone())
        assert torch.equal(q.codes, p.codes) and torch.equal(q.scales, p.scales)


def weights(ops, N, K, seed=0, sigma=0.02):
    return ops.quantize_mxfp4(normal(N, K, sigma=sigma, seed=seed))


def check_product(got, x, w):
    """x, w float64. Every MXFP4 value is a bfloat16, and products are exact in float32; the sum is off by
    at most 2 K 2^-24 of the magnitudes, the result by 2^-8 of itself."""
    value = x @ w.t()
    far = 2.0 * x.shape[1] * 2.0 ** -24 * (x.abs() @ w.abs().t())
    ffn_case.check(got, value, far + 2.0 ** -8 * (value.abs() + far), "product %s x %s" % (tuple(x.shape), tuple(w.shape)))


PRODUCTS = [(1, 8, 32), (1, 1, 32), (2, 129, 96), (5, 136, 4096), (16, 64, 64), (17, 300, 160), (31, 257, 2048), (64, 128, 512),
            (65, 384, 288), (130, 257, 320), (257, 520, 544), (300, 1000, 1056), (33, 1000, 384), (257, 136, 640), (3841, 3600, 384),
            (3841, 3600, 160), (1024, 8200, 256), (256, 8200, 512), (64, 8200, 1056), (520, 8192, 2080),
            (40, 37, 5120), (93, 200, 7520), (703, 72, 4096),
            (8, 300, 16384), (16, 300, 16384), (32, 300, 16384), (32, 300, 16416)]  # the longest rows whose scales fit LDS, and longer


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear(ops, M, N, K):
    x, w = normal(M, K, seed=1), weights(ops, N, K)
    got = ops.mxfp4_linear(x, w)
    assert got.shape == (M, N) and got.dtype == torch.bfloat16 and got.is_contiguous()
    check_product(got, x.double(), ffn_case.mx_values(*w))


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear_of_two_in_four_bits(ops, M, N, K):
    x, w = ops.quantize_mxfp4(normal(M, K, seed=1) * torch.exp(normal(M, 1, seed=2))), weights(ops, N, K)
    got = ops.mxfp4_linear(x, w)
    assert got.shape == (M, N) and got.dtype == torch.bfloat16
    check_product(got, ffn_case.mx_values(*x), ffn_case.mx_values(*w))


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M", [1, 3, 12, 30, 40, 200])
def test_scales_of_every_size_and_nan(ops, M, both):
    """Blocks whose scales lie 2^60 apart, a zero block, and a weight row with a block of NaN: its results are NaN,
    no other's are."""
    N, K = 72, 256
    x, w = normal(M, K, seed=4), normal(N, K, seed=5, dtype=torch.float32)
    w = w.reshape(N, -1, 32) * torch.exp2(torch.randint(-30, 31, (N, K // 32, 1), generator=torch.Generator().manual_seed(0)).cuda().float())
    w[3, 2] = 0
    w = ops.quantize_mxfp4(w.reshape(N, K))
    w.scales[0, 1] = 255
    w.scales[N - 1, K // 32 - 1] = 255
    if both:
        x = ops.quantize_mxfp4(x)
    got = ops.mxfp4_linear(x, w)
    bad = torch.zeros(N, dtype=torch.bool, device="cuda")
    bad[[0, N - 1]] = True
    assert torch.isnan(got[:, bad]).all()
    values = ffn_case.mx_values(*w)[~bad]
    check_product(got[:, ~bad], ffn_case.mx_values(*x) if both else x.double(), values)


def test_infinite_rows_keep_to_themselves(ops):
    w = weights(ops, 130, 160)
    for M in (2, 70):
        x = normal(M, 160, seed=6)
        clean = ops.mxfp4_linear(x, w)
        x[1, 33] = float("inf")
        got = ops.mxfp4_linear(x, w)
        rest = [m for m in range(M) if m != 1]
        assert torch.equal(got[rest], clean[rest]) and not torch.isfinite(got[1]).any()


def test_strides_and_leading_dimensions(ops):
    w = weights(ops, 100, 96)
    wide = normal(14, 300, seed=7)
    x = wide[:, 100:196].contiguous()
    want = ops.mxfp4_linear(x, w)
    assert torch.equal(ops.mxfp4_linear(wide[:, 100:196], w), want)  # rows of 600 bytes: copied
    assert torch.equal(ops.mxfp4_linear(x.view(2, 7, 96), w), want.view(2, 7, 100))
    q = ops.quantize_mxfp4(x)
    both = ops.mxfp4_linear(q, w)
    assert torch.equal(ops.mxfp4_linear(ops.Mxfp4(q.codes.view(2, 7, 48), q.scales.view(2, 7, 3)), w), both.view(2, 7, 100))
    assert ops.mxfp4_linear(x[:0], w).shape == (0, 100)
    assert ops.mxfp4_linear(x, ops.Mxfp4(w.codes[:0], w.scales[:0])).shape == (14, 0)


def mx_block_bound(x, w13, w2, act):
    """The bfloat16 block's bounds hold: the weights are bfloat16 values."""
    v13, v2 = (ffn_case.mx_values(*w).to(torch.bfloat16) for w in (w13, w2))
    assert torch.equal(v13.double(), ffn_case.mx_values(*w13))
    return ffn_case.block(x, v13, v2, act)["y"]


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T,H,I", [(1, 32, 32), (1, 256, 160), (4, 1344, 736), (16, 256, 128), (17, 96, 288), (63, 512, 1024),
                                   (65, 160, 96), (200, 544, 320), (300, 128, 256), (3841, 256, 1920), (16, 512, 12288), (3, 96, 12288), (70, 1024, 2080), (67, 384, 7680),
                                   (50, 4352, 96), (32, 16384, 6144)])
def test_block_on_mxfp4_weights(ops, T, H, I, act):
    x = normal(T, H, seed=8)
    w13, w2 = weights(ops, 2 * I, H, seed=9, sigma=H ** -0.5), weights(ops, H, I, seed=10, sigma=I ** -0.5)
    got = ops.gated_ffn(x, w13, w2, activation=act)
    ffn_case.check(got, *mx_block_bound(x, w13, w2, act), "T=%d H=%d I=%d" % (T, H, I))


class _Linear(torch.nn.Module):
    def __init__(self, weight):
        super().__init__()
        self.weight = torch.nn.Parameter(weight)


class _DenseBlock(torch.nn.Module):
    def __init__(self, w13, w2):
        super().__init__()
        self.gate_up_proj, self.down_proj = _Linear(w13), _Linear(w2)


@pytest.mark.parametrize("T", [1, 24, 200])
def test_sparse_layer_and_shared_expert_together(ops, T):
    """A layer as a model has it: the sparse block and, on the same rows, a shared expert, first in bfloat16 and
    then with its weights converted to 4 bits; eager and as one captured graph."""
    from flash_distributed_moe_amd.flashMoeOp import FlashMoeBlockWrapper
    from tests.test_gpu_module import StandInSparseMoeBlock

    cfg = synth.CONFIGS["qwen3_30b_decode"].replace(T=T)
    inp = synth.make_inputs_torch(cfg, 7907, torch.device("cuda:0"))
    sparse = FlashMoeBlockWrapper(StandInSparseMoeBlock(inp, cfg.k), maxTokens=T)
    block = _DenseBlock(normal(1536, 2048, sigma=0.02, seed=11), normal(2048, 768, sigma=0.02, seed=12))
    for quantize in (None, "mxfp4"):
        shared = ops.FlashGatedFfn(block, quantize=quantize)
        x = inp["tokens"].clone()

        def layer():
            with torch.no_grad():
                s = shared(x)
                return sparse(x.clone()) + s

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer()
        for rep in range(3):
            x.copy_(synth.make_inputs_torch(cfg, 50 + rep, torch.device("cuda:0"))["tokens"])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer())
        with torch.no_grad():
            y = shared(x)
        w13, w2 = block.gate_up_proj.weight, block.down_proj.weight
        if quantize:
            q13, q2 = ops.quantize_mxfp4(w13), ops.quantize_mxfp4(w2)
            ffn_case.check(y, *mx_block_bound(x, q13, q2, "silu"), "shared expert in 4 bits")
        else:
            ffn_case.check(y, *ffn_case.block(x, w13, w2, "silu")["y"], "shared expert")
    sparse.launcher.destroy()
