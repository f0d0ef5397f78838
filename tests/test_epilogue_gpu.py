"""The GEMM with activation, dropout and residual in its epilogue (``nvfp4.epilogue_mm``) against a
64-bit oracle, and ``FP4Linear`` / ``FP4FeedForward`` with it: outputs, gradients, fallback, refusals."""

import pytest
import torch
import torch.nn.functional as F

from tests import _epilogue_oracle as O
from tests._nvfp4_helpers import dequantize_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nv():
    import radiance_b200.nvfp4 as nv

    assert nv.nvfp4_supported()
    return nv


@pytest.fixture(autouse=True)
def _status():
    yield
    from radiance_b200 import _lib

    assert _lib.device_status(clear=True) == 0


def _rand(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _operands(nv, m, n, k, seed=0):
    a, b = _rand(m, k, seed=seed), _rand(n, k, seed=seed + 1, std=2 * k**-0.5)
    qa, qb = nv.quantize(a, -1), nv.quantize(b, -1)
    da = dequantize_gpu(qa.packed, qa.scale, qa.global_scale.double(), m, k).double()
    db = dequantize_gpu(qb.packed, qb.scale, qb.global_scale.double(), n, k).double()
    return qa, qb, da, db


def _check(y, z_out, da, db, k, bias, act, p, seed, residual):
    z = da @ db.t()
    mag = da.abs() @ db.abs().t()
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    # The dequantized factors were rounded to fp32 (2^-24 each); products are exact, 64-wide steps add in
    # fp32; the scales' product, alpha and the bias are one rounding each.
    zerr = (k / 64 + 8) * 2.0**-23 * mag
    hs = O.half_step(y.dtype)
    if z_out is not None:
        assert ((z_out.double() - z).abs() <= hs * z.abs() * 1.01 + zerr).all()
    v = O.activation(z, act)
    slope = (2 * z.abs() + 2 * zerr) if act == "relu2" else torch.full_like(z, 1.13)
    # exp and erf of 2 ulp with an argument off by a few roundings of itself; gelu's 1 + erf loses up to
    # 2^-23 of 1, times |z| / 2: all under 2^-20 |z| (|z|^2 for relu2).
    verr = slope * zerr + 2.0**-20 * (z * z if act == "relu2" else z.abs())
    if act is None:
        verr = zerr
    scale = 65536 / max(1, 65536 - O.threshold(p))
    want, err = O.drop(v, p, seed), verr * scale + 2.0**-22 * v.abs() * scale
    if residual is not None:
        want = want + residual.double()
        err = err + 2.0**-23 * residual.double().abs()
    assert ((y.double() - want).abs() <= hs * want.abs() * 1.01 + err).all()


# (m, n, k): one tile and less, a half-empty pair (m % 256 == 128) with a 128-wide N tail, short last K
# steps, more tiles than CTA pairs (so boxes and barriers go round), many K steps.
SHAPES = [(128, 128, 64), (256, 256, 64), (384, 640, 1088), (128, 2048, 512), (896, 384, 192), (4096, 2304, 128),
          (256, 128, 5632)]
VARIANTS = [  # act, p, residual, preact, bias dtype
    ("gelu", 0.0, False, True, torch.bfloat16),
    (None, 0.1, True, False, torch.float32),
    ("silu", 0.3, True, True, torch.bfloat16),
    ("relu2", 0.0, True, False, None),
    ("gelu_tanh", 0.5, False, False, torch.float32),
    ("relu", 0.0, False, False, None),
    (None, 0.0, True, True, torch.bfloat16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matches_the_oracle(nv, m, n, k, dtype):
    qa, qb, da, db = _operands(nv, m, n, k, seed=m + n)
    for i, (act, p, has_res, pre, bdt) in enumerate(VARIANTS):
        seed = 1000 * i + k
        bias = None if bdt is None else _rand(n, dtype=bdt, seed=5)
        res = _rand(m, n, dtype=dtype, seed=6) if has_res else None
        got = nv.epilogue_mm(qa, qb, bias=bias, activation=act, dropout_p=p, seed=seed, residual=res, out_dtype=dtype,
                             save_preact=pre)
        y, z = got if pre else (got, None)
        assert y.dtype == dtype and y.shape == (m, n)
        _check(y, z, da, db, k, bias, act, p, seed, res)
        again = nv.epilogue_mm(qa, qb, bias=bias, activation=act, dropout_p=p, seed=seed, residual=res,
                               out_dtype=dtype)
        assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_agrees_with_mm_and_dropout(nv, dtype):
    qa, qb, _, _ = _operands(nv, 640, 768, 320)
    bias = _rand(768, dtype=torch.bfloat16, seed=3)
    plain = nv.mm(qa, qb, out_dtype=dtype, bias=bias)
    y, z = nv.epilogue_mm(qa, qb, bias=bias, out_dtype=dtype, save_preact=True)
    assert torch.equal(y, plain) and torch.equal(z, plain)
    if dtype == torch.float32:  # no rounding in between: the same mask, the same product
        assert torch.equal(nv.epilogue_mm(qa, qb, bias=bias, out_dtype=dtype, dropout_p=0.4, seed=9),
                           nv.dropout(plain, 0.4, seed=9))
    assert (nv.epilogue_mm(qa, qb, bias=bias, out_dtype=dtype, dropout_p=1.0, seed=9) == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [128, 4096])
def test_in_place_and_strided(nv, m, dtype):
    n, k = 2304, 128
    qa, qb, _, _ = _operands(nv, m, n, k)
    res = _rand(m, n, dtype=dtype, seed=4)
    want = nv.epilogue_mm(qa, qb, activation="silu", dropout_p=0.2, seed=1, residual=res, out_dtype=dtype)
    stream = res.clone()
    assert nv.epilogue_mm(qa, qb, activation="silu", dropout_p=0.2, seed=1, residual=stream, out=stream,
                          out_dtype=dtype) is stream
    assert torch.equal(stream, want)
    # Columns of a wider buffer, the residual beside the output in it; nothing else of it changes.
    wide = torch.full((m, 2 * n + 64), 7.0, dtype=dtype, device="cuda")
    wide[:, :n] = res
    out = wide[:, n + 32:2 * n + 32]
    nv.epilogue_mm(qa, qb, activation="silu", dropout_p=0.2, seed=1, residual=wide[:, :n], out=out, out_dtype=dtype)
    assert torch.equal(out, want) and torch.equal(wide[:, :n], res)
    assert (wide[:, n:n + 32] == 7).all() and (wide[:, 2 * n + 32:] == 7).all()
    # A residual that TMA cannot read in place (odd alignment), or transposed.
    odd = torch.empty(m * n + 1, dtype=dtype, device="cuda")[1:].view(m, n).copy_(res)
    tr = res.t().contiguous().t()
    for r in (odd, tr):
        assert torch.equal(nv.epilogue_mm(qa, qb, activation="silu", dropout_p=0.2, seed=1, residual=r,
                                          out_dtype=dtype), want)


def test_nan_and_infinite_residuals(nv):
    qa, qb, _, _ = _operands(nv, 256, 256, 64)
    res = _rand(256, 256, dtype=torch.bfloat16, seed=4)
    res[3, 4], res[200, 130], res[255, 255] = float("nan"), float("inf"), -float("inf")
    y = nv.epilogue_mm(qa, qb, residual=res)
    assert torch.equal(torch.isnan(y), torch.isnan(res)) and torch.equal(torch.isinf(y), torch.isinf(res))


def test_stream_and_graph(nv):
    qa, qb, _, _ = _operands(nv, 512, 512, 256)
    res, seed = _rand(512, 512, dtype=torch.bfloat16, seed=4), torch.tensor(3, device="cuda")

    def call():
        return nv.epilogue_mm(qa, qb, activation="gelu", dropout_p=0.2, seed=seed, residual=res, save_preact=True)

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    seed.fill_(4)
    res.mul_(2)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, call())) and not torch.equal(out[0], want[0])


# ------------------------------------------------------------------------------------------------
# FP4Linear and FP4FeedForward
# ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("act,p,has_res", [("gelu", 0.0, False), (None, 0.2, True), ("silu", 0.1, True),
                                           (None, 0.0, True)])
def test_linear_gradients(nv, act, p, has_res, bias, dtype):
    """The epilogue's gradients are the plain layer's on the gradient of the pre-activations."""
    torch.manual_seed(1)
    layer = nv.FP4Linear(256, 384, bias=bias).cuda()
    if bias:
        torch.nn.init.normal_(layer.bias)
    layer.refresh_fp4_cache()
    x = _rand(2, 128, 256, dtype=dtype, seed=1).requires_grad_()
    res = _rand(2, 128, 384, dtype=dtype, seed=2).requires_grad_() if has_res else None
    gy = _rand(2, 128, 384, dtype=dtype, seed=3, std=1e-2)
    y = layer(x, activation=act, dropout_p=p, dropout_seed=77, residual=res)
    assert y.shape == (2, 128, 384) and y.dtype == dtype
    leaves = [x, layer.weight] + ([layer.bias] if bias else []) + ([res] if has_res else [])
    got = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, gy)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # The same through the plain layer: its output is the pre-activation, the gradient comes from the oracle.
    z = layer(x)
    zd, hs = z.detach().double(), O.half_step(dtype)
    want = O.drop(O.activation(zd, act).reshape(256, 384), p, 77).reshape(y.shape)
    # z was rounded to its type here and not in the epilogue (|act'| <= 1.13).
    room = 1.13 * hs * zd.abs() / (1 - p) + 2.0**-19 * (zd.abs() + 1)
    if has_res:
        want = want + res.detach().double()
    assert ((y.detach().double() - want).abs() <= hs * want.abs() * 1.01 + room).all()
    gz = gy.reshape(256, 384)
    if act is not None or p > 0:
        gz, _, sums = nv.epilogue_backward(gz, z.detach().reshape(256, 384), activation=act, dropout_p=p, seed=77,
                                           bias_grad=True)
        # One rounding to the type, and the derivative's fp32 evaluation: under 2^-18 of max(1, 2 |z|)'s 1 here
        # (exp and erf of 2 ulp, arguments off by 2^-22 of themselves, terms of at most 1.2).
        g = O.drop(gy.reshape(256, 384).double(), p, 77)
        wz = g * O.derivative(zd.reshape(256, 384), act)
        assert ((gz.double() - wz).abs() <= hs * wz.abs() * 1.01 + 2.0**-18 * g.abs()).all()
    ref = torch.autograd.grad(z, leaves[:2 + bias], gz.reshape(2, 128, 384))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    if bias:
        # The plain layer sums the rounded gradient and rounds the sum to the gradient's type, as does this one.
        exact = gz.double().sum(0)
        bound = 2 * hs * exact.abs() + hs * gz.double().abs().sum(0) + 256 * 2.0**-24 * gz.double().abs().sum(0)
        assert ((got[2].double() - exact).abs() <= bound).all()
    if has_res:
        assert torch.equal(got[-1], gy)


@pytest.mark.parametrize("recipe", [dict(save_activations=False), dict(grad_gemms=False),
                                    dict(stochastic_rounding=False, hadamard=False)])
def test_linear_recipes(nv, recipe):
    """Every recipe's backward takes the epilogue's gradient as it takes the plain layer's."""
    torch.manual_seed(1)
    layer = nv.FP4Linear(256, 384, recipe=nv.FP4Recipe(**recipe)).cuda()
    layer.refresh_fp4_cache()
    x = _rand(128, 256, dtype=torch.bfloat16, seed=1).requires_grad_()
    res, gy = _rand(128, 384, dtype=torch.bfloat16, seed=2), _rand(128, 384, dtype=torch.bfloat16, seed=3, std=1e-2)
    y = layer(x, activation="silu", dropout_p=0.1, dropout_seed=7, residual=res)
    got = torch.autograd.grad(y, (x, layer.weight), gy)
    z = layer(x)
    gz, _, _ = nv.epilogue_backward(gy, z.detach(), activation="silu", dropout_p=0.1, seed=7)
    ref = torch.autograd.grad(z, (x, layer.weight), gz)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_linear_fallback_and_refusals(nv):
    torch.manual_seed(1)
    layer = nv.FP4Linear(256, 384).cuda()
    layer.refresh_fp4_cache()
    x, res = _rand(100, 256, dtype=torch.bfloat16, seed=1), _rand(100, 384, dtype=torch.bfloat16, seed=2)
    y = layer(x, activation="gelu", dropout_p=0.2, dropout_seed=4, residual=res)  # 100 rows: the bf16 path
    z = F.gelu(F.linear(x, layer.weight.bfloat16(), layer.bias.bfloat16()))
    assert torch.equal(y, nv.dropout(z, 0.2, seed=4, residual=res))
    for name in ("relu", "relu2", "silu", "gelu_tanh"):
        w = layer(x, activation=name).double()
        zd = F.linear(x, layer.weight.bfloat16(), layer.bias.bfloat16()).double()
        # bf16 roundings of the torch ops: one, or two for the square
        assert ((w - O.activation(zd, name)).abs() <= 2.5 * 2.0**-8 * O.activation(zd, name).abs() + 1e-6).all()
    x = _rand(128, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="activation"):
        layer(x, activation="swish")
    with pytest.raises(ValueError, match="residual"):
        layer(x, residual=_rand(128, 384))
    with pytest.raises(ValueError, match="residual"):
        layer(x, residual=res)
    with pytest.raises(ValueError, match="probability"):
        layer(x, dropout_p=1.5)
    with pytest.raises(ValueError, match="unsupported dtype"):
        layer(x.half(), dropout_p=0.5)
    layer.output_gemm = lambda *a: None
    with pytest.raises(ValueError, match="N-split"):
        layer(x, dropout_p=0.5)


def test_mm_refusals(nv):
    qa, qb, _, _ = _operands(nv, 256, 256, 64)
    short = nv.quantize(_rand(256, 128), -1)
    res = _rand(256, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="contraction"):
        nv.epilogue_mm(qa, short)
    for bad in (qa.packed.view(torch.uint8)[:, ::2].view(torch.uint8), qa.packed):
        scale = qa.scale[:100] if bad is qa.packed else qa.scale
        with pytest.raises(ValueError, match="contraction|needs contiguous"):
            nv.epilogue_mm(nv.NVFP4Tensor(bad, scale, qa.global_scale), qb)
    with pytest.raises(ValueError, match="needs contiguous"):
        nv.epilogue_mm(nv.NVFP4Tensor(qa.packed, qa.scale, qa.global_scale.double()), qb)
    with pytest.raises(ValueError, match="must be on"):
        nv.epilogue_mm(qa, nv.NVFP4Tensor(qb.packed, qb.scale, qb.global_scale.cpu()))
    with pytest.raises(ValueError, match="output dtype"):
        nv.epilogue_mm(qa, qb, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="activation"):
        nv.epilogue_mm(qa, qb, activation="elu")
    with pytest.raises(ValueError, match="bias"):
        nv.epilogue_mm(qa, qb, bias=_rand(255))
    with pytest.raises(ValueError, match="residual"):
        nv.epilogue_mm(qa, qb, residual=res.float())
    with pytest.raises(ValueError, match="out must be 16-byte"):
        nv.epilogue_mm(qa, qb, out=torch.empty(256 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(256, 256))
    buf = torch.zeros(257 * 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        nv.epilogue_mm(qa, qb, residual=buf[:65536].view(256, 256), out=buf[256:].view(256, 256))
    with pytest.raises(ValueError, match="m % 128"):
        nv.epilogue_mm(nv.NVFP4Tensor(qa.packed[:100], qa.scale, qa.global_scale), qb)


def test_feed_forward_with_residual(nv):
    torch.manual_seed(2)
    ff = nv.FP4FeedForward(256, 512, dropout=0.25).cuda()
    nv.refresh_fp4_weights(ff)
    x = _rand(4, 64, 256, dtype=torch.bfloat16, seed=1).requires_grad_()
    ff.eval()
    y, plain = ff(x, residual=x), ff(x)
    want = x.detach().double() + plain.detach().double()
    room = O.half_step(torch.bfloat16) * (want.abs() + plain.detach().double().abs()) * 1.01 + 2.0**-20
    assert ((y.detach().double() - want).abs() <= room).all()
    ff.train()
    torch.manual_seed(5)
    y = ff(x, residual=x)
    torch.manual_seed(5)
    assert torch.equal(ff(x, residual=x), y)
    gone = (y == x).float().mean().item()
    assert 0.2 < gone < 0.3  # a dropped element leaves the residual as it is
    y.float().square().mean().backward()
    assert torch.isfinite(x.grad).all() and torch.isfinite(ff.down_proj.weight.grad).all()
