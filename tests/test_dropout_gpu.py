"""Counter-based dropout (``nvfp4.dropout``) and the epilogue's backward (``nvfp4.epilogue_backward``)
against 64-bit oracles: masks bit for bit, values to their roundings, gradients, odd sizes, strides
and alignments, streams and captured graphs, refusals."""

import pytest
import torch

from tests import _epilogue_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nv():
    import radiance_b200.nvfp4 as nv

    assert nv.nvfp4_supported()
    return nv


def _rand(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _check_dropout(y, x, residual, p, seed):
    want = O.drop(x.double(), p, seed)
    # The scale, the product and the sum are rounded to fp32 (2^-24 each), the result to y's type.
    room = 2.0**-22 * (want.abs() + (0 if residual is None else residual.double().abs()))
    if residual is not None:
        want = want + residual.double()
    assert ((y.double() - want).abs() <= O.half_step(y.dtype) * want.abs() * (1 + 2.0**-8) + room).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.25), ((8,), 0.5), ((3, 5, 43), 0.1), ((37, 129), 0.25),
                                     ((1000, 136), 0.9), ((2049, 1024), 0.1), ((9,), 1.0), ((64, 64), 1e-6)])
def test_dropout_matches_the_oracle(nv, shape, p, dtype):
    x, r = _rand(*shape, dtype=dtype, seed=1), _rand(*shape, dtype=dtype, seed=2)
    seed = 0x1234_5678_9ABC_DEF0 ^ x.numel()
    _check_dropout(nv.dropout(x, p, seed=seed), x, None, p, seed)
    _check_dropout(nv.dropout(x, p, seed=seed, residual=r), x, r, p, seed)
    assert torch.equal(nv.dropout(x, p, seed=seed), nv.dropout(x, p, seed=torch.tensor(seed, device="cuda")))


@pytest.mark.parametrize("seed", [0, 1, -1, 2**63 - 1, -2**63])
def test_every_seed_is_a_key(nv, seed):
    x = torch.ones(4096, device="cuda")
    assert torch.equal(nv.dropout(x, 0.5, seed=seed) > 0, O.kept((4096,), 0.5, seed, "cuda"))


def test_counter_passes_32_bits(nv):
    """A tensor of more than 2^32 elements: the groups' indexes past 2^29 reach the same draws, those at
    its very end included."""
    n = 2**32 + 13
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = nv.dropout(x, 0.5, seed=99)
    for at in (0, 2**31 - 8, 2**32 - 16, n - 21):
        at = at // 8 * 8
        m = min(64, n - at)
        ctr = torch.zeros(8, 4, dtype=torch.int64)
        ctr[:, 0] = torch.arange(8) + at // 8
        words = torch.from_numpy(O.philox4x32_10(ctr.numpy().astype("uint32"), (99, 0)).astype("int64"))
        draws = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:m]
        assert torch.equal((y[at:at + m] > 0).cpu(), draws >= 32768), at


def test_dropped_elements_hold_nothing(nv):
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep = O.kept((4096,), 0.5, 3, "cuda")
    y = nv.dropout(x, 0.5, seed=3)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    assert (nv.dropout(x, 1.0, seed=3) == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_misaligned(nv, dtype):
    base = _rand(130, 261, dtype=dtype, seed=5)
    for x in (base[:, 1:200], base.t(), base.reshape(-1)[3:1003], base[:1].expand(4, 261)):
        r = _rand(*x.shape, dtype=dtype, seed=6)
        _check_dropout(nv.dropout(x, 0.3, seed=8, residual=r), x, r, 0.3, 8)


def test_identity_cases(nv):
    x, r = _rand(5, 9), _rand(5, 9, seed=1)
    assert nv.dropout(x, 0.0) is x and nv.dropout(x, 0.7, training=False) is x
    assert torch.equal(nv.dropout(x, 0.7, training=False, residual=r), x + r)
    assert nv.dropout(x[:0], 0.5, seed=1).shape == (0, 9)
    # Zero-step edge: a probability below half of 2^-16 keeps everything, unscaled.
    assert torch.equal(nv.dropout(x, 1e-7, seed=4), x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(nv, dtype):
    x, r = _rand(33, 65, dtype=dtype, seed=1).requires_grad_(), _rand(33, 65, dtype=dtype, seed=2).requires_grad_()
    gy = _rand(33, 65, dtype=dtype, seed=3)
    y = nv.dropout(x, 0.4, seed=11, residual=r)
    gx, gr = torch.autograd.grad(y, (x, r), gy)
    assert torch.equal(gr, gy)
    _check_dropout(gx, gy, None, 0.4, 11)
    # Against differences: the map is linear, so f(x + d) - f(x) is exact up to fp32 rounding.
    if dtype == torch.float32:
        d = _rand(33, 65, seed=4)
        diff = nv.dropout((x + d).detach(), 0.4, seed=11).double() - nv.dropout(x.detach(), 0.4, seed=11).double()
        lhs, rhs = (diff * gy.double()).sum(), (gx.double() * d.double()).sum()
        bound = 2.0**-21 * ((x.abs() + d.abs()).double() * gy.double().abs()).sum()
        assert (lhs - rhs).abs() <= 2 * bound
    # Only the residual needs a gradient, and one through an expanded (stride 0) upstream gradient.
    (gr,) = torch.autograd.grad(nv.dropout(x.detach(), 0.4, seed=11, residual=r).sum(), r)
    assert (gr == 1).all()


def test_fresh_seeds_follow_the_generator(nv):
    x = torch.ones(4096, device="cuda")
    torch.manual_seed(7)
    a, b = nv.dropout(x, 0.5), nv.dropout(x, 0.5)
    torch.manual_seed(7)
    assert torch.equal(nv.dropout(x, 0.5), a) and not torch.equal(a, b)

    from torch.utils.checkpoint import checkpoint

    w = torch.ones(4096, device="cuda", requires_grad=True)
    y = checkpoint(lambda v: nv.dropout(v, 0.5) * v, w, use_reentrant=False)
    (g,) = torch.autograd.grad(y.sum(), w)
    assert torch.equal(g, 2 * y.detach())  # the recomputed mask is the first one (w = 1)


def test_seed_must_stay_until_backward(nv):
    x = _rand(64).requires_grad_()
    seed = torch.tensor(5, device="cuda")
    y = nv.dropout(x, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_unbiased(nv):
    """16-bit draws: the mean of 2^24 kept-and-scaled ones is 1 within six standard deviations."""
    n, p = 1 << 24, 0.3
    y = nv.dropout(torch.ones(n, device="cuda"), p, seed=42).double()
    q = O.threshold(p) / 65536
    assert abs(y.mean().item() - 1) <= 6 * (q / (1 - q) / n) ** 0.5


def test_stream_and_graph(nv):
    x = _rand(1000, 40, dtype=torch.bfloat16)
    seed = torch.tensor(1, device="cuda")
    want = {s: nv.dropout(x, 0.2, seed=s) for s in (1, 2)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = nv.dropout(x, 0.2, seed=seed)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = nv.dropout(x, 0.2, seed=seed)
    for s in (2, 1):
        seed.fill_(s)
        g.replay()
        assert torch.equal(out, want[s])


def test_fresh_seeds_in_a_graph(nv):
    """Without a seed every replay draws another mask, and its backward the same one again."""
    x = torch.ones(4096, device="cuda", requires_grad=True)
    gy = torch.ones(4096, device="cuda")
    torch.autograd.grad(nv.dropout(x, 0.5), x, gy)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = nv.dropout(x, 0.5)
        (gx,) = torch.autograd.grad(y, x, gy)
    seen = []
    for _ in range(3):
        g.replay()
        assert torch.equal(gx, y) and 0.4 < (y > 0).float().mean().item() < 0.6  # x = gy = 1
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_second_order_is_refused(nv):
    x = _rand(64).requires_grad_()
    (g,) = torch.autograd.grad(nv.dropout(x, 0.5, seed=1).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


# ------------------------------------------------------------------------------------------------
# epilogue_backward
# ------------------------------------------------------------------------------------------------


def _check_backward(nv, gy, z, act, p, seed, out, gs, sums):
    g = O.drop(gy.double(), p, seed)
    d = torch.ones_like(g) if z is None else O.derivative(z.double(), act)
    want = g * d
    # The derivative in fp32: its terms are at most 1.2 in size (2 |z| for relu2), each a few roundings and
    # one exponential or erf of 2 ulp, whose argument is off by 2^-22 of itself; s (1 - s) |u| <= 0.23 and
    # z u' <= 5 where that factor counts: under 2^-18 in all, relative to max(1, 2 |z|).
    room = 2.0**-18 * g.abs() * (1 if z is None else (2 * z.double().abs()).clamp_min(1))
    assert ((out.double() - want).abs() <= O.half_step(out.dtype) * want.abs() * (1 + 2.0**-8) + room).all()
    assert torch.equal(gs, nv.global_scale_of(out)) or (torch.isnan(gs) and torch.isnan(nv.global_scale_of(out)))
    if sums is not None:
        rows = gy.shape[0]
        bound = rows * 2.0**-24 * want.abs().sum(0) + room.sum(0)
        assert ((sums.double() - want.sum(0)).abs() <= bound + 1e-38).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 1), (5, 13), (16, 256), (17, 264), (640, 1152), (1001, 40),
                                       (4096, 8), (300, 4100)])
@pytest.mark.parametrize("act,p", [("gelu", 0.0), ("silu", 0.1), (None, 0.25), ("relu2", 0.5), ("gelu_tanh", 0.0),
                                   ("relu", 0.9)])
def test_backward_matches_the_oracle(nv, rows, cols, dtype, act, p):
    gy, z = _rand(rows, cols, dtype=dtype, seed=rows), _rand(rows, cols, dtype=dtype, seed=cols, std=2.0)
    seed = rows * 1000 + cols
    out, gs, sums = nv.epilogue_backward(gy, z, activation=act, dropout_p=p, seed=seed, bias_grad=True)
    _check_backward(nv, gy, None if act is None else z, act, p, seed, out, gs, sums)
    again = nv.epilogue_backward(gy, z, activation=act, dropout_p=p, seed=seed, bias_grad=True)
    assert all(torch.equal(a, b) for a, b in zip((out, gs, sums), again))
    assert nv.epilogue_backward(gy, z, activation=act, dropout_p=p, seed=seed)[2] is None


@pytest.mark.parametrize("act", O.ACTIVATIONS[1:])
def test_far_preactivations(nv, act):
    """Huge, tiny and zero pre-activations: finite derivatives stay finite."""
    mag = torch.tensor([0.0, 1e-38, 1e-20, 1e-3, 5.0, 30.0, 88.0, 1e4, 1e13, 1e19, 1e30], device="cuda")
    z = torch.cat([mag, -mag]).float().view(1, -1)
    gy = torch.ones_like(z)
    out, gs, _ = nv.epilogue_backward(gy, z, activation=act)
    assert torch.isfinite(out).all()
    _check_backward(nv, gy, z, act, 0.0, 0, out, gs, None)


def test_backward_is_the_mask_of_dropout(nv):
    gy = _rand(96, 200, dtype=torch.bfloat16)
    out, _, _ = nv.epilogue_backward(gy, dropout_p=0.3, seed=17)
    assert torch.equal(out, nv.dropout(gy, 0.3, seed=17))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_backward_strides(nv, dtype):
    base, zb = _rand(200, 528, dtype=dtype, seed=1), _rand(200, 528, dtype=dtype, seed=2)
    for gy, z in ((base[:, 16:272], zb[:, 8:264]), (base[:, 3:260], zb[:, 5:262]), (base.t(), zb.t()),
                  (base[:1].expand(200, 528), zb)):
        out, gs, sums = nv.epilogue_backward(gy, z, activation="silu", dropout_p=0.2, seed=3, bias_grad=True)
        _check_backward(nv, gy, z, "silu", 0.2, 3, out, gs, sums)
    buf = torch.full((200, 300), 7.0, dtype=dtype, device="cuda")
    out, _, _ = nv.epilogue_backward(base[:, :256], zb[:, :256], activation="silu", out=buf[:, 8:264])
    want, _, _ = nv.epilogue_backward(base[:, :256], zb[:, :256], activation="silu")
    assert torch.equal(out, want) and torch.equal(buf[:, 8:264], want)
    assert (buf[:, :8] == 7).all() and (buf[:, 264:] == 7).all()
    g = base[:, :256].contiguous()
    out, _, _ = nv.epilogue_backward(g, zb[:, :256], activation="silu", out=g)  # in place
    assert out is g and torch.equal(g, want)


def test_backward_nan_scale(nv):
    gy = _rand(64, 64)
    gy[3, 5] = float("nan")
    _, gs, _ = nv.epilogue_backward(gy, _rand(64, 64), activation="gelu")
    assert torch.isnan(gs)
    _, gs, _ = nv.epilogue_backward(torch.zeros_like(gy))
    assert gs.item() == pytest.approx(1e-12)


def test_backward_in_a_graph(nv):
    gy, z = _rand(512, 512, dtype=torch.bfloat16), _rand(512, 512, dtype=torch.bfloat16, seed=1)
    nv.epilogue_backward(gy, z, activation="gelu", bias_grad=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = nv.epilogue_backward(gy, z, activation="gelu", dropout_p=0.1, seed=5, bias_grad=True)
    gy.mul_(2)
    g.replay()
    want = nv.epilogue_backward(gy, z, activation="gelu", dropout_p=0.1, seed=5, bias_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(nv):
    x = _rand(8, 16)
    with pytest.raises(ValueError, match="unsupported dtype"):
        nv.dropout(x.half(), 0.5)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            nv.dropout(x, p)
    with pytest.raises(ValueError, match="residual"):
        nv.dropout(x, 0.5, residual=x[:4])
    with pytest.raises(ValueError, match="residual"):
        nv.dropout(x, 0.5, residual=x.bfloat16())
    with pytest.raises(ValueError, match="seed"):
        nv.dropout(x, 0.5, seed=torch.tensor(1))
    with pytest.raises(ValueError, match="seed"):
        nv.dropout(x, 0.5, seed=torch.tensor(1.0, device="cuda"))
    with pytest.raises(ValueError, match="activation"):
        nv.epilogue_backward(x, x, activation="tanh")
    with pytest.raises(ValueError, match="pre-activations"):
        nv.epilogue_backward(x, activation="silu")
    with pytest.raises(ValueError, match="preact"):
        nv.epilogue_backward(x, x[:, :8], activation="silu")
    with pytest.raises(ValueError, match="seed"):
        nv.epilogue_backward(x, dropout_p=0.5)
    with pytest.raises(ValueError, match="non-empty"):
        nv.epilogue_backward(x[:0])
    buf = torch.zeros(9, 16, device="cuda")
    with pytest.raises(ValueError, match="overlaps the gradient"):
        nv.epilogue_backward(buf[:8], out=buf[1:])
    with pytest.raises(ValueError, match="overlaps the pre-activations"):
        nv.epilogue_backward(x, buf[1:], activation="silu", out=buf[:8])
    with pytest.raises(ValueError, match="out must have contiguous rows"):
        nv.epilogue_backward(x, out=torch.empty(16, 8, device="cuda").t())
