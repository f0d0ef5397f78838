"""Expert routing (``nvfp4.route``) and the moves of token rows (``token_dispatch``,
``token_combine``) against 64-bit oracles: picks, counts and rows exactly, weights, loss and
gradients to their roundings; masked, unrouted and NaN tokens; ties; odd sizes and strides."""

import numpy as np
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


def _check_route(nv, logits, k, bias=None, valid=None, renormalize=True, backward=True):
    x = logits.detach().clone().requires_grad_(backward)
    if logits.stride() != x.stride():
        x = logits.detach().requires_grad_(backward)
    r = nv.route(x, k, expert_bias=bias, valid=valid, renormalize=renormalize)
    t, e = logits.shape
    w, ex, counts, offsets, rows, loss, prob = O.route(logits, k, bias, valid, renormalize)
    np.testing.assert_array_equal(r.experts.cpu().numpy(), ex)
    np.testing.assert_array_equal(r.counts.cpu().numpy(), counts)
    np.testing.assert_array_equal(r.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(r.rows.cpu().numpy(), rows)
    assert r.num_rows % 128 == 0 and r.num_rows >= offsets[-1]
    # fp32 softmax: the exponent's argument x - max is exact to 2^-24 of at most ~20, the exponential 2 ulp, the
    # sum of e terms and the quotient a few more roundings: under (20 + 16 + e) 2^-24 relative.
    rel = (36 + e) * 2.0**-24
    got = r.weights.detach().double().cpu().numpy()
    assert (np.abs(got - w) <= rel * w + 1e-37).all()
    # The loss adds t probabilities of each expert in fp32.
    assert abs(r.balance_loss.item() - loss) <= (rel + t * 2.0**-24) * loss
    if not backward:
        return r
    gw = _rand(t, k, seed=t + k)
    gl = 0.7
    (g,) = torch.autograd.grad((r.weights, r.balance_loss), x, (gw, torch.tensor(gl, device="cuda")))
    gwn = gw.double().cpu().numpy()
    want = O.route_gradient(w, ex, counts, prob, gwn, gl, renormalize)
    n = max(1, int((ex[:, 0] >= 0).sum()))
    c = gl * e * counts.max() / max(1, counts.sum()) / n
    # Each gradient is a sum of products w g and p c: their relative errors are the weights', twice.
    room = 4 * rel * ((np.abs(gwn) * (ex >= 0)).sum(1, keepdims=True) + 2 * c)
    got = g.double().cpu().numpy()
    assert (np.abs(got - want) <= O.half_step(x.dtype) * np.abs(want) * 1.01 + room + 1e-37).all()
    assert (got[ex[:, 0] < 0] == 0).all()
    return r


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 2, 2), (33, 3, 1), (64, 8, 8), (257, 16, 4), (130, 17, 3), (1000, 32, 5),
          (300, 33, 6), (301, 64, 8), (99, 100, 32), (515, 128, 7), (77, 160, 6), (200, 256, 8), (3000, 5, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,e,k", SHAPES)
def test_route_matches_the_oracle(nv, t, e, k, dtype):
    _check_route(nv, _rand(t, e, dtype=dtype, seed=t * e + k, std=2.0), k)


@pytest.mark.parametrize("t,e,k", [(1, 4, 2), (257, 8, 2), (640, 60, 6), (130, 256, 4)])
@pytest.mark.parametrize("renormalize", [False, True])
def test_bias_and_padding(nv, t, e, k, renormalize):
    logits = _rand(t, e, seed=3)
    valid = torch.rand(t, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.7
    logits[~valid] = float("nan")
    _check_route(nv, logits, k, _rand(e, seed=4), valid, renormalize)


@pytest.mark.parametrize("renormalize", [False, True])
def test_masked_experts(nv, renormalize):
    """-inf logits: fewer picks than k, and tokens that no expert is left for."""
    logits = _rand(200, 12, seed=5)
    gone = torch.rand(200, 12, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) < 0.75
    gone[::7] = True
    logits[gone] = float("-inf")
    r = _check_route(nv, logits, 4, renormalize=renormalize)
    assert (r.experts[::7] == -1).all() and (r.weights[::7] == 0).all()
    none = nv.route(torch.full((9, 4), float("-inf"), device="cuda"), 2)
    assert none.balance_loss.item() == 0 and (none.counts == 0).all() and (none.offsets == 0).all()
    bias = torch.zeros(12, device="cuda")
    bias[3] = float("-inf")  # an expert switched off by its bias
    r = _check_route(nv, _rand(100, 12, seed=6), 5, bias, renormalize=renormalize)
    assert r.counts[3] == 0


def test_ties_go_to_the_lower_expert(nv):
    logits = torch.zeros(50, 40, device="cuda")
    logits[:, 1::2] = -0.0
    r = _check_route(nv, logits, 6)
    assert (r.experts == torch.arange(6, device="cuda", dtype=torch.int32)).all()
    coarse = _rand(400, 24, seed=9).mul(2).round().bfloat16()
    _check_route(nv, coarse, 5)


def test_nan_and_infinite_logits(nv):
    """A NaN or +inf logit of a routed token: picked first, NaN weights for that token alone."""
    logits = _rand(64, 40, seed=8)
    logits[5, 33] = float("nan")
    logits[6, 2] = float("inf")
    r = nv.route(logits, 3)
    assert r.experts[5, 0] == 33 and r.experts[6, 0] == 2
    assert torch.isnan(r.weights[5]).all() and torch.isnan(r.weights[6, 0])
    rest = [i for i in range(64) if i not in (5, 6)]
    assert torch.isfinite(r.weights[rest]).all()
    assert torch.equal(r.weights[rest], nv.route(logits[rest], 3).weights)
    p = nv.route(logits, 3, renormalize=False).weights
    assert torch.isnan(p[5]).all() and torch.isnan(p[6]).all()


@pytest.mark.parametrize("scale", [30.0, 80.0])
def test_far_logits(nv, scale):
    """Picks far below the largest logit (a selection bias): renormalized weights do not underflow."""
    logits = _rand(64, 16, seed=1)
    logits[:, 0] += scale
    bias = torch.zeros(16, device="cuda")
    bias[0] = -1000.0
    r = _check_route(nv, logits, 2, bias, backward=False)
    assert torch.allclose(r.weights.sum(1), torch.ones(64, device="cuda"), atol=2.0**-20)


def test_many_tokens(nv):
    """More chunks than blocks of the plan; a group per expert past one tile."""
    logits = _rand(40000, 16, seed=2)
    r = nv.route(logits, 8)
    ex = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(r.experts.long(), ex)
    flat = ex.reshape(-1)
    assert torch.equal(r.counts, torch.bincount(flat, minlength=16))
    order = torch.sort(flat, stable=True).indices
    rank = torch.empty_like(flat)
    rank[order] = torch.arange(flat.numel(), device="cuda")
    start = torch.cumsum(r.counts, 0) - r.counts
    assert torch.equal(r.rows.long().reshape(-1), r.offsets[flat] + rank - start[flat])
    again = nv.route(logits, 8)
    assert all(torch.equal(a, b) for a, b in zip(r[:6], again[:6]))


def test_no_tokens(nv):
    r = nv.route(torch.empty(0, 6, device="cuda"), 2)
    assert r.num_rows == 0 and (r.counts == 0).all() and r.balance_loss == 0 and r.rows.shape == (0, 2)
    assert nv.token_dispatch(torch.empty(0, 8, device="cuda"), r).shape == (0, 8)
    assert nv.token_combine(torch.empty(0, 8, device="cuda"), r).shape == (0, 8)


def test_strided_logits(nv):
    base = _rand(130, 80, seed=1)
    _check_route(nv, base[:, 5:18], 3)
    _check_route(nv, base.t()[:, :20], 2)
    _check_route(nv, base[:1].expand(50, 80), 4)


def test_only_one_gradient(nv):
    logits = _rand(100, 9, seed=1).requires_grad_()
    r = nv.route(logits, 2)
    gw = _rand(100, 2, seed=2)
    (a,) = torch.autograd.grad(r.weights, logits, gw, retain_graph=True)
    (b,) = torch.autograd.grad(r.balance_loss, logits, retain_graph=True)
    (c,) = torch.autograd.grad((r.weights, r.balance_loss), logits, (gw, torch.ones((), device="cuda")))
    assert torch.allclose(a + b, c, atol=2.0**-20)
    assert a.abs().max() > 0 and b.abs().max() > 0


def test_counts_may_be_reduced_in_place(nv):
    """A data-parallel job adds up the counts of its ranks before the backward pass."""
    logits = _rand(100, 9, seed=1).requires_grad_()
    want = torch.autograd.grad(nv.route(logits, 2).balance_loss, logits)[0]
    r = nv.route(logits, 2)
    r.counts.mul_(4)
    r.rows.add_(1)
    assert torch.equal(torch.autograd.grad(r.balance_loss, logits)[0], want)


def test_route_gradient_against_differences(nv):
    """Central differences of the fp32 forward, with the selection unchanged by the step."""
    logits = _rand(16, 6, seed=4).requires_grad_()
    gw = _rand(16, 3, seed=5)
    for renorm in (True, False):
        r = nv.route(logits, 3, renormalize=renorm)
        (g,) = torch.autograd.grad((r.weights, r.balance_loss), logits, (gw, torch.tensor(2.0, device="cuda")))
        h = 2.0**-9

        def f(x):
            q = nv.route(x, 3, renormalize=renorm)
            assert torch.equal(q.experts, r.experts)
            return (q.weights.double() * gw.double()).sum().item() + 2.0 * q.balance_loss.double().item()

        for i, j in ((0, 0), (3, 5), (9, 2), (15, 1)):
            up, dn = logits.detach().clone(), logits.detach().clone()
            up[i, j] += h
            dn[i, j] -= h
            diff = (f(up) - f(dn)) / (2 * h)
            # truncation h^2 |f'''| / 6 with |f'''| <= 6 |g| of the token; fp32 noise 2^-22 of 16 x 3 terms over 2h
            room = h * h * 6 * gw[i].abs().sum().item() + 48 * 2.0**-22 * gw.abs().max().item() / (2 * h)
            assert abs(diff - g[i, j].item()) <= room


# ------------------------------------------------------------------------------------------------
# Rows
# ------------------------------------------------------------------------------------------------


def _rows_case(nv, t, e, k, d, dtype, mask=False, seed=0):
    logits = _rand(t, e, seed=seed + 1)
    valid = None
    if mask:
        valid = torch.rand(t, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) < 0.6
        logits[:, 0] = float("-inf")
    r = nv.route(logits, k, valid=valid)
    return (r, _rand(t, d, dtype=dtype, seed=seed + 2), _rand(r.num_rows, d, dtype=dtype, seed=seed + 3),
            _rand(t, d, dtype=dtype, seed=seed + 4))


def _check_rows(nv, r, x, y, res, gxs, gy):
    t, k = r.rows.shape
    at = r.rows.long()
    used = at >= 0
    x, y, w = x.detach().requires_grad_(), y.detach().requires_grad_(), r.weights.detach().requires_grad_()
    r = r._replace(weights=w)
    xs = nv.token_dispatch(x, r)
    want = torch.zeros_like(y.detach())
    tok = torch.arange(t, device="cuda").view(-1, 1).expand(t, k)
    want[at[used]] = x.detach()[tok[used]]
    assert torch.equal(xs.detach(), want)
    out = nv.token_combine(y, r, residual=res)
    yd, wd = y.detach().double(), w.detach().double()
    terms = torch.where(used.unsqueeze(-1), yd[at.clamp_min(0)], 0.0) * wd.unsqueeze(-1)
    ref, mag = terms.sum(1), terms.abs().sum(1)
    if res is not None:
        ref, mag = ref + res.double(), mag + res.double().abs()
    hs = O.half_step(x.dtype)
    # k fused multiply-adds and the residual's sum in fp32, then one rounding.
    assert ((out.detach().double() - ref).abs() <= hs * ref.abs() * 1.01 + (k + 2) * 2.0**-24 * mag).all()
    gx, gr, gw = torch.autograd.grad((xs, out), (x, y, w), (gxs, gy))
    parts = torch.where(used.unsqueeze(-1), gxs.double()[at.clamp_min(0)], 0.0)
    assert ((gx.double() - parts.sum(1)).abs() <= hs * parts.sum(1).abs() * 1.01
            + (k + 1) * 2.0**-24 * parts.abs().sum(1)).all()
    want = torch.zeros_like(y.detach())
    want[at[used]] = (gy.float()[tok[used]] * w.detach()[used].unsqueeze(-1)).to(x.dtype)
    assert torch.equal(gr, want)  # one fp32 product, rounded
    prod = torch.where(used.unsqueeze(-1), yd[at.clamp_min(0)], 0.0) * gy.double().unsqueeze(1)
    assert ((gw.double() - prod.sum(-1)).abs() <= x.shape[1] * 2.0**-24 * prod.abs().sum(-1)).all()
    assert (gw[~used] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,e,k,d", [(1, 4, 2, 8), (33, 16, 4, 1408), (200, 8, 2, 2048), (130, 3, 1, 1),
                                     (77, 60, 6, 129), (500, 5, 5, 264), (64, 256, 8, 128), (40, 12, 12, 2056)])
def test_rows_match_the_oracle(nv, t, e, k, d, dtype):
    for mask in (False, True):
        r, x, y, res = _rows_case(nv, t, e, k, d, dtype, mask, seed=t + d)
        gxs, gy = _rand(r.num_rows, d, dtype=dtype, seed=1), _rand(t, d, dtype=dtype, seed=2)
        _check_rows(nv, r, x, y, res, gxs, gy)
        _check_rows(nv, r, x, y, None, gxs, gy)


def test_unused_rows_are_not_read(nv):
    r, x, y, _ = _rows_case(nv, 50, 6, 2, 72, torch.float32, True)
    y = torch.full_like(y, float("nan"))
    used = r.rows[r.rows >= 0].long()
    y[used] = 1.0
    w = r.weights.detach().requires_grad_()
    y.requires_grad_()
    out = nv.token_combine(y, r._replace(weights=w))
    assert torch.isfinite(out).all()
    gy, gw = torch.autograd.grad(out.sum(), (y, w))
    assert torch.isfinite(gy).all() and torch.isfinite(gw).all()
    assert torch.isfinite(nv.token_dispatch(x, r)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_strides(nv, dtype):
    r, _, _, _ = _rows_case(nv, 90, 4, 2, 8, dtype)
    bx, by = _rand(90, 300, dtype=dtype, seed=1), _rand(r.num_rows, 300, dtype=dtype, seed=2)
    br = _rand(90, 300, dtype=dtype, seed=3)
    for lo, hi in ((0, 128), (8, 136), (3, 130), (1, 2)):
        _check_rows(nv, r, bx[:, lo:hi], by[:, lo:hi], br[:, lo:hi], by[:, lo:hi], bx[:, lo:hi])
    _check_rows(nv, r, bx[:1].expand(90, 300), by, br, by[:1].expand(r.num_rows, 300), bx[:1].expand(90, 300))


def test_rows_outside_the_layout_are_skipped(nv):
    """A plan whose rows, counts or offsets lie outside the tensors touches nothing outside them."""
    r, x, y, _ = _rows_case(nv, 40, 4, 2, 64, torch.float32)
    bad = r.rows.clone()
    bad[0, 0], bad[1, 1], bad[2, 0] = r.num_rows, 2**31 - 1, -5
    q = r._replace(rows=bad, offsets=r.offsets - 7, counts=r.counts + 1000)
    out = nv.token_combine(y, q)
    want = (torch.where((bad >= 0) & (bad < r.num_rows), r.weights, 0.0).unsqueeze(-1)
            * y[bad.long().clamp(0, r.num_rows - 1)]).sum(1)
    assert torch.allclose(out, want, atol=1e-5)
    nv.token_dispatch(x, q)
    torch.cuda.synchronize()


def test_stream_and_graph(nv):
    logits = _rand(300, 10, seed=1)
    x = _rand(300, 64, dtype=torch.bfloat16, seed=2)

    def step():
        r = nv.route(logits, 3)
        return nv.token_combine(nv.token_dispatch(x, r) * 2, r), r.balance_loss, r.rows

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    logits.copy_(_rand(300, 10, seed=7))
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals(nv):
    x = _rand(10, 8)
    for k in (0, 9):
        with pytest.raises(ValueError, match="needs 1 <= experts"):
            nv.route(x, k)
    with pytest.raises(ValueError, match="needs 1 <= experts"):
        nv.route(_rand(4, 257), 2)
    with pytest.raises(ValueError, match="needs 1 <= experts"):
        nv.route(_rand(4, 64), 33)
    with pytest.raises(ValueError, match="unsupported dtype"):
        nv.route(x.half(), 2)
    with pytest.raises(ValueError, match=r"\(tokens, experts\)"):
        nv.route(x[0], 2)
    with pytest.raises(ValueError, match="valid"):
        nv.route(x, 2, valid=torch.ones(9, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="valid"):
        nv.route(x, 2, valid=torch.ones(10, device="cuda"))
    with pytest.raises(ValueError, match="expert_bias"):
        nv.route(x, 2, expert_bias=torch.ones(7, device="cuda"))
    r = nv.route(x, 2)
    with pytest.raises(ValueError, match="expected"):
        nv.token_dispatch(_rand(9, 16), r)
    with pytest.raises(ValueError, match="expected"):
        nv.token_combine(_rand(9, 16), r)
    with pytest.raises(ValueError, match="residual"):
        nv.token_combine(_rand(r.num_rows, 16), r, residual=_rand(10, 8))
    with pytest.raises(ValueError, match="weights"):
        nv.token_combine(_rand(r.num_rows, 16), r._replace(weights=r.weights.bfloat16()))
    with pytest.raises(ValueError, match="int32 rows"):
        nv.token_dispatch(_rand(10, 16), r._replace(rows=r.rows.long()))
    with pytest.raises(ValueError, match="the routing is on"):
        nv.token_dispatch(_rand(10, 16), r._replace(rows=r.rows.cpu()))
