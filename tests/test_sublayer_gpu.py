"""The operators together, as a block uses them: an ungated feed-forward whose activation, dropout
and residual run in its GEMMs, then a mixture-of-experts sublayer with its balance loss
(``FP4BatchedExperts.forward_routed``), forward, backward and in a captured graph."""

import pytest
import torch

from tests import _epilogue_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nv():
    import radiance_b200.nvfp4 as nv

    assert nv.nvfp4_supported()
    return nv


def _rand(*shape, dtype=torch.bfloat16, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _experts(nv, e=6, d=256, f=384):
    from radiance_b200.nvfp4.grouped import FP4BatchedExperts

    torch.manual_seed(3)
    ex = FP4BatchedExperts(e, d, f, device="cuda")
    with torch.no_grad():
        ex.gate_up_b.normal_(std=0.5)
        ex.down_b.normal_(std=0.5)
    ex.refresh_fp4_cache()
    return ex


def test_routed_experts_match_their_parts(nv):
    """forward_routed against the experts run one at a time on their own rows, with the biases, and every
    gradient against the same composition's (the rows' zero padding changes no group's scale)."""
    ex = _experts(nv)
    x = _rand(2, 150, 256, seed=1).requires_grad_()
    logits = _rand(2, 150, 6, dtype=torch.float32, seed=2).requires_grad_()
    valid = torch.ones(2, 150, dtype=torch.bool, device="cuda")
    valid[1, 100:] = False
    y, r = ex.forward_routed(x, logits, 2, valid=valid, residual=x)
    assert y.shape == x.shape
    xs = nv.token_dispatch(x.detach().view(-1, 256), r)
    parts = torch.zeros(r.num_rows, 256, dtype=torch.bfloat16, device="cuda")
    offs, cnt = r.offsets.tolist(), r.counts.tolist()
    for g in range(6):
        lo, hi = offs[g], offs[g + 1]
        if lo == hi:
            continue
        only = torch.zeros(7, dtype=torch.int64, device="cuda")
        only[g + 1:] = hi - lo
        h = ex.gate_up(xs[lo:hi], only) + ex.gate_up_b[g].to(torch.bfloat16)
        h[cnt[g]:] = 0
        z = ex.down(nv.swiglu(h, "split"), only) + ex.down_b[g].to(torch.bfloat16)
        parts[lo:lo + cnt[g]] = z[:cnt[g]].detach()
    want = nv.token_combine(parts, r, residual=x.detach().view(-1, 256)).view(x.shape)
    assert torch.equal(y.detach(), want)
    assert torch.equal(y[1, 100:], x[1, 100:])  # padding tokens keep their residual
    # Gradients: finite everywhere, and exactly the upstream gradient for padding tokens.
    gy = _rand(2, 150, 256, seed=5, std=1e-2)
    (y.float() * gy.float()).sum().add(r.balance_loss * 0.01).backward()
    for name, p in ex.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    assert torch.isfinite(x.grad).all() and torch.isfinite(logits.grad).all()
    assert torch.equal(x.grad[1, 100:], gy[1, 100:]) and (logits.grad[1, 100:] == 0).all()
    # The down bias gradient is each expert's sum of w * dy over its pairs.
    dy, at = gy.view(-1, 256).double(), r.experts.view(-1).long()
    w = r.weights.detach().double().view(-1, 1)
    terms = (w * dy.repeat_interleave(2, 0))[at >= 0]
    exact = torch.zeros(6, 256, dtype=torch.float64, device="cuda").index_add_(0, at[at >= 0], terms)
    mag = torch.zeros(6, 256, dtype=torch.float64, device="cuda").index_add_(0, at[at >= 0], terms.abs())
    # bf16 rows (two roundings of each term: w dy, and the bias's cast), one bf16 rounding of the sum
    assert ((ex.down_b.grad.squeeze(1).double() - exact).abs() <= 2.0**-8 * exact.abs() + 2.0**-7 * mag).all()


def test_balance_loss_gradient_evens_the_load(nv):
    """The loss's gradient is the oracle's through the whole layer's graph (its only path is the logits)."""
    ex = _experts(nv)
    x, logits = _rand(300, 256, seed=1), _rand(300, 6, dtype=torch.float32, seed=2).requires_grad_()
    _, r = ex.forward_routed(x, logits, 2)
    (g,) = torch.autograd.grad(r.balance_loss, logits)
    w, e, counts, _, _, loss, prob = O.route(logits, 2)
    want = torch.from_numpy(O.route_gradient(w, e, counts, prob, w * 0, 1.0)).cuda()
    assert (g.double() - want).abs().max() <= 64 * 2.0**-24 * want.abs().max()
    assert abs(r.balance_loss.item() - loss) <= 400 * 2.0**-24 * loss


def _block(nv):
    torch.manual_seed(0)
    up, down = nv.FP4Linear(256, 512).cuda(), nv.FP4Linear(512, 256).cuda()
    for m in (up, down):
        m.refresh_fp4_cache()
    router = torch.nn.Linear(256, 6, bias=False).cuda()
    ex = _experts(nv)

    def step(x, seed):
        h = up(x, activation="gelu")
        x = down(h, dropout_p=0.1, dropout_seed=seed, residual=x)
        y, r = ex.forward_routed(x, router(x.float()), 2, residual=x)
        return nv.dropout(y, 0.1, seed=seed, residual=x), r

    return step, [p for m in (up, down, router, ex) for p in m.parameters()]


def test_block_trains(nv):
    step, params = _block(nv)
    x = _rand(256, 256, seed=7).requires_grad_()
    seed = torch.tensor(11, device="cuda")
    y, r = step(x, seed)
    grads = torch.autograd.grad((y.float().square().mean() + 0.01 * r.balance_loss), [x, *params])
    again_y, again_r = step(x, seed)
    again = torch.autograd.grad((again_y.float().square().mean() + 0.01 * again_r.balance_loss), [x, *params])
    assert torch.equal(y, again_y) and all(torch.isfinite(g).all() for g in grads)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)


def test_block_in_a_graph(nv):
    """Forward and backward captured once and replayed on new inputs and a new dropout seed."""
    step, params = _block(nv)
    static, seed = _rand(256, 256, seed=7).requires_grad_(), torch.tensor(11, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up: workspaces, occupancy queries, library handles
        y, r = step(static, seed)
        torch.autograd.grad(y.float().square().mean() + 0.01 * r.balance_loss, [static, *params])
        del y, r
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, r = step(static, seed)
        grads = torch.autograd.grad(y.float().square().mean() + 0.01 * r.balance_loss, [static, *params])
    with torch.no_grad():
        static.copy_(_rand(256, 256, seed=8))
    seed.fill_(12)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (y.detach(), r.balance_loss.detach(), *grads)]
    x = static.detach().clone().requires_grad_()
    want_y, want_r = step(x, seed)
    want = torch.autograd.grad(want_y.float().square().mean() + 0.01 * want_r.balance_loss, [x, *params])
    assert torch.equal(got[0], want_y) and torch.equal(got[1], want_r.balance_loss)
    for a, b in zip(got[2:], want):
        assert torch.equal(a, b)


def test_a_batch_of_padding(nv):
    """No token takes part: the output is the residual, every gradient of the experts and the logits is zero."""
    ex = _experts(nv)
    x = _rand(130, 256, seed=1).requires_grad_()
    logits = torch.full((130, 6), float("nan"), device="cuda", requires_grad=True)
    y, r = ex.forward_routed(x, logits, 2, valid=torch.zeros(130, dtype=torch.bool, device="cuda"), residual=x)
    assert torch.equal(y, x) and r.balance_loss == 0 and (r.counts == 0).all()
    gy = _rand(130, 256, seed=2)
    ((y * gy).float().sum() + r.balance_loss).backward()
    assert torch.equal(x.grad, gy) and (logits.grad == 0).all()
    for name, p in ex.named_parameters():
        assert (p.grad == 0).all(), name


def test_routed_experts_without_tokens(nv):
    ex = _experts(nv)
    y, r = ex.forward_routed(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16),
                             torch.empty(0, 6, device="cuda"), 2)
    assert y.shape == (0, 256) and (r.counts == 0).all()
    with pytest.raises(ValueError, match="forward_routed"):
        ex.forward_routed(_rand(4, 256), _rand(4, 5), 2)
