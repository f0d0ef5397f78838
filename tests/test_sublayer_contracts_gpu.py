"""What the sublayer operators promise beside their formulas: counts that may be changed in place, derivatives
that are refused and never dropped, plans that reach past the tensors, types under autocast, accuracy far out."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nv():
    import radiance_b200.nvfp4 as nv

    assert nv.nvfp4_supported()
    return nv


def _rand(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _poison(*shape, dtype=torch.bfloat16):
    """Leaves NaN in the memory that the next allocations of this size get."""
    blocks = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(6)]
    del blocks


# ------------------------------------------------------------------------------------------------
# Counts changed in place between the passes
# ------------------------------------------------------------------------------------------------

CHANGES = {
    "sum": lambda c: c.mul_(4),
    "untracked sum": lambda c: c.data.mul_(4),  # as a collective writes: autograd's version counter stays
    "untracked mean": lambda c: c.data.div_(3, rounding_mode="floor"),
    "untracked zero": lambda c: c.data.zero_(),
}


@pytest.mark.parametrize("change", list(CHANGES))
def test_moves_keep_their_counts(nv, change):
    """Dispatch, combine and both backwards after an all-reduce of the counts."""
    x, res = _rand(300, 96, seed=1), _rand(300, 96, seed=3)
    gy = _rand(300, 96, seed=4)

    def run(first, second):
        logits, xs_in = _rand(300, 6, seed=2).requires_grad_(), x.clone().requires_grad_()
        r = nv.route(logits, 2)
        first(r.counts)
        _poison(r.num_rows, 96, dtype=torch.float32)
        xs = nv.token_dispatch(xs_in, r)
        ys = xs * 2
        y = nv.token_combine(ys, r, residual=res)
        second(r.counts)
        _poison(r.num_rows, 96, dtype=torch.float32)
        return xs.detach().clone(), y.detach(), *torch.autograd.grad(y, (xs, ys, xs_in, logits), gy)

    want = run(lambda c: None, lambda c: None)
    for at in ((CHANGES[change], lambda c: None), (lambda c: None, CHANGES[change])):
        for a, b in zip(run(*at), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("change", list(CHANGES))
def test_routed_experts_keep_their_counts(nv, change):
    """A job that reduces the returned counts before the backward pass gets the gradients of one that does not."""
    from radiance_b200.nvfp4.grouped import FP4BatchedExperts

    torch.manual_seed(3)
    ex = FP4BatchedExperts(6, 256, 384, device="cuda")
    ex.refresh_fp4_cache()

    def run(f):
        x, logits = _rand(300, 256, dtype=torch.bfloat16, seed=1).requires_grad_(), _rand(300, 6, seed=2).requires_grad_()
        y, r = ex.forward_routed(x, logits, 2, residual=x)
        f(r.counts)
        _poison(r.num_rows, 256)
        loss = (y.float() * _rand(300, 256, seed=5)).sum() + r.balance_loss
        return torch.autograd.grad(loss, [x, logits, *ex.parameters()])

    for a, b in zip(run(CHANGES[change]), run(lambda c: None)):
        assert torch.isfinite(a).all() and torch.equal(a, b)


# ------------------------------------------------------------------------------------------------
# Second derivatives
# ------------------------------------------------------------------------------------------------


def _linear(nv, n=256, k=256, **recipe):
    torch.manual_seed(1)
    layer = nv.FP4Linear(k, n, recipe=nv.FP4Recipe(**recipe)).cuda()
    layer.refresh_fp4_cache()
    return layer


@pytest.mark.parametrize("recipe", [dict(), dict(grad_gemms=False)])
@pytest.mark.parametrize("act,p", [("gelu", 0.0), (None, 0.0), (None, 0.2), ("silu", 0.1)])
def test_linear_second_order_is_refused(nv, act, p, recipe):
    """With residual=x the gradient of x stays differentiable through the residual's part: differentiating it must
    not silently leave out the linear's."""
    layer = _linear(nv, **recipe)
    x = _rand(256, 256, dtype=torch.bfloat16).requires_grad_()
    y = layer(x, activation=act, dropout_p=p, dropout_seed=3, residual=x)
    (g,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().square().sum().backward()


def _twice(loss, x):
    """Differentiates a gradient again beside another term that is differentiable twice."""
    (g,) = torch.autograd.grad(loss + x.float().pow(3).sum(), x, create_graph=True)
    g.float().square().sum().backward()


def test_second_order_under_a_constant_upstream(nv):
    """Gradients that depend on the inputs are refused even where the upstream gradient is a constant."""
    layer, x = _linear(nv), _rand(256, 256, dtype=torch.bfloat16).requires_grad_()
    for kw in (dict(activation="gelu"), dict(residual=x), dict(dropout_p=0.1, dropout_seed=1)):
        with pytest.raises(RuntimeError, match="once_differentiable"):
            _twice(layer(x, **kw).float().sum(), x)
    logits = _rand(200, 6).requires_grad_()
    for pick in (lambda r: r.balance_loss, lambda r: r.weights[:, 0].sum()):
        with pytest.raises(RuntimeError, match="once_differentiable"):
            _twice(pick(nv.route(logits, 2)), logits)
    r = nv.route(logits, 2)
    y = _rand(r.num_rows, 16).requires_grad_()
    with pytest.raises(RuntimeError, match="once_differentiable"):
        _twice(nv.token_combine(y, r).sum(), y)


def test_constant_gradients_stay_constants(nv):
    """A linear map's gradient under a constant upstream is a constant, and what multiplies it may be differentiated."""
    x = _rand(200, 16).requires_grad_()
    r = nv.route(_rand(200, 6), 2)
    y = _rand(r.num_rows, 16).requires_grad_()
    for f, v in ((lambda v: nv.dropout(v, 0.4, seed=3), x), (lambda v: nv.token_dispatch(v, r), x),
                 (lambda v: nv.token_combine(v, r), y)):
        (g,) = torch.autograd.grad(f(v).sum(), v, create_graph=True)
        assert not g.requires_grad
        (got,) = torch.autograd.grad((g * v).sum(), v)
        assert torch.equal(got, g)


# ------------------------------------------------------------------------------------------------
# Forward mode
# ------------------------------------------------------------------------------------------------


def test_tangents_are_refused_not_dropped(nv):
    """There are no forward-mode formulas: a dual tensor raises, and other tensors work beside one."""
    from torch.autograd import forward_ad

    layer, x = _linear(nv), _rand(256, 256, dtype=torch.bfloat16)
    logits = _rand(256, 6)
    r = nv.route(logits, 2)
    y = _rand(r.num_rows, 256, dtype=torch.bfloat16)
    calls = {
        "dropout": (lambda v: nv.dropout(v, 0.5, seed=1), x),
        "dropout residual": (lambda v: nv.dropout(x, 0.5, seed=1, residual=v), x),
        "linear": (lambda v: layer(v, activation="gelu"), x),
        "linear residual": (lambda v: layer(x, residual=v), x),
        "route": (lambda v: nv.route(v, 2).weights, logits),
        "dispatch": (lambda v: nv.token_dispatch(v, r), x),
        "combine": (lambda v: nv.token_combine(v, r), y),
        "combine weights": (lambda v: nv.token_combine(y, r._replace(weights=v)), r.weights),
        "combine residual": (lambda v: nv.token_combine(y, r, residual=v), x),
    }
    for name, (f, v) in calls.items():
        want = f(v)
        with forward_ad.dual_level():
            assert torch.equal(f(v), want), name
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    f(forward_ad.make_dual(v, torch.ones_like(v)))


# ------------------------------------------------------------------------------------------------
# Functional forms without a gradient
# ------------------------------------------------------------------------------------------------


def test_functional_forms_say_that_they_have_no_gradient(nv):
    """A bias, residual or gradient that requires a gradient is no constant: the result raises in backward."""
    from torch.autograd import forward_ad

    qa, qb = nv.quantize(_rand(256, 128, seed=1), -1), nv.quantize(_rand(384, 128, seed=2), -1)
    bias, res = _rand(384, seed=3), _rand(256, 384, seed=4)
    kw = dict(activation="silu", out_dtype=torch.float32)
    want, wz = nv.epilogue_mm(qa, qb, bias=bias, residual=res, save_preact=True, **kw)
    for name in ("bias", "residual"):
        args = dict(bias=bias, residual=res)
        args[name] = args[name].clone().requires_grad_()
        y, z = nv.epilogue_mm(qa, qb, save_preact=True, **args, **kw)
        assert torch.equal(y, want) and torch.equal(z, wz)
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward()
        with pytest.raises(ValueError, match="out="):
            nv.epilogue_mm(qa, qb, out=torch.empty_like(want), **args, **kw)
        with torch.no_grad():
            out = torch.empty_like(want)
            assert nv.epilogue_mm(qa, qb, out=out, **args, **kw) is out and torch.equal(out, want)
            assert not nv.epilogue_mm(qa, qb, **args, **kw).requires_grad
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            args[name] = forward_ad.make_dual(args[name].detach(), torch.ones_like(args[name]))
            nv.epilogue_mm(qa, qb, **args, **kw)
    leaf = torch.zeros_like(want).requires_grad_()
    with pytest.raises(ValueError, match="out="):
        nv.epilogue_mm(qa, qb, bias=bias, residual=res, out=leaf, **kw)
    gy = _rand(256, 384, seed=5)
    gz, gs, sums = nv.epilogue_backward(gy, wz, activation="silu", bias_grad=True)
    for g, z in ((gy.clone().requires_grad_(), wz), (gy, wz.clone().requires_grad_())):
        got = nv.epilogue_backward(g, z, activation="silu", bias_grad=True)
        assert all(torch.equal(a, b) for a, b in zip(got, (gz, gs, sums)))
        with pytest.raises(RuntimeError, match="no gradient"):
            got[0].sum().backward()
        got = nv.epilogue_backward(g, z, activation="silu")
        assert torch.equal(got[0], gz) and got[2] is None
        with pytest.raises(ValueError, match="out="):
            nv.epilogue_backward(g, z, activation="silu", out=torch.empty_like(gz))


def test_writing_to_out_is_seen_by_autograd(nv):
    """A tensor that another op saved for its backward and that out= then overwrites: backward raises."""
    qa, qb = nv.quantize(_rand(256, 128, seed=1), -1), nv.quantize(_rand(256, 128, seed=2), -1)
    calls = (lambda t: nv.epilogue_mm(qa, qb, residual=t, out=t, out_dtype=torch.float32),
             lambda t: nv.epilogue_mm(qa, qb, out=t, out_dtype=torch.float32),
             lambda t: nv.epilogue_backward(t, dropout_p=0.5, seed=1, out=t))
    for call in calls:
        w, stream = _rand(256, 256, seed=3).requires_grad_(), _rand(256, 256, seed=4)
        loss = (w * stream).sum()
        call(stream)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # tensors without a version counter
        t = _rand(256, 256, seed=4)
        calls[0](t)


# ------------------------------------------------------------------------------------------------
# Autocast
# ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [256, 100])  # NVFP4 and the bf16 fallback
@pytest.mark.parametrize("kw", [dict(), dict(activation="gelu"), dict(activation="silu", dropout_p=0.1, dropout_seed=2)])
def test_linear_keeps_its_type_under_autocast(nv, tokens, kw):
    """An fp32 stream under bf16 autocast: the residual has the input's type on either path, and so has the output."""
    layer = _linear(nv)
    x, res = _rand(tokens, 256, seed=1).requires_grad_(), _rand(tokens, 256, seed=2).requires_grad_()
    with torch.autocast("cuda", torch.bfloat16):
        y = layer(x, residual=res, **kw)
        if kw:
            assert layer(x, **kw).dtype == torch.float32
    assert y.dtype == torch.float32
    gx, gr = torch.autograd.grad(y, (x, res), torch.ones_like(y))
    assert torch.isfinite(gx).all() and (gr == 1).all()


# ------------------------------------------------------------------------------------------------
# Another thread's SM budget
# ------------------------------------------------------------------------------------------------


def test_sm_budget_may_change_between_and_during_calls(nv):
    """Workspaces hold whatever budget another thread sets meanwhile; picks, plans and gradients do not depend on it."""
    import threading

    from radiance_b200 import _lib

    logits, gy, z = _rand(20000, 64, seed=1), _rand(2000, 520, seed=2), _rand(2000, 520, seed=3)
    want, wz = nv.route(logits, 4), nv.epilogue_backward(gy, z, activation="silu", bias_grad=True)
    stop = threading.Event()

    def toggle():
        while not stop.is_set():
            for sms in (1, 148, 7, 0, 90):
                _lib.set_sm_budget(sms)

    before = _lib.set_sm_budget(0)
    thread = threading.Thread(target=toggle)
    thread.start()
    try:
        for _ in range(200):
            r, got = nv.route(logits, 4), nv.epilogue_backward(gy, z, activation="silu", bias_grad=True)
            for a, b in ((r.experts, want.experts), (r.rows, want.rows), (r.counts, want.counts),
                         (r.weights, want.weights), (got[0], wz[0]), (got[1], wz[1])):
                assert torch.equal(a, b)
            # fp32 sums of 2000 terms in another order
            assert ((got[2] - wz[2]).abs() <= 2000 * 2.0**-23 * wz[0].abs().sum(0)).all()
    finally:
        stop.set()
        thread.join()
        _lib.set_sm_budget(before)


# ------------------------------------------------------------------------------------------------
# In place
# ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1 << 22, (1 << 22) + 5])
def test_dropout_in_place(nv, n, dtype):
    """The C entry with y = x and with y = residual, more elements than one round of the blocks takes."""
    from radiance_b200 import _lib

    lib = _lib.load()
    x, res, seed = _rand(n, dtype=dtype, seed=1), _rand(n, dtype=dtype, seed=2), torch.tensor(7, device="cuda")
    code = {torch.bfloat16: _lib.RB_DTYPE_BF16, torch.float32: _lib.RB_DTYPE_F32}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    for r in (None, res):
        want = nv.dropout(x, 0.3, seed=seed, residual=r)
        for into_x in (True, False) if r is not None else (True,):
            a, b = x.clone(), res.clone()
            y = a if into_x else b
            _lib.check(lib.rb_nvfp4_dropout(a.data_ptr(), None if r is None else b.data_ptr(), code, n, 0.3,
                                            seed.data_ptr(), y.data_ptr(), stream), "dropout")
            assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [1024, 1021])
def test_epilogue_backward_into_its_inputs(nv, cols, dtype):
    gy, z = _rand(3000, cols, dtype=dtype, seed=1), _rand(3000, cols, dtype=dtype, seed=2)
    kw = dict(activation="gelu", dropout_p=0.2, seed=5, bias_grad=True)
    want = nv.epilogue_backward(gy, z, **kw)
    for into_gradient in (True, False):
        a, b = gy.clone(), z.clone()
        got = nv.epilogue_backward(a, b, out=a if into_gradient else b, **kw)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


# ------------------------------------------------------------------------------------------------
# Plans that reach past the tensors
# ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 61])
def test_a_wrong_plan_writes_nothing_outside(nv, d, dtype):
    """Rows just past the layout, far past it and below it are skipped, padding ranges are cut to the tensor: the
    rows around it keep what they held, and the pairs that lie inside it their results."""
    from radiance_b200 import _lib

    lib = _lib.load()
    code = {torch.bfloat16: _lib.RB_DTYPE_BF16, torch.float32: _lib.RB_DTYPE_F32}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    r = nv.route(_rand(40, 4, seed=1), 2)
    n, t, k, guard = r.num_rows, 40, 2, 64
    x, y, gy = (_rand(rows, d, dtype=dtype, seed=s) for rows, s in ((t, 2), (n, 3), (t, 4)))
    rows = r.rows.clone()
    rows[0, 0], rows[1, 1], rows[2, 0], rows[3, 1], rows[4, 0] = n, n + guard - 1, 2**31 - 1, -1, -5
    inside = (rows >= 0) & (rows < n)
    at = rows.long()
    token = torch.arange(t, device="cuda").view(-1, 1).expand(t, k)
    for counts, offsets in ((r.counts, r.offsets), (r.counts + 1000, r.offsets), (r.counts - 500, r.offsets),
                            (r.counts, r.offsets - 9), (r.counts, r.offsets + n), (r.counts * 0 - 2**40, r.offsets * 2**40)):
        def buffer():
            b = torch.full((guard + n + guard, d), 7.0, dtype=dtype, device="cuda")
            return b, b[guard:guard + n]

        buf, out = buffer()
        _lib.check(lib.rb_nvfp4_token_dispatch(x.data_ptr(), code, t, d, d, rows.data_ptr(), k, counts.data_ptr(),
                                               offsets.data_ptr(), 4, out.data_ptr(), n, d, stream), "dispatch")
        assert (buf[:guard] == 7).all() and (buf[-guard:] == 7).all()
        if counts is r.counts and offsets is r.offsets:
            assert torch.equal(out[at[inside]], x[token[inside]])
        buf, out = buffer()
        gw = torch.full((t, k), 7.0, device="cuda")
        _lib.check(lib.rb_nvfp4_token_combine_backward(gy.data_ptr(), d, y.data_ptr(), d, code, t, d, rows.data_ptr(), k,
                                                       r.weights.data_ptr(), counts.data_ptr(), offsets.data_ptr(), 4,
                                                       out.data_ptr(), n, d, gw.data_ptr(), stream), "combine backward")
        assert (buf[:guard] == 7).all() and (buf[-guard:] == 7).all()
        assert (gw[~inside] == 0).all()
        prod = gy.double().unsqueeze(1) * torch.where(inside.unsqueeze(-1), y.double()[at.clamp(0, n - 1)], 0.0)
        assert ((gw.double() - prod.sum(-1)).abs() <= d * 2.0**-24 * prod.abs().sum(-1)).all()
        if counts is r.counts and offsets is r.offsets:
            want = (gy.float()[token[inside]] * r.weights[inside].unsqueeze(-1)).to(dtype)
            assert torch.equal(out[at[inside]], want)
        # The combine reads through the same rows.
        buf = torch.full((guard + t + guard, d), 7.0, dtype=dtype, device="cuda")
        out = buf[guard:guard + t]
        _lib.check(lib.rb_nvfp4_token_combine(y.data_ptr(), code, n, d, d, rows.data_ptr(), k, r.weights.data_ptr(),
                                              None, 0, out.data_ptr(), t, d, stream), "combine")
        assert (buf[:guard] == 7).all() and (buf[-guard:] == 7).all()
        terms = torch.where(inside.unsqueeze(-1), y.double()[at.clamp(0, n - 1)], 0.0) * r.weights.double().unsqueeze(-1)
        hs = torch.finfo(dtype).eps / 2
        assert ((out.double() - terms.sum(1)).abs()
                <= hs * terms.sum(1).abs() * 1.01 + (k + 2) * 2.0**-24 * terms.abs().sum(1)).all()


# ------------------------------------------------------------------------------------------------
# Accuracy of the activations, relative to their own values
# ------------------------------------------------------------------------------------------------

REACH = {"silu": 80.0, "gelu": 12.0, "gelu_tanh": 9.0}  # beyond, results leave fp32's normal numbers on the left


def _grid(act, n=8192):
    """Even steps over the range, and magnitudes down to 2^-30 of either sign."""
    line = torch.linspace(-REACH[act], REACH[act], n - 1024, device="cuda")
    small = 2.0 ** torch.linspace(-30, 0, 512, device="cuda")
    return torch.cat([line, small, -small])


def _parts(z, act):
    """The value, and the derivative's two terms, in float64."""
    s = {"silu": lambda: torch.sigmoid(z), "gelu": lambda: 0.5 * torch.special.erfc(-z * 0.5**0.5),
         "gelu_tanh": lambda: torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z**3))}[act]()
    up = {"silu": lambda: s * torch.sigmoid(-z), "gelu": lambda: torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5,
          "gelu_tanh": lambda: (s * torch.sigmoid(-2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z**3))
                                * 2 * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z))}[act]()
    return z * s, s, z * up


def _exact_room(act):
    # In units of 2^-23 of the value: the exponential 2, the reciprocal 1 (times at most 2.6 where GELU's tail
    # follows it), GELU's polynomial 1.1, and half of one for each of at most six roundings: under 9.
    return 9 * 2.0**-23


@pytest.mark.parametrize("act", list(REACH))
def test_fp32_activations_are_accurate_everywhere(nv, act):
    z = _grid(act)
    a, b = nv.quantize(torch.zeros(128, 64, device="cuda"), -1), nv.quantize(torch.zeros(z.numel(), 64, device="cuda"), -1)
    y, pre = nv.epilogue_mm(a, b, bias=z, activation=act, out_dtype=torch.float32, save_preact=True)  # 0 + bias
    assert torch.equal(pre[0], z) and torch.equal(y, y[:1].expand_as(y))
    value, s, t = _parts(z.double(), act)
    assert ((y[0].double() - value).abs() <= _exact_room(act) * value.abs()).all()
    d = nv.epilogue_backward(torch.ones(1, z.numel(), device="cuda"), z[None], activation=act)[0][0].double()
    # Each term as the value; the sum is one rounding, the second term's factors two more.
    assert ((d - s - t).abs() <= (_exact_room(act) + 1.5 * 2.0**-23) * (s + t.abs())).all()


@pytest.mark.parametrize("act", list(REACH))
def test_bf16_activations_are_rounded_about_once(nv, act):
    """Before its one rounding GELU is off by 7.5e-8 of |z| near 0 and 3.8e-4 of itself far out on the left, the
    others as in fp32 but for the exponent's roundings: 2^-23 of an exponent of at most 127."""
    z = _grid(act).bfloat16()
    a, b = nv.quantize(torch.zeros(128, 64, device="cuda"), -1), nv.quantize(torch.zeros(z.numel(), 64, device="cuda"), -1)
    y = nv.epilogue_mm(a, b, bias=z, activation=act)[0].double()
    zd = z.double()
    value, s, t = _parts(zd, act)
    room = 2.0**-20 + 127 * 2.0**-23
    # GELU's tail q carries into z > 0 as z (1 - q) and into z < 0 as z q.
    q = torch.minimum(s, 1 - s) if act == "gelu" else torch.zeros_like(s)
    tail = torch.minimum(3.9e-4 * q, torch.full_like(q, 8e-8)) if act == "gelu" else q
    err = room * value.abs() + tail * zd.abs()
    assert ((y - value).abs() <= 2.0**-8 * (value.abs() + err) + err).all()
    d = nv.epilogue_backward(torch.ones(1, z.numel(), dtype=torch.bfloat16, device="cuda"), z[None],
                             activation=act)[0][0].double()
    # 1 - s is taken from the rounded s here: 2^-23 of 1, times |z| times its factor (its slope).
    slope = {"gelu": 0.0, "silu": 1.0, "gelu_tanh": 1.6 + 0.22 * zd * zd}[act]
    err = room * (s + t.abs()) + tail + 2.0**-22 * s * zd.abs() * slope
    assert ((d - s - t).abs() <= 2.0**-8 * ((s + t).abs() + err) + err).all()
