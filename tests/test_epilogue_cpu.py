"""The epilogue, dropout and routing operators without a GPU: the oracle's generator against published
vectors, the sizes computed on the host, and the C entry points' refusals."""

import ctypes

import numpy as np
import pytest
import torch

from radiance_b200 import _lib
from tests import _epilogue_oracle as O


def test_philox_known_answers():
    """The known-answer vectors published with Random123 for philox4x32-10."""
    zero = O.philox4x32_10(np.zeros((1, 4), np.uint32), (0, 0))[0]
    assert [hex(v) for v in zero] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = O.philox4x32_10(np.full((1, 4), 0xFFFFFFFF, np.uint32), (0xFFFFFFFF, 0xFFFFFFFF))[0]
    assert [hex(v) for v in ones] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]
    ctr = np.array([[0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], np.uint32)
    pi = O.philox4x32_10(ctr, (0xA4093822, 0x299F31D0))[0]
    assert [hex(v) for v in pi] == ["0xd16cfe09", "0x94fdcceb", "0x5001e420", "0x24126ea1"]


def test_oracle_derivatives_against_differences():
    z = torch.linspace(-6, 6, 241, dtype=torch.float64) + 0.013
    h = 1e-6
    for name in O.ACTIVATIONS:
        diff = (O.activation(z + h, name) - O.activation(z - h, name)) / (2 * h)
        # truncation h^2 |f'''| / 6 and cancellation 2^-52 |f| / h
        assert (diff - O.derivative(z, name)).abs().max() < 1e-8, name


@pytest.mark.parametrize("t,k,e", [(0, 2, 4), (1, 1, 1), (1, 2, 256), (100, 2, 8), (127, 1, 3), (4099, 6, 160)])
def test_routed_rows_bound(t, k, e):
    """The worst routing of these sizes fits, and no smaller multiple of 128 would hold it."""
    import radiance_b200.nvfp4 as nv

    pairs, n = t * k, min(e, t * k)
    counts = [0] * e
    for i in range(n):
        counts[i] = 1  # every expert that can start a group does; the rest goes where it starts new tiles
    left = pairs - n
    for i in range(n):
        while left >= 128:
            counts[i] += 128
            left -= 128
    if n:
        counts[0] += left
    need = sum((c + 127) // 128 * 128 for c in counts)
    assert need <= nv.routed_rows(t, k, e) and nv.routed_rows(t, k, e) % 128 == 0
    assert nv.routed_rows(t, k, e) - need < 256


def test_entry_points_refuse_on_the_host():
    lib = _lib.load()
    buf, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)  # never dereferenced: validation fails first

    def msg():
        return lib.rb_nvfp4_last_error().decode()

    assert lib.rb_nvfp4_dropout(buf, None, 7, 8, 0.5, buf, buf, None) == 2 and "dtype" in msg()
    for p in (-0.5, 1.5, float("nan")):
        assert lib.rb_nvfp4_dropout(buf, None, 0, 8, p, buf, buf, None) == 2 and "probability" in msg()
    assert lib.rb_nvfp4_dropout(buf, None, 0, 8, 0.5, None, buf, None) == 2 and "seed" in msg()
    assert lib.rb_nvfp4_dropout(buf, None, 0, 8, 0.5, odd, buf, None) == 2 and "seed" in msg()
    assert lib.rb_nvfp4_dropout(None, None, 0, 8, 0.0, None, buf, None) == 2 and "null" in msg()
    assert lib.rb_nvfp4_dropout(buf, None, 0, -1, 0.0, None, buf, None) == 1
    assert lib.rb_nvfp4_dropout(None, None, 0, 0, 0.0, None, None, None) == 0  # nothing to do

    def gemm(act=0, p=0.0, seed=None, res=None, ldr=128, z=None, ldz=128, out=buf, m=128, dt=0):
        return lib.rb_nvfp4_gemm_epilogue(buf, buf, buf, buf, m, 128, 64, None, None, None, 0, act, p, seed, res, ldr,
                                          z, ldz, out, dt, 128, None)

    assert gemm(m=100) == 1 and "m % 128" in msg()
    for kw in (dict(act=6), dict(act=-1), dict(p=1.5), dict(p=float("nan")), dict(p=0.5), dict(p=0.5, seed=odd)):
        assert gemm(**kw) == 2 and "activation" in msg(), kw
    for kw in (dict(res=odd), dict(res=buf, ldr=127), dict(res=buf, ldr=132), dict(z=odd), dict(z=buf, ldz=64)):
        assert gemm(**kw) == 2 and "residual" in msg(), kw
    assert gemm(out=None) == 2 and gemm(dt=5) == 2

    def back(rows=4, cols=8, ldg=8, z=buf, act=4, ws=buf, out=buf, p=0.0, seed=None):
        return lib.rb_nvfp4_epilogue_backward(buf, ldg, z, 8, 0, rows, cols, act, p, seed, out, 8, buf, None, ws,
                                              1 << 20, None)

    assert back(act=6) == 2 and "activation" in msg()
    assert back(act=-1) == 2
    assert back(rows=0) == 1 and back(cols=0) == 1 and back(ldg=7) == 1
    assert back(z=None) == 2 and back(ws=None) == 2 and back(out=None) == 2
    assert back(p=0.5) == 2 and "seed" in msg()

    def route(dtype=1, tokens=4, experts=8, ld=8, k=2, logits=buf, counts=buf, ws=buf):
        return lib.rb_nvfp4_route(logits, dtype, tokens, experts, ld, k, None, None, 1, buf, buf, buf, counts, buf,
                                  buf, buf, ws, 1 << 20, None)

    assert route(dtype=3) == 2 and "dtype" in msg()
    for kw in (dict(k=0), dict(k=9), dict(experts=0), dict(experts=257, ld=257), dict(experts=64, ld=64, k=33),
               dict(ld=7), dict(tokens=-1), dict(tokens=1 << 31)):
        assert route(**kw) == 1, kw
    assert route(logits=None) == 2 and route(ws=None) == 2 and route(counts=ctypes.c_void_p(4)) == 2
    assert lib.rb_nvfp4_route_backward(buf, 1, 4, 8, 8, 2, 1, buf, buf, buf, None, None, buf, 7, None) == 1
    assert lib.rb_nvfp4_route_backward(buf, 1, 4, 8, 8, 2, 1, None, buf, buf, None, None, buf, 8, None) == 2

    def disp(dtype=0, tokens=4, d=8, ld=8, k=2, e=4, n=512, ldo=8, out=buf):
        return lib.rb_nvfp4_token_dispatch(buf, dtype, tokens, d, ld, buf, k, buf, buf, e, out, n, ldo, None)

    assert disp(dtype=9) == 2
    for kw in (dict(tokens=-1), dict(d=0), dict(ld=7), dict(k=0), dict(e=0), dict(e=257), dict(n=-1), dict(ldo=7),
               dict(n=1 << 31)):
        assert disp(**kw) == 1, kw
    assert disp(out=None) == 2
    assert lib.rb_nvfp4_token_combine(buf, 0, 512, 8, 8, buf, 2, None, buf, 7, buf, 4, 8, None) == 1
    assert lib.rb_nvfp4_token_combine(None, 0, 512, 8, 8, buf, 2, None, None, 0, buf, 4, 8, None) == 2
    assert lib.rb_nvfp4_token_combine_backward(buf, 7, buf, 8, 0, 4, 8, buf, 2, buf, buf, buf, 4, buf, 512, 8, buf,
                                               None) == 1
    assert lib.rb_nvfp4_token_combine_backward(buf, 8, buf, 8, 0, 4, 8, buf, 2, None, buf, buf, 4, buf, 512, 8, buf,
                                               None) == 2


def test_operators_refuse_cpu_tensors():
    import radiance_b200.nvfp4 as nv

    x = torch.randn(128, 64)
    r = nv.Routing(torch.zeros(128, 2), torch.zeros(128, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64),
                   torch.zeros(()), torch.zeros(5, dtype=torch.int64), torch.zeros(128, 2, dtype=torch.int32), 512)
    q = nv.NVFP4Tensor(torch.zeros(128, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), torch.ones(()))
    for call in (lambda: nv.dropout(x, 0.5), lambda: nv.epilogue_mm(q, q), lambda: nv.epilogue_backward(x), lambda: nv.route(x, 2),
                 lambda: nv.token_dispatch(x, r), lambda: nv.token_combine(x, r)):
        with pytest.raises(RuntimeError, match="no CPU"):
            call()
