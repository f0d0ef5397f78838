"""What the sublayer operators promise, as far as it shows without a GPU."""

import ctypes

import pytest
import torch

from radiance_b200 import _lib


def test_row_moves_go_by_the_plan_counts():
    """The moves read the routing's private counts, and `counts` only in a plan that has none."""
    import radiance_b200.nvfp4 as nv
    from radiance_b200.nvfp4 import routing

    counts, kept = torch.full((4,), 9), torch.arange(4)
    rows, offsets = torch.zeros(8, 2, dtype=torch.int32), torch.zeros(5, dtype=torch.int64)
    r = nv.Routing(torch.zeros(8, 2), rows, counts, torch.zeros(()), offsets, rows, 512)
    cpu = torch.device("cpu")
    assert routing._plan(r, cpu, "x")[1] is counts
    assert routing._plan(r._replace(plan_counts=kept), cpu, "x")[1] is kept
    with pytest.raises(ValueError, match="counts"):
        routing._plan(r._replace(plan_counts=kept.int()), cpu, "x")


def test_route_plan_refuses_on_the_host():
    lib = _lib.load()
    buf = ctypes.c_void_p(256)  # never dereferenced: validation fails first

    def plan(k=2, counts=buf, kept=buf):
        return lib.rb_nvfp4_route_plan(buf, 1, 4, 8, 8, k, None, None, 1, buf, buf, buf, counts, kept, buf, buf, buf,
                                       buf, 1 << 20, None)

    assert plan(k=0) == 1 and plan(counts=None) == 2 and plan(kept=ctypes.c_void_p(260)) == 2


def test_workspaces_hold_for_every_sm_budget():
    """Sizes do not follow the SM budget, which may change between the question and the call; and they hold the
    most blocks that any budget leads to."""
    lib = _lib.load()
    sizes = [(lambda t=t, e=e, k=k: lib.rb_nvfp4_route_workspace(t, e, k))
             for t, e, k in ((0, 8, 2), (1, 1, 1), (4099, 160, 6), (16384, 8, 2), (131072, 64, 8), (300, 256, 32))]
    sizes += [(lambda r=r, c=c: lib.rb_nvfp4_epilogue_backward_workspace(r, c))
              for r, c in ((1, 1), (640, 1152), (16384, 5632), (17, 40000), (1 << 22, 8))]
    sizes += [(lambda d=d, r=r, c=c: lib.rb_nvfp4_global_scale_colsum_workspace(d, r, c))
              for d, r, c in ((0, 16384, 5632), (1, 640, 1152), (0, 1 << 20, 64))]
    before = _lib.set_sm_budget(0)
    try:
        full = [f() for f in sizes]
        for sms in (1, 2, 37, 100, 147):
            _lib.set_sm_budget(sms)
            assert [f() for f in sizes] == full
    finally:
        _lib.set_sm_budget(before)
    for (t, e, k), size in zip(((4099, 160, 6), (16384, 8, 2), (131072, 64, 8), (300, 256, 32)), full[2:6]):
        lanes = 1
        while lanes < min(e, 32):
            lanes *= 2
        groups, most = 512 // lanes, 4096 // k
        for sms in range(1, 149):  # the kernel's chunks: whole steps of its groups, at most `most` tokens
            turns = -(-t // (sms * most))
            chunk = min(most, -(-(-(-t // (sms * turns))) // groups) * groups)
            assert -(-t // chunk) * (6 * e + 4) <= size
