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
