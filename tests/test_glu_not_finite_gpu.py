"""Gated products of what is not a number: the clamp of a gate or of an up must not turn it into one."""
import numpy as np
import pytest

from tests.test_linear4_gpu import ACTS, LIMIT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


@pytest.mark.parametrize("form", ["four", "bf16", "f32"])
@pytest.mark.parametrize("act", ["gelu", "swish"])
@pytest.mark.parametrize("m", [1, 3, 16, 17, 130, 300])
def test_rows_and_columns(lm, form, act, m):
    from peregrine_b200.layers import Device, Linear, Linear4

    d = Device(lm, "float32" if form == "f32" else "bfloat16", 300)
    t = d.torch
    g = np.random.Generator(np.random.PCG64(m))
    F, k = 40, 128
    gate, up = ((g.standard_normal((F, k)) * 0.1).astype(np.float32) for _ in range(2))
    gate[3, 70], up[17, 5] = np.nan, np.nan                       # columns 3 and 17 of the output
    lin = (Linear4 if form == "four" else Linear)(d, (d.bf16(gate), d.bf16(up)), gated=True)
    a = g.standard_normal((m, k))
    if m > 1:
        a[m - 2, 9] = np.nan                                      # a row
    x = d.f32(a).to(d.act)
    y = t.zeros(m, F, dtype=d.act, device=d.dev)
    t.cuda.synchronize()
    lin.run(x, m, y, ACTS[act], LIMIT)
    lm.sync()
    bad = np.isnan(y.float().cpu().numpy())
    want = np.zeros((m, F), bool)
    want[:, [3, 17]] = True
    if m > 1:
        want[m - 2] = True
    assert np.array_equal(bad, want) and lm.device_status() == 0
    lin.free()
