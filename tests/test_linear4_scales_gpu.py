"""Products with 4-bit weights whose groups have very different scales: every form of the product takes the weights that pg_linear4_read says.
Bounds as in tests/test_linear4_gpu.py."""
import numpy as np
import pytest

from tests.test_linear4_gpu import bf16, device, handle, rng, run, sums, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 4, 9, 16, 17, 40, 100, 300])
def test_a_small_group_beside_a_large_one(lm, m, group):
    """Row r has one group of scales around 1 and the others 2^-r of that (2^-32 at last); the activations are zero outside the small groups, so that
    nothing covers their digits up."""
    import torch

    d = device(lm, 300)
    n, k = 33, 4 * group
    g = rng(m + group)
    q = g.integers(0, 16, (n, k)).astype(np.uint8)
    s = g.uniform(1.0, 2.0, (n, 4)).astype(np.float32)
    s[:, 1:] *= 2.0 ** -np.arange(n, dtype=np.float32)[:, None]
    lin = handle(d, torch.from_numpy(q[:, 0::2] | q[:, 1::2] << 4), torch.from_numpy(s).bfloat16())
    w = lin.values().cpu().numpy()[0].astype(np.float64)
    a = g.standard_normal((m, k))
    a[:, :group] = 0.0
    x = bf16(d, a)
    want, bound = sums(x.double().cpu().numpy(), w)
    within(run(d, lin, x, m, n), want, bound)
    lin.free()


def test_scales_apart(lm):
    """Eight bits of a scale of 2^-28 beside one of 1."""
    import torch

    d = device(lm)
    q = np.full((1, 128), 15, np.uint8)
    s = np.array([[1.0, 255 / 128 * 2.0 ** -28]], np.float32)
    lin = handle(d, torch.from_numpy(q[:, 0::2] | q[:, 1::2] << 4), torch.from_numpy(s).bfloat16())
    assert np.array_equal(lin.values().cpu().numpy()[0], 7 * np.repeat(s, 64, 1))
    lin.free()


@pytest.mark.parametrize("m", [3, 16, 17, 130])
def test_small_activations_beside_a_large_one(lm, m):
    """Activations of 2^-27 of the row's largest, where they stand alone: the large one meets weights of zero."""
    import torch

    d = device(lm, 300)
    n, k, group = 20, 256, 64
    g = rng(m)
    q = g.integers(0, 16, (n, k)).astype(np.uint8)
    q[:, 5] = 8
    s = g.uniform(0.01, 0.02, (n, k // group)).astype(np.float32)
    lin = handle(d, torch.from_numpy(q[:, 0::2] | q[:, 1::2] << 4), torch.from_numpy(s).bfloat16())
    w = lin.values().cpu().numpy()[0].astype(np.float64)
    a = g.uniform(1.0, 2.0, (m, k)) * np.sign(g.standard_normal((m, k))) * 2.0 ** -27
    a[:, 5] = 1.0
    x = bf16(d, a)
    want, bound = sums(x.double().cpu().numpy(), w)
    within(run(d, lin, x, m, n), want, bound)
    lin.free()
