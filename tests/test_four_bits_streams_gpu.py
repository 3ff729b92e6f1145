"""Values of weights and caches of 4 bits, read while torch's stream is busy: the memory that they are read into may be that of a tensor which the
stream has not finished with."""
import numpy as np
import pytest

from tests.test_attention4_gpu import Case
from tests.test_linear4_gpu import device, handle, quants, rng

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


def busy(t, dev, *shape):
    """Torch's stream writes to tensors of this shape in a tenth of a second; their memory is free for the next tensor at once."""
    many = [t.empty(*shape, dtype=t.float32, device=dev).fill_(4.0) for _ in range(16)]    # (a kernel's first launch would wait)
    t.cuda.synchronize()
    t.cuda._sleep(200_000_000)
    for x in many:
        x.fill_(5.0)


def test_weights(lm):
    d = device(lm)
    q, s, w = quants(rng(3), 2, 200, 512, group=64)
    lin = handle(d, q, s)
    lin.values()                                            # (the same of its kernel)
    busy(d.torch, d.dev, 2, 200, 512)
    got = lin.values()
    d.torch.cuda.synchronize()
    assert np.array_equal(got.cpu().numpy().astype(np.float64), w)
    lin.free()


@pytest.mark.parametrize("values", [False, True])
def test_caches(lm, values):
    c = Case(lm, 7, 4, 2, 64, 64, 600, 2, 64)
    c.append(0, 0, c.rows(300))
    cache = c.vc if values else c.kc
    want = c.plan.values(cache, 600, values).cpu()
    c.d.torch.cuda.synchronize()
    busy(c.d.torch, c.d.dev, 4, 600, 64)
    got = c.plan.values(cache, 600, values)
    c.d.torch.cuda.synchronize()
    assert want.any() and c.d.torch.equal(got.cpu(), want)
