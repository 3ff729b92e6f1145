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


def words(entries, rows, seqs):
    """A batch's array: tokens, positions and sequence of each row, first rows, slots."""
    host = np.zeros(3 * rows + 2 * seqs + 1, np.int32)
    at = 0
    for i, (slot, pos, n) in enumerate(entries):
        host[rows + at:rows + at + n], host[2 * rows + at:2 * rows + at + n] = np.arange(pos, pos + n), i
        at += n
        host[3 * rows + i + 1], host[3 * rows + seqs + 1 + i] = at, slot
    return host


def test_a_recorded_portion_is_for_its_positions(lm):
    """Replayed over a batch with other positions, or another slot, a longer portion is reported; over its own it is as good as ever."""
    from tests.test_attention4_digits_gpu import want

    c = Case(lm, 17, 8, 2, 64, 96, 700, 2, 400)
    t = c.d.torch
    c.append(1, 0, c.rows(300)), c.append(0, 0, c.rows(300))
    entries = [(1, 200, 150)]
    b = c.batch(entries, fixed=True)
    proj = c.rows(150)
    x, out = t.from_numpy(proj).to(c.d.dev), t.zeros(150, c.H * c.V, dtype=t.bfloat16, device=c.d.dev)
    t.cuda.synchronize()
    with lm.record() as g:
        c.plan.run(b, x, c.kc, c.vc, out)
    for now, status in (([(1, 200, 150)], 0), ([(1, 250, 150)], -1), ([(0, 200, 150)], -1), ([(1, 200, 150)], 0)):
        b.write(words(now, 150, 1))
        g.launch()
        lm.sync()
        assert lm.device_status() == status
    y, bound = want(c, entries, proj)
    assert (np.abs(out.float().cpu().numpy().reshape(y.shape) - y) <= bound).all()
    g.free()


def test_a_later_plan_leaves_a_recorded_one_its_workspaces(lm):
    """A wider plan on the same device takes larger workspaces; what a graph was recorded with stays its own."""
    from peregrine_b200.layers import Attention4Plan

    c = Case(lm, 18, 8, 2, 64, 64, 3000, 2, 200)
    t = c.d.torch
    c.append(0, 0, c.rows(2500)), c.append(1, 0, c.rows(300))
    entries = [(0, 2500, 2), (1, 300, 150)]
    b = c.batch(entries, fixed=True)
    proj = c.rows(152)
    x, out = t.from_numpy(proj).to(c.d.dev), t.zeros(152, c.H * c.V, dtype=t.bfloat16, device=c.d.dev)
    t.cuda.synchronize()
    with lm.record() as g:
        c.plan.run(b, x, c.kc, c.vc, out)
    sizes = [c.d.buffer("attn4.part", 1, 1, t.float32).numel(), c.d.buffer("attn4.work", 1, 1).numel() // 2]
    Attention4Plan(c.d, 8, 2, 64, 256, 9000, 2, 2, scale=1.0)
    others = [t.full((n,), 9.0, device=c.d.dev) for n in sizes for _ in range(8)]
    t.cuda.synchronize()
    g.launch()
    lm.sync()
    assert all((o == 9.0).all() for o in others)
    graph = out.clone()
    t.cuda.synchronize()
    c.plan.run(b, x, c.kc, c.vc, out)
    lm.sync()
    assert t.equal(out, graph) and lm.device_status() == 0
    g.free()
