"""Experts beside a token whose router scores are not numbers: such a token chooses nothing, and the others' results are those of a step in which it
chose other experts, bit for bit (rows do not meet in any sum)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
LIMIT = 7.0


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


class Experts:
    """Two products on a route, the weights in 16 bits (bf16 or f32 steps) or in 4."""

    def __init__(self, lm, form, tokens, experts, identity, width=128, ff=64, seed=3):
        from peregrine_b200.layers import Device, Linear, Linear4

        self.lm = lm
        d = self.d = Device(lm, "float32" if form == "f32" else "bfloat16", tokens)
        t = d.torch
        self.E, self.I, self.width, self.ff = experts, identity, width, ff
        g = np.random.Generator(np.random.PCG64(seed))
        w = lambda n, k: d.bf16((g.standard_normal((experts, n, k)) / k ** 0.5).astype(np.float32))
        make = Linear4 if form == "four" else Linear
        self.gate_up, self.down = make(d, w(2 * ff, width)), make(d, w(width, ff))
        self.x0 = d.f32(g.standard_normal((tokens, width)))
        self.ones = t.ones(width, device=d.dev)

    def step(self, logits, top, correction=None):
        """x behind the step, the choices and their weights, from buffers full of what an earlier step may have left."""
        d, lib, h = self.d, self.d.lib, self.lm.handle
        t, (m, n) = d.torch, logits.shape
        route = C.c_void_p()
        d.check(lib.pg_route_create(h, m, self.E, self.I, top, C.byref(route)))
        rows = lib.pg_route_max_rows(route)
        act, out = (t.full((rows, c), 1e4, dtype=d.act, device=d.dev) for c in (self.ff, self.width))
        x, hx = self.x0[:m].clone(), self.x0[:m].to(d.act)
        hy = t.zeros_like(hx)
        z, corr = d.f32(logits), d.f32(np.zeros(n) if correction is None else correction)
        t.cuda.synchronize()
        d.check(lib.pg_route_run(h, route, d.code, z.data_ptr(), n, m, corr.data_ptr(), 1, 1))
        self.gate_up.run_routed(route, hx, True, act, 2, LIMIT)
        self.down.run_routed(route, act, False, out)
        d.check(lib.pg_routed_norm_add(h, route, out.data_ptr(), out.stride(0), x.data_ptr(), self.ones.data_ptr(), self.ones.data_ptr(), m, self.width, 1e-5, hy.data_ptr(),
                                       d.code, self.width))
        ids, w = np.zeros((m, top), np.int32), np.zeros((m, top), np.float32)
        d.check(lib.pg_route_read(h, route, ids.ctypes.data, w.ctypes.data))
        d.check(lib.pg_route_free(h, route))
        assert self.lm.device_status() == 0
        return x.cpu().numpy(), ids, w

    def free(self):
        self.gate_up.free(), self.down.free()


@pytest.mark.parametrize("form", ["four", "bf16", "f32"])
@pytest.mark.parametrize("m", [2, 5, 8, 9, 16, 40])
@pytest.mark.parametrize("bad,identity", [(1, 0), (2, 0), (2, 3)])
def test_a_token_without_a_choice(lm, form, m, bad, identity):
    if bad >= m:
        bad = m - 1
    E, top = 12, 8
    e = Experts(lm, form, m, E, identity)
    g = np.random.Generator(np.random.PCG64(m))
    z = g.standard_normal((m, E + identity)).astype(np.float32)
    z[:, E - 1] += 20.0                                       # everyone's best choice
    where = np.arange(bad) * 3 % m                            # the first token is among them: its pairs come first
    other = z.copy()
    other[where] = np.where(np.arange(E + identity) < top, 5.0, -5.0)
    for what in (np.nan, np.inf):
        z[where, 4] = what                                    # one is enough: no score of the token is a number
        for again in range(3):                                # (which row a pair gets is left to the order of arrival)
            x, ids, w = e.step(z, top)
            want, want_ids, want_w = e.step(other, top)
            good = np.delete(np.arange(m), where)
            assert np.array_equal(ids[good], want_ids[good]) and np.array_equal(w[good], want_w[good])
            assert np.array_equal(x[good], want[good])
            assert (ids[where] == E + identity - 1).all() and not w[where].any()
            assert np.array_equal(x[where], e.x0[where.tolist()].cpu().numpy())          # nothing is added
    e.free()


@pytest.mark.parametrize("form", ["four", "bf16", "f32"])
@pytest.mark.parametrize("m", [1, 7, 16, 30])
def test_no_token_with_a_choice(lm, form, m):
    """A route without a row."""
    e = Experts(lm, form, m, 5, 0)
    x, ids, w = e.step(np.full((m, 5), np.nan, np.float32), 3)
    assert np.array_equal(x, e.x0[:m].cpu().numpy()) and (ids == 4).all() and not w.any()
    e.free()


@pytest.mark.parametrize("form", ["four", "bf16", "f32"])
@pytest.mark.parametrize("m", [3, 8, 16, 30])
def test_fewer_scores_than_choices(lm, form, m):
    """Outputs whose correction is not a number are never chosen: the other choices are those of a smaller `top`."""
    E, left = 9, 5
    e = Experts(lm, form, m, E, 0)
    z = np.random.Generator(np.random.PCG64(m)).standard_normal((m, E)).astype(np.float32)
    correction = np.zeros(E, np.float32)
    correction[:E - left] = np.nan
    x, ids, w = e.step(z, 8, correction)
    want, want_ids, want_w = e.step(z, left, correction)
    assert np.array_equal(ids[:, :left], want_ids) and np.array_equal(w[:, :left], want_w) and (want_ids >= E - left).all()
    assert (ids[:, left:] == E - 1).all() and not w[:, left:].any()
    assert np.array_equal(x, want)
    e.free()
