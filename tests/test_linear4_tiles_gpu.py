"""Products with 4-bit weights of few rows on the tensor cores: tiles of 32 rows, which are the narrowest that a pair's products with the weights in
TMEM take, partly empty and not.  Bounds as in tests/test_linear4_gpu.py."""
import ctypes as C

import numpy as np
import pytest

from tests.test_linear4_gpu import ACTS, LIMIT, bf16, device, gated, handle, quants, rng, run, sums, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


@pytest.mark.parametrize("n,k", [(1024, 1024), (256, 2048), (300, 192)])
def test_few_rows_of_small_matrices(lm, n, k):
    d = device(lm, 64)
    g = rng(n + k)
    q, s, w = quants(g, n, k, group=64)
    lin = handle(d, q, s)
    for m in (17, 24, 31, 32, 33, 47, 48, 49, 64):
        x = bf16(d, g.standard_normal((m, k)))
        want, bound = sums(x.double().cpu().numpy(), w)
        within(run(d, lin, x, m, n), want, bound, f"m {m}")
    lin.free()


@pytest.mark.parametrize("per", [1, 3, 12, 13, 24, 25, 31, 32, 33])
def test_few_rows_of_an_expert(lm, per):
    """`per` tokens to each of some experts, one to the last, none to the first; every row of the route against its token's product."""
    E, n, k = 7, 272, 128
    m = per * (E - 2) + 1
    if m <= 16:
        E, m = 18, 17 * max(per, 1)
    d = device(lm, m)
    t, lib, h = d.torch, d.lib, lm.handle
    g = rng(per)
    q, s, w = quants(g, E, n, k, group=64)
    lin = handle(d, q, s)
    chosen = np.minimum(1 + np.arange(m) // per, E - 1)
    logits = np.full((m, E), -9.0, np.float32)
    logits[np.arange(m), chosen] = 9.0
    x = bf16(d, g.standard_normal((m, k)))
    z, corr, route = d.f32(logits), t.zeros(E, device=d.dev), C.c_void_p()
    d.check(lib.pg_route_create(h, m, E, 0, 1, C.byref(route)))
    out = t.full((lib.pg_route_max_rows(route), n), 3.0, device=d.dev)
    t.cuda.synchronize()
    d.check(lib.pg_route_run(h, route, d.code, z.data_ptr(), E, m, corr.data_ptr(), 1, 1))
    lin.run_routed(route, x, True, out)
    lm.sync()
    assert lm.device_status() == 0
    got, at = out.cpu().numpy(), 0
    for e in range(E):
        tokens = np.nonzero(chosen == e)[0]
        if not len(tokens):
            continue
        want, bound = sums(x[tokens.tolist()].double().cpu().numpy(), w[e])
        rows = got[at:at + len(tokens)]
        order = lambda v: np.argsort(v[:, 0], kind="stable")      # (an expert's tokens come in any order)
        within(rows[order(rows)], want[order(want)], bound[order(want)], f"expert {e}")
        at += -(-len(tokens) // 128) * 128
    d.check(lib.pg_route_free(h, route))
    lin.free()


@pytest.mark.parametrize("act", ["none", "gelu", "swish"])
@pytest.mark.parametrize("m", [1, 6, 8, 9, 16, 17, 100])
def test_activations_of_a_stack_in_groups_of_128(lm, m, act):
    E, n, k, top = 5, 176, 256, 2
    d = device(lm, m)
    t, lib, h = d.torch, d.lib, lm.handle
    g = rng(m)
    q, s, w = quants(g, E, n, k, group=128)
    lin = handle(d, q, s)
    logits = g.standard_normal((m, E)).astype(np.float32)
    x = bf16(d, g.standard_normal((m, k)) * 3)
    z, corr, route = d.f32(logits), t.zeros(E, device=d.dev), C.c_void_p()
    d.check(lib.pg_route_create(h, m, E, 0, top, C.byref(route)))
    cols = n if act == "none" else n // 2
    out = t.full((lib.pg_route_max_rows(route), cols), 3.0, dtype=t.bfloat16, device=d.dev)
    t.cuda.synchronize()
    d.check(lib.pg_route_run(h, route, d.code, z.data_ptr(), E, m, corr.data_ptr(), 1, 1))
    lin.run_routed(route, x, True, out, ACTS[act], LIMIT)
    lm.sync()
    assert lm.device_status() == 0
    got, at = out.float().cpu().numpy(), 0
    chosen = np.argsort(-logits, 1, kind="stable")[:, :top]
    for e in range(E):
        tokens = np.nonzero((chosen == e).any(1))[0]
        if not len(tokens):
            continue
        want, bound = sums(x[tokens.tolist()].double().cpu().numpy(), w[e])
        if act != "none":
            want, bound = gated(want, bound, act)
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound) + 2.0 ** -134
        rows = got[at:at + len(tokens)]
        # (an expert's tokens come in any order: each row is its token's, in every column)
        near = (np.abs(rows[:, None] - want[None]) <= bound[None]).all(2)
        assert near.any(1).all() and near.any(0).all(), f"expert {e}"
        block = 16 if m <= 16 else 128
        at += -(-len(tokens) // block) * block
    d.check(lib.pg_route_free(h, route))
    lin.free()
