"""Products with weights of 4 bits (pg_linear4_*), on the GPU against sums in 64 bits.

Bounds.  A product of a bf16 number and a weight's value is exact in the kernels; a sum of K of them goes through K / 16 matrix instructions, a
group's and a part's joins.  Each may cut its result off below 2^-23 of the largest sum that it meets, which is at most S = sum |a w|; every
instruction adds 16 products that are aligned to the largest of them, the same once more.  So |error| <= (K / 8 + 64) 2^-23 S.  A bf16 output
adds half a step, 2^-8 of its value."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ACTS = {"none": 0, "gelu": 1, "swish": 2}
LIMIT = 7.0


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


def device(lm, rows=64, dtype="bfloat16"):
    from peregrine_b200.layers import Device

    return Device(lm, dtype, rows)


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


def bf16(d, a):
    out = d.torch.from_numpy(np.asarray(a, np.float32)).to(d.dev).to(d.torch.bfloat16)
    d.torch.cuda.synchronize()
    return out


def quants(g, *shape, group):
    """Random quants, scales and the values they stand for (f64)."""
    import torch

    q = g.integers(0, 16, shape).astype(np.uint8)
    s = torch.from_numpy((g.standard_normal((*shape[:-1], shape[-1] // group)) * 0.02).astype(np.float32)).bfloat16()
    w = (q.astype(np.float64) - 8).reshape(*shape[:-1], -1, group) * s.double().numpy()[..., None]
    return torch.from_numpy(q[..., 0::2] | q[..., 1::2] << 4), s, w.reshape(shape)


def handle(d, q, s):
    from peregrine_b200.layers import Linear4

    return Linear4.from_quants(d, q.to(d.dev), s.to(d.dev))


def sums(a, w):
    """a W^T in 64 bits and the bound of the f32 sums."""
    return a @ w.T, (a.shape[1] / 8 + 64) * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)


def gated(y, b, act):
    """The gated outputs of sums y with bounds b, and their bounds before the output's rounding.  Slopes: |gelu'| <= 1.13, |(g sigmoid(1.702 g))'| <= 1.1;
    the functions themselves are good to 2^-20 of their terms."""
    y, b = y.reshape(len(y), -1, 2, 8), b.reshape(len(b), -1, 2, 8)
    (g, u), (bg, bu) = (y[:, :, i].reshape(len(y), -1) for i in (0, 1)), (b[:, :, i].reshape(len(y), -1) for i in (0, 1))
    if act == "gelu":
        f = 0.5 * g * (1 + np.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)))
        return f * u, 1.13 * (np.abs(u) + bu) * bg + np.abs(f) * bu + 2.0 ** -20 * np.abs(g * u)
    g, u = np.minimum(g, LIMIT), np.clip(u, -LIMIT, LIMIT)
    f = g / (1 + np.exp(-1.702 * g))
    return f * (u + 1), 1.1 * (np.abs(u + 1) + bu) * bg + np.abs(f) * bu + 2.0 ** -20 * np.abs(g) * (np.abs(u) + 1)


def within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    worst = np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
    assert worst <= 1, f"{what}: {worst:.3g} times the bound at {np.unravel_index(np.argmax(np.abs(got - want) / np.maximum(bound, 1e-300)), want.shape)}"


def run(d, lin, x, m, cols, out="float32", act="none", pad=5):
    """Outputs [m, cols], with a guard of untouched columns behind them."""
    t = d.torch
    y = t.full((m + 1, cols + pad), 7.0, dtype=getattr(t, out), device=d.dev)
    t.cuda.synchronize()
    lin.run(x, m, y, ACTS[act], LIMIT)
    d.gpu.sync()
    assert d.gpu.device_status() == 0
    y = y.float().cpu().numpy()
    assert (y[:m, cols:] == 7.0).all() and (y[m] == 7.0).all(), "written outside the output"
    return y[:m, :cols]


# ---- layout and quantiser ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,k,group,experts", [(1, 64, 32, 1), (17, 128, 128, 1), (40, 192, 64, 3), (130, 1024, 128, 2), (16, 4160, 32, 1)])
def test_values_of_quants(lm, n, k, group, experts):
    d = device(lm)
    q, s, w = quants(rng(n + k), experts, n, k, group=group)
    lin = handle(d, q, s)
    assert np.array_equal(lin.values().cpu().numpy().astype(np.float64), w)
    assert lin.bytes() >= experts * n * k // 2
    lin.free()


def quantised(w, group):
    """The formula, operation by operation in f32: values [n, k]."""
    import torch

    v = torch.from_numpy(w).view(w.shape[0], -1, group)
    a = v.abs()
    first = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    top = v.gather(-1, first)[..., 0]
    s = (top / torch.tensor(-8.0)).bfloat16().float()
    q = torch.where(s[..., None] == 0, torch.tensor(8.0), (torch.round(v / s[..., None]) + 8).clamp(0, 15))
    out = torch.where(s[..., None] == 0, torch.zeros_like(v), (q - 8) * s[..., None])
    fine = torch.isfinite(v).all(-1)
    out[~fine] = float("nan")
    return out.reshape(w.shape).numpy()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantiser(lm, group):
    from peregrine_b200.layers import Linear4

    d = device(lm)
    g = rng(group)
    w = (g.standard_normal((37, 384)) * 0.02).astype(np.float32)
    w[3, :128] = 0.0                       # groups of zeros
    w[4] = np.abs(w[4])                    # all of one sign
    w[5, 7], w[5, 9] = 1.0, -1.0           # equal magnitudes: the first one is -8 steps
    w[6, 300] = np.inf
    w[7, 200] = np.nan
    w[8, :128] = np.arange(128) % 15 - 7.5   # ties of the rounding
    w[9] *= 1e-38
    w[10] *= 1e30
    x = bf16(d, w)
    lin = Linear4(d, x, group=group)
    got = lin.values().cpu().numpy()[0]
    want = quantised(x.float().cpu().numpy(), group)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # scales at the edge of the f32 range: a row's are kept over a power of two, which is exact
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    lin.free()


def test_rows_of_very_different_groups(lm):
    """Scales of a row within 2^21 of each other are exact; a group of 2^-30 beside one of 1 is off by 2^-36 of the larger one's scale at most."""
    import torch

    d = device(lm)
    q = np.full((16, 128), 15, np.uint8)
    s = np.ones((16, 2), np.float32)
    s[:, 1] = 2.0 ** -np.arange(15, 31)
    lin = handle(d, torch.from_numpy(q[:, 0::2] | q[:, 1::2] << 4), torch.from_numpy(s).bfloat16())
    got = lin.values().cpu().numpy()[0].astype(np.float64)
    want = 7 * np.repeat(s.astype(np.float64), 64, 1)
    assert np.array_equal(got[:7], want[:7])
    assert np.abs(got - want).max() <= 7 * 2.0 ** -36
    lin.free()


# ---- products --------------------------------------------------------------------------------------------------------
SHAPES = [(4, 64, 32), (24, 64, 64), (41, 192, 64), (200, 320, 32), (513, 576, 64), (48, 4224, 128), (40, 8960, 32), (1030, 128, 128), (2000, 1024, 64)]


@pytest.mark.parametrize("n,k,group", SHAPES)
def test_product(lm, n, k, group):
    d = device(lm)
    g = rng(n + k + group)
    q, s, w = quants(g, n, k, group=group)
    lin = handle(d, q, s)
    for m in (1, 2, 7, 8, 9, 16, 17, 32, 33, 64, 65, 129, 200, 300):
        x = bf16(d, g.standard_normal((m, k)))
        want, bound = sums(x.double().cpu().numpy(), w)
        within(run(d, lin, x, m, n), want, bound, f"m {m}")
        within(run(d, lin, x, m, n, "bfloat16"), want, bound + 2.0 ** -8 * (np.abs(want) + bound), f"m {m} bf16")
    lin.free()


@pytest.mark.parametrize("act", ["gelu", "swish"])
@pytest.mark.parametrize("n,k,group", [(16, 64, 32), (48, 192, 64), (528, 1024, 128), (176, 4608, 64)])
def test_gated(lm, n, k, group, act):
    d = device(lm)
    g = rng(n + k)
    q, s, w = quants(g, n, k, group=group)
    lin = handle(d, q, s)
    for m in (1, 8, 9, 16, 17, 63, 128, 250):
        x = bf16(d, g.standard_normal((m, k)) * 3)
        want, bound = gated(*sums(x.double().cpu().numpy(), w), act)
        within(run(d, lin, x, m, n // 2, "bfloat16", act), want, bound + 2.0 ** -8 * (np.abs(want) + bound) + 2.0 ** -134, f"m {m}")
    lin.free()


@pytest.mark.parametrize("m", [1, 5, 16, 40, 200])
def test_large_tiles_and_parts(lm, m):
    """Wide and long matrices: several rounds of tiles, K over several CTAs."""
    d = device(lm)
    for n, k, group in ((9000, 512, 128), (256, 16384, 64)):
        g = rng(m + n)
        q, s, w = quants(g, n, k, group=group)
        lin = handle(d, q, s)
        x = bf16(d, g.standard_normal((m, k)))
        want, bound = sums(x.double().cpu().numpy(), w)
        within(run(d, lin, x, m, n), want, bound, f"{n} {k}")
        lin.free()


@pytest.mark.parametrize("m,n,k", [(3, 12005, 8192), (8, 12005, 8192), (16, 16000, 4096), (11, 24000, 2048)])
def test_many_tiles_of_a_block(lm, m, n, k):
    """Several times more tiles than a block holds sums of at once, K in as many parts as it has warps; again with the same result."""
    d = device(lm)
    g = rng(m + n)
    q, s, w = quants(g, 1, n, k, group=64)
    lin = handle(d, q, s)
    x = bf16(d, g.standard_normal((m, k)))
    want, bound = sums(x.double().cpu().numpy(), w[0])
    first = run(d, lin, x, m, n)
    within(first, want, bound)
    for _ in range(3):
        assert np.array_equal(run(d, lin, x, m, n), first)
    lin.free()


@pytest.mark.parametrize("m", [3, 20])
def test_activations_of_any_size(lm, m):
    """Rows of the largest and smallest magnitudes; an infinity or a not-a-number stays in its row."""
    d = device(lm)
    k, n = 576, 70
    g = rng(m)
    q, s, w = quants(g, n, k, group=64)
    q = q & 0x77                            # (no quant of 8: no zero weight beside an infinity)
    w = ((np.stack([q.numpy() & 15, q.numpy() >> 4], -1).reshape(n, k).astype(np.float64) - 8).reshape(n, -1, 64) * s.double().numpy()[..., None]).reshape(n, k)
    lin = handle(d, q, s)
    a = g.standard_normal((m, k))
    a[0] *= 1e36
    a[1] *= 1e-36
    x = bf16(d, a)
    want, bound = sums(x.double().cpu().numpy(), w)
    within(run(d, lin, x, m, n), want, bound + 2.0 ** -149)
    clean = run(d, lin, x, m, n)
    a[1, 100], a[2, 5] = np.inf, np.nan
    a[1, 200] = 3e38
    y = run(d, lin, bf16(d, a), m, n)
    assert np.array_equal(y[0], clean[0]) and np.array_equal(y[3:], clean[3:])
    assert np.isnan(y[2]).all() and np.array_equal(y[1], np.sign(w[:, 100]) * np.inf)
    # channels that stand out by 2^20 leave the others' share exact
    a = g.standard_normal((m, k))
    a[:, ::50] *= 2.0 ** 20
    x = bf16(d, a)
    w0 = w.copy()
    want, bound = sums(x.double().cpu().numpy(), w0)
    within(run(d, lin, x, m, n), want, bound)
    lin.free()


def test_not_a_number_in_a_group(lm):
    from peregrine_b200.layers import Linear4

    d = device(lm)
    w = np.ones((20, 128), np.float32)
    w[3, 70] = np.nan
    lin = Linear4(d, bf16(d, w), group=64)
    for m in (2, 30):
        y = run(d, lin, bf16(d, np.ones((m, 128))), m, 20)
        assert np.isnan(y[:, 3]).all() and np.isfinite(np.delete(y, 3, 1)).all()
    lin.free()


def test_rows_apart(lm):
    d = device(lm)
    g = rng(5)
    n, k = 50, 128
    q, s, w = quants(g, n, k, group=32)
    lin = handle(d, q, s)
    for m in (1, 6, 16, 50):
        wide = bf16(d, g.standard_normal((m, k + 24)))
        x = wide[:, 8:8 + k]
        y = d.torch.zeros(m, n, device=d.dev)
        d.torch.cuda.synchronize()
        d.check(d.lib.pg_linear4_run(d.gpu.handle, lin.handle, x.data_ptr(), wide.stride(0), d.code, m, 0, 0.0, y.data_ptr(), 0, n))
        d.gpu.sync()
        want, bound = sums(x.double().cpu().numpy(), w)
        within(y.cpu().numpy(), want, bound, f"m {m}")
    lin.free()


def test_a_row_is_the_same_in_any_company(lm):
    """Rows do not meet in any sum: a row's outputs do not depend on what the others hold, to the last bit."""
    d = device(lm)
    g = rng(6)
    q, s, _ = quants(g, 300, 4608, group=64)
    lin = handle(d, q, s)
    for m in (2, 12, 40, 150):
        a = g.standard_normal((m, 4608))
        one = run(d, lin, bf16(d, a), m, 300)
        a[1:] = g.standard_normal((m - 1, 4608)) * 100
        assert np.array_equal(run(d, lin, bf16(d, a), m, 300)[0], one[0])
        assert np.array_equal(run(d, lin, bf16(d, a), m, 300), run(d, lin, bf16(d, a), m, 300))
    lin.free()


# ---- routes ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [1, 4, 16, 17, 90, 400])
@pytest.mark.parametrize("E,I,top,width,ff,group", [(6, 2, 3, 128, 64, 32), (3, 0, 1, 192, 128, 64), (40, 4, 6, 256, 192, 64), (2, 5, 2, 4224, 64, 64)])
def test_experts(lm, m, E, I, top, width, ff, group):
    """gate|up by token, down by row of the route; the pairs' outputs are picked up by the weighted sum of pg_routed_norm_add."""
    d = device(lm, m)
    t, lib, h = d.torch, d.lib, lm.handle
    g = rng(m + E + width)
    gu, down = quants(g, E, 2 * ff, width, group=group), quants(g, E, width, ff, group=group)
    a, b = handle(d, gu[0], gu[1]), handle(d, down[0], down[1])
    logits = t.from_numpy(g.standard_normal((m, E + I)).astype(np.float32)).to(d.dev)
    if m > 2:
        logits[:, 1] -= 30.0               # an expert without a token
    corr, ones = t.zeros(E + I, device=d.dev), t.ones(width, device=d.dev)
    x0 = t.from_numpy(g.standard_normal((m, width)).astype(np.float32)).to(d.dev)
    hx = x0.bfloat16()
    route = C.c_void_p()
    d.check(lib.pg_route_create(h, m, E, I, top, C.byref(route)))
    rows = lib.pg_route_max_rows(route)
    act, out = (t.full((rows, c), 3.0, dtype=t.bfloat16, device=d.dev) for c in (ff, width))
    x, hy = x0.clone(), t.zeros_like(hx)
    t.cuda.synchronize()
    d.check(lib.pg_route_run(h, route, d.code, logits.data_ptr(), E + I, m, corr.data_ptr(), 1, 1))
    a.run_routed(route, hx, True, act, 2, LIMIT)
    b.run_routed(route, act, False, out)
    d.check(lib.pg_routed_norm_add(h, route, out.data_ptr(), out.stride(0), x.data_ptr(), ones.data_ptr(), ones.data_ptr(), m, width, 1e-5, hy.data_ptr(), d.code, width))
    ids, w = np.zeros((m, top), np.int32), np.zeros((m, top), np.float32)
    d.check(lib.pg_route_read(h, route, ids.ctypes.data, w.ctypes.data))
    assert lm.device_status() == 0
    xs, y, bound = x0.double().cpu().numpy(), np.zeros((m, width)), np.zeros((m, width))
    for r in range(m):
        for e, wt in zip(ids[r], w[r].astype(np.float64)):
            if e >= E:
                y[r] += wt * xs[r]
                continue
            z, bz = gated(*sums(hx[r:r + 1].double().cpu().numpy(), gu[2][e]), "swish")
            o, bo = sums(z, down[2][e])
            # the activations are rounded to bf16 between the products, the outputs behind them
            bo = bo + (bz + 2.0 ** -8 * (np.abs(z) + bz)) @ np.abs(down[2][e]).T
            y[r] += wt * o[0]
            bound[r] += wt * (bo[0] + 2.0 ** -8 * (np.abs(o[0]) + bo[0]))
    # x += y / rms(y): the norm moves by the bound's rms at most
    rms = np.sqrt((y ** 2).mean(1, keepdims=True) + 1e-5)
    moved = np.sqrt((bound ** 2).mean(1, keepdims=True))
    within(x.cpu().numpy(), xs + y / rms, (bound + np.abs(y) * moved / rms) / rms * 1.05 + 2.0 ** -20 * (np.abs(xs) + np.abs(y / rms)), "x")
    d.check(lib.pg_route_free(h, route))
    a.free(), b.free()


def test_a_route_of_very_many_tiles(lm):
    """More tiles to a pair of blocks than are looked up beforehand.  All tokens are the same, so an expert's rows are all the same, bit for bit."""
    E, N, K, m = 2, 28800, 64, 16384
    d = device(lm, m)
    t, lib, h = d.torch, d.lib, lm.handle
    g = rng(77)
    q, s, w = quants(g, E, N, K, group=64)
    lin = handle(d, q, s)
    x = bf16(d, g.standard_normal((1, K))).expand(m, K).contiguous()
    logits = t.zeros(m, E, device=d.dev)
    logits[:, 0] = t.arange(m, device=d.dev) % 3 - 0.5        # one token in three goes to the second expert
    route = C.c_void_p()
    d.check(lib.pg_route_create(h, m, E, 0, 1, C.byref(route)))
    rows = lib.pg_route_max_rows(route)
    out = t.full((rows, N), 3.0, dtype=t.bfloat16, device=d.dev)
    corr = t.zeros(E, device=d.dev)
    t.cuda.synchronize()
    d.check(lib.pg_route_run(h, route, d.code, logits.data_ptr(), E, m, corr.data_ptr(), 1, 1))
    lin.run_routed(route, x, True, out)
    lm.sync()
    assert lm.device_status() == 0
    second = int((t.arange(m) % 3 == 0).sum())
    xs = x[:1].double().cpu().numpy()
    for e, n in ((0, m - second), (1, second)):
        want, bound = sums(xs, w[e])
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
        near = (out[:, :64].double().cpu().numpy() - want[:, :64]) / bound[:, :64]
        mine = np.nonzero((np.abs(near) <= 1).all(1))[0]
        assert len(mine) >= n                                 # (rows without a token may hold anything)
        one = out[int(mine[0])]
        within(one.float().cpu().numpy()[None], want, bound)
        assert int((out[t.from_numpy(mine).to(d.dev)] == one).all(1).sum()) >= n
    d.check(lib.pg_route_free(h, route))
    lin.free()


# ---- graphs, contexts, refusals --------------------------------------------------------------------------------------
def test_two_recordings_share_the_workspace(lm):
    """Products whose K goes over several CTAs, recorded twice, replayed in turn with other inputs, beside calls that are not recorded."""
    d = device(lm)
    g = rng(8)
    k, n = 8960, 200
    q, s, w = quants(g, n, k, group=64)
    lin = handle(d, q, s)
    t = d.torch
    cases = []
    for m in (3, 40):
        x, y = bf16(d, np.zeros((m, k))), t.zeros(m, n, device=d.dev)
        t.cuda.synchronize()
        lin.run(x, m, y)
        lm.sync()
        with lm.record() as graph:
            lin.run(x, m, y)
        cases.append((m, x, y, graph))
    for turn in range(3):
        for m, x, y, graph in cases:
            a = bf16(d, g.standard_normal((m, k)))
            x.copy_(a)
            t.cuda.synchronize()
            graph.launch()
            lm.sync()
            want, bound = sums(a.double().cpu().numpy(), w)
            within(y.cpu().numpy(), want, bound)
            within(run(d, lin, a, m, n), want, bound)
    for c in cases:
        c[3].free()
    lin.free()


def test_first_call_in_a_recording(lm):
    """The workspace is there when the handle is: nothing has to be run before recording."""
    from peregrine_b200.runtime import GpuContext

    ctx = GpuContext(component="lm")
    d = device(ctx)
    g = rng(9)
    q, s, w = quants(g, 300, 8960, group=64)
    lin = handle(d, q, s)
    for m in (2, 16, 24, 200):
        x, y = bf16(d, g.standard_normal((m, 8960))), d.torch.zeros(m, 300, device=d.dev)
        d.torch.cuda.synchronize()
        with ctx.record() as graph:
            lin.run(x, m, y)
        graph.launch()
        ctx.sync()
        want, bound = sums(x.double().cpu().numpy(), w)
        within(y.cpu().numpy(), want, bound, f"m {m}")
        graph.free()
    lin.free()
    ctx.close()


def test_weights_of_more_than_four_gigabytes(lm):
    """The last rows lie behind 2^32 bytes."""
    d = device(lm)
    t = d.torch
    n, k, last = (1 << 20) + 40, 8192, 72
    gen = t.Generator(device=d.dev).manual_seed(3)
    q = t.randint(0, 256, (n, k // 2), dtype=t.uint8, device=d.dev, generator=gen)
    s = t.full((n, k // 128), 0.01, dtype=t.bfloat16, device=d.dev)
    s[-last:] = (t.randn(last, k // 128, device=d.dev, generator=gen) * 0.02).bfloat16()
    from peregrine_b200.layers import Linear4

    lin = Linear4.from_quants(d, q, s)
    assert lin.bytes() > 1 << 32
    tail = q[-last:].cpu().numpy()
    w = np.stack([tail & 15, tail >> 4], -1).reshape(last, k).astype(np.float64) - 8
    w *= np.repeat(s[-last:].double().cpu().numpy(), 128, 1)
    del q
    for m in (1, 12, 40):
        x = bf16(d, rng(m).standard_normal((m, k)))
        y = t.zeros(m, n, device=d.dev)
        t.cuda.synchronize()
        lin.run(x, m, y)
        lm.sync()
        want, bound = sums(x.double().cpu().numpy(), w)
        within(y[:, -last:].cpu().numpy(), want, bound)
    lin.free()


def test_two_contexts_at_once(lm):
    """The same weights read from two streams."""
    from peregrine_b200.runtime import GpuContext

    other = GpuContext(component="lm")
    d, e = device(lm), device(other)
    g = rng(10)
    q, s, w = quants(g, 4000, 4224, group=64)
    lin = handle(d, q, s)
    mine = handle(e, q[:16], s[:16])        # (reserves the other context's workspace)
    a = [bf16(d, g.standard_normal((m, 4224))) for m in (8, 50)]
    ys = [[d.torch.zeros(len(x), 4000, device=d.dev) for x in a] for _ in range(2)]
    d.torch.cuda.synchronize()
    for _ in range(10):
        for c, y in ((lm, ys[0]), (other, ys[1])):
            for x, out in zip(a, y):
                c.check(c.lib.pg_linear4_run(c.handle, lin.handle, x.data_ptr(), 4224, 1, len(x), 0, 0.0, out.data_ptr(), 0, 4000))
    lm.sync(), other.sync()
    for i, x in enumerate(a):
        want, bound = sums(x.double().cpu().numpy(), w)
        within(ys[0][i].cpu().numpy(), want, bound)
        assert d.torch.equal(ys[0][i], ys[1][i])
    lin.free(), mine.free()
    other.close()


def test_refusals(lm):
    from peregrine_b200._lib import InvalidArgument

    d = device(lm)
    t = d.torch
    g = rng(11)
    q, s, _ = quants(g, 32, 128, group=64)
    lin = handle(d, q, s)
    x, y = bf16(d, np.zeros((4, 136))), t.zeros(4, 64, device=d.dev)
    h = C.c_void_p()

    def refused(f, *args):
        with pytest.raises(InvalidArgument):
            d.check(f(lm.handle, *args))

    p, ps = q.to(d.dev), s.to(d.dev)
    for n, k, group, e in ((32, 128, 16, 1), (32, 96, 32, 1), (32, 192, 128, 1), (0, 128, 64, 1), (32, 0, 64, 1), (32, 128, 64, 0), (32, 1 << 17, 64, 1)):
        refused(d.lib.pg_linear4_pack, p.data_ptr(), ps.data_ptr(), n, k, group, e, C.byref(h))
    refused(d.lib.pg_linear4_pack, p.data_ptr(), None, 32, 128, 64, 1, C.byref(h))
    refused(d.lib.pg_linear4_quantize, None, 32, 128, 64, 1, C.byref(h))
    run4 = d.lib.pg_linear4_run
    for args in ((None, x.data_ptr(), 128, 1, 4, 0, 0.0, y.data_ptr(), 0, 64), (lin.handle, None, 128, 1, 4, 0, 0.0, y.data_ptr(), 0, 64),
                 (lin.handle, x.data_ptr(), 128, 0, 4, 0, 0.0, y.data_ptr(), 0, 64),          # f32 activations
                 (lin.handle, x.data_ptr(), 120, 1, 4, 0, 0.0, y.data_ptr(), 0, 64),          # rows that overlap
                 (lin.handle, x.data_ptr(), 132, 1, 4, 0, 0.0, y.data_ptr(), 0, 64),          # rows that are not aligned
                 (lin.handle, x.data_ptr() + 2, 128, 1, 4, 0, 0.0, y.data_ptr(), 0, 64),
                 (lin.handle, x.data_ptr(), 128, 1, 4, 1, 0.0, y.data_ptr(), 0, 64),          # gated outputs are bf16
                 (lin.handle, x.data_ptr(), 128, 1, 4, 3, 0.0, y.data_ptr(), 1, 64), (lin.handle, x.data_ptr(), 128, 1, 4, 0, 0.0, y.data_ptr(), 2, 64),
                 (lin.handle, x.data_ptr(), 128, 1, 4, 0, 0.0, y.data_ptr(), 0, 31), (lin.handle, x.data_ptr(), 128, 1, -1, 0, 0.0, y.data_ptr(), 0, 64)):
        refused(run4, *args)
    d.check(run4(lm.handle, lin.handle, x.data_ptr(), 128, 1, 0, 0, 0.0, y.data_ptr(), 0, 64))   # no rows: nothing to do
    stack = handle(d, q.view(2, 16, 64), s.view(2, 16, 2))
    refused(run4, stack.handle, x.data_ptr(), 128, 1, 4, 0, 0.0, y.data_ptr(), 0, 64)            # a stack of experts needs a route
    route = C.c_void_p()
    d.check(d.lib.pg_route_create(lm.handle, 4, 3, 0, 1, C.byref(route)))
    refused(d.lib.pg_linear4_run_routed, stack.handle, route, x.data_ptr(), 1, 1, 0, 0.0, y.data_ptr(), 0, 64)
    d.check(d.lib.pg_route_free(lm.handle, route))
    with lm.record() as graph:
        refused(d.lib.pg_linear4_pack, p.data_ptr(), ps.data_ptr(), 32, 128, 64, 1, C.byref(h))
    graph.free()
    from peregrine_b200.layers import Linear4

    with pytest.raises(ValueError):
        Linear4.from_quants(d, p, ps[:16])
    with pytest.raises(ValueError):
        Linear4.from_quants(d, p.float(), ps)
    lin.free(), stack.free()
    lm.sync()
    assert lm.device_status() == 0
