"""Attention over a cache in 4 bits: longer portions held to what they compute in, f16.

Bounds as in tests/test_attention4_gpu.py, each sequence by the form that it takes.  Few tokens: queries f16 (2^-11), a probability times a value's scale
bf16 (2^-8).  Longer portions: queries f16, keys and values exact, probabilities f16 (2^-11), 2^-14 and less of them by a smallest half step, 2^-25; the
largest of a row enters as 2^7 at least, so that is 2^-32 of it."""
import math

import numpy as np
import pytest

from tests.test_attention4_gpu import Case, rng

pytestmark = pytest.mark.gpu
SMALLEST = 2.0 ** -32


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


def want(c, entries, proj):
    """The formula over what the cache holds now, and the bounds of its outputs, [rows, H, V]."""
    K, Vv = c.held()
    kw, H, G, D, V = c.kw, c.H, c.G, c.D, c.V
    chunk, sink = kw.get("chunk", 0), kw.get("sink", False)
    out, bound = np.zeros((len(proj), H, V)), np.zeros((len(proj), H, V))
    at = 0
    for slot, pos0, n in entries:
        half = n > c.plan.few
        for pos in range(pos0, pos0 + n):
            q = proj[at, :H * D].astype(np.float64).reshape(H, D)
            if kw.get("q_norm") is not None:
                q = q / np.sqrt((q ** 2).mean(1, keepdims=True) + kw["eps"]) * kw["q_norm"]
            coef, every = kw.get("temp", (0.0, 0.0))
            if every:
                q = q * (1 + coef * math.log(math.floor((pos + 1) / every) + 1))
            low = pos - pos % chunk if chunk else 0
            j = np.arange(low, pos + 1)
            rows = j % c.cap if chunk else j
            for h in range(H):
                k, v = K[slot, h // (H // G), rows], Vv[slot, h // (H // G), rows]
                z = c.scale * (k @ q[h])
                ds = abs(c.scale) * (np.abs(k) @ np.abs(q[h])).max() * (2.0 ** -11 + 2.0 ** -18)
                if kw.get("slopes") is not None:
                    z = z - float(kw["slopes"][h]) * (pos - j)
                    ds += 2.0 ** -22 * float(kw["slopes"][h]) * (pos - low)
                top = z.max()
                p = np.exp(z - top)
                l = p.sum() + (math.exp(min(-top, 700.0)) if sink else 0.0)
                out[at, h] = p @ v / l
                A = p @ np.abs(v) / l
                e = math.expm1(2 * ds)
                b = A * (e + (2.0 ** -11 if half else 2.0 ** -8) * (1 + e) + 2.0 ** -17)
                if half:
                    b = b + SMALLEST * np.abs(v).sum(0) / l * (1 + e)
                bound[at, h] = b + 2.0 ** -8 * (np.abs(out[at, h]) + b)
            at += 1
    return out, bound


def check(c, entries, proj, what=""):
    got = c.step(entries, proj).reshape(len(proj), c.H, c.V)
    out, bound = want(c, entries, proj)
    worst = np.abs(got - out) / np.maximum(bound, 1e-300)
    assert np.isfinite(got).all() and worst.max() <= 1, f"{what} {entries}: {worst.max():.3g} times the bound at {np.unravel_index(worst.argmax(), worst.shape)}"


@pytest.mark.parametrize("H,G,D,V", [(4, 2, 128, 128), (8, 8, 64, 64), (8, 1, 80, 96), (3, 3, 20, 40), (20, 1, 32, 64), (16, 2, 256, 256)])
def test_longer_portions(lm, H, G, D, V):
    c = Case(lm, H * D + V + 2, H, G, D, V, 500, 4, 400)
    c.append(1, 0, c.rows(33)), c.append(2, 0, c.rows(100)), c.append(3, 0, c.rows(499))
    n = c.plan.few + 1
    for entries in ([(0, 0, max(n, 150))], [(3, 499, 1), (1, 33, max(n, 130)), (2, 100, 1)], [(2, 101, n), (0, max(n, 150), min(2, c.plan.few))]):
        check(c, entries, c.rows(sum(e[2] for e in entries)))


@pytest.mark.parametrize("kw", [{"sink": True}, {"slopes": True}, {"norms": True}, {"temp": (0.3, 40.0)}, {"sink": True, "slopes": True, "norms": True, "temp": (0.1, 7.0)}])
def test_what_a_layer_may_have(lm, kw):
    H, G, D, V = 8, 2, 64, 96
    g = rng(4)
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = (2.0 ** -np.arange(1, H + 1)).astype(np.float32)
    if kw.pop("norms", False):
        kw.update(q_norm=(1 + 0.1 * g.standard_normal(D)).astype(np.float32), k_norm=(1 + 0.1 * g.standard_normal(D)).astype(np.float32), eps=1e-5)
    c = Case(lm, 4, H, G, D, V, 1200, 2, 400, **kw)
    c.append(0, 0, c.rows(1000)), c.append(1, 0, c.rows(60))
    check(c, [(0, 1000, 150), (1, 60, 150)], c.rows(300), str(sorted(kw)))


@pytest.mark.parametrize("chunk,rows", [(5, 8), (48, 64), (100, 400)])
def test_chunks(lm, chunk, rows):
    H, G, D, V = 4, 2, 64, 64
    positions = 40 * chunk
    cap = chunk * min((chunk + rows - 2) // chunk + 1, positions // chunk)
    c = Case(lm, chunk + 1, H, G, D, V, cap, 2, rows, chunk=chunk, positions=positions, slopes=(2.0 ** -np.arange(1, H + 1)).astype(np.float32))
    at = 0
    for n in (1, min(rows, chunk + 3), 1, min(rows, 7), min(rows, 2 * chunk), 1, min(rows, chunk), min(rows, 2 * chunk), 2):
        check(c, [(1, at, n)], c.rows(n), f"chunk {chunk}")
        at += n


@pytest.mark.parametrize("H,G,D,V", [(6, 2, 18, 10), (2, 1, 130, 7), (3, 1, 33, 250)])
def test_odd_widths(lm, H, G, D, V):
    c = Case(lm, D + V + 1, H, G, D, V, 333, 3, 300)
    c.append(1, 0, c.rows(33)), c.append(2, 0, c.rows(100))
    n = c.plan.few + 70
    entries = [(2, 100, n), (1, 33, 1), (0, 0, 2)]
    check(c, entries, c.rows(n + 3))


@pytest.mark.parametrize("H,G,D,V", [(4, 2, 128, 128), (8, 1, 80, 96), (6, 2, 18, 10), (4, 2, 160, 64)])
@pytest.mark.parametrize("kw", [{}, {"sink": True}, {"slopes": True}])
def test_many_small_probabilities_beside_a_large_one(lm, H, G, D, V, kw):
    """One position takes nearly all of the weight and its value is zero: what is left of an output is what hundreds of probabilities of about 2^-29 of
    the largest add up to."""
    kw = {k: (2.0 ** -np.arange(H, dtype=np.float32) * 1e-3 if k == "slopes" else v) for k, v in kw.items()}
    n = 150
    c = Case(lm, D + V, H, G, D, V, 500, 1, 400, **kw)
    before = c.rows(300)
    # keys: one column, -7 and 0 of its scale's steps; so a score is 20 (or a sink's 0) above the others'
    before[:, H * D:(H + G) * D] = 0.0
    before[17, H * D:(H + G) * D:D] = 1.0
    before[:, (H + G) * D:] = np.abs(before[:, (H + G) * D:]) + 1.0
    before[17, (H + G) * D:] = 0.0
    c.append(0, 0, before)
    proj = c.rows(n)
    proj[:, :H * D] = 0.0
    proj[:, :H * D:D] = 20.0 / c.scale
    proj[:, H * D:(H + G) * D] = 0.0
    proj[:, (H + G) * D:] = np.abs(proj[:, (H + G) * D:]) + 1.0
    check(c, [(0, 300, n)], proj)


@pytest.mark.parametrize("n", [1, 4, 150])
@pytest.mark.parametrize("keys", [1e35, 1e-35])
def test_keys_and_queries_of_opposite_sizes(lm, n, keys):
    """Scores up to a hundred from keys at one end of the range and queries at the other."""
    H, G, D, V = 8, 2, 64, 64
    c = Case(lm, n, H, G, D, V, 600, 2, 400)
    resize = lambda x: np.concatenate([x[:, :H * D] * 12 / keys, x[:, H * D:(H + G) * D] * keys, x[:, (H + G) * D:]], 1).astype(np.float32)
    c.append(0, 0, resize(c.rows(300)))
    check(c, [(0, 300, n)], resize(c.rows(n)))


@pytest.mark.parametrize("n", [1, 3, 150])
@pytest.mark.parametrize("at", [5, 40, 299, 300])
def test_a_value_that_is_not_finite_is_seen_however_small_its_weight(lm, n, at):
    """A position whose score is 300 below the others', with values that are not numbers: rows that see it say so, the others do not."""
    H, G, D, V = 4, 2, 64, 64
    c = Case(lm, n + at, H, G, D, V, 600, 1, 400)
    rows = c.rows(300 + n)
    rows[:, :(H + G) * D] = 0.0
    rows[:, :H * D:D] = 150.0 / c.scale
    rows[:, H * D:(H + G) * D:D] = 1.0
    rows[at, H * D:(H + G) * D:D] = -1.0
    rows[at, (H + G) * D + 40] = np.nan                       # head 0's value, columns 32 .. 63
    c.append(0, 0, rows[:300])
    bad = np.isnan(c.step([(0, 300, n)], rows[300:]).reshape(n, H, V))
    sees = 300 + np.arange(n) >= at
    assert (bad[:, :2, 32:] == sees[:, None, None]).all()
    assert not bad[:, :2, :32].any() and not bad[:, 2:].any()
