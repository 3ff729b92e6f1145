"""Attention over a cache in 4 bits (pg_attention4_*), on the GPU against the formula in 64 bits.

Bounds.  What the cache holds is read back, and the outputs are compared with attention over exactly that.  Few tokens: a query enters as f16
(half a step, 2^-11 of a value), so a score is off by ds <= 2^-11 scale sum |q k| and what the f32 sums lose (2^-18 of the same); a probability
times a value's scale is rounded to bf16 (2^-8).  With A = sum p |v| / l an output is off by A (2 ds + 2^-8) at most, and rounded once
(2^-8 of itself).  Longer portions: queries, keys and values are bf16 each, so ds <= 2 * 2^-8 scale sum |q k|, and A (2 ds + 2 * 2^-8)."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


def quantised(x):
    """The formula in f32: values [..., W], W a multiple of 32."""
    import torch

    v = torch.from_numpy(np.ascontiguousarray(x)).unflatten(-1, (-1, 32))
    a = v.abs()
    first = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    s = (v.gather(-1, first)[..., 0] / torch.tensor(-8.0)).bfloat16().float()[..., None]
    q = (torch.round(v / s) + 8).clamp(0, 15)
    return torch.where(s == 0, torch.zeros_like(v), (q - 8) * s).flatten(-2).numpy()


def padded(x, to=32):
    return np.pad(x, [(0, 0)] * (x.ndim - 1) + [(0, -x.shape[-1] % to)])


class Case:
    """Slots of random contexts and the plan over them."""

    def __init__(self, lm, seed, H, G, D, V, cap, slots, rows, **kw):
        from peregrine_b200.layers import Attention4Plan, Device

        self.lm, self.g = lm, rng(seed)
        d = self.d = Device(lm, "bfloat16", rows)
        t = d.torch
        self.H, self.G, self.D, self.V, self.cap, self.slots = H, G, D, V, cap, slots
        self.kw = kw
        dev = {k: (t.from_numpy(v).to(d.dev) if isinstance(v, np.ndarray) else v) for k, v in kw.items()}
        self.scale = dev.pop("scale", D ** -0.5)
        self.plan = Attention4Plan(d, H, G, D, V, cap, slots, slots, scale=self.scale, **dev)
        self.kc = t.zeros(slots, G, self.plan.key_bytes, dtype=t.uint8, device=d.dev)
        self.vc = t.zeros(slots, G, self.plan.value_bytes, dtype=t.uint8, device=d.dev)
        self.width = (H + G) * D + G * V
        t.cuda.synchronize()

    def rows(self, n):
        x = self.g.standard_normal((n, self.width)).astype(np.float32)
        x[:, :self.H * self.D] *= 1.5
        return x

    def batch(self, entries, **kw):
        """entries: (slot, first position, tokens)."""
        from peregrine_b200.layers import Batch

        return Batch(self.d, [(s, p, [0] * n) for s, p, n in entries], **kw)

    def append(self, slot, pos0, proj):
        """Only the keys and values, no attention."""
        d, c = self.d, self.plan.c
        t = d.torch
        for i in range(0, len(proj), d.rows):
            part = proj[i:i + d.rows]
            x = t.from_numpy(part).to(d.dev)
            b = self.batch([(slot, pos0 + i, len(part))])
            c.d_q, c.d_part, c.d_tickets = (d.buffer(*a).data_ptr() for a in (("attn.q", self.plan.q_cols), ("attn4.part", 1, 1, t.float32), ("attn4.tickets", 1, 1, t.int32)))
            t.cuda.synchronize()
            d.check(d.lib.pg_attention4_run(self.lm.handle, C.byref(c), C.byref(b.c), 0, 0, 0, x.data_ptr(), self.width, self.kc.data_ptr(), self.vc.data_ptr(), x.data_ptr(),
                                            1, 1 << 20))
            self.lm.sync()

    def step(self, entries, proj, pad=3):
        """Outputs [rows, H V] of a step."""
        d = self.d
        t = d.torch
        x = t.from_numpy(proj).to(d.dev)
        out = t.full((len(proj), (self.H * self.V + 7) // 8 * 8 + 8 * pad), 7.0, dtype=t.bfloat16, device=d.dev)
        b = self.batch(entries)
        t.cuda.synchronize()
        self.plan.run(b, x, self.kc, self.vc, out)
        self.lm.sync()
        assert self.lm.device_status() == 0
        out = out.float().cpu().numpy()
        assert (out[:, self.H * self.V:] == 7.0).all(), "written behind the rows"
        return out[:, :self.H * self.V]

    def held(self):
        return self.plan.values(self.kc, self.cap, False).double().cpu().numpy(), self.plan.values(self.vc, self.cap, True).double().cpu().numpy()

    def want(self, entries, proj, half=False):
        """The formula over what the cache holds now, and the bounds of its outputs.  half: longer portions as they are computed, in f16: queries and
        probabilities are off by half a step, 2^-11, keys and values not at all; a probability below 2^-14 of its row's largest by 2^-25 of that."""
        K, Vv = self.held()
        kw, H, G, D, V = self.kw, self.H, self.G, self.D, self.V
        chunk, sink = kw.get("chunk", 0), kw.get("sink", False)
        out, bound = np.zeros((len(proj), H, V)), np.zeros((len(proj), H, V))
        at = 0
        for slot, pos0, n in entries:
            few = n <= self.plan.few or half
            for i in range(n):
                pos = pos0 + i
                q = proj[at, :H * D].astype(np.float64).reshape(H, D)
                if kw.get("q_norm") is not None:
                    q = q / np.sqrt((q ** 2).mean(1, keepdims=True) + kw["eps"]) * kw["q_norm"]
                coef, every = kw.get("temp", (0.0, 0.0))
                if every:
                    q = q * (1 + coef * math.log(math.floor((pos + 1) / every) + 1))
                low = pos - pos % chunk if chunk else 0
                j = np.arange(low, pos + 1)
                rows = j % self.cap if chunk else j
                for h in range(H):
                    g = h // (H // G)
                    k, v = K[slot, g, rows], Vv[slot, g, rows]
                    z = self.scale * (k @ q[h])
                    ds = abs(self.scale) * (np.abs(k) @ np.abs(q[h])).max() * ((2.0 ** -11 if few else 2 * 2.0 ** -8 + 2.0 ** -16) + 2.0 ** -18)
                    if kw.get("slopes") is not None:
                        z = z - float(kw["slopes"][h]) * (pos - j)
                        ds += 2.0 ** -22 * float(kw["slopes"][h]) * (pos - low)
                    top = max(z.max(), 0.0) if sink else z.max()
                    p = np.exp(z - top)
                    l = p.sum() + (math.exp(-top) if sink else 0.0)
                    out[at, h] = p @ v / l
                    A = p @ np.abs(v) / l
                    e = math.expm1(2 * ds)
                    b = A * (e + (2.0 ** -11 if half else 2.0 ** -8 if few else 2 * 2.0 ** -8) * (1 + e) + 2.0 ** -17)
                    if half:
                        b = b + 2.0 ** -24 * np.abs(v).sum(0) * (1 + e)
                    bound[at, h] = b + 2.0 ** -8 * (np.abs(out[at, h]) + b)
                at += 1
        return out.reshape(len(proj), -1), bound.reshape(len(proj), -1)

    def run_and_check(self, entries, what=""):
        """A step's outputs, and that the cache holds the formula's values of its keys and values."""
        proj = self.rows(sum(e[2] for e in entries))
        got = self.step(entries, proj)
        want, bound = self.want(entries, proj)
        worst = np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
        assert np.isfinite(got).all() and worst <= 1, f"{what} {entries}: {worst:.3g} times the bound"
        return proj


# ---- append ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,V", [(128, 128), (64, 80), (20, 24), (256, 200)])
@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_append_holds_the_formula(lm, D, V, tokens):
    c = Case(lm, D + V + tokens, 4, 2, D, V, 100, 2, 64)
    kc0 = c.kc.clone()
    for pos in (0, 15, 33):
        proj = c.rows(tokens)
        proj[0, c.H * D:c.H * D + 8] = [0.5, -0.5, 1.5, 2.5, -3.5, 7.5, -7.5, 4.0]     # ties of the rounding
        proj[-1, c.H * D + D:] = 0.0                                                   # a head of zeros
        c.step([(1, pos, tokens)], proj)
        K, V_ = c.held()
        k = quantised(padded(proj[:, c.H * D:(c.H + c.G) * D].reshape(tokens, c.G, D)))[..., :D]
        v = quantised(padded(proj[:, (c.H + c.G) * D:].reshape(tokens, c.G, V)))[..., :V]
        assert np.array_equal(K[1, :, pos:pos + tokens], k.transpose(1, 0, 2)) and np.array_equal(V_[1, :, pos:pos + tokens], v.transpose(1, 0, 2))
        assert not K[0].any() and not K[1, :, pos + tokens:].any()                     # nobody else's rows
    assert c.d.torch.equal(c.kc[0], kc0[0])


def test_layout(lm):
    """Bytes and halves where the header says."""
    c = Case(lm, 5, 2, 1, 64, 96, 48, 1, 64)
    proj = c.rows(40)
    c.append(0, 0, proj)
    raw_k, raw_v = c.kc[0, 0].cpu().numpy(), c.vc[0, 0].cpu().numpy()
    K, V = c.held()
    for raw, held, W, values in ((raw_k, K[0, 0], 64, False), (raw_v, V[0, 0], 96, True)):
        gs, tile = W // 32, W * 9
        for p in (0, 5, 8, 15, 16, 27, 39):
            for col in (0, 3, 6, 9, 17, 30, 31, W - 1):
                at = p // 16 * tile
                x, g, s, cc = p % 16, col // 32, col % 32 // 16, col % 16
                if values:
                    byte, half = raw[at + g * 256 + ((cc % 8 * 4 + x % 8 // 2) * 2 + s) * 4 + 2 * (x % 2) + x // 8], cc // 8
                else:
                    byte, half = raw[at + g * 256 + ((x % 8 * 4 + cc // 4) * 2 + s) * 4 + 2 * (cc % 2) + x // 8], cc % 4 // 2
                sc = raw[at + gs * 256 + ((x // 2 * gs + g) * 2 + x % 2) * 2:][:2].copy().view(np.uint16).astype(np.uint32) << 16
                assert float(sc.view(np.float32)[0]) * ((int(byte) >> 4 * half & 15) - 8) == held[p, col]


def test_not_finite_stays_in_its_columns(lm):
    c = Case(lm, 6, 4, 2, 64, 64, 64, 2, 64)
    c.append(0, 0, c.rows(20)), c.append(1, 0, c.rows(20))
    proj = c.rows(2)
    proj[0, (c.H + c.G) * 64 + 40] = np.inf           # head 0's value, columns 32 .. 63
    got = c.step([(0, 20, 1), (1, 20, 1)], proj)
    bad = np.isnan(got).reshape(2, 4, 64)
    assert bad[0, :2, 32:].all() and not bad[0, :2, :32].any() and not bad[0, 2:].any() and not bad[1].any()
    # what a row does not see does not touch it, whatever it holds
    proj = c.rows(3)
    proj[2, c.H * 64:] = np.nan
    got = c.step([(1, 21, 3)], proj).reshape(3, 4, 64)
    assert np.isfinite(got[:2]).all() and np.isnan(got[2]).all()
    # a slot that changes hands holds the other sequence's positions behind the new one's end
    got = c.step([(1, 5, 1)], c.rows(1))
    assert np.isfinite(got).all()


# ---- attention ---------------------------------------------------------------------------------------------------------
SHAPES = [(4, 2, 128, 128), (8, 8, 64, 64), (8, 1, 80, 96), (3, 3, 20, 40), (20, 1, 32, 64), (16, 2, 256, 256), (32, 2, 128, 64), (2, 1, 160, 24)]


@pytest.mark.parametrize("H,G,D,V", SHAPES)
def test_single_tokens(lm, H, G, D, V):
    c = Case(lm, H * D + V, H, G, D, V, 700, 5, 64)
    for s, n in enumerate((0, 1, 15, 300, 699)):
        if n:
            c.append(s, 0, c.rows(n))
    c.run_and_check([(0, 0, 1)])
    c.run_and_check([(4, 699, 1), (2, 15, 1), (1, 1, 1), (0, 1, 1), (3, 300, 1)])
    for pos in range(16, 34):
        c.run_and_check([(2, pos, 1), (0, pos - 14, 1)])


@pytest.mark.parametrize("H,G,D,V", SHAPES)
@pytest.mark.parametrize("n", [2, 5, 16])
def test_few_tokens(lm, H, G, D, V, n):
    c = Case(lm, H * D + V + n, H, G, D, V, 400, 3, 64)
    c.append(1, 0, c.rows(17)), c.append(2, 0, c.rows(301))
    c.run_and_check([(0, 0, n)])
    c.run_and_check([(2, 301, n), (1, 17, 1), (0, n, 2)])
    c.run_and_check([(1, 18, n), (2, 301 + n, n)])


@pytest.mark.parametrize("H,G,D,V", SHAPES[:5] + [(16, 2, 256, 256)])
def test_longer_portions(lm, H, G, D, V):
    c = Case(lm, H * D + V, H, G, D, V, 500, 4, 400)
    c.append(1, 0, c.rows(33)), c.append(2, 0, c.rows(100)), c.append(3, 0, c.rows(499))
    n = c.plan.few + 1
    c.run_and_check([(0, 0, max(n, 150))])
    # longer and shorter ones and single tokens in one step
    c.run_and_check([(3, 499, 1), (1, 33, max(n, 130)), (2, 100, 1)])
    c.run_and_check([(2, 101, n), (0, max(n, 150), min(2, c.plan.few))])


@pytest.mark.parametrize("H,G,D,V", SHAPES)
@pytest.mark.parametrize("sink", [False, True])
def test_longer_portions_keep_their_digits(lm, H, G, D, V, sink):
    """Scores of a wide range, keys and values of positions (and a head's from another's) that are thousands of times larger than the rest."""
    c = Case(lm, H * D + V + 1, H, G, D, V, 300, 2, 400, sink=sink)
    before = c.rows(60)
    before[17, H * D:] *= 3000.0
    before[40] *= 1e-3
    c.append(1, 0, before)
    n = max(c.plan.few + 1, 140)
    proj = c.rows(2 * n)
    proj[:, :H * D] *= 4.0
    proj[:, H * D:H * D + D] *= 1e-6
    proj[5], proj[7] = 0.0, proj[7] * 1e-12
    entries = [(1, 60, n), (0, 0, n)]
    got = c.step(entries, proj)
    want, bound = c.want(entries, proj, half=True)
    got = got.reshape(want.shape)
    assert np.isfinite(got).all()
    worst = np.abs(got - want) / np.maximum(bound, 1e-300)
    assert worst.max() <= 1, f"{worst.max():.3g} times the bound at {np.unravel_index(worst.argmax(), worst.shape)}"


@pytest.mark.parametrize("kw,D,V", [({}, 64, 96), ({}, 160, 64), ({"chunk": 50, "positions": 300}, 64, 96), ({"chunk": 40, "positions": 240}, 64, 256)])
def test_longer_portions_beside_what_is_not_finite(lm, kw, D, V):
    """Values (32 columns) and keys that are not numbers are seen by the rows that see their positions, and by no others."""
    H, G, n = 4, 2, 170
    cap = kw["chunk"] * -(-300 // kw["chunk"]) if kw else 300
    c = Case(lm, 12, H, G, D, V, cap, 2, 400, **kw)
    c.append(1, 0, c.rows(20))
    proj = c.rows(n)
    for at, what in ((30, np.inf), (90, np.nan), (133, -np.inf)):
        proj[at, (H + G) * D + 40] = what                                 # head 0's value, columns 32 .. 63
    proj[120, H * D + D + 3] = np.nan                                     # head 1's key
    got = c.step([(1, 20, n)], proj).reshape(n, H, V)
    bad = np.isnan(got)
    pos, chunk = 20 + np.arange(n), kw.get("chunk", 1 << 30)
    sees = lambda at: (pos >= 20 + at) & (pos // chunk == (20 + at) // chunk)
    value = sees(30) | sees(90) | sees(133)
    assert (bad[:, :2, 32:64] == value[:, None, None]).all()
    assert not bad[:, :2, :32].any() and not bad[:, :2, 64:].any()
    assert (bad[:, 2:] == sees(120)[:, None, None]).all()


@pytest.mark.parametrize("kw", [{"sink": True}, {"slopes": True}, {"norms": True}, {"temp": (0.3, 40.0)}, {"sink": True, "slopes": True, "norms": True, "temp": (0.1, 7.0)}])
@pytest.mark.parametrize("n", [1, 4, 150])
def test_what_a_layer_may_have(lm, kw, n):
    H, G, D, V = 8, 2, 64, 96
    g = rng(3)
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = (2.0 ** -np.arange(1, H + 1)).astype(np.float32)
    if kw.pop("norms", False):
        kw.update(q_norm=(1 + 0.1 * g.standard_normal(D)).astype(np.float32), k_norm=(1 + 0.1 * g.standard_normal(D)).astype(np.float32), eps=1e-5)
    c = Case(lm, n, H, G, D, V, 1200, 2, 400, **kw)
    c.append(0, 0, c.rows(1000)), c.append(1, 0, c.rows(60))
    proj = c.run_and_check([(0, 1000, n), (1, 60, n)], str(sorted(kw)))
    if "k_norm" in kw:
        # held to half a step of the normalised key (a step on the side that has one level less)
        k = proj[:, H * D:(H + G) * D].astype(np.float64).reshape(-1, G, D)
        k = k / np.sqrt((k ** 2).mean(-1, keepdims=True) + 1e-5) * kw["k_norm"]
        K = c.held()[0]
        got = np.concatenate([K[0, :, 1000:1000 + n], K[1, :, 60:60 + n]], 1).transpose(1, 0, 2)
        step = np.abs(k).reshape(-1, G, 2, 32).max(-1, keepdims=True) / 8 * (1 + 2.0 ** -8)
        off = np.abs(got - k).reshape(-1, G, 2, 32)
        assert (off <= step * (1 + 2.0 ** -6)).all() and np.median(off / step) < 0.51


@pytest.mark.parametrize("chunk,rows", [(5, 8), (48, 64), (100, 400)])
def test_chunks(lm, chunk, rows):
    """A ring of whole chunks: single tokens, portions that end inside a chunk, and turns of the ring."""
    H, G, D, V = 4, 2, 64, 64
    positions = 40 * chunk
    cap = chunk * min((chunk + rows - 2) // chunk + 1, positions // chunk)
    c = Case(lm, chunk, H, G, D, V, cap, 2, rows, chunk=chunk, positions=positions, slopes=(2.0 ** -np.arange(1, H + 1)).astype(np.float32))
    at = [0, 0]
    for n in (1, 1, min(rows, chunk + 3), 1, 1, min(rows, 7), min(rows, 2 * chunk), 1, 1):
        c.run_and_check([(1, at[1], n)], f"chunk {chunk}")
        at[1] += n
    while at[1] < 3 * cap + 2:
        n = min(rows, max(1, chunk // 3))
        c.run_and_check([(1, at[1], n)], f"chunk {chunk}")
        at[1] += n
    c.run_and_check([(0, 0, 1), (1, at[1], 1)])


def test_slices(lm):
    """Long contexts in many slices, few and many of them, and slices that hold nothing that an early token sees."""
    c = Case(lm, 9, 8, 2, 64, 64, 9000, 3, 1024, sink=True)
    c.append(0, 0, c.rows(8997)), c.append(1, 0, c.rows(4095)), c.append(2, 0, c.rows(255))
    c.run_and_check([(0, 8997, 1)])
    c.run_and_check([(2, 255, 1), (0, 8998, 1), (1, 4095, 1)])
    c.run_and_check([(1, 4096, 3), (2, 256, 2)])
    assert not c.d.buffer("attn4.tickets", 1, 1, c.d.torch.int32).any()


@pytest.mark.parametrize("H,G,D,V,kw", [(8, 2, 64, 64, {}), (16, 2, 128, 96, {"sink": True}), (4, 1, 64, 64, {"chunk": 1500, "positions": 6000})])
def test_slices_of_unequal_contexts(lm, H, G, D, V, kw):
    """Slices are dealt out over the sequences of a step: one long context among short ones, new ones, all equal, more sequences than a warp has lanes,
    a longer portion and a sequence outside its cache among them."""
    kw = dict(kw)
    if kw.get("chunk"):
        kw["slopes"] = (2.0 ** -np.arange(1, H + 1)).astype(np.float32)
    cap = 6000
    c = Case(lm, H + D, H, G, D, V, cap, 40, 256, **kw)
    lens = [5800, 0, 1, 700, 256, 255, 31, 2600]
    for s, n in enumerate(lens):
        if n:
            c.append(s, 0, c.rows(n))
    at = list(lens) + [0] * 32
    for slots in ([0], [7, 0], [1, 2], list(range(8)), [6, 5, 4, 3, 2, 1, 0], list(range(40)), [3, 0, 39, 38, 1]):
        c.run_and_check([(s, at[s], 1) for s in slots], str(kw))
        for s in slots:
            at[s] += 1
    if not kw.get("chunk"):
        few = min(3, c.plan.few)
        c.run_and_check([(0, at[0], few), (2, at[2], 1), (7, at[7], 1), (1, at[1], c.plan.few + 60)], "mixed")
        at[0], at[2], at[7] = at[0] + few, at[2] + 1, at[7] + 1
    # a sequence outside its cache is reported and the others are as ever
    d = c.d
    proj = c.rows(3)
    got = None
    x, out = d.torch.from_numpy(proj).to(d.dev), d.torch.full((3, (H * V + 7) // 8 * 8), 7.0, dtype=d.torch.bfloat16, device=d.dev)
    entries = [(0, at[0], 1), (5, cap, 1), (7, at[7], 1)]
    b = c.batch(entries)
    d.torch.cuda.synchronize()
    c.plan.run(b, x, c.kc, c.vc, out)
    lm.sync()
    assert lm.device_status() != 0
    got = out.float().cpu().numpy()[:, :H * V]
    want, bound = c.want([entries[0], entries[2]], proj[[0, 2]])
    assert (np.abs(got[[0, 2]] - want) <= bound).all() and (got[1] == 7.0).all()
    assert not d.buffer("attn4.tickets", 1, 1, d.torch.int32).any()


def test_positions_outside_the_cache(lm):
    """Recorded as a status, nothing written; the next call is as good as ever."""
    c = Case(lm, 11, 4, 2, 64, 64, 64, 2, 64)
    c.append(0, 0, c.rows(60)), c.append(1, 0, c.rows(20))
    for n in (1, 3):
        kc, vc = c.kc.clone(), c.vc.clone()
        t = c.d.torch
        x, out = t.from_numpy(c.rows(n + 1)).to(c.d.dev), t.full((n + 1, 256), 7.0, dtype=t.bfloat16, device=c.d.dev)
        b = c.batch([(0, 65 - n, n), (1, 20, 1)])
        t.cuda.synchronize()
        c.plan.run(b, x, c.kc, c.vc, out)
        c.lm.sync()
        assert c.lm.device_status() == -1
        assert (out[:n] == 7.0).all() and (out[n] != 7.0).all()
        if n == 1:
            assert t.equal(kc[0], c.kc[0]) and t.equal(vc[0], c.vc[0])
        c.append(1, 20, c.rows(1))
    c.run_and_check([(1, 21, 1)])


def test_rows_do_not_depend_on_their_company(lm):
    c = Case(lm, 12, 8, 2, 128, 128, 2100, 4, 64)
    for s in range(4):
        c.append(s, 0, c.rows(500 * s + 300))
    proj = c.rows(4)
    entries = [(s, 500 * s + 300, 1) for s in range(4)]
    a = c.step(entries, proj)
    assert np.array_equal(a, c.step(entries, proj))              # appended again, the same
    proj2 = c.rows(4)
    proj2[2] = proj[2]
    assert np.array_equal(c.step(entries, proj2)[2], a[2])


@pytest.mark.parametrize("H,G,D,V", [(6, 2, 18, 10), (2, 1, 130, 7), (3, 1, 33, 250)])
def test_odd_widths(lm, H, G, D, V):
    """Rows that are no whole 16-byte words, widths of which the last 32 columns are partly there."""
    c = Case(lm, D + V, H, G, D, V, 333, 3, 300)
    c.append(1, 0, c.rows(33)), c.append(2, 0, c.rows(100))
    c.run_and_check([(0, 0, 1), (1, 33, 1), (2, 100, 1)])
    c.run_and_check([(0, 1, 3), (2, 101, 2)])
    n = c.plan.few + 70
    c.run_and_check([(2, 103, n), (1, 34, 1)])


def test_a_recorded_longer_portion(lm):
    """A portion of 150 tokens recorded once, replayed over other rows of the projection."""
    c = Case(lm, 15, 8, 2, 64, 96, 700, 2, 400, sink=True)
    t = c.d.torch
    c.append(1, 0, c.rows(200))
    entries = [(1, 200, 150), (0, 0, 2)]
    b = c.batch(entries, fixed=True)
    x, out = t.zeros(152, c.width, device=c.d.dev), t.zeros(152, c.H * c.V, dtype=t.bfloat16, device=c.d.dev)
    t.cuda.synchronize()
    with lm.record() as g:
        c.plan.run(b, x, c.kc, c.vc, out)
    for _ in range(3):
        proj = c.rows(152)
        x.copy_(t.from_numpy(proj).to(c.d.dev))
        t.cuda.synchronize()
        g.launch()
        lm.sync()
        want, bound = c.want(entries, proj)
        assert (np.abs(out.float().cpu().numpy() - want) <= bound).all()
    g.free()
    assert lm.device_status() == 0


def test_two_contexts_at_once(lm):
    """Steps on two contexts' streams, each with its caches and workspaces."""
    from peregrine_b200.runtime import GpuContext

    other = GpuContext(component="lm")
    cases = [Case(c, 16, 8, 2, 128, 64, 1200, 3, 300) for c in (lm, other)]
    t = cases[0].d.torch
    for c in cases:
        c.append(0, 0, c.rows(1000)), c.append(1, 0, c.rows(31))
    entries = [(0, 1000, 1), (1, 31, 1), (2, 0, 150)]
    work = []
    for c in cases:
        proj = c.rows(152)
        x, out = t.from_numpy(proj).to(c.d.dev), t.zeros(152, c.H * c.V, dtype=t.bfloat16, device=c.d.dev)
        work.append((c, proj, x, out, c.batch(entries)))
    t.cuda.synchronize()
    for _ in range(10):
        for c, _proj, x, out, b in work:
            c.plan.run(b, x, c.kc, c.vc, out)
    lm.sync(), other.sync()
    for c, proj, x, out, b in work:
        want, bound = c.want(entries, proj)
        assert (np.abs(out.float().cpu().numpy() - want) <= bound).all()
    other.close()


def test_a_cache_of_more_than_four_gigabytes(lm):
    """Slots whose keys and values lie behind 2^32 bytes: a prompt, few and single tokens in the last of them, beside the first."""
    H, G, D, V, cap, slots = 16, 8, 128, 128, 60000, 140
    c = Case(lm, 14, H, G, D, V, cap, slots, 256)
    assert c.kc.numel() > 1 << 32
    c.held = lambda: _first_rows(c, 400)
    c.run_and_check([(139, 0, 150)])
    c.run_and_check([(139, 150, 3), (0, 0, 2)])
    c.run_and_check([(0, 2, 1), (139, 153, 1)])


def _first_rows(c, rows):
    """What the first rows of the first and the last slot hold; nothing of the others."""
    out = []
    for cache, values, width in ((c.kc, False, c.D), (c.vc, True, c.V)):
        full = np.zeros((c.slots, c.G, rows, width))
        for s in (0, c.slots - 1):
            full[s] = c.plan.values(cache[s:s + 1], rows, values)[0].double().cpu().numpy()
        out.append(full)
    return out


def test_recorded_steps(lm):
    """Two recordings over one plan's workspaces, replayed in turn with other positions and rows."""
    c = Case(lm, 13, 8, 2, 128, 128, 3000, 3, 64, sink=True)
    t = c.d.torch
    for s in range(3):
        c.append(s, 0, c.rows(2000 + 50 * s))
    made = []
    for entries in ([(0, 2000, 1), (2, 2100, 1)], [(1, 2050, 2)]):
        n = sum(e[2] for e in entries)
        b = c.batch(entries, fixed=True)
        x, out = t.zeros(n, c.width, device=c.d.dev), t.zeros(n, c.H * c.V, dtype=t.bfloat16, device=c.d.dev)
        t.cuda.synchronize()
        with lm.record() as g:
            c.plan.run(b, x, c.kc, c.vc, out)
        made.append((entries, b, x, out, g))
    for turn in range(3):
        for entries, b, x, out, g in made:
            now = [(s, p + turn * n, n) for s, p, n in entries]
            proj = c.rows(sum(e[2] for e in now))
            x.copy_(t.from_numpy(proj).to(c.d.dev))
            n = b.rows
            host = np.zeros(3 * n + 2 * b.seqs + 1, np.int32)
            at = 0
            for i, (s, p, k) in enumerate(now):
                host[n + at:n + at + k], host[2 * n + at:2 * n + at + k] = np.arange(p, p + k), i
                at += k
                host[3 * n + i + 1], host[3 * n + b.seqs + 1 + i] = at, s
            t.cuda.synchronize()
            b.write(host)
            g.launch()
            lm.sync()
            want, bound = c.want(now, proj)
            assert (np.abs(out.float().cpu().numpy() - want) <= bound).all()
    for m in made:
        m[4].free()
    assert lm.device_status() == 0


def test_refusals(lm):
    from peregrine_b200._lib import InvalidArgument
    from peregrine_b200.layers import Attention4Plan, Device

    c = Case(lm, 14, 4, 2, 64, 64, 64, 2, 64)
    d, p = c.d, c.plan.c
    t = d.torch
    x, out = t.zeros(4, c.width, device=d.dev), t.zeros(4, 256, dtype=t.bfloat16, device=d.dev)
    b = c.batch([(0, 0, 2), (1, 0, 2)], fixed=True)
    p.d_q, p.d_part, p.d_tickets = (d.buffer(*a).data_ptr() for a in (("attn.q", c.plan.q_cols), ("attn4.part", 1, 1, t.float32), ("attn4.tickets", 1, 1, t.int32)))
    run, prompt = d.lib.pg_attention4_run, d.lib.pg_attention4_prompt
    work = d.buffer("attn4.work", 1, 1)

    def go(few=4, rows=4, longest=2, proj=x.data_ptr(), ldp=c.width, kc=c.kc.data_ptr(), vc=c.vc.data_ptr(), o=out.data_ptr(), dtype=1, ldo=256):
        return run(lm.handle, C.byref(p), C.byref(b.c), few, rows, longest, proj, ldp, kc, vc, o, dtype, ldo)

    d.check(go())
    for kw in ({"dtype": 0}, {"ldp": c.width - 1}, {"ldo": 255}, {"proj": None}, {"kc": None}, {"o": None}, {"kc": c.kc.data_ptr() + 8}, {"few": -1}, {"rows": 5}, {"rows": 0},
               {"longest": 5}, {"longest": 0}):
        with pytest.raises(InvalidArgument):
            d.check(go(**kw))
    for field, bad in (("heads", 3), ("dim", 257), ("vdim", 0), ("cap", 0), ("slots", 0), ("positions", 65), ("chunk", 5), ("chunk", 32)):
        old = getattr(p, field)
        setattr(p, field, bad)
        with pytest.raises(InvalidArgument):
            d.check(go())
        setattr(p, field, old)
    for args in ((2, 2, 2, 0), (-1, 2, 2, 0), (0, 0, 2, 0), (0, 3, 3, 0), (0, 2, 1, 0), (0, 2, 65, 0), (0, 2, 2, 2), (0, 2, 2, -1)):
        with pytest.raises(InvalidArgument):
            d.check(prompt(lm.handle, C.byref(p), C.byref(b.c), *args, c.kc.data_ptr(), c.vc.data_ptr(), work.data_ptr(), out.data_ptr(), 1, 256))
    with pytest.raises(InvalidArgument):
        d.check(prompt(lm.handle, C.byref(p), C.byref(b.c), 0, 2, 2, 0, c.kc.data_ptr(), c.vc.data_ptr(), work.data_ptr() + 64, out.data_ptr(), 1, 256))
    with pytest.raises(InvalidArgument):
        d.check(d.lib.pg_cache4_read(lm.handle, c.kc.data_ptr(), 0, 64, 64, 4, 65, x.data_ptr()))
    with pytest.raises(ValueError):
        Attention4Plan(Device(lm, "float32", 4), 4, 2, 64, 64, 64, 2, 2, scale=1.0)
    lm.sync()
    assert lm.device_status() == 0
