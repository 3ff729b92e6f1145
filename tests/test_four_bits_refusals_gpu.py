"""Pointers that the kernels of the 4-bit operators cannot read or write in whole words are refused on the host."""
import ctypes as C

import numpy as np
import pytest

from tests.test_attention4_gpu import Case
from tests.test_linear4_gpu import device, handle, quants, rng

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from peregrine_b200.runtime import GpuContext

    return GpuContext(component="lm")


def test_attention(lm):
    from peregrine_b200._lib import InvalidArgument

    c = Case(lm, 1, 4, 2, 64, 64, 64, 2, 64)
    d, p = c.d, c.plan.c
    t = d.torch
    x, out = t.zeros(5, c.width, device=d.dev), t.zeros(5, 256, dtype=t.bfloat16, device=d.dev)
    b = c.batch([(0, 0, 2), (1, 0, 2)], fixed=True)
    good = {"d_q": d.buffer("attn.q", c.plan.q_cols).data_ptr(), "d_part": d.buffer("attn4.part", 1, 1, t.float32).data_ptr(),
            "d_tickets": d.buffer("attn4.tickets", 1, 1, t.int32).data_ptr()}

    def go(few=4, rows=4, longest=2, proj=x.data_ptr(), o=out.data_ptr(), **fields):
        for k, v in {**good, **fields}.items():
            setattr(p, k, v)
        return d.lib.pg_attention4_run(lm.handle, C.byref(p), C.byref(b.c), few, rows, longest, proj, c.width, c.kc.data_ptr(), c.vc.data_ptr(), o, 1, 256)

    t.cuda.synchronize()
    for kw in ({"d_part": good["d_part"] + 4}, {"proj": x.data_ptr() + 2}, {"o": out.data_ptr() + 1}, {"few": 1, "rows": 0, "longest": 0, "d_q": good["d_q"] + 8}):
        with pytest.raises(InvalidArgument, match="aligned|boundary"):
            d.check(go(**kw))
    d.check(go(d_q=good["d_q"] + 8))          # (not used where nothing follows)
    d.check(go())
    with pytest.raises(InvalidArgument):
        d.check(d.lib.pg_cache4_read(lm.handle, c.kc.data_ptr(), 0, 64, 64, 4, 64, x.data_ptr() + 2))
    lm.sync()
    assert lm.device_status() == 0


def test_weights(lm):
    from peregrine_b200._lib import InvalidArgument

    d = device(lm)
    q, s, _ = quants(rng(2), 32, 128, group=64)
    lin, h = handle(d, q, s), C.c_void_p()
    q, s = q.to(d.dev), s.to(d.dev)
    out = d.torch.zeros(32, 130, device=d.dev)
    w = d.bf16(np.zeros((33, 128), np.float32))
    d.torch.cuda.synchronize()
    for call in (lambda: d.lib.pg_linear4_pack(lm.handle, q.data_ptr(), s.data_ptr() + 1, 16, 128, 64, 1, C.byref(h)),
                 lambda: d.lib.pg_linear4_quantize(lm.handle, w.data_ptr() + 1, 32, 128, 64, 1, C.byref(h)),
                 lambda: d.lib.pg_linear4_read(lm.handle, lin.handle, out.data_ptr() + 2)):
        with pytest.raises(InvalidArgument):
            d.check(call())
        assert not h.value
    lin.free()
