"""Weights and caches of 4 bits without a GPU: the library's refusals and sizes, and the options' checks."""
import ctypes as C

import pytest

from peregrine_b200 import _lib, registry


@pytest.fixture(scope="module")
def lib():
    from peregrine_b200.build import ensure_built

    ensure_built("lm")
    return _lib.load("lm")


def test_null_contexts_are_refused(lib):
    h, p, b = C.c_void_p(), _lib.PgAttention(), _lib.PgBatch()
    null = None
    calls = [lambda: lib.pg_linear4_pack(null, null, null, 16, 64, 64, 1, C.byref(h)),
             lambda: lib.pg_linear4_quantize(null, null, 16, 64, 64, 1, C.byref(h)),
             lambda: lib.pg_linear4_read(null, null, null),
             lambda: lib.pg_linear4_run(null, null, null, 64, _lib.BF16, 1, 0, 0.0, null, _lib.F32, 16),
             lambda: lib.pg_linear4_run_routed(null, null, null, null, _lib.BF16, 1, 0, 0.0, null, _lib.F32, 16),
             lambda: lib.pg_attention4_run(null, C.byref(p), C.byref(b), 1, 0, 0, null, 64, null, null, null, _lib.BF16, 64),
             lambda: lib.pg_attention4_prompt(null, C.byref(p), C.byref(b), 0, 1, 1, 0, null, null, null, null, _lib.BF16, 64),
             lambda: lib.pg_cache4_read(null, null, 0, 64, 64, 1, 1, null)]
    for i, call in enumerate(calls):
        assert call() == _lib.PG_ERR_INVALID, i
        assert b"null" in lib.pg_last_error(), i
    assert not h.value


def test_sizes(lib):
    # 16 positions of 32 columns: 256 bytes of quants, 32 of scales
    for width, positions, want in ((32, 16, 288), (1, 1, 288), (33, 16, 576), (128, 17, 2 * 1152), (256, 16, 2304), (0, 16, 0), (32, 0, 0), (-1, 4, 0)):
        assert lib.pg_cache4_bytes(width, positions) == want
    assert lib.pg_cache4_bytes(128, 1 << 40) == (1 << 40) // 16 * 1152
    p = _lib.PgAttention(8, 2, 64, 96, 1000, 1, 0.0, 1.0, 0.0, 0.0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    assert lib.pg_attention4_unfold_bytes(C.byref(p)) >= 2 * 1000 * (64 + 96) * 2
    assert lib.pg_attention4_unfold_bytes(None) == 0 and lib.pg_attention4_part_floats(None, C.byref(p)) == 0 and lib.pg_attention4_tickets(None) == 0
    assert lib.pg_linear4_bytes(None) == 0


@pytest.mark.parametrize("options", [{"weight_bits": 4}, {"cache_bits": 4}])
def test_a_model_without_them_refuses(tmp_path, monkeypatch, options):
    with pytest.raises(ValueError, match="4 bits"):
        registry._llama(str(tmp_path / "none"), **options)


def test_the_command_line_takes_16_and_4(capsys):
    from peregrine_b200.__main__ import main

    for flag in ("--weight-bits", "--cache-bits"):
        with pytest.raises(SystemExit):
            main(["generate", "--model", "none", "--max-new", "1", "--prompt", "1", flag, "8"])
        assert "invalid choice" in capsys.readouterr().err
