"""The attention path's operators without a GPU: the references against their definitions, and every refusal of the C
ABI (arguments are checked on the host before anything is launched)."""
import numpy as np
import pytest

import q4_ref
from kore_amd import _lib

P = 0x100000  # fake, never dereferenced
M = 1 << 20
NULL, DIM, OVER, ALIAS = (_lib.KORE_HIP_ERR_NULL_PTR, _lib.KORE_HIP_ERR_BAD_DIM, _lib.KORE_HIP_ERR_OVERFLOW,
                          _lib.KORE_HIP_ERR_ALIAS)


# ---------------------------------------------------------------- references
def test_quantise_is_the_nearest_value():
    x = np.random.default_rng(0).standard_normal((64, 96)).astype(np.float32) * 10.0
    codes, scales = q4_ref.quantise(x)
    got = q4_ref.values(codes, scales, 96)
    step = np.repeat(2.0 ** (scales.astype(np.float64) - 127), 32, -1)
    grid = np.concatenate([q4_ref.MAGNITUDES, -q4_ref.MAGNITUDES])
    best = np.abs(x[..., None] - step[..., None] * grid).min(-1)
    assert (np.abs(got - x) == best).all()
    amax = np.abs(x).reshape(64, 3, 32).max(-1)
    s = 2.0 ** (scales.astype(np.float64) - 127)
    assert (amax <= 7 * s).all() and (amax > 3.5 * s).all()


def test_quantise_ties_and_special_blocks():
    x = np.zeros((8, 32), np.float32)
    x[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0]
    x[1, :2] = [7.0, 6.9]
    x[2, 0] = np.float32(7.0000005)
    x[3, 0] = np.inf
    x[4, 3] = np.nan
    x[5, 0] = np.float32(3.4e38)
    x[6, 0] = 2.0 ** -140
    codes, scales = q4_ref.quantise(x)
    v = q4_ref.values(codes, scales, 32)
    assert v[0, :9].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -4] and scales[0, 0] == 127
    assert v[1, :2].tolist() == [6, 6]
    assert scales[2, 0] == 128 and v[2, 0] == 8  # 3.5 units: a tie, the even code
    assert np.isnan(v[3]).all() and np.isnan(v[4]).all()
    assert v[5, 0] == 3 * 2.0 ** 126 and scales[5, 0] == 253
    assert v[6, 0] == 0 and scales[6, 0] == 27
    assert scales[7, 0] == 27 and (codes[7] == 0).all()


@pytest.mark.parametrize("page,d", [(16, 32), (16, 128), (64, 80), (32, 256)])
def test_layout_has_every_byte_once(page, d):
    used = np.concatenate([np.concatenate(q4_ref.places(page, d, t, v)) for v in (False, True) for t in range(page)])
    assert sorted(used.tolist()) == list(range(page * q4_ref.blocks(d) * 34))


def test_backward_formula_against_differences():
    r = np.random.default_rng(3)
    t, h, d = 3, 2, 12
    x, dy, w = r.standard_normal((t, h, d)), r.standard_normal((t, h, d)), r.standard_normal(d) + 1.0
    pos, inv = np.array([0, 5, 1000]), 1.0 / 10000.0 ** (np.arange(d // 2) * 2 / d)
    for inter in (False, True):
        dx, dw, _, _ = q4_ref.qk_norm_rope_backward(dy, x, w, pos, inv, 1e-3, inter)

        def f(xx, ww):
            return (q4_ref.qk_norm_rope(xx, ww, pos, inv, 1e-3, inter)[0] * dy).sum()

        eps = 1e-5
        for i in np.ndindex(t, h, d):
            e = np.zeros_like(x)
            e[i] = eps
            assert abs((f(x + e, w) - f(x - e, w)) / (2 * eps) - dx[i]) < 1e-7
        for i in range(d):
            e = np.zeros(d)
            e[i] = eps
            assert abs((f(x, w + e) - f(x, w - e)) / (2 * eps) - dw[i]) < 1e-7


# ------------------------------------------------------------------- refusals
def norm_rope(q=P, k=P + M, qw=P + 8 * M, kw=P + 8 * M, inv=P + 9 * M, pos=None, qo=P + 2 * M, ko=P + 3 * M, batch=2, seq=3,
              hq=4, hk=2, d=64, qs=0, ks=0, qos=0, kos=0, start=0):
    return _lib.load().kore_hip_qk_norm_rope_f32(q, k, qw, kw, inv, pos, qo, ko, batch, seq, hq, hk, d, qs, ks, qos, kos,
                                                 start, 1e-6, 0, None)


def test_norm_rope_refusals():
    assert norm_rope(batch=0, q=None) == 0 and norm_rope(d=0) == 0 and norm_rope(hq=0, hk=0, inv=None) == 0
    for name in ("q", "k", "qw", "kw", "inv", "qo", "ko"):
        assert norm_rope(**{name: None}) == NULL, name
    assert norm_rope(d=63) == DIM and norm_rope(d=1026) == DIM
    assert norm_rope(qs=4 * 64 - 1) == DIM and norm_rope(kos=2 * 64 - 4) == DIM
    assert norm_rope(batch=2 ** 40, seq=2 ** 40) == OVER and norm_rope(batch=2 ** 31, seq=1) == OVER
    assert norm_rope(start=2 ** 64 - 2) == OVER
    assert norm_rope(qs=2 ** 45) == OVER
    # outputs over each other, over the other's input, or shifted over their own
    assert norm_rope(ko=P + 2 * M + 64) == ALIAS
    assert norm_rope(qo=P + M) == ALIAS and norm_rope(ko=P) == ALIAS
    assert norm_rope(qo=P + 64) == ALIAS
    # in place, but with another stride
    assert norm_rope(qo=P, qos=512) == ALIAS
    # rows of k inside the gaps of q's, but one float too far in
    assert norm_rope(q=P, qo=P, qs=512, qos=512, k=P + 4 * (4 * 64 - 1), ko=P + 4 * (4 * 64 - 1), ks=512, kos=512) == ALIAS
    # outputs over what every row reads
    row, end = 4 * 64 * 4, 6 * 4 * 64 * 4
    for name, size in (("qw", 256), ("kw", 256), ("inv", 128), ("pos", 24)):
        assert norm_rope(**{name: P + 2 * M}) == norm_rope(**{name: P + 2 * M + end - 4}) == ALIAS, name
        assert norm_rope(**{name: P + 3 * M - 4}) == norm_rope(**{name: P + 3 * M + 64}) == ALIAS, name
        assert norm_rope(**{name: P + 2 * M + 5 * 2 * row - 4}, qos=512) == ALIAS, name  # the last token's row


def norm_rope_bwd(dq=P, dk=P + M, q=P + 2 * M, k=P + 3 * M, qw=P + 8 * M, kw=P + 8 * M, inv=P + 9 * M, gq=P + 4 * M,
                  gk=P + 5 * M, gqw=P + 6 * M, gkw=P + 7 * M, ws=P + 10 * M, wsb=None, batch=2, seq=3, hq=4, hk=2, d=64,
                  strides=(0,) * 6, start=0):
    lib = _lib.load()
    if wsb is None:
        wsb = lib.kore_hip_qk_norm_rope_backward_workspace_bytes(batch * seq, hq, hk, d)
    return lib.kore_hip_qk_norm_rope_backward_f32(dq, dk, q, k, qw, kw, inv, None, gq, gk, gqw, gkw, ws, wsb, batch, seq, hq,
                                                  hk, d, *strides, start, 1e-6, 0, None)


def test_norm_rope_backward_refusals():
    assert norm_rope_bwd(d=0) == 0 and norm_rope_bwd(hq=0, hk=0) == 0
    for name in ("dq", "dk", "q", "k", "qw", "kw", "inv", "gq", "gk", "gqw", "gkw", "ws"):
        assert norm_rope_bwd(**{name: None}) == NULL, name
    lib = _lib.load()
    need = lib.kore_hip_qk_norm_rope_backward_workspace_bytes(6, 4, 2, 64)
    assert need > 0 and norm_rope_bwd(wsb=need - 1) == DIM
    assert norm_rope_bwd(d=7, wsb=M) == DIM and norm_rope_bwd(d=2048, wsb=M) == DIM
    for i in range(6):
        s = [0] * 6
        s[i] = 100
        assert norm_rope_bwd(strides=s) == DIM, i
    assert norm_rope_bwd(gq=P + 5 * M + 4) == ALIAS and norm_rope_bwd(gq=P + M) == ALIAS and norm_rope_bwd(gk=P + 2 * M) == ALIAS
    assert norm_rope_bwd(gq=P + 4) == ALIAS
    for name in ("qw", "kw", "inv", "gqw", "gkw"):
        assert norm_rope_bwd(**{name: P + 4 * M + 64}) == norm_rope_bwd(**{name: P + 5 * M}) == ALIAS, name
        assert norm_rope_bwd(**{name: P + 10 * M + 4}) == ALIAS, name
    for name in ("dq", "dk", "q", "k", "gq", "gk"):
        assert norm_rope_bwd(**{name: P + 10 * M - 4}) == ALIAS, name
    assert norm_rope_bwd(gkw=P + 6 * M + 252) == ALIAS
    assert norm_rope_bwd(batch=2 ** 30, seq=1, wsb=2 ** 40) == OVER  # more than 32 bits of rows
    ws = lib.kore_hip_qk_norm_rope_backward_workspace_bytes
    assert ws(0, 4, 2, 64) == 0 and ws(5, 0, 0, 64) == 0 and ws(1, 1, 1, 64) == 512 and ws(1, 3, 0, 64) == 256
    assert ws(2 ** 30, 32, 8, 128) == 1023 * 128 * 4 and ws(20, 2, 1, 128) == 5 * 128 * 4


def cache_write(k=P, v=P + M, slots=P + 2 * M, cache=P + 3 * M, tokens=5, heads=2, d=64, pages=4, page=16, ks=0, vs=0):
    return _lib.load().kore_hip_kv_cache_write_q4_f32(k, v, slots, cache, tokens, heads, d, pages, page, ks, vs, None)


def cache_read(cache=P, slots=P + M, k=P + 2 * M, v=P + 3 * M, tokens=5, heads=2, d=64, pages=4, page=16):
    return _lib.load().kore_hip_kv_cache_read_q4_f32(cache, slots, k, v, tokens, heads, d, pages, page, None)


def test_cache_refusals():
    for f in (cache_write, cache_read):
        assert f(tokens=0, k=None) == 0 and f(heads=0) == 0 and f(d=0) == 0
        for name in ("k", "v", "slots", "cache"):
            assert f(**{name: None}) == NULL, name
        for bad in ({"d": 257}, {"page": 8}, {"page": 24}, {"page": 0}, {"page": 1 << 17}, {"cache": P + 3 * M + 8}):
            assert f(**bad) == DIM, bad
        assert f(heads=70000) == OVER and f(pages=2 ** 33) == OVER and f(pages=2 ** 32 - 1, page=65536) == OVER
    assert cache_write(pages=0, cache=None) == 0
    assert cache_write(ks=127) == DIM and cache_write(vs=64) == DIM and cache_write(ks=2 ** 45) == OVER
    assert cache_write(k=P + 3 * M + 64) == ALIAS and cache_write(v=P + 3 * M - 64) == ALIAS and cache_write(slots=P + 3 * M) == ALIAS
    assert cache_read(k=P + 64) == ALIAS and cache_read(v=P + 2 * M + 16) == ALIAS and cache_read(k=P + M) == ALIAS
    b = _lib.load().kore_hip_kv_cache_q4_bytes
    assert b(3, 16, 2, 65) == 3 * 2 * 16 * 3 * 34 and b(3, 20, 2, 64) == 0 and b(3, 16, 2, 300) == 0


def attention(q=P, cache=P + M, table=P + 2 * M, lens=P + 3 * M, starts=P + 4 * M, out=P + 5 * M, ws=P + 8 * M, wsb=None, seqs=2,
              tokens=5, hq=4, hk=2, d=64, pages=8, page=16, most=4, qs=0):
    lib = _lib.load()
    if wsb is None:
        wsb = lib.kore_hip_attention_q4_workspace_bytes(seqs, tokens, hq, hk, d, page, most)
    return lib.kore_hip_attention_q4_f32(q, cache, table, lens, starts, out, ws, wsb, seqs, tokens, hq, hk, d, pages, page, most,
                                         qs, 0.125, 1, None)


def test_attention_refusals():
    assert attention(seqs=0, q=None) == 0 and attention(tokens=0) == 0 and attention(hq=0) == 0 and attention(d=0) == 0
    for name in ("q", "cache", "table", "lens", "starts", "out"):
        assert attention(**{name: None}) == NULL, name
    for bad in ({"d": 300}, {"page": 12}, {"hq": 5}, {"hk": 0}, {"hk": 3}, {"cache": P + M + 4}, {"qs": 255}):
        assert attention(**bad) == DIM, bad
    for bad in ({"tokens": 2 ** 32}, {"seqs": 2 ** 32}, {"most": 2 ** 29}, {"hq": 2 ** 17}, {"qs": 2 ** 44},
                {"tokens": 2 ** 30, "hq": 32, "hk": 8}):
        assert attention(**bad) == OVER, bad
    for over in (P, P + M, P + 2 * M, P + 3 * M, P + 4 * M):
        assert attention(out=over) == ALIAS
    # long tables split the keys: a workspace
    lib = _lib.load()
    need = lib.kore_hip_attention_q4_workspace_bytes(2, 5, 4, 2, 64, 16, 1024)
    assert need > 0
    assert attention(most=1024, wsb=need - 1) == DIM and attention(most=1024, ws=None) == NULL
    assert attention(most=1024, ws=P + 8 * M + 4) == DIM and attention(most=1024, out=P + 8 * M) == ALIAS
    for name in ("q", "cache", "table", "lens", "starts"):
        assert attention(most=1024, **{name: P + 8 * M}) == ALIAS, name
    assert lib.kore_hip_attention_q4_workspace_bytes(2, 5, 4, 3, 64, 16, 1024) == 0
    assert lib.kore_hip_attention_q4_workspace_bytes(2, 0, 4, 2, 64, 16, 1024) == 0
