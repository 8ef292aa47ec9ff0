"""The paged 4-bit cache: every byte that a write leaves against the definition, the rest of the cache untouched, and
values read back exactly."""
import numpy as np
import pytest

import q4_ref
from inputs import normal

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from kore_amd import rocm  # noqa: E402
from kore_amd.rocm import HipBuffer, RocmError  # noqa: E402

DEV = 0


def up(a):
    return HipBuffer.from_host(DEV, np.ascontiguousarray(a))


def special(x):
    """Blocks that are zero, tiny, huge, at ties, and not finite, into the first tokens of x [T, H, D]."""
    x = x.copy()
    t, d = x.shape[0], x.shape[-1]
    rows = [np.zeros(d), np.full(d, 2.0 ** -140), np.full(d, 3.4e38), np.where(np.arange(d) % 2, 1e38, -1.5e38),
            np.resize([6, 0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0, 7.0, -7.0, 0.0, -0.0], d), np.full(d, 7.0000005),
            np.where(np.arange(d) == d // 2, np.inf, 1.0), np.where(np.arange(d) == 0, np.nan, 1.0),
            np.where(np.arange(d) == d - 1, -np.inf, 1.0), np.full(d, 1.75 * 2.0 ** 127), np.full(d, 2.0 ** -98), np.full(d, 1e-45)]
    for i, row in enumerate(rows[:t]):
        x[i, i % x.shape[1]] = row.astype(np.float32)
    return x


@pytest.mark.parametrize("page,heads,d,tokens,pad", [(16, 1, 32, 1, 0), (16, 2, 128, 40, 0), (64, 8, 128, 13, 0), (16, 3, 80, 30, 5),
                                                     (32, 2, 96, 33, 0), (128, 1, 256, 20, 4), (16, 2, 1, 14, 0), (16, 5, 33, 18, 1),
                                                     (1024, 2, 64, 50, 3), (16, 1, 200, 17, 0), (64, 7, 7, 29, 2)])
def test_write_then_read(page, heads, d, tokens, pad):
    r = np.random.default_rng(page + d)
    pages = tokens // page + 5
    host = q4_ref.Cache(pages, page, heads, d, seed=1)
    slots = r.permutation(pages * page)[:tokens].astype(np.uint32)
    slots[tokens // 2] = 0xFFFFFFFF  # padding: skipped
    if tokens > 20:
        slots[3] = pages * page  # just past the end
    stride = heads * d + pad
    kbuf, vbuf = normal((tokens, stride), 2), normal((tokens, stride), 3, 0.0, 40.0)
    k = special(kbuf[:, :heads * d].reshape(tokens, heads, d))
    v = special(vbuf[:, :heads * d].reshape(tokens, heads, d)[::-1])[::-1]
    kbuf[:, :heads * d], vbuf[:, :heads * d] = k.reshape(tokens, -1), v.reshape(tokens, -1)
    assert host.bytes.nbytes == rocm.rocm_kv_cache_q4_bytes(pages, page, heads, d)
    cache = up(host.bytes)
    rocm.rocm_kv_cache_write_q4_f32(DEV, up(kbuf.ravel()[:tokens * stride - pad]), up(vbuf), up(slots), cache, tokens, heads, d, pages,
                                    page, stride, stride)
    host.write(slots, k, v)
    got = cache.to_host().reshape(host.bytes.shape)
    assert got.tobytes() == host.bytes.tobytes(), np.argwhere(got != host.bytes)[:5]
    ko, vo = rocm.rocm_kv_cache_read_q4_f32(DEV, cache, up(slots), tokens, heads, d, pages, page)
    wk, wv = host.read(slots)
    for out, want in ((ko, wk), (vo, wv)):
        g = out.to_host(np.float32).reshape(want.shape)
        assert np.array_equal(g.astype(np.float64), want, equal_nan=True)
    assert (ko.to_host(np.float32).reshape(wk.shape)[tokens // 2] == 0).all()


def test_read_of_any_bytes():
    """Bytes that no write leaves: scales below 2^-100 read as what they stand for, those past f32's range as infinite."""
    page, heads, d, pages = 16, 2, 64, 40
    host = q4_ref.Cache(pages, page, heads, d, seed=9)
    slots = np.arange(pages * page, dtype=np.uint32)
    ko, vo = rocm.rocm_kv_cache_read_q4_f32(DEV, up(host.bytes), up(slots), len(slots), heads, d, pages, page)
    for out, want in zip((ko, vo), host.read(slots)):
        with np.errstate(over="ignore"):
            want = want.astype(np.float32)
        assert np.array_equal(out.to_host(np.float32).reshape(want.shape), want, equal_nan=True)


def test_every_code_boundary():
    """Values a step of f32 to both sides of every rounding edge, in blocks whose scale is held by a 6."""
    edges = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    near = np.concatenate([edges, np.nextafter(edges, np.float32(0)), np.nextafter(edges, np.float32(9))])
    x = np.zeros((1, 1, 32), np.float32)
    x[0, 0, 0], x[0, 0, 1:1 + len(near)] = 6.0, near
    ladder = np.float32(2.0) ** np.arange(-90, 110, 7, dtype=np.float32)
    k = np.concatenate([x * s for s in ladder] + [-x * s for s in ladder])
    t = k.shape[0]
    host = q4_ref.Cache(8, 16, 1, 32, fill=0)
    cache = up(host.bytes)
    slots = np.arange(t, dtype=np.uint32)
    rocm.rocm_kv_cache_write_q4_f32(DEV, up(k), up(k), up(slots), cache, t, 1, 32, 8, 16)
    host.write(slots, k, k)
    assert cache.to_host().tobytes() == host.bytes.tobytes()


def test_offsets_past_32_bits():
    """Pages beyond the first 4 GiB of a cache."""
    page, heads, d = 4096, 8, 128
    each = rocm.rocm_kv_cache_q4_bytes(1, page, heads, d)
    pages = (5 << 30) // each + 1
    cache = HipBuffer.empty(DEV, rocm.rocm_kv_cache_q4_bytes(pages, page, heads, d))
    t = 6
    slots = np.array([pages * page - 1, pages * page - 2, (pages - 1) * page, 5, pages * page // 2, pages * page], np.uint32)
    k, v = normal((t, heads, d), 1), normal((t, heads, d), 2)
    rocm.rocm_kv_cache_write_q4_f32(DEV, up(k), up(v), up(slots), cache, t, heads, d, pages, page)
    ko, vo = rocm.rocm_kv_cache_read_q4_f32(DEV, cache, up(slots), t, heads, d, pages, page)
    for out, x in ((ko, k), (vo, v)):
        want = q4_ref.values(*q4_ref.quantise(x), d)
        want[5] = 0
        assert (out.to_host(np.float32).reshape(x.shape) == want).all()
    last = cache.tensor()[(pages - 1) * each:].cpu().numpy().reshape(heads, -1)
    c, _ = q4_ref.places(page, d, page - 1, False)
    codes, _ = q4_ref.quantise(k[0])
    assert (last[:, c] == (codes[:, 0::2] | codes[:, 1::2] << 4)).all()


def test_small_buffers_are_refused():
    z, s = up(np.zeros(512, np.float32)), up(np.zeros(4, np.uint32))
    cache = HipBuffer.zeros(DEV, rocm.rocm_kv_cache_q4_bytes(2, 16, 1, 64))
    with pytest.raises(RocmError, match="cache"):
        rocm.rocm_kv_cache_write_q4_f32(DEV, z, z, s, cache, 4, 1, 64, 3, 16)
    with pytest.raises(RocmError, match="slots"):
        rocm.rocm_kv_cache_write_q4_f32(DEV, z, z, s, cache, 5, 1, 64, 2, 16)
    with pytest.raises(RocmError, match="kv_cache_write v"):
        rocm.rocm_kv_cache_write_q4_f32(DEV, z, z, s, cache, 4, 1, 64, 2, 16, 0, 160)
    with pytest.raises(RocmError, match="v_out"):
        rocm.rocm_kv_cache_read_q4_f32(DEV, cache, s, 4, 1, 64, 2, 16, v_out=up(np.zeros(255, np.float32)))
    with pytest.raises(RocmError):
        rocm.rocm_kv_cache_q4_bytes(2, 24, 1, 64)
