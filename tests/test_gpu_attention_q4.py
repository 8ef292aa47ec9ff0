"""Attention over the paged 4-bit cache against 64 bits: every head dimension's form, shared key heads, ragged sequences
down to empty ones, pages that end inside a tile, masked places that hold NaN, and the split over long contexts."""
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


class Case:
    """Sequences with `lens` cached tokens and `news` query tokens, in pages of any order; slots that no sequence owns hold
    any bytes (NaN scales among them)."""

    def __init__(self, hq, hk, d, page, lens, news, seed=0, spare=0, std=1.0):
        r = np.random.default_rng(seed)
        self.hq, self.hk, self.d, self.page = hq, hk, d, page
        self.lens, self.news = np.array(lens, np.uint32), np.array(news)
        each = [(n + page - 1) // page for n in lens]
        self.most = max(each + [1]) + spare
        self.cache = q4_ref.Cache(sum(each) + 2, page, hk, d, seed=seed)
        ids = r.permutation(sum(each) + 2)
        self.table = r.integers(0, 2 ** 32, (len(lens), self.most), dtype=np.uint64).astype(np.uint32)  # past the end: anything
        at = 0
        for s, n in enumerate(each):
            self.table[s, :n] = ids[at:at + n]
            at += n
        for s, n in enumerate(lens):
            i = np.arange(n)
            slots = self.table[s, i // page].astype(np.int64) * page + i % page
            self.cache.write(slots, r.standard_normal((n, hk, d), np.float32), r.standard_normal((n, hk, d), np.float32))
        self.starts = np.concatenate([[0], np.cumsum(self.news)]).astype(np.uint32)
        self.tokens = int(self.starts[-1])
        self.q = r.standard_normal((self.tokens, hq, d), np.float32) * np.float32(std)
        self.scale = d ** -0.5

    def run(self, causal=True, out=None, q=None, q_stride=0, tokens=None, workspace=None):
        t = self.tokens if tokens is None else tokens
        return rocm.rocm_attention_q4_f32(
            DEV, up(self.q) if q is None else q, up(self.cache.bytes), up(self.table), up(self.lens), up(self.starts), len(self.lens),
            t, self.hq, self.hk, self.d, self.cache.bytes.shape[0], self.page, self.most, self.scale, causal, q_stride, workspace, out)

    def check(self, causal=True, what="", **kw):
        got = self.run(causal, **kw).to_host(np.float32)[:self.q.size].reshape(self.q.shape)
        want, tol = q4_ref.attention(self.q, self.cache, self.table, self.lens, self.starts, self.scale, causal, np.zeros(self.q.shape))
        q4_ref.assert_within(got, want, tol, what)
        return got


# hq, hk, head_dim, page, lens, news
CASES = [
    (1, 1, 32, 16, [1], [1]), (2, 1, 64, 16, [16], [1]), (4, 2, 128, 16, [17], [1]), (3, 3, 96, 32, [31, 32, 33], [1, 1, 1]),
    (8, 1, 128, 64, [63, 64, 65, 129], [1, 1, 1, 1]), (5, 1, 80, 16, [100, 1, 47], [1, 1, 1]), (6, 2, 16, 16, [20, 40], [1, 2]),
    (4, 4, 256, 16, [70, 5], [1, 3]), (2, 2, 160, 32, [50], [4]), (2, 1, 200, 16, [90], [2]), (7, 7, 40, 16, [33], [5]),
    (4, 1, 1, 16, [19], [3]), (10, 2, 7, 64, [77, 3], [2, 3]), (20, 1, 64, 16, [60], [3]), (33, 1, 32, 16, [40], [2]),
    (4, 2, 64, 16, [0, 5, 0, 30, 0], [1, 2, 0, 3, 2]), (4, 4, 64, 16, [3, 10], [8, 10]), (2, 2, 128, 128, [200, 130], [150, 1]),
    (8, 2, 64, 16, [300, 77, 12], [61, 77, 5]), (4, 1, 128, 16, [257], [40]), (1, 1, 128, 16, [150], [150]), (2, 1, 256, 64, [130], [70]),
    (16, 2, 128, 32, [500, 480, 16, 33], [1, 1, 1, 1]), (3, 1, 64, 16, [65] * 70, [1] * 70), (2, 2, 32, 16, [9] * 130, [0, 1] * 65)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%dx%dx%d-p%d-%s-%s" % (*c[:4], c[4][:4], c[5][:4]))
def test_against_64_bits(case, causal):
    Case(*case, seed=len(case[4])).check(causal)


@pytest.mark.parametrize("hq,hk,d,page,lens,news", [(4, 1, 128, 16, [3000], [1]), (8, 2, 64, 64, [5000, 1500], [1, 1]),
                                                    (2, 2, 256, 16, [1200, 0, 40], [2, 1, 1]), (4, 2, 128, 32, [2100], [9]),
                                                    (6, 1, 96, 16, [1700, 300], [40, 2]), (2, 2, 256, 16, [2300, 0, 40], [2, 1, 1]),
                                                    (6, 1, 96, 16, [3100, 300], [40, 2]), (4, 1, 128, 64, [4097, 700, 2048], [100, 3, 33]),
                                                    (2, 1, 64, 16, [2500] + [30] * 300, [1] * 301)])
def test_split_contexts(hq, hk, d, page, lens, news):
    """Few rows over many keys: shares of the keys, joined at the end; some shares of the shorter sequences are empty."""
    c = Case(hq, hk, d, page, lens, news, seed=3, std=3.0)
    # keys are cut where the table has room for 2048 tokens of a sequence
    assert (rocm.rocm_attention_q4_workspace_bytes(len(lens), c.tokens, hq, hk, d, page, c.most) > 0) == (max(lens) >= 2048)
    c.check()
    c.check(causal=False)


@pytest.mark.parametrize("seqs,hq,hk,d,most,first,news", [(400, 8, 4, 32, 40, 3, [1]), (300, 18, 6, 64, 20, 0, [0, 1, 2, 40]), (5000, 3, 1, 16, 3, 0, [0, 0, 1]),
                                                          (257, 24, 8, 16, 40, 1, [9, 0]), (2300, 4, 2, 16, 8, 7, [1]), (2100, 6, 3, 16, 4, 0, [0, 35, 2])])
def test_many_sequences(seqs, hq, hk, d, most, first, news):
    """More sequences than a wave looks at in one go, some of them empty, rows before the first and behind the last."""
    r = np.random.default_rng(seqs)
    c = Case(hq, hk, d, 16, [int(x) for x in r.integers(0, most, seqs)], (news * seqs)[:seqs], seed=seqs)
    c.starts = c.starts + np.uint32(first)
    c.tokens += first + 2
    c.q = normal((c.tokens, hq, d), seqs)
    for causal in (True, False):
        out = HipBuffer.from_host(DEV, np.full(c.q.size * 4, 0xFF, np.uint8))
        c.run(causal, out)
        got = out.to_host(np.float32).reshape(c.q.shape)
        want, tol = q4_ref.attention(c.q, c.cache, c.table, c.lens, c.starts, c.scale, causal, np.full(c.q.shape, np.nan))
        q4_ref.assert_within(got, want, tol)


@pytest.mark.parametrize("hq,hk,d,lens,news", [(4, 2, 64, [30, 300, 5, 200, 17], [1, 150, 1, 90, 1]), (8, 2, 128, [2500, 40, 2100], [1, 40, 100]),
                                               (6, 3, 32, [3000] + [20] * 90 + [260], [1] * 91 + [200])])
def test_decode_steps_beside_chunks(hq, hk, d, lens, news):
    """Sequences of one tile among those of several, uncut and cut."""
    c = Case(hq, hk, d, 16, lens, news, seed=22)
    c.check()
    c.check(causal=False)


def test_table_longer_than_the_sequences():
    """A table sized for long contexts in front of short ones: most splits have nothing to do."""
    c = Case(4, 2, 64, 16, [5, 40, 0], [1, 1, 1], seed=4, spare=2000)
    assert rocm.rocm_attention_q4_workspace_bytes(3, 3, 4, 2, 64, 16, c.most) > 0
    got = c.check()
    assert (got[2] == 0).all()


def test_peaked_and_flat_scores():
    c = Case(4, 2, 128, 16, [600, 333], [3, 1], seed=5, std=60.0)
    c.check(what="peaked")
    c.scale = 0.0
    c.check(what="flat")
    c.scale = -0.3
    c.check(what="negative")


@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_nan_and_inf_in_places_that_are_not_seen(d):
    """NaN keys and values of later tokens leave earlier rows alone, block by block; what sees them is NaN."""
    n, new = 75, 40
    c = Case(4, 2, d, 16, [n], [new], seed=6)
    r = np.random.default_rng(7)
    k, v = r.standard_normal((n, 2, d), np.float32), r.standard_normal((n, 2, d), np.float32)
    v[60, 1, 33 % d] = np.nan  # one block of V, key head 1, seen by the last 15 rows
    v[70, 0, d - 1] = np.inf
    k[72, 0, 0] = np.nan       # a key: whole rows of key head 0
    i = np.arange(n)
    c.cache.write(c.table[0, i // 16].astype(np.int64) * 16 + i % 16, k, v)
    got = c.run().to_host(np.float32).reshape(c.q.shape)
    want, tol = q4_ref.attention(c.q, c.cache, c.table, c.lens, c.starts, c.scale, True, np.zeros(c.q.shape))
    assert np.isfinite(want[:25]).all() and np.isnan(want).any()
    q4_ref.assert_within(got, want, tol)
    first = n - new  # token of row 0
    b = slice(33 % d // 32 * 32, min(d, 33 % d // 32 * 32 + 32))
    assert np.isnan(got[60 - first:, 2:, b]).all() and np.isfinite(got[:72 - first, :2, :(d - 1) // 32 * 32]).all()


def test_nan_before_every_row():
    """A NaN value that all rows see, in a step without masks."""
    c = Case(2, 1, 128, 16, [200], [2], seed=8)
    k, v = normal((1, 1, 128), 1), normal((1, 1, 128), 2)
    v[0, 0, 40] = np.nan
    c.cache.write([int(c.table[0, 2]) * 16 + 3], k, v)
    got = c.check()
    assert np.isnan(got[..., 32:64]).all() and np.isfinite(got[..., :32]).all() and np.isfinite(got[..., 64:]).all()
    k[0, 0, 5] = np.inf
    c.cache.write([int(c.table[0, 2]) * 16 + 3], k, v)
    assert np.isnan(c.check()).all()


def test_queries_that_are_not_finite():
    c = Case(4, 2, 64, 16, [50], [4], seed=9)
    c.q[1, 2, 3], c.q[2, 0, 0] = np.nan, np.inf
    got = c.run().to_host(np.float32).reshape(c.q.shape)
    assert np.isnan(got[1, 2]).all() and np.isnan(got[2, 0]).all()
    got[1, 2], got[2, 0] = 0, 0
    c.q[1, 2, 3] = c.q[2, 0, 0] = 0
    want, tol = q4_ref.attention(c.q, c.cache, c.table, c.lens, c.starts, c.scale, True, np.zeros(c.q.shape))
    want[1, 2], want[2, 0] = 0, 0
    q4_ref.assert_within(got, want, tol)


def test_pages_that_do_not_exist():
    """Page ids past the cache: their tokens are left out, whatever lies where."""
    c = Case(4, 2, 64, 16, [100, 40], [5, 1], seed=10)
    c.table[0, 2] = c.cache.bytes.shape[0]
    c.table[0, 5] = 0xFFFFFFFF
    c.table[1, :3] = 1 << 30
    got = c.check()
    assert (got[5] == 0).all()


def test_lengths_past_the_table_and_rows_of_no_sequence():
    """Lengths count up to the table's end; starts up to `tokens`; rows of no sequence stay as they are."""
    c = Case(2, 1, 64, 16, [64, 30], [3, 2], seed=11)
    t = c.tokens + 4
    c.lens = np.array([5000, 30], np.uint32)
    c.q = normal((t, 2, 64), 12)
    c.starts = np.array([1, 4, 6], np.uint32)
    out = torch.full((t, 2, 64), 55.0, device="cuda")
    c.run(tokens=t, out=HipBuffer.from_tensor(out))
    got = out.cpu().numpy()
    want, tol = q4_ref.attention(c.q, c.cache, c.table, c.lens, c.starts, c.scale, True, np.full(c.q.shape, 55.0))
    q4_ref.assert_within(got, want, tol)
    assert (got[0] == 55).all() and (got[6:] == 55).all()
    c.starts = np.array([0, 3, 100], np.uint32)
    c.check(tokens=t)


@pytest.mark.parametrize("pad,off", [(128, 0), (3, 1), (64, 2)])
def test_queries_inside_a_projection(pad, off):
    c = Case(4, 2, 64, 16, [80, 33], [6, 1], seed=13)
    stride = 4 * 64 + pad
    buf = torch.full((c.tokens * stride + off,), float("nan"), device="cuda")
    buf[off:].view(c.tokens, stride)[:, :256] = torch.from_numpy(c.q.reshape(c.tokens, 256)).cuda()
    c.check(q=HipBuffer.from_tensor(buf[off:]), q_stride=stride)


def test_repeats_bit_for_bit_and_on_another_stream():
    c = Case(8, 2, 128, 16, [900, 700], [1, 3], seed=14)
    first = c.run().to_host().tobytes()
    assert c.run().to_host().tobytes() == first
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run()
    s.synchronize()
    assert got.to_host().tobytes() == first


def test_capture_with_growing_contexts():
    """A captured call replayed with other lengths and queries in the same buffers."""
    c = Case(4, 2, 64, 16, [700, 300], [1, 1], seed=15)
    ws = HipBuffer.empty(DEV, max(16, rocm.rocm_attention_q4_workspace_bytes(2, 2, 4, 2, 64, 16, c.most)))
    b = [up(c.q), up(c.cache.bytes), up(c.table), up(c.lens), up(c.starts)]
    out = HipBuffer.empty(DEV, c.q.nbytes)

    def step():
        rocm.rocm_attention_q4_f32(DEV, *b, 2, 2, 4, 2, 64, c.cache.bytes.shape[0], 16, c.most, c.scale, True, 0, ws, out)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for lens in ([700, 300], [1, 299], [0, 17], [650, 0], [700, 300]):
        c.lens = np.array(lens, np.uint32)
        c.q = normal(c.q.shape, sum(lens))
        b[3].tensor(torch.int32).copy_(torch.from_numpy(c.lens.view(np.int32)))
        b[0].tensor(torch.float32).copy_(torch.from_numpy(c.q.ravel()))
        out.tensor().fill_(0xFF)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.to_host(np.float32)
        step()
        torch.cuda.synchronize()
        assert out.to_host(np.float32).tobytes() == got.tobytes()
        want, tol = q4_ref.attention(c.q, c.cache, c.table, c.lens, c.starts, c.scale, True, np.zeros(c.q.shape))
        q4_ref.assert_within(got.reshape(c.q.shape), want, tol, str(lens))


def test_small_buffers_are_refused():
    c = Case(2, 1, 64, 16, [64], [2], seed=16)
    with pytest.raises(RocmError, match="attention q"):
        c.run(q=up(np.zeros(255, np.float32)))
    with pytest.raises(RocmError, match="attention out"):
        c.run(out=up(np.zeros(255, np.float32)))
    with pytest.raises(RocmError, match="page_table"):
        c.most += 1
        c.run()
    c.most = 400
    c.table = np.zeros((1, 400), np.uint32)
    with pytest.raises(RocmError, match="invalid dimension"):
        c.run(workspace=HipBuffer.empty(DEV, 64))


@pytest.mark.parametrize("page,lens,news", [(65536, [70, 300], [1, 3]), (4096, [4100, 17], [1, 1]), (1024, [1025, 2049, 5], [60, 1, 5])])
def test_large_pages(page, lens, news):
    Case(4, 2, 32, page, lens, news, seed=16).check()


def test_sequences_that_share_pages():
    """A common beginning cached once: the same pages in several rows of the table, and the whole table of one row twice."""
    c = Case(6, 2, 64, 16, [64, 75, 90], [1, 2, 1], seed=17)
    c.table[0, :4] = c.table[2, :4]
    c.table[1, :3] = c.table[2, :3]
    c.check()
    c.table[1], c.lens[1] = c.table[2], c.lens[2]
    c.check()
    c.table[2, 1] = c.table[2, 0]  # one page at two places
    c.check()


def test_nothing_cached_and_nothing_new():
    c = Case(4, 2, 64, 16, [20, 30], [2, 1], seed=18)
    for pages, most in ((0, c.most), (c.cache.bytes.shape[0], 0), (0, 0)):
        out = HipBuffer.from_host(DEV, np.full(c.q.size * 4, 0xFF, np.uint8))
        rocm.rocm_attention_q4_f32(DEV, up(c.q), up(c.cache.bytes), up(c.table), up(c.lens), up(c.starts), 2, c.tokens, 4, 2, 64, pages, 16,
                                   most, c.scale, True, 0, None, out)
        assert (out.to_host(np.float32) == 0).all(), (pages, most)
    for starts in ([0, 0, 0], [3, 3, 3], [99, 99, 99]):
        out = HipBuffer.from_host(DEV, np.full(c.q.size * 4, 0xFF, np.uint8))
        rocm.rocm_attention_q4_f32(DEV, up(c.q), up(c.cache.bytes), up(c.table), up(c.lens), up(np.array(starts, np.uint32)), 2, c.tokens, 4, 2,
                                   64, c.cache.bytes.shape[0], 16, c.most, c.scale, True, 0, None, out)
        assert (out.to_host(np.uint8) == 0xFF).all(), starts


def test_two_calls_at_once():
    """Two calls on two streams, over one cache and with workspaces of their own, many times over."""
    c = Case(8, 2, 64, 16, [2600, 900], [1, 1], seed=19)
    n = rocm.rocm_attention_q4_workspace_bytes(2, 2, 8, 2, 64, 16, c.most)
    assert n > 0
    b = [up(c.cache.bytes), up(c.table), up(c.lens), up(c.starts)]
    qs = [normal(c.q.shape, 20 + i) for i in range(2)]
    each = [(up(q), HipBuffer.empty(DEV, n), HipBuffer.empty(DEV, q.nbytes), torch.cuda.Stream()) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for q, ws, out, stream in each:
            with torch.cuda.stream(stream):
                rocm.rocm_attention_q4_f32(DEV, q, *b, 2, 2, 8, 2, 64, c.cache.bytes.shape[0], 16, c.most, c.scale, True, 0, ws, out)
    torch.cuda.synchronize()
    for q, (_, _, out, _) in zip(qs, each):
        want, tol = q4_ref.attention(q, c.cache, c.table, c.lens, c.starts, c.scale, True, np.zeros(q.shape))
        q4_ref.assert_within(out.to_host(np.float32).reshape(q.shape), want, tol)


def test_offsets_past_32_bits():
    """Pages past 4 GiB of the cache, and query rows 4 GiB apart: the same bits as from a small cache and dense rows."""
    hq, hk, d, page, lens = 4, 2, 256, 64, [70, 150]
    c = Case(hq, hk, d, page, lens, [1, 2], seed=21)
    small = c.run(out=None).to_host(np.float32)[:c.q.size]
    each = c.cache.bytes[0].nbytes
    far = (1 << 32) // each + 1
    cache = torch.empty(((far + c.cache.bytes.shape[0]) * each,), dtype=torch.uint8, device="cuda")
    cache[far * each:].copy_(torch.from_numpy(c.cache.bytes.reshape(-1)))
    cache[:c.cache.bytes.nbytes].fill_(0xFF)  # what a wrapped offset would meet
    stride = 1 << 30
    q = torch.empty(((c.tokens - 1) * stride + hq * d,), device="cuda")
    for t in range(c.tokens):
        q[t * stride:t * stride + hq * d].copy_(torch.from_numpy(c.q[t].reshape(-1)))
    got = rocm.rocm_attention_q4_f32(DEV, HipBuffer.from_tensor(q), HipBuffer.from_tensor(cache), up(c.table + np.uint32(far)), up(c.lens), up(c.starts),
                                     2, c.tokens, hq, hk, d, far + c.cache.bytes.shape[0], page, c.most, c.scale, True, stride)
    torch.cuda.synchronize()
    assert got.to_host(np.float32)[:c.q.size].tobytes() == small.tobytes()
