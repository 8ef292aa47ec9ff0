"""Per-head norm of Q and K with the rotation in the same pass, and its backward, against 64 bits: both pairings, head
dimensions of every lane count and of the general path, fused projections' strides, positions, in place, refusals of
small buffers, capture."""
import numpy as np
import pytest

import q4_ref
from inputs import normal

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from kore_amd import rocm  # noqa: E402
from kore_amd.rocm import HipBuffer, RocmError  # noqa: E402

DEV, EPS = 0, 1e-6


def up(a):
    return HipBuffer.from_host(DEV, np.ascontiguousarray(a))


def case(batch, seq, hq, hk, d, start, seed, positions=None):
    t = batch * seq
    size = np.exp(normal((1, hq + hk, 1), seed + 5))
    x = normal((t, hq + hk, d), seed) * size
    inv = rocm.rope_inv_freq_host(d, 10000.0)
    pos = np.tile(np.arange(start, start + seq, dtype=np.uint64), batch) if positions is None else positions.astype(np.uint64)
    return x[:, :hq], x[:, hq:], normal((d,), seed + 1, 1.0, 0.2), normal((d,), seed + 2, 1.0, 0.2), inv, pos


SHAPES = [  # batch, seq, q heads, k heads, head_dim, start
    (1, 1, 1, 1, 2, 0), (1, 1, 1, 0, 8, 3), (1, 3, 0, 2, 8, 0), (2, 5, 3, 1, 16, 7), (1, 7, 5, 5, 24, 0), (3, 1, 4, 2, 32, 99),
    (1, 4, 6, 2, 64, 4095), (2, 3, 8, 2, 80, 0), (1, 5, 3, 3, 96, 131071), (2, 9, 32, 8, 128, 2040), (1, 2, 17, 1, 192, 5),
    (1, 3, 4, 2, 256, 0), (1, 2, 3, 1, 512, 11), (1, 3, 2, 1, 36, 0), (2, 2, 3, 2, 100, 1 << 20), (1, 2, 2, 1, 1024, 1),
    (1, 2, 1, 1, 520, 0), (1, 2, 3, 1, 64, 4000000000), (1, 300, 5, 3, 64, 0)]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(shape, inter):
    batch, seq, hq, hk, d, start = shape
    q, k, qw, kw, inv, pos = case(*shape, seed=sum(shape) % 1000)
    qo, ko = rocm.rocm_qk_norm_rope_f32(DEV, up(q), up(k), up(qw), up(kw), up(inv), batch, seq, hq, hk, d, EPS, start, None, inter)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        want, tol = q4_ref.qk_norm_rope(x, w, pos, inv, EPS, inter)
        q4_ref.assert_within(got.to_host(np.float32).reshape(x.shape), want, tol, f"forward {shape}")


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES + [(4, 1100, 4, 2, 32, 0), (1, 4500, 1, 1, 20, 0)], ids=str)
def test_backward(shape, inter):
    batch, seq, hq, hk, d, start = shape
    q, k, qw, kw, inv, pos = case(*shape, seed=sum(shape) % 1000 + 3)
    dq, dk = normal(q.shape, 8), normal(k.shape, 9)
    got = rocm.rocm_qk_norm_rope_backward_f32(DEV, up(dq), up(dk), up(q), up(k), up(qw), up(kw), up(inv), batch, seq, hq, hk, d,
                                              EPS, start, None, inter)
    for dx, dw, dy, x, w in ((got[0], got[2], dq, q, qw), (got[1], got[3], dk, k, kw)):
        if x.size == 0:
            continue
        wdx, wdw, tx, tw = q4_ref.qk_norm_rope_backward(dy, x, w, pos, inv, EPS, inter)
        q4_ref.assert_within(dx.to_host(np.float32).reshape(x.shape), wdx, tx, f"dx {shape}")
        q4_ref.assert_within(dw.to_host(np.float32), wdw, tw, f"dw {shape}")


@pytest.mark.parametrize("d,pad,off", [(64, 0, 0), (64, 3, 1), (20, 5, 2), (128, 4, 4)])
def test_parts_of_a_projection_with_positions(d, pad, off):
    """q and k inside one [tokens, (hq + 2 hk) d + pad] output, at any offset, every token with its own position; out of
    place, in place, and the backward's gradients into a buffer of the same kind.  Nothing else is touched."""
    t, hq, hk = 13, 4, 2
    stride = (hq + 2 * hk) * d + pad
    buf = normal((t * stride + off,), 4)
    r = np.random.default_rng(5)
    pos = r.integers(0, 200000, t).astype(np.uint32)
    rows = buf[off:].reshape(t, stride)
    q, k = rows[:, :hq * d].reshape(t, hq, d), rows[:, hq * d:(hq + hk) * d].reshape(t, hk, d)
    qw, kw, inv = normal((d,), 6, 1.0, 0.1), normal((d,), 7, 1.0, 0.1), rocm.rope_inv_freq_host(d, 500000.0)
    wq, tq = q4_ref.qk_norm_rope(q, qw, pos, inv, EPS, False)
    wk, tk = q4_ref.qk_norm_rope(k, kw, pos, inv, EPS, False)
    dev = torch.from_numpy(buf.copy()).cuda()
    qb, kb = HipBuffer.from_tensor(dev[off:]), HipBuffer.from_tensor(dev[off + hq * d:])
    args = (up(qw), up(kw), up(inv), 1, t, hq, hk, d, EPS, 0, up(pos), False, stride, stride)
    qo, ko = rocm.rocm_qk_norm_rope_f32(DEV, qb, kb, *args)
    q4_ref.assert_within(qo.to_host(np.float32).reshape(q.shape), wq, tq, "q")
    q4_ref.assert_within(ko.to_host(np.float32).reshape(k.shape), wk, tk, "k")
    assert (dev.cpu().numpy() == buf).all()
    dq, dk = normal(q.shape, 8), normal(k.shape, 9)
    g = torch.full_like(dev, 77.0)
    rocm.rocm_qk_norm_rope_backward_f32(DEV, up(dq), up(dk), qb, kb, *args, grad_q=HipBuffer.from_tensor(g[off:]),
                                        grad_k=HipBuffer.from_tensor(g[off + hq * d:]), grad_q_stride=stride, grad_k_stride=stride)
    g = g.cpu().numpy()
    gr = g[off:].reshape(t, stride)
    wdx, _, tx, _ = q4_ref.qk_norm_rope_backward(dq, q, qw, pos, inv, EPS, False)
    q4_ref.assert_within(gr[:, :hq * d].reshape(q.shape), wdx, tx, "grad q")
    wdx, _, tx, _ = q4_ref.qk_norm_rope_backward(dk, k, kw, pos, inv, EPS, False)
    q4_ref.assert_within(gr[:, hq * d:(hq + hk) * d].reshape(k.shape), wdx, tx, "grad k")
    assert (gr[:, (hq + hk) * d:] == 77.0).all() and (g[:off] == 77.0).all()
    rocm.rocm_qk_norm_rope_f32(DEV, qb, kb, *args, q_out=qb, k_out=kb, q_out_stride=stride, k_out_stride=stride)
    got = dev.cpu().numpy()
    assert got[off:].reshape(t, stride)[:, :hq * d].tobytes() == qo.to_host(np.float32).reshape(t, hq * d).tobytes()
    assert got[off:].reshape(t, stride)[:, hq * d:(hq + hk) * d].tobytes() == ko.to_host(np.float32).reshape(t, hk * d).tobytes()
    assert (got[off:].reshape(t, stride)[:, (hq + hk) * d:] == rows[:, (hq + hk) * d:]).all()


@pytest.mark.parametrize("d", [128, 36])
def test_backward_in_place_and_repeatable(d):
    t, hq, hk = 700, 4, 2
    q, k, qw, kw, inv, pos = case(1, t, hq, hk, d, 0, 21)
    dq, dk = normal(q.shape, 8), normal(k.shape, 9)

    def call(over):
        b = [up(a) for a in (dq, dk, q, k)]
        kwargs = {"grad_q": b[over], "grad_k": b[over + 1]} if over is not None else {}
        r = rocm.rocm_qk_norm_rope_backward_f32(DEV, *b, up(qw), up(kw), up(inv), 1, t, hq, hk, d, EPS, **kwargs)
        return [x.to_host(np.float32).tobytes() for x in r]

    first = call(None)
    assert call(None) == first and call(0) == first and call(2) == first


def test_rows_of_zeros_inf_and_nan():
    d, t = 64, 6
    q, k, qw, kw, inv, pos = case(1, t, 2, 1, d, 0, 31)
    q = q.copy()
    q[0] = 0.0
    q[1, 0, 5] = np.inf
    q[2, 1, 7] = np.nan
    q[3] *= np.float32(1e-30)  # squares underflow: eps alone is left
    qo, _ = rocm.rocm_qk_norm_rope_f32(DEV, up(q), up(k), up(qw), up(kw), up(inv), 1, t, 2, 1, d, EPS)
    got = qo.to_host(np.float32).reshape(t, 2, d)
    with np.errstate(invalid="ignore"):
        want, tol = q4_ref.qk_norm_rope(q, qw, pos, inv, EPS, False)
    assert (got[0] == 0).all() and np.isnan(got[2, 1]).all()
    # inf * (1 / inf) is NaN, and the others times zero are 0; the NaN reaches its pair
    assert np.isnan(got[1, 0, [5, 37]]).all() and (np.delete(got[1, 0], [5, 37]) == 0).all()
    for i in ((1, 1), (2, 0), (3, 0), (3, 1), (4, 0), (5, 1)):
        q4_ref.assert_within(got[i], want[i], tol[i], str(i))


def test_empty_and_small_buffers():
    z = up(np.zeros(64, np.float32))
    gq, gk, gqw, gkw = rocm.rocm_qk_norm_rope_backward_f32(
        DEV, z, z, z, z, z, z, z, 0, 5, 2, 1, 32, EPS, grad_q_weight=up(np.ones(32, np.float32)),
        grad_k_weight=up(np.ones(32, np.float32)))
    assert (gqw.to_host(np.float32) == 0).all() and (gkw.to_host(np.float32) == 0).all()
    with pytest.raises(RocmError, match="q_weight"):
        rocm.rocm_qk_norm_rope_f32(DEV, z, z, up(np.zeros(31, np.float32)), z, z, 1, 1, 2, 1, 32, EPS)
    with pytest.raises(RocmError, match="qk_norm_rope k"):
        rocm.rocm_qk_norm_rope_f32(DEV, z, z, z, z, z, 1, 2, 1, 1, 32, EPS, k_stride=33)
    with pytest.raises(RocmError, match="positions"):
        rocm.rocm_qk_norm_rope_f32(DEV, z, z, z, z, z, 1, 2, 1, 1, 32, EPS, positions=up(np.zeros(1, np.uint32)))


def test_capture_of_forward_and_backward():
    t, hq, hk, d = 40, 4, 2, 64
    q, k, qw, kw, inv, pos = case(1, t, hq, hk, d, 0, 41)
    b = [up(a) for a in (q, k, qw, kw, inv)]
    dq, dk, p = up(normal(q.shape, 1)), up(normal(k.shape, 2)), up(pos.astype(np.uint32))
    outs = [HipBuffer.empty(DEV, n) for n in (q.nbytes, k.nbytes, q.nbytes, k.nbytes, d * 4, d * 4)]
    ws = HipBuffer.empty(DEV, rocm.rocm_qk_norm_rope_backward_workspace_bytes(t, hq, hk, d))

    def step():
        rocm.rocm_qk_norm_rope_f32(DEV, *b, 1, t, hq, hk, d, EPS, 0, p, q_out=outs[0], k_out=outs[1])
        rocm.rocm_qk_norm_rope_backward_f32(DEV, dq, dk, *b, 1, t, hq, hk, d, EPS, 0, p, workspace=ws, grad_q=outs[2],
                                            grad_k=outs[3], grad_q_weight=outs[4], grad_k_weight=outs[5])

    step()
    want = [o.to_host().tobytes() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        for o in outs:
            o.tensor().fill_(0xFF)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert [o.to_host().tobytes() for o in outs] == want
        step()
        torch.cuda.synchronize()
        assert [o.to_host().tobytes() for o in outs] == want


@pytest.mark.parametrize("start", [2 ** 20, 2 ** 32 + 5])
def test_far_positions_without_a_table(start):
    """Positions past 32 bits and far past an f32's exact integers."""
    t, hq, hk, d = 5, 2, 1, 64
    q, k = normal((t, hq, d), 30), normal((t, hk, d), 31)
    w, inv = normal((d,), 32, 1.0, 0.1), rocm.rope_inv_freq_host(d, 10000.0)
    pos = start + np.arange(t)
    qo, ko = rocm.rocm_qk_norm_rope_f32(DEV, up(q), up(k), up(w), up(w), up(inv), 1, t, hq, hk, d, EPS, start)
    for got, x in ((qo, q), (ko, k)):
        want, tol = q4_ref.qk_norm_rope(x, w, pos, inv, EPS, False)
        q4_ref.assert_within(got.to_host(np.float32).reshape(x.shape), want, tol)


def test_two_backward_calls_at_once():
    """On two streams with workspaces of their own: each the same bits as alone."""
    t, hq, hk, d = 700, 4, 2, 64
    n = rocm.rocm_qk_norm_rope_backward_workspace_bytes(t, hq, hk, d)
    w, inv = up(normal((d,), 40, 1.0, 0.1)), up(rocm.rope_inv_freq_host(d, 10000.0))
    calls = []
    for i in range(2):
        a = [up(normal((t, h, d), 41 + 10 * i + j)) for j, h in enumerate((hq, hk, hq, hk))]
        out = dict(grad_q=HipBuffer.empty(DEV, t * hq * d * 4), grad_k=HipBuffer.empty(DEV, t * hk * d * 4), workspace=HipBuffer.empty(DEV, n))
        calls.append((a, out, torch.cuda.Stream()))

    def run(a, out):
        return rocm.rocm_qk_norm_rope_backward_f32(DEV, *a, w, w, inv, 1, t, hq, hk, d, EPS, **out)

    want = []
    for a, out, _ in calls:
        r = run(a, out)
        torch.cuda.synchronize()
        want.append([b.tensor().clone() for b in r])
    for _ in range(10):
        got = []
        for a, out, stream in calls:
            with torch.cuda.stream(stream):
                got.append(run(a, out))
        torch.cuda.synchronize()
        for g, x in zip(got, want):
            assert all(torch.equal(b.tensor()[:y.numel()], y) for b, y in zip(g, x))


@pytest.mark.parametrize("d,inter", [(96, False), (128, True)])
def test_more_than_the_caches_hold(d, inter):
    """Rows that are read past the caches: the same bits as from small calls on some of the tokens, and dw in 64 bits."""
    t, hq, hk = 7000, 32, 8
    gen = torch.Generator(device="cuda").manual_seed(50)
    q, k, dq, dk = (torch.randn(t, h, d, device="cuda", generator=gen) for h in (hq, hk, hq, hk))
    qw, kw, inv = normal((d,), 51, 1.0, 0.1), normal((d,), 52, 1.0, 0.1), rocm.rope_inv_freq_host(d, 10000.0)
    pos = np.random.default_rng(53).integers(0, 100000, t).astype(np.uint32)
    w = (up(qw), up(kw), up(inv))

    def call(lo, hi):
        b = [HipBuffer.from_tensor(x[lo:hi].contiguous()) for x in (q, k, dq, dk)]
        n = hi - lo
        y = rocm.rocm_qk_norm_rope_f32(DEV, b[0], b[1], *w, n, 1, hq, hk, d, EPS, 0, up(pos[lo:hi]), inter)
        g = rocm.rocm_qk_norm_rope_backward_f32(DEV, b[2], b[3], b[0], b[1], *w, n, 1, hq, hk, d, EPS, 0, up(pos[lo:hi]), inter)
        torch.cuda.synchronize()
        return [x.tensor(torch.float32) for x in (*y, *g)]

    big = call(0, t)
    for lo, hi in ((0, 50), (3333, 3400), (t - 31, t)):
        for i, (a, b) in enumerate(zip(big[:4], call(lo, hi)[:4])):
            row = (hq, hk)[i % 2] * d
            assert torch.equal(a[lo * row:hi * row], b[:(hi - lo) * row]), (i, lo)
    angle = torch.from_numpy(pos.astype(np.float64)).cuda()[:, None] * torch.from_numpy(inv.astype(np.float64)).cuda()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    for i, (x, dy) in enumerate(((q, dq), (k, dk))):
        x, dy = x.double(), dy.double()
        a, b = (dy[..., 0::2], dy[..., 1::2]) if inter else (dy[..., :d // 2], dy[..., d // 2:])
        g0, g1, both = a * c + b * s, b * c - a * s, a.abs() + b.abs()
        g, size = (torch.stack(p, -1).flatten(-2) if inter else torch.cat(p, -1) for p in ((g0, g1), (both, both)))
        n = x / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
        want, tol = (g * n).sum((0, 1)), ((192 + 64) * q4_ref.U + 3 * 2.0 ** -53 * 1e5) * (size * n.abs()).sum((0, 1))
        assert ((big[4 + i][:d].double() - want).abs() <= tol).all()
