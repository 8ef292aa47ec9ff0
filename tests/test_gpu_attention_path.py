"""The attention path's operators one after the other, as a program runs them: an attention layer that serves ragged
prompts and then decode steps (eager, and as a captured graph), and a training step through norm, projection and heads.

Every stage is checked against 64 bits on what the stage before it gave, so that a value next to a border of the 4-bit
codes falls on the same side in both."""
import numpy as np
import pytest

import oracle
import q4_ref
from inputs import normal, raw_packed
from q4_ref import U

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from kore_amd import rocm  # noqa: E402
from kore_amd.rocm import HipBuffer  # noqa: E402

DEV = 0
EPS = 1e-6
NOWHERE = 0xFFFFFFFF  # the slot of a padding token


def up(a):
    return HipBuffer.from_host(DEV, np.ascontiguousarray(a))


def u32(a):
    return np.ascontiguousarray(a, np.uint32)


class Layer:
    """Norm, BitLinear projection to Q, K and V, head norms with rotation in place in that buffer, cache, attention,
    BitLinear output."""

    def __init__(self, hidden, hq, hk, d, page, seqs, most, cap, interleaved=False):
        self.hidden, self.hq, self.hk, self.d, self.page, self.seqs, self.most = hidden, hq, hk, d, page, seqs, most
        self.interleaved, self.wide = interleaved, (hq + 2 * hk) * d
        self.pages = seqs * most + 1
        self.host = {"g": normal((hidden,), 1, 1.0, 0.1), "qw": normal((d,), 2, 1.0, 0.1), "kw": normal((d,), 3, 1.0, 0.1),
                     "inv": rocm.rope_inv_freq_host(d, 10000.0), "wqkv": raw_packed(self.wide, hidden, 4),
                     "sqkv": np.abs(normal((self.wide,), 5, 0.05, 0.01)), "wo": raw_packed(hidden, hq * d, 6),
                     "so": np.abs(normal((hidden,), 7, 0.05, 0.01))}
        self.w = {k: up(v) for k, v in self.host.items()}
        self.cache = HipBuffer.from_host(DEV, np.random.default_rng(8).integers(
            0, 256, rocm.rocm_kv_cache_q4_bytes(self.pages, page, hk, d)).astype(np.uint8))
        self.table = np.random.default_rng(9).permutation(self.pages)[:seqs * most].reshape(seqs, most)
        f32 = lambda n: HipBuffer.empty(DEV, n * 4)  # noqa: E731
        self.x, self.n, self.out, self.o = f32(cap * hidden), f32(cap * hidden), f32(cap * hidden), f32(cap * hq * d)
        self.t = torch.zeros(cap * self.wide, device="cuda")
        self.qkv = [HipBuffer.from_tensor(self.t[i * d:]) for i in (0, hq, hq + hk)]
        self.pos, self.slots, self.lens, self.starts = (HipBuffer.empty(DEV, n * 4) for n in (cap, cap, seqs, seqs + 1))
        self.pages_of = up(u32(self.table))
        self.ws = HipBuffer.empty(DEV, max([16] + [rocm.rocm_attention_q4_workspace_bytes(seqs, n, hq, hk, d, page, most)
                                                   for n in range(1, cap + 1)]))

    def give(self, x, pos, slots, lens, starts):
        for b, a in ((self.x, np.float32(x)), (self.pos, u32(pos)), (self.slots, u32(slots)), (self.lens, u32(lens)), (self.starts, u32(starts))):
            a = np.ascontiguousarray(a)
            b.tensor()[:a.nbytes].copy_(torch.from_numpy(a.reshape(-1).view(np.uint8)))
        torch.cuda.synchronize()

    def project(self, n):
        w, h = self.w, self.hidden
        rocm.rocm_rms_norm_f32(DEV, self.x, w["g"], n, h, EPS, self.n)
        rocm.rocm_bit_linear_f32(DEV, w["wqkv"], w["sqkv"], self.n, None, self.wide, n, h, self.qkv[0])

    def attend(self, n):
        w, (q, k, v), s = self.w, self.qkv, self.wide
        rocm.rocm_qk_norm_rope_f32(DEV, q, k, w["qw"], w["kw"], w["inv"], n, 1, self.hq, self.hk, self.d, EPS, 0, self.pos,
                                   self.interleaved, s, s, q, k, s, s)
        rocm.rocm_kv_cache_write_q4_f32(DEV, k, v, self.slots, self.cache, n, self.hk, self.d, self.pages, self.page, s, s)
        rocm.rocm_attention_q4_f32(DEV, q, self.cache, self.pages_of, self.lens, self.starts, self.seqs, n, self.hq, self.hk, self.d,
                                   self.pages, self.page, self.most, self.d ** -0.5, True, s, self.ws, self.o)
        rocm.rocm_bit_linear_f32(DEV, w["wo"], w["so"], self.o, None, self.hidden, n, self.hq * self.d, self.out)

    def slot(self, seq, i):
        return self.table[seq, i // self.page] * self.page + i % self.page

    def check(self, n, x, pos, slots, lens, starts, before):
        """Runs n tokens and compares each stage; before: the cache's bytes so far."""
        hq, hk, d = self.hq, self.hk, self.d
        self.give(x, pos, slots, lens, starts)
        self.o.tensor().fill_(0xFF)
        self.project(n)
        torch.cuda.synchronize()
        raw = self.t.cpu().numpy()[:n * self.wide].reshape(n, hq + 2 * hk, d)
        norm = oracle.rms_norm(np.float32(x), self.host["g"], EPS)
        want = oracle.bit_linear_forward(self.host["wqkv"], self.host["sqkv"], norm, None, self.wide, n, self.hidden)
        assert raw.reshape(n, -1).tobytes() == want.tobytes()
        self.attend(n)
        torch.cuda.synchronize()
        got = self.t.cpu().numpy()[:n * self.wide].reshape(n, hq + 2 * hk, d)
        p = np.asarray(pos)
        for name, a, b in (("q", 0, hq), ("k", hq, hq + hk)):
            want, tol = q4_ref.qk_norm_rope(raw[:, a:b], self.host[name + "w"], p, self.host["inv"], EPS, self.interleaved)
            q4_ref.assert_within(got[:, a:b], want, tol, name)
        assert (got[:, hq + hk:] == raw[:, hq + hk:]).all()
        cache = q4_ref.Cache(0, self.page, hk, d)
        cache.bytes = before.copy()
        cache.write(u32(slots), got[:, hq:hq + hk], got[:, hq + hk:])
        assert (self.bytes() == cache.bytes).all()
        want, tol = q4_ref.attention(got[:, :hq], cache, u32(self.table), u32(lens), u32(starts), d ** -0.5, True, np.zeros((n, hq, d)))
        o = self.o.to_host(np.float32)[:n * hq * d].reshape(n, hq, d)
        mine = np.arange(n) < int(starts[-1])
        q4_ref.assert_within(o[mine], want[mine], tol[mine], "attention")
        assert np.isnan(o[~mine]).all()  # left as they were
        return cache.bytes

    def bytes(self):
        return self.cache.to_host(np.uint8).reshape(self.pages, self.hk, -1)


@pytest.mark.parametrize("hidden,hq,hk,d,page,prompts,inter", [
    (160, 4, 2, 64, 16, [37, 5, 16], False), (96, 6, 2, 80, 32, [1, 70], True), (128, 4, 4, 128, 16, [33], False), (64, 8, 1, 32, 16, [17, 16, 15, 1], False)])
def test_prompts_then_decode(hidden, hq, hk, d, page, prompts, inter):
    """Ragged prompts in one batch, the second half of one of them in a chunk of its own, then decode steps with a sequence
    that leaves the batch (its row becomes padding)."""
    seqs, steps = len(prompts), 4
    most = max(prompts) // page + 2
    layer = Layer(hidden, hq, hk, d, page, seqs, most, sum(prompts) + 1, inter)
    r = np.random.default_rng(10)
    at, cache = np.zeros(seqs, int), layer.bytes()
    for part in range(2):
        new = [n // 2 if part == 0 else n - n // 2 for n in prompts]
        n = sum(new)
        if n == 0:
            continue
        pos = np.concatenate([np.arange(at[s], at[s] + new[s]) for s in range(seqs)])
        slots = np.concatenate([[layer.slot(s, i) for i in range(at[s], at[s] + new[s])] for s in range(seqs)])
        at += new
        cache = layer.check(n, r.standard_normal((n, hidden)), pos, slots, at, np.concatenate([[0], np.cumsum(new)]), cache)
    for step in range(steps):
        there = np.arange(seqs) < (seqs if step < 2 else max(1, seqs - 1))
        slots = [layer.slot(s, at[s]) if there[s] else NOWHERE for s in range(seqs)]
        pos = at.copy()
        at += there
        starts = np.concatenate([[0], np.cumsum(there)])
        cache = layer.check(seqs, r.standard_normal((seqs, hidden)), pos, slots, at * there, starts, cache)


def test_decode_step_as_a_graph():
    """A whole step captured once and replayed as contexts grow, a row turns into padding and comes back: bit for bit the
    eager step on the same cache, over contexts on either side of the length from which keys are cut in shares."""
    seqs, hidden = 3, 128
    layer = Layer(hidden, 8, 2, 64, 16, seqs, 160, seqs)
    r = np.random.default_rng(11)
    n = 2300
    for s in range(seqs):  # contexts of any values
        k, v = (torch.from_numpy(r.standard_normal((n, 2, 64), np.float32)).cuda() for _ in range(2))
        slots = up(u32([layer.slot(s, i) for i in range(n)]))
        rocm.rocm_kv_cache_write_q4_f32(DEV, HipBuffer.from_tensor(k), HipBuffer.from_tensor(v), slots, layer.cache, n, 2, 64, layer.pages, 16)

    def step():
        layer.project(seqs)
        layer.attend(seqs)

    lens = np.array([2290, 40, 0])
    layer.give(np.ones((seqs, hidden)), lens, [NOWHERE] * seqs, lens, np.arange(seqs + 1))
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(6):
        there = np.array([True, i % 3 != 1, True])
        slots = [layer.slot(s, lens[s]) if there[s] else NOWHERE for s in range(seqs)]
        x, pos = r.standard_normal((seqs, hidden)), lens.copy()
        lens += there
        layer.give(x, pos, slots, lens * there, np.arange(seqs + 1))
        before = layer.cache.tensor().clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [b.tensor().clone() for b in (layer.cache, layer.o, layer.out)]
        layer.cache.tensor().copy_(before)
        layer.o.tensor().fill_(0xFF)
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (layer.cache, layer.o, layer.out)):
            assert torch.equal(a, b.tensor())
        o = layer.o.to_host(np.float32).reshape(seqs, -1)
        assert (o[~there] == 0).all() and np.isfinite(o).all() and (o[there] != 0).any(-1).all()


def test_two_graphs_on_two_streams():
    """Two captured layers with caches and workspaces of their own, replayed at the same time on two streams."""
    both = []
    for i in range(2):
        layer = Layer(64, 4, 1, 128, 16, 2, 140, 2)
        r = np.random.default_rng(20 + i)
        k = torch.from_numpy(r.standard_normal((2200, 1, 128), np.float32)).cuda()
        for s in range(2):
            rocm.rocm_kv_cache_write_q4_f32(DEV, HipBuffer.from_tensor(k), HipBuffer.from_tensor(k), up(u32([layer.slot(s, j) for j in range(2200)])),
                                            layer.cache, 2200, 1, 128, layer.pages, 16)
        layer.give(r.standard_normal((2, 64)), [2200, 70], [layer.slot(0, 2200), layer.slot(1, 70)], [2201, 71], [0, 1, 2])
        layer.project(2)
        layer.attend(2)
        torch.cuda.synchronize()
        want = layer.out.tensor().clone()
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            layer.project(2)
            layer.attend(2)
        both.append((layer, want, stream, graph))
    for _ in range(5):
        for layer, _, _, _ in both:
            layer.out.tensor().fill_(0xFF)
        torch.cuda.synchronize()
        for _, _, stream, graph in both:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for layer, want, _, _ in both:
            assert torch.equal(layer.out.tensor(), want)


@pytest.mark.parametrize("hq,hk,d,tokens,inter", [(4, 2, 32, 19, False), (2, 1, 20, 33, True), (3, 3, 128, 9, False)])
def test_training_step_against_differences(hq, hk, d, tokens, inter):
    """loss = sum(q a) + sum(k b) behind RMSNorm, a projection and the head norms with rotation: the chain's gradients for
    the input, the projection and all weights, against differences of the loss in 64 bits along random directions.

    Off by: a projection's sums have as many roundings as terms, the head norms' gradient 256, the outer norm's as many as
    columns and 64; each relative to the sum of the absolute values of what is added, carried through the chain."""
    hidden, wide = 48, (hq + hk) * d
    host = {"x": normal((tokens, hidden), 1), "g": normal((hidden,), 2, 1.0, 0.1), "w": normal((hidden, wide), 3) / np.float32(hidden ** 0.5),
            "qw": normal((d,), 4, 1.0, 0.1), "kw": normal((d,), 5, 1.0, 0.1)}
    a, b = normal((tokens, hq, d), 6), normal((tokens, hk, d), 7)
    inv, pos = rocm.rope_inv_freq_host(d, 10000.0), np.arange(100, 100 + tokens)

    def norm64(p):
        return p["x"] / np.sqrt((p["x"] ** 2).mean(-1, keepdims=True) + EPS) * p["g"]

    def loss(p):
        y = (norm64(p) @ p["w"]).reshape(tokens, hq + hk, d)
        q, _ = q4_ref.qk_norm_rope(y[:, :hq], p["qw"], pos, inv, EPS, inter)
        k, _ = q4_ref.qk_norm_rope(y[:, hq:], p["kw"], pos, inv, EPS, inter)
        return (q * a).sum() + (k * b).sum()

    dev = {k: up(v) for k, v in host.items()}
    n = rocm.rocm_rms_norm_f32(DEV, dev["x"], dev["g"], tokens, hidden, EPS)
    nt, wt = n.tensor(torch.float32)[:tokens * hidden].view(tokens, hidden), dev["w"].tensor(torch.float32).view(hidden, wide)
    y = (nt @ wt).contiguous()
    dy = torch.empty_like(y)
    parts = [HipBuffer.from_tensor(t.view(-1)[i:]) for t in (y, dy) for i in (0, hq * d)]
    args = (dev["qw"], dev["kw"], up(inv), 1, tokens, hq, hk, d, EPS, 100, None, inter, wide, wide)
    rocm.rocm_qk_norm_rope_f32(DEV, *parts[:2], *args)
    r = rocm.rocm_qk_norm_rope_backward_f32(DEV, up(a), up(b), *parts[:2], *args, grad_q=parts[2], grad_k=parts[3], grad_q_stride=wide, grad_k_stride=wide)
    dw = nt.t().contiguous() @ dy
    dn = (dy @ wt.t().contiguous()).contiguous()
    dx, dg = rocm.rocm_rms_norm_backward_f32(DEV, HipBuffer.from_tensor(dn), dev["x"], dev["g"], tokens, hidden, EPS)
    torch.cuda.synchronize()
    got = {"x": dx.to_host(np.float32)[:tokens * hidden].reshape(tokens, hidden), "g": dg.to_host(np.float32)[:hidden], "w": dw.cpu().numpy(),
           "qw": r[2].to_host(np.float32)[:d], "kw": r[3].to_host(np.float32)[:d]}
    p64 = {k: v.astype(np.float64) for k, v in host.items()}
    # Absolute values carried through the chain.
    y64, size, tol = (norm64(p64) @ p64["w"]).reshape(tokens, hq + hk, d), {}, {}
    spread = np.abs(norm64(p64)) @ np.abs(p64["w"])  # what y's roundings are relative to
    sdy = np.zeros((tokens, hq + hk, d))
    for name, lo, hi, up_ in (("qw", 0, hq, a), ("kw", hq, hq + hk, b)):
        yy = y64[:, lo:hi]
        rms = 1.0 / np.sqrt((yy * yy).mean(-1, keepdims=True) + EPS)
        both, part = q4_ref._both(up_.astype(np.float64), inter), np.abs(yy * rms)
        u = both * np.abs(p64[name])
        # dx is of size rms (u + n mean(u n)); an error of y moves it by rms times that, relative to y's row
        sdy[:, lo:hi] = rms * (u + part * (u * part).mean(-1, keepdims=True))
        rel = (spread.reshape(tokens, -1, d)[:, lo:hi] * rms).max(-1, keepdims=True)
        sdy[:, lo:hi] *= 1.0 + 4.0 * rel
        size[name] = (both * part * (1.0 + 2.0 * rel)).sum((0, 1))
    sdy = sdy.reshape(tokens, wide)
    inv0 = 1.0 / np.sqrt((p64["x"] ** 2).mean(-1, keepdims=True) + EPS)
    size["w"], sdn = np.abs(norm64(p64)).T @ sdy, sdy @ np.abs(p64["w"]).T
    n0 = np.abs(p64["x"] * inv0)
    size["g"], ug = (sdn * n0).sum(0), sdn * np.abs(p64["g"])
    size["x"] = inv0 * (ug + n0 * (ug * n0).mean(-1, keepdims=True))
    steps = hidden + 256 + wide + hidden + 64 + tokens
    rng = np.random.default_rng(12)
    for name in host:
        for _ in range(3):
            v = rng.standard_normal(host[name].shape)
            h = 1e-5
            diff = (loss({**p64, name: p64[name] + h * v}) - loss({**p64, name: p64[name] - h * v})) / (2 * h)
            whole = (size[name] * np.abs(v)).sum()
            assert abs((got[name].astype(np.float64) * v).sum() - diff) <= (steps * U + 1e-8) * whole, name
