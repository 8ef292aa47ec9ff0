"""Cases of the attention path's operators: query/key norm with rotation and its backward, the 4-bit paged key/value
cache (write and read back), and attention over that cache.

With ``own`` false, ``run`` computes them in their plain form, from elementary torch operations in 32 bits; with
``own`` true it makes the calls that a program makes through ``kore_amd.rocm``.  Both take the same inputs: the cache
is the same bytes for both, in the layout below.

``norm_rope``           per head RMSNorm of Q and K (one weight of head_dim for all heads) and rotation, one pass;
                        the angle is position x inv_freq without a rounding to f32;
``norm_rope_backward``  its gradients for q, k and both weights;
``cache``               K and V of some tokens quantised into their slots, and read back from them;
``attention``           softmax(scale q k^T) v over each sequence's pages, query heads sharing key heads.

Cache layout, for ``page`` tokens a page (a multiple of 16) and blocks = ceil(head_dim / 32).  Every 32 values of a
head are a block: 32 E2M1 codes (sign, 2 exponent bits, 1 mantissa bit; the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) and
a scale byte b, the power of two 2^(b - 127), or NaN for b = 255.  Values past head_dim are zeros.  The bytes of
[page, kv head] are, one after the other,
    K codes   [page tokens][16 blocks bytes]: dimension 2j in the low half of byte j, 2j + 1 in the high half;
    V codes   [page / 16][4 token groups][4 blocks chunks][4 tokens][4 bytes]: a chunk is 8 dimensions of one token,
              token 4 g + i of its 16 in group g at place i, halves as in K;
    K scales  [page tokens][blocks];
    V scales  [page / 16][blocks][16 tokens].
The scale of a block is the smallest power of two, from 2^-100 on, with which its largest magnitude is at most 7 (2^126
at most, where magnitudes past 3 * 2^126 count as that); a code is the nearest magnitude, ties to the even code, past 6
the code of 6.  A block that holds an infinity or a NaN has scale byte 255 and codes of zero.
"""
import math

import torch

own = False

DEV = 0
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # One token of one layer, as a decode step of a single stream makes it.
        {"name": "norm_rope decode 1", "kind": "norm_rope", "batch": 1, "seq": 1, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "start": 4095, "interleaved": False, "fused": True, "positions": False},
        # A continuous-batching decode step: every token at its own far position, Q and K inside one projection's output.
        {"name": "norm_rope decode 45", "kind": "norm_rope", "batch": 45, "seq": 1, "q_heads": 16, "k_heads": 16,
         "head_dim": 64, "start": 0, "interleaved": True, "fused": True, "positions": True},
        # A training batch's forward, outputs apart from the inputs (which the backward needs).
        {"name": "norm_rope train 8x2048", "kind": "norm_rope", "batch": 8, "seq": 2048, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "start": 0, "interleaved": False, "fused": False, "positions": False},
        # The backward of a short, odd sequence.
        {"name": "norm_rope_backward 1x1023", "kind": "norm_rope_backward", "batch": 1, "seq": 1023, "q_heads": 16,
         "k_heads": 4, "head_dim": 96, "start": 0, "interleaved": False, "fused": True, "positions": False},
        # The backward of the training batch.
        {"name": "norm_rope_backward 8x2048", "kind": "norm_rope_backward", "batch": 8, "seq": 2048, "q_heads": 32,
         "k_heads": 8, "head_dim": 128, "start": 0, "interleaved": False, "fused": False, "positions": False},
        # A decode step's new tokens, one for each of the running sequences, into the cache and back.
        {"name": "cache 45 tokens", "kind": "cache", "tokens": 45, "kv_heads": 8, "head_dim": 128, "page": 16,
         "prompt": False},
        # A prompt's tokens into consecutive slots of its pages and back, as a prefill and a later dense pass do.
        {"name": "cache prompt 8192", "kind": "cache", "tokens": 8192, "kv_heads": 8, "head_dim": 128, "page": 64,
         "prompt": True},
        # A decode step of a single stream: few rows, so latency counts.
        {"name": "attention decode 1x2048", "kind": "attention", "seqs": 1, "kv": 2048, "q": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "causal": True},
        # A continuous-batching decode step over contexts of every length.
        {"name": "attention decode 45x8192", "kind": "attention", "seqs": 45, "kv": 8192, "q": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "causal": True},
        # Decode over very long contexts: the cache's bytes are the work.
        {"name": "attention decode 2x131072", "kind": "attention", "seqs": 2, "kv": 131072, "q": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True},
        # Ragged prompts whose earlier part is cached already, one key head for each query head.
        {"name": "attention chunks 5x1023", "kind": "attention", "seqs": 5, "kv": 2777, "q": 1023, "q_heads": 16,
         "kv_heads": 16, "head_dim": 64, "page": 16, "causal": True},
        # A whole prompt: the products are the work.
        {"name": "attention prompt 4096", "kind": "attention", "seqs": 1, "kv": 4096, "q": 4096, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["norm_rope", "norm_rope_backward", "cache", "attention", "attention", "attention"])
    if kind in ("norm_rope", "norm_rope_backward"):
        kh = rng.choice([1, 2, 4, 8])
        qh = kh * rng.choice([1, 2, 4])
        d = rng.choice([32, 64, 80, 96, 128, 256])
        seq = log(1, 2048)
        batch = log(1, max(1, min(64, (1 << 26) // (seq * (qh + kh) * d))))
        return {"kind": kind, "batch": batch, "seq": seq, "q_heads": qh, "k_heads": kh, "head_dim": d,
                "start": rng.choice([0, rng.randrange(100000)]), "interleaved": rng.random() < 0.5,
                "fused": rng.random() < 0.5, "positions": rng.random() < 0.3}
    if kind == "cache":
        return {"kind": kind, "tokens": log(1, 8192), "kv_heads": rng.choice([1, 2, 3, 4, 8]),
                "head_dim": rng.choice([32, 64, 80, 96, 128]), "page": rng.choice([16, 32, 64, 128]),
                "prompt": rng.random() < 0.5}
    kh, d = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 80, 96, 128, 256])
    qh = kh * rng.choice([1, 2, 3, 4, 5, 8])
    kv = log(1, 32768)
    q = min(kv, rng.choice([1, 1, 1, rng.randint(2, 8), log(9, 2048)]))
    most = min((1 << 28) // (kv * kh * d), (1 << 33) // (q * kv * qh))
    return {"kind": kind, "seqs": log(1, max(1, min(64, most))), "kv": kv, "q": q, "q_heads": qh, "kv_heads": kh,
            "head_dim": d, "page": rng.choice([16, 32, 64, 128]), "causal": rng.random() < 0.8}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda:%d" % DEV).manual_seed(seed)


def _normal(g, *shape, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device=g.device).normal_(mean, std, generator=g)


def _rope_table(head_dim):
    """1 / theta^(2i / D) rounded to f32."""
    i = torch.arange(head_dim // 2, dtype=torch.float64)
    return (THETA ** (-2.0 * i / head_dim)).to(torch.float32).to("cuda:%d" % DEV)


def _blocks(d):
    return (d + 31) // 32


def _page_bytes(page, d):
    """Bytes of one page of one key head."""
    return page * _blocks(d) * 34


_MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _quantise(x):
    """x [..., D] f32 -> codes [..., 16 blocks] uint8 and scale bytes [..., blocks] uint8, in 32 bits (every step but the
    choice of the code is exact)."""
    d, nb = x.shape[-1], _blocks(x.shape[-1])
    x = torch.nn.functional.pad(x, (0, nb * 32 - d)).view(*x.shape[:-1], nb, 32)
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, torch.zeros_like(x))
    amax = x.abs().amax(-1)
    # exponent of the least power of two that amax / 1.75 does not exceed, two below it the scale
    e = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 129).clamp(-100, 126)
    up = torch.ldexp(torch.ones_like(amax), -e)
    y = (x.clamp(-3.0 * 2.0 ** 126, 3.0 * 2.0 ** 126) * up[..., None]).abs()
    code = torch.zeros_like(y, dtype=torch.uint8)
    for edge, tie_up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (y >= edge) if tie_up else (y > edge)
    code += 8 * torch.signbit(x).to(torch.uint8)
    code = code.view(*x.shape[:-2], nb * 16, 2)
    scale = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code[..., 0] + 16 * code[..., 1], scale


def _dequantise(codes, scales, d):
    lut = torch.tensor(_MAGNITUDES + [-m for m in _MAGNITUDES], dtype=torch.float32, device=codes.device)
    v = torch.stack([lut[(codes & 15).to(torch.int32)], lut[(codes >> 4).to(torch.int32)]], -1).flatten(-2)
    s = torch.exp2(scales.to(torch.float32) - 127.0)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (v.view(*scales.shape, 32) * s[..., None]).flatten(-2)[..., :d]


def _parts(pages, page, d):
    """Views of pages [..., page bytes] as K codes [..., page, 16 nb], V codes [..., page/16, 4, 4 nb, 4, 4],
    K scales [..., page, nb] and V scales [..., page/16, nb, 16]."""
    nb, lead = _blocks(d), pages.shape[:-1]
    n = page * nb
    return (pages[..., :16 * n].unflatten(-1, (page, nb * 16)), pages[..., 16 * n:32 * n].unflatten(-1, (page // 16, 4, 4 * nb, 4, 4)),
            pages[..., 32 * n:33 * n].unflatten(-1, (page, nb)), pages[..., 33 * n:].unflatten(-1, (page // 16, nb, 16)))


def _fill(pages, page, k, v):
    """Whole pages [n, H, page bytes] from k, v [n * page, H, D]."""
    n, heads, d = pages.shape[0], pages.shape[1], k.shape[-1]
    nb = _blocks(d)
    kc, vc, ks, vs = _parts(pages, page, d)
    c, s = _quantise(k)
    kc.copy_(c.view(n, page, heads, nb * 16).transpose(1, 2))
    ks.copy_(s.view(n, page, heads, nb).transpose(1, 2))
    c, s = _quantise(v)
    vc.copy_(c.view(n, page // 16, 4, 4, heads, 4 * nb, 4).permute(0, 4, 1, 2, 5, 3, 6))
    vs.copy_(s.view(n, page // 16, 16, heads, nb).permute(0, 3, 1, 4, 2))


def _unfill(pages, page, d):
    """k, v [n * page, H, D] of whole pages [n, H, page bytes]."""
    n, heads = pages.shape[0], pages.shape[1]
    nb = _blocks(d)
    kc, vc, ks, vs = _parts(pages, page, d)
    k = _dequantise(kc, ks, d)
    v = _dequantise(vc.permute(0, 1, 2, 3, 5, 4, 6).reshape(n, heads, page, nb * 16), vs.transpose(-1, -2).reshape(n, heads, page, nb), d)
    return k.transpose(1, 2).reshape(n * page, heads, d), v.transpose(1, 2).reshape(n * page, heads, d)


def _lengths(case):
    """Keys and new tokens of each sequence: the first has the most, the others are spread down to a quarter of that."""
    part = [1.0 - 0.75 * (s * 0.6180339887 % 1.0) for s in range(case["seqs"])]
    kv = [math.ceil(case["kv"] * x) for x in part]
    return kv, [min(k, math.ceil(case["q"] * x)) for k, x in zip(kv, reversed(part[1:] + part[:1]))]


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind in ("norm_rope", "norm_rope_backward"):
        t, hq, hk, d = case["batch"] * case["seq"], case["q_heads"], case["k_heads"], case["head_dim"]
        i = {"qw": _normal(g, d, std=0.1, mean=1.0), "kw": _normal(g, d, std=0.1, mean=1.0)}
        # the projection's output: activations whose size differs from head to head
        size = _normal(g, 1, hq + 2 * hk, 1).exp()
        x = _normal(g, t, hq + 2 * hk, d) * size
        if case["fused"]:
            i["qkv"] = x
        else:
            i["q"], i["k"] = x[:, :hq].contiguous(), x[:, hq:hq + hk].contiguous()
        if case["positions"]:
            i["positions"] = torch.randint(0, 131072, (t,), device=g.device, generator=g, dtype=torch.int32)
        if kind == "norm_rope_backward":
            i["dq"], i["dk"] = _normal(g, t, hq, d), _normal(g, t, hk, d)
        return i
    d, page, heads = case["head_dim"], case["page"], case["kv_heads"]
    if kind == "cache":
        t = case["tokens"]
        used = (t + page - 1) // page if case["prompt"] else t
        pages = used + 3
        perm = torch.randperm(pages, device=g.device, generator=g)[:used]
        if case["prompt"]:  # consecutive tokens of a sequence in pages of any order, from the middle of the first one
            at = torch.arange(t, device=g.device) + (page // 3 if t % page else 0)
            at = at % (used * page)
            slots = perm[at // page] * page + at % page
        else:  # one token for each sequence, in a page of its own
            slots = perm * page + torch.randint(0, page, (t,), device=g.device, generator=g)
        return {"k": _normal(g, t, heads, d) * _normal(g, 1, heads, d, std=0.3, mean=1.0), "v": _normal(g, t, heads, d),
                "slots": slots.to(torch.int32), "cache": torch.zeros(pages, heads, _page_bytes(page, d), dtype=torch.uint8, device=g.device)}
    n = case["seqs"]
    kv, qn = _lengths(case)
    each = [(k + page - 1) // page for k in kv]
    pages = sum(each) + 2
    perm = torch.randperm(pages, device=g.device, generator=g)
    cache = torch.empty(pages, heads, _page_bytes(page, d), dtype=torch.uint8, device=g.device)
    table = torch.zeros(n, max(each), dtype=torch.int32, device=g.device)
    chan = _normal(g, 1, heads, d, std=0.3, mean=1.0)
    at = 0
    for s in range(n):
        ids = perm[at:at + each[s]]
        at += each[s]
        table[s, :each[s]] = ids.to(torch.int32)
        some = max(1, (1 << 24) // (page * heads * d))
        for j in range(0, each[s], some):
            m = min(some, each[s] - j)
            new = torch.empty(m, heads, cache.shape[2], dtype=torch.uint8, device=g.device)
            _fill(new, page, _normal(g, m * page, heads, d) * chan, _normal(g, m * page, heads, d))
            cache[ids[j:j + m]] = new
    starts = [sum(qn[:s]) for s in range(n + 1)]
    return {"q": _normal(g, starts[-1], case["q_heads"], d, std=1.5), "cache": cache, "table": table,
            "lens": torch.tensor(kv, dtype=torch.int32, device=g.device),
            "starts": torch.tensor(starts, dtype=torch.int32, device=g.device), "kv": kv, "q_at": starts}


def _q_and_k(case, i):
    if not case["fused"]:
        return i["q"], i["k"]
    hq, hk = case["q_heads"], case["k_heads"]
    return i["qkv"][:, :hq], i["qkv"][:, hq:hq + hk]


def _positions(case, i):
    if case["positions"]:
        return i["positions"].to(torch.int64)
    return (torch.arange(case["seq"], device=i["qw"].device) + case["start"]).repeat(case["batch"])


def prepare(case, seed):
    i, kind = _inputs(case, seed), case["kind"]
    s = {"case": case, "in": i}
    if kind in ("norm_rope", "norm_rope_backward"):
        i["inv"] = _rope_table(case["head_dim"])
    if own:
        from kore_amd import rocm
        from kore_amd.rocm import HipBuffer

        s["buf"] = {k: HipBuffer.from_tensor(v) for k, v in i.items() if isinstance(v, torch.Tensor)}
        t, dev = case.get("tokens"), i["cache" if "cache" in i else "inv"].device

        def empty(*shape):
            return torch.empty(shape, dtype=torch.float32, device=dev)

        if kind in ("norm_rope", "norm_rope_backward"):
            t, hq, hk, d = case["batch"] * case["seq"], case["q_heads"], case["k_heads"], case["head_dim"]
            s["stride"] = (hq + 2 * hk) * d if case["fused"] else 0
            if case["fused"]:
                s["buf"]["q"] = s["buf"]["qkv"]
                s["buf"]["k"] = HipBuffer.from_tensor(i["qkv"].view(-1)[hq * d:])
            s["out"] = {"q": empty(t, hq, d), "k": empty(t, hk, d)}
            if kind == "norm_rope_backward":
                s["out"]["qw"], s["out"]["kw"] = empty(d), empty(d)
                s["ws"] = HipBuffer.empty(DEV, max(16, rocm.rocm_qk_norm_rope_backward_workspace_bytes(t, hq, hk, d)))
        elif kind == "cache":
            s["out"] = {"k": empty(t, case["kv_heads"], case["head_dim"]), "v": empty(t, case["kv_heads"], case["head_dim"])}
        else:
            rows = i["q_at"][-1]
            s["out"] = {"o": empty(rows, case["q_heads"], case["head_dim"])}
            s["ws"] = HipBuffer.empty(DEV, max(16, rocm.rocm_attention_q4_workspace_bytes(
                case["seqs"], rows, case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], i["table"].shape[1])))
        s["obuf"] = {k: HipBuffer.from_tensor(v) for k, v in s["out"].items()}
    return s


# -------------------------------------------------------------- the two forms
def _run_own(s):
    from kore_amd import rocm

    c, b, o = s["case"], s["buf"], s["obuf"]
    kind = c["kind"]
    if kind == "norm_rope":
        rocm.rocm_qk_norm_rope_f32(DEV, b["q"], b["k"], b["qw"], b["kw"], b["inv"], c["batch"], c["seq"], c["q_heads"],
                                   c["k_heads"], c["head_dim"], EPS, c["start"], b.get("positions"), c["interleaved"],
                                   s["stride"], s["stride"], o["q"], o["k"])
    elif kind == "norm_rope_backward":
        rocm.rocm_qk_norm_rope_backward_f32(DEV, b["dq"], b["dk"], b["q"], b["k"], b["qw"], b["kw"], b["inv"], c["batch"],
                                            c["seq"], c["q_heads"], c["k_heads"], c["head_dim"], EPS, c["start"],
                                            b.get("positions"), c["interleaved"], s["stride"], s["stride"], s["ws"], o["q"],
                                            o["k"], o["qw"], o["kw"])
    elif kind == "cache":
        pages = s["in"]["cache"].shape[0]
        rocm.rocm_kv_cache_write_q4_f32(DEV, b["k"], b["v"], b["slots"], b["cache"], c["tokens"], c["kv_heads"],
                                        c["head_dim"], pages, c["page"])
        rocm.rocm_kv_cache_read_q4_f32(DEV, b["cache"], b["slots"], c["tokens"], c["kv_heads"], c["head_dim"], pages,
                                       c["page"], o["k"], o["v"])
    else:
        rocm.rocm_attention_q4_f32(DEV, b["q"], b["cache"], b["table"], b["lens"], b["starts"], c["seqs"],
                                   s["in"]["q_at"][-1], c["q_heads"], c["kv_heads"], c["head_dim"],
                                   s["in"]["cache"].shape[0], c["page"], s["in"]["table"].shape[1],
                                   c["head_dim"] ** -0.5, c["causal"], workspace=s["ws"], out=o["o"])
    return s["out"]


def _rotate(x, cos, sin, interleaved):
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    r0, r1 = a * cos - b * sin, a * sin + b * cos
    return torch.stack([r0, r1], -1).flatten(-2) if interleaved else torch.cat([r0, r1], -1)


def _angles(case, i):
    a = _positions(case, i).double()[:, None] * i["inv"].double()
    return torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]


def run(s):
    if own:
        return _run_own(s)
    c, i = s["case"], s["in"]
    kind = c["kind"]
    if kind == "norm_rope":
        cos, sin = _angles(c, i)
        out = {}
        for name, x in zip(("q", "k"), _q_and_k(c, i)):
            y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * i[name + "w"]
            out[name] = _rotate(y, cos, sin, c["interleaved"])
        return out
    if kind == "norm_rope_backward":
        cos, sin = _angles(c, i)
        out = {}
        for name, x in zip(("q", "k"), _q_and_k(c, i)):
            dy = _rotate(i["d" + name], cos, -sin, c["interleaved"])  # back through the rotation
            inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            n = x * inv
            out[name + "w"] = (dy * n).sum((0, 1), dtype=torch.float64).float()
            dn = dy * i[name + "w"]
            out[name] = inv * (dn - n * (dn * n).mean(-1, keepdim=True))
        return out
    d, page = c["head_dim"], c["page"]
    if kind == "cache":
        cache, slots = i["cache"], i["slots"].to(torch.int64)
        p, at = slots // page, slots % page
        kc, vc, ks, vs = _parts(cache, page, d)
        nb = _blocks(d)
        codes, scales = _quantise(i["k"])
        kc[p, :, at], ks[p, :, at] = codes, scales
        codes, scales = _quantise(i["v"])
        vc[p, :, at // 16, at % 16 // 4, :, at % 4] = codes.unflatten(-1, (4 * nb, 4))
        vs[p, :, at // 16, :, at % 16] = scales
        return {"k": _dequantise(kc[p, :, at], ks[p, :, at], d),
                "v": _dequantise(vc[p, :, at // 16, at % 16 // 4, :, at % 4].flatten(-2), vs[p, :, at // 16, :, at % 16], d)}
    group = c["q_heads"] // c["kv_heads"]
    out = torch.empty_like(i["q"])
    for n in range(c["seqs"]):
        kv, q0, q1 = i["kv"][n], i["q_at"][n], i["q_at"][n + 1]
        ids = i["table"][n, :(kv + page - 1) // page].to(torch.int64)
        k, v = _unfill(i["cache"][ids], page, d)
        k, v = k[:kv].transpose(0, 1), v[:kv].transpose(0, 1)  # [heads, kv, D]
        last = torch.arange(kv - (q1 - q0), kv, device=k.device) if c["causal"] else torch.full((q1 - q0,), kv, device=k.device)
        hidden = torch.arange(kv, device=k.device) > last[:, None]
        for h in range(c["kv_heads"]):
            q = i["q"][q0:q1, h * group:(h + 1) * group].transpose(0, 1)  # [group, rows, D]
            x = torch.matmul(q, k[h].t().contiguous()) * d ** -0.5
            x = x.masked_fill(hidden, -math.inf)
            e = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(e, v[h].contiguous()) / e.sum(-1, keepdim=True)
            out[q0:q1, h * group:(h + 1) * group] = o.transpose(0, 1)
    return {"o": out}


def work(case):
    """Inputs read once and outputs written once; a multiply and an add are two."""
    kind = case["kind"]
    if kind in ("norm_rope", "norm_rope_backward"):
        n = case["batch"] * case["seq"] * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        extra = 4 * case["batch"] * case["seq"] * case["positions"] + 10 * case["head_dim"]
        return {"bytes": (8 if kind == "norm_rope" else 12) * n + extra, "flops": (8 if kind == "norm_rope" else 18) * n}
    d, heads = case["head_dim"], case["kv_heads"]
    if kind == "cache":  # the values in, their codes and scales, and the values out
        n = case["tokens"] * heads
        return {"bytes": n * (16 * d + 2 * 17 * _blocks(d)) + 4 * case["tokens"], "flops": 10 * n * d}
    total_kv, rows, pairs = 0, 0, 0  # pairs of a row and a key that it sees
    for kv, q in zip(*_lengths(case)):
        total_kv, rows = total_kv + kv, rows + q
        pairs += q * (kv - q) + q * (q + 1) // 2 if case["causal"] else q * kv
    return {"bytes": total_kv * heads * 2 * 17 * _blocks(d) + 8 * rows * case["q_heads"] * d,
            "flops": 4 * pairs * case["q_heads"] * d}


# -------------------------------------------------------------- in 64 bits
def _cached64(cache, page, d, slots, value):
    """K (value False) or V of the slots [T] in 64 bits, [T, H, D], byte by byte from the layout's definition."""
    nb, dev = _blocks(d), cache.device
    flat = cache.view(-1)
    heads, size = cache.shape[1], cache.shape[2]
    p, t = (slots // page)[:, None, None], (slots % page)[:, None, None]
    h = torch.arange(heads, device=dev)[None, :, None]
    x = torch.arange(d, device=dev)[None, None, :]
    base = (p * heads + h) * size
    if value:
        code = base + 16 * page * nb + ((((t // 16) * 4 + t % 16 // 4) * 4 * nb + x // 8) * 4 + t % 4) * 4 + x % 8 // 2
        scale = base + 33 * page * nb + (t // 16 * nb + x // 32) * 16 + t % 16
    else:
        code = base + t * 16 * nb + x // 2
        scale = base + 32 * page * nb + t * nb + x // 32
    c = (flat[code].to(torch.int32) >> (4 * (x % 2)).to(torch.int32)) & 15
    sign, e, m = (c >> 3).double(), ((c >> 1) & 3).double(), (c & 1).double()
    mag = torch.where(e == 0, m * 0.5, (1.0 + 0.5 * m) * torch.pow(torch.full_like(e, 2.0), e - 1.0))
    b = flat[scale].double()
    return torch.where(b == 255, math.nan, (1.0 - 2.0 * sign) * mag * torch.pow(torch.full_like(b, 2.0), b - 127.0))


def _nearest64(x):
    """x [T, H, D] f32 as the cache holds it, in 64 bits: the nearest of the block's values, the even code of two."""
    d, nb = x.shape[-1], _blocks(x.shape[-1])
    w = torch.nn.functional.pad(x.double(), (0, nb * 32 - d)).unflatten(-1, (nb, 32))
    amax = w.abs().amax(-1, keepdim=True)
    step = torch.pow(torch.full_like(amax, 2.0), torch.ceil(torch.log2(torch.clamp(amax, min=1e-300) / 7.0)).clamp(-100, 126))
    step = torch.where(amax > 7.0 * step, 2.0 * step, torch.where((amax <= 3.5 * step) & (step > 2.0 ** -100), 0.5 * step, step))
    # the even code wins a tie: order the candidates by distance, then the even codes first
    best, far = torch.zeros_like(w), torch.full_like(w, math.inf)
    y = (w / step).abs()
    for c in (0, 2, 4, 6, 1, 3, 5, 7):
        dist = (y - _MAGNITUDES[c]).abs()
        best, far = torch.where(dist < far, torch.full_like(w, _MAGNITUDES[c]), best), torch.minimum(dist, far)
    return (torch.sign(w) * best * step).flatten(-2)[..., :d]


def exact(case, seed):
    kind, i = case["kind"], _inputs(case, seed)
    if kind in ("norm_rope", "norm_rope_backward"):
        inv_freq = _rope_table(case["head_dim"]).double()
        # a pair as a complex number, turned by the angle
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=inv_freq.device), _positions(case, i).double()[:, None] * inv_freq)[:, None, :]
        d, out = case["head_dim"], {}
        for name, x in zip(("q", "k"), _q_and_k(case, i)):
            leaf, w = x.double().requires_grad_(), i[name + "w"].double().requires_grad_()
            y = leaf * torch.rsqrt(leaf.square().mean(-1, keepdim=True) + EPS) * w
            pairs = y.unflatten(-1, (d // 2, 2)) if case["interleaved"] else y.unflatten(-1, (2, d // 2)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            if kind == "norm_rope":
                out[name] = y.detach()
            else:
                out[name], out[name + "w"] = torch.autograd.grad(y, (leaf, w), i["d" + name].double())
        return out
    if kind == "cache":
        return {"k": _nearest64(i["k"]), "v": _nearest64(i["v"])}
    d, page, group = case["head_dim"], case["page"], case["q_heads"] // case["kv_heads"]
    o = torch.empty(i["q"].shape, dtype=torch.float64, device=i["q"].device)
    for s in range(case["seqs"]):
        kv, q0, q1 = i["kv"][s], i["q_at"][s], i["q_at"][s + 1]
        rows = q1 - q0
        at = torch.arange(kv, device=o.device)
        slots = i["table"][s].to(torch.int64)[at // page] * page + at % page
        k, v = _cached64(i["cache"], page, d, slots, False), _cached64(i["cache"], page, d, slots, True)
        seen = (at[None, :] <= torch.arange(rows, device=o.device)[:, None] + (kv - rows)) if case["causal"] else None
        for h in range(case["q_heads"]):
            x = i["q"][q0:q1, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(d)
            if seen is not None:
                x = torch.where(seen, x, -math.inf)
            o[q0:q1, h] = torch.softmax(x, -1) @ v[:, h // group].contiguous()
    return {"o": o}
