"""The decode-step operators around the 4-bit KV cache, as they are measured: the rotary append into the cache, the
attention over it (whole context, or a sliding window with sinks) and the sampler with temperature, top-k, top-p and
min-p. `run` computes an operator's plain form with elementary torch operations, or, with `own`, makes the library's
calls on the same data."""
import ctypes as C
import math

import torch

own = False

BLOCK, TILE = 32, 16        # values of a quantised block; positions of a cache tile
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    def attn(name, seqs, rows, heads, kv_heads, hd, start, window=0, sinks=0, pad=0):
        return dict(name=name, op="attention", seqs=seqs, rows=rows, heads=heads, kv_heads=kv_heads, hd=hd, start=start,
                    window=window, sinks=sinks, pad=pad)

    def append(name, seqs, rows, heads, kv_heads, hd, rope, neox, start):
        return dict(name=name, op="append", seqs=seqs, rows=rows, heads=heads, kv_heads=kv_heads, hd=hd, rope=rope, neox=neox,
                    start=start)

    def sample(name, rows, vocab, mix):
        return dict(name=name, op="sample", rows=rows, vocab=vocab, mix=mix)

    return [
        # one token of a single user's reply on the 70B head layout: a launch's latency
        append("append_1", 1, 1, 64, 8, 128, 128, False, 1100),
        # a decode step of 61 requests on the mixture-of-experts head layout, half of each head rotated
        append("append_61", 61, 1, 32, 4, 128, 64, True, 700),
        # a prompt of 2048 tokens
        append("append_2048", 1, 2048, 64, 8, 128, 128, False, 0),
        # one token of the smallest configuration, a short reply
        attn("attend_1_short", 1, 1, 8, 8, 64, 299),
        # one token at the end of a long document
        attn("attend_1_long", 1, 1, 64, 8, 128, 131000),
        # eight users mid-reply, their lengths apart, one slot of the batch unused
        attn("attend_8", 8, 1, 64, 8, 128, 4100, pad=1),
        # a full batch of chats that see a window and the first tokens
        attn("attend_64_window", 64, 1, 32, 8, 128, 6000, window=1024, sinks=4),
        # a prompt
        attn("attend_prompt", 1, 1500, 64, 8, 128, 0),
        # the next part of a long prompt, with a window
        attn("attend_chunk_window", 1, 512, 32, 4, 128, 20001, window=4096, sinks=16),
        # one row of the benchmark vocabularies; a batch of rows with options of their own
        sample("sample_1", 1, 32000, "topk"),
        sample("sample_8", 8, 151936, "mixed"),
        sample("sample_64", 64, 128256, "mixed"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("append", "attention", "attention", "sample"))
    heads, kv_heads, hd = rng.choice(((8, 8, 64), (32, 8, 128), (64, 8, 128), (32, 4, 128), (16, 1, 96), (8, 4, 256), (24, 24, 64), (20, 4, 128)))
    if op == "append":
        seqs = rng.choice((1, log(1, 64)))
        return dict(op=op, seqs=seqs, rows=log(1, 2048 // seqs), heads=heads, kv_heads=kv_heads, hd=hd,
                    rope=rng.choice((hd, hd // 2, hd // 4, 0)), neox=rng.random() < 0.5, start=rng.randrange(0, 4000))
    if op == "sample":
        return dict(op=op, rows=log(1, 64), vocab=log(500, 128256), mix=rng.choice(("topk", "topp", "minp", "plain", "mixed", "masked")))
    window, sinks = (0, 0) if rng.random() < 0.5 else (log(16, 4096), rng.choice((0, 1, 4, 16)))
    if rng.random() < 0.6:
        seqs = log(1, 64)
        return dict(op=op, seqs=seqs, rows=1, heads=heads, kv_heads=kv_heads, hd=hd, start=log(1, 60000 // seqs),
                    window=window, sinks=sinks, pad=rng.choice((0, 0, seqs // 5)))
    seqs = rng.choice((1, 1, 3))
    rows = log(2, 1000 // seqs)
    return dict(op=op, seqs=seqs, rows=rows, heads=heads, kv_heads=kv_heads, hd=hd, start=rng.choice((0, log(1, 4000 // seqs))),
                window=window, sinks=sinks, pad=0)


def _starts(case):
    """Where each sequence's rows begin: spread below case["start"], the first of them at it."""
    n, s = case["seqs"], case["start"]
    return [s - (s * (7 * i % 16)) // 24 for i in range(n)]


def _capacity(case):
    return (case["start"] + case["rows"] + TILE - 1) // TILE * TILE


def _visible(case):
    """Positions seen by each sequence's rows together, and pairs (row, position) in all."""
    seen, pairs = 0, 0
    for i, s in enumerate(_starts(case)):
        if i >= case["seqs"] - case["pad"]:
            continue
        lo = None
        for r in range(case["rows"]):
            p = s + r
            first = max(0, p - case["window"] + 1) if case["window"] else 0
            lo = first if lo is None else lo
            pairs += p + 1 - first + min(case["sinks"], first)
        seen += s + case["rows"] - lo + min(case["sinks"], lo)
    return seen, pairs


def work(case):
    if case["op"] == "sample":
        return dict(bytes=case["rows"] * (4.0 * case["vocab"] + 44), flops=0.0)
    t = case["seqs"] * case["rows"]
    qd, kd = case["heads"] * case["hd"], case["kv_heads"] * case["hd"]
    if case["op"] == "append":
        # q in and out, k and v in, the rows of the table, the codes and scales out and back, and the values they stand for
        return dict(bytes=t * (8.0 * qd + 8.0 * kd + 4.0 * case["rope"] + 2 * 2 * 0.5625 * kd + 4.0 * kd + 12), flops=0.0)
    seen, pairs = _visible(case)
    return dict(bytes=seen * kd * 2 * 0.5625 + 8.0 * t * qd + 12 * t, flops=4.0 * qd * pairs)


# ---------------------------------------------------------------------------------------------------------------------
# the cache's bytes
# ---------------------------------------------------------------------------------------------------------------------
# A tile holds 16 positions of one KV head: the keys' codes, the values' codes (each 8 * hd bytes of 32-bit words of
# eight 4-bit codes), then the keys' and the values' fp16 scales [16][hd / 32].
def _split(cache, hd):
    """The four parts of tiles [..., 18 * hd]."""
    return cache[..., :8 * hd], cache[..., 8 * hd:16 * hd], cache[..., 16 * hd:17 * hd], cache[..., 17 * hd:]


def _decode(cache, hd):
    """float32 keys and values [seqs, positions, kv_heads, hd] of tiles [seqs, tiles, kv_heads, 18 * hd]."""
    n, tiles, kvh = cache.shape[:3]
    nb = hd // BLOCK
    w = min(4, nb)
    kc, vc, ks, vs = _split(cache, hd)

    def nibbles(x):
        x = torch.stack((x & 15, x >> 4), -1)
        # plane, half, g, c, block in the plane, nibble
        return x.reshape(n, tiles, kvh, nb // w, 2, 8, 4, w, 8).float() - 8

    def scales(x):
        return x.contiguous().view(torch.float16).reshape(n, tiles, kvh, TILE, nb, 1).float()

    k = nibbles(kc).permute(0, 1, 2, 4, 5, 3, 7, 6, 8).reshape(n, tiles, kvh, TILE, nb, BLOCK) * scales(ks)
    v = nibbles(vc).reshape(n, tiles, kvh, nb // w, 2, 8, 4, w, 2, 4)      # ..., odd position, dim
    v = v.permute(0, 1, 2, 4, 6, 8, 3, 7, 5, 9).reshape(n, tiles, kvh, TILE, nb, BLOCK) * scales(vs)
    return tuple(x.permute(0, 1, 3, 2, 4, 5).reshape(n, tiles * TILE, kvh, hd) for x in (k, v))


def _quantise(x):
    """Codes (uint8, 0 to 15) and fp16 scales of blocks of 32: in 64 bits, where a code's border falls."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) / -8).to(torch.float32).to(torch.float16)
    inv = torch.where(d == 0, torch.zeros_like(hi), 1 / d.double())
    return torch.floor(b * inv[..., None] + 8.5).clamp(0, 15).to(torch.uint8).flatten(-2), d


def _pack(kc, kd, vc, vd):
    """Tiles [seqs, tiles, kv_heads, 18 * hd] of codes [seqs, positions, kv_heads, hd] and scales [..., hd / 32]."""
    n, p, kvh, hd = kc.shape
    nb, tiles = hd // BLOCK, p // TILE
    w = min(4, nb)

    def words(x):
        return (x[..., 0::2] | (x[..., 1::2] << 4)).reshape(n, tiles, kvh, 8 * hd)

    # [seq, tile, half, g, head, plane, block, c, nibble]
    k = kc.reshape(n, tiles, 2, 8, kvh, nb // w, w, 4, 8).permute(0, 1, 4, 5, 2, 3, 7, 6, 8)
    # [seq, tile, half, c, odd, head, plane, block, g, nibble]
    v = vc.reshape(n, tiles, 2, 4, 2, kvh, nb // w, w, 8, 4).permute(0, 1, 5, 6, 2, 8, 3, 7, 4, 9)

    def scales(x):
        return x.reshape(n, tiles, TILE, kvh, nb).permute(0, 1, 3, 2, 4).contiguous().view(torch.uint8).reshape(n, tiles, kvh, hd)

    return torch.cat((words(k), words(v), scales(kd), scales(vd)), -1)


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------
def _filled(case, gen):
    """A cache whose keys and values have the spread of a model's: a few strong key channels, the first tokens' large."""
    kvh, hd, cap = case["kv_heads"], case["hd"], _capacity(case)
    cache = torch.empty(case["seqs"], cap // TILE, kvh, 18 * hd, dtype=torch.uint8, device=DEV)
    chan = 1 + 4 * (torch.rand(kvh, hd, generator=gen, device=DEV) > 0.96)
    for i in range(case["seqs"]):
        for at in range(0, cap, 16384):
            m = min(16384, cap - at)
            k = torch.randn(1, m, kvh, hd, generator=gen, device=DEV) * chan
            v = torch.randn(1, m, kvh, hd, generator=gen, device=DEV)
            cache[i, at // TILE:(at + m) // TILE] = _pack(*_quantise(k), *_quantise(v))[0]
    return cache


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "sample":
        return _prepare_sample(case, gen, s)
    kvh, hd, heads = case["kv_heads"], case["hd"], case["heads"]
    n, r = case["seqs"], case["rows"]
    pos = torch.tensor(_starts(case), dtype=torch.int32)[:, None] + torch.arange(r, dtype=torch.int32)
    if case.get("pad"):
        pos[n - case["pad"]:] = -1
    s["pos"] = pos.reshape(-1).to(DEV)
    s["capacity"] = _capacity(case)
    s["q"] = torch.randn(n * r, heads, hd, generator=gen, device=DEV)
    if case["op"] == "append":
        s["cache"] = torch.zeros(n, s["capacity"] // TILE, kvh, 18 * hd, dtype=torch.uint8, device=DEV)
        s["k"] = torch.randn(n * r, kvh, hd, generator=gen, device=DEV)
        s["v"] = torch.randn(n * r, kvh, hd, generator=gen, device=DEV)
        s["q_out"] = torch.empty_like(s["q"])
        s["k16"] = torch.empty(n * r, kvh, hd, dtype=torch.float16, device=DEV)
        s["v16"] = torch.empty_like(s["k16"])
        # the model's table of angles: 500000 to the -2i / dims, stretched four times over the trained length
        i = torch.arange(case["rope"] // 2, dtype=torch.float64, device=DEV)
        angle = torch.arange(s["capacity"], dtype=torch.float64, device=DEV)[:, None] * 0.25 * 500000.0 ** (-2 * i / max(1, case["rope"]))
        s["table"] = torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()
    else:
        s["cache"] = _filled(case, gen)
        s["out"] = torch.empty_like(s["q"])
        # one workspace for every call, as a server keeps it: the tickets in its first bytes start at zero
        s["ws"] = torch.zeros(256 << 20, dtype=torch.uint8, device=DEV)
    s["scale"] = hd ** -0.5
    row_cache = torch.arange(n, device=DEV).repeat_interleave(r) * s["cache"][0].numel() + s["cache"].data_ptr()
    s["caches"] = row_cache.contiguous()
    return s


def _prepare_sample(case, gen, s):
    rows, v, mix = case["rows"], case["vocab"], case["mix"]
    x = torch.randn(rows, v, generator=gen, device=DEV) * 2.2
    # a model's row: a handful of ids that stand out
    lead = torch.randint(0, v, (rows, 12), generator=gen, device=DEV)
    x.scatter_(1, lead, 9 + 3 * torch.rand(rows, 12, generator=gen, device=DEV))
    if mix in ("masked", "mixed"):      # a grammar that leaves a twentieth of the ids, on some rows
        off = torch.rand(rows, v, generator=gen, device=DEV) > 0.05
        off[:, 0] = False
        if mix == "mixed":
            off[torch.arange(rows, device=DEV) % 5 != 3] = False
        x = x.masked_fill(off, float("-inf"))
    u = torch.rand(rows, 4, generator=gen, device=DEV, dtype=torch.float64)
    r = torch.arange(rows, device=DEV)
    kind = {"topk": 0, "topp": 1, "minp": 2, "plain": 3, "masked": 1}.get(mix)
    kind = r % 6 if kind is None else torch.full_like(r, kind)
    s["x"] = x.contiguous()
    s["temperature"] = torch.where(kind == 5, 0.0, 0.6 + 0.6 * u[:, 0])
    s["top_k"] = torch.where((kind == 0) | (kind == 4), (1 + u[:, 1] * 100).long(), torch.zeros_like(r))
    s["top_p"] = torch.where((kind == 1) | (kind == 4), 0.5 + 0.49 * u[:, 2], torch.ones_like(u[:, 2]))
    s["min_p"] = torch.where((kind == 2) | (kind == 4), 0.01 + 0.1 * u[:, 1], torch.zeros_like(u[:, 1]))
    s["draw"] = u[:, 3].contiguous()
    # the same five numbers a row, as the library takes them
    s["opts"] = torch.stack((s["temperature"], s["top_p"], s["min_p"], s["draw"]), 1).view(torch.int64)
    s["opts"] = torch.cat((s["opts"], s["top_k"][:, None]), 1).contiguous()
    s["ids"] = torch.empty(rows, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"append": _append, "attention": _attention, "sample": _sample}[s["case"]["op"]](s)


def _run_own(s):
    from windlass_b200 import _lib
    lib, c = _lib.lib(), s["case"]

    def p(t):
        return C.c_void_p(t.data_ptr())

    if c["op"] == "sample":
        v = c["vocab"]
        _lib.check(lib.wl_sample_rows(p(s["x"]), v, v, c["rows"], p(s["opts"]), p(s["ids"]), None))
        return s["ids"]
    t = c["seqs"] * c["rows"]
    if c["op"] == "append":
        _lib.check(lib.wl_kv4_append(p(s["q"]), p(s["q_out"]), p(s["k"]), p(s["v"]), t, c["heads"], c["kv_heads"], c["hd"],
                                     p(s["table"]), c["rope"], int(c["neox"]), p(s["caches"]), p(s["pos"]), s["capacity"], None))
        _lib.check(lib.wl_kv4_read(p(s["caches"]), p(s["pos"]), t, c["kv_heads"], c["hd"], s["capacity"], p(s["k16"]), p(s["v16"]), None))
        return s["q_out"], s["k16"], s["v16"]
    _lib.check(lib.wl_kv4_attention(p(s["q"]), t, c["rows"], c["heads"], c["kv_heads"], c["hd"], s["scale"], p(s["caches"]),
                                    p(s["pos"]), s["capacity"], c["window"], c["sinks"], p(s["out"]), p(s["ws"]), s["ws"].numel(), None))
    return s["out"]


def _rotate(x, cs, rope, neox):
    """x [rows, heads, hd] with its first `rope` dims turned by cs [rows, 1, rope / 2, 2]; in x's type."""
    if not rope:
        return x
    a = x[..., :rope]
    x0, x1 = (a[..., :rope // 2], a[..., rope // 2:]) if neox else (a[..., 0::2], a[..., 1::2])
    c, sn = cs[..., 0], cs[..., 1]
    y0, y1 = x0 * c - x1 * sn, x0 * sn + x1 * c
    y = torch.cat((y0, y1), -1) if neox else torch.stack((y0, y1), -1).flatten(-2)
    return torch.cat((y, x[..., rope:]), -1)


def _append(s):
    c = s["case"]
    n, r, hd, kvh = c["seqs"], c["rows"], c["hd"], c["kv_heads"]
    pos = s["pos"].long()
    cs = s["table"][pos][:, None]
    q = _rotate(s["q"], cs, c["rope"], c["neox"])
    kc, kd = _quantise(_rotate(s["k"].double(), cs.double(), c["rope"], c["neox"]))
    vc, vd = _quantise(s["v"])
    # into the cache: each row's position of its own tile
    seq = torch.arange(n, device=pos.device).repeat_interleave(r)
    nb, tile, half, g = hd // BLOCK, pos // TILE, pos % TILE // 8, pos % 8
    w = min(4, nb)
    kt, vt, ks, vs = _split(s["cache"], hd)
    kw = kc.reshape(n * r, kvh, nb // w, w, 4, 4, 2).transpose(3, 4)                     # row, head, plane, c, block, byte, nibble
    vw = vc.reshape(n * r, kvh, nb // w, w, 8, 2, 2).transpose(3, 4)                     # row, head, plane, g, block, byte, nibble
    kt.unflatten(-1, (nb // w, 2, 8, 4, w, 4))[seq, tile, :, :, half, g] = kw[..., 0] | (kw[..., 1] << 4)
    vt.unflatten(-1, (nb // w, 2, 8, 4, w, 2, 2))[seq, tile, :, :, half, :, g // 2, :, g % 2] = vw[..., 0] | (vw[..., 1] << 4)
    ks.unflatten(-1, (TILE, 2 * nb))[seq, tile, :, pos % TILE] = kd.view(torch.uint8)
    vs.unflatten(-1, (TILE, 2 * nb))[seq, tile, :, pos % TILE] = vd.view(torch.uint8)

    def values(codes, d):
        return ((codes.unflatten(-1, (-1, BLOCK)).float() - 8) * d[..., None].float()).flatten(-2).half()

    return q, values(kc, kd), values(vc, vd)


def _attention(s):
    c = s["case"]
    n, r, hd, kvh, heads = c["seqs"], c["rows"], c["hd"], c["kv_heads"], c["heads"]
    g = heads // kvh
    k, v = _decode(s["cache"], hd)
    q = s["q"].reshape(n, r, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * r, hd)
    score = (q @ k.permute(0, 2, 3, 1)) * s["scale"]
    pos = s["pos"].reshape(n, 1, 1, r, 1).long()
    j = torch.arange(k.shape[1], device=k.device)
    seen = j <= pos
    if c["window"]:
        seen = seen & ((j > pos - c["window"]) | (j < c["sinks"]))
    score = score.reshape(n, kvh, g, r, -1).masked_fill(~seen, float("-inf"))
    m = score.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(score - m)
    del score
    out = e.reshape(n, kvh, g * r, -1) @ v.permute(0, 2, 1, 3)
    out = out.reshape(n, kvh, g, r, hd) / e.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(n * r, heads, hd)


def _sample(s):
    x = s["x"]
    v = x.shape[1]
    t, top_k, top_p, min_p, u = (s[k][:, None] for k in ("temperature", "top_k", "top_p", "min_p", "draw"))
    xs, idx = torch.sort(x, dim=1, descending=True, stable=True)
    warm = torch.where(t > 0, t, torch.ones_like(t))
    p = torch.exp((xs - xs[:, :1]).double() / warm)
    place = torch.arange(v, device=x.device)
    k1 = torch.where(top_k > 0, top_k.clamp(max=v), torch.full_like(top_k, v))
    run_sum = torch.cumsum(p * (place < k1), 1)
    s1 = run_sum[:, -1:]
    k2 = torch.where(top_p < 1, 1 + (run_sum < top_p * s1).sum(1, keepdim=True), k1)
    k3 = (p >= min_p).sum(1, keepdim=True)
    k = torch.minimum(torch.minimum(k1, k2), k3).clamp(1, v)
    kept = run_sum.gather(1, k - 1)
    at = torch.minimum((run_sum < u * kept).sum(1, keepdim=True), k - 1)
    chosen = idx.gather(1, at)
    # no filter: the ids' own order
    c0 = torch.cumsum(torch.exp((x - xs[:, :1]).double() / warm), 1)
    plain = ((c0 < u * c0[:, -1:]) | (c0 <= 0)).sum(1, keepdim=True).clamp(max=v - 1)
    free = (k1 == v) & (top_p >= 1) & (min_p <= 0)
    chosen = torch.where(free, plain, chosen)
    return torch.where(t > 0, chosen, idx[:, :1])[:, 0].int()


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)


def _exact_append(s):
    c = s["case"]
    hd, rope = c["hd"], c["rope"]

    def turned(x):
        x = x.double().clone()
        z = s["table"].double()[s["pos"].long()]
        for i in range(rope // 2):
            a, b = (i, i + rope // 2) if c["neox"] else (2 * i, 2 * i + 1)
            co, si = z[:, i, 0:1], z[:, i, 1:2]
            x[:, :, a], x[:, :, b] = x[:, :, a] * co - x[:, :, b] * si, x[:, :, a] * si + x[:, :, b] * co
        return x

    def held(x):
        for b in range(0, hd, BLOCK):
            part = x[:, :, b:b + BLOCK]
            top = part.abs().amax(-1, keepdim=True)
            sign = torch.where((part == top).any(-1, keepdim=True), 1.0, -1.0).double()
            d = (top * sign / -8).half().double()
            x[:, :, b:b + BLOCK] = torch.where(d == 0, torch.zeros_like(part), d * ((part / d + 0.5).floor().clamp(-8, 7)))
        return x

    return turned(s["q"]), held(turned(s["k"])), held(s["v"].double().clone())


def _exact_attention(s):
    c = s["case"]
    hd, kvh, g = c["hd"], c["kv_heads"], c["heads"] // c["kv_heads"]
    nb = hd // BLOCK
    w = min(4, nb)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    dim = torch.arange(hd, device=DEV)
    b = dim // BLOCK
    for i in range(c["seqs"]):
        at = s["pos"][i * c["rows"]:(i + 1) * c["rows"]].long()
        if int(at[-1]) < 0:
            continue
        n = int(at[-1]) + 1
        p = torch.arange(n, device=DEV)[:, None]
        for h in range(kvh):
            tiles = s["cache"][i, :, h]
            r = p % TILE

            def part(word, nibble, base, scale_base):
                byte = (b // 4 * 1024 + word * 4) + nibble // 2
                code = (tiles[p // TILE, base + byte].int() >> (4 * (nibble % 2))) & 15
                lo, up = (tiles[p // TILE, scale_base + 2 * (r * nb + b) + e].int() for e in (0, 1))
                return (code - 8).double() * (lo + 256 * up).to(torch.int16).view(torch.float16).double()

            lane = (r // 8) * 32
            k = part((lane + r % 8 * 4 + dim % 32 // 8) * w + b % 4, dim % 8, 0, 16 * hd)
            v = part((lane + dim % 32 // 4 * 4 + r % 8 // 2) * w + b % 4, dim % 4 + 4 * (r % 2), 8 * hd, 17 * hd)
            for lo in range(0, c["rows"], 256):
                rows = at[lo:lo + 256]
                q = s["q"][i * c["rows"] + lo:i * c["rows"] + lo + len(rows), h * g:(h + 1) * g].double()
                a = torch.einsum("thd,jd->thj", q, k) * s["scale"]
                j = p[:, 0]
                hide = j > rows[:, None]
                if c["window"]:
                    hide = hide | ((j <= rows[:, None] - c["window"]) & (j >= c["sinks"]))
                a = torch.softmax(a.masked_fill(hide[:, None], -math.inf), -1)
                out[i * c["rows"] + lo:i * c["rows"] + lo + len(rows), h * g:(h + 1) * g] = torch.einsum("thj,jd->thd", a, v)
    return out


def _exact_sample(s):
    import numpy as np
    ids = []
    for r in range(s["x"].shape[0]):
        x = s["x"][r].cpu().numpy().astype(np.float64)
        t, k, tp, mp, u = (s[n][r].item() for n in ("temperature", "top_k", "top_p", "min_p", "draw"))
        if t <= 0:
            ids.append(int(np.argmax(x)))
            continue
        p = np.exp((x - x.max()) / t)
        order = np.lexsort((np.arange(x.size), -x))
        if k <= 0 and tp >= 1 and mp <= 0:
            order = np.flatnonzero(p > 0)
        if k > 0:
            order = order[:k]
        keep = len(order)
        if tp < 1:
            keep = 1 + int(np.searchsorted(np.cumsum(p[order]), tp * p[order].sum()))
        if mp > 0:
            keep = min(keep, int((p[order] >= mp).sum()))
        order = order[:max(1, keep)]
        c = np.cumsum(p[order])
        ids.append(int(order[min(len(order) - 1, int(np.searchsorted(c, u * c[-1])))]))
    return torch.tensor(ids, dtype=torch.int32)
