"""Cases of the 4-bit paged key/value cache operators: append (RMSNorm, rotary
positions, quantisation), attend and read.

Each case is one call as a serving step makes it.  `run` computes it in plain
torch operations, or through q3t.KV4Cache where `own` is true.

The cache holds every (page of 16 tokens, kv head) in one block of 20 D bytes:

  K digits   8 D bytes   token c, dim 32 j + 8 t + 4 b0 + 2 h + b1 in byte
                         c D / 2 + 4 (G t + j) + 2 b1 + b0, nibble h
  V digits   8 D bytes   token 8 b0 + 2 t + b1, dim 64 M + 16 m + 8 h + g in byte
                         8 D + 512 M + 16 (4 g + t) + 4 m + 2 b1 + b0, nibble h
  scales     4 D bytes   token 8 p1 + 2 t + p0, group j: K scale, K zero, V scale,
                         V zero as bf16 at 16 D + 8 (4 (4 j + t) + 2 p1 + p0)

with G = D / 32 groups of 32 dims, and a digit n standing for n * scale + zero.
Of a group's values: zero is their minimum, rounded down to bf16; scale is
(maximum - zero) / 15 in bf16; a digit is round((x - zero) / scale) within
0..15.
"""
import math
import random

import torch

own = False

PAGE = 16
EPS = 1e-6


# ----------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------
def _case(op, name=None, *, D=128, kv_heads=8, group=2, seqs=1, q=(1, 1), past=(0, 0), chunks=0, chunk=(0, 0),
          lens=1, **more):
    c = {"op": op, "D": D, "kv_heads": kv_heads, "group": group, "seqs": seqs, "q_lo": q[0], "q_hi": q[1],
         "past_lo": past[0], "past_hi": past[1], "chunks": chunks, "chunk_lo": chunk[0], "chunk_hi": chunk[1],
         "lens": lens}
    if op == "append":
        c |= {"dtype": "bf16", "norm": False, "layout": "half", "rot": D, "theta": 1e6, "scaling": "none",
              "factor": 1.0, "low": 1.0, "high": 4.0, "original": 4096, "amplitude": 1.0}
    if op == "attend":
        c |= {"window": 0}
    c |= more
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the talker's decode frame at 64 requests: one token each, f32 rows from the projection, q/k RMSNorm
        _case("append", "append_frame64", seqs=64, past=(100, 1500), dtype="f32", norm=True),
        # prompts of odd lengths; 64-wide heads, half of each rotated, adjacent pairs, positions divided by 4
        _case("append", "append_prompts_d64", D=64, kv_heads=16, group=1, seqs=7, q=(33, 700), past=(0, 50),
              layout="interleaved", rot=32, theta=1e4, scaling="linear", factor=4.0),
        # two long prompts continued far out, frequencies blended for the long context
        _case("append", "append_far", seqs=2, q=(4001, 4096), past=(99_000, 101_000), norm=True, scaling="bands",
              factor=32.0, low=1.0, high=32.0, amplitude=1.34375),
        # one request's decode step (the batch-1 talker step at 1024 cached keys)
        _case("attend", "attend_one", past=(1023, 1023)),
        # the decode frame of 64 requests with the serving workload's ragged lengths
        _case("attend", "attend_frame64", seqs=64, past=(100, 1500)),
        # 64 requests whose caches are full
        _case("attend", "attend_full64", seqs=64, past=(4095, 4095)),
        # one very long cache, an odd length
        _case("attend", "attend_long", past=(131_070, 131_070)),
        # a frame that carries prompt chunks next to the decode tokens, 128 tokens in all
        _case("attend", "attend_mixed", seqs=61, past=(60, 900), chunks=3, chunk=(15, 30)),
        # a whole prompt at the cache's capacity
        _case("attend", "attend_prompt", q=(4096, 4096)),
        # sixteen requests with 64-wide heads, four query heads to a kv head, a sliding window
        _case("attend", "attend_window_d64", D=64, kv_heads=4, group=4, seqs=16, past=(700, 5000), window=1000),
        # saving one request's cache
        _case("read", "read_one", past=(369, 369)),
        # copying out the caches of 64 requests
        _case("read", "read_64", seqs=64, past=(100, 1500)),
    ]


def _span(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "read"])
    lens = rng.randrange(1 << 30)
    while True:
        D = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
        group = rng.choice([1, 2, 2, 4, 5, 8])
        seqs, chunks, chunk = _span(rng, 1, 64), 0, (0, 0)
        more = {}
        if op == "append" or (op == "attend" and rng.random() < 0.4):  # prompts, or one token each
            q_hi = 1 if rng.random() < 0.4 else _span(rng, 2, 4096)
        else:
            q_hi = 1
        q = (rng.randint(max(1, q_hi // 3), q_hi), q_hi)
        past_hi = _span(rng, 1, 131_000) if rng.random() < 0.7 else 0
        past = (past_hi // 4, past_hi)
        if op == "append":
            rot = rng.choice([D, D, D // 2, 16, 0])
            scaling = rng.choice(["none", "linear", "bands"])
            more = {"dtype": rng.choice(["bf16", "f32"]), "norm": rng.random() < 0.5,
                    "layout": rng.choice(["half", "interleaved"]), "rot": rot, "theta": rng.choice([1e4, 1e6]),
                    "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0])}
        elif op == "attend":
            more = {"window": rng.choice([0, 0, 0, _span(rng, 1, 4096)])}
            if q_hi == 1 and rng.random() < 0.3:
                chunks, chunk = rng.randint(1, 3), (5, 40)
        c = _case(op, D=D, kv_heads=kv_heads, group=group, seqs=seqs, q=q, past=past, chunks=chunks, chunk=chunk,
                  lens=lens, **more)
        nq, kv = _lengths(c)
        heads, B = kv_heads * group, len(nq)
        scores = B * heads * max(nq) * max(kv)
        cells = B * max(kv) * kv_heads * D  # keys of the padded caches
        if op == "append":
            fine = sum(nq) * max(heads, kv_heads) * D <= 8192 * 16 * 128 and sum(kv) * kv_heads * D <= 1 << 28
        elif op == "attend":
            fine = scores <= 1 << 28 and cells <= 1 << 28
        else:
            fine = sum(kv) * kv_heads * D <= 1 << 26 and cells <= 1 << 28
        if fine:
            return c


def _lengths(case):
    """(query tokens, keys) of each sequence; the same for every seed."""
    r = random.Random(case["lens"])
    nq, kv = [], []
    for i in range(case["seqs"] + case["chunks"]):
        n = r.randint(case["q_lo"], case["q_hi"]) if i < case["seqs"] else r.randint(case["chunk_lo"], case["chunk_hi"])
        nq.append(n)
        kv.append(n + r.randint(case["past_lo"], case["past_hi"]))
    if case["op"] == "read":  # a read takes whole caches
        nq = list(kv)
    return nq, kv


def _pairs(case):
    """(query, key) pairs that the masks let through, and keys that any query sees, summed over sequences."""
    pairs = keys = 0
    w = case.get("window", 0)
    for n, k in zip(*_lengths(case)):
        if not w:
            pairs += n * k - n * (n - 1) // 2
            keys += k
        else:
            pairs += sum(min(p + 1, w) for p in range(k - n, k))
            keys += min(k, n + w - 1)
    return pairs, keys


def work(case):
    nq, kv = _lengths(case)
    D, kvh, heads = case["D"], case["kv_heads"], case["kv_heads"] * case["group"]
    cached = kvh * D * 5 / 4  # bytes of a token's keys and values: 4 bits a digit, 4 bf16 to 32 + 32 of them
    T = sum(nq)
    if case["op"] == "append":
        size = 4 if case["dtype"] == "f32" else 2
        rows = T * (heads + 2 * kvh) * D
        # rows in, rotated queries out, digits and scales out, and the stored values back
        return {"bytes": rows * size + T * heads * D * 2 + T * cached + T * 2 * kvh * D * 2, "flops": rows * 10}
    if case["op"] == "attend":
        pairs, keys = _pairs(case)
        return {"bytes": keys * cached + 2 * T * heads * D * 2, "flops": 4 * pairs * heads * D}
    return {"bytes": sum(kv) * cached + sum(kv) * 2 * kvh * D * 2, "flops": sum(kv) * kvh * D * 4}


# ----------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    nq, kv = _lengths(case)
    D, kvh, heads, B, T = case["D"], case["kv_heads"], case["kv_heads"] * case["group"], len(nq), sum(nq)
    pages = [-(-k // PAGE) for k in kv]
    stride = max(pages) + 1
    num_pages = sum(pages) + 3
    order = torch.randperm(num_pages, generator=gen, device=dev).to(torch.int32).cpu()  # a pool's pages are scattered
    table = torch.zeros(B, stride, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": dict(case), "max_q": max(nq), "max_kv": max(kv), "tokens": T, "table": table.to(dev),
         "q_start": torch.tensor([0] + nq).cumsum(0).to(torch.int32).to(dev),
         "kv_len": torch.tensor(kv, dtype=torch.int32, device=dev)}
    # a pool that other requests have used before: stale bytes wherever this case has no keys
    s["pool"] = torch.randint(0, 256, (num_pages, kvh, 20 * D), generator=gen, device=dev, dtype=torch.uint8)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    offset = 2.0 * normal(kvh, 1, D) * (torch.rand(kvh, 1, D, generator=gen, device=dev) < 0.1)  # channels with a bias
    if case["op"] == "append":
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        rows = normal(T, (heads + 2 * kvh) * D) * 1.5  # one projection's rows: queries, keys, values
        rows[:, heads * D:(heads + kvh) * D] += offset.reshape(1, -1)
        s["rows"] = rows.to(dt)
        s["q_gamma"] = 1.0 + 0.3 * normal(D) if case["norm"] else None
        s["k_gamma"] = 1.0 + 0.3 * normal(D) if case["norm"] else None
        s["q_out"] = torch.empty(T, heads, D, dtype=torch.bfloat16, device=dev)
    else:
        for p0 in range(0, num_pages, 4096):
            n = min(4096, num_pages - p0)
            s["pool"][p0:p0 + n] = _pack_pages(normal(n, kvh, PAGE, D) + offset, normal(n, kvh, PAGE, D))
        # slots behind a sequence's last key hold whatever was there: here digits of 15 and NaN scales
        tails = [(int(table[b, k // PAGE]), c) for b, k in enumerate(kv) if k % PAGE for c in range(k % PAGE, PAGE)]
        if tails:
            at = torch.tensor(tails, device=dev)
            off = _row_offsets(at[:, 1], D)
            idx = (at[:, :1, None] * kvh + torch.arange(kvh, device=dev)[None, :, None]) * (20 * D) + off[:, None, :]
            s["pool"].view(-1)[idx.reshape(-1)] = 255
    if case["op"] == "attend":
        s["q"] = (1.3 * normal(T, heads, D)).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
    if case["op"] != "attend":
        s["k_out"] = torch.empty(T, kvh, D, dtype=torch.bfloat16, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


# ----------------------------------------------------------------------------
# the plain forms
# ----------------------------------------------------------------------------
def _quantise(x):
    """(digits, scale, zero) of x [..., D] in groups of 32."""
    g = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    hi, lo = g.amax(-1), g.amin(-1)
    bits = lo.view(torch.int32)
    zero = (torch.where(lo < 0, bits + 0xffff, bits) & ~0xffff).view(torch.float32)  # towards minus infinity
    scale = ((hi * 0.5 - zero * 0.5) * (2.0 / 15.0)).bfloat16().float()
    some = torch.where(scale > 0, scale, torch.ones_like(scale))
    digit = ((g - zero[..., None]) / some[..., None]).round().clamp(0, 15)
    digit = torch.where((scale > 0)[..., None], digit, torch.zeros_like(digit))
    return digit.to(torch.uint8).reshape(x.shape), scale.bfloat16(), zero.bfloat16()


def _pack_pages(k, v):
    """Blocks [pages, kv heads, 20 D] of whole pages of keys and values [pages, kv heads, 16, D]."""
    n, h, _, D = k.shape
    G = D // 32
    kd, ks, kz = _quantise(k)
    vd, vs, vz = _quantise(v)
    kd = kd.view(n, h, 16, G, 4, 2, 2, 2).permute(0, 1, 2, 4, 3, 7, 5, 6)  # token, t, j, b1, b0, nibble
    kb = kd[..., 0] | (kd[..., 1] << 4)
    vd = vd.view(n, h, 2, 4, 2, D // 64, 4, 2, 8).permute(0, 1, 5, 8, 3, 6, 4, 2, 7)  # M, g, t, m, b1, b0, nibble
    vb = vd[..., 0] | (vd[..., 1] << 4)
    sc = torch.stack([ks, kz, vs, vz], -1).view(n, h, 2, 4, 2, G, 4).permute(0, 1, 5, 3, 2, 4, 6)  # j, t, p1, p0
    return torch.cat([kb.reshape(n, h, -1), vb.reshape(n, h, -1),
                      sc.contiguous().view(torch.uint8).reshape(n, h, -1)], -1)


def _row_offsets(c, D):
    """Byte offsets within a block of what token c [T] owns: its D/2 key bytes, D/2 value bytes, D/4 scale bytes."""
    dev, G = c.device, D // 32
    ar = lambda n: torch.arange(n, device=dev)  # noqa: E731
    c = c.long()[:, None]
    k = c * (D // 2) + ar(D // 2)
    t, b1, b0 = (c >> 1) & 3, c & 1, c >> 3
    M, m, g = ar(D // 64)[:, None, None], ar(4)[None, :, None], ar(8)[None, None, :]
    v = 8 * D + (512 * M + 64 * g + 4 * m).reshape(1, -1) + 16 * t + 2 * b1 + b0
    j, e = ar(G)[:, None], ar(8)[None, :]
    s = 16 * D + (128 * j + e).reshape(1, -1) + 32 * t + 8 * (2 * b0 + b1)
    return torch.cat([k, v, s], -1)


def _pack_rows(k, v):
    """The bytes [T, kv heads, 5 D / 4] at _row_offsets of keys and values [T, kv heads, D]."""
    T, h, D = k.shape
    G = D // 32
    kd, ks, kz = _quantise(k)
    vd, vs, vz = _quantise(v)
    kd = kd.view(T, h, G, 4, 2, 2, 2).permute(0, 1, 3, 2, 6, 4, 5)
    kb = (kd[..., 0] | (kd[..., 1] << 4)).reshape(T, h, -1)
    vd = vd.view(T, h, D // 64, 4, 2, 8)
    vb = (vd[:, :, :, :, 0] | (vd[:, :, :, :, 1] << 4)).reshape(T, h, -1)
    sc = torch.stack([ks, kz, vs, vz], -1).contiguous().view(torch.uint8).reshape(T, h, -1)
    return torch.cat([kb, vb, sc], -1)


def _unpack(blocks):
    """Keys and values [..., 16, D] in f32 of blocks [..., 20 D]."""
    lead, D = blocks.shape[:-1], blocks.shape[-1] // 20
    G, n = D // 32, len(blocks.shape) - 1
    at = list(range(n))
    both = torch.stack([blocks[..., :16 * D] & 15, blocks[..., :16 * D] >> 4], -1)
    kd = both[..., :8 * D, :].reshape(*lead, 16, 4, G, 2, 2, 2)  # token, t, j, b1, b0, nibble
    kd = kd.permute(*at, n, n + 2, n + 1, n + 4, n + 5, n + 3).reshape(*lead, 16, G, 32)
    vd = both[..., 8 * D:, :].reshape(*lead, D // 64, 8, 4, 4, 2, 2, 2)  # M, g, t, m, b1, b0, nibble
    vd = vd.permute(*at, n + 5, n + 2, n + 4, n, n + 3, n + 6, n + 1).reshape(*lead, 16, G, 32)
    sc = blocks[..., 16 * D:].contiguous().view(torch.bfloat16).float().reshape(*lead, G, 4, 2, 2, 4)
    sc = sc.permute(*at, n + 2, n + 1, n + 3, n, n + 4).reshape(*lead, 16, G, 4)
    k = kd.float() * sc[..., 0:1] + sc[..., 1:2]
    v = vd.float() * sc[..., 2:3] + sc[..., 3:4]
    return k.reshape(*lead, 16, D), v.reshape(*lead, 16, D)


def _places(s):
    """(sequence, index in it, position, page, slot) of every token row."""
    tok = torch.arange(s["tokens"], device=s["pool"].device)
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), tok.to(torch.int32), right=True)
    i = tok - s["q_start"][seq]
    pos = s["kv_len"][seq] - (s["q_start"][seq + 1] - s["q_start"][seq]) + i
    page = s["table"][seq, pos // PAGE].long()
    return seq, i, pos, page, pos % PAGE


def _frequencies(case):
    rot = case["rot"]
    f = [case["theta"] ** (-2.0 * i / rot) for i in range(rot // 2)]
    if case["scaling"] == "linear":
        f = [x / case["factor"] for x in f]
    if case["scaling"] == "bands":  # turns over the original context: few are slowed down, many are kept
        ramp = [min(1.0, max(0.0, (case["original"] * x / (2 * math.pi) - case["low"]) / (case["high"] - case["low"])))
                for x in f]
        f = [(1 - r) * x / case["factor"] + r * x for x, r in zip(f, ramp)]
    return f


def _normed(x, gamma):
    """RMSNorm of each head; its sum of squares in 64 bits."""
    if gamma is None:
        return x
    r = (1.0 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    return x * r * gamma


def _rotated(x, pos, case):
    """Rotary positions on x [T, heads, D] in f32; the angles in 64 bits."""
    rot = case["rot"]
    if not rot:
        return x
    a = pos.double()[:, None] * torch.tensor(_frequencies(case), dtype=torch.float64, device=x.device)
    cos, sin = ((f(a) * case["amplitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    if case["layout"] == "half":
        u, w = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([u * cos - w * sin, w * cos + u * sin, x[..., rot:]], -1)
    u, w = x[..., 0:rot:2], x[..., 1:rot:2]
    turned = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _split_rows(s):
    c = s["case"]
    D, kvh, heads = c["D"], c["kv_heads"], c["kv_heads"] * c["group"]
    rows = s["rows"].view(s["tokens"], heads + 2 * kvh, D)
    return rows[:, :heads], rows[:, heads:heads + kvh], rows[:, heads + kvh:]


def _plain_read(s):
    _, _, _, page, slot = _places(s)
    distinct, back = torch.unique(page, return_inverse=True)
    k, v = _unpack(s["pool"][distinct])
    return {"k": k[back, :, slot].bfloat16(), "v": v[back, :, slot].bfloat16()}


def _plain_append(s):
    c = s["case"]
    D, kvh = c["D"], c["kv_heads"]
    q, k, v = (x.float() for x in _split_rows(s))
    _, _, pos, page, slot = _places(s)
    q = _rotated(_normed(q, s["q_gamma"]), pos, c)
    k = _rotated(_normed(k, s["k_gamma"]), pos, c)
    base = (page[:, None, None] * kvh + torch.arange(kvh, device=q.device)[None, :, None]) * (20 * D)
    s["pool"].view(-1)[base + _row_offsets(slot, D)[:, None, :]] = _pack_rows(k, v)
    return {"q": q.bfloat16(), **_plain_read(s)}


def _plain_attend(s):
    c = s["case"]
    D, kvh, g = c["D"], c["kv_heads"], c["group"]
    dev = s["pool"].device
    n_pages = -(-s["max_kv"] // PAGE)
    keys = torch.arange(n_pages * PAGE, device=dev)
    held = keys[None, :] < s["kv_len"][:, None]
    page = s["table"][:, :n_pages].long()
    k, v = _unpack(s["pool"][page])  # [B, pages, kv heads, 16, D]
    hide = ~held.view(page.shape[0], n_pages, 1, PAGE, 1)
    k = k.masked_fill_(hide, 0.0).transpose(1, 2).reshape(page.shape[0], kvh, 1, -1, D)
    v = v.masked_fill_(hide, 0.0).transpose(1, 2).reshape(page.shape[0], kvh, 1, -1, D)
    i = torch.arange(s["max_q"], device=dev)
    n = s["q_start"][1:] - s["q_start"][:-1]
    tok = (s["q_start"][:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][tok].float().view(page.shape[0], s["max_q"], kvh, g, D).permute(0, 2, 3, 1, 4)
    pos = (s["kv_len"] - n)[:, None] + i
    seen = held[:, None, :] & (keys <= pos[..., None])
    if c["window"]:
        seen &= keys > pos[..., None] - c["window"]
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    score = score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    seq, at, _, _, _ = _places(s)
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(page.shape[0], s["max_q"], kvh * g, D)[seq, at].bfloat16()}


# ----------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------
def _program(s):
    """What a program keeps over its calls: the cache over its pool, the step's batch, the rotation."""
    if "program" not in s:
        import os
        import sys
        path = os.path.join(os.getcwd(), "tts-rs_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import q3t
        c = s["case"]
        cache = q3t.KV4Cache(s["pool"], s["table"], c["kv_heads"], c["D"])
        batch = q3t.KV4Batch(s["q_start"], s["kv_len"], s["tokens"], max_q=s["max_q"], max_kv=s["max_kv"])
        rope = None
        if c["op"] == "append" and c["rot"]:
            rope = q3t.Rope(c["D"], rotary_dim=c["rot"], layout=c["layout"], theta=c["theta"], scaling=c["scaling"],
                            factor=c["factor"], low=c["low"], high=c["high"], original=c["original"],
                            amplitude=c["amplitude"])
        s["program"] = cache, batch, rope
    return s["program"]


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        cache, batch, rope = _program(s)
        if op == "attend":
            return {"out": cache.attend(batch, s["q"], window=s["case"]["window"], out=s["out"])}
        if op == "append":
            q, k, v = _split_rows(s)
            cache.append(batch, k, v, q=q, rope=rope, q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=EPS,
                         q_out=s["q_out"])
            k, v = cache.read(batch, k=s["k_out"], v=s["v_out"])
            return {"q": s["q_out"], "k": k, "v": v}
        k, v = cache.read(batch, k=s["k_out"], v=s["v_out"])
        return {"k": k, "v": v}
    if op == "attend":
        return _plain_attend(s)
    if op == "append":
        return _plain_append(s)
    return _plain_read(s)


# ----------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------
def _exact_tables(D, dev):
    """Byte and shift of every (token, dim) digit and the place of every (token, group) scale, spelled out."""
    kb, ks, vb, vs, sc = [], [], [], [], []
    for c in range(16):
        for d in range(D):
            j, t, e = d // 32, d % 32 // 8, d % 8
            kb.append(c * D // 2 + 4 * (D // 32 * t + j) + 2 * (e % 2) + e // 4)
            ks.append(4 * (e // 2 % 2))
            M, m, h, g = d // 64, d % 64 // 16, d % 16 // 8, d % 8
            vb.append(8 * D + 512 * M + 16 * (4 * g + c % 8 // 2) + 4 * m + 2 * (c % 2) + c // 8)
            vs.append(4 * h)
            sc.append((16 * D + 8 * (4 * (4 * j + c % 8 // 2) + 2 * (c // 8) + c % 2)) // 2)
    return [torch.tensor(x, device=dev) for x in (kb, ks, vb, vs, sc)]


def _exact_keys(pool, pages, n, D, tables):
    """The first n keys and values [n, kv heads, D] of a list of pages, in 64 bits."""
    kb, ks, vb, vs, sc = tables
    raw = pool[pages].long()
    half = pool[pages].view(torch.bfloat16).double()
    k = (raw[..., kb] >> ks & 15) * half[..., sc] + half[..., sc + 1]
    v = (raw[..., vb] >> vs & 15) * half[..., sc + 2] + half[..., sc + 3]
    shape = (len(pages), pool.shape[1], 16, D)
    k, v = (x.reshape(shape).transpose(1, 2).reshape(-1, pool.shape[1], D)[:n] for x in (k, v))
    return k, v


def _exact_stored(x):
    """What the cache keeps of x [..., D]: bf16 scale and zero of each 32, whole digits, no other rounding."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    _, e = torch.frexp(lo)
    ulp = torch.ldexp(torch.ones_like(lo), e - 8)
    zero = torch.floor(lo / ulp) * ulp
    want = (hi - zero) / 15
    _, e = torch.frexp(want)
    ulp = torch.ldexp(torch.ones_like(want), e - 8)
    scale = torch.round(want / ulp) * ulp
    n = torch.where(scale > 0, torch.round((g - zero) / torch.where(scale > 0, scale, 1.0)).clamp(0, 15), 0.0)
    return (n * scale + zero).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    D, kvh, heads, group = case["D"], case["kv_heads"], case["kv_heads"] * case["group"], case["group"]
    dev = s["pool"].device
    nq, kv = _lengths(case)
    table = s["table"].cpu().long()
    if case["op"] == "append":
        rows = s["rows"].double().view(-1, heads + 2 * kvh, D)
        pos = torch.tensor([k - n + i for n, k in zip(nq, kv) for i in range(n)], dtype=torch.float64, device=dev)
        x = rows[:, :heads + kvh]
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
            x = torch.cat([x[:, :heads] * s["q_gamma"].double(), x[:, heads:] * s["k_gamma"].double()], 1)
        x = x.clone()
        for i in range(case["rot"] // 2):
            f = case["theta"] ** (-2 * i / case["rot"])
            if case["scaling"] == "linear":
                f /= case["factor"]
            if case["scaling"] == "bands":
                turns = case["original"] * f / (2 * math.pi)
                keep = min(1.0, max(0.0, (turns - case["low"]) / (case["high"] - case["low"])))
                f = keep * f + (1 - keep) * f / case["factor"]
            a, b = (i, i + case["rot"] // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(pos, case["amplitude"]), pos * f)[:, None]
            x[..., a], x[..., b] = z.real, z.imag
        return {"q": x[:, :heads], "k": _exact_stored(x[:, heads:]), "v": _exact_stored(rows[:, heads + kvh:])}
    tables = _exact_tables(D, dev)
    if case["op"] == "read":
        both = [_exact_keys(s["pool"], table[b, :-(-k // 16)].to(dev), k, D, tables) for b, k in enumerate(kv)]
        return {"k": torch.cat([x[0] for x in both]), "v": torch.cat([x[1] for x in both])}
    if case["op"] == "attend" and heads * sum(n * k for n, k in zip(nq, kv)) * D > 1 << 41:
        return None
    out, at = [], 0
    for b, (n, m) in enumerate(zip(nq, kv)):
        k, v = _exact_keys(s["pool"], table[b, :-(-m // 16)].to(dev), m, D, tables)
        q = s["q"][at:at + n].double()
        at += n
        own_pos, key = torch.arange(m - n, m, device=dev)[:, None], torch.arange(m, device=dev)[None, :]
        hidden = key > own_pos
        if case["window"]:
            hidden = hidden | (key <= own_pos - case["window"])
        per_head = []
        for h in range(heads):
            w = (q[:, h] @ k[:, h // group].T / math.sqrt(D)).masked_fill(hidden, float("-inf"))
            per_head.append(torch.softmax(w, -1) @ v[:, h // group])
        out.append(torch.stack(per_head, 1))
    return {"out": torch.cat(out)}
