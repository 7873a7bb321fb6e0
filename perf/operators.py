"""What is measured of the paged key/value cache: appending to it, and attention of one new token over it.

Three kinds of pass (``case["op"]``):

``append``  keys and values of new tokens go into the pages of each sequence, with the rotary embedding
            applied to the keys on the way (prompts of different lengths in one padded batch, or one new
            token per sequence); with ``query`` the rotated query and key are handed back as well, which is
            what a prompt's attention needs next.
``attend``  attention of one query token per sequence over the sequence's pages; every sequence has its own
            length, several query heads may share a key/value head, and a head may see only its first ``sink``
            and last ``local`` tokens.
``step``    both at once, the decode step: rotate, append the new token, attend over the sequence with it.

``own = False`` computes the plain form with elementary torch operations in fp32; ``own = True`` calls
``moa_b200.paged_append`` and ``moa_b200.paged_decode``.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
LOCALS = (256, 512, 1024, 2048, 4096)      # windows of the per-head spans; the sink is 64 tokens
SINK = 64
THETA = 10000.0
MOST_BYTES = 1.1e9                         # a drawn case moves no more than the largest listed one


def listed():
    return [
        # one new token of each of 16 sequences, 32 heads: the append of one layer of a small decode batch
        dict(name="append 16x1 fp16", op="append", dtype="fp16", B=16, H=32, KV=32, N=1, D=128, page=64, layout="heads",
             short=200, long=4000, spans=False, table="token", query=False),
        # a batch of chat prompts of different lengths, grouped heads, small pages
        dict(name="append 8x1500 ragged bf16", op="append", dtype="bf16", B=8, H=32, KV=8, N=1500, D=128, page=16,
             layout="tokens", short=0, long=700, spans=False, table="position", query=False),
        # one long prompt of a 32-head model: rotation of query and key, append, rotated tensors for the prefill
        dict(name="append 1x16384 query fp16", op="append", dtype="fp16", B=1, H=32, KV=32, N=16384, D=128, page=64,
             layout="heads", short=0, long=0, spans=False, table="token", query=True),
        # odd sizes: 5 heads of 64, prompt pieces that start in the middle of a page
        dict(name="append 3x333 odd bf16", op="append", dtype="bf16", B=3, H=5, KV=5, N=333, D=64, page=32,
             layout="heads", short=5, long=91, spans=False, table="position", query=True),
        # a single short conversation, eight heads: latency
        dict(name="attend 1x129 fp16", op="attend", dtype="fp16", B=1, H=8, KV=8, D=128, page=64, layout="heads",
             short=129, long=129, spans=False),
        # 16 sequences at 16k with per-head spans (64 + 256..4096): the decode batch of the ring caches, paged
        dict(name="attend 16x16384 spans fp16", op="attend", dtype="fp16", B=16, H=32, KV=32, D=128, page=64,
             layout="heads", short=16384, long=16384, spans=True),
        # a server's batch, lengths from a few tokens to 8k, four query heads to a key head, small pages
        dict(name="attend 64x8192 ragged bf16", op="attend", dtype="bf16", B=64, H=32, KV=8, D=128, page=16,
             layout="tokens", short=3, long=8192, spans=False),
        # one long document, eight key heads: work split over the length
        dict(name="attend 1x131071 bf16", op="attend", dtype="bf16", B=1, H=64, KV=8, D=128, page=64, layout="heads",
             short=131071, long=131071, spans=False),
        # a single key head under 16 query heads, narrow heads, odd lengths
        dict(name="attend 7x20011 one head fp16", op="attend", dtype="fp16", B=7, H=16, KV=1, D=64, page=128,
             layout="heads", short=999, long=20011, spans=False),
        # the decode step of one short conversation: latency
        dict(name="step 1x1000 fp16", op="step", dtype="fp16", B=1, H=32, KV=32, D=128, page=64, layout="heads",
             short=1000, long=1000, spans=False, table="token"),
        # the decode step of a server's batch of ragged requests
        dict(name="step 128x2048 ragged bf16", op="step", dtype="bf16", B=128, H=32, KV=8, D=128, page=16,
             layout="tokens", short=1, long=2048, spans=False, table="position"),
        # the decode step of 32 sequences at 16k under per-head spans, one layer of a 32-head model
        dict(name="step 32x16384 spans fp16", op="step", dtype="fp16", B=32, H=32, KV=32, D=128, page=64,
             layout="heads", short=15000, long=16384, spans=True, table="token"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "attend", "step"])
        KV = rng.choice([1, 2, 4, 5, 8, 16, 32])
        G = rng.choice([g for g in (1, 2, 3, 4, 6, 8, 12, 16) if KV * g <= 64])
        c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), B=_spread(rng, 1, 128), H=KV * G, KV=KV,
                 D=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]), layout=rng.choice(["heads", "tokens"]))
        if op == "append":
            c["N"] = rng.choice([1, _spread(rng, 2, 16384)])
            c["short"], c["long"] = 0, rng.randint(0, 4000)
            c["query"], c["spans"] = rng.random() < 0.3, False
        else:
            c["long"] = _spread(rng, 16, 131072)
            c["short"] = rng.choice([1, c["long"], rng.randint(1, c["long"])])
            c["spans"] = rng.random() < 0.3
        if op != "attend":
            c["table"] = rng.choice(["token", "position"])
        if work(c)["bytes"] <= MOST_BYTES and _pool_bytes(c) <= 10e9:
            return c


# ---------------------------------------------------------------------------------------- sizes of a case

def _lengths(c):
    """Tokens in each sequence's pages before the pass (fixed by the case, not by the seed)."""
    rng = random.Random("lengths %d %d %d" % (c["B"], c["short"], c["long"]))
    got = [rng.randint(c["short"], c["long"]) for _ in range(c["B"])]
    got[-1] = c["long"]
    return got


def _counts(c):
    """New tokens of each sequence (append): between a quarter of N and N."""
    rng = random.Random("counts %d %d" % (c["B"], c["N"]))
    got = [rng.randint(max(1, c["N"] // 4), c["N"]) for _ in range(c["B"])]
    got[0] = c["N"]
    return got


def _locals(c):
    rng = random.Random("spans %d" % c["KV"])
    return [rng.choice(LOCALS) for _ in range(c["KV"])]


def _new(c):
    return {"append": c.get("N", 0), "attend": 0, "step": 1}[c["op"]]


def _pages_each(c):
    return -(-(c["long"] + max(_new(c), 1)) // c["page"])


def _pages_needed(c):
    most = [n + m for n, m in zip(_lengths(c), _counts(c) if c["op"] == "append" else [_new(c)] * c["B"])]
    return [-(-n // c["page"]) for n in most]


def _pool_bytes(c):
    """The larger of the pools and the padded view of them that the plain form makes, in 16 bits."""
    row = c["KV"] * c["page"] * c["D"] * 2 * 2
    view = 0 if c["op"] == "append" else c["B"] * _pages_each(c)
    return row * max(sum(_pages_needed(c)), view)


def _rows(c):
    """Key rows that the attention of a pass has to read, over all sequences and key heads."""
    total = 0
    for n in _lengths(c):
        n += _new(c)
        if c["spans"]:
            total += sum(min(n, SINK + w) for w in _locals(c))
        else:
            total += n * c["KV"]
    return total


def work(c):
    B, H, KV, D = c["B"], c["H"], c["KV"], c["D"]
    cell = 2 if c.get("table") == "token" else 4
    if c["op"] == "append":
        tokens = sum(_counts(c))
        data = tokens * KV * D * 2 * 4                                   # k, v read and written
        if c["query"]:
            data += tokens * H * D * 2 * 2 + tokens * KV * D * 2         # q read, q and k handed back
        return {"bytes": data + tokens * D * cell * 2, "flops": 3 * tokens * D * (KV + (H if c["query"] else 0))}
    rows = _rows(c)
    data = rows * D * 2 * 2 + B * H * D * 2 * 2 + sum(_pages_needed(c)) * 4
    flops = 4 * rows * D * (H // KV)
    if c["op"] == "step":
        data += B * KV * D * 2 * 4 + B * D * cell * 2
        flops += 3 * B * D * (H + KV)
    return {"bytes": data, "flops": flops}


# ---------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    c = case
    dtype = DTYPES[c["dtype"]]
    B, H, KV, D, page = c["B"], c["H"], c["KV"], c["D"], c["page"]
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    lengths, need = _lengths(c), _pages_needed(c)
    # pages are handed out in a shuffled order, as they are after some hours of serving; rows of the table end in -1
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((B, _pages_each(c)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": c, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "page_table": table.cuda(),
         "scale": D ** -0.5, "sink": None, "local": None}
    if c["layout"] == "heads":      # (pages, heads, slots, D) in memory
        s["key_pages"], s["value_pages"] = normal(sum(need), KV, page, D), normal(sum(need), KV, page, D)
    else:                           # (pages, slots, heads, D) in memory
        s["key_pages"] = normal(sum(need), page, KV, D).transpose(1, 2)
        s["value_pages"] = normal(sum(need), page, KV, D).transpose(1, 2)
    N = c["N"] if c["op"] == "append" else 1
    # query, key and value as they come out of one projection: (B, N, heads, D) slices of its output, seen heads first
    qkv = normal(B, N, H + 2 * KV, D)
    s["query"] = (qkv[:, :, :H] * 1.5).transpose(1, 2) if c["op"] == "attend" else qkv[:, :, :H].transpose(1, 2)
    s["key"], s["value"] = qkv[:, :, H:H + KV].transpose(1, 2), qkv[:, :, H + KV:].transpose(1, 2)
    if c["op"] == "append":
        s["counts"] = torch.tensor(_counts(c), dtype=torch.int32, device="cuda")
    if c["spans"]:
        s["sink"] = torch.full((KV,), SINK, dtype=torch.int64, device="cuda")
        s["local"] = torch.tensor(_locals(c), dtype=torch.int64, device="cuda")
    if c["op"] != "attend":
        inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        if c["table"] == "position":        # one fp32 row for every position
            pos = torch.arange(_pages_each(c) * page, device="cuda").double()
        else:                               # one row for every new token, in the tensors' type
            pos = s["lengths"].double()[:, None] + torch.arange(N, device="cuda")
        angle = pos[..., None] * inv
        angle = torch.cat([angle, angle], dim=-1)
        kind = torch.float32 if c["table"] == "position" else dtype
        s["cos"], s["sin"] = angle.cos().to(kind), angle.sin().to(kind)
    return s


# ---------------------------------------------------------------------------------------- the pass

def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    import moa_b200

    op = s["case"]["op"]
    pages = (s["key_pages"], s["value_pages"], s["page_table"], s["lengths"])
    if op == "append":
        got = moa_b200.paged_append(s["key"], s["value"], *pages, counts=s["counts"], rope=(s["cos"], s["sin"]),
                                    query=s["query"] if s["case"]["query"] else None)
        out = {"key_pages": s["key_pages"], "value_pages": s["value_pages"]}
        if got is not None:
            out["query"], out["key"] = got
        return out
    if op == "attend":
        return {"out": moa_b200.paged_decode(s["query"], *pages, s["scale"], sink_size=s["sink"], local_size=s["local"])}
    out = moa_b200.paged_decode(s["query"], *pages, s["scale"], key=s["key"], value=s["value"],
                                rope=(s["cos"], s["sin"]), sink_size=s["sink"], local_size=s["local"])
    return {"out": out, "key_pages": s["key_pages"], "value_pages": s["value_pages"]}


def _rotate(x, cos, sin):
    """(B, heads, N, D) in fp32 rotated by (B, 1, N, D) tables: the halves of a head are the two coordinates."""
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _attention(q, key_pages, value_pages, table, n, scale, sink, local):
    """q (B, H, 1, D) in fp32 over the first n[b] tokens of each sequence -> (B, 1, H, D) in fp32."""
    B, H, _, D = q.shape
    KV, page = key_pages.shape[1], key_pages.shape[2]
    table = table.clamp(min=0).long()
    S = table.shape[1] * page
    k = key_pages[table].permute(0, 2, 1, 3, 4).reshape(B, KV, S, D).float()
    scores = torch.matmul(q.reshape(B, KV, H // KV, D), k.transpose(2, 3)) * scale
    del k
    v = value_pages[table].permute(0, 2, 1, 3, 4).reshape(B, KV, S, D).float()
    pos = torch.arange(S, device=q.device)
    seen = (pos < n[:, None])[:, None, None, :]
    if sink is not None:
        near = pos >= n[:, None, None] - local[None, :, None]
        seen = seen & (near | (pos < sink[None, :, None]))[:, :, None, :]
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(B, 1, H, D)


def _plain(s):
    c = s["case"]
    kp, vp, table, lengths = s["key_pages"], s["value_pages"], s["page_table"], s["lengths"].long()
    if c["op"] == "attend":
        out = _attention(s["query"].float(), kp, vp, table, lengths, s["scale"], s["sink"], s["local"])
        return {"out": out.to(kp.dtype)}
    key, value, query = s["key"], s["value"], s["query"]
    N, page = key.shape[2], kp.shape[2]
    at = torch.arange(N, device=key.device)
    pos = lengths[:, None] + at
    if c["table"] == "position":
        last = s["cos"].shape[0] - 1
        cos, sin = s["cos"][pos.clamp(max=last)][:, None], s["sin"][pos.clamp(max=last)][:, None]
    else:
        cos, sin = s["cos"].float()[:, None], s["sin"].float()[:, None]
    rotated = _rotate(key.float(), cos, sin)
    rows = rotated.to(kp.dtype)
    if c["op"] == "append":
        # a row behind a sequence's count repeats its last counted one, so that every write is of the row it should be
        i = torch.minimum(at, s["counts"].long()[:, None] - 1)
    else:
        i = torch.zeros_like(pos)
    b = torch.arange(key.shape[0], device=key.device)[:, None]
    pos = lengths[:, None] + i
    pages, slots = table.long().gather(1, pos // page), pos % page
    kp[pages, :, slots] = rows.transpose(1, 2)[b, i]
    vp[pages, :, slots] = value.transpose(1, 2)[b, i]
    out = {"key_pages": kp, "value_pages": vp}
    if c["op"] == "step":
        q = _rotate(query.float(), cos, sin)
        out["out"] = _attention(q, kp, vp, table, lengths + 1, s["scale"], s["sink"], s["local"]).to(kp.dtype)
    elif c["query"]:
        counted = (at < s["counts"].long()[:, None])[:, None, :, None]
        out["query"] = torch.where(counted, _rotate(query.float(), cos, sin), 0.0).to(kp.dtype)
        out["key"] = torch.where(counted, rotated, 0.0).to(kp.dtype)
    return out


# ---------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    dtype = DTYPES[c["dtype"]]
    page, D, KV, G = c["page"], c["D"], c["KV"], c["H"] // c["KV"]
    lengths = _lengths(c)
    new = _counts(c) if c["op"] == "append" else [_new(c)] * c["B"]
    half = D // 2

    def turned(x, b, n, m):
        """x (heads, m, D) of sequence b at positions n .. n + m - 1, as pairs of coordinates turned by the angles."""
        if c["table"] == "position":
            cos, sin = s["cos"][n:n + m].double(), s["sin"][n:n + m].double()
        else:
            cos, sin = s["cos"][b, :m].double(), s["sin"][b, :m].double()
        first, second = x[..., :half].double(), x[..., half:].double()
        return torch.cat([first * cos[:, :half] - second * sin[:, :half],
                          second * cos[:, half:] + first * sin[:, half:]], dim=-1)

    result = {}
    if c["op"] != "attend":
        kp, vp = s["key_pages"].double(), s["value_pages"].double()
        if c["op"] == "append" and c["query"]:
            result["query"] = torch.zeros(c["B"], c["H"], c["N"], D, dtype=torch.float64, device="cuda")
            result["key"] = torch.zeros(c["B"], KV, c["N"], D, dtype=torch.float64, device="cuda")
        for b, (n, m) in enumerate(zip(lengths, new)):
            k = turned(s["key"][b, :, :m], b, n, m)
            if "query" in result:
                result["query"][b, :, :m] = turned(s["query"][b, :, :m], b, n, m)
                result["key"][b, :, :m] = k
            v = s["value"][b, :, :m].double()
            done = 0
            while done < m:         # page by page
                slot = (n + done) % page
                take = min(page - slot, m - done)
                p = int(s["page_table"][b, (n + done) // page])
                kp[p, :, slot:slot + take] = k[:, done:done + take]
                vp[p, :, slot:slot + take] = v[:, done:done + take]
                done += take
        result["key_pages"], result["value_pages"] = kp, vp
    if c["op"] == "append":
        return result
    out = torch.zeros(c["B"], 1, c["H"], D, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(lengths, new)):
        n += m
        pages = s["page_table"][b, :-(-n // page)].long()
        if c["op"] == "step":       # the new key is attended as it is stored
            k = kp[pages].to(dtype).double().transpose(0, 1).reshape(KV, -1, D)[:, :n]
            v = vp[pages].transpose(0, 1).reshape(KV, -1, D)[:, :n]
            q = turned(s["query"][b], b, n - 1, 1)[:, 0]
        else:
            k = s["key_pages"][pages].double().transpose(0, 1).reshape(KV, -1, D)[:, :n]
            v = s["value_pages"][pages].double().transpose(0, 1).reshape(KV, -1, D)[:, :n]
            q = s["query"][b, :, 0].double()
        for h in range(KV):
            w = int(s["local"][h]) if c["spans"] else n
            rows = None
            if c["spans"] and n > SINK + w:
                rows = torch.cat([torch.arange(SINK), torch.arange(n - w, n)]).cuda()
            kh, vh = (k[h], v[h]) if rows is None else (k[h][rows], v[h][rows])
            p = torch.softmax(q[h * G:(h + 1) * G] @ kh.T * s["scale"], dim=-1)
            out[b, 0, h * G:(h + 1) * G] = p @ vh
    result["out"] = out
    return result
