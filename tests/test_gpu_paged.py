"""Paged cache on the GPU against a plain implementation in 64 bits.

Tolerances, derived and not measured.  u = 2^-23 bounds one fp32 operation (a tensor core may truncate where
an FMA rounds).  Stored values are off by half a step of their type, eps/2 of the value (plus the smallest
step of fp16 near zero).

A score is a sum of D products scaled once: off by at most (D + 8) u sum|q_d k_d| scale.  A rotated coordinate is
two products and a sum: off by 3u (|a cos| + |b sin|), which adds at most 6u * 2 max|..| per factor and is covered by
counting 16 more operations.  exp of a score that is off by e is off by the factor 1 + e (and 2^-20 for the
exponential itself, its argument rounded at a magnitude up to 64).  With every weight off by at most f, a weighted
mean is off by at most 2 f sum p|v| (numerator and denominator), and its sums over n rows add n u sum p|v|.
"""
import pytest
import torch

import moa_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
F16, BF16 = torch.float16, torch.bfloat16


def _half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return 2.0 ** -25 if dtype == F16 else 0.0


class Case:
    """A pool with pages handed out in a shuffled order; what no token is in holds NaN."""

    def __init__(self, lengths, H, KV, D, page, dtype, layout="heads", room=1, seed=0, width=None):
        gen = torch.Generator().manual_seed(seed)
        self.H, self.KV, self.D, self.page, self.dtype = H, KV, D, page, dtype
        self.B = len(lengths)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        need = [-(-(max(n, 0) + room) // page) if n >= 0 else 0 for n in lengths]
        total = sum(need) + 3
        order = torch.randperm(total, generator=gen).int()
        width = width or max(need + [1]) + 1
        table = torch.full((self.B, width), -1, dtype=torch.int32)
        table[:, -1] = 2 ** 31 - 1
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table.cuda()
        self.kp = self.empty_pool(total, layout)
        self.vp = self.empty_pool(total, layout)
        self.gen = gen
        for b, n in enumerate(lengths):
            if n > 0:
                pages, slots = self.places(b, torch.arange(n))
                self.kp[pages, :, slots] = self.normal(n, KV, D)
                self.vp[pages, :, slots] = self.normal(n, KV, D)

    def empty_pool(self, total, layout):
        nan = float("nan")
        if layout == "heads":
            return torch.full((total, self.KV, self.page, self.D), nan, dtype=self.dtype, device="cuda")
        if layout == "tokens":
            return torch.full((total, self.page, self.KV, self.D), nan, dtype=self.dtype, device="cuda").transpose(1, 2)
        both = torch.full((total, 2, self.KV, self.page + 1, self.D + 8), nan, dtype=self.dtype, device="cuda")
        return both[:, 1, :, 1:, 8:]            # padded rows and heads, a pool inside a larger one

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen).to(self.dtype).cuda()

    def places(self, b, pos):
        pos = pos.to("cuda")
        return self.table[b, pos // self.page].long(), pos % self.page

    def pool(self):
        return self.kp, self.vp, self.table, self.lengths


def tables(D, positions, kind, theta=10000.0):
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    angle = positions.to("cuda").double()[..., None] * inv
    angle = torch.cat([angle, angle], -1)
    return angle.cos().to(kind), angle.sin().to(kind)


def rotated64(x, cos, sin):
    """x (..., D) in 64 bits with tables that broadcast; returns the value and |a cos| + |b sin|."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    half = x.shape[-1] // 2
    other = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos + other * sin, (x * cos).abs() + (other * sin).abs()


def attention64(case, q, n, scale, sink=None, local=None, dropped=()):
    """(B, 1, H, D) in 64 bits over the first n[b] tokens as the pool holds them, and the tolerance of an fp32 result."""
    B, H, D, G = case.B, case.H, case.D, case.H // case.KV
    out = torch.zeros(B, 1, H, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for b in range(B):
        m = max(int(n[b]), 0)
        pos_all = torch.tensor([j for j in range(m) if (b, j) not in dropped], dtype=torch.long, device="cuda")
        for g in range(case.KV):
            pos = pos_all
            if sink is not None:
                pos = pos[(pos < sink[g]) | (pos >= m - local[g])]
            if len(pos) == 0:
                continue
            pages, slots = case.places(b, pos)
            k, v = case.kp[pages, g, slots].double(), case.vp[pages, g, slots].double()
            qh = q[b, g * G:(g + 1) * G, 0].double()
            p = torch.softmax(qh @ k.T * scale, -1)
            out[b, 0, g * G:(g + 1) * G] = p @ v
            off = ((D + 24) * U * scale * (qh.abs() @ k.abs().T)).max(-1).values + 2.0 ** -20
            tol[b, 0, g * G:(g + 1) * G] = (2 * off[:, None] + len(pos) * U) * (p @ v.abs())
    return out, tol


def close(out, ref, tol, what=""):
    tol = tol + _half_step(out.dtype) * ref.abs() * (1 + 2 ** -8) + _tiny(out.dtype) + 1e-30
    worst = ((out.double() - ref).abs() / tol).max().item() if out.numel() else 0.0
    assert not torch.isnan(out).any(), what
    assert worst <= 1.0, (what, worst)


def same_pool(pool, before, rows):
    """The pool is as before but for the (page, slot) rows given."""
    touched = torch.zeros(pool.shape[0], pool.shape[2], dtype=torch.bool, device="cuda")
    for pages, slots in rows:
        touched[pages, slots] = True
    a, b = pool.transpose(1, 2)[~touched], before.transpose(1, 2)[~touched]
    assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


# ------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,KV,page,layout", [(128, 8, 2, 16, "heads"), (64, 3, 3, 32, "tokens"), (64, 5, 1, 1, "heads"),
                                               (128, 4, 4, 64, "inside")])
@pytest.mark.parametrize("N,lengths,counts", [(1, [0, 15, 16, 63, 200], None), (37, [5, 0, 64, 31], [37, 1, 0, 20]),
                                             (130, [7, -1, 100], [129, 130, 500]), (3, [9], [-4])])
@pytest.mark.parametrize("kind", ["none", "position", "position16", "token", "shared token"])
def test_append(dtype, D, H, KV, page, layout, N, lengths, counts, kind):
    c = Case(lengths, H, KV, D, page, dtype, layout, room=N)
    qkv = c.normal(c.B, N, H + 2 * KV, D)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([H, KV, KV], 2))
    pos = c.lengths.cpu()[:, None] + torch.arange(N)
    rope = None
    if kind.startswith("position"):
        cos, sin = rope = tables(D, torch.arange(max(lengths) + N), torch.float32 if kind == "position" else dtype)
        cos, sin = cos[pos.clamp(min=0)], sin[pos.clamp(min=0)]
    elif kind == "token":
        cos, sin = rope = tables(D, pos, dtype)
    elif kind == "shared token":
        cos, sin = rope = tables(D, torch.arange(N)[None] + 11, torch.float32)
        cos, sin = cos.expand(c.B, -1, -1), sin.expand(c.B, -1, -1)
    kb, vb, qkvb, before = c.kp.clone(), c.vp.clone(), qkv.clone(), c.lengths.clone()
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    got = moa_b200.paged_append(k, v, *c.pool(), counts=cnt, rope=rope, query=q if rope is not None else None)
    moa_b200.check_device_status()
    assert torch.equal(c.lengths, before) and torch.equal(qkv, qkvb)
    rows = []
    for b in range(c.B):
        m = 0 if lengths[b] < 0 else min(max(counts[b], 0), N) if counts is not None else N
        pages, slots = c.places(b, lengths[b] + torch.arange(m))
        rows.append((pages, slots))
        kk, vv = k[b, :, :m].transpose(0, 1), v[b, :, :m].transpose(0, 1)
        assert torch.equal(c.vp[pages, :, slots], vv)
        if rope is None:
            assert got is None and torch.equal(c.kp[pages, :, slots], kk)
        else:
            ref, parts = rotated64(kk, cos[b, :m, None], sin[b, :m, None])
            close(c.kp[pages, :, slots], ref, 3 * U * parts)
            ref_q, parts = rotated64(q[b, :, :m], cos[b, :m], sin[b, :m])
            close(got[0][b, :, :m], ref_q, 3 * U * parts)
            assert torch.equal(got[1][b, :, :m].transpose(0, 1), c.kp[pages, :, slots])
            assert not got[0][b, :, m:].any() and not got[1][b, :, m:].any()
    same_pool(c.kp, kb, rows)
    same_pool(c.vp, vb, rows)


def test_append_rotates_as_the_prefill_does():
    """Bit for bit what apply_rotary_pos_emb makes of the same query and key."""
    from moa_b200.module import apply_rotary_pos_emb, rotary_cos_sin

    c = Case([0, 0], 4, 4, 128, 64, F16, room=77)
    q, k, v = c.normal(2, 4, 77, 128), c.normal(2, 4, 77, 128), c.normal(2, 4, 77, 128)
    cos, sin = rotary_cos_sin(torch.arange(77, device="cuda")[None].expand(2, -1), 128, 10000.0, F16)
    qr, kr = moa_b200.paged_append(k, v, *c.pool(), rope=(cos, sin), query=q)
    q2, k2 = apply_rotary_pos_emb(q.clone(), k.clone(), cos, sin)
    assert torch.equal(qr, q2) and torch.equal(kr, k2)


def test_append_advances_when_asked():
    c = Case([3, -1, 60], 2, 2, 64, 16, F16, room=9)
    k, v = c.normal(3, 2, 9, 64), c.normal(3, 2, 9, 64)
    counts = torch.tensor([2, 5, 77], dtype=torch.int32, device="cuda")
    moa_b200.paged_append(k, v, *c.pool(), counts=counts, advance=True)
    assert c.lengths.tolist() == [5, -1, 69]
    moa_b200.paged_append(k[:, :, :1], v[:, :, :1], *c.pool(), advance=True)
    assert c.lengths.tolist() == [6, -1, 70]


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
def test_append_without_a_page_stores_nothing_and_says_so(bad):
    c = Case([10, 20], 2, 2, 64, 16, F16, room=20)
    c.table[1, 2] = bad                       # positions 32..47 of the second sequence
    k, v = c.normal(2, 2, 20, 64), c.normal(2, 2, 20, 64)
    kb = c.kp.clone()
    moa_b200.paged_append(k, v, *c.pool())
    rows = [c.places(0, torch.arange(10, 30)), c.places(1, torch.arange(20, 32))]
    same_pool(c.kp, kb, rows)
    assert torch.equal(c.kp[rows[1][0], :, rows[1][1]], k[1, :, :12].transpose(0, 1))
    with pytest.raises(moa_b200.MoaError, match="no page"):
        moa_b200.check_device_status()
    moa_b200.check_device_status()            # said once


def test_append_behind_the_page_table_or_the_rope_table():
    c = Case([30], 1, 1, 64, 16, F16, room=2, width=2)
    c.table[0, :2] = torch.tensor([0, 1], dtype=torch.int32)
    k, v = c.normal(1, 1, 4, 64), c.normal(1, 1, 4, 64)
    kb = c.kp.clone()
    moa_b200.paged_append(k, v, *c.pool())    # positions 30..33; the table holds 32
    same_pool(c.kp, kb, [c.places(0, torch.arange(30, 32))])
    with pytest.raises(moa_b200.MoaError, match="no page"):
        moa_b200.check_device_status()
    c = Case([30], 1, 1, 64, 16, F16, room=4)
    kb = c.kp.clone()
    moa_b200.paged_append(k, v, *c.pool(), rope=tables(64, torch.arange(33), torch.float32))
    same_pool(c.kp, kb, [c.places(0, torch.arange(30, 33))])
    with pytest.raises(moa_b200.MoaError, match="rope row"):
        moa_b200.check_device_status()


def test_append_copies_rows_it_cannot_read_in_place():
    c = Case([4, 9], 2, 2, 64, 16, BF16, room=5)
    wide = c.normal(2, 2, 5, 67)
    k = wide[..., 1:65]                       # rows that start at odd addresses
    v = c.normal(2, 2, 64, 5).transpose(2, 3)
    moa_b200.paged_append(k, v, *c.pool())
    for b in range(2):
        pages, slots = c.places(b, int(c.lengths[b]) + torch.arange(5))
        assert torch.equal(c.kp[pages, :, slots], k[b].transpose(0, 1))
        assert torch.equal(c.vp[pages, :, slots], v[b].transpose(0, 1))


# ------------------------------------------------------------------------------------------- attention
def _decode(c, scale=None, spans=None, qscale=1.5, out_dtype=None, check=True, n=None):
    q = (c.normal(c.B, 1, c.H, c.D) * qscale).transpose(1, 2)
    scale = scale if scale is not None else c.D ** -0.5
    sink = local = None
    if spans is not None:
        sink, local = (torch.tensor(s, dtype=torch.int64, device="cuda") for s in spans)
    out = moa_b200.paged_decode(q, *c.pool(), scale, sink_size=sink, local_size=local, out_dtype=out_dtype)
    if check:
        ref, tol = attention64(c, q, c.lengths if n is None else n, scale, *(spans or (None, None)))
        close(out, ref, tol)
    return q, out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV", [(1, 1), (4, 4), (6, 2), (8, 1), (16, 2), (24, 2), (12, 1), (40, 1), (35, 5)])
@pytest.mark.parametrize("lengths,page", [([0, 1, 2, 15, 16, 17, 0], 16), ([127, 128, 129, 255, 257, 31], 32),
                                         ([1000, 1, 2047], 64), ([5, 300], 1), ([700, 0, 65], 256)])
def test_decode(dtype, D, H, KV, lengths, page):
    c = Case(lengths, H, KV, D, page, dtype, layout="tokens" if page == 64 else "heads", room=0)
    _decode(c)
    _decode(c, out_dtype=torch.float32)
    moa_b200.check_device_status()


@pytest.mark.parametrize("H,KV,lengths", [(8, 8, [20011]), (64, 8, [30001]), (16, 1, [40007, 3]), (4, 1, [9001] * 5),
                                         (8, 2, [0] * 37 + [8000]), (2, 2, list(range(0, 260, 7)) * 5)])
def test_decode_long_and_ragged(H, KV, lengths):
    for D, dtype in ((128, BF16), (64, F16)):
        c = Case(lengths, H, KV, D, 64, dtype, room=0)
        _decode(c, out_dtype=torch.float32)
        _decode(c)
    moa_b200.check_device_status()


@pytest.mark.parametrize("spans", [([64] * 4, [256, 64, 1024, 0]), ([0] * 4, [1, 17, 64, 5000]), ([0, 3, 5000, 33], [0, 0, 0, 100]),
                                   ([2 ** 62] * 4, [2 ** 62] * 4), ([-5, -1, 0, 1], [-7, 2, -1, -2 ** 62])])
@pytest.mark.parametrize("H,page", [(4, 16), (12, 64)])
def test_decode_spans(spans, H, page):
    c = Case([0, 1, 63, 64, 321, 1500], H, 4, 128, page, F16, room=0)
    clamped = tuple([max(0, min(x, 10 ** 6)) for x in s] for s in spans)
    q, out = _decode(c, spans=spans, check=False)
    ref, tol = attention64(c, q, c.lengths, c.D ** -0.5, *clamped)
    close(out, ref, tol)
    moa_b200.check_device_status()


def test_pages_outside_the_span_are_not_touched():
    """A sliding window lets the pages behind it go: their entries in the table may be anything."""
    c = Case([1000, 400], 2, 2, 64, 16, F16, room=0)
    q = c.normal(2, 2, 1, 64)
    sink, local = torch.tensor([16, 16], device="cuda"), torch.tensor([100, 64], device="cuda")
    ref = moa_b200.paged_decode(q, *c.pool(), 0.125, sink_size=sink, local_size=local)
    c.table[0, 1:56] = -7
    c.table[1, 1:18] = 2 ** 31 - 1
    assert torch.equal(ref, moa_b200.paged_decode(q, *c.pool(), 0.125, sink_size=sink, local_size=local))
    moa_b200.check_device_status()


@pytest.mark.parametrize("G", [1, 12])
def test_decode_leaves_out_tokens_without_a_page(G):
    c = Case([100, 40], 2 * G, 2, 64, 16, F16, room=0)
    gone = c.table[0, 2].item()
    q = c.normal(2, 2 * G, 1, 64)
    for bad in (-1, 12345, gone):
        c.table[0, 2] = bad if bad != gone else -1
        out = moa_b200.paged_decode(q, *c.pool(), 0.2)
        c.table[0, 2] = gone
        ref, tol = attention64(c, q, c.lengths, 0.2, dropped={(0, j) for j in range(32, 48)})
        close(out, ref, tol)
        with pytest.raises(moa_b200.MoaError, match="no page for position"):
            moa_b200.check_device_status()
    c.table[1, :] = -1                        # a sequence without any page: zeros
    out = moa_b200.paged_decode(q, *c.pool(), 0.2)
    assert not out[1].any()
    with pytest.raises(moa_b200.MoaError, match="no page"):
        moa_b200.check_device_status()


def test_lengths_beyond_the_page_table_are_cut_and_reported():
    c = Case([64, 10], 2, 2, 64, 16, F16, room=0, width=4)
    c.table[0, :4] = torch.arange(4, dtype=torch.int32)
    c.table[1, :] = torch.tensor([4, -1, -1, -1], dtype=torch.int32)
    c.kp.normal_(), c.vp.normal_()
    q = c.normal(2, 2, 1, 64)
    ref = moa_b200.paged_decode(q, *c.pool(), 0.2)
    moa_b200.check_device_status()
    c.lengths[0] = 2 ** 31 - 1
    assert torch.equal(ref, moa_b200.paged_decode(q, *c.pool(), 0.2))
    with pytest.raises(moa_b200.MoaError, match="more than its row"):
        moa_b200.check_device_status()
    c.lengths[0] = -5                          # no sequence
    assert not moa_b200.paged_decode(q, *c.pool(), 0.2)[0].any()
    moa_b200.check_device_status()


def test_extreme_scores():
    """Scores far from zero on either side, all equal, and rows whose weights underflow."""
    for dtype in (F16, BF16):
        c = Case([50, 333], 4, 2, 64, 16, dtype, room=0)
        for scale in (0.0, 1.0, -1.0, 20.0, 1e-30):
            _decode(c, scale=scale, qscale=2.0, out_dtype=torch.float32)


def test_non_finite_values_go_where_the_formula_puts_them():
    c = Case([40, 40], 2, 2, 64, 16, BF16, room=0)
    q = c.normal(2, 2, 1, 64).abs() + 0.1
    pages, slots = c.places(0, torch.tensor([7]))
    c.vp[pages, 0, slots, 5] = float("inf")
    c.kp[pages, 1, slots] = -float("inf")      # score -inf: no weight
    out = moa_b200.paged_decode(q, *c.pool(), 0.1)
    assert out[0, 0, 0, 5] == float("inf") and torch.isfinite(out).sum() == out.numel() - 1
    ref, tol = attention64(c, q, c.lengths, 0.1, dropped={(0, 7)})
    close(out[0, :, 1], ref[0, :, 1], tol[0, :, 1])
    c.kp[pages, 1, slots, 3] = float("nan")
    out = moa_b200.paged_decode(q, *c.pool(), 0.1)
    assert torch.isnan(out[0, 0, 1]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("dtype,D,H,KV,page", [(F16, 128, 4, 4, 16), (BF16, 128, 24, 3, 64), (F16, 64, 2, 2, 8), (BF16, 64, 36, 3, 16),
                                              (F16, 64, 40, 2, 32), (BF16, 128, 24, 2, 16)])
@pytest.mark.parametrize("step", ["attend", "plain step", "step"])
@pytest.mark.parametrize("spanned", [False, True])
def test_many_short_sequences(dtype, D, H, KV, page, step, spanned):
    """More (sequence, key head) pairs than blocks, and page tables that reach 256 tokens at most."""
    gen = torch.Generator().manual_seed(5)
    lengths = [int(n) for n in torch.randint(0, 190, (210,), generator=gen)]
    lengths[3], lengths[50], lengths[209], lengths[7] = 0, 1, 191, 190
    if step != "attend":
        lengths[11], lengths[208] = -1, -9
    c = Case(lengths, H, KV, D, page, dtype, layout="tokens" if KV == 3 else "heads", room=1, width=256 // page)
    assert c.table.shape[1] * page == 256 and c.B * KV > 296
    c.table[:, -1] = -1
    spans = ([0, 5, 16, 200][:KV], [33, 64, 0, 7][:KV]) if spanned else (None, None)
    sink, local = (None, None) if not spanned else (torch.tensor(x, device="cuda") for x in spans)
    q = c.normal(c.B, H, 1, D)
    kb, vb = c.kp.clone(), c.vp.clone()
    if step == "attend":
        args, n, qr, rows = {}, c.lengths, q, []
    else:
        k, v = c.normal(c.B, KV, 1, D), c.normal(c.B, KV, 1, D)
        args, qr = dict(key=k, value=v), q
        n = torch.where(c.lengths < 0, c.lengths, c.lengths + 1)
        live = (c.lengths >= 0).nonzero()[:, 0]
        rows = [c.places(b, c.lengths[b:b + 1].long()) for b in live.tolist()]
        if step == "step":
            args["rope"] = tables(D, torch.arange(256), torch.float32)
            cos, sin = (t[c.lengths.long().clamp(min=0)] for t in args["rope"])
            qr = rotated64(q, cos[:, None, None], sin[:, None, None])[0]
    out32 = moa_b200.paged_decode(q, *c.pool(), 0.11, sink_size=sink, local_size=local, out_dtype=torch.float32, **args)
    out = moa_b200.paged_decode(q, *c.pool(), 0.11, sink_size=sink, local_size=local, **args)
    moa_b200.check_device_status()
    same_pool(c.kp, kb, rows)
    same_pool(c.vp, vb, rows)
    if rows:
        for b, (pages, slots) in zip(live.tolist(), rows):
            assert torch.equal(c.vp[pages, :, slots][0], v[b, :, 0])
            if step == "step":
                ref, parts = rotated64(k[b, :, 0], cos[b], sin[b])
                close(c.kp[pages, :, slots][0], ref, 3 * U * parts)
            else:
                assert torch.equal(c.kp[pages, :, slots][0], k[b, :, 0])
    ref, tol = attention64(c, qr, n, 0.11, *spans)
    close(out32, ref, tol)
    close(out, ref, tol)
    assert torch.equal(out32.to(dtype), out)


@pytest.mark.parametrize("B,H,KV,page,top", [(300, 2, 2, 64, 500), (2, 300, 300, 16, 40), (600, 1, 1, 16, 90), (270, 12, 1, 32, 700)])
def test_more_sequences_or_heads_than_are_held_in_shared_memory(B, H, KV, page, top):
    gen = torch.Generator().manual_seed(8)
    lengths = [int(n) for n in torch.randint(0, top, (B,), generator=gen)]
    c = Case(lengths, H, KV, 64, page, F16, room=1)
    spans = ([int(x) for x in torch.randint(0, 20, (KV,), generator=gen)], [int(x) for x in torch.randint(0, 300, (KV,), generator=gen)])
    _decode(c)
    _decode(c, spans=spans)
    q, k, v = c.normal(B, H, 1, 64), c.normal(B, KV, 1, 64), c.normal(B, KV, 1, 64)
    out = moa_b200.paged_decode(q, *c.pool(), 0.2, key=k, value=v, advance=True)
    assert c.lengths.tolist() == [n + 1 for n in lengths]
    ref, tol = attention64(c, q, c.lengths, 0.2)
    close(out, ref, tol)
    moa_b200.check_device_status()


def test_decode_into_a_wider_buffer_and_from_strided_queries():
    c = Case([70, 5, 200], 6, 3, 128, 32, F16, layout="inside", room=0)
    wide = torch.full((3, 1, 10, 128), 7.0, dtype=F16, device="cuda")
    qkv = c.normal(3, 1, 12, 128)
    q = qkv[:, :, 2:8].transpose(1, 2)
    got = moa_b200.paged_decode(q, *c.pool(), 0.09, out=wide[:, :, 3:9])
    assert got.data_ptr() == wide[:, :, 3:9].data_ptr() and (wide[:, :, :3] == 7).all() and (wide[:, :, 9:] == 7).all()
    ref, tol = attention64(c, q, c.lengths, 0.09)
    close(got, ref, tol)
    odd = c.normal(3, 6, 1, 131)[..., 3:]
    ref, tol = attention64(c, odd, c.lengths, 0.09)
    close(moa_b200.paged_decode(odd, *c.pool(), 0.09), ref, tol)
    one = c.normal(1, 6, 1, 128).expand(3, 6, 1, 128)
    ref, tol = attention64(c, one, c.lengths, 0.09)
    close(moa_b200.paged_decode(one, *c.pool(), 0.09), ref, tol)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 elements with its tokens in the last pages."""
    D, KV, page, total = 128, 2, 64, 2 ** 32 // (128 * 2 * 64) + 40
    c = Case([150, 33], 4, KV, D, page, F16, room=1)
    need = int((c.table[:, :-1] >= 0).sum())
    kp, vp = (torch.empty(total, KV, page, D, dtype=F16, device="cuda") for _ in range(2))
    far = torch.where((c.table >= 0) & (c.table < 2 ** 30), total - 1 - c.table, c.table)
    assert far.max() == 2 ** 31 - 1 and need > 3
    pages = torch.arange(c.kp.shape[0], device="cuda")
    kp[total - 1 - pages], vp[total - 1 - pages] = c.kp, c.vp
    q, k, v = c.normal(2, 4, 1, D), c.normal(2, KV, 1, D), c.normal(2, KV, 1, D)
    ref = moa_b200.paged_decode(q, *c.pool(), 0.09, key=k, value=v)
    got = moa_b200.paged_decode(q, kp, vp, far, c.lengths, 0.09, key=k, value=v)
    assert torch.equal(ref, got)
    moa_b200.paged_append(k, v, kp, vp, far, c.lengths + 1)
    for b in range(2):
        n = int(c.lengths[b]) + 1
        assert torch.equal(kp[far[b, n // page].long(), :, n % page], k[b, :, 0])
    moa_b200.check_device_status()


# ------------------------------------------------------------------------------------------- the step
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,KV,page,layout", [(128, 4, 4, 16, "heads"), (64, 12, 1, 32, "tokens"), (128, 16, 2, 64, "inside"),
                                               (64, 40, 2, 1, "heads"), (128, 20, 1, 16, "tokens")])
@pytest.mark.parametrize("lengths", [[0, 1, 15, 16, -1, 127], [1000, 0, 2047, -3], [128]])
@pytest.mark.parametrize("kind", ["none", "position", "token"])
@pytest.mark.parametrize("spanned", [False, True])
def test_step(dtype, D, H, KV, page, layout, lengths, kind, spanned):
    c = Case(lengths, H, KV, D, page, dtype, layout, room=1)
    qkv = c.normal(c.B, 1, H + 2 * KV, D)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([H, KV, KV], 2))
    rope = None
    if kind == "position":
        rope = tables(D, torch.arange(max(lengths) + 1), torch.float32)
        cos, sin = (t[c.lengths.long().clamp(min=0)] for t in rope)
    elif kind == "token":
        rope = tables(D, c.lengths.cpu()[:, None], dtype)
        cos, sin = (t[:, 0] for t in rope)
    spans = None
    if spanned:
        spans = ([3, 0, 64, 16][:KV] + [1] * max(0, KV - 4), [100, 1, 64, 0][:KV] + [9] * max(0, KV - 4))
    kb, vb, before = c.kp.clone(), c.vp.clone(), c.lengths.clone()
    sink, local = (None, None) if spans is None else (torch.tensor(s, device="cuda") for s in spans)
    args = dict(key=k, value=v, rope=rope, sink_size=sink, local_size=local)
    out32 = moa_b200.paged_decode(q, *c.pool(), D ** -0.5, out_dtype=torch.float32, **args)
    out = moa_b200.paged_decode(q, *c.pool(), D ** -0.5, **args)
    moa_b200.check_device_status()
    assert torch.equal(c.lengths, before)
    rows = []
    for b, n in enumerate(lengths):
        if n < 0:
            assert not out[b].any() and not out32[b].any()
            continue
        pages, slots = c.places(b, torch.tensor([n]))
        rows.append((pages, slots))
        assert torch.equal(c.vp[pages, :, slots][0], v[b, :, 0])
        if rope is None:
            assert torch.equal(c.kp[pages, :, slots][0], k[b, :, 0])
        else:
            ref, parts = rotated64(k[b, :, 0], cos[b], sin[b])
            close(c.kp[pages, :, slots][0], ref, 3 * U * parts)
    same_pool(c.kp, kb, rows)
    same_pool(c.vp, vb, rows)
    qr = q if rope is None else rotated64(q, cos[:, None, None], sin[:, None, None])[0]
    ref, tol = attention64(c, qr, torch.where(c.lengths < 0, c.lengths, c.lengths + 1), D ** -0.5, *(spans or (None, None)))
    close(out32, ref, tol)
    close(out, ref, tol)
    assert torch.equal(out32.to(dtype), out)
    # the two calls that the step stands for, without the rotation of the query
    if rope is None:
        n = torch.where(c.lengths < 0, c.lengths, c.lengths + 1)
        two = moa_b200.paged_decode(q, c.kp, c.vp, c.table, n, D ** -0.5, sink_size=sink, local_size=local)
        close(two, ref, tol)     # not bit for bit: the step adds the new token first, and fp32 sums depend on their order


def test_step_advances_and_decodes_on():
    """Sixty steps by the kernel's own bookkeeping: pages and lengths are what sixty appends make of them."""
    c = Case([0, 13, -1, 64], 4, 2, 64, 16, BF16, room=61)
    d = Case([0, 13, -1, 64], 4, 2, 64, 16, BF16, room=61)
    assert torch.equal(c.table, d.table)
    cos, sin = tables(64, torch.arange(200), torch.float32)
    for step in range(60):
        q, k, v = c.normal(4, 4, 1, 64), c.normal(4, 2, 1, 64), c.normal(4, 2, 1, 64)
        out = moa_b200.paged_decode(q, *c.pool(), 0.125, key=k, value=v, rope=(cos, sin), advance=True)
        moa_b200.paged_append(k, v, *d.pool(), rope=(cos, sin), advance=True)
        assert torch.equal(c.lengths, d.lengths)
        if step % 20 == 19:
            at = (d.lengths.long() - 1).clamp(min=0)
            qr = rotated64(q, cos[at][:, None, None], sin[at][:, None, None])[0]
            ref, tol = attention64(d, qr, d.lengths, 0.125)
            close(out, ref, tol)
    assert c.lengths.tolist() == [60, 73, -1, 124]
    for a, b in ((c.kp, d.kp), (c.vp, d.vp)):
        assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def test_step_without_a_page_or_a_rope_row_attends_the_rest():
    c = Case([32, 20], 4, 2, 64, 16, F16, room=1)
    q, k, v = c.normal(2, 4, 1, 64), c.normal(2, 2, 1, 64), c.normal(2, 2, 1, 64)
    c.table[0, 2] = -1
    kb = c.kp.clone()
    out = moa_b200.paged_decode(q, *c.pool(), 0.2, key=k, value=v)
    same_pool(c.kp, kb, [c.places(1, torch.tensor([20]))])
    ref, tol = attention64(c, q, c.lengths + 1, 0.2, dropped={(0, 32)})
    close(out, ref, tol)
    with pytest.raises(moa_b200.MoaError, match="no page"):
        moa_b200.check_device_status()
    c = Case([32, 20], 4, 2, 64, 16, F16, room=1)
    kb = c.kp.clone()
    out = moa_b200.paged_decode(q, *c.pool(), 0.2, key=k, value=v, rope=tables(64, torch.arange(32), torch.float32))
    same_pool(c.kp, kb, [c.places(1, torch.tensor([20]))])
    assert torch.isfinite(out).all()
    with pytest.raises(moa_b200.MoaError, match="rope row"):
        moa_b200.check_device_status()
    c = Case([32, 20], 4, 2, 64, 16, F16, room=0, width=2)     # the table ends where the new token would go
    c.table[0] = torch.tensor([0, 1], dtype=torch.int32)
    c.table[1] = torch.tensor([2, 3], dtype=torch.int32)
    c.kp.normal_(), c.vp.normal_()
    out = moa_b200.paged_decode(q, *c.pool(), 0.2, key=k, value=v)
    ref, tol = attention64(c, q, torch.tensor([32, 21]), 0.2)
    close(out, ref, tol)
    with pytest.raises(moa_b200.MoaError):
        moa_b200.check_device_status()


# ------------------------------------------------------------------------------------------- around them
def test_results_do_not_depend_on_the_run():
    c = Case([5000, 1, 777, 12000], 16, 4, 128, 64, BF16, room=0)
    q = c.normal(4, 16, 1, 128)
    first = moa_b200.paged_decode(q, *c.pool(), 0.09)
    for _ in range(20):
        assert torch.equal(first, moa_b200.paged_decode(q, *c.pool(), 0.09))


def test_calls_on_two_streams_at_once():
    c = Case([9000, 30], 8, 2, 128, 64, F16, room=0)
    d = Case([50, 7000, 400], 8, 8, 64, 16, BF16, room=0)
    qc, qd = c.normal(2, 8, 1, 128), d.normal(3, 8, 1, 64)
    rc, rd = moa_b200.paged_decode(qc, *c.pool(), 0.09), moa_b200.paged_decode(qd, *d.pool(), 0.125)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        with torch.cuda.stream(s):
            got.append((rc, moa_b200.paged_decode(qc, *c.pool(), 0.09)))
        with torch.cuda.stream(t):
            got.append((rd, moa_b200.paged_decode(qd, *d.pool(), 0.125)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


def test_two_captured_graphs_replayed_at_once():
    c = Case([9000, 30], 8, 2, 128, 64, F16, room=400)
    d = Case([50, 7000, 400], 8, 8, 64, 16, BF16, room=400)
    graphs = []
    for x in (c, d):
        q, k, v = x.normal(x.B, x.H, 1, x.D), x.normal(x.B, x.KV, 1, x.D), x.normal(x.B, x.KV, 1, x.D)
        x.start = x.lengths.clone()
        x.want = moa_b200.paged_decode(q, *x.pool(), 0.1, key=k, value=v)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = moa_b200.paged_decode(q, *x.pool(), 0.1, key=k, value=v, advance=True)
        graphs.append((g, torch.cuda.Stream(), out, x, q, k, v))
        assert torch.equal(x.lengths, x.start)
    torch.cuda.synchronize()
    for _ in range(40):
        for g, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for g, stream, out, x, q, k, v in graphs:
        assert torch.equal(x.lengths, x.start + 40)
        again = moa_b200.paged_decode(q, x.kp, x.vp, x.table, x.lengths, 0.1)
        assert torch.equal(out, again)
        x.lengths.copy_(x.start)
        assert torch.equal(x.want, moa_b200.paged_decode(q, *x.pool(), 0.1, key=k, value=v))


def test_empty_batches():
    c = Case([5], 4, 2, 64, 16, F16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    out = moa_b200.paged_decode(c.normal(0, 4, 1, 64), c.kp, c.vp, c.table[:0], none, 0.1)
    assert out.shape == (0, 1, 4, 64)
    moa_b200.paged_append(c.normal(0, 2, 3, 64), c.normal(0, 2, 3, 64), c.kp, c.vp, c.table[:0], none)
    before = c.kp.clone()
    moa_b200.paged_append(c.normal(1, 2, 0, 64), c.normal(1, 2, 0, 64), *c.pool())
    same_pool(c.kp, before, [])


def test_the_ring_cache_and_pages_with_spans_agree():
    """Decode of a prompt and 150 further tokens: per-head rings of sink + window against pages with those spans."""
    caps, sinks, B, D, N = [128, 192, 320], [64, 16, 64], 2, 64, 200
    H = len(caps)
    ring = moa_b200.StaticCircularCache([caps], B, D, [sinks], "cuda", F16)
    c = Case([0] * B, H, H, D, 16, F16, room=N + 150)
    k, v = c.normal(B, H, N, D), c.normal(B, H, N, D)
    ring.update(k, v, 0)
    moa_b200.paged_append(k, v, *c.pool(), advance=True)
    sink, local = ring.static_cache_size[0], ring.circular_cache_size[0]
    for step in range(150):
        q, k, v = c.normal(B, H, 1, D), c.normal(B, H, 1, D), c.normal(B, H, 1, D)
        a = ring.decode_attention(q, k, v, 0, 0.125, out_dtype=torch.float32)
        b = moa_b200.paged_decode(q, *c.pool(), 0.125, key=k, value=v, sink_size=sink, local_size=local, advance=True,
                                  out_dtype=torch.float32)
        if step % 30 == 29:
            ref, tol = attention64(c, q, c.lengths, 0.125, sink.tolist(), local.tolist())
            close(b, ref, tol)
            close(a, ref, tol)
    moa_b200.check_device_status()


@pytest.mark.parametrize("page,lengths", [(2048, [5000, 1, 2048]), (65536, [70000, 3]), (512, [511, 512, 513])])
def test_large_pages(page, lengths):
    c = Case(lengths, 4, 2, 64, page, BF16, room=1)
    _decode(c)
    k, v = c.normal(c.B, 2, 1, 64), c.normal(c.B, 2, 1, 64)
    moa_b200.paged_append(k, v, *c.pool(), advance=True)
    _decode(c)
    moa_b200.check_device_status()


def test_pools_whose_heads_are_one_head_repeated():
    """An expanded dimension (stride zero) for reading: every key head is the same memory."""
    c = Case([100, 333], 6, 1, 128, 64, F16, room=0)
    q = c.normal(2, 6, 1, 128)
    one = moa_b200.paged_decode(q, *c.pool(), 0.09)
    three = moa_b200.paged_decode(q, c.kp.expand(-1, 3, -1, -1), c.vp.expand(-1, 3, -1, -1), c.table, c.lengths, 0.09)
    ref, tol = attention64(c, q, c.lengths, 0.09)
    close(one, ref, tol)
    close(three, ref, tol)


@pytest.mark.parametrize("G", [2, 12])
def test_a_rotated_query_beyond_the_range_of_fp16(G):
    """Coordinates of 60000 become up to 84852 when they are turned; the query is not rounded to fp16 on the way."""
    c = Case([50, 7], 2 * G, 2, 64, 16, F16, room=1)
    q = torch.where(c.normal(2, 2 * G, 1, 64) > 0, 60000.0, -60000.0).half()
    k, v = c.normal(2, 2, 1, 64), c.normal(2, 2, 1, 64)
    cos, sin = tables(64, torch.arange(64), torch.float32)
    out = moa_b200.paged_decode(q, *c.pool(), 1e-6, key=k, value=v, rope=(cos, sin), out_dtype=torch.float32)
    at = c.lengths.long()
    qr = rotated64(q, cos[at][:, None, None], sin[at][:, None, None])[0]
    assert qr.abs().max() > 70000
    ref, tol = attention64(c, qr, c.lengths + 1, 1e-6)
    close(out, ref, tol)


def test_the_output_may_replace_the_query():
    c = Case([3000, 40, 0], 8, 2, 64, 64, BF16, room=0)
    q = c.normal(3, 1, 8, 64)
    ref = moa_b200.paged_decode(q.transpose(1, 2), *c.pool(), 0.125)
    got = moa_b200.paged_decode(q.transpose(1, 2), *c.pool(), 0.125, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, ref)


CHILD = """
import torch, moa_b200
kp, vp = torch.randn(9, 2, 16, 64, device="cuda").half(), torch.randn(9, 2, 16, 64, device="cuda").half()
table, lengths = torch.arange(9, device="cuda", dtype=torch.int32)[None], torch.full((1,), 100, device="cuda", dtype=torch.int32)
q, k = torch.randn(1, 4, 1, 64, device="cuda").half(), torch.randn(1, 2, 1, 64, device="cuda").half()
if CAPTURE:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moa_b200.paged_append(k, k, kp, vp, table, lengths)
        out = moa_b200.paged_decode(q, kp, vp, table, lengths, 0.125, key=k, value=k, advance=True)
    graph.replay(); graph.replay()
else:
    moa_b200.paged_append(k, k, kp, vp, table, lengths, advance=True)
    moa_b200.paged_decode(q, kp, vp, table, lengths, 0.125, key=k, value=k, advance=True)
    out = None
moa_b200.check_device_status()
assert lengths.tolist() == [102], lengths
if out is not None:
    assert torch.equal(out, moa_b200.paged_decode(q, kp, vp, table, lengths - 1, 0.125, key=k, value=k))
print("child ok")
"""


@pytest.mark.parametrize("capture,env", [(True, {}), (False, {"MOA_B200_NVTX": "1"})])
def test_a_process_whose_first_call_is_captured_and_one_with_ranges(capture, env):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", "CAPTURE = %r\n%s" % (capture, CHILD)], cwd=root, text=True,
                          capture_output=True, timeout=300, env={**os.environ, **env, "PYTHONPATH": root})
    assert done.returncode == 0 and "child ok" in done.stdout, done.stderr[-2000:]


def test_compiled_and_python_checks_make_the_same_calls(monkeypatch):
    """The compiled common case against the calls from Python alone, and what it leaves to Python."""
    from moa_b200 import paged

    assert paged._host is not None, "moa_b200/_paged_host.so is not built"
    c = Case([100, 333, -1, 0], 12, 3, 128, 32, BF16, room=9)
    qkv = c.normal(4, 9, 18, 128)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([12, 3, 3], 2))
    counts = torch.tensor([9, 4, 1, 0], dtype=torch.int32, device="cuda")
    sink, local = torch.tensor([4, 0, 64], device="cuda"), torch.tensor([99, 10, 0], device="cuda")
    where, token = tables(128, torch.arange(400), torch.float32), tables(128, torch.arange(9)[None] + 5, BF16)
    one = [t[:, :, :1] for t in (q, k, v)]
    shared = tables(128, torch.arange(1)[None] + 7, torch.float32)
    calls = [lambda: moa_b200.paged_append(k, v, *c.pool()),
             lambda: moa_b200.paged_append(k, v, *c.pool(), counts=counts, rope=where, query=q),
             lambda: moa_b200.paged_append(k, v, *c.pool(), counts=counts, rope=token, query=q[:, :5]),
             lambda: moa_b200.paged_append(k, v, *c.pool(), counts=counts, advance=True),
             lambda: moa_b200.paged_decode(one[0], *c.pool(), 0.1),
             lambda: moa_b200.paged_decode(one[0], *c.pool(), 0.1, sink_size=sink, local_size=local),
             lambda: moa_b200.paged_decode(one[0], *c.pool(), 0.1, key=one[1], value=one[2]),
             lambda: moa_b200.paged_decode(one[0], *c.pool(), 0.1, key=one[1], value=one[2], rope=where, advance=True),
             lambda: moa_b200.paged_decode(one[0], *c.pool(), 0.1, key=one[1], value=one[2], rope=shared, sink_size=sink,
                                           local_size=local)]
    moa_b200.paged_decode(one[0], *c.pool(), 0.1)          # this stream's scratch
    start = [t.clone() for t in (c.kp, c.vp, c.lengths)]

    def results():
        got = []
        for call in calls:
            for t, was in zip((c.kp, c.vp, c.lengths), start):
                t.copy_(was)
            out = call()
            got.append([t.clone() for t in (out if isinstance(out, tuple) else () if out is None else (out,))] +
                       [t.clone() for t in (c.kp, c.vp, c.lengths)])
        return got

    counted = {"decode": 0, "append": 0}

    class Counting:
        def __getattr__(self, name):
            inner = getattr(host, name)

            def call(*args):
                got = inner(*args)
                counted[name] = counted.get(name, 0) + (got is not None)
                return got
            return call

    host = paged._host
    monkeypatch.setattr(paged, "_host", Counting())
    compiled = results()
    assert counted["append"] == 4 and counted["decode"] == 5     # none of them was left to Python
    # what it leaves: copies, an output of the caller's, fp32, gradients, refusals, captures
    before = dict(counted)
    moa_b200.paged_decode(c.normal(4, 12, 1, 131)[..., 3:], *c.pool(), 0.1)
    moa_b200.paged_decode(one[0], *c.pool(), 0.1, out_dtype=torch.float32)
    moa_b200.paged_append(k[..., 1:65].contiguous()[:, :, :0], v[..., :64][:, :, :0], c.kp[..., :64], c.vp[..., :64], c.table, c.lengths)
    with pytest.raises(NotImplementedError):
        moa_b200.paged_decode(one[0].detach().requires_grad_(), *c.pool(), 0.1)
    for bad in (dict(lengths=c.lengths.long()), dict(page_table=c.table[:2]), dict(key=one[1]), dict(sink_size=sink),
                dict(advance=True), dict(rope=where), dict(query=q), dict(query=one[0].half())):
        args = dict(query=one[0], key_pages=c.kp, value_pages=c.vp, page_table=c.table, lengths=c.lengths, sm_scale=0.1)
        args.update(bad)
        with pytest.raises(AssertionError):
            moa_b200.paged_decode(**args)
    for bad in (dict(value=v[:, :2]), dict(counts=counts.long()), dict(query=q), dict(rope=(where[0], where[1][:7]), query=q),
                dict(rope=tuple(t[:, :3] for t in token))):
        args = dict(key=k, value=v, key_pages=c.kp, value_pages=c.vp, page_table=c.table, lengths=c.lengths)
        args.update(bad)
        with pytest.raises(AssertionError):
            moa_b200.paged_append(**args)
    with pytest.raises(moa_b200.MoaError, match="power of two"):     # an error of the C entry point comes through it
        moa_b200.paged_append(k, v, c.kp[:, :, :24], c.vp[:, :, :24], c.table, c.lengths)
    before["append"] += 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moa_b200.paged_decode(one[0], *c.pool(), 0.1)
    assert counted["decode"] == before["decode"] and counted["append"] == before["append"]
    with torch.no_grad():
        moa_b200.paged_decode(one[0].detach().requires_grad_(), *c.pool(), 0.1)
    assert counted["decode"] == before["decode"] + 1
    monkeypatch.setattr(paged, "_host", None)
    for a, b in zip(compiled, results()):
        assert len(a) == len(b) and all(x.shape == y.shape and x.stride() == y.stride() and torch.equal(
            x.view(torch.int16) if x.dtype == BF16 else x, y.view(torch.int16) if y.dtype == BF16 else y) for x, y in zip(a, b))
