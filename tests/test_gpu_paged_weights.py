"""Attention weights of the paged cache that are small beside the largest, and values that are infinite, against 64 bits.

Tolerance for one token with a score `gap` above all others, whose value is zero, so that nothing but the small weights
makes the result.  u = 2^-23 bounds one fp32 operation.  Scores are products of single coordinates and exact; turned into
an exponent of two they pass through a constant and a product (half a step of 1.45 gap each), and the differences to the
reference through two subtractions of up to 1.45 gap + 15: off by (2 * 1.45 gap + 15) u at most, and the weights by that
times ln 2, and 4 u of the exponential itself.  A weight is held in 16-bit parts: fp16 to 2^-22 of itself and to 2^-39 of
the largest, bf16 to 2^-17 of itself.  All terms are positive, and a sum runs over the units of 16 tokens that one warp
takes, the 16 of them, and the warps' and parts' results: depth (units + 80).  Weights and sums count twice, in numerator
and denominator; what is left of 2^-39 of the largest weight is a share of the values."""
import math

import pytest
import torch

import moa_b200
from test_gpu_paged import BF16, F16, U, Case, _half_step, _tiny, tables

pytestmark = pytest.mark.gpu


def _filled(n, H, KV, D, B, dtype, page, width, keys):
    """Sequences of n tokens with zero keys but for `keys(kp, pages, slots)`, and values in [0.5, 1.5)."""
    c = Case([0] * B, H, KV, D, page, dtype, room=n + 1, width=width, seed=3)
    pages, slots = c.table[:, torch.arange(n, device="cuda") // page].long(), torch.arange(n, device="cuda") % page
    slots = slots.expand(B, -1)
    c.kp[pages, :, slots] = torch.zeros((), dtype=dtype, device="cuda")
    c.vp[pages, :, slots] = (torch.rand(B, n, KV, D, generator=c.gen) + 0.5).to(dtype).cuda()
    c.lengths.fill_(n)
    c.values = c.vp[pages, :, slots]                      # (B, n, KV, D), a copy
    keys(c, pages, slots)
    return c


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 8), (64, 12), (128, 16)])
@pytest.mark.parametrize("form", ["blocks", "warps"])
@pytest.mark.parametrize("gap", [10.0, 17.0, 17.5, 20.0])
@pytest.mark.parametrize("call", ["attend", "step", "turned", "new token"])
def test_many_small_weights_beside_a_large_one(dtype, D, G, form, gap, call):
    B, KV, page = 150, 2, 16
    n, width = (1000, 80) if form == "blocks" else (250, 16)
    H, at = G * KV, 5

    def sink(c, pages, slots):
        if call != "new token":
            c.kp[pages[:, at], :, slots[:, at], 0] = 1.0
            c.vp[pages[:, at], :, slots[:, at]] = 0.0
            c.values[:, at] = 0.0

    c = _filled(n, H, KV, D, B, dtype, page, width, sink)
    assert c.B * KV > 296 and (c.table.shape[1] * page <= 256) == (form == "warps")
    q = torch.zeros(B, H, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = gap
    scores = torch.zeros(n, dtype=torch.float64, device="cuda")
    values, args = c.values.double(), {}
    if call != "new token":
        scores[at] = gap
    if call != "attend":
        k, v = torch.zeros(B, KV, 1, D, dtype=dtype, device="cuda"), c.values[:, 7].unsqueeze(2).clone()
        if call == "new token":
            k[..., 0] = 1.0
            v.zero_()
        args = dict(key=k, value=v)
        if call == "turned":                              # by an angle of zero
            args["rope"] = tuple(t[:1].expand(n + 1, -1).contiguous() for t in tables(D, torch.zeros(1), torch.float32))
        scores = torch.cat([scores, scores.new_full((1,), gap if call == "new token" else 0.0)])
        values = torch.cat([values, v.transpose(1, 2).double()], 1)
    p = torch.softmax(scores, 0)
    ref = torch.einsum("n,bnkd->bkd", p, values).repeat_interleave(G, 1)[:, None]
    units = math.ceil(len(p) / 16)
    weight = 2.0 ** -22 if dtype == F16 else 2.0 ** -17
    rel = 2 * (math.log(2) * (2.9 * gap + 15) * U + 4 * U + weight + (units + 80) * U)
    tol = rel * ref + (2.0 ** -39 * p.max() * values.abs().sum(1).repeat_interleave(G, 1)[:, None] if dtype == F16 else 0.0)
    for out_dtype in (torch.float32, dtype):
        out = moa_b200.paged_decode(q, *c.pool(), 1.0, out_dtype=out_dtype, **args)
        off = (out.double() - ref).abs() / (tol + _half_step(out_dtype) * ref * (1 + 2 ** -8) + _tiny(out_dtype))
        assert off.max().item() <= 1.0, (out_dtype, off.max().item(), (out.double() / ref).min().item())
    moa_b200.check_device_status()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form", ["blocks", "warps"])
@pytest.mark.parametrize("G", [1, 12])
@pytest.mark.parametrize("step", [False, True])
def test_scores_so_large_that_fp32_has_no_fractions(dtype, form, G, step):
    """Scores of 2^10 .. 2^39 times 0, 1/2 and 1 (differences of hundreds and more): the largest takes all the weight."""
    B, KV, D, page = 150, 2, 64, 16
    n, width = (600, 48) if form == "blocks" else (250, 16)

    def keys(c, pages, slots):
        c.kp[pages, :, slots, 0] = 0.5
        c.kp[pages[:, 100], :, slots[:, 100], 0] = 1.0
        c.kp[pages[:, 101], :, slots[:, 101], 0] = 0.0

    c = _filled(n, G * KV, KV, D, B, dtype, page, width, keys)
    q = torch.zeros(B, G * KV, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 2.0
    k, v = torch.zeros(B, KV, 1, D, dtype=dtype, device="cuda"), torch.ones(B, KV, 1, D, dtype=dtype, device="cuda")
    want = c.values[:, 100].double().repeat_interleave(G, 1)[:, None]
    for power in (10, 15, 23, 24, 25, 27, 33, 39):        # half the score is 2^9 at least: nothing is left of the others
        out = moa_b200.paged_decode(q, *c.pool(), 2.0 ** (power - 1), out_dtype=torch.float32, **(dict(key=k, value=v) if step else {}))
        off = ((out.double() - want).abs() / want).max().item()
        assert off <= 8 * U, (power, off)                 # one weight, a product with it, a division by it
    moa_b200.check_device_status()
