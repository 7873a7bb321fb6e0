"""Infinite values and keys in a paged cache: the result is what the formula gives for them, whatever the number of query
heads per key head, the type and the kernel's form.  Tolerances of the finite rest: those of test_gpu_paged."""
import pytest
import torch

import moa_b200
from test_gpu_paged import BF16, F16, Case, attention64, close, rotated64, tables

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,G", [(64, 1), (64, 9), (64, 16), (128, 8), (128, 12)])
@pytest.mark.parametrize("form", ["blocks", "warps"])
@pytest.mark.parametrize("call", ["attend", "step", "turned step", "step turned by nothing"])
def test_infinite_values_and_keys(dtype, D, G, form, call):
    B, KV, page = (150, 2, 16) if form == "warps" else (7, 2, 16)
    n, width = (200, 16) if form == "warps" else (611, 48)
    c = Case([n] * B, G * KV, KV, D, page, dtype, room=1, width=width)
    slow = D // 2 - 1                                     # a coordinate that rotation hardly turns
    at = lambda j: c.places(slice(None), torch.tensor(j))
    for j in range(0, n):
        pages, slots = at(j)
        c.kp[pages, :, slots] *= 0.1
    for j, score in ((20, -20.0), (40, -60.0)):           # weights of e^-20 and e^-60 of the largest, or so
        c.kp[at(j)[0], 0, at(j)[1], slow] = score
    for j, d, x in ((7, 5, INF), (90, 6, -INF), (7, 7, INF), (91, 7, -INF), (20, 9, INF), (40, 10, -INF), (15, 11, float("nan"))):
        c.vp[at(j)[0], 0, at(j)[1], d] = x
    c.kp[at(11)[0], 1, at(11)[1], slow] = -INF            # the second key head: score -inf, no weight
    q = c.normal(B, G * KV, 1, D) * 0.3
    q[..., slow] = 1.0 + 0.1 * c.normal(B, G * KV, 1).abs()
    args, qr, length = {}, q, c.lengths
    if call != "attend":
        k, v = c.normal(B, KV, 1, D) * 0.1, c.normal(B, KV, 1, D)
        v[:, 0, :, 12] = -INF
        args, length = dict(key=k, value=v), c.lengths + 1
        if call not in ("attend", "step"):                # (turned by nothing: queries have no part beyond 16 bits)
            args["rope"] = tables(D, torch.arange(n + 1) * (call == "turned step"), torch.float32)
            cos, sin = (t[n] for t in args["rope"])
            qr = rotated64(q, cos, sin)[0]
            assert qr[..., slow].min() > 0.5
    for out_dtype in (torch.float32, dtype):
        out = moa_b200.paged_decode(q, *c.pool(), 1.0, out_dtype=out_dtype, **args)
        ref, tol = attention64(c, qr, length, 1.0)
        ref1, tol1 = attention64(c, qr, length, 1.0, dropped={(b, 11) for b in range(B)})
        ref[:, :, G:], tol[:, :, G:] = ref1[:, :, G:], tol1[:, :, G:]
        finite = torch.isfinite(ref)
        special = {5: INF, 6: -INF, 7: None, 9: INF, 10: -INF, 11: None}
        if call != "attend":
            special[12] = -INF
        assert (~finite).sum() == len(special) * B * G
        for d, x in special.items():
            got = out[:, 0, :G, d]
            assert (torch.isnan(got) if x is None else got == x).all(), (d, x, got.flatten()[:4])
        close(out[finite], ref[finite], tol[finite])
    moa_b200.check_device_status()
