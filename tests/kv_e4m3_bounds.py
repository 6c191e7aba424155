"""Attention over a cache kept in 8 bits against float64 with a bound of its own for every sequence: that of the kernel that takes it, and
relative to what the row itself looks at."""
import math
import os

import torch

from kv_e4m3_util import F64, scale_values, two_to
from rllm_b200.kernels import ops

BF16, F32 = torch.bfloat16, torch.float32


def forms_of(st, window, scale, num_decode, forced):
    """The kernel that takes each sequence: the launches' own sharing out (native/csrc/launch.cc, e4m3_attention), for tensors on 16 bytes."""
    S, g = len(st.lens), st.nq // st.nkv
    most, max_q = max(st.totals), max(st.lens)
    keys = min(window + max_q, most) if window else most
    few = max_q * g
    together = forced is None and 0 < num_decode <= S - num_decode and (few <= 16 or (few <= 32 and S * st.nkv <= 148))
    if together:
        num_decode = 0
    forms = []
    for i, (first, end, longest) in enumerate(((0, num_decode, 1), (num_decode, S, max_q))):
        if first < end:
            form = forced[i] if forced else ops.attention_e4m3_form(st.dtype, st.nq, st.nkv, st.d, st.page, scale, longest, end - first, keys)
            forms += [form] * (end - first)
    return forms


def expected(st, window=0, scale=None, num_decode=None, forced=None):
    """(result, bound) float64 [T, nq d].

    s: scores in units of the natural logarithm, p = e^(s - max s), l = sum p >= 1, w = p / l, P_j = p_j 2^ev_j, n visible keys.
    Scores.  Products and sums in float32: (d + 4) 2^-24 of the products' absolute sum.  Queries: two halves of float32 22 bits (2^-22);
    halves and e4m3 terms end at a fraction of the row's largest number, 2^-38 ("rows", "tcgen05") or 2^-22 ("columns"), of which a
    key's absolute sum is taken.  "columns": sums of e4m3 products are off by 2^-21 of their absolute sum.
    Exponentials: the argument's rounding, |s| log2(e) 2^-23 (two roundings), and the exponential's own 2^-22, for p and for the weight
    with its value's power each, whose argument is of up to 2^8 more: 2 (|s| + 2^8) 2^-24.
    Weights.  Rounded to a half (2^-11), two halves (float32, 2^-22), bfloat16 with exponentials partly a polynomial's ("dense", 2^-8
    and 4e-5).  Where the steps end: "rows" 2^-25 over 2^11 of a power of two that is less than twice the row's largest P_j (2^-35),
    "columns" 2^-24 over 2^2 of it (2^-26); "tcgen05" as "rows" (2^-35) for the weight.
    There the error is n 448 times that of max P_j, over l.
    "simt", "dense": none.
    Sums over the keys: n 2^-24.  The result: rounded once to its type."""
    scale = st.d ** -0.5 if scale is None else scale
    num_decode = st.num_decode if num_decode is None else num_decode
    forms = forms_of(st, window, scale, num_decode, forced)
    outs, bounds, at, g = [], [], 0, st.nq // st.nkv
    for s, (n, form) in enumerate(zip(st.lens, forms)):
        k, held = st.rows_of(s, st.k, st.ks)
        v, _ = st.rows_of(s, st.v, st.vs)
        pages = st.table[s, :-(-st.totals[s] // st.page)].long().clamp(0, st.pages - 1)
        power = scale_values(st.vs[pages]).transpose(0, 1).reshape(st.nkv, -1)[:, :st.totals[s]]
        kpower = scale_values(st.ks[pages]).transpose(0, 1).reshape(st.nkv, -1)[:, :st.totals[s]]
        q = st.q[at:at + n].to(F64).view(n, st.nq, st.d)
        at += n
        pos = torch.arange(st.totals[s] - n, st.totals[s], device=q.device)[:, None]
        key = torch.arange(st.totals[s], device=q.device)[None]
        seen = (key <= pos) & held[None]
        if window:
            seen = seen & (key > pos - window)
        res, bnd = torch.empty_like(q), torch.empty_like(q)
        many = seen.sum(-1, keepdim=True)
        f32 = st.dtype is F32
        half = {"dense": 2.0 ** -8 + 4e-5, "simt": 0.0}.get(form, 2.0 ** -22 if f32 else 2.0 ** -11)
        step = {"dense": 0.0, "simt": 0.0, "columns": 2.0 ** -26}.get(form, 2.0 ** -35)
        for h in range(st.nq):
            qq, kk, vv = q[:, h], k[h // g], v[h // g]
            bad = (seen & (torch.isnan(kk).any(-1) | torch.isnan(vv).any(-1))[None]).any(-1)
            kk, vv, pw = torch.nan_to_num(kk), torch.nan_to_num(vv), torch.nan_to_num(power[h // g])
            sc = ((qq @ kk.T) * scale).masked_fill(~seen, -math.inf)
            top = sc.amax(-1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(sc - top)
            l = p.sum(-1, keepdim=True).clamp(min=1.0)
            w = p / l
            out = w @ vv
            products = (qq.abs() @ kk.abs().T) * abs(scale)
            largest = qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1)[None] * abs(scale)
            off = products * ((st.d + 4) * 2.0 ** -24 + (2.0 ** -22 if f32 and form == "rows" else 0.0) + (2.0 ** -21 if form == "columns" else 0.0))
            if form in ("rows", "tcgen05", "columns"):
                off = off + largest * (2.0 ** -22 if form == "columns" else 2.0 ** -38)
            off = off.masked_fill(~seen, 0).amax(-1, keepdim=True)
            size = sc.masked_fill(~seen, 0).abs().amax(-1, keepdim=True) * 1.4427
            rel = 2 * (off + size * 2.0 ** -23) + 2 * (2.0 ** -22 + (size + 256) * 2.0 ** -24) + half + many * 2.0 ** -24
            rel = rel + (2.0 ** -21 if form == "columns" else 0.0)
            floor = many * 448 * step * (p * pw[None]).amax(-1, keepdim=True) / l
            out[bad] = math.nan
            res[:, h] = out
            bnd[:, h] = rel * (w @ vv.abs()) + floor + torch.finfo(st.dtype).eps / 2 * out.abs() + torch.finfo(st.dtype).tiny
        outs.append(res.view(n, -1))
        bounds.append(bnd.view(n, -1))
    return torch.cat(outs), torch.cat(bounds)


def check(st, out, window=0, scale=None, num_decode=None, forced=None):
    want, bound = expected(st, window, scale, num_decode, forced)
    got = out[:want.shape[0]].to(F64)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN where none belongs, or none where one does"
    fine = ~torch.isnan(want)
    off = ((got - want).abs() / bound)[fine]
    if os.environ.get("RLLM_TEST_SHOW"):
        print(f"  {float(off.max()):.3f} of the bound, off by {float(((got - want)[fine]).norm() / want[fine].norm()):.2e}")
    assert off.numel() == 0 or float(off.max()) <= 1.0, f"{float(off.max()):.2f} times the bound"
