"""A cache kept in 8 bits, in float64: what a row becomes, what it reads back as, and the attention over it; with the inputs
and the bounds that the tests of the kernels share."""
import math

import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
F64 = torch.float64


def two_to(e):
    """2^e in float64 by its bits (a power function may be an ulp off)."""
    return ((e.long() + 1023) << 52).view(F64)


def power_of(top):
    """The exponent e of float64 magnitudes: the least whole e >= -127 with top <= 448 * 2^e."""
    m, e = torch.frexp(top.to(F64))                      # top = m 2^e, m in [1/2, 1); 448 = (7/8) 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(top == 0, torch.full_like(e, -127), e.clamp(min=-127))


def to_e4m3(x):
    """The e4m3 number nearest to each float64 number of at most 448, ties to even."""
    _, e = torch.frexp(x)
    step = two_to((e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def quantise(x):
    """(numbers float64, scale bytes) of rows [..., d]; a row with a number that is not finite: zeros and 255."""
    x = x.to(F64)
    fine = torch.isfinite(x).all(-1)
    e = power_of(torch.where(fine, x.abs().amax(-1), torch.zeros(x.shape[:-1], dtype=F64, device=x.device)))
    c = to_e4m3(torch.where(fine[..., None], x, torch.zeros_like(x)) / two_to(e)[..., None])
    return c, torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def values(codes, scale):
    """float64 values of a cache's tensors."""
    return codes.to(torch.float32).to(F64) * scale_values(scale)[..., None]


def scale_values(scale):
    b = scale.view(torch.uint8).to(torch.int32)
    p = two_to(b - 127)
    return torch.where(b == 255, torch.full_like(p, math.nan), p)


class Step:
    """A step of sequences that bring ``lens`` tokens behind ``starts`` cached ones, and the cache, filled with random rows."""

    def __init__(self, lens, starts, nq, nkv, d, page, dtype, seed=0, device="cuda", spread=1.0, qscale=1.0, more_rows=0, stride_pad=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.totals = list(lens), [a + b for a, b in zip(lens, starts)]
        self.nq, self.nkv, self.d, self.page, self.dtype, self.device = nq, nkv, d, page, dtype, device
        S, T = len(lens), sum(lens)
        need = [max(1, -(-n // page)) for n in self.totals]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.full((S, max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n].int()
            at += n
        rows = torch.randn(2, self.pages, nkv, page, d, generator=g) * torch.exp(spread * torch.randn(2, self.pages, nkv, page, 1, generator=g))
        codes, byte = quantise(rows)
        self.k, self.v = (codes[i].float().to(E4M3).to(device) for i in range(2))
        self.ks, self.vs = (byte[i].to(device).view(E8M0) for i in range(2))
        self.table = self.table.to(device)
        i32 = dict(dtype=torch.int32, device=device)
        self.q_start = torch.tensor([sum(lens[:i]) for i in range(S + 1)], **i32)
        self.seq_lens = torch.tensor(self.totals, **i32)
        self.positions = torch.tensor([p for n, a in zip(lens, starts) for p in range(a, a + n)], **i32)
        self.token_seq = torch.tensor([s for s, n in enumerate(lens) for _ in range(n)], **i32)
        wide = torch.randn(T + more_rows, nq * d + stride_pad, generator=g).mul_(qscale).to(dtype).to(device)
        self.q = wide[:, :nq * d]
        self.err = torch.zeros(1, **i32)
        self.num_decode = next((i for i, n in enumerate(lens) if n != 1), S)

    def attend(self, ops, window=0, scale=None, out=None, **over):
        out = torch.full((self.q.shape[0], self.nq * self.d), 7.0, dtype=self.dtype, device=self.device) if out is None else out
        a = dict(num_decode=self.num_decode, max_q_len=max(self.lens), max_seq_len=max(self.totals))
        a.update(over)
        ops.attention_e4m3(self.q, out, self.k, self.v, self.ks, self.vs, self.table, self.q_start, self.seq_lens,
                           a["num_decode"], a["max_q_len"], a["max_seq_len"], self.nq, self.nkv, window,
                           self.d ** -0.5 if scale is None else scale, self.err)
        return out

    def rows_of(self, s, codes, scale):
        """float64 [nkv, keys, d] of sequence s; NaN rows where the scale says so."""
        n = self.totals[s]
        at = self.table[s, :-(-n // self.page)].long()
        held = (at >= 0) & (at < self.pages)
        at = at.clamp(0, self.pages - 1)
        x = values(codes[at], scale[at]).transpose(0, 1).reshape(self.nkv, -1, self.d)[:, :n]
        return x, held.repeat_interleave(self.page)[:n]

    def expected(self, window=0, scale=None, prompts=False, columns=False):
        """(result, bound of the error) float64 [T, nq d].

        The bound, from the kernels' arithmetic.  A score's sum of d products in float32 is off by at most (d + 4) 2^-24 of
        the products' absolute sum (the last 4: scale and power factors), q itself being exact as one or two halves or off by
        2^-22; a weight p is off by that, by 2^-21 (the exponential and its argument, of up to 2^5 in the log2 domain times
        2^-24, counted with 2^-17) and by the rounding of p to a half (2^-11), or to two of them (2^-22); the sums over the keys
        add n 2^-24; the result is rounded once to its type.  A half's step does not fall below 2^-24, so a weight, held as
        p 2^ev 2^7 over a power of two that is at most the largest 2^ev in sight, is off by 2^-32 of that at least: over n keys
        with numbers of at most 448, n 448 2^-32 max 2^ev, p being 1 at the row's reference and the weights' sum 1 at least.

        ``columns``: there a weight is p 2^ev over a reference that is at most the row's largest p 2^ev, times 2^2; a half is off by
        2^-25 at least, and the last of the four terms it is taken apart into, of a step of 2^-9 over 2^15, by as much: by 2^-24 over
        2^2 of the row's largest p 2^ev together, n 448 2^-26 max p 2^ev over n keys.  (Its products' sums are off by 2^-21 of the
        absolute sum, which the score's (d + 4) 2^-24 and the weights' 2^-17 cover.)"""
        scale = self.d ** -0.5 if scale is None else scale
        # prompts on tcgen05: the weights are bfloat16 (2^-8), some exponentials a polynomial's (4e-5)
        half = 2.0 ** -8 + 4e-5 if prompts else 2.0 ** -11 if self.dtype is torch.bfloat16 else 2.0 ** -22
        outs, bounds = [], []
        at = 0
        for s, n in enumerate(self.lens):
            k, held = self.rows_of(s, self.k, self.ks)
            v, _ = self.rows_of(s, self.v, self.vs)
            q = self.q[at:at + n].to(F64).view(n, self.nq, self.d)
            at += n
            pos = torch.arange(self.totals[s] - n, self.totals[s], device=q.device)[:, None]
            key = torch.arange(self.totals[s], device=q.device)[None]
            seen = (key <= pos) & held[None]
            if window:
                seen = seen & (key > pos - window)
            g = self.nq // self.nkv
            for h in range(self.nq):
                kk, vv = k[h // g], v[h // g]
                sc = torch.where(seen, (q[:, h] @ kk.T) * scale, torch.full((1, 1), -math.inf, dtype=F64, device=q.device))
                top = sc.amax(-1, keepdim=True)
                p = torch.where(seen, torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(sc))
                l = p.sum(-1, keepdim=True)
                bad = (seen & torch.isnan(kk).any(-1)[None]).any(-1) | (seen & torch.isnan(vv).any(-1)[None]).any(-1)
                vz = torch.nan_to_num(vv)
                p = torch.nan_to_num(p)
                w = torch.where(l > 0, p / l.clamp(min=1e-300), torch.zeros_like(p))
                out = w @ vz
                out[bad] = math.nan
                off = ((q[:, h].abs() @ torch.nan_to_num(kk).abs().T) * abs(scale) * (self.d + 4) * 2.0 ** -24).masked_fill(~seen, 0).amax(-1, keepdim=True)
                # scores above 32 in the log2 domain lose more in the exponent's argument
                arg = torch.nan_to_num(sc.masked_fill(~seen, 0).abs()).amax(-1, keepdim=True) * 1.4427 * 2.0 ** -23
                rel = 2 * (off + arg) + 2.0 ** -17 * (1.0 if self.dtype is torch.bfloat16 else 2.0 ** -4) + half + key.numel() * 2.0 ** -24
                outs.append(out)
                power = torch.where(seen.any(0)[:, None], vz.abs(), torch.zeros_like(vz)).amax() / 224        # 2^ev <= max|v| / 224
                floor = key.numel() * 448 * 2.0 ** -32 * power
                if columns:
                    floor = floor + key.numel() * 448 * 2.0 ** -26 * (p * (vz.abs().amax(-1) / 224)[None]).amax(-1, keepdim=True)
                bounds.append(rel * (w @ vz.abs()) + floor + torch.finfo(self.dtype).eps / 2 * out.abs() + 1e-30)
        T = sum(self.lens)
        place = []
        i = 0
        res = torch.empty((T, self.nq, self.d), dtype=F64, device=self.device)
        bnd = torch.empty_like(res)
        at = 0
        for n in self.lens:
            for h in range(self.nq):
                res[at:at + n, h], bnd[at:at + n, h] = outs[i], bounds[i]
                i += 1
            at += n
        return res.view(T, -1), bnd.view(T, -1)

    def check(self, out, window=0, scale=None):
        from rllm_b200.kernels import ops
        forms = ops.E4M3_FORMS or (ops.attention_e4m3_form(
            self.dtype, self.nq, self.nkv, self.d, self.page, 1.0, max(self.lens), len(self.lens) - self.num_decode, max(self.totals)),)
        want, bound = self.expected(window, scale, "dense" in forms, "columns" in forms)
        got = out[:want.shape[0]].to(F64)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN where none belongs, or none where one does"
        fine = ~torch.isnan(want)
        off = ((got - want).abs() / bound)[fine]
        assert off.numel() == 0 or float(off.max()) <= 1.0, f"{float(off.max()):.2f} times the bound"
