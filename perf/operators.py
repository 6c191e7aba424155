"""The quantised cache's operators as cases that can be timed and compared: keys and values kept in 8 bits.

A cache page holds its rows as float8 e4m3 numbers, and one power of two (e8m0) a row beside them: a token's key (or
value) of one kv head is the row of numbers times that power.  Kinds of cases:

write   rotation of a step's queries and keys, and its keys and values quantised into their pages
read    tokens' keys and values read back from the pages
attend  causal attention of a step's tokens (single decoded ones, a few drafted ones, portions of prompts) over the
        pages, the tokens' own keys and values among them

"lens": the tokens that every sequence of the step brings; "starts": how many it had in the cache before.
"""
import math

import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bfloat16": BF16, "float32": F32}
MOST = 448.0                       # the largest e4m3 number
own = False


def listed():
    return [
        # one decoded token: the launch is what counts
        dict(name="write_one_token", kind="write", nq=32, nkv=8, dim=64, page=16, lens="1", starts="2047", dtype="bfloat16"),
        # a step of prompts, one of them a later portion
        dict(name="write_prompts", kind="write", nq=32, nkv=8, dim=128, page=16, lens="4096,1531,700", starts="0,0,2048",
             dtype="bfloat16"),
        # the exact path
        dict(name="write_float32", kind="write", nq=16, nkv=4, dim=64, page=16, lens="301,45", starts="0,77", dtype="float32"),
        # what a request holds behind a short prompt
        dict(name="read_prompt", kind="read", nq=32, nkv=8, dim=64, page=16, lens="333", starts="0", dtype="bfloat16"),
        # long prefixes of eight requests
        dict(name="read_batch", kind="read", nq=32, nkv=8, dim=128, page=16,
             lens="16384,9001,12288,16000,4099,8192,15871,6007", starts="0,0,0,0,0,0,0,0", dtype="bfloat16"),
        # one request that decodes
        dict(name="attend_one_token", kind="attend", nq=32, nkv=8, dim=64, page=16, window=0, lens="1", starts="2047",
             dtype="bfloat16"),
        # eight that decode behind prompts of about 4,096 tokens
        dict(name="attend_decode_8", kind="attend", nq=24, nkv=8, dim=128, page=16, window=0, lens="1,1,1,1,1,1,1,1",
             starts="4096,4100,2047,4200,3061,4303,1048,2111", dtype="bfloat16"),
        # a full batch over long contexts
        dict(name="attend_decode_64", kind="attend", nq=32, nkv=8, dim=128, page=16, window=0, lens=",".join(["1"] * 64),
             starts=",".join(str(4000 + (i * 1237) % 8192) for i in range(64)), dtype="bfloat16"),
        # drafted tokens of eight requests
        dict(name="attend_drafts", kind="attend", nq=32, nkv=8, dim=64, page=16, window=0, lens="5,5,4,5,2,5,5,3",
             starts="8000,4100,6047,8200,7061,4303,8048,2111", dtype="bfloat16"),
        # a whole prompt
        dict(name="attend_prompt", kind="attend", nq=32, nkv=8, dim=64, page=16, window=0, lens="2048", starts="0",
             dtype="bfloat16"),
        # portions of long prompts, one of them short
        dict(name="attend_portions", kind="attend", nq=32, nkv=8, dim=128, page=32, window=0, lens="1024,57", starts="15360,12001",
             dtype="bfloat16"),
        # the exact path, under a window
        dict(name="attend_float32", kind="attend", nq=16, nkv=4, dim=64, page=16, window=512, lens="1,96", starts="1200,500",
             dtype="float32"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend"])
    nq, nkv = rng.choice([(32, 8), (24, 8), (16, 4), (8, 8), (16, 2), (32, 4)])
    case = dict(kind=kind, nq=nq, nkv=nkv, dim=rng.choice([64, 128]), page=rng.choice([16, 16, 32, 64]),
                dtype="float32" if rng.random() < 0.2 else "bfloat16")
    n = rng.choice([1, 1, 2, 3, 5, 8])
    if kind == "write":
        lens = [_log(rng, 1, max(1, 6144 // n)) for _ in range(n)]
        starts = [rng.choice([0, _log(rng, 1, 16384)]) for _ in lens]
    elif kind == "read":
        lens = [_log(rng, 1, 65536 // n) for _ in range(n)]
        starts = [0 for _ in lens]
    elif case["dtype"] == "float32":
        lens = [rng.choice([1, _log(rng, 1, 128)]) for _ in range(n)]
        starts = [_log(rng, 1, 2048) for _ in lens]
    else:
        how = rng.choice(["decode", "drafts", "portions"])
        if how == "decode":
            n = _log(rng, 1, 64)
            lens = [1] * n
            starts = [_log(rng, 16, min(32768, 262144 // n)) for _ in lens]
        elif how == "drafts":
            lens = [rng.randint(1, 8) for _ in range(n)]
            starts = [_log(rng, 16, 16384) for _ in lens]
        else:
            n = rng.choice([1, 1, 2, 3])
            lens = [_log(rng, 9, 1024 // n) for _ in range(n)]
            starts = [rng.choice([0, _log(rng, 1, 15360 // n)]) for _ in lens]
    if kind == "attend":
        case["window"] = 0 if rng.random() < 0.7 else _log(rng, 16, 4096)
        pairs = sorted(zip(lens, starts), key=lambda p: p[0] != 1)          # single tokens come first in a step
        lens, starts = [p[0] for p in pairs], [p[1] for p in pairs]
    case["lens"], case["starts"] = ",".join(map(str, lens)), ",".join(map(str, starts))
    return case


def _ints(text):
    return [int(x) for x in text.split(",")]


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _two_to(e):
    """2^e in float32 for whole e from -126 to 127, by its bits (a power function may be an ulp off)."""
    return ((e.to(torch.int32) + 127) << 23).view(F32)


def _quantise(x):
    """Rows (the last axis) of float32 numbers as e4m3 numbers and each row's power of two, the least with which no number
    passes the largest e4m3 one; as bytes."""
    top = x.abs().amax(-1)
    fraction, e = torch.frexp(top)                            # top = fraction 2^e, fraction from a half to 1
    e = torch.where(fraction > MOST / 512.0, e - 8, e - 9).clamp(min=-127)
    e = torch.where(top == 0, torch.full_like(e, -127), e)
    half = torch.div(-e, 2, rounding_mode="floor")
    scaled = x * _two_to(half).unsqueeze(-1) * _two_to(-e - half).unsqueeze(-1)
    return scaled.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _pages(g, pages, nkv, page, dim):
    """Pages that earlier steps left: rows whose sizes differ, a few channels larger than the rest (as keys have)."""
    dev = g.device
    codes = torch.empty((pages, nkv, page, dim), dtype=torch.uint8, device=dev)
    powers = torch.empty((pages, nkv, page), dtype=torch.uint8, device=dev)
    channel = torch.exp(torch.randn(nkv, 1, dim, device=dev, generator=g) * 0.5)
    step = max(1, (1 << 26) // (nkv * page * dim))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        rows = torch.exp(torch.randn(n, nkv, page, 1, device=dev, generator=g) * 0.3)
        codes[a:a + n], powers[a:a + n] = _quantise(torch.randn(n, nkv, page, dim, device=dev, generator=g) * rows * channel)
    return codes.view(torch.float8_e4m3fn), powers.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 7919 + 17)
    lens, starts = _ints(case["lens"]), _ints(case["starts"])
    nq, nkv, dim, page, dtype = case["nq"], case["nkv"], case["dim"], case["page"], DTYPES[case["dtype"]]
    S, T, totals = len(lens), sum(lens), [a + b for a, b in zip(lens, starts)]
    need = [-(-n // page) for n in totals]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=dev, generator=g).int()
    table = torch.full((S, max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    st = dict(case=case, nq=nq, nkv=nkv, dim=dim, table=table, lens=lens, totals=totals)
    st["k"], st["ks"] = _pages(g, pages, nkv, page, dim)
    st["v"], st["vs"] = _pages(g, pages, nkv, page, dim)
    i32 = dict(dtype=torch.int32, device=dev)
    st["positions"] = torch.cat([torch.arange(a, a + n, **i32) for a, n in zip(starts, lens)])
    st["token_seq"] = torch.repeat_interleave(torch.arange(S, **i32), torch.tensor(lens, device=dev))
    st["q_start"] = torch.tensor([sum(lens[:i]) for i in range(S + 1)], **i32)
    st["seq_lens"] = torch.tensor(totals, **i32)
    st["err"] = torch.zeros(1, **i32)
    st["dtype"] = dtype
    if case["kind"] == "write":
        st["inv_freq"] = 500000.0 ** (-torch.arange(dim // 2, dtype=F64, device=dev) * 2 / dim)
        st["qkv"] = torch.randn(T, (nq + 2 * nkv) * dim, device=dev, generator=g).to(dtype)
    elif case["kind"] == "attend":
        st["q"] = torch.randn(T, nq * dim, device=dev, generator=g).to(dtype)
        st["num_decode"] = sum(1 for n in lens if n == 1)
        st["scale"] = 1.0 / math.sqrt(dim)
        st["rows_at"] = torch.arange(T, device=dev) - st["q_start"].long()[st["token_seq"].long()]
    return st


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"write": _own_write, "read": _own_read, "attend": _own_attend}[kind](st)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[kind](st)


def _own_write(st):
    from rllm_b200.kernels import ops
    q = torch.empty_like(st["qkv"][:, :st["nq"] * st["dim"]], memory_format=torch.contiguous_format)
    ops.rope_kv_write_e4m3(st["qkv"], st["positions"], st["token_seq"], st["inv_freq"], st["dim"], st["table"], st["k"], st["v"],
                           st["ks"], st["vs"], st["nq"], st["nkv"], st["dim"], st["err"], q_out=q)
    return {"q": q, "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _own_read(st):
    from rllm_b200.kernels import ops
    shape = (st["positions"].numel(), st["nkv"] * st["dim"])
    k = torch.empty(shape, dtype=st["dtype"], device=st["k"].device)
    v = torch.empty(shape, dtype=st["dtype"], device=st["k"].device)
    ops.kv_read_e4m3(st["positions"], st["token_seq"], st["table"], st["k"], st["v"], st["ks"], st["vs"], k, v, st["err"])
    return {"k": k, "v": v}


def _own_attend(st):
    from rllm_b200.kernels import ops
    out = torch.empty_like(st["q"])
    ops.attention_e4m3(st["q"], out, st["k"], st["v"], st["ks"], st["vs"], st["table"], st["q_start"], st["seq_lens"],
                       st["num_decode"], max(st["lens"]), max(st["totals"]), st["nq"], st["nkv"], st["case"]["window"],
                       st["scale"], st["err"])
    return {"out": out}


def _values(codes, powers):
    """Float32 numbers of bytes and of their rows' powers."""
    return codes.float() * powers.float().unsqueeze(-1)


def _plain_write(st):
    nq, nkv, d, T = st["nq"], st["nkv"], st["dim"], st["positions"].numel()
    x = st["qkv"].float().view(T, nq + 2 * nkv, d)
    angle = st["positions"].to(F64).unsqueeze(1) * st["inv_freq"]
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    a, b = x[:, :nq + nkv, :d // 2], x[:, :nq + nkv, d // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    q = turned[:, :nq].to(st["dtype"]).reshape(T, nq * d)
    size = st["k"].shape[2]
    pos = st["positions"].long()
    page, slot = st["table"][st["token_seq"].long(), pos // size].long(), pos % size
    for name, rows in (("k", turned[:, nq:]), ("v", x[:, nq + nkv:])):
        codes, powers = _quantise(rows.contiguous())
        st[name].view(torch.uint8)[page, :, slot] = codes
        st[name + "s"].view(torch.uint8)[page, :, slot] = powers
    return {"q": q, "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _plain_read(st):
    size, pos = st["k"].shape[2], st["positions"].long()
    page, slot = st["table"][st["token_seq"].long(), pos // size].long(), pos % size
    return {n: _values(st[n].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn),
                       st[n + "s"].view(torch.uint8)[page, :, slot].view(torch.float8_e8m0fnu)).to(st["dtype"])
            .view(pos.numel(), -1) for n in ("k", "v")}


def _plain_attend(st):
    nq, nkv, d, window = st["nq"], st["nkv"], st["dim"], st["case"]["window"]
    S, Q, C, size = len(st["lens"]), max(st["lens"]), max(st["totals"]), st["k"].shape[2]
    seq, row = st["token_seq"].long(), st["rows_at"]
    pages = st["table"].long().clamp(min=0)
    k, v = (_values(st[n].view(torch.uint8)[pages].view(torch.float8_e4m3fn), st[n + "s"].view(torch.uint8)[pages].view(torch.float8_e8m0fnu))
            .transpose(1, 2).reshape(S, nkv, -1, d)[:, :, :C] for n in ("k", "v"))
    q = torch.zeros((S, Q, nq, d), dtype=F32, device=k.device)
    q[seq, row] = st["q"].float().view(-1, nq, d)
    q = q.view(S, Q, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(S, nkv, -1, d)
    scores = (q @ k.transpose(-1, -2)).view(S, nkv, nq // nkv, Q, C) * st["scale"]
    key = torch.arange(C, device=k.device)
    first = (st["seq_lens"] - (st["q_start"][1:] - st["q_start"][:-1])).long()
    at = first.view(S, 1, 1) + torch.arange(Q, device=k.device).view(1, Q, 1)
    seen = (key <= at) & (key < st["seq_lens"].view(S, 1, 1))
    if window:
        seen = seen & (key > at - window)
    seen = seen.view(S, 1, 1, Q, C)
    scores = scores.masked_fill(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = (p.view(S, nkv, -1, C) @ v).view(S, nkv, nq // nkv, Q, d) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(S, Q, nq * d)
    return {"out": out[seq, row].to(st["dtype"])}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    lens, starts = _ints(case["lens"]), _ints(case["starts"])
    nq, nkv, d, T = case["nq"], case["nkv"], case["dim"], sum(lens)
    size = DTYPES[case["dtype"]].itemsize
    row = nkv * 2 * (d + 1)                                   # a token's bytes in the cache
    if case["kind"] == "write":
        return {"bytes": T * ((2 * nq + 2 * nkv) * d * size + row), "flops": T * (nq + nkv) * d * 3}
    if case["kind"] == "read":
        return {"bytes": T * (row + 2 * nkv * d * size), "flops": T * 2 * nkv * d}
    window = case["window"] or (1 << 60)
    pairs = keys = 0
    for n, a in zip(lens, starts):
        pairs += sum(min(p + 1, window) for p in range(a, a + n))
        keys += a + n - max(0, a - window + 1)
    return {"bytes": T * 2 * nq * d * size + keys * row, "flops": 4 * pairs * nq * d}


def _e4m3(x):
    """The nearest e4m3 numbers of float64 ones (ties to even)."""
    _, e = torch.frexp(x)
    step = ((e.long() - 4).clamp(min=-9) + 1023 << 52).view(F64)
    return torch.round(x / step) * step                        # torch.round: halves to even


def _rows64(rows):
    top = rows.abs().amax(-1, keepdim=True)
    power = (torch.ceil(torch.log2(top.clamp(min=1e-300) / MOST)).clamp(min=-127).long() + 1023 << 52).view(F64)
    power = torch.where(power * MOST < top, power * 2, power)  # (the logarithm's rounding)
    power = torch.where(power * (MOST / 2) >= top, (power / 2).clamp(min=2.0 ** -127), power)
    return _e4m3(rows / power), power.squeeze(-1)


def exact(case, seed):
    st = prepare(case, seed)
    nq, nkv, d, size = st["nq"], st["nkv"], st["dim"], st["k"].shape[2]
    lens, totals, table = st["lens"], st["totals"], st["table"].cpu()
    k, v = st["k"].to(F64), st["v"].to(F64)
    ks, vs = st["ks"].to(F64), st["vs"].to(F64)
    begin = [sum(lens[:i]) for i in range(len(lens))]
    if case["kind"] == "write":
        qs = []
        for s, n in enumerate(lens):
            x = st["qkv"][begin[s]:begin[s] + n].to(F64).view(n, -1, d)
            pos = torch.arange(totals[s] - n, totals[s], dtype=F64, device=x.device)
            turn = torch.polar(torch.ones_like(pos)[:, None] * torch.ones_like(st["inv_freq"]), pos[:, None] * st["inv_freq"])
            z = torch.complex(x[:, :nq + nkv, :d // 2], x[:, :nq + nkv, d // 2:]) * turn[:, None]
            z = torch.cat([z.real, z.imag], -1)
            qs.append(z[:, :nq].reshape(n, nq * d))
            for (codes, powers), rows in (((k, ks), z[:, nq:]), ((v, vs), x[:, nq + nkv:])):
                c, p = _rows64(rows)
                for j in range(0, totals[s], size):
                    a, b = max(j, totals[s] - n), min(j + size, totals[s])
                    if a < b:
                        there = int(table[s, j // size])
                        codes[there, :, a - j:b - j] = c[a - totals[s] + n:b - totals[s] + n].transpose(0, 1)
                        powers[there, :, a - j:b - j] = p[a - totals[s] + n:b - totals[s] + n].transpose(0, 1)
        return {"q": torch.cat(qs), "k": k, "v": v, "ks": ks, "vs": vs}
    outs, keys, values = [], [], []
    for s, n in enumerate(lens):
        at = st["table"][s, :-(-totals[s] // size)].long()
        ke = (k[at] * ks[at][..., None]).transpose(0, 1).reshape(nkv, -1, d)[:, :totals[s]]
        ve = (v[at] * vs[at][..., None]).transpose(0, 1).reshape(nkv, -1, d)[:, :totals[s]]
        if case["kind"] == "read":
            keys.append(ke.transpose(0, 1).reshape(-1, nkv * d))
            values.append(ve.transpose(0, 1).reshape(-1, nkv * d))
            continue
        q = st["q"][begin[s]:begin[s] + n].to(F64).view(n, nq, d)
        out = torch.empty((n, nq, d), dtype=F64, device=q.device)
        pos = torch.arange(totals[s] - n, totals[s], device=q.device)[:, None]
        key = torch.arange(totals[s], device=q.device)[None]
        hidden = (key > pos) | ((pos - key >= case["window"]) if case["window"] else torch.zeros_like(key > pos))
        for h in range(nq):
            kv = h // (nq // nkv)
            scores = (q[:, h] @ ke[kv].T) * st["scale"]
            out[:, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ ve[kv]
        outs.append(out.view(n, nq * d))
    if case["kind"] == "read":
        return {"k": torch.cat(keys), "v": torch.cat(values)}
    return {"out": torch.cat(outs)}
