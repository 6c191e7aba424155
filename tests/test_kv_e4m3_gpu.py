"""A cache kept in 8 bits on the GPU: writing it, reading it back, attention over it, and the three in a row, against float64."""
import math

import pytest
import torch

from kv_e4m3_util import E4M3, E8M0, F64, Step, quantise, scale_values, values
from rllm_b200.kernels import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def freqs(rd):
    return 10000.0 ** (-torch.arange(rd // 2, dtype=F64, device="cuda") * 2 / max(rd, 1))


def fresh_cache(step, seed=3):
    """Pages with bytes of earlier use: whatever a write leaves alone has to stay."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    byte = lambda shape: torch.randint(0, 120, shape, dtype=torch.uint8, device="cuda", generator=g)  # noqa: E731
    return byte(step.k.shape).view(E4M3), byte(step.v.shape).view(E4M3), byte(step.ks.shape).view(E8M0), byte(step.vs.shape).view(E8M0)


def turned(x, pos, rd, inv):
    """float64 rotation of halves of the first rd dims."""
    if rd == 0:
        return x
    a = pos.to(F64)[:, None] * inv
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    h = rd // 2
    return torch.cat([x[..., :h] * c - x[..., h:rd] * s, x[..., h:rd] * c + x[..., :h] * s, x[..., rd:]], -1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,rd,page,lens,starts", [
    (4, 2, 64, 64, 16, [1], [0]), (32, 8, 64, 64, 16, [5, 1, 33], [0, 4095, 17]), (24, 8, 128, 128, 16, [300, 7], [2, 99991]),
    (3, 3, 48, 48, 4, [9, 2], [3, 30]), (4, 4, 16, 8, 7, [3, 20], [0, 6]), (8, 1, 256, 128, 32, [40], [31]),
    (5, 1, 80, 0, 1, [4, 4], [0, 2]), (16, 2, 128, 0, 64, [129], [63]), (8, 4, 96, 64, 8, [11], [5]), (2, 2, 32, 32, 16, [600], [0])])
def test_write(dtype, nq, nkv, d, rd, page, lens, starts):
    st = Step(lens, starts, nq, nkv, d, page, dtype, seed=d + rd)
    T = sum(lens)
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(T, nq + 2 * nkv, d, generator=g) * torch.exp(2 * torch.randn(T, nq + 2 * nkv, 1, generator=g))
    qkv[0, nq] = 0                                                       # a row of zeros
    if T > 1:
        qkv[1, nq + nkv] = 2.0 ** -140                                   # a row of numbers below the least scale (zeros in neither type)
        qkv[T - 1, nq + nkv, 1:] = 0
        qkv[T - 1, nq + nkv, 0] = 448.0 * 2.0 ** 100
    if T > 2:
        qkv[2, nq + nkv + nkv - 1, d // 2] = 3.0e38
    qkv = qkv.to(dtype).cuda()
    x = qkv.to(F64)
    cache = fresh_cache(st)
    old = [c.clone() for c in cache]
    inv = freqs(rd)
    before = qkv.clone()
    q = torch.full((T + 2, nq * d + 16), 5.0, dtype=dtype, device="cuda")
    ops.rope_kv_write_e4m3(qkv.view(T, -1), st.positions, st.token_seq, inv if rd else None, rd, st.table, *cache, nq, nkv, d, st.err,
                           q_out=q[:T, :nq * d])
    assert int(st.err) == 0 and torch.equal(qkv, before)
    assert (q[T:] == 5).all() and (q[:, nq * d:] == 5).all()
    want = turned(x[:, :nq + nkv], st.positions, rd, inv)
    # cosine and sine are off by 2^-21, two products and a sum by 3 2^-24 of what they are made of
    slack = 2.0 ** -20 * (turned(x[:, :nq + nkv].abs(), torch.zeros_like(st.positions), 0, inv) + torch.roll(x[:, :nq + nkv].abs(), rd // 2, -1)
                          + torch.roll(x[:, :nq + nkv].abs(), -(rd // 2), -1)) if rd else torch.zeros_like(want)
    got = q[:T, :nq * d].view(T, nq, d).to(F64)
    assert ((got - want[:, :nq]).abs() <= torch.finfo(dtype).eps / 2 * want[:, :nq].abs() + slack[:, :nq] * 1.01).all()
    # in place gives the same bits
    ops.rope_kv_write_e4m3(qkv.view(T, -1), st.positions, st.token_seq, inv if rd else None, rd, st.table, *[c.clone() for c in cache], nq,
                           nkv, d, st.err)
    assert torch.equal(qkv[:, :nq].reshape(T, -1), q[:T, :nq * d]) and torch.equal(qkv[:, nq:], before[:, nq:])
    pos = st.positions.long()
    at = (st.table[st.token_seq.long(), pos // page].long(), slice(None), pos % page)
    untouched = torch.ones(st.ks.shape, dtype=torch.bool, device="cuda")
    untouched[at[0], :, at[2]] = False
    for codes, scale, co, so, rows, sl, exact in ((cache[0], cache[2], old[0], old[2], want[:, nq:], slack[:, nq:], rd == 0),
                                                  (cache[1], cache[3], old[1], old[3], x[:, nq + nkv:], None, True)):
        assert torch.equal(codes.view(torch.uint8)[untouched], co.view(torch.uint8)[untouched])
        assert torch.equal(scale.view(torch.uint8)[untouched], so.view(torch.uint8)[untouched])
        c, b = quantise(rows)
        gc, gb = codes.view(torch.uint8)[at].view(E4M3).to(F64), scale.view(torch.uint8)[at]
        if exact:
            assert torch.equal(gb, b) and torch.equal(gc, c)
            continue
        # rotated rows: the nearest number of what float32 gave, so at most half a step (of the written scale) and the slack off;
        # and the scale is that of a largest magnitude within the slack
        power = scale_values(gb.view(E8M0))
        step = torch.maximum(2.0 ** -4 * (rows.abs() + sl * 1.01) / power[..., None], torch.tensor(2.0 ** -10, device="cuda", dtype=F64))
        assert ((gc - rows / power[..., None]).abs() <= step * 1.0001 + sl * 1.01 / power[..., None]).all()
        top = rows.abs().amax(-1)
        sl_top = sl.amax(-1) * 1.01
        assert (top - sl_top <= 448 * power).all() and ((top + sl_top > 224 * power) | (gb == 0)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_rows_with_numbers_that_are_not_finite(dtype, what):
    nq, nkv, d, page = 4, 2, 64, 16
    st = Step([3], [0], nq, nkv, d, page, dtype)
    qkv = torch.randn(3, (nq + 2 * nkv) * d).to(dtype).cuda()
    qkv[1, nq * d + 5] = what                      # the key of head 0
    qkv[2, (nq + nkv + 1) * d + 63] = what         # the value of head 1
    cache = fresh_cache(st)
    ops.rope_kv_write_e4m3(qkv, st.positions, st.token_seq, freqs(d), d, st.table, *cache, nq, nkv, d, st.err)
    there = int(st.table[0, 0])
    kb, vb = cache[2].view(torch.uint8)[there], cache[3].view(torch.uint8)[there]
    assert kb[0, 1] == 255 and vb[1, 2] == 255
    assert (kb[:, :3] == 255).sum() == 1 and (vb[:, :3] == 255).sum() == 1
    assert (cache[0].view(torch.uint8)[there, 0, 1] == 0).all() and (cache[1].view(torch.uint8)[there, 1, 2] == 0).all()
    k, v = (torch.empty(3, nkv * d, dtype=dtype, device="cuda") for _ in range(2))
    ops.kv_read_e4m3(st.positions, st.token_seq, st.table, *cache, k, v, st.err)
    kn, vn = torch.isnan(k.view(3, nkv, d)), torch.isnan(v.view(3, nkv, d))
    assert kn[1, 0].all() and kn.sum() == d and vn[2, 1].all() and vn.sum() == d and int(st.err) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nkv,d,page,lens", [(8, 64, 16, [333]), (2, 128, 16, [1]), (1, 16, 3, [7, 1, 50]), (3, 48, 4, [9, 2]),
                                             (8, 128, 32, [2000, 31, 777]), (1, 256, 64, [65])])
def test_read(dtype, nkv, d, page, lens):
    st = Step(lens, [0] * len(lens), nkv, nkv, d, page, dtype, seed=d)
    order = torch.randperm(sum(lens), device="cuda")
    order = torch.cat([order, order[:1]])          # in any order, a token twice
    k, v = (torch.full((order.numel() + 1, nkv * d), 3.0, dtype=dtype, device="cuda") for _ in range(2))
    n = order.numel()
    ops.kv_read_e4m3(st.positions[order], st.token_seq[order], st.table, st.k, st.v, st.ks, st.vs, k[:n], v[:n], st.err)
    assert int(st.err) == 0 and (k[n:] == 3).all() and (v[n:] == 3).all()
    at = 0
    for s, m in enumerate(lens):
        for got, codes, scale in ((k, st.k, st.ks), (v, st.v, st.vs)):
            want = st.rows_of(s, codes, scale)[0].transpose(0, 1).reshape(m, -1)
            here = torch.empty((sum(lens), nkv * d), dtype=dtype, device="cuda")
            here[order] = got[:n]
            assert torch.equal(here[at:at + m].to(F64), want)       # exact in both types at these sizes
        at += m


def test_read_and_write_report_pages_that_are_not_held():
    nq, nkv, d, page = 4, 2, 64, 16
    st = Step([40], [0], nq, nkv, d, page, BF16)
    st.table[0, 1] = -1
    k, v = (torch.full((40, nkv * d), 3.0, dtype=BF16, device="cuda") for _ in range(2))
    ops.kv_read_e4m3(st.positions, st.token_seq, st.table, st.k, st.v, st.ks, st.vs, k, v, st.err)
    assert int(st.err) == 4 and (k[16:32] == 0).all() and not (k[:16] == 0).all()
    st.err.zero_()
    cache = fresh_cache(st)
    old = [c.clone() for c in cache]
    st.table[0, 0] = st.pages                       # behind the last page
    qkv = torch.randn(40, (nq + 2 * nkv) * d).to(BF16).cuda()
    ops.rope_kv_write_e4m3(qkv, st.positions, st.token_seq, freqs(d), d, st.table, *cache, nq, nkv, d, st.err)
    assert int(st.err) == 2
    third = int(st.table[0, 2])
    for a, b in zip(cache, old):
        same = (a.view(torch.uint8) == b.view(torch.uint8)).reshape(a.shape[0], -1).all(1)
        assert not same[third] and same.sum() == a.shape[0] - 1
    st.err.zero_()
    far = st.positions.clone()
    far[3], far[4] = -1, 1 << 20                    # no position of the table's
    ops.kv_read_e4m3(far, st.token_seq, st.table, st.k, st.v, st.ks, st.vs, k, v, st.err)
    assert int(st.err) == 4 and (k[3:5] == 0).all()


SHAPES = [  # nq, nkv, d, page, lens, starts, window
    (4, 2, 64, 16, [1], [0], 0), (32, 8, 64, 16, [1], [2047], 0), (32, 8, 128, 16, [1, 1, 1], [4000, 15, 16], 0),
    (24, 8, 128, 16, [1] * 8, [1, 300, 31, 32, 33, 1000, 2000, 64], 0), (8, 8, 64, 16, [1, 1], [700, 5], 100),
    (16, 2, 128, 32, [1, 1, 1, 1], [129, 0, 1500, 77], 16), (32, 1, 64, 64, [1, 1], [999, 63], 0), (8, 1, 256, 16, [1], [515], 0),
    (32, 8, 64, 16, [5, 3, 2, 8], [800, 0, 33, 1234], 0), (32, 8, 128, 16, [1, 1, 4, 2], [800, 0, 33, 1234], 0),
    (16, 4, 64, 16, [1, 96], [1200, 500], 512), (8, 8, 128, 16, [33], [1000], 0), (24, 8, 128, 16, [130], [0], 0),
    (32, 4, 64, 32, [200, 1 + 64], [1000, 3], 0), (32, 8, 64, 16, [300], [77], 64), (4, 4, 64, 16, [257], [255], 1),
    (3, 3, 48, 4, [9, 2], [3, 30], 0), (5, 1, 80, 1, [1, 4], [44, 2], 7), (4, 2, 16, 16, [3, 20], [0, 300], 0),
    (8, 4, 96, 8, [1, 11], [5, 50], 0), (2, 1, 128, 7, [1, 30], [100, 9], 0), (6, 2, 32, 16, [1, 40], [600, 0], 33),
    (32, 8, 64, 16, [1] * 6, [5000, 0, 255, 256, 257, 1023], 0), (24, 8, 128, 16, [1] * 5, [4999, 127, 128, 129, 3], 0), (32, 8, 64, 16, [5, 1, 6, 8], [4000, 1, 255, 2000], 0),
    (32, 8, 128, 48, [5, 1, 6, 8], [4000, 1, 255, 2000], 0), (16, 2, 64, 32, [1] * 12, [100 * i for i in range(12)], 900), (64, 2, 128, 16, [1] * 9, [900] * 9, 0),
    (32, 8, 64, 16, [1, 1, 1, 5, 2, 8], [4000, 0, 700, 30, 2500, 0], 0), (32, 8, 128, 16, [1, 4, 2], [40, 0, 700], 100), (32, 8, 128, 16, [1, 1, 1, 1, 2], [900] * 5, 0),
    (20, 4, 128, 16, [6] * 6, [1500, 30, 0, 700, 122, 1], 1000), (8, 8, 128, 16, [1] * 20, [150 * i for i in range(20)], 0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,page,lens,starts,window", SHAPES)
def test_attention(dtype, nq, nkv, d, page, lens, starts, window):
    st = Step(lens, starts, nq, nkv, d, page, dtype, seed=nq + d, more_rows=2, stride_pad=16)
    out = st.attend(ops, window)
    assert int(st.err) == 0
    assert (out[sum(lens):] == 7).all()             # rows behind the last sequence's
    st.check(out, window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,starts", [([1], [200]), ([1, 1, 6], [40, 300, 500]), ([140], [60])])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_over_rows_of_very_different_sizes(dtype, lens, starts, d):
    """Rows up to e^12 times larger and smaller than others, scores far apart, and values of one size only where weights are large."""
    st = Step(lens, starts, 8, 2, d, 16, dtype, seed=9, spread=3.0, qscale=0.3)
    out = st.attend(ops)
    st.check(out)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,starts", [([1], [100]), ([5], [100]), ([1, 1, 150], [40, 70, 30])])
def test_a_key_that_is_nan_reaches_the_rows_that_see_it_alone(dtype, lens, starts):
    st = Step(lens, starts, 8, 2, 64, 16, dtype, seed=4)
    s = len(lens) - 1
    for where, scale, codes in ((0, st.ks, st.k), (1, st.vs, st.v)):
        j = starts[s] + max(0, lens[s] // 2)        # a token of the step itself: earlier rows do not see it
        page = int(st.table[s, j // 16])
        scale.view(torch.uint8)[page, where, j % 16] = 255
        codes.view(torch.uint8)[page, where, j % 16] = 0
    out = st.attend(ops)
    st.check(out)
    assert torch.isnan(out[:sum(lens)]).any() and (lens[s] == 1 or not torch.isnan(out[sum(lens[:s]):sum(lens[:s]) + lens[s] // 2]).any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_lies_behind_a_sequence_and_ahead_of_its_window_is_not_seen(dtype):
    """NaN scales and NaN numbers in the last page behind the sequence's end, and in rows that the window hides from all."""
    for lens, starts, window in (([1, 1], [37, 99], 0), ([1, 7], [400, 99], 50), ([130], [3], 0)):
        st = Step(lens, starts, 8, 2, 64, 16, dtype, seed=6)
        plain = st.attend(ops, window)
        for s, n in enumerate(st.totals):
            last = int(st.table[s, (n - 1) // 16])
            for t in (st.k, st.v, st.ks, st.vs):
                t.view(torch.uint8)[last, :, (n - 1) % 16 + 1:] = 255
            if window and n - lens[s] - window > 16:
                first = int(st.table[s, 0])
                for t in (st.k, st.v, st.ks, st.vs):
                    t.view(torch.uint8)[first] = 255
        out = st.attend(ops, window)
        assert torch.equal(out, plain) and not torch.isnan(out).any() and int(st.err) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,starts", [([1], [60]), ([4], [60]), ([140], [60])])
def test_pages_that_are_not_held_are_left_out_and_reported(dtype, lens, starts):
    for page, d in ((16, 64), (8, 48)):
        st = Step(lens, starts, 4, 2, d, page, dtype, seed=8)
        st.table[0, 1] = -1
        st.table[0, 2] = st.pages + 3
        out = st.attend(ops)
        assert int(st.err) == 4
        st.check(out)


FORMS = ["rows", "columns", "tcgen05", "dense"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("nq,nkv,d,page,lens,starts,window", [
    (4, 4, 64, 16, [1], [0], 0), (32, 8, 64, 16, [40], [3000], 0), (32, 8, 128, 16, [33, 1, 7], [2500, 64, 0], 0), (8, 2, 64, 16, [64], [0], 0),
    (8, 8, 128, 32, [127, 129], [1, 63], 0), (24, 8, 128, 16, [43, 42], [64, 65], 0), (32, 1, 64, 16, [9], [500], 70), (16, 2, 128, 64, [100], [300], 1),
    (8, 1, 128, 16, [20, 50], [1000, 10], 128), (40, 8, 64, 16, [30], [90], 0), (5, 1, 128, 48, [28], [200], 33), (128, 1, 64, 16, [2], [200], 0)])
def test_every_form_of_the_attention(form, nq, nkv, d, page, lens, starts, window, monkeypatch):
    monkeypatch.setattr(ops, "E4M3_FORMS", (form, form))
    for spread, qscale in ((1.0, 1.0), (3.0, 0.3)):
        st = Step(lens, starts, nq, nkv, d, page, BF16, seed=nq + d, more_rows=2, stride_pad=16, spread=spread, qscale=qscale)
        out = st.attend(ops, window, num_decode=0)
        assert int(st.err) == 0 and (out[sum(lens):] == 7).all()
        st.check(out, window)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,starts", [([5], [100]), ([3, 150], [40, 30]), ([70, 2], [200, 1000])])
def test_keys_that_are_nan_missing_or_out_of_sight_in_every_form(form, d, lens, starts, monkeypatch):
    monkeypatch.setattr(ops, "E4M3_FORMS", (form, form))
    s, n = len(lens) - 1, lens[-1]
    for where in (0, 1):                                          # a key, a value that is NaN, of a token of the step
        st = Step(lens, starts, 8, 2, d, 16, BF16, seed=4)
        j = starts[s] + n // 2
        scale, codes = (st.ks, st.k) if where == 0 else (st.vs, st.v)
        scale.view(torch.uint8)[int(st.table[s, j // 16]), where, j % 16] = 255
        codes.view(torch.uint8)[int(st.table[s, j // 16]), where, j % 16] = 0
        out = st.attend(ops, num_decode=0)
        st.check(out)
        assert torch.isnan(out[:sum(lens)]).any() and not torch.isnan(out[:sum(lens[:s]) + n // 2]).any()
    st = Step(lens, starts, 8, 2, d, 16, BF16, seed=5)            # pages that are not held
    st.table[s, 1], st.table[s, 2] = -1, st.pages
    out = st.attend(ops, num_decode=0)
    assert int(st.err) == 4
    st.check(out)
    for window in (0, 50):                                        # NaN behind the sequence's end and ahead of the window
        st = Step(lens, starts, 8, 2, d, 16, BF16, seed=6)
        plain = st.attend(ops, window, num_decode=0)
        for i, m in enumerate(st.totals):
            last = int(st.table[i, (m - 1) // 16])
            first = int(st.table[i, 0]) if window and m - lens[i] - window > 16 else None
            for t in (st.k, st.v, st.ks, st.vs):
                t.view(torch.uint8)[last, :, (m - 1) % 16 + 1:] = 255
                if first is not None:
                    t.view(torch.uint8)[first] = 255
        out = st.attend(ops, window, num_decode=0)
        assert torch.equal(out, plain) and not torch.isnan(out).any() and int(st.err) == 0


@pytest.mark.parametrize("form", FORMS)
def test_rows_that_are_zeros_in_every_form(form, monkeypatch):
    """Queries, keys and values of zeros (the least scales of all), alone and beside others."""
    monkeypatch.setattr(ops, "E4M3_FORMS", (form, form))
    st = Step([40, 3], [100, 200], 8, 2, 64, 16, BF16, seed=7)
    st.q[::3] = 0
    for t in (st.k, st.v, st.ks, st.vs):
        t.view(torch.uint8)[int(st.table[0, 2])] = 0
        t.view(torch.uint8)[st.table[1, :13].long()] = 0
    out = st.attend(ops, num_decode=0)
    st.check(out)
    assert (out[40:43] == 0).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_a_query_that_is_not_finite_reaches_its_own_row_alone(form, d, what, monkeypatch):
    monkeypatch.setattr(ops, "E4M3_FORMS", (form, form))
    st = Step([5, 3], [300, 40], 8, 2, d, 16, BF16, seed=3)
    plain = st.attend(ops, num_decode=0)
    st.q[2, 3 * d + 7] = what
    out = st.attend(ops, num_decode=0)
    assert torch.isnan(out[2, 3 * d:4 * d]).all() and int(st.err) == 0
    out[2, 3 * d:4 * d] = plain[2, 3 * d:4 * d]
    assert torch.equal(out, plain)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
def test_queries_whose_numbers_lie_far_apart(form, d, monkeypatch):
    """A few of a row's numbers 2^10 and more above the others, rows up to 2^30 apart."""
    monkeypatch.setattr(ops, "E4M3_FORMS", (form, form))
    for size in (1.0, 2.0 ** -20):
        st = Step([6, 1], [500, 900], 8, 2, d, 16, BF16, seed=11, spread=0.5)
        g = torch.Generator().manual_seed(2)
        st.q.mul_(torch.exp(2.5 * torch.randn(st.q.shape, generator=g)).to(BF16).cuda() * (0.02 * size))
        st.check(st.attend(ops, scale=d ** -0.5 / size, num_decode=0), scale=d ** -0.5 / size)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,starts", [([1, 1], [60, 2000]), ([5], [100]), ([140], [60])])
def test_results_off_16_bytes(dtype, lens, starts):
    """out anywhere in a buffer: kernels that store 16 bytes are not the ones that take it."""
    st = Step(lens, starts, 8, 2, 64, 16, dtype, seed=4)
    buffer = torch.full((sum(lens) * 8 * 64 + 3,), 7.0, dtype=dtype, device="cuda")
    out = buffer[1:-2].view(sum(lens), -1)
    st.attend(ops, out=out)
    st.check(out)
    assert int(st.err) == 0 and float(buffer[0]) == 7 and (buffer[-2:] == 7).all()


def test_prompts_in_groups_of_what_the_scratch_holds(monkeypatch):
    monkeypatch.setattr(ops, "E4M3_FORMS", ("dense", "dense"))
    st = Step([40, 3, 70, 9], [100, 200, 0, 30], 8, 2, 64, 16, BF16, seed=7)
    whole = st.attend(ops, num_decode=0)
    monkeypatch.setattr(ops, "E4M3_DENSE_SCRATCH", 1)              # a sequence at a time
    assert torch.equal(st.attend(ops, num_decode=0), whole) and int(st.err) == 0
    st.check(whole)


def test_a_sequence_all_of_whose_pages_are_missing_gives_zeros():
    for lens, starts in (([1, 1], [60, 30]), ([4, 3], [60, 30]), ([140, 20], [5, 30])):
        st = Step(lens, starts, 4, 2, 64, 16, BF16)
        st.table[0, :] = -1
        out = st.attend(ops)
        assert int(st.err) == 4 and (out[:lens[0]] == 0).all()
        st.check(out)


def test_sequences_without_tokens_and_calls_without_any():
    st = Step([1, 5, 3], [30, 40, 7], 4, 2, 64, 16, BF16)
    st.lens = [1, 5, 3]
    out = st.attend(ops)
    # a sequence between them that brings none
    st2 = Step([1, 5, 3], [30, 40, 7], 4, 2, 64, 16, BF16)
    st2.q_start = torch.tensor([0, 1, 6, 6, 9], dtype=torch.int32, device="cuda")
    st2.seq_lens = torch.tensor([31, 45, 0, 10], dtype=torch.int32, device="cuda")
    st2.table = torch.stack([st2.table[0], st2.table[1], torch.full_like(st2.table[0], -1), st2.table[2]])
    assert torch.equal(st2.attend(ops), out) and int(st2.err) == 0
    empty = torch.empty(0, 4 * 64, dtype=BF16, device="cuda")
    st.q = st.q[:0]
    assert st.attend(ops, out=empty).numel() == 0


@pytest.mark.parametrize("form,d", [(None, 64), ("columns", 64), ("columns", 128), ("tcgen05", 64), ("dense", 128)])
def test_the_operators_in_a_row_on_another_stream_and_captured(form, d, monkeypatch):
    """Tokens written step by step, attended to and read back, eagerly and in a captured graph that is replayed with other inputs."""
    monkeypatch.setattr(ops, "E4M3_FORMS", form and (form, form))
    nq, nkv, page = 8, 2, 16
    st = Step([1, 1, 1], [37, 100, 15], nq, nkv, d, page, BF16)
    inv = freqs(d)
    side = torch.cuda.Stream()
    qkv = torch.randn(3, (nq + 2 * nkv) * d, device="cuda").to(BF16)

    def step(cache):
        q, out = torch.empty(3, nq * d, dtype=BF16, device="cuda"), torch.empty(3, nq * d, dtype=BF16, device="cuda")
        k, v = (torch.empty(3, nkv * d, dtype=BF16, device="cuda") for _ in range(2))
        ops.rope_kv_write_e4m3(qkv, st.positions, st.token_seq, inv, d, st.table, *cache, nq, nkv, d, st.err, q_out=q)
        ops.attention_e4m3(q, out, *cache, st.table, st.q_start, st.seq_lens, 3, 1, 128, nq, nkv, 0, d ** -0.5, st.err)
        ops.kv_read_e4m3(st.positions, st.token_seq, st.table, *cache, k, v, st.err)
        return q, out, k, v

    cache = [st.k, st.v, st.ks, st.vs]
    first = [x.clone() for x in step(cache)]
    st.q = first[0]
    st.check(first[1])
    assert torch.equal(first[3].to(F64).view(3, nkv, d),
                       values(*[(c.to(E4M3), b.view(E8M0)) for c, b in [quantise(qkv.view(3, -1, d)[:, nq + nkv:])]][0]))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(cache)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step(cache)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, static))
    # the next token of each, through the graph
    qkv.copy_(torch.randn(3, (nq + 2 * nkv) * d, device="cuda").to(BF16))
    st.table[2, 1] = next(p for p in range(st.pages) if not (st.table == p).any())
    st.positions += 1
    st.seq_lens += 1
    st.totals = [n + 1 for n in st.totals]
    graph.replay()
    torch.cuda.synchronize()
    st.q = static[0]
    st.check(static[1])
    assert int(st.err) == 0


def test_attention_does_not_depend_on_how_a_prompt_was_cut():
    """A portion of many tokens against its tokens a few at a time: the same arithmetic up to the order of additions."""
    st = Step([70], [50], 8, 2, 64, 16, BF16, seed=2)
    whole = st.attend(ops)
    st.check(whole)
    for n in (1, 3, 70 - 4):
        part = Step([70], [50], 8, 2, 64, 16, BF16, seed=2)
        part.lens, part.totals = [n], [50 + n]
        part.q = part.q[:n]
        part.q_start[1] = n
        part.seq_lens[0] = 50 + n
        part.num_decode = 1 if n == 1 else 0
        part.check(part.attend(ops))


class TheLongWay:
    """The extension module without its checking and launching in one go."""

    def __init__(self, module):
        self.module = module

    def __getattr__(self, name):
        return (lambda *args: False) if name in ("e4m3_write", "e4m3_read") else getattr(self.module, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,rd,page,window,start", [
    (8, 2, 64, 64, 16, 0, 100), (6, 2, 128, 64, 32, 20, 100), (5, 1, 256, 0, 16, 0, 100), (4, 4, 48, 48, 7, 9, 100), (64, 1, 64, 64, 16, 0, 100),
    (32, 1, 64, 64, 16, 33, 100), (32, 1, 128, 64, 16, 0, 100), (32, 8, 64, 64, 16, 0, 2729), (32, 8, 64, 64, 16, 0, 2730), (16, 16, 128, 128, 16, 0, 766),
    (16, 16, 128, 128, 16, 0, 767), (16, 16, 128, 128, 16, 767, 2000), (16, 16, 128, 128, 16, 766, 2000), (32, 1, 128, 64, 48, 0, 6000), (12, 4, 256, 64, 16, 0, 3000)])
def test_calls_checked_in_one_go_and_the_long_way_give_the_same_bits(dtype, nq, nkv, d, rd, page, window, start, monkeypatch):
    results = []
    for long_way in (False, True):
        if long_way:
            module = TheLongWay(ops._launch())
            monkeypatch.setattr(ops, "_launch", lambda: module)
        st = Step([1, 1, 1], [37, start, 15], nq, nkv, d, page, dtype, seed=d, more_rows=1, stride_pad=16)
        g = torch.Generator().manual_seed(1)
        qkv = torch.randn(3, (nq + 2 * nkv) * d, generator=g).to(dtype).cuda()
        cache = (st.k, st.v, st.ks, st.vs)
        inv = freqs(rd) if rd else None
        out = [torch.full((4, nq * d + 8), 3.0, dtype=dtype, device="cuda")]
        ops.rope_kv_write_e4m3(qkv, st.positions, st.token_seq, inv, rd, st.table, *cache, nq, nkv, d, st.err, q_out=out[0][:3, :nq * d])
        ops.rope_kv_write_e4m3(qkv, st.positions, st.token_seq, inv, rd, st.table, *cache, nq, nkv, d, st.err)
        out += [qkv, st.attend(ops, window)] + [torch.full((4, nkv * d), 3.0, dtype=dtype, device="cuda") for _ in range(2)]
        ops.kv_read_e4m3(st.positions, st.token_seq, st.table, *cache, out[3][:3], out[4][:3], st.err)
        assert int(st.err) == 0
        results.append(out + [c.view(torch.uint8) for c in cache])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def on_gpu(x):
    """A copy on the GPU with the same strides."""
    if not isinstance(x, torch.Tensor):
        return x
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    y.view(torch.uint8).copy_(x.view(torch.uint8)) if x.dtype in (E4M3, E8M0) else y.copy_(x)
    return y


I32 = dict(dtype=torch.int32)
WRITES = [dict(qkv=torch.zeros(2, 7 * 64, dtype=BF16)), dict(qkv=torch.zeros(2, 8 * 64, dtype=torch.float16)), dict(positions=torch.zeros(1, **I32)),
          dict(token_seq=torch.zeros(2, dtype=torch.int64)), dict(inv_freq=None), dict(inv_freq=torch.zeros(32)),
          dict(inv_freq=torch.zeros(16, dtype=torch.float64)), dict(inv_freq=torch.zeros(64, dtype=torch.float64)[::2]),
          dict(q_out=torch.zeros(2, 4 * 64)), dict(q_out=torch.zeros(3, 4 * 64, dtype=BF16)), dict(q_out=torch.zeros(2, 5 * 64, dtype=BF16)),
          dict(q_out=torch.zeros(4 * 64, 2, dtype=BF16).t()), dict(q_out=torch.zeros(1, 4 * 64, dtype=BF16).expand(2, -1)),
          dict(qkv=torch.zeros(8 * 64, 2, dtype=BF16).t()), dict(block_table=torch.zeros(2, **I32)), dict(err=torch.zeros(1, dtype=torch.int64)),
          dict(nkv=1, qkv=torch.zeros(2, 6 * 64, dtype=BF16)), dict(d=32, qkv=torch.zeros(2, 8 * 32, dtype=BF16)), dict(rotary_dim=65),
          dict(rotary_dim=-64), dict(nq=-4, qkv=torch.zeros(2, 0, dtype=BF16))]
DECODES = [dict(q=torch.zeros(2, 4 * 64)), dict(q=torch.zeros(2, 3 * 64, dtype=BF16)), dict(q=torch.zeros(1, 4 * 64, dtype=BF16)),
           dict(q=torch.zeros(4 * 64, 2, dtype=BF16).t()), dict(out=torch.zeros(2, 8 * 64, dtype=BF16)[:, ::2]),
           dict(q=torch.zeros(2, 4 * 64, dtype=torch.float16), out=torch.zeros(2, 4 * 64, dtype=torch.float16)),
           dict(q_start=torch.zeros(2, **I32)), dict(seq_lens=torch.zeros(2, dtype=torch.int64)), dict(nd=3), dict(nd=-1), dict(ms=33), dict(ms=-1),
           dict(mq=-1), dict(nkv=4), dict(nq=3), dict(nkv=0), dict(table=torch.zeros(1, 2, **I32)), dict(table=torch.zeros(2, 4, **I32)[:, ::2]),
           dict(window=-1), dict(scale=math.nan), dict(scale=math.inf)]


@pytest.mark.parametrize("over", WRITES)
def test_a_write_that_does_not_fit_is_refused_on_the_gpu_too(over):
    a = dict(qkv=torch.zeros(2, 8 * 64, dtype=BF16), positions=torch.arange(2, **I32), token_seq=torch.zeros(2, **I32),
             inv_freq=torch.zeros(32, dtype=torch.float64), rotary_dim=64, block_table=torch.arange(2, **I32).view(1, 2), nq=4, nkv=2, d=64,
             err=torch.zeros(1, **I32), q_out=None)
    a.update(over)
    a = {k: on_gpu(x) if k != "q_out" or x is None or x.stride(0) else x[:1].cuda().expand(2, -1) for k, x in a.items()}
    cache = [torch.full((3, 2, 16) + tail, 9, dtype=torch.uint8, device="cuda") for tail in ((64,), (64,), (), ())]
    with pytest.raises(ops.KernelError):
        ops.rope_kv_write_e4m3(a["qkv"], a["positions"], a["token_seq"], a["inv_freq"], a["rotary_dim"], a["block_table"], cache[0].view(E4M3),
                               cache[1].view(E4M3), cache[2].view(E8M0), cache[3].view(E8M0), a["nq"], a["nkv"], a["d"], a["err"], q_out=a["q_out"])
    assert all((c == 9).all() for c in cache)


@pytest.mark.parametrize("over", DECODES)
def test_an_attention_of_single_tokens_that_does_not_fit_is_refused_on_the_gpu_too(over):
    a = dict(q=torch.zeros(2, 4 * 64, dtype=BF16), out=torch.zeros(2, 4 * 64, dtype=BF16), table=torch.zeros(2, 2, **I32),
             q_start=torch.arange(3, **I32), seq_lens=torch.full((2,), 20, **I32), nd=2, mq=1, ms=20, nq=4, nkv=2, window=0, scale=0.125,
             err=torch.zeros(1, **I32))
    a.update(over)
    a = {k: on_gpu(x) for k, x in a.items()}
    cache = [torch.zeros((3, 2, 16) + tail, dtype=torch.uint8, device="cuda") for tail in ((64,), (64,), (), ())]
    with pytest.raises(ops.KernelError):
        ops.attention_e4m3(a["q"], a["out"], cache[0].view(E4M3), cache[1].view(E4M3), cache[2].view(E8M0), cache[3].view(E8M0), a["table"],
                           a["q_start"], a["seq_lens"], a["nd"], a["mq"], a["ms"], a["nq"], a["nkv"], a["window"], a["scale"], a["err"])


def test_a_reading_that_does_not_fit_is_refused_on_the_gpu_too():
    st = Step([2], [0], 4, 2, 64, 16, BF16)
    good = dict(pos=st.positions, seq=st.token_seq, k=torch.zeros(2, 128, dtype=BF16, device="cuda"), v=torch.zeros(2, 128, dtype=BF16, device="cuda"))
    for over in (dict(seq=st.token_seq[:1]), dict(pos=st.positions.long()), dict(k=good["k"][:1]), dict(v=good["v"].float()),
                 dict(k=good["k"].half(), v=good["v"].half()), dict(k=torch.zeros(2, 256, dtype=BF16, device="cuda")[:, ::2]), dict(v=good["v"].cpu())):
        a = {**good, **over}
        with pytest.raises(ops.KernelError):
            ops.kv_read_e4m3(a["pos"], a["seq"], st.table, st.k, st.v, st.ks, st.vs, a["k"], a["v"], st.err)
    with pytest.raises(ops.KernelError):
        ops.kv_read_e4m3(good["pos"], good["seq"], st.table, st.k, st.v, st.k, st.vs, good["k"], good["v"], st.err)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(8, 2), (32, 2), (16, 8)])
def test_the_same_bits_again_and_again_beside_other_work(d, nq, nkv, monkeypatch):
    """Calls whose warps hand tiles to one another, repeated, two streams at a time, each over a cache of its own: no result depends
    on who was first."""
    monkeypatch.setattr(ops, "E4M3_FORMS", ("columns", "columns"))
    steps = [Step(lens, starts, nq, nkv, d, 16, BF16, seed=i, spread=2.0) for i, (lens, starts) in enumerate(
        [([1] * 7, [3000, 5, 777, 128, 255, 2000, 1]), ([1, 1, 2, 1 + 3 % nkv], [1500, 900, 640, 64]), ([1], [9000])])]
    streams = [torch.cuda.Stream() for _ in range(2)]
    first = [st.attend(ops) for st in steps]
    torch.cuda.synchronize()
    for st, out in zip(steps, first):
        st.check(out)
    outs = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((i % 3, steps[i % 3].attend(ops)))
    torch.cuda.synchronize()
    assert all(torch.equal(first[which], out) for which, out in outs) and all(int(st.err) == 0 for st in steps)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [10, 22, 25, 27])
def test_a_small_value_that_has_all_the_weight(form, d, gap, monkeypatch):
    """One key that every row looks at, whose value lies 2^gap below those that weigh nothing."""
    monkeypatch.setattr(ops, "E4M3_FORMS", (form, form))
    st = Step([1, 2], [46, 600], 8, 2, d, 16, BF16, seed=5, spread=0.3)
    for s, j in ((0, 1), (1, 333)):
        page, slot = int(st.table[s, j // 16]), j % 16
        k = (st.k[page, :, slot].float() * 2.0 ** (st.ks.view(torch.uint8)[page, :, slot].float() - 127)[:, None])     # [nkv, d]
        first, last = int(st.q_start[s]), int(st.q_start[s + 1])
        st.q[first:last] = (k * 60 / k.square().sum(-1, keepdim=True) * d ** 0.5).repeat_interleave(4, 0).reshape(-1).to(BF16)
        st.vs.view(torch.uint8)[page, :, slot] -= gap
    out = st.attend(ops, num_decode=0)
    st.check(out)
    assert (out[:3] != 0).any(-1).all()


@pytest.mark.parametrize("dtype,forms", [(BF16, None), (F32, None)] + [(BF16, (a, b)) for a in FORMS for b in FORMS])
def test_single_tokens_and_portions_side_by_side(dtype, forms, monkeypatch):
    """The portions' kernel does not wait for the single tokens' one, but for the write ahead of both, and what comes behind waits for
    both: written, attended to and overwritten many times without a stop in between, each result that of its own inputs."""
    monkeypatch.setattr(ops, "E4M3_FORMS", forms)
    nq, nkv, d, page = 8, 2, 64, 16
    lens, starts = [1] * 6 + [40, 200, 3], [3000, 5, 900, 2000, 0, 77, 500, 0, 64]
    st = Step(lens, starts, nq, nkv, d, page, dtype, seed=3)
    T, inv = sum(lens), freqs(d)
    g = torch.Generator(device="cuda").manual_seed(1)
    inputs = [torch.randn(T, (nq + 2 * nkv) * d, device="cuda", generator=g).to(dtype) for _ in range(24)]
    cache = [st.k, st.v, st.ks, st.vs]

    def step(x, out, q):
        ops.rope_kv_write_e4m3(x, st.positions, st.token_seq, inv, d, st.table, *cache, nq, nkv, d, st.err, q_out=q)
        ops.attention_e4m3(q, out, *cache, st.table, st.q_start, st.seq_lens, 6, 200, max(st.totals), nq, nkv, 0, d ** -0.5, st.err)

    apart = []
    q = torch.empty(T, nq * d, dtype=dtype, device="cuda")
    for x in inputs:
        out = torch.empty(T, nq * d, dtype=dtype, device="cuda")
        step(x, out, q)
        torch.cuda.synchronize()
        apart.append(out)
    st.q = q.clone()
    st.check(apart[-1])
    outs = [torch.empty(T, nq * d, dtype=dtype, device="cuda") for _ in inputs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = []
        for x, out in zip(inputs, outs):
            step(x, out, q)
            kept.append(out.clone())
            out.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(apart, kept)) and int(st.err) == 0
