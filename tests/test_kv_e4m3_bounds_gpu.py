"""Attention over a cache kept in 8 bits, each sequence within the bound of the kernel that takes it and of what its own rows look at."""
import pytest
import torch

from kv_e4m3_bounds import check
from kv_e4m3_util import Step
from rllm_b200.kernels import ops
from test_kv_e4m3_gpu import SHAPES

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
FORMS = [(F32, None)] + [(BF16, f) for f in ("rows", "columns", "tcgen05", "dense")]


def attend(st, form, monkeypatch, window=0, num_decode=None):
    forced = form and (form, form)
    monkeypatch.setattr(ops, "E4M3_FORMS", forced)
    num_decode = st.num_decode if num_decode is None else num_decode
    out = st.attend(ops, window, num_decode=num_decode)
    assert int(st.err) == 0 and (out[sum(st.lens):] == 7).all()
    check(st, out, window, num_decode=num_decode, forced=forced)
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nkv,d,page,lens,starts,window", SHAPES)
def test_steps_of_all_kinds(dtype, nq, nkv, d, page, lens, starts, window, monkeypatch):
    attend(Step(lens, starts, nq, nkv, d, page, dtype, seed=nq + d, more_rows=2, stride_pad=16), None, monkeypatch, window)


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,starts,window", [([1], [200], 0), ([1, 2, 7], [46, 600, 3000], 0), ([40], [60], 0), ([9, 30], [500, 90], 70)])
@pytest.mark.parametrize("spread,qscale", [(1.0, 1.0), (3.0, 0.3)])
def test_rows_of_like_and_of_very_different_sizes(dtype, form, d, lens, starts, window, spread, qscale, monkeypatch):
    attend(Step(lens, starts, 8, 2, d, 16, dtype, seed=9, spread=spread, qscale=qscale), form, monkeypatch, window, 0)


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [8, 20, 25, 32, 45])
def test_values_that_a_row_does_not_see_are_larger_by_far(dtype, form, d, gap, monkeypatch):
    """Values of the portion's later tokens 2^gap times the others: the rows of the earlier ones keep all of their bits."""
    for lens, starts in (([12], [20]), ([1, 7], [40, 300])):
        st = Step(lens, starts, 8, 2, d, 16, dtype, seed=5, spread=0.3, qscale=0.5)
        s = len(lens) - 1
        for j in range(st.totals[s] - lens[s] // 2, st.totals[s]):
            st.vs.view(torch.uint8)[int(st.table[s, j // 16]), :, j % 16] += gap
        out = attend(st, form, monkeypatch, num_decode=0)
        assert (out[:sum(lens) - lens[s] // 2] != 0).all()


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [8, 20, 25, 32, 45, 90])
def test_values_that_have_the_weight_are_smaller_by_far(dtype, form, d, gap, monkeypatch):
    """A few like keys that a row looks at, whose values lie 2^gap below those that weigh nothing, in one tile with them and tiles away."""
    st = Step([1, 2], [46, 600], 8, 2, d, 16, dtype, seed=5, spread=0.3)
    for s, keys in ((0, (1, 2, 40)), (1, (333, 5, 590))):
        place = [(int(st.table[s, j // 16]), j % 16) for j in keys]
        page, slot = place[0]
        for other, at in place[1:]:                                # its neighbour, but for a number
            for t in (st.k, st.ks):
                t.view(torch.uint8)[other, :, at] = t.view(torch.uint8)[page, :, slot]
            st.k.view(torch.uint8)[other, :, at, 3] = 0
        k = (st.k[page, :, slot].float() * 2.0 ** (st.ks.view(torch.uint8)[page, :, slot].float() - 127)[:, None])
        first, last = int(st.q_start[s]), int(st.q_start[s + 1])
        st.q[first:last] = (k * 120 / k.square().sum(-1, keepdim=True) * d ** 0.5).repeat_interleave(4, 0).reshape(-1).to(dtype)
        for other, at in place:
            st.vs.view(torch.uint8)[other, :, at] -= gap
    out = attend(st, form, monkeypatch, num_decode=0)
    assert (out[:3] != 0).any(-1).all()


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("power", [-118, -60, 60, 110])
def test_values_near_the_ends_of_the_range(dtype, form, power, monkeypatch):
    """All values about 2^power."""
    for lens, starts in (([3], [100]), ([1, 20], [900, 30])):
        st = Step(lens, starts, 8, 2, 64, 16, dtype, seed=5, spread=0.3)
        scale = st.vs.view(torch.uint8)
        scale.copy_((scale.int() + power).clamp(0, 247).to(torch.uint8))
        attend(st, form, monkeypatch, num_decode=0)


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [18, 20, 21, 30, 60])
@pytest.mark.parametrize("lens,starts", [([12], [20]), ([1, 70], [40, 300])])
def test_keys_that_a_row_does_not_see_are_larger_by_far(dtype, form, d, gap, lens, starts, monkeypatch):
    """Keys of the portion's later tokens 2^gap times the others; some values too, and a row of zeros among each."""
    st = Step(lens, starts, 8, 2, d, 16, dtype, seed=5, spread=0.3, qscale=0.5)
    s = len(lens) - 1
    for j in range(st.totals[s] - lens[s] // 2, st.totals[s]):
        page, slot = int(st.table[s, j // 16]), j % 16
        st.ks.view(torch.uint8)[page, :, slot] += gap
        if j % 3 == 0:
            st.vs.view(torch.uint8)[page, :, slot] += gap + 1
    for t in (st.k, st.v, st.ks, st.vs):
        t.view(torch.uint8)[int(st.table[s, 0]), :, 5] = 0
    out = attend(st, form, monkeypatch, num_decode=0)
    assert (out[:sum(lens) - lens[s] // 2] != 0).all()


@pytest.mark.parametrize("dtype,form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [200.0, 2.0 ** 14, 2.0 ** 20, 2.0 ** 26, 2.0 ** 32, 2.0 ** 62])
@pytest.mark.parametrize("lens,starts", [([1], [700]), ([2, 20], [900, 700])])
def test_keys_that_are_alike_weigh_the_same_however_large_scores_are(dtype, form, d, size, lens, starts, monkeypatch):
    """Five like keys, tiles apart, whose scores of ``size`` leave all others behind: the result is their values' mean.  Like scores are
    rounded alike, so what large ones lose does not count: a weight is off by its rounding, two exponentials and their arguments of up to
    2^6 (2 (2^-22 + 2^6 2^-24)), and the sums by n 2^-24."""
    st = Step(lens, starts, 8, 2, d, 16, dtype, seed=12, spread=0.1)
    for s in range(len(lens)):
        place = [(int(st.table[s, j // 16]), j % 16) for j in (3, 130, 333, 400, 690)]
        page, slot = place[0]
        for i, (other, at) in enumerate(place):
            for t in (st.k, st.ks):
                t.view(torch.uint8)[other, :, at] = t.view(torch.uint8)[page, :, slot]
            st.vs.view(torch.uint8)[other, :, at] += (0, 3, 7, 1, 10)[i]
        k = (st.k[page, :, slot].float() * 2.0 ** (st.ks.view(torch.uint8)[page, :, slot].float() - 127)[:, None])
        first, last = int(st.q_start[s]), int(st.q_start[s + 1])
        st.q[first:last] = (k * size / k.square().sum(-1, keepdim=True) * d ** 0.5).repeat_interleave(4, 0).reshape(-1).to(dtype)
    forced = form and (form, form)
    monkeypatch.setattr(ops, "E4M3_FORMS", forced)
    out = st.attend(ops, num_decode=0)
    assert int(st.err) == 0
    at = 0
    for s, n in enumerate(lens):
        v, _ = st.rows_of(s, st.v, st.vs)
        k, _ = st.rows_of(s, st.k, st.ks)
        q = st.q[at:at + n].double().view(n, 2, 4, d)
        scores = torch.einsum("nghd,gkd->nghk", q, k) * d ** -0.5
        rest = scores.clone()
        rest[..., [3, 130, 333, 400, 690]] = float("-inf")
        assert (scores[..., 3] - rest.amax(-1) > 0.3 * size).all()
        mean = v[:, [3, 130, 333, 400, 690]].mean(1)[None, :, None]
        size_of = v[:, [3, 130, 333, 400, 690]].abs().mean(1)[None, :, None]
        rel = {"dense": 2.0 ** -8 + 4e-5, None: 2.0 ** -22}.get(form, 2.0 ** -11) + 2 * (2.0 ** -22 + 64 * 2.0 ** -24) + st.totals[s] * 2.0 ** -24
        bound = rel * size_of + torch.finfo(dtype).eps / 2 * mean.abs()
        got = out[at:at + n].double().view(n, 2, 4, d)
        assert ((got - mean).abs() <= bound).all(), float(((got - mean).abs() / bound).max())
        at += n


@pytest.mark.parametrize("nq,nkv,d,page,window,total", [(8, 2, 64, 16, 0, 700), (8, 2, 64, 16, 100, 700), (32, 8, 128, 16, 0, 190), (8, 1, 256, 32, 33, 300),
                                                        (24, 8, 128, 48, 500, 2100), (3, 3, 48, 4, 0, 90), (4, 4, 64, 8, 20, 130)])
def test_a_float32_result_does_not_depend_on_the_step(nq, nkv, d, page, window, total):
    """The last 40 tokens of a sequence in one portion, cut in any way, one by one, and beside others: the same bits."""
    st = Step([40], [total - 40], nq, nkv, d, page, F32, seed=3, spread=1.5)
    whole = st.attend(ops, window)
    check(st, whole, window)
    q, table, pages = st.q, st.table, st.pages

    def step(parts, num_decode=None):
        """Sequences over the same pages: (first, last) of the tokens of each."""
        st.lens = [b - a for a, b in parts]
        st.totals = [total - 40 + b for _, b in parts]
        st.q = torch.cat([q[a:b] for a, b in parts])
        st.q_start = torch.tensor([sum(st.lens[:i]) for i in range(len(parts) + 1)], dtype=torch.int32, device="cuda")
        st.seq_lens = torch.tensor(st.totals, dtype=torch.int32, device="cuda")
        st.table = table.expand(len(parts), -1).contiguous()
        st.num_decode = next((i for i, n in enumerate(st.lens) if n != 1), len(parts))
        out = st.attend(ops, window)
        assert int(st.err) == 0
        at = 0
        for (a, b), n in zip(parts, st.lens):
            assert torch.equal(out[at:at + n], whole[a:b]), (a, b)
            at += n

    for cut in ([0, 1, 2, 5, 21, 40], [0, 39, 40], [0, 8, 16, 24, 32, 40]):
        for a, b in zip(cut, cut[1:]):
            step([(a, b)])
    step([(i, i + 1) for i in range(40)])
    step([(0, 1)])
    step([(3, 4)] * 70 + [(39, 40), (0, 40), (5, 9)])
    step([(7, 8), (1, 4), (36, 40)])
