"""Attention over a cache kept in 8 bits at the limits of its arguments: bounds beyond 32 bits, tensors off 16 bytes, more rows and
sequences than a kernel's grid has places for."""
import pytest
import torch

from kv_e4m3_util import E8M0, Step
from rllm_b200.kernels import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def call(st, out, window=0, max_q_len=None, max_seq_len=None, scale=None):
    ops.attention_e4m3(st.q, out, st.k, st.v, st.ks, st.vs, st.table, st.q_start, st.seq_lens, st.num_decode,
                       max(st.lens) if max_q_len is None else max_q_len, max(st.totals) if max_seq_len is None else max_seq_len, st.nq, st.nkv,
                       window, st.d ** -0.5 if scale is None else scale, st.err)
    assert int(st.err) == 0
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,starts", [([1, 5], [300, 100]), ([1], [4000]), ([40], [60]), ([300], [20])])
def test_bounds_beyond_32_bits(dtype, lens, starts):
    """Larger than anything that they bound: they hide nothing, cut nothing off and change no result."""
    st = Step(lens, starts, 8, 2, 64, 16, dtype, seed=1)
    plain = st.attend(ops)
    st.check(plain)
    for window in ((1 << 31) - 1, 1 << 31, (1 << 32) + 5, (1 << 62) + 1):
        assert torch.equal(call(st, torch.full_like(plain, 7.0), window), plain)
    for most in ((1 << 31) - 1, 1 << 31, (1 << 32) + 1, 1 << 62):
        got = call(st, torch.full_like(plain, 7.0), max_q_len=most)
        st.check(got)
    for window in (-1, -(1 << 32) + 5, -(1 << 31)):
        with pytest.raises(ops.KernelError):
            call(st, torch.full_like(plain, 7.0), window)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_queries_far_apart(dtype):
    """A single row's stride is no matter; rows 2^31 numbers apart and more are refused."""
    st = Step([1], [70], 8, 2, 64, 16, dtype, seed=2)
    plain = st.attend(ops)
    for stride in (1 << 33, (1 << 32) + 1, 0):
        q = st.q
        st.q = st.q.as_strided((1, 8 * 64), (stride, 1))
        assert torch.equal(call(st, torch.full_like(plain, 7.0)), plain)
        st.q = q
    st = Step([1, 1], [70, 30], 8, 2, 64, 16, dtype, seed=2)
    buffer = torch.zeros((1 << 31) + 1024, dtype=dtype, device="cuda")
    st.q = buffer.as_strided((2, 8 * 64), (1 << 31, 1))
    with pytest.raises(ops.KernelError, match="apart"):
        call(st, torch.full((2, 8 * 64), 7.0, dtype=dtype, device="cuda"))


def off_16(x, pad=3):
    """The same rows one number into a buffer, an odd number of them apart."""
    buffer = torch.zeros(x.shape[0] * (x.shape[1] + pad) + 1, dtype=x.dtype, device="cuda")
    y = buffer[1:].view(x.shape[0], -1)[:, :x.shape[1]]
    y.copy_(x)
    return y


@pytest.mark.parametrize("dtype,form", [(BF16, None), (F32, None)] + [(BF16, f) for f in ("rows", "columns", "tcgen05", "dense")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("lens,starts", [([1, 1], [60, 2000]), ([5], [900]), ([1, 150], [30, 60]), ([9, 7], [0, 3000])])
def test_queries_off_16_bytes(dtype, form, d, page, lens, starts, monkeypatch):
    monkeypatch.setattr(ops, "E4M3_FORMS", form and (form, form))
    st = Step(lens, starts, 8, 2, d, page, dtype, seed=4)
    st.q = off_16(st.q)
    out = call(st, torch.full((sum(lens), 8 * d), 7.0, dtype=dtype, device="cuda"))
    monkeypatch.setattr(ops, "E4M3_FORMS", None)
    st.check(out)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,starts", [([1, 1], [60, 2000]), ([5], [900]), ([1, 150], [30, 60])])
def test_scales_off_16_bytes(dtype, d, lens, starts):
    st = Step(lens, starts, 8, 2, d, 16, dtype, seed=4)
    for name in ("ks", "vs"):
        scale = getattr(st, name).view(torch.uint8)
        buffer = torch.zeros(scale.numel() + 1, dtype=torch.uint8, device="cuda")
        moved = buffer[1:].view(scale.shape)
        moved.copy_(scale)
        setattr(st, name, moved.view(E8M0))
    st.check(call(st, torch.full((sum(lens), 8 * d), 7.0, dtype=dtype, device="cuda")))


@pytest.mark.parametrize("d", [64, 128])
def test_more_rows_than_a_grid_has_places_for(d):
    """A bound of so many tokens that neither the tensor-core kernels, for queries off 16 bytes, nor the one for few rows can take the call."""
    most = 16500
    st = Step([25], [60], 128, 1, d, 16, BF16, seed=3)
    q = torch.zeros(most, 128 * d, dtype=BF16, device="cuda")
    q[:25] = st.q
    st.q = off_16(q, 1)
    out = call(st, torch.full((most, 128 * d), 7.0, dtype=BF16, device="cuda"), max_q_len=most)
    assert (out[25:] == 7).all()
    st.check(out)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_sequences_than_a_grid_has_places_for(dtype):
    S, nq, d = 65537, 2, 64
    st = Step([1], [15], nq, 1, d, 16, dtype, seed=3)                    # all read one page
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(S, nq * d, device="cuda", generator=g).to(dtype)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = torch.arange(S, **i32) % 16 + 1
    out = torch.full((S, nq * d), 7.0, dtype=dtype, device="cuda")
    ops.attention_e4m3(q, out, st.k, st.v, st.ks, st.vs, st.table[:1, :1].expand(S, 1).contiguous(), torch.arange(S + 1, **i32), lens, S, 1, 16,
                       nq, 1, 0, d ** -0.5, st.err)
    k, v = (st.rows_of(0, a, b)[0][0] for a, b in ((st.k, st.ks), (st.v, st.vs)))
    scores = (q.double().view(S, nq, d) @ k.T * d ** -0.5).masked_fill((torch.arange(16, device="cuda") >= lens[:, None])[:, None], float("-inf"))
    w = torch.softmax(scores, -1)
    # float32 products, exponentials and sums over 16 keys, rounded once: see Step.expected
    bound = (2.0 ** -11 if dtype is BF16 else 2.0 ** -17) * (w @ v.abs()) + torch.finfo(dtype).eps / 2 * (w @ v).abs()
    assert int(st.err) == 0 and ((out.double().view(S, nq, d) - w @ v).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [1e-60, 0.0, -0.2])
@pytest.mark.parametrize("lens,starts", [([1, 1], [60, 2000]), ([150], [20]), ([1, 5], [900, 30])])
def test_factors_that_are_no_positive_numbers(dtype, scale, lens, starts):
    """1e-60 is 0 in float32: every visible key then weighs the same."""
    st = Step(lens, starts, 8, 2, 64, 16, dtype, seed=6)
    st.check(call(st, torch.full((sum(lens), 8 * 64), 7.0, dtype=dtype, device="cuda"), scale=scale), scale=scale)


@pytest.mark.parametrize("form", [None, "rows", "columns", "tcgen05", "dense"])
def test_one_query_for_all_tokens(form, monkeypatch):
    """Rows that lie 0 apart."""
    monkeypatch.setattr(ops, "E4M3_FORMS", form and (form, form))
    st = Step([3, 150], [40, 60], 8, 2, 64, 16, BF16, seed=4)
    st.q = st.q[:1].expand(153, -1)
    got = call(st, torch.full((153, 8 * 64), 7.0, dtype=BF16, device="cuda"))
    st.q = st.q.contiguous()
    assert torch.equal(got, call(st, torch.full((153, 8 * 64), 7.0, dtype=BF16, device="cuda")))
