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
