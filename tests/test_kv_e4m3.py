"""What the operators over a cache kept in 8 bits refuse before anything is launched; no GPU."""
import pytest
import torch

from kv_e4m3_util import E4M3, E8M0, quantise, to_e4m3
from rllm_b200.kernels import ops

BF16 = torch.bfloat16


def cache(pages=3, nkv=2, page=16, d=64):
    code = lambda: torch.zeros(pages, nkv, page, d, dtype=torch.uint8).view(E4M3)  # noqa: E731
    scale = lambda: torch.zeros(pages, nkv, page, dtype=torch.uint8).view(E8M0)  # noqa: E731
    return [code(), code(), scale(), scale()]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def write(c=None, **over):
    a = dict(qkv=torch.zeros(2, 8 * 64, dtype=BF16), positions=i32(0, 1), token_seq=i32(0, 0), inv_freq=torch.zeros(32, dtype=torch.float64),
             rotary_dim=64, block_table=i32(0, 1).view(1, 2), nq=4, nkv=2, d=64, err=i32(0), q_out=None)
    a.update(over)
    k, v, ks, vs = c or cache()
    ops.rope_kv_write_e4m3(a["qkv"], a["positions"], a["token_seq"], a["inv_freq"], a["rotary_dim"], a["block_table"], k, v, ks, vs,
                           a["nq"], a["nkv"], a["d"], a["err"], q_out=a["q_out"])


def attend(c=None, **over):
    a = dict(q=torch.zeros(2, 4 * 64, dtype=BF16), out=torch.zeros(2, 4 * 64, dtype=BF16), table=i32(0, 1).view(1, 2), q_start=i32(0, 2),
             seq_lens=i32(20), nd=0, mq=2, ms=20, nq=4, nkv=2, window=0, scale=0.125, err=i32(0))
    a.update(over)
    ops.attention_e4m3(a["q"], a["out"], *(c or cache()), a["table"], a["q_start"], a["seq_lens"], a["nd"], a["mq"], a["ms"], a["nq"],
                       a["nkv"], a["window"], a["scale"], a["err"])


@pytest.mark.parametrize("over", [
    dict(qkv=torch.zeros(2, 7 * 64, dtype=BF16)), dict(qkv=torch.zeros(2, 8 * 64, dtype=torch.float16)), dict(positions=i32(0)),
    dict(token_seq=torch.zeros(2, dtype=torch.int64)), dict(inv_freq=None), dict(inv_freq=torch.zeros(32)),
    dict(inv_freq=torch.zeros(16, dtype=torch.float64)), dict(q_out=torch.zeros(2, 4 * 64)), dict(q_out=torch.zeros(3, 4 * 64, dtype=BF16)),
    dict(qkv=torch.zeros(8 * 64, 2, dtype=BF16).t()), dict(block_table=i32(0, 1)), dict(nkv=1, qkv=torch.zeros(2, 6 * 64, dtype=BF16)),
    dict(d=32, qkv=torch.zeros(2, 8 * 32, dtype=BF16))])
def test_a_write_that_does_not_fit(over):
    with pytest.raises(ops.KernelError):
        write(**over)


@pytest.mark.parametrize("over", [
    dict(q=torch.zeros(2, 4 * 64)), dict(q=torch.zeros(2, 3 * 64, dtype=BF16)), dict(q=torch.zeros(1, 4 * 64, dtype=BF16)),
    dict(q=torch.zeros(4 * 64, 2, dtype=BF16).t()), dict(out=torch.zeros(2, 8 * 64, dtype=BF16)[:, ::2]),
    dict(q=torch.zeros(2, 4 * 64, dtype=torch.float16), out=torch.zeros(2, 4 * 64, dtype=torch.float16)),
    dict(q_start=i32(0, 1, 2)), dict(seq_lens=torch.zeros(1, dtype=torch.int64)), dict(nd=2), dict(nd=-1), dict(ms=33), dict(mq=-1),
    dict(nkv=4), dict(table=torch.zeros(0, 2, dtype=torch.int32)), dict(table=i32(0, 9, 1, 9).view(1, 4)[:, ::2])])
def test_an_attention_that_does_not_fit(over):
    with pytest.raises(ops.KernelError):
        attend(**over)


def test_a_cache_of_another_kind():
    for at, bad in ((0, torch.zeros(3, 2, 16, 64, dtype=BF16)), (1, torch.zeros(3, 2, 16, 32, dtype=torch.uint8).view(E4M3)),
                    (2, torch.zeros(3, 2, 16)), (3, torch.zeros(3, 2, 8, dtype=torch.uint8).view(E8M0)),
                    (0, torch.zeros(3, 16, 2, 64, dtype=torch.uint8).view(E4M3).transpose(1, 2))):
        c = cache()
        c[at] = bad
        with pytest.raises(ops.KernelError):
            write(c)
        with pytest.raises(ops.KernelError):
            attend(c)
        out = [torch.zeros(2, 2 * 64, dtype=BF16) for _ in range(2)]
        with pytest.raises(ops.KernelError):
            ops.kv_read_e4m3(i32(0, 1), i32(0, 0), i32(0, 1).view(1, 2), *c, *out, i32(0))


def test_a_reading_that_does_not_fit():
    good = [torch.zeros(2, 2 * 64, dtype=BF16) for _ in range(2)]
    for pos, seq, outs in ((i32(0, 1), i32(0), good), (i32(0, 1), i32(0, 0), [good[0], good[1].float()]),
                           (i32(0, 1), i32(0, 0), [good[0][:, :64], good[1]]), (i32(0, 1), i32(0, 0), [g.half() for g in good])):
        with pytest.raises(ops.KernelError):
            ops.kv_read_e4m3(pos, seq, i32(0, 1).view(1, 2), *cache(), *outs, i32(0))


def test_there_is_no_cpu_path():
    with pytest.raises(ops.KernelError, match="CUDA"):
        write()
    with pytest.raises(ops.KernelError, match="CUDA"):
        attend()


def test_the_tests_own_rounding():
    """to_e4m3 against every number of the type and the middles between neighbours."""
    all_ = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).to(torch.float64)          # 0 .. 448 ascending
    assert torch.equal(to_e4m3(all_), all_) and all_[-1] == 448
    mid = (all_[1:] + all_[:-1]) / 2
    even = torch.where(torch.arange(126) % 2 == 0, all_[:-1], all_[1:])
    assert torch.equal(to_e4m3(mid), even) and torch.equal(to_e4m3(-mid), -even)
    assert torch.equal(to_e4m3(mid * (1 + 1e-12)), all_[1:]) and torch.equal(to_e4m3(mid * (1 - 1e-12)), all_[:-1])
    c, b = quantise(torch.tensor([[448.0, 1.0], [448.0001, 1.0], [0.0, 0.0], [float("nan"), 1.0], [2.0 ** -140, 0.0]], dtype=torch.float64))
    assert b.tolist() == [127, 128, 0, 255, 0] and c[0].tolist() == [448.0, 1.0] and c[3].tolist() == [0.0, 0.0]


@pytest.mark.parametrize("dtype,nq,nkv,d,page,scale,q,seqs,keys,form", [
    (BF16, 32, 8, 64, 16, 0.1, 1, 64, 9000, "columns"), (BF16, 32, 8, 64, 16, 0.1, 8, 64, 9000, "columns"), (BF16, 32, 8, 64, 16, 0.1, 9, 8, 9000, "tcgen05"),
    (BF16, 32, 8, 64, 16, 0.1, 1, 64, 767, "rows"), (BF16, 32, 8, 64, 16, 0.1, 1, 64, 768, "columns"), (BF16, 32, 8, 64, 16, 0.1, 1, 1, 8191, "rows"),
    (BF16, 32, 8, 64, 16, 0.1, 1, 1, 8192, "columns"), (BF16, 32, 8, 128, 16, 0.1, 1, 1, 2048, "columns"), (BF16, 32, 8, 128, 16, 0.1, 1, 1, 2047, "rows"),
    (BF16, 32, 8, 64, 16, 0.1, 32, 1, 9000, "rows"), (BF16, 32, 8, 64, 16, 0.1, 33, 1, 9000, "tcgen05"), (BF16, 32, 8, 128, 16, 0.1, 6, 8, 9000, "columns"),
    (BF16, 32, 8, 128, 16, 0.1, 8, 8, 9000, "columns"), (BF16, 32, 8, 128, 16, 0.1, 9, 8, 9000, "tcgen05"), (BF16, 32, 8, 128, 16, 0.1, 32, 1, 4000, "columns"),
    (BF16, 32, 8, 128, 16, 0.1, 33, 1, 4000, "tcgen05"), (BF16, 32, 8, 128, 16, 0.1, 12, 1, 700, "rows"), (BF16, 32, 8, 128, 16, -0.1, 6, 8, 9000, "columns"),
    (BF16, 32, 8, 64, 16, 0.1, 128, 1, 128, "tcgen05"), (BF16, 32, 8, 64, 16, 0.1, 129, 1, 129, "dense"), (BF16, 8, 8, 128, 16, 0.1, 513, 2, 600, "dense"),
    (BF16, 32, 8, 64, 8, 0.1, 1, 1, 100, "tcgen05"), (BF16, 32, 8, 64, 16, -0.1, 200, 1, 200, "rows"), (BF16, 32, 8, 96, 16, 0.1, 1, 1, 100, "simt"),
    (BF16, 32, 8, 64, 8, 0.1, 1, 64, 9000, "tcgen05"), (BF16, 200, 1, 64, 16, 0.1, 1, 1, 100, "rows"), (torch.float32, 32, 8, 64, 16, 0.1, 1, 64, 9000, "rows"),
    (torch.float32, 32, 8, 64, 16, 0.1, 300, 1, 300, "rows"), (torch.float32, 32, 8, 64, 8, 0.1, 3, 1, 300, "simt"),
    (BF16, 8, 1, 256, 32, 0.1, 300, 1, 300, "rows"), (BF16, 8, 1, 256, 32, 0.1, 1, 64, 9000, "rows")])
def test_which_kernel_a_call_takes(dtype, nq, nkv, d, page, scale, q, seqs, keys, form, monkeypatch):
    assert ops.attention_e4m3_form(dtype, nq, nkv, d, page, scale, q, seqs, keys) == form
    monkeypatch.setenv("RLLM_ATTENTION", "mma")
    assert ops.attention_e4m3_form(dtype, nq, nkv, d, page, scale, q, seqs, keys) in ("rows", "simt")
    monkeypatch.setenv("RLLM_ATTENTION", "simt")
    assert ops.attention_e4m3_form(dtype, nq, nkv, d, page, scale, q, seqs, keys) == "simt"
