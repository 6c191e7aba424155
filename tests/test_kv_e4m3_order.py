"""Attention over a cache kept in 8 bits directly behind the kernel that makes its lengths: nothing is read ahead of the wait for it
unless the caller says that it may be."""
import re

import pytest
import torch

from kv_e4m3_util import Step
from rllm_b200.kernels import ops
from test_launch_overlap_rules import kernels

BF16, F32 = torch.bfloat16, torch.float32
READERS = {"attention_e4m3_simt_kernel", "attention_e4m3_rows_kernel", "attention_e4m3_columns_kernel", "attention_e4m3_tcgen05_kernel",
           "kv_e4m3_widen_kernel"}


@pytest.mark.parametrize("file,name,params,body", [k for k in kernels() if k[1] in READERS], ids=lambda v: v if len(v) < 60 else "")
def test_lengths_are_read_behind_the_wait(file, name, params, body):
    """By its text: a step's lengths, row ranges and block table are made anew behind a wait before anything is read through them."""
    wait = re.search(r"(?:kv8_inputs|pdl_wait_on)\(([^)]*)\)", body)
    assert wait and {"block_table", "q_start", "seq_lens"} <= set(re.findall(r"\w+", wait.group(1))), f"{file}: {name}"
    assert not re.search(r"\b(?:block_table|q_start|seq_lens|bt)\b", body[:wait.start()]), f"{file}: {name}"


def test_every_reader_was_looked_at():
    assert READERS <= {k[1] for k in kernels()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,form", [(BF16, 64, None), (F32, 64, None), (BF16, 48, None)] + [
    (BF16, d, f) for d in (64, 128) for f in ("rows", "columns", "tcgen05", "dense")])
@pytest.mark.parametrize("ready", [False, True])
def test_directly_behind_the_kernel_that_counts_the_lengths_up(dtype, d, form, ready, monkeypatch):
    """``decode_advance``, then the attention, many times without a stop in between, eagerly and in a captured graph: each result is that
    of the lengths as they are then.  With ``lengths_ready`` the queries' copy stands between the two, as a cache's write would."""
    monkeypatch.setattr(ops, "E4M3_FORMS", form and (form, form))
    for lens in ([40], [5 * i % 61 + 30 for i in range(64)]):
        S, most = len(lens), 24
        st = Step([1] * S, lens, 8, 2, d, 16, dtype, seed=S)
        start = st.seq_lens - most                                 # every result is a prefix's
        token, sampled = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.ones(S, dtype=torch.int32, device="cuda")
        between = torch.empty_like(st.q)

        def run(outs, stop):
            st.seq_lens.copy_(start)
            for out in outs:
                ops.decode_advance(token, st.positions, st.seq_lens, sampled, None)
                if ready:
                    ops.softcap_rows(between.copy_(st.q).float(), 1.0)
                ops.attention_e4m3(st.q, out, st.k, st.v, st.ks, st.vs, st.table, st.q_start, st.seq_lens, S, 1, max(lens) + 1, st.nq, st.nkv, 0,
                                   d ** -0.5, st.err, lengths_ready=ready)
                if stop:
                    torch.cuda.synchronize()

        want = [torch.empty(S, 8 * d, dtype=dtype, device="cuda") for _ in range(most)]
        run(want, True)
        st.totals = [n + 1 for n in lens]
        st.check(want[-1])
        assert not any(torch.equal(a, b) for a, b in zip(want, want[1:]))
        outs = [torch.full_like(w, 7.0) for w in want]
        for _ in range(4):
            run(outs, False)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(outs, False)
        for _ in range(4):
            for out in outs:
                out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)) and int(st.err) == 0
