"""What the engine sets aside beside a cache kept in 8 bits: the scratch of calls that the run can make; no GPU."""
import pytest
import torch

from conftest import TINY_C
from rllm_b200.cache import page_bytes
from rllm_b200.config import resolve_architecture
from rllm_b200.config.engine_args import EngineArgs
from rllm_b200.engine import engine_core
from rllm_b200.kernels import ops
from rllm_b200.models.decoder import DecoderModel

GiB = 1 << 30


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_run_plans_with_the_scratch_that_its_own_calls_take(dtype, monkeypatch):
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (20 * GiB, 180 * GiB))
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    arch = resolve_architecture(TINY_C)
    model = DecoderModel(arch.build_spec(arch.parse_config(dict(TINY_C, max_position_embeddings=1 << 21))))
    model.dtype = dtype
    args = EngineArgs(max_num_seqs=4096, max_num_batched_tokens=64, gpu_memory_utilization=0.95)
    need, layers = model.layout.groups[0], len(model.layout.owners[0])
    wide = 2 if dtype is torch.bfloat16 else 4
    most = 1 << 21
    plain = engine_core.plan_cache_pages(model, args, most, torch.device("cpu"))[0] * page_bytes(need, 16, wide) * layers
    args.kv_cache_dtype = "fp8"
    narrow = engine_core.plan_cache_pages(model, args, most, torch.device("cpu"))[0] * page_bytes(need, 16, 1, 1) * layers
    forms = {ops.attention_e4m3_form(dtype, 4, 2, 64, page, model.blocks[0].mixer.scale, q, seqs, most) for page in (1, 16)
             for q in (1, 9, 300, most) for seqs in (1, 100)}
    scratch = 4 * most * 2 * 64 if "dense" in forms else 0         # keys and values of one sequence as bfloat16
    assert abs(plain - narrow - scratch) <= (1 << 20) + layers * page_bytes(need, 16, wide)


@pytest.mark.parametrize("dtype,nq,nkv,d,scale", [
    (torch.bfloat16, 32, 8, 64, 0.1), (torch.bfloat16, 32, 8, 128, 0.1), (torch.float32, 32, 8, 64, 0.1), (torch.bfloat16, 32, 8, 96, 0.1),
    (torch.bfloat16, 8, 1, 256, 0.1), (torch.bfloat16, 128, 1, 64, 0.1), (torch.bfloat16, 129, 1, 64, 0.1), (torch.bfloat16, 32, 8, 64, -0.1)])
def test_scratch_is_for_calls_that_the_rule_gives_to_the_dense_form(dtype, nq, nkv, d, scale):
    dense = any(ops.attention_e4m3_form(dtype, nq, nkv, d, page, scale, q, 1, 9000) == "dense" for page in (1, 16) for q in (1, 200, 9000))
    assert (ops.e4m3_dense_scratch(nkv, d, 9000, dtype, nq, scale) > 0) == dense
