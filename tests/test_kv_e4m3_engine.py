"""A cache kept in 8 bits as the engine sees it: the option, what it refuses, pages and bytes, copies for forks; no GPU."""
import pytest
import torch

from conftest import TINY_C
from kv_e4m3_util import E4M3, E8M0
from rllm_b200.cache import CacheStorage, page_bytes
from rllm_b200.config import ConfigError, resolve_architecture
from rllm_b200.config.engine_args import EngineArgs
from rllm_b200.engine import engine_core
from rllm_b200.engine.replay import build_parser as replay_parser
from rllm_b200.cli import build_parser
from rllm_b200.models.decoder import CacheLayout, DecoderModel
from rllm_b200.parts.spec import KVPagesNeed, StateNeed


def model_of(config):
    arch = resolve_architecture(config)
    return DecoderModel(arch.build_spec(arch.parse_config(config)))


def test_the_option():
    assert not EngineArgs().cache_in_8_bits and EngineArgs(kv_cache_dtype="fp8").cache_in_8_bits
    assert EngineArgs(kv_cache_dtype="fp8_e4m3").cache_in_8_bits
    for bad in ("int8", "fp8_e5m2", ""):
        with pytest.raises(ConfigError, match="kv_cache_dtype"):
            EngineArgs(kv_cache_dtype=bad).validate()
    EngineArgs(kv_cache_dtype="fp8").validate()
    assert build_parser().parse_args(["generate", "x", "--kv-cache-dtype", "fp8"]).kv_cache_dtype == "fp8"
    a = replay_parser().parse_args(["--model", "x", "--dtype", "float32", "--out", "y", "--max-tokens", "9", "--kv-cache-dtype", "fp8_e4m3"])
    assert a.kv_cache_dtype == "fp8_e4m3"


def test_which_models_take_it():
    model_of(TINY_C).check_8_bit_cache()
    from fasulix_util import FX_A
    from munupel_util import MU_A
    for config in (FX_A, MU_A):
        with pytest.raises(ConfigError, match="kv_cache_dtype fp8_e4m3: layer"):
            model_of(config).check_8_bit_cache()


def test_pages_scales_and_copies():
    need = KVPagesNeed(2, 64)
    assert page_bytes(need, 16, 1, 1) == 2 * 16 * 2 * 65 and page_bytes(need, 16, 2) == 2 * 16 * 2 * 128
    st = CacheStorage(CacheLayout([need, StateNeed((3,))], [[0], [1]], [0, 1], [0, 1]), 16, [5], 2, torch.bfloat16, torch.device("cpu"), e4m3=True)
    view = st.view(0)
    assert view.k.shape == (6, 2, 16, 64) and view.k.dtype is E4M3 and view.v.dtype is E4M3
    assert view.k_scale.shape == (6, 2, 16) and view.k_scale.dtype is E8M0 and view.v_scale.dtype is E8M0
    assert st.num_bytes() == 6 * page_bytes(need, 16, 1, 1) + 3 * 3 * 4
    for i, t in enumerate((view.k, view.v, view.k_scale, view.v_scale)):
        t.view(torch.uint8)[1] = 17 + i
    st.copy_for_fork([(0, 1, 4)], (0, 1))
    for i, t in enumerate((view.k, view.v, view.k_scale, view.v_scale)):
        assert (t.view(torch.uint8)[4] == 17 + i).all() and (t.view(torch.uint8)[3] == 0).all()
    with pytest.raises(ValueError, match="no 8-bit form"):
        CacheStorage(CacheLayout([KVPagesNeed(1, 64, values=False)], [[0]], [0], [0]), 16, [5], 2, torch.bfloat16, torch.device("cpu"), e4m3=True)
    plain = CacheStorage(CacheLayout([need], [[0]], [0], [0]), 16, [5], 2, torch.bfloat16, torch.device("cpu"))
    assert plain.view(0).k_scale is None
    with pytest.raises(ValueError, match="no pages in 8 bits"):
        plain.read_tokens(0, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_pages_are_planned_with_what_a_step_takes(monkeypatch):
    from rllm_b200.kernels import ops
    GiB = 1 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (20 * GiB, 180 * GiB))
    monkeypatch.setattr(torch.cuda, "empty_cache", lambda: None)
    model = model_of(dict(TINY_C, max_position_embeddings=1 << 20))
    model.dtype = torch.bfloat16
    args = EngineArgs(max_num_seqs=4096, max_num_batched_tokens=64, gpu_memory_utilization=0.95)
    plain = engine_core.plan_cache_pages(model, args, 1 << 20, torch.device("cpu"))
    args.kv_cache_dtype = "fp8"
    narrow = engine_core.plan_cache_pages(model, args, 1 << 20, torch.device("cpu"))
    need = model.layout.groups[0]
    layers = len(model.layout.owners[0])
    scratch = ops.e4m3_dense_scratch(2, 64, 1 << 20)
    assert scratch >= 4 * (1 << 20) * 2 * 64
    left = plain[0] * page_bytes(need, 16, 2) * layers - narrow[0] * page_bytes(need, 16, 1, 1) * layers
    assert abs(left - scratch) <= 2 * layers * page_bytes(need, 16, 2)
    assert narrow[0] > 1.85 * plain[0]
