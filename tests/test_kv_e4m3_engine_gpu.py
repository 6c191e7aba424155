"""A cache kept in 8 bits under the mixer and the engine on the GPU."""
import pytest
import torch

from conftest import TINY
from kv_e4m3_util import F64, Step, quantise, two_to
from test_engine_gpu import make_llm, prompts_for
from test_parts_gpu import DEV, context_for, load_part

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,page,window", [(64, 16, None), (128, 16, 40), (48, 4, None), (64, 8, 9)])
@pytest.mark.parametrize("entries", [[("a", 1, 70), ("b", 1, 15)], [("a", 1, 33), ("b", 5, 90), ("c", 3, 0)], [("a", 1, 7), ("p", 150, 20), ("r", 40, 0)]])
def test_the_mixer_writes_and_attends(dtype, d, page, window, entries):
    """From a step's projections to the attention's result: the tokens' rows are in the pages as float64 quantises them (up to
    a step where the rotation's rounding decides), and the result is the attention over what the pages hold."""
    from rllm_b200.cache import CacheStorage
    from rllm_b200.models.decoder import CacheLayout
    from rllm_b200.parts import PartSpec, build_part
    hidden, nq, nkv = 96, 6, 2
    spec = PartSpec.of("attention", tensor_names={k: k for k in "qkvo"}, hidden_size=hidden, num_heads=nq, num_kv_heads=nkv, head_dim=d,
                       window=window, position=PartSpec.of("rotary", head_dim=d, rotary_dim=d, theta=5000.0, scaling=None, interleaved=False))
    part = build_part("mixer", spec)
    load_part(part, dtype)
    assert part.no_8_bit_cache() is None
    lens, starts = [e[1] for e in entries], [e[2] for e in entries]
    pages = sum(-(-(n + a) // page) for n, a in zip(lens, starts)) + 4
    storage = CacheStorage(CacheLayout([part.cache_need()], [[0]], [0], [0]), page, [pages], len(entries), dtype, DEV, e4m3=True)
    ctx, cache = context_for([part.cache_need()], page, pages, [(r, [0] * n, a) for r, n, a in entries], dtype)
    view = storage.view(0)
    st = Step(lens, starts, nq, nkv, d, page, dtype, seed=d)      # its rows are what earlier steps left
    n = min(st.k.shape[0], view.k.shape[0])
    for mine, theirs in ((view.k, st.k), (view.v, st.v), (view.k_scale, st.ks), (view.v_scale, st.vs)):
        mine.view(torch.uint8)[:n] = theirs.view(torch.uint8)[:n]
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(ctx.num_tokens, (nq + 2 * nkv) * d, device="cuda", generator=g).to(dtype)
    v_rows = qkv.view(-1, nq + 2 * nkv, d)[:, nq + nkv:].clone()
    out = part.attend(qkv, ctx, view)
    assert int(ctx.err.item()) == 0
    # the attention over what the pages hold now, from the queries as they were rotated in place
    st.q, st.k, st.v, st.ks, st.vs = qkv[:, :nq * d], view.k, view.v, view.k_scale, view.v_scale
    st.table, st.pages, st.device = ctx.block_tables[0], view.k.shape[0], qkv.device
    st.check(out, int(window or 0))
    # the values as they were written
    _, v = storage.read_tokens(0, ctx.block_tables[0], ctx.positions, ctx.token_seq, torch.float32)
    codes, byte = quantise(v_rows)
    assert torch.equal(v.to(F64), codes * two_to(byte.int() - 127)[..., None])


@pytest.mark.parametrize("name,dtype", [("C", "fp32"), ("C", "bf16"), ("D", "fp32"), ("B", "bf16")])
def test_generation_with_graphs_and_without(model_dirs, name, dtype):
    from rllm_b200 import SamplingParams
    prompts = prompts_for(name, [5, 40, 71, 19], 7)
    params = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    outs = []
    for graphs in (True, False):
        llm = make_llm(model_dirs, name, dtype=dtype, kv_cache_dtype="fp8", enable_cuda_graphs=graphs)
        assert llm.engine.storage.e4m3
        outs.append([o.outputs[0].token_ids for o in llm.generate(prompts, params)])
        assert all(len(o) == 12 for o in outs[-1])
        llm.engine.runner.check_errors()
    assert outs[0] == outs[1]


def test_prefixes_that_are_shared_samples_that_fork_and_requests_that_are_preempted(model_dirs):
    """In float32, where a token's row and result do not depend on how its prompt was cut or whom it ran beside."""
    from rllm_b200 import SamplingParams
    prompts = prompts_for("C", [90, 40, 64], 3)
    prompts = [prompts[0], prompts[0][:64] + prompts[1], prompts[2]]
    params = SamplingParams(temperature=0.0, max_tokens=16, ignore_eos=True)
    alone = [make_llm(model_dirs, "C", kv_cache_dtype="fp8").generate([p], params)[0].outputs[0].token_ids for p in prompts]
    together = make_llm(model_dirs, "C", kv_cache_dtype="fp8", max_num_batched_tokens=64, long_prefill_token_threshold=32)
    assert [o.outputs[0].token_ids for o in together.generate(prompts, params)] == alone
    again = together.generate(prompts, params)                    # from the prefix cache
    assert [o.outputs[0].token_ids for o in again] == alone and together.engine.cache.usage()["num_requests"] == 0
    tight = make_llm(model_dirs, "C", kv_cache_dtype="fp8", num_gpu_blocks=17, enable_prefix_caching=False)
    assert [o.outputs[0].token_ids for o in tight.generate(prompts, params)] == alone
    forks = make_llm(model_dirs, "C", kv_cache_dtype="fp8").generate([prompts[0]], SamplingParams(temperature=1e-4, max_tokens=16, ignore_eos=True, n=3, seed=1))
    assert all(c.token_ids == alone[0] for c in forks[0].outputs)


@pytest.mark.parametrize("name", ["C", "B"])
def test_logits_are_near_those_of_the_runs_own_type(model_dirs, name):
    """Rows of 4 significant bits: a key's or value's rounding is 2^-4 of it at most, half that on average in the square; the
    logits of a two- or three-layer model stay within a tenth of their spread, and with a cache of the run's own type they are others."""
    from rllm_b200.engine.loading import load_model
    from rllm_b200.engine.replay import TraceSession
    _, model = load_model(model_dirs[name], dtype="float32")
    prompt = prompts_for(name, [100], 5)[0]
    got = []
    for e4m3 in (False, True):
        session = TraceSession(model, 256, TINY[name][2], 2, e4m3)
        got.append(session.step({"step": 0, "entries": [{"id": "a", "tokens": prompt, "want": list(range(100))}]}).double())
    off = (got[1] - got[0]).norm() / (got[0] - got[0].mean()).norm()
    assert 1e-5 < float(off) < 0.1


def test_models_that_have_no_such_cache_say_so(tmp_path):
    from fasulix_util import FX_A
    from rllm_b200 import LLM
    from rllm_b200.config import ConfigError
    from rllm_b200.engine.loading import write_random_model
    write_random_model(str(tmp_path), FX_A, 0, "float32")
    with pytest.raises(ConfigError, match="kv_cache_dtype"):
        LLM(str(tmp_path), dtype="fp32", kv_cache_dtype="fp8", num_gpu_blocks=64)
