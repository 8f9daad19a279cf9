"""What an engine with a 4-bit cache refuses before anything is loaded, its cache's bookkeeping, and what the command line says (CPU)."""
import json
import types

import pytest
import torch

from helpers import TINY_A, TINY_D
from questwend_b200 import cli
from questwend_b200.cache.manager import CacheError, CacheManager
from questwend_b200.config.registry import config_from_dict, get_architecture
from questwend_b200.engine import generate, score
from questwend_b200.engine.engine import EngineError, require_cache_bits
from questwend_b200.engine.model import Model
from questwend_b200.kernels import ops
from questwend_b200.parts.base import KVSpec, Runtime
from movudra_helpers import MIXED


def plan_of(cfgd):
    cfg = config_from_dict(cfgd)
    return get_architecture(cfg.architecture).plan(cfg)


def test_a_plan_that_can_and_plans_that_cannot():
    plan = plan_of(TINY_D)
    require_cache_bits(plan, 0)
    require_cache_bits(plan, 4)
    units = Model(plan, Runtime(torch.device("cpu"), torch.bfloat16, 4)).cache_units()
    assert all(kv.bits == 4 for kv, _, _ in units)
    assert all(kv.bits == 0 for kv, _, _ in Model(plan, Runtime(torch.device("cpu"), torch.bfloat16)).cache_units())
    with pytest.raises(EngineError, match="not in 8"):
        require_cache_bits(plan, 8)
    with pytest.raises(EngineError, match="multiple of 32"):
        require_cache_bits(plan_of(TINY_A), 4)                  # heads of 16


def test_a_mixer_that_keeps_its_cache_in_the_engines_dtype_is_refused():
    with pytest.raises(EngineError, match="keeps its cache in the engine's dtype only"):
        require_cache_bits(plan_of(MIXED), 4)


def test_the_cache_in_4_bits():
    spec = KVSpec(2, 64, bits=4)
    c = CacheManager([(spec, None, None), (spec, None, None), (KVSpec(2, 64), None, None)], 200, 4, 200, torch.bfloat16, "cpu")
    assert c.n_groups() == 2 and c.group_spec(0).bits == 4
    u = c.unit_cache(1)
    assert u.k_pool.dtype == torch.uint8 and tuple(u.k_pool.shape) == (4, 2, ops.kv4_page_bytes(64)) and u.v_pool is None
    assert c.unit_cache(2).k_pool.dtype == torch.bfloat16 and c.unit_cache(2).v_pool is not None
    assert c.bytes_held() == 4 * 64 * (2 * spec.token_bytes(2) + KVSpec(2, 64).token_bytes(2))
    slots = c.open(2)
    c.reserve({slots[0]: 130, slots[1]: 1})
    assert [len(p) for p in c.page_lists(0, slots)] == [3, 1]
    for bad in (KVSpec(2, 64, bits=8), KVSpec(2, 64, bits=4, stride=4), KVSpec(2, 64, bits=4, value_dim=32), KVSpec(1, 64, values=False, bits=4)):
        with pytest.raises(CacheError, match="4 bits"):
            CacheManager([(bad, None, None)], 64, 1, 64, torch.bfloat16, "cpu")


def test_info_and_refused_options(tmp_path, capsys):
    cfg = tmp_path / "config.json"
    cfg.write_text(json.dumps(TINY_D))
    sizes = []
    for bits in ("0", "4"):
        assert cli.main(["--random", str(cfg), "--info", "--cache-bits", bits]) == 0
        sizes.append(json.loads(capsys.readouterr().out)["memory"]["cache_bytes_per_token"])
    per_layer = TINY_D["num_key_value_heads"] * TINY_D["head_dim"] * 2
    assert sizes == [2 * per_layer * 2, 2 * per_layer * 9 // 16]
    with pytest.raises(SystemExit, match="--logprobs"):
        cli.main(["--random", str(cfg), "-p", "1", "--logprobs", "-1"])


def test_score_and_generate_refusals():
    engine = types.SimpleNamespace(vocab_size=10, cache=types.SimpleNamespace(max_seq_len=5))
    for seqs, kw, what in [([[1, 2]], {"top": 11}, "top"), ([[1, 2]], {"top": -1}, "top"), ([[1, 2]], {"max_rows": 0}, "max_rows"), ([[]], {}, "empty"),
                           ([[1] * 7], {}, "longest"), ([[1, 10]], {}, "token id"), ([[-1]], {}, "token id")]:
        with pytest.raises(ValueError, match=what):
            score(engine, seqs, **kw)
    with pytest.raises(ValueError, match="logprobs"):
        generate(engine, [[1]], logprobs=65)


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf")])
def test_a_scale_that_the_attention_does_not_take_is_refused_before_a_weight_is_read(scale):
    from questwend_b200.parts.attention import GroupedQueryAttention
    from questwend_b200.parts.base import PartSpec
    spec = PartSpec("gqa", {"hidden_size": 64, "n_heads": 2, "n_kv_heads": 1, "head_dim": 32, "scale": scale}, "layers.0.self_attn.")
    with pytest.raises(ValueError, match="scale above 0"):
        GroupedQueryAttention(spec, Runtime(torch.device("cpu"), torch.bfloat16, 4))
    GroupedQueryAttention(spec, Runtime(torch.device("cpu"), torch.bfloat16))
