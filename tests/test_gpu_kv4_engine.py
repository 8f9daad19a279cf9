"""The engine with a 4-bit cache, a step's tables, scores of tokens: through the public entry points (needs a B200)."""
import json

import numpy as np
import pytest
import torch

import plain_kv4 as pk
import plain_model as pm
import questwend_b200 as qw
from helpers import BF16_TOL, FP32_TOL, TINY, make_folder
from questwend_b200 import cli
from questwend_b200.cache.manager import CacheManager
from questwend_b200.engine.engine import EngineError, StepEntry, build_step_context
from questwend_b200.parts.base import KVSpec
from questwend_b200.sampling import GREEDY, SamplingParams

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {(name, dtype): make_folder(tmp_path_factory.mktemp(f"{name}_{dtype}"), TINY[name][0], TINY[name][1], dtype)
            for name in "BCD" for dtype in ("float32", "bfloat16")}


def tol(dtype):
    return FP32_TOL if dtype == "float32" else BF16_TOL


def cached(engine, slot):
    """Keys and values of a slot's tokens, layer by layer, as the cache's bytes say, and the steps of their groups."""
    g = engine.cache._groups[0]
    n, pages, out = engine.cache.length(slot), g.pages[slot], []
    for unit in range(len(g.units)):
        raw = g.k[unit][pages].cpu().numpy()
        flat = lambda x: x.transpose(0, 2, 1, 3).reshape(-1, g.spec.n_kv_heads, x.shape[3])[:n]
        kc, kw, vc, vw = pk.unpack(raw, g.spec.head_dim)
        steps = [np.repeat(((flat(w).astype(np.uint32) & 0xFFF0) << 16).view(np.float32), 32, -1).astype(np.float64) for w in (kw, vw)]
        out.append((flat(pk.stands_for(kc, kw)), flat(pk.stands_for(vc, vw)), *steps))
    return out


def logits_over(cfg, w, tokens, held, dtype):
    """The model's logits with each layer's attention reading these keys and values; what the layer itself gives is within a step
    of them (half a step, or where the 16 numbers end a little more)."""
    r16 = pm.round_bf16 if dtype == "bfloat16" else (lambda a: a)
    T, eps, hd = len(tokens), cfg["rms_norm_eps"], cfg["head_dim"]
    Hq, Hkv = cfg["num_attention_heads"], cfg["num_key_value_heads"]
    h = pm.embed(w["model.embed_tokens.weight"], tokens)
    angles = pm.rope_angles(np.arange(T), hd, cfg["rope_theta"])
    for i, (k, v, ks, vs) in enumerate(held):
        px = f"model.layers.{i}."
        x = r16(pm.rms_norm(h, w[px + "input_layernorm.weight"], eps))
        proj = lambda n, heads: pm.linear(x, w[f"{px}self_attn.{n}_proj.weight"]).reshape(T, heads, hd)
        q = r16(pm.apply_rope_neox(pm.rms_norm(proj("q", Hq), w[px + "self_attn.q_norm.weight"], eps), angles, hd))
        own = pm.apply_rope_neox(pm.rms_norm(proj("k", Hkv), w[px + "self_attn.k_norm.weight"], eps), angles, hd)
        slack = 2 * tol(dtype) * np.abs(own).max()
        assert (np.abs(own - k) <= 1.5 * ks + slack).all() and (np.abs(proj("v", Hkv) - v) <= 1.5 * vs + slack).all()
        att = r16(pm.attention_causal(q, k, v).reshape(T, Hq * hd))
        h = h + pm.linear(att, w[px + "self_attn.o_proj.weight"])
        x = r16(pm.rms_norm(h, w[px + "post_attention_layernorm.weight"], eps))
        a = pm.swiglu(pm.linear(x, w[px + "mlp.gate_proj.weight"]), pm.linear(x, w[px + "mlp.up_proj.weight"]))
        h = h + pm.linear(r16(a), w[px + "mlp.down_proj.weight"])
    x = r16(pm.rms_norm(h, w["model.norm.weight"], eps))
    return pm.linear(x, w.get("lm_head.weight", w["model.embed_tokens.weight"]))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "C", "D"])
@pytest.mark.parametrize("pieces", [[130], [1] * 70, [64, 64, 1, 1, 40], [3, 90, 1, 5, 1]])
def test_logits_over_the_cache_that_the_engine_keeps(folders, name, dtype, pieces):
    cfg, w = pm.read_model_folder(folders[name, dtype])
    eng = qw.Engine.from_folder(folders[name, dtype], dtype=dtype, max_tokens=512, cache_bits=4)
    rng = np.random.default_rng(sum(pieces))
    seqs = [rng.integers(0, cfg["vocab_size"], sum(pieces)).tolist() for _ in range(2)]
    eng.close_sequences(eng.open_sequences(1))
    slots = eng.open_sequences(2)
    rows, at = [[], []], 0
    for n in pieces:                                       # the second sequence comes in the same pieces, but one token later
        entries = [StepEntry(slots[0], seqs[0][at:at + n], list(range(n)))]
        lo, hi = max(0, at - 1), at + n - 1
        if hi > lo:
            entries.append(StepEntry(slots[1], seqs[1][lo:hi], list(range(hi - lo))))
        got = eng.step(entries).cpu().numpy()
        rows[0].append(got[:n])
        rows[1].append(got[n:])
        at += n
    for b, seq in ((0, seqs[0]), (1, seqs[1][:-1])):
        ref = logits_over(cfg, w, seq, cached(eng, slots[b]), dtype)
        err = np.abs(np.concatenate(rows[b]) - ref).max(axis=1) / np.abs(ref).max()
        assert err.max() < tol(dtype), (b, int(np.argmax(err)), err.max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_4_bit_cache_is_near_the_other(folders, dtype):
    """Not a tolerance of the kernels: rows off by 2 % of their size move logits by a few per cent, not more than the logits' size."""
    folder = folders["D", dtype]
    toks = np.random.default_rng(1).integers(0, TINY["D"][0]["vocab_size"], 200).tolist()
    out, held = [], []
    for bits in (0, 4):
        eng = qw.Engine.from_folder(folder, dtype=dtype, max_tokens=256, cache_bits=bits)
        (s,) = eng.open_sequences(1)
        out.append(eng.step([StepEntry(s, toks, [199])]).cpu().numpy())
        held.append(eng.describe()["cache_bytes"])
    assert held[0] / held[1] == (2 if dtype == "bfloat16" else 4) * 16 / 9
    assert 0 < np.abs(out[0] - out[1]).max() < 0.5 * np.abs(out[0]).max()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("sampling", [GREEDY, SamplingParams(temperature=0.9, top_k=20, seed=5, repeat_penalty=1.3, repeat_last_n=8)])
def test_generation_with_scores_from_graphs_and_plain_steps(folders, dtype, bits, sampling):
    eng = qw.Engine.from_folder(folders["C", dtype], dtype=dtype, max_tokens=1024, cache_bits=bits)
    prompts = [[1, 2, 3], list(range(70)), [9] * 20, [4]]
    runs = [qw.generate(eng, prompts, max_new_tokens=12, sampling=sampling, ignore_eos=True, use_graph=g, logprobs=4) for g in (True, False, True)]
    for a, b in zip(runs[0], runs[1]):
        assert a.tokens == b.tokens and a.scores == b.scores and len(a.scores) == 12
    assert [r.scores for r in runs[0]] == [r.scores for r in runs[2]]                       # pages used before
    without = qw.generate(eng, prompts, max_new_tokens=12, sampling=sampling, ignore_eos=True)
    assert [r.tokens for r in without] == [r.tokens for r in runs[0]] and without[0].scores == []
    for r in runs[0]:
        for t, s in zip(r.tokens, r.scores):
            assert s.token == t and len(s.top) == 4 and s.logprob <= 0 < s.entropy
            assert list(s.top) == sorted(s.top, key=lambda x: (-x[1], x[0]))
            if sampling.greedy:
                assert s.top[0] == (t, s.logprob)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_of_sequences(folders, dtype):
    """Against log probabilities of the plain model; whatever pieces the sequences run in."""
    folder = folders["D", dtype]
    cfg, w = pm.read_model_folder(folder)
    eng = qw.Engine.from_folder(folder, dtype=dtype, max_tokens=512, max_batch=3)
    rng = np.random.default_rng(7)
    seqs = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in (40, 1, 2, 90, 7, 30)]
    free = eng.cache.free_pages()
    for max_rows in (2048, 33, 1 if dtype == "float32" else 50):
        got = qw.score(eng, seqs, top=3, max_rows=max_rows)
        assert [len(g) for g in got] == [len(s) - 1 for s in seqs]
        for s, g in zip(seqs, got):
            if len(s) < 2:
                continue
            ref = pm.forward_logits(cfg, w, s, round16=None if dtype == "float32" else "bf16")
            lp, H, ids, lps, _, _ = pk.logprobs(ref[:-1], s[1:], 3)
            lim = 2 * tol(dtype) * np.abs(ref).max()         # a logit and the logarithm of the sum are off by a logit's tolerance each
            assert (np.abs(np.array([x.logprob for x in g]) - lp) <= lim).all() and [x.token for x in g] == s[1:]
            assert (np.abs(np.array([[p for _, p in x.top] for x in g]) - lps) <= lim).all()
            # dH = sum p |d lp| (1 + |lp|)
            assert (np.abs(np.array([x.entropy for x in g]) - H) <= lim * (1 + H)).all()
    assert eng.cache.free_pages() == free and eng.cache.slots.n_free == 3
    with pytest.raises(ValueError):
        qw.score(eng, [[1, 10 ** 6]])


def test_scores_with_the_4_bit_cache_match_its_logits(folders):
    eng = qw.Engine.from_folder(folders["D", "bfloat16"], max_tokens=512, cache_bits=4)
    seq = np.random.default_rng(8).integers(0, eng.vocab_size, 100).tolist()
    (got,) = qw.score(eng, [seq], top=2)
    (s,) = eng.open_sequences(1)
    logits = eng.step([StepEntry(s, seq[:-1], list(range(99)))]).double().cpu().numpy()
    lp, _, ids, _, _, _ = pk.logprobs(logits, seq[1:], 2)
    assert np.abs(np.array([x.logprob for x in got]) - lp).max() < 1e-5                     # the same kernels: the same logits
    assert [[i for i, _ in x.top] for x in got] == ids.tolist()


@pytest.mark.parametrize("lens,new", [([0, 0, 0], [1, 1, 1]), ([70, 0, 63], [3, 200, 1]), ([130], [1])])
def test_a_steps_context_is_what_the_lengths_say(lens, new):
    specs = [KVSpec(1, 64), KVSpec(2, 32, stride=4), KVSpec(1, 32, bits=4)]
    cache = CacheManager([(tuple(specs), None, None)], 2000, 5, 1000, torch.bfloat16, "cuda:0")
    spare = cache.open(1)
    cache.reserve({spare[0]: 100})
    slots = cache.open(len(lens))
    for s, n in zip(slots, lens):
        if n:
            cache.reserve({s: n})
            cache.advance(s, n)
    cache.close(spare)
    ctx, want = build_step_context(cache, [StepEntry(s, list(range(n)), [n - 1]) for s, n in zip(slots, new)], 1000, "cuda:0")
    cu = np.concatenate([[0], np.cumsum(new)])
    assert ctx.token_ids.tolist() == [t for n in new for t in range(n)] and ctx.cu_seqlens.tolist() == cu.tolist()
    assert ctx.tok_seq.tolist() == np.repeat(np.arange(len(new)), new).tolist()
    assert ctx.tok_pos.tolist() == [p + i for p, n in zip(lens, new) for i in range(n)]
    assert ctx.pos0.tolist() == lens and ctx.seq_len.tolist() == [a + b for a, b in zip(lens, new)] and ctx.slots.tolist() == slots
    assert want.tolist() == (cu[1:] - 1).tolist()
    assert (ctx.max_new, ctx.min_new, ctx.max_len) == (max(new), min(new), max(a + b for a, b in zip(lens, new)))
    assert ctx.single_token == all(n == 1 for n in new) and ctx.all_start == (not any(lens)) and ctx.host_slots == slots
    for g in range(3):
        assert (ctx.page_tables[g].cpu().numpy() == cache.page_table_host(g, slots)).all()
    pages = cache.page_lists(2, slots)
    assert ctx.tables[2].slot_map.tolist() == [pages[b][(lens[b] + i) // 64] * 64 + (lens[b] + i) % 64 for b in range(len(new)) for i in range(new[b])]
    assert ctx.tables[2].pages.tolist() == [p for row in pages for p in row]


def test_a_truncated_sequence_goes_on(folders):
    eng = qw.Engine.from_folder(folders["D", "bfloat16"], max_tokens=512, cache_bits=4)
    toks = np.random.default_rng(2).integers(0, eng.vocab_size, 100).tolist()
    a, b = eng.open_sequences(2)
    eng.step([StepEntry(a, toks[:80], [])])
    eng.step([StepEntry(a, [1] * 30, [])])
    eng.cache.truncate(a, 80)
    eng.step([StepEntry(b, toks[:80], [])])
    la = eng.step([StepEntry(a, toks[80:], [19])])
    lb = eng.step([StepEntry(b, toks[80:], [19])])
    assert torch.equal(la, lb)


def test_refused_engines(folders):
    with pytest.raises(EngineError, match="cache_bits"):
        qw.Engine.from_folder(folders["B", "float32"], dtype="float32", max_tokens=64, cache_bits=2)


def test_the_command_line(folders, capsys):
    folder = folders["D", "bfloat16"]
    args = ["-m", folder, "-p", "1 2 3 4", "-n", "5", "--n-ctx", "64", "--ignore-eos", "--cache-bits", "4"]
    assert cli.main(args) == 0
    (ids,) = capsys.readouterr().out.strip().splitlines()
    assert cli.main(args + ["--logprobs", "2"]) == 0
    again, scores = capsys.readouterr().out.strip().splitlines()
    assert again == ids and [str(s["token"]) for s in json.loads(scores)] == ids.split() and all(len(s["top"]) == 2 for s in json.loads(scores))
    assert cli.main(args + ["--score", "1"]) == 0
    assert [s["token"] for s in json.loads(capsys.readouterr().out)] == [2, 3, 4]
