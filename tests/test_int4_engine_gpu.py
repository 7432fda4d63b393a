"""A model whose weights and cache are held in 4 bits, through the engine, beside the plain implementation on the values that 4 bits hold."""
import numpy as np
import pytest
import torch

import int4_cases
import plain_qwen3 as plain
from helpers import TINY, TOL, TOL_MODEL_BF16_MEDIAN, make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
GROUP = {"D": 64, "E": 32}
QUANTISED = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    tmp = str(tmp_path_factory.mktemp("models"))
    out = {}
    for name in ("D", "E"):
        folder = make_model_dir(tmp, name)
        out[name] = (folder, *plain.read_model(folder))
    return out


def make_engine(folder, dtype, name, **kw):
    from carbon_engine_b200 import Engine
    args = dict(dtype=dtype, page_size=TINY[name]["page_size"], kv_tokens=2048, max_seq_len=1024, poison_cache=True, int4_group=GROUP[name])
    args.update(kw)
    return Engine(folder, **args)


def held_weights(w, group, dtype):
    """The weights that the engine multiplies with: as stored (rounded to the compute type), then in 4 bits where the width allows."""
    out = {}
    for n, t in w.items():
        if any(f".{q}.weight" in n for q in QUANTISED) and t.shape[1] % group == 0:
            out[n] = int4_cases.held(t.to(dtype), group).to(t.dtype)
        else:
            out[n] = t
    return out


def logits_of(eng, tokens, cuts):
    """Logits of every token, the tokens brought in portions that end at ``cuts``."""
    from carbon_engine_b200.engine.batch import StepEntry
    eng.runner.open_request(1)
    rows, at = [], 0
    for end in cuts:
        rows.append(eng.runner.step([StepEntry(1, tokens[at:end], list(range(end - at)))]).double().cpu())
        eng.runner.check_status()
        at = end
    eng.runner.close_request(1)
    return torch.cat(rows)


@pytest.mark.parametrize("name", ["D", "E"])
def test_weights_in_4_bits_float32(models, name):
    """Portions below and above the tokens that read the codes themselves: the same values either way."""
    folder, cfg, w = models[name]
    eng = make_engine(folder, "float32", name, weight_bits=4)
    tokens = random_tokens(np.random.default_rng(2), 150, cfg["vocab_size"])
    got = logits_of(eng, tokens, [70, 71, 72, 100, 150])
    want = plain.forward(cfg, held_weights(w, GROUP[name], torch.float32), tokens).double()
    assert float((got - want).abs().max()) <= TOL["float32"] * float(want.abs().max())
    # ... and they are not the unquantised model's
    assert float((want - plain.forward(cfg, w, tokens).double()).abs().max()) > 20 * TOL["float32"] * float(want.abs().max())


@pytest.mark.parametrize("name", ["D", "E"])
def test_cache_in_4_bits_float32(models, name, monkeypatch):
    """Keys and values that differ by a rounding may take the code next to theirs, which moves them by a step: the engine has to lie five times
    nearer to the plain implementation on quantised keys and values than the plain implementation without them does (norms of all
    logits; one code in some hundred thousand flips, where quantisation moves all of them)."""
    folder, cfg, w = models[name]
    eng = make_engine(folder, "float32", name, kv_bits=4)
    tokens = random_tokens(np.random.default_rng(3), 90, cfg["vocab_size"])
    exact = plain.forward(cfg, w, tokens).double()
    whole = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, scale, window=0: whole(
        q, int4_cases.held(k, GROUP[name]).to(k.dtype), int4_cases.held(v, GROUP[name]).to(v.dtype), scale, window))
    want = plain.forward(cfg, w, tokens).double()
    for cuts in ([90], [33, 34, 35, 90], list(range(1, 91))):
        got = logits_of(eng, tokens, cuts)
        assert float((got - want).norm()) <= 0.2 * float((exact - want).norm())


@pytest.mark.parametrize("kv_bits,weight_bits", [(4, 16), (4, 4)])
def test_generation_with_graphs_is_generation_without(models, kv_bits, weight_bits):
    """bfloat16: steps replayed as graphs, requests that come and go, portions beside decoding requests."""
    from carbon_engine_b200 import SamplingParams
    folder, cfg, w = models["D"]
    rng = np.random.default_rng(4)
    prompts = [random_tokens(rng, n, cfg["vocab_size"]) for n in (3, 130, 64, 17, 300)]
    outs = []
    for graphs in (False, True):
        eng = make_engine(folder, "bfloat16", "D", kv_bits=kv_bits, weight_bits=weight_bits, cuda_graphs=graphs, max_running_requests=3,
                          max_prefill_tokens=100, run_ahead=graphs)
        outs.append([o.token_ids for o in eng.generate(prompts, SamplingParams(max_tokens=12, ignore_eos=True))])
        assert eng.cuda_graphs == graphs
        eng.storage.manager.check()
    assert all(len(t) == 12 for t in outs[0]) and outs[0] == outs[1]


def test_weights_and_cache_in_4_bits_bfloat16(models, monkeypatch):
    """A key or value rounded to bfloat16 is off by up to 2^-9 of itself, at most 1.5 % of a step (of 2/15 of the group's largest): as many codes
    flip, and move it by a step, 0.12 steps in the mean square where quantisation moves it by 0.29 - less than half.  Beside that, the
    roundings of a bfloat16 model, 2e-2 of the logits."""
    folder, cfg, w = models["D"]
    eng = make_engine(folder, "bfloat16", "D", kv_bits=4, weight_bits=4)
    tokens = random_tokens(np.random.default_rng(5), 120, cfg["vocab_size"])
    held = held_weights(w, 64, torch.bfloat16)
    exact = plain.forward(cfg, held, tokens).double()
    whole = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, scale, window=0: whole(
        q, int4_cases.held(k, 64).to(k.dtype), int4_cases.held(v, 64).to(v.dtype), scale, window))
    want = plain.forward(cfg, held, tokens).double()
    got = logits_of(eng, tokens, [100, 101, 120])
    assert float((got - want).norm()) <= 0.5 * float((exact - want).norm()) + TOL_MODEL_BF16_MEDIAN * float(want.norm())


def test_memory_and_sizes(models):
    folder, cfg, w = models["D"]
    a, b = make_engine(folder, "bfloat16", "D"), make_engine(folder, "bfloat16", "D", kv_bits=4, weight_bits=4)
    per = a.storage.bytes_per_token()
    assert b.storage.bytes_per_token() * 16 == per * 4.5 and b._bytes_per_token() == b.storage.bytes_per_token()
    assert all(v.k_pool is None and v.int4 is not None for v in b.storage.paged_views())
    from carbon_engine_b200.engine.engine import linears
    assert all(p.weight is None and p.int4 is not None for p in linears(b.model))


def test_command_line(models, capsys):
    from carbon_engine_b200.cli import main
    folder = models["D"][0]
    assert main(["generate", "--model", folder, "--prompt-ids", "1,2,3", "--max-tokens", "4", "--ignore-eos", "--print-ids", "--kv-tokens", "512",
                 "--kv-bits", "4", "--weight-bits", "4", "--cuda-graphs"]) == 0
    assert capsys.readouterr().out


def test_refusals(models):
    folder = models["D"][0]
    for kw in (dict(kv_bits=4, page_size=8), dict(weight_bits=5), dict(kv_bits=4, int4_group=16)):
        with pytest.raises(ValueError):
            make_engine(folder, "bfloat16", "D", **kw)
