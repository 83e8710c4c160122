"""Engines with 8-bit projections and with adapters on the GPU."""
import pytest
import torch

from gpustack_amd import ops
from gpustack_amd.engine import EngineConfig, LLMEngine, SamplingParams
from test_lora_bank import make, sizes

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]


def engine(**kw):
    cfg = EngineConfig(model="llama-3-8b", device="cuda:0", max_model_len=256,
                       max_num_seqs=8, kv_cache_blocks=128, **kw)
    s = cfg.spec
    s.num_layers, s.hidden_size, s.intermediate_size = 3, 1024, 2048
    s.num_heads, s.num_kv_heads, s.vocab_size = 8, 2, 2048
    return LLMEngine(cfg)


def run(e, prompts, params):
    ids = [e.add_request(p, s) for p, s in zip(prompts, params)]
    got = {i: [] for i in ids}
    while e.has_unfinished():
        for o in e.step():
            got[o.request_id].append(o.token_id)
    return [got[i] for i in ids]


def P(name=None, n=12):
    return SamplingParams(max_tokens=n, ignore_eos=True, lora_name=name)


PROMPTS = [[5, 6, 7, 8, 9] * 9, [100, 3, 50], [1] * 20 + [2]]


def test_hidden_states_stay_near():
    """Embeddings of an 8-bit engine against the same weights' in bf16: an e4m3
    product's terms are off by up to 2^-4 on both sides, at random, so a sum
    of them by far less than an eighth of its size."""
    e = engine(quantize_runtime="fp8", seed=3)
    assert all(l.attn.qkv_pack is not None and l.mlp.down_pack is not None
               for l in e.runner.model.layers)
    got = torch.tensor(e.runner.embed(PROMPTS))
    want = torch.tensor(engine(seed=3).runner.embed(PROMPTS))
    off = (got - want).norm(dim=1) / want.norm(dim=1)
    assert (off > 0).all() and (off < .125).all()


def test_decode_graphs_are_the_eager_steps(monkeypatch):
    """Captured decode steps of an 8-bit engine give an eager engine's tokens."""
    a = run(engine(quantize_runtime="fp8", seed=4), PROMPTS, [P()] * 3)
    monkeypatch.setenv("GPUSTACK_AMD_NO_GRAPHS", "1")
    b = run(engine(quantize_runtime="fp8", seed=4), PROMPTS, [P()] * 3)
    assert a == b and all(len(t) == 12 for t in a)


@pytest.mark.parametrize("quantize", [None, "fp8"])
def test_adapter_rows_beside_others(tmp_path, quantize):
    """Each request of a mixed batch gets the tokens it gets alone, before,
    between and after others come and go."""
    e = engine(quantize_runtime=quantize, seed=5)
    spec = e.runner.cfg.spec
    base = run(e, PROMPTS[:1], [P()])[0]
    for name, r in (("a", 8), ("b", 24), ("c", 5)):
        make(tmp_path / name, spec, ord(name), r, list(sizes(spec)))
        if name != "c":
            e.add_lora(name, str(tmp_path / name))
    calls = []
    own = ops.lora_add
    try:
        ops.lora_add = lambda *a: (calls.append(1), own(*a))[1]
        solo = {n: run(e, PROMPTS[:1], [P(n)])[0] for n in "ab"}
    finally:
        ops.lora_add = own
    assert calls                                  # the kernel, not the library
    assert solo["a"] != solo["b"] and base not in solo.values()
    # prompts of one batch share its products' tiles, not their rows: first
    # tokens agree with those alone wherever the logits are apart
    mixed = run(e, [PROMPTS[0]] * 3, [P("a"), P(), P("b")])
    assert [t[0] for t in mixed] == [solo["a"][0], base[0], solo["b"][0]]
    assert e.remove_lora("a")
    e.add_lora("c", str(tmp_path / "c"))
    assert run(e, PROMPTS[:1], [P("b")])[0] == solo["b"]
    assert run(e, PROMPTS[:1], [P("c")])[0] not in (base, solo["a"], solo["b"])
    assert run(e, PROMPTS[:1], [P()])[0] == base
