"""Many continuations of one prompt on the GPU: draws from one row, forked requests whose steps attend to the shared
positions once for all, and draws from given numbers."""

import pytest
import torch

from tests import draw_plain
from tests.plain import qwen2_plain as plain
from tests.tiny import random_tokens

pytestmark = pytest.mark.gpu

SIZES = dict(architectures=["Qwen2ForCausalLM"], model_type="qwen2", num_hidden_layers=2, hidden_size=256, intermediate_size=384,
             vocab_size=700, rope_theta=1000000.0, rms_norm_eps=1e-6, tie_word_embeddings=True, max_position_embeddings=1024,
             use_sliding_window=False, hidden_act="silu")
HEADS = {64: dict(num_attention_heads=4, num_key_value_heads=2, head_dim=64),
         128: dict(num_attention_heads=7, num_key_value_heads=1, head_dim=128)}


@pytest.fixture(scope="module", params=list(HEADS))
def model(request, tmp_path_factory):
    from somi_inference_b200.config import Qwen2Config
    from somi_inference_b200.weights import write_random_model
    d = write_random_model(Qwen2Config.from_dict(SIZES | HEADS[request.param]), 5, str(tmp_path_factory.mktemp("fork") / "m"),
                           dtype=torch.float32, std=0.08)
    cfg, w = plain.load_folder(d)
    # the weights that an engine of bfloat16 holds, so that what differs is the step's own rounding
    return d, cfg, w, {k: v.bfloat16().float() for k, v in w.items()}


def engine(d, dtype="bfloat16", saves=1):
    from somi_inference_b200 import Engine
    from somi_inference_b200.ops import CudaOps
    ops = CudaOps()
    ops.SHARED_PREFIX_POSITIONS = 0
    ops.SHARED_PREFIX_VALUES = ops.SHARED_PREFIX_VALUES_PORTIONS = saves          # (the tests' prefixes are short)
    calls = []
    inner = ops.shared_prefix_attention
    ops.shared_prefix_attention = lambda *a, **k: calls.append(a) or inner(*a, **k)
    return Engine(d, dtype=dtype, page_size=16, num_pages=200, max_requests=30, ops=ops), ops, calls


def close(got, usual, want):
    """Both steps round the same formula: outside attention at the same places, and in attention both round the
    probabilities and the output to bfloat16 once and hold everything else in 32 bits (the parts of a row are merged in
    32 bits).  So their errors against the plain model are of one size, whatever the model makes of a rounding; they are
    sums over thousands of roundings, which leaves their rms a spread of some percent.  A row that misses a part of its
    keys is off by as much as its logits are large."""
    got, usual = got.float().cpu() - want, usual.float().cpu() - want
    assert got.square().mean().sqrt() <= 1.5 * usual.square().mean().sqrt()
    assert got.abs().max() <= 2 * usual.abs().max() <= 0.1 * want.abs().max()


def test_continuations_of_one_prompt(model):
    from somi_inference_b200 import SamplingParams, StepEntry
    from somi_inference_b200.sampling import Sampler
    d, cfg, _, w = model
    (eng, ops, calls), (usual, usual_ops, usual_calls) = engine(d), engine(d)
    usual_ops.use_shared_prefix = False
    sampler = Sampler(ops, "cuda")
    g = torch.Generator().manual_seed(1)
    n, prompt = 12, random_tokens(333, cfg["vocab_size"], 7)
    sp = SamplingParams(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)
    row = eng.step([StepEntry("prompt", prompt, [len(prompt) - 1])])
    u = torch.rand(1, n, generator=g)
    tokens, prob = sampler.draw(row, [sp], u.cuda())
    want, want_p = draw_plain.draw(row[0].cpu(), u[0], 0.8, 50, float(torch.tensor(0.95)), float(torch.tensor(0.01)))
    assert tokens[0].tolist() == want.tolist() and torch.allclose(prob[0].cpu(), want_p, rtol=2.0 ** -21, atol=0)
    texts = {f"c{i}": prompt + [t] for i, t in enumerate(tokens[0].tolist())}
    usual.step([StepEntry("prompt", prompt, [])])
    for e in (eng, usual):
        assert [e.fork(r, "prompt") for r in texts] == [320] * n
        e.end("prompt")
    todo = {r: t[320:] for r, t in texts.items()}
    for step in range(7):
        logits, other = (e.step([StepEntry(r, t, [len(t) - 1]) for r, t in todo.items()]) for e in (eng, usual))
        # from the second sighting of a layout on, the step is a captured graph; lengths change, the graph does not
        if step in (0, 1, 6):
            close(logits, other, torch.stack([plain.logits(cfg, w, texts[r])[-1] for r in texts]))
        u = torch.rand(n, generator=g)
        drawn, _ = sampler.draw(logits, [sp] * n, u.cuda(), probabilities=False)
        for i, r in enumerate(texts):
            assert int(drawn[i]) == int(draw_plain.draw(logits[i].cpu(), u[i:i + 1], 0.8, 50, float(torch.tensor(0.95)),
                                                        float(torch.tensor(0.01)))[0])
            texts[r] = texts[r] + [int(drawn[i])]
        todo = {r: [t[-1]] for r, t in texts.items()}
    assert len(calls) >= 4 * cfg["num_hidden_layers"]     # (the prompt's rest, an eager and a captured single token)
    assert not usual_calls
    for r in texts:
        eng.end(r)
    eng.cache.check_consistency()
    assert eng.cache.free_pages() == [200]
    ops.check_errors()


def test_short_portions_beside_other_requests(model):
    """Two families, portions of unequal length, single tokens, and a request that shares nothing, in one step."""
    from somi_inference_b200 import StepEntry
    d, cfg, _, w = model
    (eng, ops, calls), (usual, usual_ops, _) = engine(d), engine(d)
    usual_ops.use_shared_prefix = False
    first = {"x": random_tokens(200, cfg["vocab_size"], 11), "y": random_tokens(97, cfg["vocab_size"], 12),
             "z": random_tokens(50, cfg["vocab_size"], 13)}
    for e in (eng, usual):
        e.step([StepEntry(r, t, []) for r, t in first.items()])
    text = dict(first)
    for i, (r, of, more) in enumerate((("x1", "x", 30), ("x2", "x", 1), ("x3", "x", 9), ("y1", "y", 40), ("y2", "y", 2))):
        n = eng.fork(r, of)
        assert usual.fork(r, of) == n
        text[r] = first[of][:n] + random_tokens(more, cfg["vocab_size"], 20 + i)
    for r in first:
        text[r] = first[r] + random_tokens(1, cfg["vocab_size"], 40 + len(r))
    order = ["x1", "x2", "x", "x3", "z", "y1", "y", "y2"]
    entries = [StepEntry(r, text[r][eng.length(r):], [len(text[r]) - eng.length(r) - 1]) for r in order]
    before = len(calls)
    got = eng.step(entries)
    assert len(calls) == before + cfg["num_hidden_layers"]
    close(got, usual.step(entries), torch.stack([plain.logits(cfg, w, text[r])[-1] for r in order]))


def test_steps_that_save_little_and_float32_keep_their_kernels(model):
    from somi_inference_b200 import StepEntry
    d, cfg, w, _ = model
    prompt = random_tokens(64, cfg["vocab_size"], 3)
    for dtype, saves in (("bfloat16", 1 << 30), ("float32", 1)):
        rows = []
        for use in (True, False):
            eng, ops, calls = engine(d, dtype, saves)
            ops.use_shared_prefix = use
            eng.step([StepEntry("p", prompt, [])])
            for r in ("a", "b"):
                eng.fork(r, "p", 48)
            rows.append(eng.step([StepEntry(r, prompt[48:] + [5], [16]) for r in ("a", "b")]).cpu())
            assert not calls
        assert torch.equal(*rows)
        if dtype == "float32":
            assert (rows[0] - plain.logits(cfg, w, prompt + [5])[-1]).abs().max() < 1e-4


def test_generation_with_min_p_does_not_depend_on_the_batch(model):
    from somi_inference_b200 import LLM, SamplingParams
    d, cfg, w, _ = model
    llm = LLM(d, num_blocks=64, block_size=16, max_concurrent=4, dtype="float32")
    prompts = [random_tokens(n, cfg["vocab_size"], 60 + n) for n in (3, 20, 41)]
    sps = [SamplingParams(temperature=0.9, min_p=0.05, seed=1), SamplingParams(temperature=0.9, seed=2),
           SamplingParams(temperature=0.9, min_p=0.2, top_k=40, repetition_penalty=1.2, seed=3)]
    together = llm.generate_many(prompts, max_new_tokens=10, sampling_params=sps, ignore_eos=True)
    for p, sp, out in zip(prompts, sps, together):
        assert llm.generate_many([p], max_new_tokens=10, sampling_params=[sp], ignore_eos=True) == [out]
    # every token was one that min-p keeps
    for p, sp, out in ((prompts[0], sps[0], together[0]),):
        text = list(p)
        for t in out:
            x = plain.logits(cfg, w, text)[-1]
            prob = torch.softmax(x.double() / 0.9, -1)
            assert prob[t] >= 0.05 * prob.max() * (1 - 1e-4)
            text.append(t)
