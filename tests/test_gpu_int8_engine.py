"""The engine with its layers' products in 8-bit integers, against the plain model with the same rows and matrices in 8 bits (64 bits
otherwise): whole prompts, portions, decoded tokens beside prompts, recorded graphs."""

import pytest
import torch

import plain_model as pm
from helpers import errors, plain_logits, random_ids, weights_for, write_model_dir
from plain_int8 import held_weights
from test_gpu_replay import run_cut
from ullm_b200.csrc import kernels

pytestmark = [pytest.mark.gpu, pytest.mark.needs_cuda]

# An element next to a border goes to the other side where 32 bits (or a 16-bit row in front of it) cannot tell.  One such element is off
# by a step, 1 / 127 of its row's largest, among 64 and more of a product: below 1 / 127 * (largest / rms, 4) / sqrt(64) = 4e-3 of the
# row's results.  float32: a few of them in a run (3e-5 of the elements).  bfloat16: rows rounded to 2^-8 move one element in ten,
# together as much as half a step of noise in each of 12 to 20 products, beside the engine's own tolerance of 4e-2.
TOL = {"float32": 1e-2, "bfloat16": 8e-2, "float16": 2e-2}


def make_runner(tmp_path, tag, dtype, **kw):
    from ullm_b200.engine import ModelRunner

    cfg, w, page = weights_for(tag, dtype)
    d = write_model_dir(str(tmp_path / f"model_{tag}_{dtype}"), cfg, w)
    args = dict(dtype=dtype, page_size=page, num_pages=64, max_requests=4, max_context=cfg["max_position_embeddings"], max_step_tokens=64,
                poison_cache=True, quantization="int8")
    return ModelRunner(d, **{**args, **kw}), cfg, w


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("tag", ["A", "B", "C"])  # C: sizes that are no multiples of 16, a bias, a window
def test_prompts_in_portions(tmp_path, tag, dtype):
    runner, cfg, w = make_runner(tmp_path, tag, dtype)
    n = 60
    ids = random_ids(cfg["vocab_size"], n, 11)
    ref = pm.forward_logits(ids, held_weights(w), cfg)
    for name, cuts in (("whole", [n]), ("cut", [1, 33, 7, 1, 1, 17])):
        mx, _ = errors(run_cut(runner, name, ids, cuts).double(), ref)
        assert mx <= TOL[dtype], f"{name}: {mx:.2e}"
    # (and these are not the products of the weights as they came)
    apart, _ = errors(plain_logits(ids, w, cfg).double(), ref)
    if dtype == "float32":
        assert mx < apart / 3


def test_matrices_are_held_in_8_bits_only(tmp_path):
    runner, cfg, w = make_runner(tmp_path, "B", "bfloat16")
    left = runner.model.all_tensors()
    assert not [n for n in left if n.endswith("_proj.weight")]
    mlp = runner.model.blocks[0].feed_forward
    assert mlp.w_gate_up.q.dtype == torch.int8 and mlp.w_gate_up.shape == (2 * cfg["intermediate_size"], cfg["hidden_size"])


@pytest.mark.parametrize("eager", [True, False])
def test_generation(tmp_path, eager):
    """Greedy tokens under a token budget that cuts prompts, with recorded graphs and without: every token is the plain model's best
    within the tolerance, given the tokens before it."""
    from ullm_b200 import LLM, EngineConfig, SamplingParams

    cfg, w, page = weights_for("B", "bfloat16")
    d = write_model_dir(str(tmp_path / "m"), cfg, w)
    llm = LLM(EngineConfig(model=d, max_bs=4, context_len=256, page_size=page, num_pages=64, max_num_batched_tokens=24,
                           dtype="bfloat16", quantization="int8", enforce_eager=eager))
    prompts = [random_ids(331, n, 70 + n) for n in (1, 7, 33, 64)]
    outs = llm.generate_batch(prompts, SamplingParams(temperature=0.0, max_new_tokens=10, ignore_eos=True))
    held = held_weights(w)
    for p, o in zip(prompts, outs):
        assert len(o.token_ids) == 10
        lg = pm.forward_logits(p + o.token_ids, held, cfg)
        scale = lg.abs().max()
        for i, tok in enumerate(o.token_ids):
            row = lg[len(p) - 1 + i]
            assert row.max() - row[tok] <= 2 * TOL["bfloat16"] * scale
    if not eager:
        assert llm.engine.decode_graphs.replays > 0
    llm.engine.runner.cache.check_invariants()


def test_random_weights_on_the_device(tmp_path):
    """Weights made on the device, at a width whose prompts take pairs of SMs and whose decode steps share tiles."""
    from ullm_b200.engine import ModelRunner, StepEntry

    cfg = dict(architectures=["Qwen3ForCausalLM"], num_hidden_layers=2, hidden_size=2048, num_attention_heads=16, num_key_value_heads=4,
               head_dim=128, intermediate_size=8192, vocab_size=1000, rope_theta=1e6, rms_norm_eps=1e-6, attention_bias=False,
               tie_word_embeddings=False, max_position_embeddings=4096, torch_dtype="bfloat16")
    runners = [ModelRunner(config=cfg, page_size=16, num_pages=300, max_requests=4, max_context=4096, max_step_tokens=2048,
                           load_format="random", seed=3, quantization=q) for q in (None, "int8")]
    logits = []
    ids = random_ids(1000, 1500, 4)
    for r in runners:
        r.add_request("a")
        logits.append([r.step([StepEntry("a", ids[:1498], [1497])]).clone(), r.step([StepEntry("a", ids[1498:1499], [0])]).clone()])
        r.check_device_status()
    for a, b in zip(*logits):
        # 8 bits beside 8 bits of mantissa: a step of noise of 1 / 254 of the largest against 2^-9 of each element
        assert torch.isfinite(b).all() and (a - b).abs().max() <= 0.1 * a.abs().max()
        assert not torch.equal(a, b)


def test_prompts_one_after_another(tmp_path):
    """Many prompt steps in a row, so that every kernel may begin beside the end of the one in front of it: each as when it runs alone.
    (Products by pairs of SMs allocate tensor memory for both: a block that did so before the other one had started waited for good.)"""
    from ullm_b200.engine import ModelRunner, StepEntry

    cfg = dict(architectures=["Qwen3ForCausalLM"], num_hidden_layers=6, hidden_size=2048, num_attention_heads=16, num_key_value_heads=4,
               head_dim=128, intermediate_size=8192, vocab_size=1000, rope_theta=1e6, rms_norm_eps=1e-6, attention_bias=False,
               tie_word_embeddings=False, max_position_embeddings=4096, torch_dtype="bfloat16")
    r = ModelRunner(config=cfg, page_size=16, num_pages=260, max_requests=2, max_context=4096, max_step_tokens=2048,
                    load_format="random", seed=3, quantization="int8")
    ids = random_ids(1000, 2000, 4)
    assert kernels().lib.ullm_linear_int8_form(2000, 2 * 8192, 2048) < 0

    def prompt(n):
        r.add_request("a")
        out = r.step([StepEntry("a", ids[:n], [n - 1])]).clone()
        r.end_request("a")
        return out

    sizes = (2000, 700, 1024)
    alone = []
    for n in sizes:
        alone.append(prompt(n))
        torch.cuda.synchronize()
    for _ in range(30):
        got = [prompt(n) for n in sizes]
    for a, b in zip(alone, got):
        assert torch.equal(a, b)
    r.check_device_status()
