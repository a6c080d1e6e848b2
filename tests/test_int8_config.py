"""Which models take quantization='int8', and the options that ask for it."""

import argparse
import importlib

import pytest

from helpers import weights_for, write_model_dir
from ullm_b200 import EngineConfig
from ullm_b200.config import int8_spec, load_model_spec
from ullm_b200.parts.model import DecoderModel


def test_spec_of_a_pre_norm_decoder():
    cfg, _, _ = weights_for("B", "float32")
    _, spec = load_model_spec(cfg)
    held = int8_spec(spec)
    assert {(s.block, s.mixer.kind, s.feed_forward.kind) for s in held.layers} == {
        ("prenorm_residual_int8", "paged_attention_int8", "gated_mlp_int8")}
    assert {(s.block, s.mixer.kind, s.feed_forward.kind) for s in spec.layers} == {("prenorm_residual", "paged_attention", "gated_mlp")}
    # the checkpoint's tensors are the same ones
    assert DecoderModel(held).all_decls() == DecoderModel(spec).all_decls()
    with pytest.raises(ValueError, match="8-bit products go with"):
        int8_spec(held)


@pytest.mark.parametrize("design", ["mafarax", "ludalix", "borosun", "pidenex", "finosun", "ninelix"])
def test_other_designs_are_refused(design):
    helpers = importlib.import_module(design + "_helpers")
    config = next(v for n, v in sorted(vars(helpers).items()) if n.startswith("CFG_") and isinstance(v, dict))
    _, spec = load_model_spec(config)
    with pytest.raises(ValueError, match="quantization 'int8'"):
        int8_spec(spec)


def test_options(tmp_path):
    cfg, w, _ = weights_for("A", "float32")
    d = write_model_dir(str(tmp_path / "m"), cfg, w)
    assert EngineConfig(model=d).quantization is None
    with pytest.raises(ValueError, match="int4"):
        EngineConfig(model=d, quantization="int4")
    parser = argparse.ArgumentParser()
    EngineConfig.add_cli_args(parser)
    assert EngineConfig.from_args(parser.parse_args(["--model", d, "--quantization", "int8"])).quantization == "int8"
    assert EngineConfig.from_args(parser.parse_args(["--model", d])).quantization is None


def test_what_the_parts_refuse():
    from ullm_b200.parts import FEED_FORWARDS, MIXERS

    with pytest.raises(ValueError, match="activation"):
        FEED_FORWARDS["gated_mlp_int8"](hidden_size=16, intermediate_size=32, activation="swiglu_clamped", limit=7.0)
    with pytest.raises(ValueError, match="plain attention"):
        MIXERS["paged_attention_int8"](hidden_size=16, num_heads=2, num_kv_heads=1, head_dim=8, score_cap=30.0)
