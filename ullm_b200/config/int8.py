"""A decoder's spec with its layers' products in 8-bit integers (parts/int8.py).  Embedding and output head stay as they are.

The reference has no quantized weights."""

from __future__ import annotations

from dataclasses import replace

from .specs import ModelSpec

QUANTIZATIONS = ("int8",)
_BLOCKS = {"prenorm_residual": "prenorm_residual_int8"}
_MIXERS = {"paged_attention": "paged_attention_int8"}
_FEED_FORWARDS = {"gated_mlp": "gated_mlp_int8"}


def int8_spec(spec: ModelSpec) -> ModelSpec:
    """The spec whose layers hold their matrices in 8 bits; ValueError for a layer made of anything but pre-norm blocks of paged
    attention and a gated feed-forward."""

    def layer(i, s):
        if s.block not in _BLOCKS or s.mixer.kind not in _MIXERS or s.feed_forward is None or s.feed_forward.kind not in _FEED_FORWARDS:
            raise ValueError(f"quantization 'int8': layer {i} of {spec.architecture} is {s.block} with {s.mixer.kind} and "
                             f"{s.feed_forward.kind if s.feed_forward else 'no feed-forward'}; 8-bit products go with pre-norm blocks of "
                             "paged attention and a gated feed-forward")
        return replace(s, block=_BLOCKS[s.block], mixer=replace(s.mixer, kind=_MIXERS[s.mixer.kind]),
                       feed_forward=replace(s.feed_forward, kind=_FEED_FORWARDS[s.feed_forward.kind]))

    if spec.stream_dtype != "engine":
        raise ValueError(f"quantization 'int8': {spec.architecture} keeps its residual stream in 32 bits")
    return replace(spec, layers=[layer(i, s) for i, s in enumerate(spec.layers)])
