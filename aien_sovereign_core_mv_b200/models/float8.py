"""A model whose layers keep their matrices in 8 bits."""
from __future__ import annotations

from dataclasses import replace

from ..config.model_config import ConfigError
from ..config.spec import ModelSpec, PartSpec
from ..registry import part_factory


def _takes(family: str, part: PartSpec) -> bool:
    return bool(getattr(part_factory(family, part.kind), "offers_float8", False))


def with_float8_weights(spec: ModelSpec) -> ModelSpec:
    """The same model with ``weights="float8"`` given to every mixer and feed-forward: their matrices are e4m3 codes with a scale for each block
    of 128 x 128, what they read is in 8 bits with a scale for each 128 numbers of a row, made by the norm ahead of them or by a step between two
    products.  Norms, the attention itself, embedding and head stay as they are.  Every layer has to be made of parts that can: a pre-norm block of an RMS
    norm, grouped-query attention and a gated feed-forward (the Llama and Qwen3 decoders)."""
    layers = []
    for i, layer in enumerate(spec.layers):
        wrong = [f"{family} {part.kind!r}" for family, part in (("mixer", layer.mixer), ("feed_forward", layer.feed_forward))
                 if part is not None and not _takes(family, part)]
        block = part_factory("block", layer.block)
        if not getattr(block, "offers_float8", False):
            wrong.append(f"block {layer.block!r}")
        wrong += [f"norm {layer.norm_for(slot).kind!r}" for slot in getattr(block, "norm_slots", ()) if not _takes("norm", layer.norm_for(slot))]
        if wrong:
            raise ConfigError(f"layer {i}: no 8-bit form of {', '.join(dict.fromkeys(wrong))}: weights float8 are for pre-norm layers of grouped-query "
                              f"attention and gated feed-forwards")
        put = lambda part: None if part is None else PartSpec(part.kind, {**dict(part.params), "weights": "float8"})
        layers.append(replace(layer, mixer=put(layer.mixer), feed_forward=put(layer.feed_forward)))
    return replace(spec, layers=tuple(layers))
