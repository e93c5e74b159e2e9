"""Which models may keep their layers' matrices in 8 bits, decided before anything is on a device."""
import pytest

import helpers as H
from aien_sovereign_core_mv_b200 import ConfigError, EngineConfig, model_spec_for
from aien_sovereign_core_mv_b200.models import Decoder
from aien_sovereign_core_mv_b200.models.float8 import with_float8_weights


@pytest.mark.parametrize("which", list(H.TINY))
def test_dense_decoders(which):
    spec = model_spec_for(H.TINY[which])[1]
    eight = with_float8_weights(spec)
    assert all("weights" not in l.mixer.params for l in spec.layers)             # the spec itself is left alone
    assert all(l.mixer.params["weights"] == l.feed_forward.params["weights"] == "float8" for l in eight.layers)
    plain, model = Decoder(spec), Decoder(eight)
    assert model.catalog() == plain.catalog() and model.group_needs == plain.group_needs
    assert all(b.mixer.takes_float8 and b.feed_forward.takes_float8 and not b.mixer.feeds_residual and not b.feed_forward.takes_prenormed for b in model.blocks)
    assert not any(b.mixer.takes_float8 or b.feed_forward.takes_float8 for b in plain.blocks)


def test_other_layers_are_refused_by_name():
    from test_config import _dulisun_config
    with pytest.raises(ConfigError, match="layer 0: no 8-bit form of mixer 'chunked_sink_attention', feed_forward 'routed_experts', block 'branchnorm'"):
        with_float8_weights(model_spec_for(_dulisun_config())[1])


def test_engine_config():
    assert EngineConfig().resolved_weights() == "stored" and EngineConfig(weights="float8").resolved_weights() == "float8"
    with pytest.raises(ValueError, match="weights must be stored or float8"):
        EngineConfig(weights="int8").resolved_weights()
    with pytest.raises(ValueError, match="bfloat16 engine"):
        EngineConfig(dtype="float32", weights="float8").resolved_weights()


def test_parts_refuse_other_kinds():
    from aien_sovereign_core_mv_b200.registry import make_part
    with pytest.raises(ValueError, match="known are 'stored' and 'float8'"):
        make_part("feed_forward", "swiglu", hidden_size=8, intermediate_size=8, weights="int4")
    with pytest.raises(ValueError, match="known are 'stored' and 'float8'"):
        make_part("mixer", "paged_attention", hidden_size=8, num_heads=1, num_kv_heads=1, head_dim=8, position=make_part("position", "none"), weights="int4")
