"""What can be held in 4 bits, and what is refused, without a GPU."""
import pytest

import carbon_engine_b200.models  # noqa: F401
from carbon_engine_b200 import ops_int4
from carbon_engine_b200.config.registry import resolve_architecture
from carbon_engine_b200.engine.engine import hold_in_4_bits, linears
from carbon_engine_b200.parts.base import Mixer, PagedCacheSpec
from helpers import TINY


def model(**over):
    from carbon_engine_b200.config.qwen3 import Qwen3Config
    raw = dict(TINY["D"]["config"], **over)
    return resolve_architecture(raw).build_model(Qwen3Config.from_dict(dict(raw)), 256)


def test_what_is_marked():
    m = model()
    hold_in_4_bits(m, 16, 16, 64, 64)
    assert all(p.int4_group is None for p in linears(m))
    assert all(s.int4_group is None for _, s in m.cache_layout())
    hold_in_4_bits(m, 4, 4, 128, 64)
    assert [p.int4_group for p in linears(m)] == [128] * (4 * len(m.blocks))        # q|k|v, o, gate|up, down
    assert [p.gated for p in linears(m)] == [False, False, True, False] * len(m.blocks)
    assert all(s == PagedCacheSpec(2, 128, 0, None, int4_group=64) for _, s in m.cache_layout())


def test_products_whose_width_does_not_fit_stay_as_they_are():
    m = model(intermediate_size=1000)
    hold_in_4_bits(m, 4, 16, 64, 16)
    assert [p.int4_group for p in linears(m)] == [64, 64, 64, None] * len(m.blocks)
    with pytest.raises(ValueError):
        hold_in_4_bits(model(hidden_size=80, num_attention_heads=6, num_key_value_heads=3, head_dim=48, intermediate_size=112), 4, 16, 128, 16)


@pytest.mark.parametrize("args", [(8, 16, 64, 16), (16, 3, 64, 16), (4, 16, 16, 16), (16, 4, 64, 8), (16, 4, 64, 24), (16, 4, 16, 16)])
def test_refusals(args):
    with pytest.raises(ValueError):
        hold_in_4_bits(model(), *args)


def test_heads_and_mixers_a_cache_cannot_hold():
    with pytest.raises(ValueError, match="head size 16"):
        hold_in_4_bits(model(head_dim=16), 16, 4, 32, 16)
    m = model()
    m.blocks[1].mixer = Mixer()
    with pytest.raises(ValueError, match="paged attention"):
        hold_in_4_bits(m, 16, 4, 64, 16)


def test_sizes():
    # codes and (step, minimum) of keys and values: what the kernels' tiles hold
    for d in ops_int4.HEAD_SIZES:
        for group in ops_int4.CACHE_GROUPS:
            assert ops_int4.cache_bytes_per_token(3, d, group) * 16 == 3 * (16 * d + 128 * (d // group))
    assert ops_int4.cache_problem(128, 64, 16) is None
    assert ops_int4.cache_problem(96, 32, 16) and ops_int4.cache_problem(64, 128, 16) and ops_int4.cache_problem(64, 64, 20)


@pytest.mark.parametrize("jobs", [1, 8, 40, 168, 512, 5000])
@pytest.mark.parametrize("tiles", [1, 7, 8, 100, 563, 8192])
def test_splits_cover_the_keys(jobs, tiles):
    splits, share = ops_int4._splits(jobs, tiles)
    assert splits * share >= tiles and (splits - 1) * share < tiles and 1 <= splits <= 64


def test_a_mixer_inside_a_sum_sees_its_own_state():
    """Views are made field by field in places that know nothing of 4-bit pages."""
    from carbon_engine_b200.cache.storage import LayerCacheView
    view = LayerCacheView("paged", 1, 16, "k", "v", "state", False, {"a": "b"})
    assert (view.state, view.writes, view.extra, view.int4) == ("state", False, {"a": "b"}, None)
