"""8-bit plans, cache needs and their storage, without a GPU."""
import pytest
import torch

from kvad_b200.cache.device import DeviceCache
from kvad_b200.cache.layout import CacheLayout, KVNeed
from kvad_b200.config import architectures
from kvad_b200.models.int8 import int8_plan
from kvad_b200.models.plan import Model
from kvad_b200.ops import Ops, libraries_for
from tests.conftest import TINY


def plan_of(name):
    from kvad_b200.config.json_view import JsonView
    arch = next(a for a in architectures() if a.id == "gpt2")
    return arch.plan(arch.read_config(JsonView(TINY[name])))


def test_an_8_bit_plan_asks_for_the_same_tensors():
    plan = plan_of("A")
    assert [(r.name, r.shape) for r in Model(int8_plan(plan)).requests()] == [(r.name, r.shape) for r in Model(plan).requests()]


def test_an_8_bit_plan_names_what_it_launches_from_and_keeps():
    model = Model(int8_plan(plan_of("A")))
    assert "int8" in model.kernel_families() and model.graph_safe
    assert "attention_int8_prompt" in libraries_for(torch.bfloat16, model.kernel_families())
    assert all(g.need.int8 for g in model.cache_layout.groups)


def test_inputs_that_no_product_takes_are_refused():
    with pytest.raises(ValueError, match="multiple of 16"):
        Model(int8_plan(plan_of("C")))               # an inner width of 200


def test_an_architecture_without_an_8_bit_form_says_so():
    from tests.nifulix_configs import CONFIGS
    from kvad_b200.config.json_view import JsonView
    arch = next(a for a in architectures() if a.id.lower() == "nifulix")
    with pytest.raises(ValueError, match="no 8-bit form"):
        int8_plan(arch.plan(arch.read_config(JsonView(CONFIGS["R"]))))


def test_storage_of_a_group_in_8_bits():
    layout = CacheLayout([KVNeed(2, 32, int8=True), KVNeed(2, 32), KVNeed(2, 32, int8=True)])
    cache = DeviceCache(layout, torch.float32, "cpu", 256, max_seqs=2)
    view, plain = cache.kv_view(2, {0: None, 1: None}), cache.kv_view(1, {0: None, 1: None})
    assert view.k_pages.dtype == view.v_pages.dtype == torch.int8 and view.k_pages.shape == (4, 2, 64, 32)
    assert view.k_scales.shape == view.v_scales.shape == (4, 2, 64) and view.k_scales.dtype == torch.float32
    assert plain.k_pages.dtype == torch.float32 and plain.k_scales is None
    assert layout.bytes_per_token(4) == 2 * (2 * 2 * (32 + 4)) + 2 * 2 * 32 * 4
    assert cache.bytes() == 256 * layout.bytes_per_token(4)
    with pytest.raises(ValueError, match="like its keys"):
        KVNeed(2, 32, value_dim=16, int8=True)


@pytest.mark.parametrize("items,reach", [(1, 1), (12, 9), (96, 16), (96, 17), (8, 126), (8, 471), (148, 40), (149, 16), (512, 129), (4000, 3)])
def test_every_page_goes_to_one_block(items, reach):
    for hd, wide in ((16, False), (64, False), (128, False), (128, True), (256, False)):
        blocks, pages, warps = Ops.int8_splits(items, reach, hd, wide, n_sms=148)
        assert 1 <= warps <= 12 and blocks >= 1 and (blocks - 1) * pages < reach <= blocks * pages
        assert reach > 16 or blocks == 1


@pytest.mark.parametrize("rows,seqs,kv,group,width,window", [(2048, 2, 16, 1, 16, 0), (330, 2, 2, 4, 43, 0), (5, 1, 2, 4, 126, 0), (5, 1, 1, 128, 126, 0), (300, 1, 4, 2, 500, 100)])
def test_every_page_goes_to_one_part(rows, seqs, kv, group, width, window):
    parts, pages = Ops.int8_parts(rows, seqs, kv, group, width, window, 4, n_sms=148)
    assert parts == 1 or (pages >= 8 and (parts - 1) * pages < width)
    tokens = 2 * (128 // group)
    reach = min(width, -(-(window + tokens) // 64) + 2) if window else width
    assert parts == 1 or parts * pages >= reach
