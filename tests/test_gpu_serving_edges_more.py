"""The edges of the operators around prompts and 4-bit caches on the GPU: the calls and
tolerances of tests/serving_edges.py."""
import os
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import serving_edges as edges  # noqa: E402
from serving_ref import BF16, F16, F32, tname  # noqa: E402

pytestmark = pytest.mark.gpu
combos = pytest.mark.parametrize("q_t,cache_t", edges.COMBOS, ids=tname)
decodes = pytest.mark.parametrize("q_t,cache_t", [*edges.COMBOS, (F32, None), (F16, None), (BF16, None)], ids=tname)


@pytest.fixture(scope="module")
def program():
    from tomoul_amd import _abi
    _abi.init()
    return edges.GpuProgram


@combos
@pytest.mark.parametrize("cap", edges.CAPS)
def test_prompt_caps(program, q_t, cache_t, cap):
    edges.prompt_caps(program, q_t, cache_t, cap)


@combos
def test_prompt_cap_of_large_scale(program, q_t, cache_t):
    edges.prompt_cap_of_large_scale(program, q_t, cache_t)


@decodes
@pytest.mark.parametrize("cap", edges.CAPS)
def test_decode_caps(program, q_t, cache_t, cap):
    edges.decode_caps(program, q_t, cache_t, cap)


@combos
@pytest.mark.parametrize("window", edges.WINDOWS)
def test_prompt_before_the_cache(program, q_t, cache_t, window):
    edges.prompt_before_the_cache(program, q_t, cache_t, window)


@combos
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
@pytest.mark.parametrize("mask", edges.ODD_MASKS, ids=lambda m: "-".join(m) or "causal")
def test_prompt_odd_values(program, q_t, cache_t, dim, mask):
    edges.prompt_odd_values(program, q_t, cache_t, dim, mask)


@combos
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
@pytest.mark.parametrize("mask", edges.KEY_MASKS, ids=lambda m: "-".join(m) or "causal")
def test_prompt_odd_keys(program, q_t, cache_t, dim, mask):
    edges.prompt_odd_keys(program, q_t, cache_t, dim, mask)


@combos
@pytest.mark.parametrize("dim", [40, 64])
def test_prompt_odd_q(program, q_t, cache_t, dim):
    edges.prompt_odd_q(program, q_t, cache_t, dim)


@decodes
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_decode_odd_q_and_keys(program, q_t, cache_t, cap):
    edges.decode_odd_q_and_keys(program, q_t, cache_t, cap)


@decodes
@pytest.mark.parametrize("scale", edges.SCALES)
def test_other_scales(program, q_t, cache_t, scale):
    edges.other_scales(program, q_t, cache_t, scale)


@pytest.mark.parametrize("q_t,cache_t", edges.COMBOS, ids=tname)
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("mask", edges.MANY_MASKS, ids=lambda m: "-".join(m) or "causal")
def test_prompt_many(program, q_t, cache_t, dim, mask):
    import torch
    edges.prompt_many(program, q_t, cache_t, dim, mask, torch.cuda.get_device_properties(0).multi_processor_count, 70)


@combos
def test_nothing_weighs(program, q_t, cache_t):
    edges.nothing_weighs(program, q_t, cache_t)
