"""The edges of the operators around prompts and 4-bit caches on the CPU, lane by lane
(tests/cpu_emu/lanes.py): the calls and tolerances of tests/serving_edges.py.
CPU only; needs /opt/rocm/llvm/bin/clang++ and an x86-64 (skipped without them)."""
import os
import platform
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import serving_edges as edges  # noqa: E402
from serving_ref import BF16, F16, F32, tname  # noqa: E402

CLANG = "/opt/rocm/llvm/bin/clang++"
pytestmark = pytest.mark.skipif(not os.path.exists(CLANG) or platform.machine() != "x86_64", reason="no clang++ for the CPU build, or not x86-64")


@pytest.fixture(scope="module")
def program():
    sys.path.insert(0, os.path.join(HERE, "cpu_emu"))
    import lanes  # tests/cpu_emu/lanes.py
    lanes.build()
    return lanes.Program


combos = pytest.mark.parametrize("q_t,cache_t", edges.COMBOS, ids=tname)
some = pytest.mark.parametrize("q_t,cache_t", [(F32, F32), (F32, F16), (BF16, BF16), (F32, BF16)], ids=tname)  # (the GPU's tests have all)
decodes = pytest.mark.parametrize("q_t,cache_t", [*edges.COMBOS, (F32, None), (F16, None), (BF16, None)], ids=tname)


@combos
@pytest.mark.parametrize("cap", edges.CAPS[::2] + edges.CAPS[-1:])
def test_prompt_caps(program, q_t, cache_t, cap):
    edges.prompt_caps(program, q_t, cache_t, cap)


@combos
def test_prompt_cap_of_large_scale(program, q_t, cache_t):
    edges.prompt_cap_of_large_scale(program, q_t, cache_t)


@decodes
@pytest.mark.parametrize("cap", edges.CAPS[::3])
def test_decode_caps(program, q_t, cache_t, cap):
    edges.decode_caps(program, q_t, cache_t, cap)


@combos
@pytest.mark.parametrize("window", edges.WINDOWS[::3])
def test_prompt_before_the_cache(program, q_t, cache_t, window):
    edges.prompt_before_the_cache(program, q_t, cache_t, window)


@some
@pytest.mark.parametrize("dim", [40])
@pytest.mark.parametrize("mask", edges.ODD_MASKS, ids=lambda m: "-".join(m) or "causal")
def test_prompt_odd_values(program, q_t, cache_t, dim, mask):
    edges.prompt_odd_values(program, q_t, cache_t, dim, mask, cus=1 if "window" in mask else 256, shares=(0.02,))


@some
@pytest.mark.parametrize("dim", [40])
@pytest.mark.parametrize("mask", edges.KEY_MASKS[::3], ids=lambda m: "-".join(m) or "causal")
def test_prompt_odd_keys(program, q_t, cache_t, dim, mask):
    edges.prompt_odd_keys(program, q_t, cache_t, dim, mask, which=slice(1, None, 2))


@combos
@pytest.mark.parametrize("dim", [40, 64])
def test_prompt_odd_q(program, q_t, cache_t, dim):
    edges.prompt_odd_q(program, q_t, cache_t, dim)


@decodes
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_decode_odd_q_and_keys(program, q_t, cache_t, cap):
    edges.decode_odd_q_and_keys(program, q_t, cache_t, cap)


@decodes
@pytest.mark.parametrize("scale", edges.SCALES[:2])
def test_other_scales(program, q_t, cache_t, scale):
    edges.other_scales(program, q_t, cache_t, scale)


@pytest.mark.parametrize("q_t,cache_t", [(BF16, BF16)], ids=tname)
@pytest.mark.parametrize("dim", [64])
@pytest.mark.parametrize("mask", edges.MANY_MASKS, ids=lambda m: "-".join(m) or "causal")
def test_prompt_many(program, q_t, cache_t, dim, mask):
    edges.prompt_many(program, q_t, cache_t, dim, mask, 1, 3)


@combos
def test_nothing_weighs(program, q_t, cache_t):
    edges.nothing_weighs(program, q_t, cache_t)
