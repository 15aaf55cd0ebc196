"""The scan of test_isa_hazards.py over the kernels of linear attention and of attention with shaped scores."""
from concurrent.futures import ThreadPoolExecutor

import pytest

import isa_hazards
from test_isa_hazards import _assembly

SOURCES = ["linear.hip", "attn_shaped.hip", "attn_shaped_tiled.hip"]


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("isa"))
    with ThreadPoolExecutor(3) as pool:
        return dict(zip(SOURCES, pool.map(lambda s: _assembly(s, out), SOURCES)))


@pytest.mark.parametrize("src", SOURCES)
def test_no_reader_of_a_matrix_result_in_another_block_comes_too_soon(listings, src):
    found, n = [], 0
    for name, lines in isa_hazards.kernels(listings[src]):
        n += any(l[0] == "ins" and l[1].startswith("v_mfma") for l in lines)
        found += [(name, v) for v in isa_hazards.violations(lines)]
    assert n >= 8 and found == [], found[:3]
