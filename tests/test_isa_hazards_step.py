"""The matrix kernels of differential attention and of the low-rank adapters, scanned as tests/test_isa_hazards.py scans the others."""
import os
from concurrent.futures import ThreadPoolExecutor

import pytest

import isa_hazards
from test_isa_hazards import HIPCC, _assembly

SOURCES = ["attn_diff.hip", "attn_diff_tiled.hip", "lowrank.hip"]


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    out = str(tmp_path_factory.mktemp("isa"))
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        texts = list(pool.map(lambda s: _assembly(s, out), SOURCES))
    return {src: list(isa_hazards.kernels(text)) for src, text in zip(SOURCES, texts)}


def test_no_matrix_result_is_read_across_a_block_boundary_too_early(listings):
    for src, kernels in listings.items():
        matrix = [(name, lines) for name, lines in kernels if any(kind == "ins" and op.startswith("v_mfma") for kind, op, _ in lines)]
        assert matrix, src
        for name, lines in matrix:
            assert isa_hazards.violations(lines) == [], (src, name)


def test_no_packed_fp32(listings):
    for src, kernels in listings.items():
        for name, lines in kernels:
            assert not [op for kind, op, _ in lines if kind == "ins" and op.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))], (src, name)
