"""Addresses that linear attention and attention with shaped scores refuse."""
import pytest

from test_layers_refusals import S, X, call, linear_args, linear_params, shaped_args, shaped_params


@pytest.mark.parametrize("what,off", [("Q", 2), ("Q", 4), ("Q", 8), ("pool", 2), ("pool", 8), ("O", 2), ("O", 4)])
def test_shaped_refuses_odd_addresses(what, off):
    rc, err = call("esp_attn_shaped", *shaped_args(shaped_params(), S, **{what: X + off}))[:2]
    assert rc == 1 and "aligned" in err, (rc, err)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_linear_refuses_odd_decays(off):
    rc, err = call("esp_linear_attn", *linear_args(linear_params(), decay=X + off))[:2]
    assert rc == 1 and "decay" in err, (rc, err)
