"""Linear attention's planner and check at the border between its two kernels: the recurrent one takes sequences of up to 8 rows."""
import numpy as np
import pytest

from test_layers_refusals import linear_params, planned, seqs
from espetero_amd import abi, device, host

FEW = 8


@pytest.mark.parametrize("workgroups", [1, 64, 512, 5000])
@pytest.mark.parametrize("rows", [[7, 8, 9], [8] * 40, [9] * 40, [0, 1, 8, 9, 16, 17, 700]])
def test_up_to_eight_rows_are_few(rows, workgroups):
    p = linear_params(n_states=2 * len(rows))
    base = np.cumsum([0] + rows)[:-1].tolist()
    s = seqs(*[(b, m, i, len(rows) + i) for i, (b, m) in enumerate(zip(base, rows))])
    tiles, n_few, n_parts = host.plan_linear(p, s, sum(rows), workgroups)
    device.validate_linear(p, tiles, n_few, n_parts, sum(rows))
    assert sorted(int(t["rows"]) for t in tiles[:n_few]) == sorted(m for m in rows if m <= FEW)
    assert sum(int(t["rows"]) for t in tiles[n_few:]) == sum(m for m in rows if m > FEW)


def test_nine_rows_are_refused_among_the_few():
    p, tiles, n_few, n_parts = planned()
    for rows, refused in ((FEW, False), (FEW + 1, True)):
        t = tiles.copy()
        t[0]["row0"], t[0]["rows"] = 1180, rows
        if refused:
            with pytest.raises(abi.EspError, match="few"):
                device.validate_linear(p, t, n_few, n_parts, 1200)
        else:
            device.validate_linear(p, t, n_few, n_parts, 1200)
