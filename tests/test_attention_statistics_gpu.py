"""Attention within segments: the statistics of a plan reach the host some time after the plan is built.  Whether they
have arrived when an operator is called must not show in its results."""
import pytest
import torch

from tests.test_attention_gpu import DEV, TYPES, _inputs, _plan, _step

pytestmark = pytest.mark.gpu


def _forget(data):
    """The plan as it is while the copy of its statistics is still under way, whenever that is."""
    data._poll(wait=True)
    known = data._plan.max_cnt
    data._plan.max_cnt = -1
    return known


LENS = {"half tiles": [32 + 7 * i % 33 for i in range(40)], "tiles": [64] * 9, "short": [1 + 11 * i % 64 for i in range(50)],
        "one": [50], "longer": [40, 65, 300], "many": [32 + 7 * i % 33 for i in range(300)]}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("shuffled", [False, True])
def test_bits_do_not_depend_on_what_the_host_knows(dtype, dim, lens, shuffled):
    lens = LENS[lens]
    ids, data = _plan(lens, shuffled, dim)
    q, k, v, g = _inputs(sum(lens), 2, 1, dim, dtype, 5)
    known = _forget(data)
    assert known == max(lens)
    early = _step(q, k, v, g, data, causal=dim == 16)
    data._plan.max_cnt = known
    late = _step(q, k, v, g, data, causal=dim == 16)
    assert all(torch.equal(a, b) for a, b in zip(early, late))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 64])
def test_bits_beside_rows_that_are_not_finite(dtype, dim):
    """Values that are not finite right behind what a tile of 64 rows sees."""
    lens = [30, 34, 9, 60, 1, 58]
    ids, data = _plan(lens, False)
    q, k, v, g = _inputs(sum(lens), 2, 1, dim, dtype, 6)
    v[ids == 2] = float("nan")
    known = _forget(data)
    early = _step(q, k, v, g, data)
    data._plan.max_cnt = known
    late = _step(q, k, v, g, data)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(early, late))
    assert early[0][ids != 2].isfinite().all() and early[0][ids == 2].isnan().all()
