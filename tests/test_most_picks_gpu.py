"""As many picks as ``order_picks`` takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_order_of_as_many_picks_as_there_may_be():
    """Two paths and picks that go nowhere, in turn."""
    from brainstorm_b200 import _lib
    from brainstorm_b200._C import router as R

    n, E, part = 2 ** 31 - 2 ** 20 - 1, 2, 1 << 27
    picks = torch.empty(n, 1, dtype=torch.int32, device="cuda")
    for i in range(0, n, part):
        at = torch.arange(i, min(i + part, n), device="cuda")
        picks[i:i + part, 0] = (at % 3).int()
    places, loads = R.order_picks(picks, E)
    count = [(n + 2 - r) // 3 for r in range(3)]
    assert loads.tolist() == count[:2]
    base = torch.tensor([0, count[0], count[0] + count[1]], device="cuda")
    for i in range(0, n, part):
        at = torch.arange(i, min(i + part, n), device="cuda")
        row = base[at % 3] + at // 3
        want = torch.where(at % 3 < 2, row, -2 - row)
        assert torch.equal(places[i:i + part, 0].long(), want), i
    del picks, places
    torch.cuda.empty_cache()
    small = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="32 bits"):
        R.order_picks(small.expand(n + 1, 1), E)
    assert _lib.query("brt_pick_order_scratch_bytes", n, E) <= 1024 * 3 * 4
