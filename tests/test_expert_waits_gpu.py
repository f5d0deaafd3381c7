"""The bounded wait inside the expert products: the lanes of a warp go on together or give up together."""
import pytest
import torch


def test_the_probe_refuses_long_limits():
    from brainstorm_b200 import _lib

    for args in ((4096, 10 ** 9, 0, 0), (4096, 0, 10 ** 9, 0), (4096, 0, 0, 10 ** 9)):
        with pytest.raises(_lib.BrtError, match="limit"):
            _lib.call("brt_expert_wait_probe", *args, None)
    with pytest.raises(_lib.BrtError, match="null"):
        _lib.call("brt_expert_wait_probe", None, 0, 0, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("first,others,arrives,done", [
    (10 ** 8, 10 ** 8, 0, 1),               # at once
    (10 ** 8, 10 ** 8, 2 * 10 ** 6, 1),     # within everybody's limit
    (10 ** 5, 10 ** 8, 5 * 10 ** 6, 0),     # behind the limit of one lane: nobody goes on alone
    (10 ** 8, 10 ** 5, 5 * 10 ** 6, 0),
    (10 ** 5, 10 ** 5, 5 * 10 ** 6, 0),
])
def test_lanes_go_on_together_or_not_at_all(first, others, arrives, done):
    from brainstorm_b200 import _lib

    for _ in range(10):
        results = torch.full((32,), 7, dtype=torch.int32, device="cuda")
        _lib.call("brt_expert_wait_probe", results.data_ptr(), first, others, arrives,
                  torch.cuda.current_stream().cuda_stream)
        assert results.tolist() == [done] * 32


def test_the_word_of_run_out_waits_needs_a_place():
    from brainstorm_b200 import _lib

    with pytest.raises(_lib.BrtError, match="null"):
        _lib.call("brt_expert_error_word", None)
