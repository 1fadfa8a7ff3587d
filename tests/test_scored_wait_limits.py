"""The limits of the waits behind the scores and the shared attention, run out by a thread that nobody signals."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,word", [("head_scores", 0), ("shared", 1), ("shared_tcgen05", 1)])
def test_a_wait_that_runs_out_sets_its_error_word(kernel, word):
    """Some 50 ms with a limit of 10^8 cycles, some 1 ms with one of 2 * 10^6: the limit that was set is the one that holds."""
    from pulsar_b200 import ops
    ops.check_wait_words()
    took = {}
    try:
        for limit in (100_000_000, 2_000_000):
            ops.set_wait_limit(limit)
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            torch.cuda.synchronize()
            a.record()
            ops.wait_selftest(kernel)
            b.record()
            b.synchronize()
            took[limit] = a.elapsed_time(b)
            words = torch.zeros(8, dtype=torch.int32, device="cuda")
            ops.gather_wait_words(words)
            assert words.tolist()[:ops.N_WAIT_WORDS] == [9 if i == word else 0 for i in range(ops.N_WAIT_WORDS)]
            with pytest.raises(ops.DeviceWaitError, match="wait self-test"):
                ops.check_wait_words()
            ops.set_wait_words(0)
    finally:
        ops.set_wait_limit(4_000_000_000)
        ops.set_wait_words(0)
    assert took[2_000_000] < 20 < took[100_000_000] < 500
    ops.check_wait_words()
    a = torch.randn(64, 64, device="cuda")
    assert torch.isfinite(a @ a).all()                  # the context still works


def test_an_unknown_kernel_is_refused():
    from pulsar_b200 import ops
    with pytest.raises(ValueError, match="unknown kernel"):
        ops.wait_selftest("nothing")
