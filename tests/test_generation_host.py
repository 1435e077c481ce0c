"""What the generation-side operators refuse, on the CPU: arguments that no kernel may see."""
import numpy as np
import pytest
import torch


def test_library_refuses_bad_sizes_before_a_launch():
    from mindformers_amd import _lib
    lib = _lib.load()

    def refused(name, args, word):
        assert getattr(lib, name)(*args) == 1
        assert word in lib.mf_last_error().decode(), lib.mf_last_error()

    fork = [8] * 9 + [4, 4, 100, 16, 1, 0, 0, 8, 1 << 20, None]
    for at, value, word in ((9, 0, "sizes"), (11, 0, "blocks"), (11, (1 << 20) + 1, "blocks"), (12, 1 << 30, "overflow"),
                            (14, -1, "sizes"), (15, 3, "window"), (2, None, "null"), (17, 8, "workspace"), (5, 8, "own")):
        args = list(fork)
        if at != 5:
            args[0], args[1] = 16, 24
        args[at] = value
        refused("mf_fork_blocks", args, word)
    compact = [8] * 5 + [4, 4, 100, 16, 8, 1 << 20, None]
    for at, value, word in ((5, 0, "sizes"), (7, 0, "blocks"), (3, None, "null"), (10, 8, "workspace")):
        args = list(compact)
        args[at] = value
        refused("mf_compact_blocks", args, word)
    beam = [8] * 7 + [0, 8, 2, 4, 100, 8, -1, 0, 8, 1 << 20, None]
    for at, value, word in ((14, 3, "dtype"), (10, 0, "sizes"), (10, 65, "beams"), (12, 3, "candidates"), (12, 65, "beams"), (11, 1, "candidates"),
                            (9, 20000, "beams"), (7, 99, "stride"), (6, None, "null"), (6, 9, "aligned"), (16, 64, "workspace")):
        args = list(beam)
        args[at] = value
        refused("mf_beam_search_select", args, word)
    args = list(beam)
    args[12], args[13] = 7, 5
    refused("mf_beam_search_select", args, "candidates")      # an end token needs two candidates a beam
    refused("mf_copy_blocks", [None, None, 1, 8, 1, 4, 4, None], "null")
    refused("mf_copy_blocks", [None, None, 1, 8, 1, 0, 4, None], "sizes")
    assert lib.mf_copy_blocks(None, None, 0, None, 3, 4, 4, None) == 0


def test_host_lists_of_copies_are_checked():
    from mindformers_amd.ops import _host_copies
    np.testing.assert_array_equal(_host_copies([[1, 2], [1, 3]], 8, 16), [[1, 2, 16], [1, 3, 16]])
    assert _host_copies(torch.zeros(0, 2, dtype=torch.int64), 8, 16).shape == (0, 3)
    for bad in ([[1, 8]], [[-1, 2]], [[1, 2, 17]], [[1, 2, -1]], [[1, 2], [3, 2]], [[1, 2], [2, 3]], [[1, 1]], [[1.5, 2.0]], [1, 2], [[1, 2, 3, 4]]):
        with pytest.raises(ValueError):
            _host_copies(bad, 8, 16)


def test_ops_refuse_tensors_that_are_not_on_the_gpu():
    from mindformers_amd import ops
    t, l = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.fork_blocks(t, l, 10, 16), lambda: ops.compact_blocks(t, 10, 16), lambda: ops.copy_blocks([torch.zeros(4, 2, 8)], [[0, 1]]),
                 lambda: ops.beam_search_select(torch.zeros(4, 9), torch.zeros(1, 4)), lambda: ops.copy_blocks([], [[0, 1]])):
        with pytest.raises(ValueError):
            call()
