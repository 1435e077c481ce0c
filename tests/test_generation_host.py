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


def test_windowed_attention_is_refused_before_a_launch():
    from mindformers_amd import _lib
    lib = _lib.load()

    def refused(name, args, word):
        assert getattr(lib, name)(*args) == 1
        assert word in lib.mf_last_error().decode(), lib.mf_last_error()

    #        out  xq x_scale smooth layout q k v key_scale value_scale kv_quant tables lens b nh nkv d block width blocks
    decode = [16, None, None, None, 0, 16, 16, 16, None, None, 0, 16, 16, 2, 8, 2, 64, 16, 200, 100, 0.125, 1000, 4, 0, 0, 16, 1 << 30, None]
    need = lib.mf_window_attention_workspace_bytes(2, 8, 64, 3200, 1000, 4)
    assert need > 0
    for at, value, word in ((21, 0, "window"), (21, -3, "window"), (22, -1, "sinks"), (10, 3, "kv_quant"), (10, -1, "kv_quant"), (10, 1, "scales"),
                            (14, 7, "multiple"), (16, 192, "head_dim"), (16, 48, "head_dim"), (17, 0, "geometry"), (18, 1 << 28, "overflows"),
                            (24, 2, "dtype"), (5, None, "null"), (11, None, "null"), (7, 24, "aligned"), (23, 100, "stride"), (23, 516, "stride"),
                            (26, need - 1, "workspace"), (25, None, "workspace"), (25, 24, "workspace")):
        args = list(decode)
        args[at] = value
        refused("mf_window_attention_decode", args, word)
    for xq, scale, smooth, layout, kvq, word in ((16, None, None, 0, 0, "quantised"), (16, 16, None, 2, 0, "quantised"), (16, 16, None, 0, 1, "quantised"),
                                                 (20, 16, None, 0, 0, "aligned"), (16, 16, 24, 0, 0, "aligned")):
        args = list(decode)
        args[1:5], args[10] = [xq, scale, smooth, layout], kvq
        refused("mf_window_attention_decode", args, word)
    args = list(decode)
    args[8:11] = [16, None, 2]
    refused("mf_window_attention_decode", args, "per-token")
    args[8:11], args[17] = [16, 16, 2], 6
    refused("mf_window_attention_decode", args, "multiple of 4")
    args = list(decode)
    args[13] = 0
    assert lib.mf_window_attention_decode(*args) == 0          # no sequence, nothing to do

    #         out q k v key_scale value_scale kv_quant tables lens starts b rows nh nkv d block width blocks
    prefill = [16, 16, 16, 16, None, None, 0, 16, 16, 16, 2, 40, 8, 2, 64, 16, 200, 100, 0.125, 1000, 4, 0, 0, 0, 16, 1 << 30, None]
    need = lib.mf_window_attention_prefill_workspace_bytes(2, 40, 8, 2, 64, 3200, 1000, 4)
    assert need > 0
    for at, value, word in ((19, 0, "window"), (20, -1, "sinks"), (6, 3, "kv_quant"), (6, 1, "scales"), (12, 7, "multiple"), (14, 192, "32, 64 or 128"),
                            (14, 48, "head_dim"), (23, 2, "dtype"), (1, None, "null"), (9, None, "null"), (3, 24, "aligned"), (21, 100, "stride"),
                            (18, -1.0, "scale"), (25, need - 1, "workspace"), (24, None, "workspace"), (24, 24, "workspace")):
        args = list(prefill)
        args[at] = value
        refused("mf_window_attention_prefill", args, word)
    for sizes in ((0, 40, 8, 2, 64, 3200, 1000, 4), (2, 40, 8, 3, 64, 3200, 1000, 4), (2, 40, 8, 2, 64, 3200, 0, 4), (2, 40, 8, 2, 64, 3200, 1000, -1)):
        assert lib.mf_window_attention_prefill_workspace_bytes(*sizes) == 0


def test_windows_that_are_none():
    from mindformers_amd import ops
    from mindformers_amd.modules import BeamSearch, FlashAttention, PagedAttentionMgr
    assert ops.check_window(None, 0) == (0, 0) and ops.check_window(7, 2) == (7, 2) and ops.check_window(7.0, 2) == (7, 2)
    assert ops.check_window(1 << 40, 1 << 50) == (0x7fffffff, 0x7fffffff)
    for window, sinks in ((0, 0), (-1, 0), (2.5, 0), (float("inf"), 0), (float("nan"), 0), (3, -1), (3, 0.5), (3, float("inf")), (None, 1)):
        with pytest.raises(ValueError):
            ops.check_window(window, sinks)
        with pytest.raises(ValueError):
            BeamSearch([torch.zeros(4, 2, 8)], 2, window=window, sinks=sinks)
        with pytest.raises(ValueError):
            PagedAttentionMgr(2, 32, 2, kv_shape=(4, 16, 2, 32), device="cpu", window=window, sinks=sinks)
    with pytest.raises(NotImplementedError):
        FlashAttention(2, head_dim=576, kv_head_num=1, pa_mla_v_dim=512, window=4)


def test_a_beam_search_is_started_first():
    from mindformers_amd.modules import BeamSearch
    search = BeamSearch([torch.zeros(4, 2, 8)], 2)
    for call in (lambda: search.step(torch.zeros(2, 9)), lambda: search.release([0]), search.compact, search.hypotheses):
        with pytest.raises(RuntimeError, match="start"):
            call()
    for beams in (0, 33):
        with pytest.raises(ValueError):
            BeamSearch([torch.zeros(4, 2, 8)], beams)
    with pytest.raises(ValueError):
        BeamSearch([], 2)
