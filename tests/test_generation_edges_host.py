"""Refusals and layouts of the generation-side operators, on the CPU."""
import pytest


def test_the_decode_step_keeps_the_struct_that_it_had_before_there_were_windows():
    """27 addresses, 17 integers and 3 doubles, 8 bytes each: a caller of mf_decode_layer_step need not be built again."""
    from mindformers_amd import _lib
    assert [len(names) for names in _lib.DECODE_LAYER_FIELDS.values()] == [27, 17, 3]
    assert _lib.load().mf_decode_layer_args_bytes() == 8 * (27 + 17 + 3)
    assert _lib.DECODE_LAYER_FIELDS["d"] == ("eps", "next_eps", "scale")


@pytest.mark.parametrize("window,sinks", [(-1, 0), (5, -1), (0, 3)])
def test_the_decode_step_refuses_a_window_before_any_launch(window, sinks):
    from mindformers_amd import _lib
    lib = _lib.load()
    args = _lib.DECODE_LAYER_ARGS.pack(*[0] * 44, 0.0, 0.0, 0.0)
    assert lib.mf_decode_layer_step_window(args, window, sinks) == 1 and "window" in lib.mf_last_error().decode()
    for rc in (lib.mf_decode_layer_step_window(args, 4, 1), lib.mf_decode_layer_step(args)):
        assert rc == 1 and "null" in lib.mf_last_error().decode()


def test_windows_over_tables_of_more_than_2_to_the_30_tokens_are_refused():
    """The plan may take the whole walk as one partition, and walk and partition are added in 32 bits."""
    from mindformers_amd import _lib
    lib = _lib.load()
    for block, width, ok in ((128, 1 << 23, True), (128, (1 << 23) + 1, False), (32768, 65535, False), (1, (1 << 30) + 1, False)):
        # without a workspace: what is served is refused for that, further down
        decode = [16, None, None, None, 0, 16, 16, 16, None, None, 0, 16, 16, 2, 8, 2, 64, block, width, 100, 0.125, 1 << 30, 4, 0, 0, None, 0, None]
        prefill = [16, 16, 16, 16, None, None, 0, 16, 16, 16, 2, 40, 8, 2, 64, block, width, 100, 0.125, 1 << 30, 4, 0, 0, 0, None, 0, None]
        for name, args in (("mf_window_attention_decode", decode), ("mf_window_attention_prefill", prefill)):
            assert getattr(lib, name)(*args) == 1
            assert ("workspace" if ok else "with a window") in lib.mf_last_error().decode(), lib.mf_last_error()
    packed = [16, 16, 16, 16, None, None, 0, None, None, 16, 1, (1 << 30) + 1, 8, 2, 64, 0, 0, 0, 0.125, 1 << 30, 4, 0, 0, 0, None, 0, None]
    assert lib.mf_window_attention_prefill(*packed) == 1 and "with a window" in lib.mf_last_error().decode()


def test_a_band_asked_for_by_the_reference_s_arguments_is_warned_of():
    import warnings
    from mindformers_amd.modules import FlashAttention, InferAttention
    flash = lambda **kw: FlashAttention(2, 32, 2, **kw)  # noqa: E731
    infer = lambda **kw: InferAttention(2, 32, 2, num_blocks=2, use_rope_rotary_emb=False, device="cpu", **kw)  # noqa: E731
    for make in (flash, infer):
        for band in (dict(sparse_mode=4), dict(pre_tokens=511), dict(pre_tokens=511, sparse_mode=4)):
            with pytest.warns(UserWarning, match="window=pre_tokens"):
                assert make(**band) is not None
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            for quiet in ({}, dict(window=512, pre_tokens=511, sparse_mode=4), dict(pre_tokens=511, sparse_mode=2), dict(sparse_mode=3),
                          dict(pre_tokens=None, sparse_mode=None), dict(pre_tokens=None)):
                make(**quiet)


def test_vocabularies_whose_columns_pass_32_bits_are_refused():
    """A wave's piece may end a 64th behind the row's end, and its next step behind that."""
    from mindformers_amd import _lib
    lib = _lib.load()
    for beams, vocab, word in ((1, 0x7c000000, "workspace"), (1, 0x7c000001, "tokens"), (1, 0x7fffffff, "tokens"), (2, 0x3e000001, "tokens"),
                               (62, 33554432, "workspace")):
        args = [8] * 7 + [0, 8, 1, beams, vocab, beams, -1, 0, None, 0, None]
        assert lib.mf_beam_search_select(*args) == 1 and word in lib.mf_last_error().decode(), lib.mf_last_error()
