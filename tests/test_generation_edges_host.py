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
