"""Settings of the whole process that a test leaves behind do not reach the next one: two
tests, in this order."""
import deep_gemm
from deep_gemm import _ffi


def pieces():
    return _ffi.lib.dg_bf16_gemm_ragged_workspace_size(0, 10, 0, 30, 640, 2)


def test_leaves_settings_behind():
    deep_gemm.set_num_sms(7)
    deep_gemm.set_tile_override(128, 5, variant=13)
    deep_gemm.set_mk_alignment_for_contiguous_layout(64)
    assert deep_gemm.get_num_sms() == 7 and pieces() == 5 * 10 * 32 * 4


def test_finds_none():
    try:
        assert deep_gemm.get_num_sms() != 7
    except RuntimeError as e:      # no device to ask
        assert 'hip' in str(e).lower()
    deep_gemm.set_num_sms(7)
    assert pieces() != 5 * 10 * 32 * 4
    assert deep_gemm.get_mk_alignment_for_contiguous_layout() == 128
