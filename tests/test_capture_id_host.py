"""The number of a stream's capture: arguments, without a GPU."""

from llama_lite_npu_amd import _lib, ops


def test_refused_without_a_place_for_the_number():
    assert _lib.load().litekv_stream_capture_id(None, None) == 1 and b"null pointer" in _lib.load().litekv_last_error()


def test_nothing_is_captured_outside_a_capture(monkeypatch):
    monkeypatch.setattr(ops.torch.cuda, "is_current_stream_capturing", lambda: False)
    assert ops.capture_id() is None
