"""What the gradients of the 16-bit products and the loss make of a backward pass that may be recorded into a graph, on the side that needs no GPU."""
import pytest
import torch

from catccos_amd import ops


def _asked(monkeypatch, capturing, held):
    def query():
        if isinstance(capturing, Exception):
            raise capturing
        return capturing

    class Native:
        @staticmethod
        def accumulates_on_default_stream():
            return held

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", query)
    monkeypatch.setattr(ops, "_direct", Native())


def test_a_recorded_backward_of_held_leaves_is_refused(monkeypatch):
    _asked(monkeypatch, True, True)
    with pytest.raises(RuntimeError, match="matmul_bias_act: .*eager graph"):
        ops._check_recording("matmul_bias_act")


@pytest.mark.parametrize("capturing,held", [(False, True), (False, False), (True, False), (False, NotImplemented)])
def test_others_go_on(monkeypatch, capturing, held):
    _asked(monkeypatch, capturing, held)
    assert ops._check_recording("matmul_bias_act") is None


@pytest.mark.parametrize("held", [True, False, NotImplemented])
def test_a_stream_that_cannot_be_asked_is_no_recording(monkeypatch, held):
    """The default stream answers with an error while another thread records: this thread's backward is an eager one."""
    _asked(monkeypatch, RuntimeError("operation would make the legacy stream depend on a capturing blocking stream"), held)
    assert ops._check_recording("matmul_bias_act") is None


def test_a_recording_without_the_native_module_is_refused(monkeypatch):
    """Nothing else says whether an eager graph holds the leaves, and if one does the process ends."""
    _asked(monkeypatch, True, NotImplemented)
    with pytest.raises(RuntimeError, match="matmul_bias_act: .*_direct"):
        ops._check_recording("matmul_bias_act")
