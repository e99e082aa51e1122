"""Page-locking host memory: what the driver refuses is logged, what fails is
raised."""
import logging

import pytest
import torch

from torched_impala_amd import ops


def test_failure_without_a_device_is_raised():
    """Not to be taken for a driver that refuses this memory."""
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    ext = ops.ext_hip(required=False)
    if ext is None:
        pytest.skip("the kernels' extension is not built")
    with pytest.raises(RuntimeError, match="hipHostRegister"):
        ext.host_register(torch.zeros(8))
    assert not ext.host_register(torch.zeros(0))


class _Ext:
    def __init__(self, answer):
        self.answer = answer

    def host_register(self, t):
        if isinstance(self.answer, Exception):
            raise self.answer
        return self.answer


def test_refusal_is_logged_with_its_reason(monkeypatch, caplog):
    monkeypatch.setattr(ops, "ext_hip", lambda required=True: _Ext("reason"))
    with caplog.at_level(logging.WARNING):
        ops.pin_host_memory(torch.zeros(8))
    assert "32 bytes" in caplog.text and "reason" in caplog.text


@pytest.mark.parametrize("answer", ["", RuntimeError("lost")])
def test_nothing_else_is_logged(monkeypatch, caplog, answer):
    monkeypatch.setattr(ops, "ext_hip", lambda required=True: _Ext(answer))
    with caplog.at_level(logging.WARNING):
        if answer:
            with pytest.raises(RuntimeError):
                ops.pin_host_memory(torch.zeros(8))
        else:
            ops.pin_host_memory(torch.zeros(8))
    assert not caplog.text
