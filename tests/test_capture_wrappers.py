"""Captured calls of the Python wrappers, on the CPU: which stream is asked about."""
import contextlib

import pytest
import torch

import dflash_qmm
from test_rotation_host import Tensor, accept_inputs, like  # noqa: F401
from test_verify_ops_wrappers import Fake, lib  # noqa: F401


@pytest.mark.parametrize("current", (0, 1))
@pytest.mark.parametrize("captured", (None, 0, 1))
def test_a_captured_accept_has_its_own_workspace_on_any_gpu(lib, monkeypatch, current,  # noqa: F811
                                                            captured):
    """A context's stream is looked at on the context's GPU, whichever is the current one."""
    at = [current]

    @contextlib.contextmanager
    def device(n):
        before, at[0] = at[0], n
        yield
        at[0] = before
    monkeypatch.setattr(torch, "Tensor", (torch.Tensor, Fake))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at[0] == captured)
    lib.need = lambda rows: 4096
    lib.current = 77     # not the default stream, which is never captured
    ctx = dflash_qmm.Context(0)
    tokens, _, _ = ctx.sample_accept(**accept_inputs())
    args = [c for c in lib.calls if c[0] == "dfq_sample_accept"][-1][1]
    shared = ctx._scratch.get(77)
    if captured == 0:
        # cut from one buffer with the outputs
        assert shared is None and tokens.data_ptr() - args[-3] == 4096
    else:
        assert shared is not None and args[-3] == shared.data_ptr()
    assert at == [current]
