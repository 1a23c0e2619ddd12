"""The Python wrappers of the cache, attention and log-probability calls over a library that only
records: which workspaces, streams and addresses a call is made with.  Nothing is launched."""
import threading
import time

import pytest
import torch

import dflash_qmm

WORKSPACE = 3   # the status of a workspace that is too small


class Fake:
    """A tensor that lies on a GPU as far as the wrappers can tell."""

    def __init__(self, shape, dtype=torch.bfloat16, device="cuda:0", address=1 << 20):
        self.shape, self.dtype, self.device = tuple(shape), dtype, torch.device(device)
        self.address = address
        self.is_cuda = self.device.type == "cuda"

    def stride(self, i=None):
        s, n = [], 1
        for d in reversed(self.shape):
            s.insert(0, n)
            n *= d
        return tuple(s) if i is None else s[i]

    def dim(self):
        return len(self.shape)

    def data_ptr(self):
        return self.address

    def is_contiguous(self):
        return True

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()


class Library:
    """Calls by name; `need` bytes of workspace, and what a call does, by its rows."""

    def __init__(self):
        self.calls, self.need, self.during = [], lambda rows: 0, lambda name, args: None

    def __getattr__(self, name):
        def call(*args):
            return self.called(name, args)
        return call

    def called(self, name, args):
        if name in ("dfq_init", "dfq_destroy"):
            return 0
        if name == "dfq_last_error":
            return b"recorded"
        self.calls.append((name, args))
        if name.endswith("workspace_bytes"):
            rows = args[1] if name == "dfq_token_logprobs_workspace_bytes" else args[6]
            n = getattr(args[-1], "_obj", args[-1])
            n.value = self.need(rows)
            self.during(name, args)
            return 0
        if name in ("dfq_token_logprobs", "dfq_cache_attention"):
            rows = args[3] if name == "dfq_token_logprobs" else args[12]
            if args[-2] < self.need(rows):
                return WORKSPACE
        self.during(name, args)
        return 0


@pytest.fixture
def lib(monkeypatch):
    """The recording library, with outputs in host memory and stream 0 current."""
    fake = Library()
    empty = torch.empty
    fake.current = 0
    monkeypatch.setattr(dflash_qmm, "load_library", lambda path=None: fake)
    monkeypatch.setattr(dflash_qmm, "_current_stream", lambda device: fake.current)

    def allocate(*shape, device=None, **kw):
        t = empty(*shape, **kw)
        fake.calls.append(("allocate", (t.data_ptr(), fake.current)))
        return t
    monkeypatch.setattr(torch, "empty", allocate)
    return fake


def in_threads(*calls):
    """Runs the calls in a thread each, 20 ms apart; the first error is raised."""
    errors = []

    def guarded(i, f):
        time.sleep(0.02 * i)
        try:
            f()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=a) for a in enumerate(calls)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


def test_threads_growing_their_workspaces_do_not_see_each_others_size(lib):
    """Two threads on streams of their own ask for the sizes that they need at the same time."""
    ctx = dflash_qmm.Context(0)
    lib.need = lambda rows: rows << 20
    lib.during = lambda name, args: time.sleep(0.05) if name.endswith("bytes") else None
    in_threads(lambda: ctx.token_logprobs(Fake((5, 8)), stream=1),
               lambda: ctx.token_logprobs(Fake((2, 8)), stream=2))
    assert ctx._scratch[1].numel() == 5 << 20 and ctx._scratch[2].numel() == 2 << 20
