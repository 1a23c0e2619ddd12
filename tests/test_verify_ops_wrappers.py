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

    def get_device(self):
        return self.device.index if self.is_cuda else -1

    def contiguous(self):
        return self

    def reshape(self, *shape):
        return Fake(shape, self.dtype, self.device, self.address)

    def element_size(self):
        return self.dtype.itemsize


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
            rows = args[6] if name.startswith("dfq_cache") else args[1]
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


class Stream:
    """Enters as torch.cuda.stream's context manager does."""

    def __init__(self, lib, handle):
        self.lib, self.cuda_stream = lib, handle

    def __enter__(self):
        self.before, self.lib.current = self.lib.current, self.cuda_stream

    def __exit__(self, *args):
        self.lib.current = self.before


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
    monkeypatch.setattr(torch.cuda, "ExternalStream",
                        lambda handle, device=None: Stream(fake, handle))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: Stream(fake, 0))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
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


def cache(device="cuda:0"):
    """A cache of one slot of one head of 64, capacity 64, 4 bits in groups of 64."""
    codes, rest = (1, 1, 64, 8), (1, 1, 64, 1)
    a = lambda at: (Fake(codes, torch.int32, device, at), Fake(rest, device=device),  # noqa: E731
                    Fake(rest, device=device))
    return dflash_qmm.KVCache.from_arrays(a(1 << 21), a(1 << 22), 4, 64)


def packed():
    return dflash_qmm.PackedWeight(Fake((64,), torch.uint8), 64, 512, 4, 64, 0)


def linear(ctx):
    return dflash_qmm.QuantizedLinear(ctx, Fake((64, 64), torch.int32), Fake((64, 8)),
                                      Fake((64, 8)), _handle=1)


# name -> a call with a workspace of the context's
SHARED = {
    "token_logprobs": lambda ctx: ctx.token_logprobs(Fake((5, 8)), stream=1),
    "cache_attention": lambda ctx: ctx.cache_attention(Fake((1, 1, 64)), cache(), stream=1),
    "qmm": lambda ctx: ctx.qmm(Fake((2, 512)), Fake((64, 64)), Fake((64, 8)), Fake((64, 8)), 4, 64,
                               stream=1),
    "qmm_silu_gate_up": lambda ctx: ctx.qmm_silu_gate_up(
        Fake((2, 512)), Fake((64, 64)), Fake((64, 8)), Fake((64, 8)), 4, 64, stream=1),
    "linear_forward": lambda ctx: linear(ctx)(Fake((2, 512)), stream=1),
    "qmm_packed": lambda ctx: ctx.qmm_packed(Fake((2, 512)), packed(), stream=1),
    "qmm_silu_gate_up_packed": lambda ctx: ctx.qmm_silu_gate_up_packed(Fake((2, 512)), packed(),
                                                                       stream=1),
}


@pytest.mark.parametrize("first", sorted(SHARED))
def test_calls_on_one_stream_do_not_share_a_workspace_at_once(lib, first):
    """A call makes several launches that meet in the workspace; another thread's on the same
    stream may come before or after all of them, not between."""
    ctx = dflash_qmm.Context(0)
    lib.need = lambda rows: 1 << 20
    state = {"inside": set(), "met": []}

    def during(name, args):
        # the addresses of the context's workspaces in the call
        known = {t.data_ptr() for d in (ctx._ws, ctx._scratch) for t in d.values()}
        mine = known & {a for a in args if isinstance(a, int)}
        if name.endswith("bytes") or not mine:
            return
        state["met"] += [name] if mine & state["inside"] else []
        state["inside"] |= mine
        time.sleep(0.05)
        state["inside"] -= mine
    lib.during = during
    in_threads(*[lambda: SHARED[first](ctx)] * 2)
    assert not state["met"] and any(name == "dfq_" + first for name, _ in lib.calls)


LAUNCHES = {
    "dfq_token_logprobs": lambda ctx, **kw: ctx.token_logprobs(
        Fake((5, 8)), Fake((5,), torch.int32), top_k=3, **kw),
    "dfq_cache_attention": lambda ctx, **kw: ctx.cache_attention(Fake((1, 1, 64)), cache(), **kw),
    "dfq_cache_read": lambda ctx, **kw: ctx.cache_read(cache(), 2, **kw),
}


@pytest.mark.parametrize("name", sorted(LAUNCHES))
@pytest.mark.parametrize("form", ["handle", "stream", "default"])
def test_outputs_and_workspaces_belong_to_the_stream_of_the_launch(lib, name, form):
    """What a call allocates on another stream than the current one may be dropped, and be the
    current stream's next allocation, while the launch has still to write it."""
    ctx = dflash_qmm.Context(0)
    lib.need = lambda rows: 3 << 20
    lib.current, launch = (9, 0) if form == "default" else (0, 7)
    given = Stream(lib, 7) if form == "stream" else launch
    before = lib.current
    outputs = LAUNCHES[name](ctx, stream=given)
    assert lib.current == before and outputs
    made = [args[1] for what, args in lib.calls if what == "allocate"]
    assert made and set(made) == {launch}
    assert [args[-1] or 0 for what, args in lib.calls if what == name][-1] == launch


def ints(*shape, device="cuda:0"):
    return Fake(shape, torch.int32, device)


# call, and its arrays by name with a maker of each for a device
TAKES = {
    "cache_append": (lambda ctx, **a: ctx.cache_append(a.pop("cache"), a.pop("k"), a.pop("v"), **a), {
        "cache": cache, "k": lambda d: Fake((1, 2, 64), device=d),
        "v": lambda d: Fake((1, 2, 64), device=d), "starts": lambda d: ints(1, device=d)}),
    "cache_read": (lambda ctx, **a: ctx.cache_read(a.pop("cache"), 2, **a), {
        "cache": cache, "starts": lambda d: ints(1, device=d),
        "k": lambda d: Fake((1, 2, 1, 64), device=d), "v": lambda d: Fake((1, 2, 1, 64), device=d)}),
    "cache_attention": (lambda ctx, **a: ctx.cache_attention(**a), {
        "q": lambda d: Fake((1, 2, 64), device=d), "cache": cache, "prefix": cache,
        "lengths": lambda d: ints(1, device=d), "tree": lambda d: ints(1, 2, device=d),
        "out": lambda d: Fake((1, 2, 64), device=d),
        "lse": lambda d: Fake((1, 2, 1), torch.float32, d)}),
    "token_logprobs": (lambda ctx, **a: ctx.token_logprobs(**a), {
        "logits": lambda d: Fake((3, 9), device=d), "tokens": lambda d: ints(3, device=d)}),
}


@pytest.mark.parametrize("name", sorted(TAKES))
@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
def test_arrays_that_are_not_on_the_gpu_are_refused(lib, name, where):
    """Each array of each call in host memory, or on another GPU: an error, and nothing is called."""
    ctx = dflash_qmm.Context(0)
    call, takes = TAKES[name]
    call(ctx, **{k: make("cuda:0") for k, make in takes.items()})
    assert any(what == "dfq_" + name for what, _ in lib.calls)
    for bad in takes:
        lib.calls.clear()
        with pytest.raises(ValueError):
            call(ctx, **{k: make(where if k == bad else "cuda:0") for k, make in takes.items()})
        assert not any(what.startswith("dfq_") for what, _ in lib.calls), bad


def test_a_cache_lies_on_one_device():
    part = (Fake((1, 1, 64, 8), torch.int32), Fake((1, 1, 64, 1)), Fake((1, 1, 64, 1)))
    other = (part[0], part[1], Fake((1, 1, 64, 1), device="cpu"))
    with pytest.raises(ValueError):
        dflash_qmm.KVCache.from_arrays(part, other, 4, 64)


BIG = 1 << 32
OUT_OF_RANGE = {
    "start of an append": lambda ctx: ctx.cache_append(cache(), Fake((1, 1, 64)), Fake((1, 1, 64)),
                                                       start=BIG),
    "rows of an append": lambda ctx: ctx.cache_append(cache(), Fake((1, BIG + 1, 64)),
                                                      Fake((1, BIG + 1, 64))),
    "start of a read": lambda ctx: ctx.cache_read(cache(), 1, start=-BIG),
    "rows of a read": lambda ctx: ctx.cache_read(cache(), BIG + 1, k=Fake((1, BIG + 1, 1, 64)),
                                                 v=Fake((1, BIG + 1, 1, 64))),
    "max_length": lambda ctx: ctx.cache_attention(Fake((1, 1, 64)), cache(), max_length=BIG + 5),
    "prefix_length": lambda ctx: ctx.cache_attention(Fake((1, 1, 64)), prefix=cache(),
                                                     prefix_length=BIG),
    "vocabulary": lambda ctx: ctx.token_logprobs(Fake((1, BIG + 7))),
    "rows of logits": lambda ctx: ctx.token_logprobs(Fake((BIG, 7))),
    "alternatives": lambda ctx: ctx.token_logprobs(Fake((1, 7)), top_k=BIG + 1),
    "capacity": lambda ctx: dflash_qmm.KVCache.from_arrays(
        *[(Fake((1, 1, BIG + 64, 8), torch.int32), *[Fake((1, 1, BIG + 64, 1))] * 2)] * 2, 4, 64),
}


@pytest.mark.parametrize("name", sorted(OUT_OF_RANGE))
def test_numbers_that_a_c_int_does_not_hold_are_refused(lib, monkeypatch, name):
    """Not taken modulo 2^32: a start of 2^32 would write position 0."""
    monkeypatch.setattr(torch, "empty", lambda *shape, **kw: pytest.fail("allocated"))
    ctx = dflash_qmm.Context(0)
    with pytest.raises(ValueError):
        OUT_OF_RANGE[name](ctx)
    assert not any(what == "dfq_cache_append" for what, _ in lib.calls)
