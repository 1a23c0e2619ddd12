"""The rotation and sampled-accept calls on the CPU: frequency tables, argument checks that need no
device, and the Python wrappers' checks over a library that only records."""
import ctypes
import math
import struct
from fractions import Fraction

import pytest
import torch

import dflash_qmm
from rotation_util import angle, distribution, accept
from test_verify_ops_wrappers import Fake, lib  # noqa: F401  (lib is a fixture)

MAX = 0x7fffffff


# ---- frequency tables ----------------------------------------------------------------------

@pytest.mark.parametrize("rotary", [2, 20, 64, 128, 512])
@pytest.mark.parametrize("base", [1.5, 1e4, 1e7])
def test_plain_and_divided_frequencies(rotary, base):
    plain = [base ** (-2 * i / rotary) for i in range(rotary // 2)]
    close = lambda a, b: all(abs(x - y) <= 1e-13 * abs(y) for x, y in zip(a, b))  # noqa: E731
    rope = dflash_qmm.Rope(rotary, base=base, device="cpu")
    assert close(rope.frequencies, plain) and rope.amplitude == 1.0
    half = dflash_qmm.Rope(rotary, base=base, scaling={"type": "linear", "factor": 2.0},
                           device="cpu")
    assert close(half.frequencies, [f / 2 for f in plain])
    ntk = dflash_qmm.Rope(rotary, base=base, scaling={"type": "ntk", "factor": 3.0}, device="cpu")
    wide = base * 3.0 ** (rotary / max(rotary - 2, 1))
    assert close(ntk.frequencies, [wide ** (-2 * i / rotary) for i in range(rotary // 2)])
    if rotary > 2:
        # the last pair turns as in the original over a context three times as long
        assert abs(ntk.frequencies[-1] * 3 - plain[-1]) <= 1e-12 * plain[-1]


def test_bands():
    rope = dflash_qmm.Rope(64, base=5e5, device="cpu", scaling={
        "type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
        "original_length": 8192})
    seen = set()
    for i, f in enumerate(rope.frequencies):
        plain = 5e5 ** (-2 * i / 64)
        turns = 8192 * plain / (2 * math.pi)
        if turns >= 4:
            want, kind = plain, "kept"
        elif turns <= 1:
            want, kind = plain / 8, "divided"
        else:
            mix = (turns - 1) / 3
            want, kind = mix * plain + (1 - mix) * plain / 8, "mixed"
        seen.add(kind)
        assert abs(f - want) <= 1e-12 * want
    assert seen == {"kept", "divided", "mixed"}


def test_yarn():
    length, factor = 32768, 4.0
    rope = dflash_qmm.Rope(128, base=1e6, device="cpu", scaling={
        "type": "yarn", "factor": factor, "original_length": length})
    # the pairs that turn 32 times and once over the original length, by search
    def first(turns):
        return next(i / 100 for i in range(0, 12800)
                    if length * 1e6 ** (-2 * (i / 100) / 128) / (2 * math.pi) <= turns)
    low, high = math.floor(first(32)), math.ceil(first(1) - 0.01)
    for i, f in enumerate(rope.frequencies):
        plain = 1e6 ** (-2 * i / 128)
        mix = min(1, max(0, (i - low) / (high - low)))
        assert abs(f - (mix * plain / factor + (1 - mix) * plain)) <= 1e-12 * plain, i
    assert abs(rope.amplitude - (0.1 * math.log(factor) + 1)) < 1e-6
    short = dflash_qmm.Rope(128, base=1e6, device="cpu", scaling={
        "type": "yarn", "factor": 0.5, "original_length": length})
    assert short.amplitude == 1.0


def test_turns_are_the_frequencies_mod_one_turn():
    values = [0.0, 1.0, 1e-9, 0.3, 2 * math.pi, 7.0, -1.0, -1e-30, 1e-300, 12345.678]
    rope = dflash_qmm.Rope(2 * len(values), frequencies=values, device="cpu")
    for f, t in zip(values, rope.turns.tolist()):
        part = Fraction(t % 2 ** 64, 2 ** 64)
        want = Fraction(angle(1, f)) / Fraction(angle(1, 1.0)) * (Fraction(1.0) /
                                                                 Fraction(2 * math.pi))
        off = abs(part - want) % 1
        # angle() rounds to 53 bits of a turn
        assert min(off, 1 - off) <= Fraction(1, 2 ** 50), f


def test_tables_that_are_refused():
    make = dflash_qmm.Rope
    for bad in (0, 1, 3, -2):
        with pytest.raises(ValueError):
            make(bad, device="cpu")
    for kw in ({"rotary_dim": 514}, {"rotary_dim": 64, "base": 1.0},
               {"rotary_dim": 64, "base": math.inf}, {"rotary_dim": 64, "base": math.nan},
               {"rotary_dim": 64, "scaling": {"type": "linear"}},
               {"rotary_dim": 64, "scaling": {"type": "linear", "factor": -1.0}},
               {"rotary_dim": 64, "scaling": {"type": "ntk", "factor": math.nan}},
               {"rotary_dim": 64, "scaling": {"type": "bands", "factor": 2.0}},
               {"rotary_dim": 64, "scaling": {"type": "bands", "factor": 2.0,
                                              "original_length": 10, "low_freq_factor": 4.0,
                                              "high_freq_factor": 1.0}},
               {"rotary_dim": 64, "scaling": {"type": "yarn", "factor": 2.0}},
               {"rotary_dim": 64, "scaling": {"type": "yarn", "factor": 2.0,
                                              "original_length": 10, "beta_slow": 40.0}},
               {"rotary_dim": 4, "frequencies": [1.0, math.inf]}):
        with pytest.raises(dflash_qmm.DfqError):
            make(device="cpu", **kw)
    for kw in ({"scaling": {"factor": 2.0}}, {"scaling": {"type": "other"}},
               {"scaling": {"type": "linear", "factor": 2.0, "depth": 1}},
               {"frequencies": [1.0] * 31},
               {"frequencies": [1.0] * 32, "scaling": {"type": "linear", "factor": 2.0}}):
        with pytest.raises(ValueError):
            make(64, device="cpu", **kw)
    c = dflash_qmm.load_library()
    assert c.dfq_rope_frequencies(None, None, None) == 1
    assert c.dfq_rope_turns(None, 1, None) == 1


# ---- the C calls' own checks, which come before any use of the context ---------------------

BLANK = ctypes.create_string_buffer(1 << 16)     # in place of a context
AT = 1 << 20                                     # addresses that no check looks behind


def heads(n=2, start=AT, out=AT, strides=(0,) * 6):
    return struct.pack("@PPqqqqqqi4x", start, out, *strides, n)


def table(turns=AT, rotary=64, interleaved=0, amplitude=1.0):
    return dflash_qmm._RopeTable(turns, rotary, interleaved, amplitude)


def rope_call(ctx=BLANK, rope="table", q="heads", k=None, dim=64, dtype=0, batch=1, rows=1, start=0,
              starts=None, positions=None, norms=None):
    c = dflash_qmm.load_library()
    t = table() if rope == "table" else rope
    at = ctypes.addressof(t) if t is not None else None
    q = heads() if q == "heads" else q
    if norms is None:
        return c.dfq_rope(ctx, at, q, k, dim, dtype, batch, rows, start, starts, positions, 0, None)
    qw, kw, wt, eps, offset = norms
    return c.dfq_qk_norm_rope(ctx, at, q, k, qw, kw, wt, eps, offset, dim, dtype, batch, rows,
                              start, starts, positions, None)


@pytest.mark.parametrize("norms", [None, (None, None, 0, 1e-6, 0.0)])
def test_rotations_that_are_refused(norms):
    def refused(status, **kw):
        assert rope_call(norms=norms, **kw) == status, kw
    refused(1, ctx=None)
    refused(1, q=None)
    refused(2, dtype=3)
    for dim in (0, -2, 63, 514):
        refused(2, dim=dim)
    refused(1, batch=0)
    refused(1, rows=-1)
    if norms is None:
        refused(1, rope=None)
    refused(1, rope=table(turns=None))
    refused(1, rope=table(turns=AT + 4))
    for rotary in (0, 3, 66, -2):
        refused(2, rope=table(rotary=rotary))
    refused(1, rope=table(amplitude=math.nan))
    refused(1, q=heads(start=0))
    refused(1, q=heads(out=0))
    refused(1, q=heads(start=AT + 1))
    refused(1, q=heads(out=AT + 2), dtype=2)
    refused(1, q=heads(0))
    refused(1, k=heads(-1))
    refused(1, k=heads(start=0))
    refused(1, starts=AT + 2)
    refused(1, positions=AT + 1)
    refused(1, positions=AT, start=1)
    refused(1, positions=AT, starts=AT)
    refused(2, batch=1 << 16, rows=1 << 16)
    refused(2, q=heads(MAX), k=heads(MAX))


def test_rotations_past_a_launch_are_refused():
    """More heads of a token than a lane's counting holds, and grids of 2^32 threads and more (a
    wave a head where chunks do not fit)."""
    for n in (65536, MAX):
        assert rope_call(q=heads(n)) == 2
        assert rope_call(k=heads(n)) == 2
    assert rope_call(rope=table(rotary=12), dim=12, batch=1 << 13, rows=1 << 13) == 2


def test_norms_that_are_refused():
    for norms, status in (((AT, AT, 1, 1e-6, 0.0), 2), ((AT + 1, None, 0, 1e-6, 0.0), 1),
                          ((None, AT + 2, 2, 1e-6, 0.0), 1), ((AT, AT, 0, -1e-6, 0.0), 1),
                          ((AT, AT, 0, math.nan, 0.0), 1), ((AT, AT, 0, 1e-6, math.inf), 1)):
        assert rope_call(norms=norms) == status, norms


def accept_call(ctx=BLANK, logits=AT, strides=(9, 9), draft_logits=None, draft_strides=(9, 9),
                batch=2, rows=3, V=9, dtype=0, drafts=AT, lengths=None, uniforms=AT, t=None,
                temperature=1.0, dt=None, draft_temperature=1.0, tokens=AT, accepted=AT,
                chances=AT, ws=AT, ws_bytes=1 << 30):
    c = dflash_qmm.load_library()
    return c.dfq_sample_accept(ctx, logits, *strides, draft_logits, *draft_strides, batch, rows, V,
                               dtype, drafts, lengths, uniforms, t, temperature, dt,
                               draft_temperature, tokens, accepted, chances, ws, ws_bytes, None)


def test_accepts_that_are_refused():
    def refused(status, **kw):
        assert accept_call(**kw) == status, kw
    refused(1, ctx=None)
    for name in ("batch", "rows", "V"):
        refused(1, **{name: 0})
    refused(2, rows=65)
    refused(2, V=MAX // 2 + 1)
    refused(2, dtype=3)
    for name in ("logits", "uniforms", "tokens", "accepted", "drafts"):
        refused(1, **{name: None})
    refused(1, strides=(-9, 9))
    refused(1, strides=(9, -9))
    refused(1, draft_logits=AT, draft_strides=(9, -1))
    for name in ("drafts", "lengths", "uniforms", "t", "dt", "tokens", "accepted", "chances"):
        refused(1, **{name: AT + 2})
    refused(1, logits=AT + 1)
    refused(1, logits=AT + 2, dtype=2)
    refused(1, draft_logits=AT + 1)
    for bad in (-1.0, math.inf, math.nan):
        refused(1, temperature=bad)
        refused(1, draft_logits=AT, draft_temperature=bad)
    refused(3, ws=None)
    refused(3, ws_bytes=8)
    refused(1, ws=AT + 8)
    refused(2, batch=MAX, rows=1, drafts=None, V=10 ** 6, ws_bytes=1 << 62)
    # more workgroups than a launch has
    refused(2, batch=1 << 24, rows=1, drafts=None, V=1, ws_bytes=1 << 62)
    refused(2, batch=1 << 23, rows=64, V=1, ws_bytes=1 << 62)
    refused(2, batch=MAX, rows=64, V=MAX // 2, ws_bytes=1 << 62)
    c = dflash_qmm.load_library()
    n = ctypes.c_size_t(7)
    assert c.dfq_sample_accept_workspace_bytes(None, 1, 1, 9, 0, 0, ctypes.byref(n)) == 1
    assert n.value == 0
    assert c.dfq_sample_accept_workspace_bytes(BLANK, 1, 1, 9, 0, 0, None) == 1
    assert c.dfq_sample_accept_workspace_bytes(BLANK, 1, 65, 9, 0, 0, ctypes.byref(n)) == 2
    assert c.dfq_sample_accept_workspace_bytes(BLANK, 1, 2, 9, 0, 1, ctypes.byref(n)) == 0
    assert n.value > 0


# ---- the wrappers --------------------------------------------------------------------------

@pytest.fixture(autouse=True)
def like(monkeypatch):
    """torch.empty_like of such a tensor, as the recording library's fixture has torch.empty."""
    monkeypatch.setattr(torch, "empty_like", lambda t, dtype=None, memory_format=None:
                        torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device))


class Tensor(Fake):
    """A Fake with strides of its own, whose dtype torch knows."""

    def __init__(self, shape, dtype=torch.bfloat16, device="cuda:0", strides=None):
        super().__init__(shape, dtype, device)
        self.strides = strides

    def stride(self, i=None):
        s = self.strides or super().stride()
        return s if i is None else s[i]

    def is_contiguous(self):
        return self.strides is None


def rope_on(device="cuda:0"):
    r = dflash_qmm.Rope.__new__(dflash_qmm.Rope)
    r._table = table()
    r.table, r.turns = ctypes.addressof(r._table), Tensor((32,), torch.int64, device)
    r.index = r.turns.get_device()
    return r


def test_rotation_arguments_reach_the_library(lib):  # noqa: F811
    ctx = dflash_qmm.Context(0)
    fused = (7 * 640, 640, 64, 1)
    q, k = Tensor((2, 7, 6, 64), strides=fused), Tensor((2, 7, 2, 64), strides=fused)
    starts = Tensor((2,), torch.int32)
    q_out, _ = ctx.rope(rope_on(), q, k, start=5, starts=starts, inverse=True)
    name, args = [c for c in lib.calls if c[0] != "allocate"][-1]
    assert name == "dfq_rope"
    got = struct.unpack("@PPqqqqqqi4x", args[2])
    assert got[2:5] == fused[:3] and got[5:8] == (7 * 6 * 64, 6 * 64, 64) and got[8] == 6
    assert got[1] == q_out.data_ptr()
    assert args[4:9] == (64, 0, 2, 7, 5) and args[9] == starts.data_ptr() and args[11]
    ctx.qk_norm_rope(rope_on(), q, None, Tensor((64,), torch.float32), eps=1e-5, weight_offset=1.0)
    name, args = [c for c in lib.calls if c[0] != "allocate"][-1]
    assert name == "dfq_qk_norm_rope" and args[3] is None and args[6:9] == (2, 1e-5, 1.0)


def test_rotation_wrappers_refuse(lib):  # noqa: F811
    ctx = dflash_qmm.Context(0)
    q, k, rope = Tensor((2, 7, 6, 64)), Tensor((2, 7, 2, 64)), rope_on()
    w = Tensor((64,))
    bad = [
        (rope, Tensor((2, 7, 384))), (rope, q, Tensor((2, 6, 2, 64))),
        (rope, q, Tensor((2, 7, 2, 32))), (rope, q, Tensor((2, 7, 2, 64), torch.float16)),
        (rope, Tensor((2, 7, 6, 64), strides=(5376, 768, 128, 2))),
        (rope, Tensor((2, 7, 6, 64), device="cpu")), (rope, q, Tensor((2, 7, 2, 64), device="cpu")),
        (rope, Tensor((2, 7, 6, 64), device="cuda:1")), (rope_on("cpu"), q),
        (rope, Tensor((1 << 32, 1, 1, 64))),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            ctx.rope(*args)
        with pytest.raises(ValueError):
            ctx.qk_norm_rope(*args)
    for kw in ({"starts": Tensor((2,), torch.int64)}, {"starts": Tensor((3,), torch.int32)},
               {"positions": Tensor((2, 6), torch.int32)},
               {"positions": Tensor((2, 7), torch.int32, "cpu")}, {"start": MAX + 1},
               {"start": -MAX - 2}, {"k_out": k}, {"q_out": Tensor((2, 7, 6, 32))},
               {"q_out": Tensor((2, 7, 6, 64), torch.float16)},
               {"q_out": Tensor((2, 7, 6, 64), device="cpu")},
               # outputs whose heads share elements
               {"q_out": Tensor((2, 7, 6, 64), strides=(0, 384, 64, 1))},
               {"q_out": Tensor((2, 7, 6, 64), strides=(2688, 384, 63, 1))},
               {"q_out": Tensor((2, 7, 6, 64), strides=(2688, 300, 64, 1))}):
        with pytest.raises(ValueError):
            ctx.rope(rope, q, **kw)
    ctx.rope(rope, q, q_out=Tensor((2, 7, 6, 64), strides=(64, 128, 896, 1)))
    for weights in ((Tensor((32,)), None), (Tensor((64,), torch.float16), None),
                    (Tensor((64,), device="cpu"), None), (w, Tensor((64,), torch.float32))):
        with pytest.raises(ValueError):
            ctx.qk_norm_rope(rope, q, k, *weights)
    assert not [c for c in lib.calls if c[0] == "dfq_qk_norm_rope"]


def accept_inputs(batch=2, rows=3, V=9):
    return {"logits": Tensor((batch, rows, V)), "uniforms": Tensor((batch, rows), torch.float32),
            "drafts": Tensor((batch, rows - 1), torch.int32)}


def test_accept_wrapper_refuses(lib, monkeypatch):  # noqa: F811
    monkeypatch.setattr(torch, "Tensor", (torch.Tensor, Fake))
    ctx = dflash_qmm.Context(0)
    ctx.sample_accept(**accept_inputs())
    calls = len([c for c in lib.calls if c[0] == "dfq_sample_accept"])
    bad = [
        {"logits": Tensor((2, 27))}, {"logits": Tensor((2, 3, 9), device="cpu")},
        {"logits": Tensor((2, 3, 9), strides=(54, 18, 2))}, {"drafts": None},
        {"drafts": Tensor((2, 3), torch.int32)}, {"drafts": Tensor((2, 2), torch.int64)},
        {"drafts": Tensor((2, 2), torch.int32, "cpu")},
        {"uniforms": Tensor((2, 2), torch.float32)}, {"uniforms": Tensor((2, 3))},
        {"uniforms": Tensor((2, 3), torch.float32, "cuda:1")},
        {"draft_logits": Tensor((2, 3, 9))}, {"draft_logits": Tensor((2, 2, 9), torch.float16)},
        {"draft_logits": Tensor((2, 2, 9), strides=(36, 18, 2))},
        {"draft_logits": Tensor((2, 2, 9), device="cpu")},
        {"draft_lengths": Tensor((3,), torch.int32)}, {"draft_lengths": Tensor((2,))},
        {"temperature": Tensor((2,))}, {"temperature": Tensor((3,), torch.float32)},
        {"temperature": Tensor((2,), torch.float32, "cpu")},
        {"draft_temperature": Tensor((1,), torch.float32)},
    ]
    for kw in bad:
        with pytest.raises(ValueError):
            ctx.sample_accept(**{**accept_inputs(), **kw})
    with pytest.raises(ValueError):
        ctx.sample_accept(**{**accept_inputs(2, 2), "logits": Tensor((2, 1, 9)),
                             "uniforms": Tensor((2, 1), torch.float32)})
    assert len([c for c in lib.calls if c[0] == "dfq_sample_accept"]) == calls


# ---- the oracle of the GPU tests against known values --------------------------------------

def test_the_oracle():
    assert abs(angle(10 ** 6, 1.0) - math.fmod(10 ** 6, 2 * math.pi)) < 1e-9
    assert abs(angle(-1, 1.0) - (2 * math.pi - 1)) < 1e-12
    import numpy as np
    p = distribution(np.array([0.0, math.log(3.0)]), 1.0)
    assert np.allclose(p, [0.25, 0.75])
    assert distribution(np.array([1.0, math.nan, 5.0, 5.0]), 0.0).tolist() == [0, 0, 1, 0]
    assert distribution(np.array([1.0, math.nan]), 1.0) is None
    x = np.log(np.array([[[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]]))
    one = np.array([1.0])
    # 0.4 < 0.5 takes the draft; the token is drawn from the second row
    t, n, c, _ = accept(x, np.array([[0.4, 0.15]]), np.array([[0]]), None, None, one, one)
    assert t.tolist() == [[0, 1]] and n.tolist() == [1] and abs(c[0, 0] - 0.5) < 1e-12
    # 0.6 refuses it; 0.3 and 0.2 are left
    t, n, _, _ = accept(x, np.array([[0.6, 0.59]]), np.array([[0]]), None, None, one, one)
    assert t.tolist() == [[1, -1]] and n.tolist() == [0]
    # drawn from q = (0.8, 0.1, 0.1): min(1, 5/8), then (0, 0.2, 0.1)
    q = np.log(np.array([[[0.8, 0.1, 0.1]]]))
    t, n, c, _ = accept(x, np.array([[0.63, 0.7]]), np.array([[0]]), None, q, one, one)
    assert t.tolist() == [[2, -1]] and n.tolist() == [0] and abs(c[0, 0] - 0.625) < 1e-12
