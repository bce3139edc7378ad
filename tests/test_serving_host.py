"""CPU tests of the serving operators' host side (rotary tables and scalings,
the paged 4-bit cache's sizes, every refusal): no GPU call is made.  The
refusals come before the library looks at the device, so a struct with the
engine's first fields (stream, head dim) and addresses that are never read
show them here."""
import ctypes
import math

import numpy as np
import pytest


def _table(f, m, positions):
    a = np.arange(positions, dtype=np.float64)[:, None] * f
    return np.stack([np.cos(a) * m, np.sin(a) * m], -1)


@pytest.mark.parametrize("rot", [16, 32, 64, 128])
def test_scaled_tables_match_their_formulas(sage, rot):
    base, n, pairs = 10000.0, 700, rot // 2
    i = np.arange(pairs)
    f = base ** (-2.0 * i / rot)
    R = sage.RopeScaling
    turns = 512 * f / (2 * math.pi)
    # a pair keeps its frequency above `high` turns and is stretched below `low`
    keep = np.clip((turns - 1.0) / 3.0, 0, 1)
    edge = [pairs * math.log(512 / (r * 2 * math.pi)) / math.log(base) for r in (32.0, 1.0)]
    lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
    ntk = (base * 4.0 ** (rot / (rot - 2))) ** (-2.0 * i / rot)
    cases = [(None, f, 1.0), (R.linear(4.0), f / 4, 1.0), (R.ntk(4.0), ntk, 1.0),
             (R.yarn(4.0, 512), f * (1 - ramp) + f / 4 * ramp, 0.1 * math.log(4.0) + 1.0),
             (R.yarn(4.0, 512, attention=1.25), f * (1 - ramp) + f / 4 * ramp, 1.25),
             (R.bands(8.0, 512), f * keep + f / 8 * (1 - keep), 1.0)]
    for scaling, freq, m in cases:
        got = sage.rope_table(base, rot, n, scaling)
        assert got.shape == (n, pairs, 2) and got.dtype == np.float32
        # f32 rounding (2^-24 relative) and angles of up to 700 in f64
        assert np.all(np.abs(got - _table(freq, m, n)) <= 2.0 ** -24 * 1.5 + 1e-10), scaling
    for d in (64, 128):
        if rot == d:
            assert np.array_equal(sage.rope_table(base, rot, n), sage.rope_table_1d(base, rot, n))


def test_table_refusals(sage):
    R = sage.RopeScaling
    for args in ((1.0, 64, 4), (10000.0, 24, 4), (10000.0, 0, 4), (10000.0, 144, 4), (10000.0, 64, 0),
                 (float("nan"), 64, 4), (float("inf"), 64, 4)):
        with pytest.raises(sage.SageError):
            sage.rope_table(*args)
    for bad in (R(9, 2.0), R(-1, 2.0), R.linear(0.5), R.linear(float("nan")), R.ntk(0.0), R.yarn(4.0, 0),
                R.yarn(4.0, 512, low=2.0, high=2.0), R.yarn(4.0, 512, low=0.0), R.bands(8.0, 512, low=5.0, high=4.0),
                R.yarn(4.0, 512, attention=-1.0), R.bands(8.0, -3)):
        with pytest.raises(sage.SageError):
            sage.rope_table(10000.0, 64, 4, bad)


def test_block_bytes(sage):
    for d in (64, 128):
        for page in (16, 32, 64, 128):
            # K and V nibbles, and a bf16 scale and zero per 64 channels of each
            assert sage.Kv4Cache.block_bytes(d, page) == page * (2 * d // 2 + 2 * (d // 64) * 4)
    for d, page in ((96, 16), (64, 8), (64, 48), (128, 256), (128, 0)):
        with pytest.raises(sage.SageError):
            sage.Kv4Cache.block_bytes(d, page)


class _Calls:
    """The four calls with good arguments, over an engine of which only the
    head dim is ever looked at, and addresses that are never read."""

    def __init__(self, sage, d=128):
        self.sage, self.L, self.d = sage, sage.lib(), d
        self.mem = (ctypes.c_int64 * 16)()
        self.mem[1] = d  # {stream, head_dim, ...}
        self.eng = ctypes.cast(self.mem, ctypes.c_void_p)
        self.ws_mem = (ctypes.c_int64 * 8)()
        self.ws_mem[0] = (d << 32)  # {device 0, head_dim, ...}
        self.ws = ctypes.cast(self.ws_mem, ctypes.c_void_p)

    def t(self, at=0x100000, n=1 << 30, token=None, head=None, heads=8):
        return self.sage._Tensor(at, n, 0, heads * self.d if token is None else token, self.d if head is None else head)

    def cache(self, **k):
        block = self.L.spl_sage_kv4_block_bytes(self.d, 64)
        a = dict(data=0x900000000, pages=10, page_stride=2 * block, page_tokens=64, kv_heads=2)
        a.update(k)
        return self.sage._Kv4(**a)

    def rotary(self, **k):
        a = dict(table=0x200000, positions=100, rot_dim=64, interleaved=0)
        a.update(k)
        return self.sage._Rotary(**a)

    def rope(self, dtype=0, tokens=5, heads=8, x=None, out=None, rotary=..., positions=0x300000, eng=...):
        r = self.rotary() if rotary is ... else rotary
        return self.L.spl_sage_rope(self.eng if eng is ... else eng, dtype, tokens, heads, x or self.t(),
                                    out or self.t(0x10000000), None if r is None else ctypes.byref(r), positions, 0)

    def append(self, cache=..., tokens=5, k=None, v=None, slots=0x400000, rotary=..., positions=0x300000, hq=8, q=None,
               q_out=None, eng=...):
        c = self.cache() if cache is ... else cache
        r = self.rotary() if rotary is ... else rotary
        return self.L.spl_sage_kv4_append(self.eng if eng is ... else eng, None if c is None else ctypes.byref(c),
                                          tokens, k or self.t(0x20000000, heads=2), v or self.t(0x30000000, heads=2),
                                          slots, None if r is None else ctypes.byref(r), positions, hq,
                                          q or self.t(), q_out or self.t(0x10000000))

    def read(self, cache=..., tokens=5, slots=0x400000, k=None, v=None, eng=...):
        c = self.cache() if cache is ... else cache
        return self.L.spl_sage_kv4_read(self.eng if eng is ... else eng, None if c is None else ctypes.byref(c), tokens,
                                        slots, k or self.t(0x20000000, heads=2), v or self.t(0x30000000, heads=2))

    def attend(self, ws=..., cache=..., q=None, q_start=0x500000, kv_len=0x600000, pages=0x700000, opts=None, out=None,
               lse=0x800000, eng=..., **k):
        c = self.cache() if cache is ... else cache
        a = dict(batch=3, heads=8, tokens=5, max_q=2, max_pages=4, causal=1, window=0)
        a.update(k)
        return self.L.spl_sage_kv4_attend(self.eng if eng is ... else eng, self.ws if ws is ... else ws,
                                          None if c is None else ctypes.byref(c),
                                          ctypes.byref(self.sage._Kv4Shape(**a)), q or self.t(), q_start, kv_len, pages,
                                          None if opts is None else ctypes.byref(opts), out or self.t(0x10000000), lse)

    def why(self):
        return self.L.spl_sage_last_error().decode()


@pytest.fixture
def calls(sage):
    return _Calls(sage)


def test_rope_refusals(calls):
    c = calls
    bad = [(dict(eng=None), "NULL engine"), (dict(dtype=3), "unknown type"), (dict(tokens=-1), "tokens"),
           (dict(heads=-1), "tokens"), (dict(heads=70000), "tokens"), (dict(tokens=1 << 30, heads=2), "tokens"),
           (dict(rotary=None), "NULL rotary"), (dict(positions=None), "NULL rotary"),
           (dict(rotary=c.rotary(table=None)), "NULL rotary"), (dict(rotary=c.rotary(rot_dim=24)), "multiple of 16"),
           (dict(rotary=c.rotary(rot_dim=0)), "multiple of 16"), (dict(rotary=c.rotary(rot_dim=144)), "multiple of 16"),
           (dict(rotary=c.rotary(positions=0)), "positions"), (dict(rotary=c.rotary(table=0x200008)), "16 bytes"),
           (dict(positions=0x300002), "4 bytes"), (dict(x=c.t(token=1020)), "multiples of 8"),
           (dict(x=c.t(head=-128)), "multiples of 8"), (dict(x=c.t(at=0)), "is NULL"),
           (dict(x=c.t(at=0x100008)), "16 bytes"), (dict(x=c.t(n=5 * 8 * 128 - 1)), "holds"),
           (dict(out=c.t(0x10000000, n=4000)), "holds"), (dict(out=c.t(0x10000000, token=0)), "overlap one another"),
           (dict(out=c.t(0x10000000, head=64)), "overlap one another"),
           (dict(out=c.t(0x10000000, token=512)), "overlap one another"), (dict(out=c.t(0x100010)), "overlaps x")]
    for args, text in bad:
        assert c.rope(**args) == 1 and text in c.why(), (args, c.why())
    assert c.rope(tokens=0, x=c.t(at=0)) == 0 and c.rope(heads=0) == 0  # nothing to do


def test_cache_refusals(calls):
    c = calls
    caches = [(None, "NULL cache"), (c.cache(page_tokens=8), "16, 32, 64 or 128"), (c.cache(page_tokens=65), "16, 32"),
              (c.cache(data=None), "NULL"), (c.cache(data=0x900000008), "16 bytes"), (c.cache(kv_heads=0), "KV heads"),
              (c.cache(kv_heads=-2), "KV heads"), (c.cache(pages=0), "31 bits"), (c.cache(pages=1 << 25), "31 bits"),
              (c.cache(pages=-1), "31 bits"), (c.cache(page_stride=18431), "page stride"),
              (c.cache(page_stride=18424), "page stride"), (c.cache(page_stride=-18432), "page stride"),
              (c.cache(kv_heads=3), "page stride")]
    for bad, text in caches:
        for call in (c.append, c.read, c.attend):
            assert call(cache=bad) == 1 and text in c.why(), (bad, text, c.why())


def test_append_and_read_refusals(calls):
    c = calls
    two = dict(heads=2)
    bad = [(dict(eng=None), "NULL engine"), (dict(tokens=-1), "tokens"), (dict(hq=-1), "tokens"),
           (dict(slots=None), "slots"), (dict(slots=0x400001), "slots"), (dict(rotary=None), "positions without"),
           (dict(rotary=None, positions=None), "no rotary table"), (dict(positions=None), "NULL rotary"),
           (dict(k=c.t(0x20000000, n=100, **two)), "K holds"), (dict(v=c.t(0x30000004, **two)), "V must start"),
           (dict(q=c.t(n=9)), "Q holds"), (dict(q_out=c.t(0x10000000, token=8)), "overlap one another"),
           (dict(q_out=c.t(0x100000, token=2048)), "overlaps an input"), (dict(q_out=c.t(0x20000100)), "overlaps an input"),
           (dict(q_out=c.t(0x30000100)), "overlaps an input")]
    for args, text in bad:
        assert c.append(**args) == 1 and text in c.why(), (args, c.why())
    assert c.append(tokens=0, k=c.t(at=0)) == 0
    for args, text in [(dict(eng=None), "NULL engine"), (dict(tokens=1 << 31), "tokens"), (dict(slots=None), "slots"),
                       (dict(k=c.t(at=0)), "NULL"), (dict(v=c.t(0x30000000, head=0, **two)), "overlap one another")]:
        assert c.read(**args) == 1 and text in c.why(), (args, c.why())
    assert c.read(tokens=0) == 0


def test_attend_refusals(calls):
    c, sage = calls, calls.sage
    o = sage._Options()
    sage.lib().spl_sage_default_options(ctypes.byref(o))

    def scaled(v):
        x = sage._Options.from_buffer_copy(o)
        x.softmax_scale, x.has_softmax_scale = v, 1
        return x

    norm = sage._Options.from_buffer_copy(o)
    norm.qk_norm_params = 0x1000
    other = _Calls(sage, 64)
    bad = [(dict(eng=None), "NULL engine"), (dict(ws=None), "NULL workspace"), (dict(ws=other.ws), "head dim 64"),
           (dict(heads=7), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(batch=-1), "sequences"),
           (dict(tokens=-1), "query tokens"), (dict(max_q=0), "queries"), (dict(max_q=1 << 40), "queries"),
           (dict(max_pages=0), "pages"), (dict(max_pages=1 << 25), "pages"), (dict(window=-1), "window"),
           (dict(kv_len=None), "lengths"), (dict(pages=None), "lengths"), (dict(pages=0x700002), "lengths"),
           (dict(kv_len=0x600001), "lengths"), (dict(q_start=0x500003), "lengths"),
           (dict(q_start=None), "without q_start"), (dict(q_start=None, max_q=1, tokens=2), "without q_start"),
           (dict(lse=0x800001), "lse"), (dict(q=c.t(n=10)), "Q holds"), (dict(out=c.t(0x10000008)), "output must start"),
           (dict(out=c.t(0x10000000, token=0)), "overlap one another"), (dict(out=c.t()), "overlaps Q"),
           (dict(opts=scaled(0.0)), "softmax scale"), (dict(opts=scaled(-1.0)), "softmax scale"),
           (dict(opts=scaled(float("nan"))), "softmax scale"), (dict(opts=scaled(float("inf"))), "softmax scale"),
           (dict(opts=norm), "LayerNorm")]
    for args, text in bad:
        assert c.attend(**args) == 1 and text in c.why(), (args, c.why())
    assert c.attend(batch=0) == 0 and c.attend(tokens=0) == 0


def test_wrappers_refuse_cpu_tensors(sage):
    import torch
    with pytest.raises(sage.SageError, match="rotary table"):
        sage.Rotary(torch.zeros(4, 32, 2), 64)
    with pytest.raises(sage.SageError, match="cache pool"):
        sage.Kv4Cache(torch.zeros(2, 2, sage.Kv4Cache.block_bytes(64, 16), dtype=torch.uint8), 16, 64)
    with pytest.raises(sage.SageError, match="head dim 96"):
        sage.Kv4Cache.empty(2, 2, 16, 96)


def test_struct_layouts(sage, tmp_path):
    import os
    import subprocess

    from conftest import ROOT
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "splsage.h"\nint main(void){printf("'
                   '%zu %zu %zu %zu %zu %zu %zu", sizeof(spl_sage_rotary), sizeof(spl_sage_rope_scaling),'
                   'sizeof(spl_sage_kv4), sizeof(spl_sage_kv4_shape), offsetof(spl_sage_rope_scaling, attention),'
                   'offsetof(spl_sage_kv4, kv_heads), offsetof(spl_sage_kv4_shape, window));return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(sage._Rotary), ctypes.sizeof(sage._RopeScaling), ctypes.sizeof(sage._Kv4),
                   ctypes.sizeof(sage._Kv4Shape), sage._RopeScaling.attention.offset, sage._Kv4.kv_heads.offset,
                   sage._Kv4Shape.window.offset]


@pytest.mark.parametrize("tokens", [1, 5])
def test_append_q_output_over_k_or_v(calls, tokens):
    """Q rotated in place beside K and V in one buffer is fine wherever the three lie; over a row of K or V it is not,
    in place or not (every pair of rows is compared here)."""
    c, d = calls, calls.d
    c.mem[1:] = [(-1 << 32) | d] + [-1] * 14  # an engine of device -1: no call gets past the check of the device
    base, hq, hk = 0x10000000, 4, 2

    def rows(at, token, head, heads):
        return [(at + 2 * (t * token + h * head), 2 * d) for t in range(tokens) for h in range(heads)]

    layouts = []  # (token stride, head stride) of q, k, v and where k and v begin
    packed = (hq + 2 * hk) * d
    layouts.append(((packed, d), (packed, d), hq * d, (hq + hk) * d))            # token by token
    layouts.append(((packed, d), (packed, d), (hq - 1) * d, (hq + hk) * d))      # k one head early: over q
    layouts.append(((packed, d), (packed, d), hq * d, packed))                   # v over the next token's q
    layouts.append(((d, tokens * d), (d, tokens * d), hq * tokens * d, (hq + hk) * tokens * d))  # head by head
    layouts.append(((d, tokens * d), (d, tokens * d), (hq * tokens - 1) * d, (hq + hk) * tokens * d))
    layouts.append(((packed, 2 * d), (packed, 4 * d), d, 3 * d))                 # between q's heads
    layouts.append(((packed, 2 * d), (packed, 4 * d), d, 4 * d))
    layouts.append(((packed, 2 * d), (packed, 4 * d), d + 64, 3 * d))            # half a row over
    layouts.append(((packed, d), (packed, d), -64, (hq + hk) * d))
    seen = set()
    for (qs, ks, at_k, at_v) in layouts:
        at = [base, base + 2 * at_k, base + 2 * at_v]
        q = rows(at[0], *qs, hq)
        apart = all(x + n <= y or y + m <= x for a, h in ((at[1], hk), (at[2], hk)) for x, n in rows(a, *ks, h) for y, m in q)
        for q_in in (at[0], 0x70000000):  # in place, and from elsewhere
            got = c.append(tokens=tokens, hq=hq, q=c.t(q_in, token=qs[0], head=qs[1]),
                           q_out=c.t(at[0], token=qs[0], head=qs[1]), k=c.t(at[1], token=ks[0], head=ks[1]),
                           v=c.t(at[2], token=ks[0], head=ks[1]))
            # (what is fine gets as far as the device)
            assert got != 0
            assert (got != 0 and "overlaps an input" in c.why()) == (not apart), (qs, ks, at_k, at_v, c.why())
        seen.add(apart)
    assert seen == {True, False}


def test_read_outputs_over_one_another(calls):
    """K and V of a read may lie between one another's rows, but not on them, nor on the cache."""
    c, d = calls, calls.d
    c.mem[1:] = [(-1 << 32) | d] + [-1] * 14  # an engine of device -1: no call gets past the check of the device
    at = 0x20000000
    both = dict(token=4 * d, head=d)  # K and V heads of a token side by side
    for k, v, text in ((c.t(at, heads=2), c.t(at, heads=2), "K and V overlap"),
                       (c.t(at, **both), c.t(at + 2 * d, **both), "K and V overlap"),
                       (c.t(at, token=2 * d, head=d), c.t(at + 2 * 9 * d, token=2 * d, head=d), "K and V overlap"),
                       (c.t(0x900000000, heads=2), c.t(at, heads=2), "overlaps the cache"),
                       (c.t(at, heads=2), c.t(0x900000000 + 9 * 18432, heads=2), "overlaps the cache")):
        assert c.read(k=k, v=v) == 1 and text in c.why(), c.why()
    assert c.read(k=c.t(at, **both), v=c.t(at + 4 * d, **both)) != 0 and "overlap" not in c.why()
    assert c.read(k=c.t(at, token=2 * d, head=d), v=c.t(at + 2 * 10 * d, token=2 * d, head=d)) != 0 and "overlap" not in c.why()


def test_outputs_between_the_rows_of_inputs(calls):
    """Rotation and attention into heads beside their input's in one buffer: not an overlap."""
    c, d = calls, calls.d
    c.mem[1:] = [(-1 << 32) | d] + [-1] * 14  # an engine of device -1: no call gets past the check of the device
    c.ws_mem[0] = (d << 32) | 0xffffffff
    at, wide = 0x20000000, dict(token=16 * d, head=d)
    for shift, fine in ((8 * d, True), (7 * d + 8, False), (-8 * d, True), (24 * d, True), (25 * d - 8, False)):
        for call, arg in ((c.rope, "x"), (c.attend, "q")):
            rc = call(**{arg: c.t(at, **wide), "out": c.t(at + 2 * shift, **wide)})
            assert rc != 0 and ("overlaps" in c.why()) == (not fine), (arg, shift, c.why())
