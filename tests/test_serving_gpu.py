"""The serving operators on the GPU against plain 64-bit forms: rotary
positions (both layouts, part of the head, three types, the gradient), tokens
into and out of the paged 4-bit cache (to the bit), attention over it (ragged
batches, one token to pieces of prompts, every mask), the way they are used
together, and calls at their edges.

Tolerances count the roundings: half a step of the output's type (bf16 2^-8,
f16 2^-11, f32 2^-24 relative), for attention also the one rounding to f16
of a probability times its V scale, and f32 sums."""
import importlib
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
sage = importlib.import_module("sota-papers-lab_b200")

DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def engines():
    made = {d: sage.SageAttention(torch.cuda.current_stream(), d) for d in (64, 128)}
    made.update({("ws", d): made[d].kv4_workspace() for d in (64, 128)})
    yield made
    for d in (64, 128):
        made[d].engine_status()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rand(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def table(rot, n, scaling=None):
    return torch.from_numpy(sage.rope_table(10000.0, rot, n, scaling)).to(DEV)


def ints(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- rotary positions

def rotate64(x, tab, pos, rot, inter, back=False):
    cs = tab.double()[pos.long()][:, None]
    c, s = cs[..., 0], cs[..., 1] * (-1 if back else 1)
    y = x.double().clone()
    i = torch.arange(rot // 2, device=DEV)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    xa, xb = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rot,inter", [(64, 64, False), (64, 32, True), (128, 128, False), (128, 128, True),
                                         (128, 96, False), (128, 16, True), (64, 48, False)])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (7, 5), (1500, 9)])
def test_rope(engines, dtype, d, rot, inter, tokens, heads):
    g = gen(1)
    tab = table(rot, 3000, sage.RopeScaling.yarn(4.0, 1024))
    pos = torch.randint(0, 3000, (tokens,), generator=g, device=DEV, dtype=torch.int32)
    pos[-1] = 2999
    wide = rand(g, tokens, heads + 3, d, dtype=dtype)  # heads of a wider row
    x = wide[:, 2:2 + heads]
    for back in (False, True):
        out = torch.full((heads, tokens, d), 7.0, dtype=dtype, device=DEV).transpose(0, 1)  # head-major
        engines[d].rope(x, out, sage.Rotary(tab, rot, inter), pos, backward=back)
        want = rotate64(x, tab, pos, rot, inter, back)
        # three f32 roundings of terms no larger than |x| * 1.2, then the type's
        tol = HALF[dtype] * want.abs() + 3 * 2.0 ** -24 * 1.2 * x.double().abs().amax() + 2.0 ** -25
        assert ((out.double() - want).abs() <= tol).all()
        assert torch.equal(out[..., rot:], x[..., rot:])
        keep = wide.clone()
        engines[d].rope(x, x, sage.Rotary(tab, rot, inter), pos, backward=back)  # in place
        assert torch.equal(x, out) and torch.equal(wide[:, :2], keep[:, :2]) and torch.equal(wide[:, 2 + heads:],
                                                                                               keep[:, 2 + heads:])
        wide.copy_(keep)
    engines[d].engine_status()


def test_rope_gradient_is_the_transposed_rotation(engines):
    """<R x, w> differs by <e, R^T w> when x moves by e (exactly, being linear), f32 rounding aside."""
    g, d, rot = gen(2), 128, 64
    tab, pos = table(rot, 50, sage.RopeScaling.yarn(4.0, 16)), ints([0, 3, 49, 17])
    x, w, e = (rand(g, 4, 3, d, dtype=torch.float32) for _ in range(3))
    r = sage.Rotary(tab, rot, True)
    y0, y1, back = (torch.empty_like(x) for _ in range(3))
    engines[d].rope(x, y0, r, pos)
    engines[d].rope(x + e, y1, r, pos)
    engines[d].rope(w, back, r, pos, backward=True)
    left = ((y1.double() - y0.double()) * w.double()).sum()
    right = (((x + e).double() - x.double()) * back.double()).sum()
    n = x.numel()
    # each element is off by a few f32 roundings of numbers below 16; they add up at most like n of them
    assert (left - right).abs() <= n * 8 * 2.0 ** -24 * 16 * float(w.abs().max())
    want = rotate64(w, tab, pos, rot, True, True)
    assert (back.double() - want).abs().max() <= 4 * 2.0 ** -24 * 1.2 * float(w.abs().max())


def test_rope_positions_out_of_the_table(engines):
    eng, g = engines[64], gen(3)
    x, tab = rand(g, 5, 2, 64), table(64, 10)
    out = torch.full_like(x, 3.0)
    eng.rope(x, out, sage.Rotary(tab, 64), ints([0, -1, 9, 10, 2**31 - 1]))
    assert (out[[1, 3, 4]] == 3.0).all() and (out[[0, 2]] != 3.0).any()
    with pytest.raises(sage.SageError):
        eng.engine_status()
    eng.engine_status()  # cleared


# ---------------------------------------------------------------- the cache

def quantise(x):
    """The stored form of f32 rows [..., D], by numpy's IEEE f32 operations:
    n uint8 [..., D], scale and zero as f32 [..., D/64]."""
    x = x.reshape(*x.shape[:-1], -1, 64)
    bf = lambda v: torch.from_numpy(np.ascontiguousarray(v)).bfloat16().float().numpy()  # noqa: E731
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1), x.max(-1)
        rng = (hi - lo).astype(np.float32)
        zero, scale = bf(lo), bf(rng * np.float32(1.0 / 15.0))
        bad = ~(np.isfinite(x).all(-1) & np.isfinite(rng) & np.isfinite(zero) & np.isfinite(scale))
        flat = scale < np.float32(2.0 ** -100)
        scale[flat] = 0
        n = np.rint((x - zero[..., None]) / scale[..., None])
        n[np.broadcast_to((bad | flat)[..., None], n.shape)] = 0
        n = np.clip(n, 0, 15).astype(np.uint8)
    scale[bad] = zero[bad] = np.nan
    return n.reshape(*n.shape[:-2], -1), scale, zero


def parts(pool, page, d):
    """Views of a pool (numpy uint8): K and V bytes [pages][heads][P][D/2], K
    and V parameter bits uint16 [pages][heads][P][D/64][2]."""
    v, p = page * d // 2, page * d // 64 * 4
    cut = [0, v, 2 * v, 2 * v + p, 2 * v + 2 * p]
    a = [pool[..., i:j].reshape(*pool.shape[:2], page, -1) for i, j in zip(cut, cut[1:])]
    return [a[0], a[1]] + [np.ascontiguousarray(x).view(np.uint16).reshape(*x.shape[:3], d // 64, 2) for x in a[2:]]


def held(pool, page, d):
    """The values a pool stands for, f64 K and V [pages][heads][P][D] (CUDA)."""
    kb, vb, kp, vp = parts(pool.cpu().numpy(), page, d)
    got = []
    for b, p in ((kb, kp), (vb, vp)):
        n = np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:3], d // 64, 64).astype(np.float64)
        s = torch.from_numpy(p.astype(np.int32) << 16).view(torch.float32).double().numpy()
        with np.errstate(invalid="ignore"):
            got.append(torch.from_numpy((s[..., 1:] + s[..., :1] * n).reshape(*b.shape[:3], d)).to(DEV))
    return got


def f32_rotate(x, tab, pos, rot, inter):
    cs = tab[pos.long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    y = x.float().clone()
    i = torch.arange(rot // 2, device=DEV)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    xa, xb = x.float()[..., a], x.float()[..., b]
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def check_append(eng, d, page, rot, inter, tokens, hkv, hq, k, v, q, seed=0):
    g = gen(seed + 50)
    pages = 2 * tokens // page + 3
    pool = torch.randint(0, 256, (pages, hkv, sage.Kv4Cache.block_bytes(d, page)), generator=g, device=DEV,
                         dtype=torch.int32).to(torch.uint8)
    before = pool.cpu().numpy().copy()
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].int()
    if tokens > 2:
        slots[1] = -1
    tab = table(rot, 5000) if rot else None
    pos = torch.randint(0, 5000, (tokens,), generator=g, device=DEV, dtype=torch.int32) if rot else None
    cache = sage.Kv4Cache(pool, page, d)
    more = {}
    if rot:
        more = dict(rotary=sage.Rotary(tab, rot, inter), positions=pos)
    if hq:
        q_out = torch.zeros(tokens, hq, d, dtype=torch.bfloat16, device=DEV)
        more.update(q=q, q_out=q_out)
    eng.kv4_append(cache, k, v, slots, **more)
    kr = f32_rotate(k, tab, pos, rot, inter) if rot else k.float()
    want = before.copy()
    block = [quantise(x.float().cpu().numpy()) for x in (kr, v)]
    half, par, ng = page * d // 2, page * d // 64 * 4, d // 64
    for t, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        p, r = divmod(slot, page)
        for i, (n, scale, zero) in enumerate(block):
            byte = n[t, :, 0::2] | (n[t, :, 1::2] << 4)
            want[p, :, i * half + r * d // 2:i * half + (r + 1) * d // 2] = byte
            bits = torch.from_numpy(np.stack([scale[t], zero[t]], -1)).bfloat16().view(torch.int16).numpy()
            at = 2 * half + i * par + r * ng * 4
            want[p, :, at:at + ng * 4] = bits.reshape(hkv, -1).view(np.uint8)
    got = pool.cpu().numpy()
    a, b = parts(got, page, d), parts(want, page, d)
    for i in (0, 1):
        assert np.array_equal(a[i], b[i]), ("K values", "V values")[i]
    for i in (2, 3):  # parameters as numbers: any NaN, either zero
        x, y = (torch.from_numpy(w[i].astype(np.int32) << 16).view(torch.float32) for w in (a, b))
        assert torch.equal(torch.nan_to_num(x, nan=123.5), torch.nan_to_num(y, nan=123.5)), ("K params", "V params")[i - 2]
    if hq:
        assert torch.equal(q_out, f32_rotate(q, tab, pos, rot, inter).bfloat16())
    ko, vo = (torch.full((tokens, hkv, d), 5.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    eng.kv4_read(cache, slots, ko, vo)
    kh, vh = held(pool, page, d)
    p, r = (slots.clamp(min=0) // page).long(), (slots.clamp(min=0) % page).long()
    for o, h in ((ko, kh), (vo, vh)):
        w = h[p, :, r].float().bfloat16()  # scale * n is exact, the sum rounds once to f32, then to bf16
        w[slots < 0] = 0
        assert torch.equal(torch.nan_to_num(o, nan=99.0), torch.nan_to_num(w, nan=99.0))
    eng.engine_status()
    return pool


@pytest.mark.parametrize("d,page,rot,inter", [(128, 64, 128, False), (64, 16, 64, False), (128, 16, 64, True),
                                              (64, 128, 16, True), (128, 32, 96, False), (64, 32, 0, False),
                                              (128, 128, 48, True)])
@pytest.mark.parametrize("tokens,hkv,hq", [(1, 1, 0), (5, 2, 6), (130, 3, 7), (700, 8, 32)])
def test_append_and_read(engines, d, page, rot, inter, tokens, hkv, hq):
    if not rot:
        hq = 0
    g = gen(tokens + d)
    qkv = rand(g, tokens, hq + 2 * hkv, d)
    check_append(engines[d], d, page, rot, inter, tokens, hkv, hq, qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], qkv[:, :hq])


@pytest.mark.parametrize("d", [64, 128])
def test_append_of_uncommon_values(engines, d):
    """Constant groups, ties, tiny and huge ranges, NaN and infinities, each in a group of its own."""
    g, tokens = gen(9), 12
    k, v = rand(g, tokens, 2, d).float(), rand(g, tokens, 2, d).float()
    k[0] = 0.0
    k[1] = -3.25
    k[2, :, :64] = torch.arange(64, device=DEV) % 16          # exactly on the steps
    k[3, :, :64] = (torch.arange(64, device=DEV) % 31) / 2    # ties between two of them
    k[4] *= 2.0 ** -110
    k[5] *= 2.0 ** 125
    k[6, 0, 3], k[6, 1, d - 1] = math.nan, math.inf
    k[7, 0, 0], k[7, 1, 63] = -math.inf, math.nan
    v[0, 0, 0], v[1, 1, d - 1], v[2] = math.nan, -math.inf, 1.0
    v[3, :, 0], v[3, :, 1] = 3.38e38, -3.38e38                # a range beyond f32
    v[4] *= 1e-39                                             # subnormal
    k, v = k.bfloat16(), v.bfloat16()
    check_append(engines[d], d, 16, 0, False, tokens, 2, 0, k, v, None)
    check_append(engines[d], d, 16, 32, True, tokens, 2, 0, k, v, None)


def test_append_bad_slots_and_positions(engines):
    eng, g, d, page = engines[128], gen(11), 128, 16
    pool = torch.full((3, 2, sage.Kv4Cache.block_bytes(d, page)), 0xAB, dtype=torch.uint8, device=DEV)
    before = pool.clone()
    k, v, q = rand(g, 4, 2, d), rand(g, 4, 2, d), rand(g, 4, 4, d)
    out = torch.full_like(q, 2.0)
    r = sage.Rotary(table(128, 8), 128)
    eng.kv4_append(sage.Kv4Cache(pool, page, d), k, v, ints([48, 2**31 - 1, 5, -1]), rotary=r,
                   positions=ints([0, 1, 8, -1]), q=q, q_out=out)
    assert torch.equal(pool, before) and (out == 2.0).all()
    with pytest.raises(sage.SageError):
        eng.engine_status()
    ko, vo = torch.full_like(k, 4.0), torch.full_like(v, 4.0)
    eng.kv4_read(sage.Kv4Cache(pool, page, d), ints([48, 47, -5, 2**31 - 1]), ko, vo)
    assert (ko[[0, 3]] == 4.0).all() and (ko[2] == 0).all()
    with pytest.raises(sage.SageError):
        eng.engine_status()
    eng.engine_status()


def test_pool_of_strided_pages(engines):
    """A pool that is every second page of a larger buffer, its heads cut from more."""
    eng, g, d, page = engines[64], gen(12), 64, 32
    block = sage.Kv4Cache.block_bytes(d, page)
    big = torch.full((8, 5, block), 0x5A, dtype=torch.uint8, device=DEV)
    pool = big[::2, 1:3]
    k, v = rand(g, 6, 2, d), rand(g, 6, 2, d)
    slots = ints([0, 31, 32, 127, 70, 64])
    eng.kv4_append(sage.Kv4Cache(pool, page, d), k, v, slots)
    dense = torch.full((4, 2, block), 0x5A, dtype=torch.uint8, device=DEV)
    eng.kv4_append(sage.Kv4Cache(dense, page, d), k, v, slots)
    assert torch.equal(pool, dense)
    assert (big[1::2] == 0x5A).all() and (big[:, 0] == 0x5A).all() and (big[:, 3:] == 0x5A).all()


# ---------------------------------------------------------------- attention

class Batch:
    """A cache filled with `kv` tokens a sequence, pages in a shuffled order,
    ids behind the last needed page wild, and everything behind the last token
    NaN; qn query tokens a sequence."""

    def __init__(self, d, page, hq, hkv, kv, qn, seed=0, kscale=1.0, tail_rows=2):
        g = gen(seed)
        self.d, self.page, self.hq, self.hkv, self.kv, self.qn = d, page, hq, hkv, kv, qn
        need = [-(-n // page) for n in kv]
        pages = sum(need) + 2
        block = sage.Kv4Cache.block_bytes(d, page)
        self.pool = torch.full((pages, hkv, block), 0xFF, dtype=torch.uint8, device=DEV)  # bf16 0xffff: NaN
        order = torch.randperm(pages, generator=g, device=DEV).cpu()
        most = max(max(need), 1) + 1
        ids = torch.full((len(kv), most), -7, dtype=torch.int32)
        ids[:, -1] = 2**31 - 1
        at, slots = 0, []
        for i, n in enumerate(need):
            ids[i, :n] = order[at:at + n]
            j = torch.arange(kv[i])
            slots.append(ids[i].long()[j // page] * page + j % page)
            at += n
        self.pages = ids.to(DEV)
        self.slots = torch.cat(slots).int().to(DEV)
        total = sum(kv)
        offset = torch.randn(hkv, d, generator=g, device=DEV)
        k = (torch.randn(total, hkv, d, generator=g, device=DEV) * kscale + offset).bfloat16()
        v = rand(g, total, hkv, d)
        self.eng = None
        self.k, self.v = k, v
        self.kv_len = ints(kv)
        starts = np.concatenate([[0], np.cumsum(qn)])
        self.q_start = ints(starts)
        self.q = rand(g, int(starts[-1]) + tail_rows, hq, d)
        self.out = torch.full_like(self.q, 3.0)
        self.lse = torch.full((self.q.shape[0], hq), 5.0, device=DEV)

    def fill(self, eng):
        if self.slots.numel():
            eng.kv4_append(sage.Kv4Cache(self.pool, self.page, self.d), self.k, self.v, self.slots)

    def attend(self, eng, ws, **k):
        a = dict(q_start=self.q_start, max_q=max(max(self.qn), 1), lse=self.lse)
        a.update(k)
        eng.kv4_attend(ws, sage.Kv4Cache(self.pool, self.page, self.d), self.q, self.out, self.pages, self.kv_len, **a)

    def check(self, causal=True, window=0, scale=None, what=""):
        d, hq, hkv, g = self.d, self.hq, self.hkv, self.hq // self.hkv
        scale = d ** -0.5 if scale is None else scale
        kb, vb, kp, vp = parts(self.pool.cpu().numpy(), self.page, d)
        kh, vh = held(self.pool, self.page, d)
        vs = torch.from_numpy(vp.astype(np.int32)[..., 0] << 16).view(torch.float32).double().to(DEV)
        vn = torch.from_numpy(np.stack([vb & 15, vb >> 4], -1).reshape(*vb.shape[:3], d)).to(DEV).double()
        row = 0
        for b, (n, qn) in enumerate(zip(self.kv, self.qn)):
            if qn == 0:
                continue
            p = self.pages[b, :-(-n // self.page)].long()
            k, v = (x[p].transpose(1, 2).reshape(-1, hkv, d)[:n] for x in (kh, vh))
            # a probability times its V scale is rounded to f16, by at most 2^-11; it weighs n
            w = vn[p].transpose(1, 2).reshape(-1, hkv, d)[:n] * vs[p].transpose(1, 2).reshape(
                -1, hkv, d // 64)[:n].repeat_interleave(64, -1)
            j = torch.arange(n, device=DEV)
            at = n - qn + torch.arange(qn, device=DEV)[:, None]
            see = torch.ones(qn, n, dtype=torch.bool, device=DEV)
            if causal:
                see &= j <= at
            if window:
                see &= j > at - window
            for h in range(hkv):
                q = self.q[row:row + qn, h * g:(h + 1) * g].double()
                x = torch.einsum("tgd,kd->tgk", q, k[:, h]) * scale
                # f32 sums of scores: 24 roundings (products' sums of 4 steps per group, parameters) of the terms' size
                most = 4 * w[:, h].amax() + 2 * k[:, h].abs().amax() if n else 0.0
                size = q.abs().sum(-1) * most * scale
                x = torch.where(see[:, None], x, -math.inf)
                lse = torch.logsumexp(x, -1) if n else torch.full((qn, g), -math.inf, dtype=torch.float64, device=DEV)
                pr = torch.where(see[:, None], torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
                o = torch.einsum("tgk,kd->tgd", pr, v[:, h])
                off = 24 * 2.0 ** -24 * size + 2.0 ** -20
                tol = (2.0 ** -8 * o.abs() + 2.0 ** -11 * torch.einsum("tgk,kd->tgd", pr, w[:, h])
                       + (2 * off[..., None]) * (v[:, h].abs().amax() if n else 0.0) + 1e-30)
                if max(self.qn) * g > 128:  # many rows: V's values and the probabilities are rounded to f16 (2^-11)
                    tol = tol + 2 * 2.0 ** -11 * torch.einsum("tgk,kd->tgd", pr, v[:, h].abs())
                got = self.out[row:row + qn, h * g:(h + 1) * g].double()
                bad = (got - o).abs() > tol
                assert not bad.any(), (what, b, h, bad.nonzero()[:4].tolist(), (got - o).abs().max().item())
                assert torch.isfinite(got).all()
                if self.lse is not None:
                    gl = self.lse[row:row + qn, h * g:(h + 1) * g].double()
                    same = (gl == lse) | ((gl - lse).abs() <= off + 2.0 ** -22 * lse.abs())
                    assert same.all(), (what, b, h, (gl - lse).abs().max().item())
            row += qn
        assert (self.out[row:] == 3.0).all() and (self.lse is None or (self.lse[row:] == 5.0).all())  # rows behind the last sequence


HEADS = [(8, 2), (4, 4), (7, 1), (32, 8), (12, 1), (24, 1), (3, 1)]


@pytest.mark.parametrize("d,page", [(64, 16), (64, 128), (128, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_attend_single_tokens(engines, d, page, hq, hkv):
    """Decoding steps over every kind of length, an idle sequence among them."""
    kv = [1, 2, 15, 16, 17, 31, 33, 0, 63, 64, 65, 127, 128, 129, 500, 1000, 3001]
    b = Batch(d, page, hq, hkv, kv, [1] * len(kv), seed=d + page + hq)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    b.check(what="ragged")
    b.attend(engines[d], engines["ws", d], causal=False, window=40)
    b.check(causal=False, window=40, what="window")
    engines[d].engine_status()


@pytest.mark.parametrize("d,page,hq,hkv", [(128, 64, 32, 8), (64, 16, 6, 2), (128, 16, 7, 1), (128, 128, 4, 4),
                                           (64, 64, 40, 1)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 37), (False, 130), (True, 10000)])
def test_attend_several_tokens(engines, d, page, hq, hkv, causal, window):
    """Drafted tokens and pieces of prompts: more queries than keys (rows that
    see nothing), sequences without queries, lengths of one."""
    kv, qn = [5, 300, 1, 0, 77, 129, 640, 16], [5, 3, 1, 2, 0, 129, 200, 40]
    b = Batch(d, page, hq, hkv, kv, qn, seed=hq + page)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], causal=causal, window=window)
    b.check(causal, window)
    small = Batch(d, page, hq, hkv, [4, 260, 1, 0, 33], [2, 2, 1, 2, 0], seed=hq + page + 1)
    small.fill(engines[d])
    small.attend(engines[d], engines["ws", d], causal=causal, window=window)
    small.check(causal, window, what="two tokens")
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
def test_attend_one_long_sequence(engines, d):
    """Split over the whole GPU; a softmax scale of its own, large scores."""
    b = Batch(d, 64, 8, 2, [20011], [1], seed=3, kscale=3.0)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], softmax_scale=0.5)
    b.check(scale=0.5)
    b.attend(engines[d], engines["ws", d], softmax_scale=1e-4)
    b.check(scale=1e-4)


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 4, 4)])
def test_attend_without_q_start(engines, d, hq, hkv):
    kv = [3, 90, 17, 0]
    b = Batch(d, 32, hq, hkv, kv, [1] * 4)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], q_start=None)
    b.check()


def test_attend_many_sequences(engines):
    """More sequences than a warp has lanes, more tiles than CTAs."""
    kv = [(i * 37) % 150 for i in range(300)]
    b = Batch(64, 16, 8, 4, kv, [1] * 300)
    b.fill(engines[64])
    b.attend(engines[64], engines["ws", 64])
    b.check()


def test_attend_strided_rows(engines):
    """q cut from a packed projection, out head-major."""
    d, eng = 128, engines[128]
    b = Batch(d, 64, 4, 2, [70, 9], [3, 2], tail_rows=0)
    b.fill(eng)
    wide = torch.zeros(5, 9, d, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:7] = b.q
    b.q = wide[:, 3:7]
    b.out = torch.full((4, 5, d), 3.0, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    b.attend(eng, engines["ws", d])
    b.check()


@pytest.mark.parametrize("rows", [1, 4, 40, 90])
def test_attend_nan_reaches_only_the_rows_that_see_it(engines, rows):
    """A cached NaN (K of one token, V of one group of another) spreads to
    the queries that see it and to no other; a V group's only to its channels."""
    d, eng, n = 128, engines[128], 300
    for part in ("k", "v"):
        b = Batch(d, 16, 2, 1, [n], [rows], tail_rows=0)
        at = n - rows + rows // 2  # seen by the later half of the queries
        getattr(b, part)[at, 0, 70] = math.nan
        b.fill(eng)
        b.attend(eng, engines["ws", d])
        see = torch.arange(n - rows, n, device=DEV) >= at
        nan = torch.isnan(b.out)
        if part == "k":
            assert nan[see].all() and not nan[~see].any()
        else:
            assert nan[see][..., 64:].all() and not nan[see][..., :64].any() and not nan[~see].any()
    eng.engine_status()


@pytest.mark.parametrize("rows", [1, 4, 90])
def test_attend_query_that_is_not_finite_stays_in_its_row(engines, rows):
    d, eng = 128, engines[128]
    b = Batch(d, 16, 4, 2, [300], [rows], tail_rows=0)
    b.fill(eng)
    b.attend(eng, engines["ws", d])
    right = b.out.clone()
    b.q[0, 0, 5], b.q[rows // 2, 1, 77], b.q[rows - 1, 3, 0] = math.nan, math.inf, -math.inf
    b.attend(eng, engines["ws", d])
    hit = torch.zeros(rows, 4, dtype=torch.bool, device=DEV)
    hit[0, 0] = hit[rows // 2, 1] = hit[rows - 1, 3] = True
    assert torch.equal(b.out[~hit], right[~hit]) and torch.isnan(b.out[hit]).any(-1).all()
    eng.engine_status()


@pytest.mark.parametrize("rows", [1, 9, 150])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_uneven_magnitudes(engines, d, rows):
    """Keys 50 and values 500 times as large as their neighbours', query rows
    a thousandth of the others', constant groups."""
    eng = engines[d]
    b = Batch(d, 32, 4, 2, [700], [rows], seed=rows + d, tail_rows=0)
    b.k[::97] *= 50
    b.v[5::89] *= 500
    b.v[3::50] = 0.75
    b.k[9::70] = 0.0
    b.q[::3] *= 1e-3
    b.fill(eng)
    b.attend(eng, engines["ws", d])
    b.check()


def test_index_errors_leave_other_kernels_alone(engines):
    """A bad slot sets the index bit; the projection and attention that follow
    on the same engine (whose waits look at the error word) run all the same."""
    eng, d = engines[128], 128
    g = gen(4)
    cache = sage.Kv4Cache.empty(2, 2, 16, d)
    x = rand(g, 1, 2, d)
    h = rand(g, 256, 512)
    w = rand(g, (4 + 2 + 2) * d, 512)
    q = torch.zeros(256, 4, d, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(256, 2, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q2 = q.clone()
    eng.qkv_gemm(h, w, None, None, q2, k, v, batch=1, tokens=256, heads=4, kv_heads=2)
    eng.kv4_append(cache, x, x, ints([99]))
    eng.qkv_gemm(h, w, None, None, q, k, v, batch=1, tokens=256, heads=4, kv_heads=2)
    b = Batch(d, 16, 4, 2, [300], [90], tail_rows=0)
    b.fill(eng)
    b.attend(eng, engines["ws", d])
    b.check()
    assert torch.equal(q, q2)
    with pytest.raises(sage.SageError, match="out of range"):
        eng.engine_status()
    eng.engine_status()


def test_attend_bad_indices_are_reported(engines):
    """Wild page ids, lengths and q_start stay inside the buffers, set the
    error word, and leave the other sequences right."""
    d, eng, ws = 64, engines[64], engines["ws", 64]
    b = Batch(d, 16, 2, 2, [40, 50, 60], [1, 1, 1], tail_rows=0)
    b.fill(eng)
    good = b.pages.clone()

    def run(**k):
        b.out.fill_(3.0)
        b.attend(eng, ws, **k)
        with pytest.raises(sage.SageError):
            eng.engine_status()
        return b.out.clone()

    b.attend(eng, ws)
    right = b.out.clone()
    eng.engine_status()
    b.pages[1, 1] = b.pool.shape[0]
    assert torch.equal(run()[[0, 2]], right[[0, 2]])
    b.pages[1, 1] = -1
    assert torch.equal(run()[[0, 2]], right[[0, 2]])
    b.pages.copy_(good)
    b.kv_len[0] = -3
    assert torch.equal(run()[1:], right[1:])
    b.kv_len[0] = 40
    b.q_start.copy_(ints([0, 1, 2, 9]))
    assert torch.equal(run()[:2], right[:2])
    b.q_start.copy_(ints([-5, 1, 2, 3]))
    assert torch.equal(run()[1:], right[1:])
    b.q_start.copy_(ints([0, 1, 2, 3]))
    b.attend(eng, ws)
    assert torch.equal(b.out, right)
    eng.engine_status()


def test_attend_is_reproducible_and_splits_do_not_matter_much(engines):
    d, eng, ws = 128, engines[128], engines["ws", 128]
    b = Batch(d, 64, 8, 2, [5000, 40, 9000], [1, 1, 1])
    b.fill(eng)
    b.attend(eng, ws)
    first = b.out.clone()
    for _ in range(5):
        b.attend(eng, ws)
        assert torch.equal(b.out, first)
    eng.reserve_sms(100)
    try:
        b.attend(eng, ws)
        b.check(what="fewer SMs")
    finally:
        eng.reserve_sms(0)


# ---------------------------------------------------------------- as they are used

@pytest.mark.parametrize("d,inter", [(128, False), (64, True)])
def test_decoding_loop(engines, d, inter):
    """A prompt laid down in two pieces, then tokens one by one: each step
    rotates and appends, then attends; checked against the held values."""
    eng, ws = engines[d], engines["ws", d]
    hq, hkv, page, n, rot = 8, 2, 16, 90, d // 2
    g = gen(21)
    pool = torch.zeros(12, hkv, sage.Kv4Cache.block_bytes(d, page), dtype=torch.uint8, device=DEV)
    cache = sage.Kv4Cache(pool, page, d)
    pages = torch.randperm(12, generator=g, device=DEV).int()[None, :8].contiguous()
    r = sage.Rotary(table(rot, 200), rot, inter)
    x = rand(g, n, hq + 2 * hkv, d)
    got = torch.zeros(n, hq, d, dtype=torch.bfloat16, device=DEV)
    rotated = torch.zeros(n, hq, d, dtype=torch.bfloat16, device=DEV)
    at = 0
    for step in [50, 30] + [1] * 10:
        sl = slice(at, at + step)
        pos = torch.arange(at, at + step, device=DEV, dtype=torch.int32)
        slots = (pages[0].long()[pos.long() // page] * page + pos.long() % page).int()
        eng.kv4_append(cache, x[sl, hq:hq + hkv], x[sl, hq + hkv:], slots, rotary=r, positions=pos, q=x[sl, :hq],
                       q_out=rotated[sl])
        at += step
        eng.kv4_attend(ws, cache, rotated[sl], got[sl], pages, ints([at]), q_start=ints([0, step]), max_q=step)
    eng.engine_status()
    b = Batch(d, page, hq, hkv, [n], [n], tail_rows=0)
    b.pool, b.pages, b.q, b.out, b.lse = pool, pages, rotated, got, torch.zeros(n, hq, device=DEV)
    check_lse = b.lse
    b.lse = torch.zeros(n, hq, device=DEV)
    eng.kv4_attend(ws, cache, rotated, torch.zeros_like(got), pages, ints([n]), q_start=ints([0, n]), max_q=n, lse=b.lse)
    b.check()
    del check_lse


def test_read_gives_a_prefix_to_the_dense_kernel(engines):
    """The values read back are what attention over the cache sees: the
    dense kernel on them agrees within its own quantisation."""
    d, eng, n = 128, engines[128], 256
    b = Batch(d, 64, 4, 4, [n], [n], tail_rows=0)
    b.fill(eng)
    b.attend(eng, engines["ws", d])
    k, v = (torch.empty(n, 4, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    eng.kv4_read(sage.Kv4Cache(b.pool, 64, d), b.slots, k, v)
    w = eng.workspace(sage.Shape(1, 4, n, causal=True))
    o = torch.empty_like(k)
    st = sage.Strides.bthd(n, 4, d)
    eng.forward(w, *[sage.Tensor(t, st) for t in (b.q, k, v, o)])
    e = (o.float() - b.out.float()).norm() / b.out.float().norm()
    assert e < 0.04  # the reference's gate for its quantised attention (rel-L2)


def test_graph_replays_match_eager_calls(engines):
    """Append and attend captured once, replayed on new inputs, lengths and slots."""
    d, page, hq, hkv, nb = 128, 16, 8, 2, 3
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        eng = sage.SageAttention(s, d)
        ws = eng.kv4_workspace()
        pool = torch.zeros(20, hkv, sage.Kv4Cache.block_bytes(d, page), dtype=torch.uint8, device=DEV)
        twin = pool.clone()
        pages = torch.arange(18, device=DEV, dtype=torch.int32).view(nb, 6).contiguous()
        x = torch.zeros(nb, hq + 2 * hkv, d, dtype=torch.bfloat16, device=DEV)
        pos, kv, slots = (torch.zeros(nb, dtype=torch.int32, device=DEV) for _ in range(3))
        q, out = (torch.zeros(nb, hq, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        r = sage.Rotary(table(d, 128), d)

        def step(p):
            c = sage.Kv4Cache(p, page, d)
            eng.kv4_append(c, x[:, hq:hq + hkv], x[:, hq + hkv:], slots, rotary=r, positions=pos, q=x[:, :hq], q_out=q)
            eng.kv4_attend(ws, c, q, out, pages, kv)

        step(pool)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(pool)
        pool.zero_()
        twin.zero_()
        g = gen(5)
        for t in range(70):
            x.copy_(rand(g, nb, hq + 2 * hkv, d))
            n = torch.tensor([t, max(0, t - 20), t // 2], device=DEV)
            pos.copy_(n)
            kv.copy_(n + 1)
            slots.copy_((pages.long()[torch.arange(nb, device=DEV), n // page] * page + n % page))
            graph.replay()
            a = out.clone()
            step(twin)
            assert torch.equal(a, out) and torch.equal(pool, twin), t
        eng.engine_status()
    s.synchronize()
    del graph


def test_two_streams_with_workspaces_of_their_own(engines):
    """Calls in flight at once on two streams, an engine and workspace each."""
    d = 128
    sets = []
    for i in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            eng = sage.SageAttention(s, d)
            ws = eng.kv4_workspace()
            b = Batch(d, 64, 8, 2, [7000 + 999 * i, 30], [1, 1], seed=30 + i)
            b.fill(eng)
        s.synchronize()
        sets.append((s, eng, ws, b))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, eng, ws, b in sets:
            b.attend(eng, ws)
    torch.cuda.synchronize()
    for s, eng, ws, b in sets:
        b.check()
        eng.engine_status()


def test_long_cache_passes_32_bit_offsets(engines):
    """Slots and pages whose byte offsets pass 2^32: the pool is 6 GB, its last
    pages are used."""
    d, page, hkv = 128, 128, 8
    eng, ws = engines[d], engines["ws", d]
    block = sage.Kv4Cache.block_bytes(d, page)
    pages = 6 * 10**9 // (block * hkv)
    pool = torch.empty(pages, hkv, block, dtype=torch.uint8, device=DEV)
    g = gen(8)
    n = 300
    ids = ints([[pages - 1, pages - 2, pages // 2 + 1]])
    k, v, q = rand(g, n, hkv, d), rand(g, n, hkv, d), rand(g, 1, 16, d)
    j = torch.arange(n, device=DEV)
    slots = (ids[0].long()[j // page] * page + j % page).int()
    cache = sage.Kv4Cache(pool, page, d)
    eng.kv4_append(cache, k, v, slots)
    ko, vo, out = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q)
    eng.kv4_read(cache, slots, ko, vo)
    small = torch.empty(3, hkv, block, dtype=torch.uint8, device=DEV)
    c2 = sage.Kv4Cache(small, page, d)
    eng.kv4_append(c2, k, v, j.int())
    k2, v2, o2 = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q)
    eng.kv4_read(c2, j.int(), k2, v2)
    eng.kv4_attend(ws, cache, q, out, ids, ints([n]))
    eng.kv4_attend(ws, c2, q, o2, ints([[0, 1, 2]]), ints([n]))
    assert torch.equal(ko, k2) and torch.equal(vo, v2) and torch.equal(out, o2)
    assert torch.equal(pool[ids[0].long()[0]], small[0])
    eng.engine_status()


def test_attend_prompt_strided_without_lse(engines):
    """Many rows, q cut from a packed projection, out head-major, no lse; a
    group of 20 heads, more sequences than a warp, some empty."""
    d, eng = 64, engines[64]
    kv = [(37 * i) % 200 for i in range(40)]
    qn = [i % 9 if i % 9 <= n else 0 for i, n in enumerate(kv)]
    b = Batch(d, 16, 40, 2, kv, qn, seed=77, tail_rows=3)
    b.fill(eng)
    n = b.q.shape[0]
    wide = torch.zeros(n, 45, d, dtype=torch.bfloat16, device=DEV)
    wide[:, 4:44] = b.q
    b.q = wide[:, 4:44]
    b.out = torch.full((40, n, d), 3.0, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    b.attend(eng, engines["ws", d], lse=None)
    b.lse = None
    b.check()
    eng.engine_status()


def test_attend_prompt_bad_indices_are_reported(engines):
    d, eng, ws = 128, engines[128], engines["ws", 128]
    b = Batch(d, 16, 2, 2, [140, 250, 260], [140, 150, 160], tail_rows=0)
    b.fill(eng)
    good = b.pages.clone()
    b.attend(eng, ws)
    right = b.out.clone()
    eng.engine_status()

    def run(keep):
        b.out.fill_(3.0)
        b.attend(eng, ws)
        with pytest.raises(sage.SageError, match="out of range"):
            eng.engine_status()
        assert torch.equal(b.out[keep], right[keep])

    for bad in (b.pool.shape[0], -1):
        b.pages[1, 3] = bad
        run(torch.tensor([*range(140), *range(290, 450)], device=DEV))
    b.pages.copy_(good)
    b.kv_len[2] = 2**31 - 1
    run(slice(0, 290))
    b.kv_len[2] = 260
    b.q_start.copy_(ints([0, 140, 290, 2**31 - 1]))
    run(slice(0, 290))
    b.q_start.copy_(ints([0, 140, 290, 450]))
    b.attend(eng, ws)
    assert torch.equal(b.out, right)
    eng.engine_status()


def test_attend_prompt_in_a_graph_and_beside_another_stream(engines):
    """Pieces of prompts captured once and replayed at other lengths, while
    single tokens run on a second stream with a workspace of its own."""
    d, page, hq, hkv, n = 128, 64, 8, 2, 200
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        eng = sage.SageAttention(s, d)
        ws = eng.kv4_workspace()
        b = Batch(d, page, hq, hkv, [1500, 900], [n, n], seed=12, tail_rows=0)
        b.fill(eng)
    s2 = torch.cuda.Stream()
    with torch.cuda.stream(s2):
        eng2 = sage.SageAttention(s2, d)
        ws2 = eng2.kv4_workspace()
        one = Batch(d, page, hq, hkv, [5000, 40], [1, 1], seed=13)
        one.fill(eng2)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            b.attend(eng, ws)
        for kv in ([1500, 900], [200, 733], [1111, 500]):
            b.kv, b.kv_len[:] = kv, ints(kv)
            b.out.fill_(3.0)
            graph.replay()
            for _ in range(3):
                with torch.cuda.stream(s2):
                    one.attend(eng2, ws2)
            s.synchronize()
            s2.synchronize()
            b.check()
            one.check()
        eng.engine_status()
        eng2.engine_status()
    del graph


def test_first_calls_of_a_process_may_be_captured():
    """Every kernel's first launch inside a capture."""
    code = """
import torch, numpy as np, sys
sys.path.insert(0, %r)
import importlib
sage = importlib.import_module("sota-papers-lab_b200")
d, page = 128, 16
s = torch.cuda.Stream()
with torch.cuda.stream(s):
    eng = sage.SageAttention(s, d)
    ws = eng.kv4_workspace()
    pool = torch.zeros(40, 2, sage.Kv4Cache.block_bytes(d, page), dtype=torch.uint8, device="cuda")
    cache = sage.Kv4Cache(pool, page, d)
    x = torch.randn(300, 8, d, device="cuda").bfloat16()
    q, out, few = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    k2, v2 = (torch.zeros(300, 2, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = torch.arange(300, device="cuda", dtype=torch.int32)
    tab = torch.from_numpy(np.ascontiguousarray(sage.rope_table(10000.0, d, 300))).cuda()
    r = sage.Rotary(tab, d)
    pages = torch.arange(40, device="cuda", dtype=torch.int32).view(1, 40)
    kv, start = (torch.tensor(t, device="cuda", dtype=torch.int32) for t in ([300], [0, 300]))
    last, lo, hi = (torch.tensor(t, device="cuda", dtype=torch.int32) for t in ([300], [0, 1], [0, 3]))
    s.synchronize()

    def run():
        eng.rope(x, q, r, at)
        eng.kv4_append(cache, q[:, :2], x[:, 2:4], at)
        eng.kv4_read(cache, at, k2, v2)
        eng.kv4_attend(ws, cache, q, out, pages, kv, q_start=start, max_q=300)
        eng.kv4_attend(ws, cache, q[299:], few[299:], pages, kv)
        eng.kv4_attend(ws, cache, q[297:], few[:3], pages, kv, q_start=hi, max_q=3)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        run()
    graph.replay()
    s.synchronize()
    a = [t.clone() for t in (q, pool, k2, v2, out, few)]
    for t in (q, pool, k2, v2, out, few):
        t.zero_()
    run()
    eng.engine_status()
    assert all(torch.equal(i, j) for i, j in zip(a, (q, pool, k2, v2, out, few))) and out.abs().sum() > 0
    del graph
""" % str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]


def test_attend_prompt_over_a_long_cache_and_shared_pages(engines):
    """Page bytes past 2^32, and two sequences that share their prefix's pages."""
    d, page, hkv, n = 64, 128, 8, 400
    eng, ws = engines[d], engines["ws", d]
    block = sage.Kv4Cache.block_bytes(d, page)
    pages = 5 * 10**9 // (block * hkv)
    g = gen(9)
    k, v, q = rand(g, n, hkv, d), rand(g, n, hkv, d), rand(g, 300, 16, d)
    j = torch.arange(n, device=DEV)
    outs = []
    for count, ids in ((pages, [pages - 1, pages - 3, pages // 2, pages - 2]), (4, [0, 1, 2, 3])):
        ids = ints([ids, ids])
        pool = torch.empty(count, hkv, block, dtype=torch.uint8, device=DEV)
        cache = sage.Kv4Cache(pool, page, d)
        eng.kv4_append(cache, k, v, (ids[0].long()[j // page] * page + j % page).int())
        out = torch.zeros_like(q)
        eng.kv4_attend(ws, cache, q, out, ids, ints([n, n - 100]), q_start=ints([0, 150, 300]), max_q=150)
        outs.append(out)
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    eng.engine_status()


@pytest.mark.parametrize("reserved", [1, 100, 10000])
def test_attend_with_reserved_sms(engines, reserved):
    """Fewer CTAs than SMs, down to one SM's, in a workspace that other calls use as well."""
    d = 128
    eng = sage.SageAttention(torch.cuda.current_stream(), d)
    ws = engines["ws", d]
    if reserved == 10000:
        reserved = torch.cuda.get_device_properties(0).multi_processor_count - 1
    eng.reserve_sms(reserved)
    few = Batch(d, 32, 8, 2, [900, 0, 3, 130], [1, 0, 1, 1], seed=40)
    some = Batch(d, 32, 8, 2, [500, 260], [4, 5], seed=41)
    many = Batch(d, 32, 8, 2, [300, 700], [150, 90], seed=42)
    for b in (few, some, many):
        b.fill(eng)
    for _ in range(2):
        for b in (few, some, many):
            b.attend(eng, ws)
            b.attend(engines[d], ws)
            b.attend(eng, ws)
    for b in (few, some, many):
        b.check()
    eng.engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,rows", [(160, 1, 1), (129, 1, 1), (128, 1, 1), (16, 2, 16), (16, 2, 17), (6, 2, 3),
                                         (5, 5, 257)])
def test_attend_around_the_kernels_limits(engines, d, hq, hkv, rows):
    """Groups of more heads than a tile has rows, and the row counts where one kernel hands over to the next."""
    b = Batch(d, 64, hq, hkv, [400, rows, 1], [rows, rows, 1], seed=hq + rows)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], window=99)
    b.check(window=99)
    engines[d].engine_status()


def test_gpu_refusals(engines):
    """What the wrappers refuse: types, shapes, devices, mixed-up arguments."""
    d, eng, ws = 128, engines[128], engines["ws", 128]
    g = gen(1)
    x = rand(g, 4, 2, d)
    r = sage.Rotary(table(64, 10), 64)
    pos = ints([0, 1, 2, 3])
    cache = sage.Kv4Cache.empty(4, 2, 16, d)
    with pytest.raises(sage.SageError):
        eng.rope(x, x.float(), r, pos)
    with pytest.raises(sage.SageError):
        eng.rope(x, torch.empty_like(x), r, pos.long())
    with pytest.raises(sage.SageError):
        eng.rope(x, torch.empty_like(x), r, pos[:3])
    with pytest.raises(sage.SageError):
        eng.rope(x.cpu(), torch.empty_like(x), r, pos)
    with pytest.raises(sage.SageError):
        eng.rope(x[..., :64], torch.empty_like(x[..., :64]), r, pos)
    with pytest.raises(sage.SageError):
        engines[64].kv4_append(cache, x, x, pos)
    with pytest.raises(sage.SageError):
        eng.kv4_append(cache, x, x, pos, rotary=r)
    with pytest.raises(sage.SageError):
        eng.kv4_append(cache, x.half(), x, pos)
    with pytest.raises(sage.SageError):
        eng.kv4_append(cache, x, x, pos, q=x)
    with pytest.raises(sage.SageError):
        eng.kv4_read(cache, pos, x[:, :1], x)
    q, o, kv, ids = rand(g, 4, 4, d), rand(g, 4, 4, d), ints([1] * 4), ints([[0]] * 4)
    for bad in (dict(q_start=pos), dict(window=-1), dict(window=2**32), dict(max_q=2), dict(softmax_scale=-1.0),
                dict(lse=torch.zeros(4, 4, device=DEV, dtype=torch.float64))):
        with pytest.raises(sage.SageError):
            eng.kv4_attend(ws, cache, q, o, ids, kv, **bad)
    with pytest.raises(sage.SageError):
        eng.kv4_attend(engines["ws", 64], cache, q, o, ids, kv)
    with pytest.raises(sage.SageError):
        eng.kv4_attend(ws, cache, rand(g, 4, 3, d), rand(g, 4, 3, d), ids, kv)
    with pytest.raises(sage.SageError):
        eng.kv4_attend(ws, cache, q, q, ids, kv)
    with pytest.raises(sage.SageError):
        sage.Kv4Cache(torch.zeros(4, 2, 100, dtype=torch.uint8, device=DEV), 16, d)
    closed = eng.kv4_workspace()
    closed.close()
    with pytest.raises(sage.SageError):
        eng.kv4_attend(closed, cache, q, o, ids, kv)
    eng.engine_status()


# ---------------------------------------------------------------- magnitudes, signs, joins

def large_query(engines, d, size, rows):
    """One query row far larger than the others, which do not change by a bit."""
    b = Batch(d, 16, 4, 2, [300], [rows], seed=rows, tail_rows=0)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    right = b.out.clone()
    b.q[rows // 2, 1] *= size
    b.attend(engines[d], engines["ws", d])
    hit = torch.zeros(rows, 4, dtype=torch.bool, device=DEV)
    hit[rows // 2, 1] = True
    assert torch.equal(b.out[~hit], right[~hit]) and torch.isfinite(b.out).all()
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [3, 5, 90])
def test_attend_large_queries_leave_other_rows_alone(engines, d, rows):
    large_query(engines, d, 1e4, rows)


def exact_attend(b, causal=True, window=0):
    """Per sequence with queries: its first row, 64-bit outputs [token][head][D], lse, and what a rounding can be
    relative to: the probabilities' products with the largest magnitude that a stored group can hold."""
    d, hkv, g = b.d, b.hkv, b.hq // b.hkv
    kh, vh = held(b.pool, b.page, d)
    row = 0
    for i, (n, qn) in enumerate(zip(b.kv, b.qn)):
        if qn and n:
            p = b.pages[i, :-(-n // b.page)].long()
            k, v = (x[p].transpose(1, 2).reshape(-1, hkv, d)[:n] for x in (kh, vh))
            top = v.unflatten(-1, (-1, 64)).abs().amax(-1).repeat_interleave(64, -1)
            j, at = torch.arange(n, device=DEV), n - qn + torch.arange(qn, device=DEV)[:, None]
            see = torch.ones(qn, n, dtype=torch.bool, device=DEV)
            if causal:
                see &= j <= at
            if window:
                see &= j > at - window
            q = b.q[row:row + qn].double().unflatten(1, (hkv, g))
            x = torch.einsum("thgd,khd->thgk", q, k) * d ** -0.5
            x = torch.where(see[:, None, None], x, -math.inf)
            lse = torch.logsumexp(x, -1)
            most = x.amax(-1, keepdim=True)
            pr = torch.exp(x - torch.where(most == -math.inf, 0.0, most))
            pr = pr / pr.sum(-1, keepdim=True).clamp(min=1e-300)
            o, size = (torch.einsum("thgk,khd->thgd", pr, y).flatten(1, 2) for y in (v, top))
            yield row, o, lse.flatten(1, 2), size
        row += qn


def check_attend(b, what, **k):
    """Against 64 bits: the output's rounding to bf16 (2^-8 of it), and of probabilities and values on the way (each
    key's part by 2^-9 of the most that its group of channels can be), scores' f32 sums (2^-15 of what they weigh:
    |scores| here are below 2^7 where they count, 2^-24 each way of up to 2^2 terms)."""
    for row, o, lse, size in exact_attend(b, **k):
        got = b.out[row:row + o.shape[0]].double()
        assert torch.isfinite(got).all(), (what, (~torch.isfinite(got)).nonzero()[:4].tolist())
        bad = (got - o).abs() > 2.0 ** -8 * o.abs() + (2.0 ** -9 + 2.0 ** -15) * size + 1e-30
        assert not bad.any(), (what, bad.nonzero()[:4].tolist(), float((got - o).abs().max()))
        gl = b.lse[row:row + o.shape[0]].double()
        assert ((gl == lse) | ((gl - lse).abs() <= 2.0 ** -15 + 2.0 ** -20 * lse.abs())).all(), (what, "lse")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e4, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("rows", [1, 5, 90])
def test_attend_scores_far_beyond_one(engines, d, size, rows):
    """Scores of up to 1e31: each row is the value of its best key, as far ahead of the second as they are large; of two
    equal keys, the mean."""
    b = Batch(d, 16, 4, 2, [400], [rows], seed=rows + d, tail_rows=0)
    b.k = (b.k.float() * size).bfloat16()
    for h in range(4):  # (a best key that is clearly the best)
        b.k[7 + 90 * h, h // 2] = (b.q[:rows, h].float().mean(0) * 8 * size).bfloat16()
    b.k[350] = b.k[7]
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    assert torch.isfinite(b.out).all()
    for row, o, lse, size64 in exact_attend(b):
        kh, _ = held(b.pool, b.page, d)
        p = b.pages[0, :25].long()
        k = kh[p].transpose(1, 2).reshape(-1, 2, d)[:400]
        x = torch.einsum("thgd,khd->thgk", b.q.double().unflatten(1, (2, 2)), k).flatten(1, 2)
        two = x.topk(3, -1).values
        # rows whose third score is behind by more than f32's rounding of scores can make up
        clear = (two[..., 0] - two[..., 2]) * d ** -0.5 > 40 + 2.0 ** -16 * two.abs().amax(-1) * d ** -0.5
        same = (two[..., 0] == two[..., 1]) | ((two[..., 0] - two[..., 1]) * d ** -0.5 > 40 + 2.0 ** -16 * two.abs().amax(-1))
        fine = clear & same & (x.abs().amax(-1) == two[..., 0].abs())
        got = b.out[row:row + rows].double()
        bad = ((got - o).abs() > 2.0 ** -8 * o.abs() + 2.0 ** -9 * size64) & fine[..., None]
        assert not bad.any()
        assert ((b.lse[row:row + rows].double() - lse).abs() <= 2.0 ** -18 * lse.abs() + 1e-4).all()
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e12, 1e30])
@pytest.mark.parametrize("rows", [3, 5, 90])
def test_attend_huge_queries_leave_other_rows_alone(engines, d, size, rows):
    large_query(engines, d, size, rows)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 6, 70])
def test_attend_scales_of_either_sign(engines, d, rows):
    """A pool that another program wrote: half of the scales negative (the largest of them the largest of all)."""
    b = Batch(d, 16, 8, 2, [500], [rows], seed=rows, tail_rows=0)
    b.v[::3] *= 8
    b.fill(engines[d])
    _, _, kp, vp = parts(b.pool.cpu().numpy(), b.page, d)
    half, par = b.page * d // 2, b.page * d // 64 * 4
    for i, p in enumerate((kp, vp)):
        p[..., 0::2, :, 0] ^= 0x8000  # every second token's scales
        at = 2 * half + i * par
        b.pool[..., at:at + par] = torch.from_numpy(p.reshape(*p.shape[:2], -1).view(np.uint8)).to(DEV)
    b.attend(engines[d], engines["ws", d])
    check_attend(b, "signs")
    engines[d].engine_status()


def huge_values(engines, d, size, rows):
    """A cached V far beyond the others', seen by the later half of the queries only, and one that all see whose
    probability is nothing: the other rows keep their precision, and the rows that see it stay finite."""
    n = 700
    b = Batch(d, 32, 4, 2, [n, 60], [rows, 1], seed=rows + d, tail_rows=0)
    hidden = n - rows + rows // 2
    b.v[hidden] *= size
    b.v[n - rows - 9, 1, 5] = size  # one channel only: its group's other values are lost in its scale
    b.v[200] *= size
    for h in range(2):
        u = torch.randn(d, generator=gen(h), device=DEV)
        b.q[:rows, 2 * h:2 * h + 2] = (u + 0.3 * b.q[:rows, 2 * h:2 * h + 2].float()).bfloat16()
        b.k[200, h] = (-30 * u).bfloat16()  # a score far below the others'
        b.k[n - rows - 9, h] = (-30 * u).bfloat16()
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    check_attend(b, "V")
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e20, 1e30, 1e32, 2e37])
@pytest.mark.parametrize("rows", [3, 5, 40])
def test_attend_huge_finite_values_stay_with_the_rows_that_see_them(engines, d, size, rows):
    huge_values(engines, d, size, rows)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e20, 1e30, 1e32, 2e37])
def test_attend_prompt_huge_finite_values_stay_with_the_rows_that_see_them(engines, d, size):
    huge_values(engines, d, size, 90)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e12, 1e30, 1e35])
@pytest.mark.parametrize("rows", [5, 40, 90])
def test_attend_huge_finite_keys_stay_with_the_rows_that_see_them(engines, d, size, rows):
    """The same of a cached K: rows that do not see it score their other keys as if it were not there."""
    n = 500
    b = Batch(d, 16, 4, 2, [n], [rows], seed=rows, tail_rows=0)
    hidden = n - rows + rows // 2
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    right, lse = b.out.clone(), b.lse.clone()
    b.k[hidden] *= size
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    before = torch.arange(rows, device=DEV) < rows // 2
    # the same scores up to f32's rounding: a step of bf16 at most, lse by a few of f32's steps of the scores
    assert ((b.out - right).abs()[before] <= 2.0 ** -7 * right.abs()[before] + 1e-3).all()
    assert ((b.lse - lse).abs()[before] <= 1e-4).all()
    assert torch.isfinite(b.out[~before]).all()
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 30, 90, 170])
@pytest.mark.parametrize("window", [0, 100])
def test_attend_of_any_magnitudes(engines, d, rows, window):
    """Every key's K and V, and every query, with a power of two of its own: each key counts as much as it weighs."""
    b = Batch(d, 32, 4, 2, [900, 333, 1500], [rows, min(rows, 64), rows], seed=rows + d, tail_rows=0)
    g = gen(rows)

    def scaled(x, low, high):
        e = torch.rand(x.shape[:2], generator=g, device=DEV)[..., None] * (high - low) + low
        return (x.float() * torch.exp2(e.round())).bfloat16()

    b.k, b.q = scaled(b.k, -30, 0), scaled(b.q, -20, 1)
    b.v = scaled(b.v, -40, 60)
    b.v[::7, 0] = 0.0
    b.k[3::11, 1] = 0.0
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], window=window)
    check_attend(b, "magnitudes", window=window)
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [4, 90])
def test_attend_far_keys_on_a_long_cache(engines, d, rows):
    """The same where tiles are cut and joined: a few huge and a few tiny keys among 9000, one V that is not finite and
    that half the queries see."""
    n = 9000
    b = Batch(d, 64, 4, 1, [n], [rows], seed=rows + d, tail_rows=0)
    b.v[::501] *= 2.0 ** 70
    b.v[100::333] *= 2.0 ** -50
    b.k[50::777] *= 2.0 ** -40
    b.v[n - rows + rows // 2, 0, 3] = math.inf
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    first = b.out.clone()
    b.attend(engines[d], engines["ws", d])
    half = rows // 2
    assert torch.equal(b.out[:half], first[:half]) and torch.isnan(b.out[half:, :, :64]).all()
    b.v[n - rows + half, 0, 3] = 1.0  # (the rows that do not see it, and its other group, are right)
    b.fill(engines[d])
    for row, o, lse, size in exact_attend(b):
        bad = (first.double() - o).abs() > 2.0 ** -8 * o.abs() + (2.0 ** -9 + 2.0 ** -15) * size
        assert not bad[:half].any() and not bad[half:, :, 64:].any()
    engines[d].engine_status()


@pytest.mark.parametrize("rows", [3, 40, 90])
@pytest.mark.parametrize("size", [1e4, 1e9, 1e25])
def test_attend_groups_of_v_far_apart(engines, rows, size):
    """One half of V's channels far larger than the other, in all keys or in some: the other keeps its precision."""
    b = Batch(128, 32, 4, 2, [700, 90], [rows, 1], seed=rows, tail_rows=0)
    b.v[:, 0, 64:] *= size
    b.v[::3, 1, :64] *= size
    b.v[1::5, 1, 64:] /= size
    b.fill(engines[128])
    b.attend(engines[128], engines["ws", 128])
    check_attend(b, "groups")
    engines[128].engine_status()


@pytest.mark.parametrize("d", [64, 128])
def test_appends_between_prompt_calls_without_a_pause(engines, d):
    """Attend, append into the page that the last call read half filled, attend again, nothing else on the stream in
    between: each call sees what was appended before it, as calls with a pause between them do."""
    eng, ws, page, n = engines[d], engines["ws", d], 64, 150
    b = Batch(d, page, 4, 2, [700], [n], seed=d, tail_rows=0)
    cache = sage.Kv4Cache(b.pool, page, d)
    steps = [range(i, i + 10) for i in range(n, 700, 10)]
    lens = [ints([s[-1] + 1]) for s in steps]
    outs = [torch.zeros(n, 4, d, dtype=torch.bfloat16, device=DEV) for _ in range(2 * len(steps))]

    def run(outs, pause):
        b.pool.zero_()
        eng.kv4_append(cache, b.k[:n], b.v[:n], b.slots[:n])
        torch.cuda.synchronize()
        for s, kv, out in zip(steps, lens, outs):
            sl = slice(s[0], s[-1] + 1)
            eng.kv4_append(cache, b.k[sl], b.v[sl], b.slots[sl])
            if pause:
                torch.cuda.synchronize()
            eng.kv4_attend(ws, cache, b.q, out, b.pages, kv, q_start=b.q_start, max_q=n)
            if pause:
                torch.cuda.synchronize()

    run(outs[:len(steps)], True)
    for _ in range(5):
        run(outs[len(steps):], False)
        assert all(torch.equal(x, y) for x, y in zip(outs, outs[len(steps):]))
    eng.engine_status()


@pytest.mark.parametrize("d,kv,rows,window", [(128, 16000, 40, 0), (64, 9000, 33, 0), (128, 20000, 75, 12000),
                                              (64, 12000, 65, 7001), (128, 8200, 65, 0)])
def test_attend_prompt_tiles_of_many_pieces(engines, d, kv, rows, window):
    """A piece of a prompt on a long cache: its tiles (the last of 160, 132, 44, 4 and 4 rows) are cut into more than
    four pieces each, joined the same way every time."""
    b = Batch(d, 64, 4, 1, [kv], [rows], seed=kv, tail_rows=1)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], window=window)
    b.check(window=window)
    first, lse = b.out.clone(), b.lse.clone()
    for _ in range(3):
        b.attend(engines[d], engines["ws", d], window=window)
        assert torch.equal(b.out, first) and torch.equal(b.lse, lse)
    engines[d].engine_status()


def kernel_nodes(graph):
    """(grid, dynamic shared memory) of a captured graph's kernels."""
    from cuda.bindings import driver
    err, _, n = driver.cuGraphGetNodes(graph.raw_cuda_graph(), 0)
    assert int(err) == 0
    err, nodes, n = driver.cuGraphGetNodes(graph.raw_cuda_graph(), n)
    assert int(err) == 0
    got = []
    for x in nodes[:n]:
        err, kind = driver.cuGraphNodeGetType(x)
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, p = driver.cuGraphKernelNodeGetParams(x)
            assert int(err) == 0
            got.append((p.gridDimX * p.gridDimY * p.gridDimZ, p.sharedMemBytes))
    return got


@pytest.mark.parametrize("reserved", [1, 20, 100])
@pytest.mark.parametrize("d,rows", [(64, 1), (128, 1), (128, 4), (128, 60)])
def test_attend_leaves_the_reserved_sms_free(d, rows, reserved):
    """No more CTAs than SMs that are not reserved, and none of them able to share an SM with another call's (two
    CTAs' shared memory is more than an SM has), so that they cannot be spread over more SMs than that either way."""
    props = torch.cuda.get_device_properties(0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        eng = sage.SageAttention(s, d)
        ws = eng.kv4_workspace()
        b = Batch(d, 32, 8, 2, [9000, 900, 4000], [rows] * 3, seed=3)
        b.fill(eng)
        eng.reserve_sms(reserved)
        b.attend(eng, ws)
        s.synchronize()
        b.check()
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph, stream=s):
            b.attend(eng, ws)
    grids = kernel_nodes(graph)
    assert len(grids) == 1
    grid, shared = grids[0]
    assert grid <= props.multi_processor_count - reserved
    assert 2 * shared > props.shared_memory_per_multiprocessor or rows == 60
    del graph


@pytest.mark.parametrize("layout", ["rows", "heads", "per head", "one head"])
def test_append_with_q_in_place(engines, layout):
    """Q rotated where it lies, K and V beside it in the same buffer: token by token, head by head, q, k and v of a
    head side by side, one head of each."""
    d, eng, t, h, page = 128, engines[128], 70, 1 if layout == "one head" else 4, 16
    g = gen(17)
    if layout == "heads":
        x = rand(g, 3 * h, t, d).transpose(0, 1)
    else:
        x = rand(g, t, 3 * h, d)
    cut = [slice(0, h), slice(h, 2 * h), slice(2 * h, 3 * h)]
    if layout == "per head":
        cut = [slice(i, 3 * h, 3) for i in range(3)]
    q, k, v = (x[:, c] for c in cut)
    r, pos, slots = sage.Rotary(table(d, 100), d), ints(range(5, 5 + t)), ints(range(t))
    pools = [torch.zeros(5, h, sage.Kv4Cache.block_bytes(d, page), dtype=torch.uint8, device=DEV) for _ in range(2)]
    out = torch.empty(t, h, d, dtype=torch.bfloat16, device=DEV)
    eng.kv4_append(sage.Kv4Cache(pools[0], page, d), k, v, slots, rotary=r, positions=pos, q=q, q_out=out)
    keep = [k.clone(), v.clone()]
    eng.kv4_append(sage.Kv4Cache(pools[1], page, d), k, v, slots, rotary=r, positions=pos, q=q, q_out=q)
    assert torch.equal(*pools) and torch.equal(q, out) and torch.equal(k, keep[0]) and torch.equal(v, keep[1])
    for other in (dict(k=q, v=v), dict(k=k, v=q), dict(k=x[:, 1:1 + h] if layout == "rows" else q, v=v)):
        with pytest.raises(sage.SageError, match="overlaps an input"):
            eng.kv4_append(sage.Kv4Cache(pools[1], page, d), other["k"], other["v"], slots, rotary=r, positions=pos, q=q,
                           q_out=q)
    eng.engine_status()


@pytest.mark.parametrize("rows", [4, 60])
def test_attend_without_max_q_takes_any_number_of_queries(engines, rows):
    """max_q is a bound that speeds a call up; left out, every query of every sequence is answered."""
    d, eng, ws = 128, engines[128], engines["ws", 128]
    b = Batch(d, 16, 8, 2, [300, 90, 200], [rows, 1, 2], seed=6)
    b.fill(eng)
    eng.kv4_attend(ws, sage.Kv4Cache(b.pool, 16, d), b.q, b.out, b.pages, b.kv_len, q_start=b.q_start, lse=b.lse)
    eng.engine_status()
    check_attend(b, "no max_q")
    assert (b.out[sum(b.qn):] == 3.0).all()


def test_tensors_that_moved_are_found_again(engines):
    """A pool and a rotary table whose tensors got other memory (set_, a larger or smaller one) after they were wrapped:
    the calls use what the tensors are now, or refuse it."""
    d, page, eng = 128, 16, engines[128]
    g = gen(3)
    block = sage.Kv4Cache.block_bytes(d, page)
    pools = [torch.zeros(n, 2, block, dtype=torch.uint8, device=DEV) for n in (4, 6, 2)]
    tabs = [table(d, 50), table(d, 80, sage.RopeScaling.linear(2.0))]
    pool, tab = pools[0].view_as(pools[0]).detach(), tabs[0].view_as(tabs[0]).detach()
    cache, r = sage.Kv4Cache(pool, page, d), sage.Rotary(tab, d)
    k, v, slots, pos = rand(g, 5, 2, d), rand(g, 5, 2, d), ints([0, 17, 35, 50, 63]), ints([1, 2, 3, 49, 30])
    eng.kv4_append(cache, k, v, slots, rotary=r, positions=pos)
    first = pools[0].clone()
    pool.set_(pools[1])
    tab.set_(tabs[1])
    slots[4], pos[4] = 95, 79
    eng.kv4_append(cache, k, v, slots, rotary=r, positions=pos)
    want = torch.zeros_like(pools[1])
    eng.kv4_append(sage.Kv4Cache(want, page, d), k, v, slots, rotary=sage.Rotary(tabs[1], d), positions=pos)
    assert torch.equal(pools[1], want) and torch.equal(pools[0], first)
    eng.engine_status()
    pool.set_(pools[2])
    eng.kv4_append(cache, k, v, slots, rotary=r, positions=pos)  # two pages: the other slots are out of range
    with pytest.raises(sage.SageError, match="out of range"):
        eng.engine_status()
    pool.set_(torch.zeros(4, 2, block - 16, dtype=torch.uint8, device=DEV))
    with pytest.raises(sage.SageError, match="cache pool"):
        eng.kv4_append(cache, k, v, slots)
    eng.engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 5, 90])
@pytest.mark.parametrize("value", [0.0, 2.5, -7.0e30])
def test_attend_constant_caches(engines, d, rows, value):
    """No group has a scale: each key's V is its zero, all keys weigh the same, the mean is exact."""
    b = Batch(d, 32, 4, 2, [800, 3], [rows, 1], seed=rows, tail_rows=0)
    b.k.fill_(0.375)
    b.v.fill_(value)
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d], causal=False)
    want = torch.tensor(value).bfloat16().to(DEV)
    # sums of equal numbers in f32, up to 800 of them: 2^-24 each, then bf16's rounding of a bf16 number
    assert ((b.out - want).abs() <= 2.0 ** -7 * want.abs()).all()
    score = (b.q.float().sum(-1) * 0.375).double() * d ** -0.5
    n = torch.cat([torch.full((rows,), 800.0), torch.full((1,), 3.0)]).to(DEV).double()[:, None]
    assert ((b.lse.double() - score - n.log()).abs() <= 1e-4).all()
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** -30, 2.0 ** -12, 2.0 ** 9, 2.0 ** 40])
@pytest.mark.parametrize("rows", [1, 90])
def test_attend_short_sequences_of_any_size_of_values(engines, d, scale, rows):
    """All keys of one magnitude, far from one, in sequences that end within a tile."""
    b = Batch(d, 16, 4, 2, [3, 130, 17, 90, 257], [min(rows, 3), rows, min(rows, 17), rows, rows], seed=rows, tail_rows=0)
    b.k, b.v = (b.k.float() * min(scale, 8.0)).bfloat16(), (b.v.float() * scale).bfloat16()
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    check_attend(b, "size")
    engines[d].engine_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-6, 1e-20])
@pytest.mark.parametrize("rows", [4, 90])
@pytest.mark.parametrize("key", [0.0, 0.25, 1e-25])
def test_attend_constant_keys_and_values_among_others(engines, d, size, rows, key):
    """Every fourth key constant (or nothing), its value too, small queries: it weighs what it should beside the others."""
    b = Batch(d, 16, 4, 2, [600, 130, 47], [rows, rows, min(rows, 47)], seed=rows, tail_rows=0)
    b.k[::4], b.v[::4] = key, 1.0
    b.q = (b.q.float() * size).bfloat16()
    b.fill(engines[d])
    b.attend(engines[d], engines["ws", d])
    check_attend(b, "constant")
    engines[d].engine_status()
