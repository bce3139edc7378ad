"""The serving operators and the work they are timed on: rotary positions, keys and values appended to a paged 4-bit
cache (with the rotation applied on the way), and attention over that cache.

`run` computes them in plain torch operations where `own` is false and makes the framework's calls where it is true.
`exact` computes them in 64 bits from their definitions.

The cache: a pool uint8 [pages][kv_heads][block]; the block of one page of P tokens and one KV head holds the K
values [P][D/2], the V values [P][D/2] (channel 2j in a byte's low half, 2j+1 in its high half), then the K parameters
[P][D/64] pairs (scale, zero) in bf16 and the V parameters likewise.  A value is zero + scale * n, n = 0..15, with one
scale and zero per 64 channels of a token: zero = bf16(min), scale = bf16((max - min) * (1/15)),
n = clamp(rint((x - zero) / scale), 0, 15)."""
import importlib
import math
import random

import torch

own = False

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# (query heads, KV heads, head dim): the repository's Llama-3-8B prefill heads, its ViT-L heads, and
# generic ones, a group that is not a power of two among them
HEADS = [(32, 8, 128), (16, 16, 64), (12, 12, 128), (28, 4, 128), (8, 2, 64)]


def listed():
    return [
        # one decoding step's q and k rows of 32 sequences, anywhere in a long context
        dict(name="rope step", op="rope", tokens=32, heads=40, d=128, rot=128, inter=False, dtype="bf16", table=131072,
             start=-1, scaling="bands", backward=False),
        # the q and k rows of an 8192-token prompt
        dict(name="rope prompt", op="rope", tokens=8192, heads=40, d=128, rot=128, inter=False, dtype="bf16",
             table=8192, start=0, scaling="none", backward=False),
        # a training step's gradient, half of each head rotated, neighbouring channels paired, an odd length
        dict(name="rope gradient", op="rope", tokens=4099, heads=32, d=64, rot=32, inter=True, dtype="f32",
             table=16384, start=517, scaling="yarn", backward=True),
        # one decoding step of 64 sequences: a row each, into pages all over the pool
        dict(name="append step", op="append", tokens=64, hq=32, hkv=8, d=128, rot=128, inter=False, page=16,
             table=131072, start=-1),
        # an 8192-token prompt laid down after 1000 cached tokens
        dict(name="append prompt", op="append", tokens=8192, hq=32, hkv=8, d=128, rot=128, inter=False, page=64,
             table=16384, start=1000),
        # a ViT-L sized prompt, half of each head rotated
        dict(name="append part", op="append", tokens=1370, hq=16, hkv=16, d=64, rot=32, inter=True, page=32,
             table=4096, start=0),
        # one user, a short context: what counts is latency
        dict(name="attend short", op="attend", batch=1, q=1, ctx=1000, low=1000, hq=32, hkv=8, d=128, page=16,
             causal=True, window=0, mix=1),
        # a serving batch, contexts of very different lengths
        dict(name="attend batch", op="attend", batch=64, q=1, ctx=8192, low=1, hq=32, hkv=8, d=128, page=64,
             causal=True, window=0, mix=2),
        # one user, the longest context
        dict(name="attend long", op="attend", batch=1, q=1, ctx=131072, low=131072, hq=32, hkv=8, d=128, page=64,
             causal=True, window=0, mix=3),
        # as many KV heads as query heads, small pages
        dict(name="attend heads", op="attend", batch=16, q=1, ctx=4096, low=200, hq=16, hkv=16, d=64, page=16,
             causal=True, window=0, mix=4),
        # a few drafted tokens of each sequence checked at once, within a sliding window
        dict(name="attend draft", op="attend", batch=8, q=5, ctx=16384, low=3000, hq=32, hkv=8, d=128, page=32,
             causal=True, window=8192, mix=5),
        # pieces of two prompts against what is cached of them already
        dict(name="attend prompt", op="attend", batch=2, q=2048, ctx=8192, low=5000, hq=32, hkv=8, d=128, page=64,
             causal=True, window=0, mix=6),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    hq, hkv, d = rng.choice(HEADS)
    kind = rng.choice(["rope", "append", "attend one", "attend one", "attend few", "attend piece"])
    if kind in ("rope", "append"):
        rot = rng.choice([d, d, d // 2, d // 4])
        c = dict(op=kind, tokens=_log(rng, 1, 8192), d=d, rot=rot, inter=rng.random() < 0.5, table=16384,
                 start=rng.choice([-1, 0, rng.randrange(8192)]))
        if kind == "append":
            return dict(c, hq=hq, hkv=hkv, page=rng.choice([16, 32, 64, 128]))
        return dict(c, heads=hq + hkv if hkv < hq else hq, dtype=rng.choice(["bf16", "f16", "f32"]),
                    scaling=rng.choice(["none", "linear", "bands", "yarn"]), backward=rng.random() < 0.4)
    c = dict(op="attend", hq=hq, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 128]), mix=rng.randrange(1 << 20),
             causal=rng.random() < 0.85, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    if kind == "attend piece":
        q = _log(rng, 9, 2048)
        ctx = q + _log(rng, 1, 6144)
        b = max(1, min(8, rng.randrange(1, 5), 4096 // q))
    else:
        q = 1 if kind == "attend one" else rng.randrange(2, 9)
        ctx = _log(rng, max(16, q), 16384)
        b = _log(rng, 1, max(1, min(64, 400000 // ctx)))
    return dict(c, batch=b, q=q, ctx=ctx, low=rng.randrange(q, ctx + 1))


def _lens(case):
    """Cached tokens and query tokens of each sequence: the case's own, whatever the seed."""
    rng = random.Random(case["mix"])
    kv = [rng.randint(case["low"], case["ctx"]) for _ in range(case["batch"])]
    kv[0] = case["ctx"]
    qn = [case["q"] if i == 0 or case["q"] == 1 else rng.randint(1, case["q"]) for i in range(case["batch"])]
    return kv, [min(q, n) for q, n in zip(qn, kv)]


# ---------------------------------------------------------------- inputs

def _frequencies(rot, scaling):
    """The angle per position of each pair, and the factor on cos and sin (64 bits)."""
    base, pairs = 500000.0, rot // 2
    f = base ** -(torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    turns = 8192 * f / (2 * math.pi)  # full turns within the original context
    if scaling == "linear":
        return f / 4, 1.0
    if scaling == "bands":  # slow pairs stretched by 8, fast ones kept, those between blended
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / 8 * (1 - keep), 1.0
    if scaling == "yarn":
        at = [pairs * math.log(8192 / (r * 2 * math.pi)) / math.log(base) for r in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((torch.arange(pairs, dtype=torch.float64, device="cuda") - low) / max(high - low, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / 4 * ramp, 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _table(rot, positions, scaling):
    f, m = _frequencies(rot, scaling)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.stack([a.cos() * m, a.sin() * m], -1).float()


def _positions(case, g):
    if case["start"] < 0:
        return torch.randint(0, case["table"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)
    return torch.arange(case["start"], case["start"] + case["tokens"], device="cuda", dtype=torch.int32)


def _block(page, d):
    return page * (d + d // GROUP * 8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = case["d"]

    def normal(*shape, dtype=torch.bfloat16, offset=0.0):
        x = torch.randn(*shape, generator=g, device="cuda")
        if offset:  # a channel's own mean, as keys have it
            x += offset * torch.randn(shape[-2:], generator=g, device="cuda")
        return x.to(dtype)

    s = dict(case=case)
    if case["op"] == "rope":
        s["x"] = normal(case["tokens"], case["heads"], d, dtype=DTYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["x"])
        s["table"] = _table(case["rot"], case["table"], case["scaling"])
        s["positions"] = _positions(case, g)
        return s
    page = case["page"]
    if case["op"] == "append":
        t, hq, hkv = case["tokens"], case["hq"], case["hkv"]
        qkv = normal(t, hq + 2 * hkv, d, offset=1.0)  # as the projection leaves them: q, k and v heads side by side
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["table"] = _table(case["rot"], case["table"], "none")
        s["positions"] = _positions(case, g)
        if case["start"] < 0:  # each token at the end of a sequence of its own
            pages = 2 * t + 3
            p = torch.randperm(pages, generator=g, device="cuda")[:t]
            row = s["positions"].long() % page
        else:
            pages = t // page + 5
            at = torch.arange(t, device="cuda") + case["start"] % page
            p = torch.randperm(pages, generator=g, device="cuda")[at // page]
            row = at % page
        s["slots"] = (p * page + row).int()
        s["pool"] = torch.zeros(pages, hkv, _block(page, d), dtype=torch.uint8, device="cuda")
        s["q_out"] = torch.empty(t, hq, d, dtype=torch.bfloat16, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty(t, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        return s
    kv, qn = _lens(case)
    hq, hkv = case["hq"], case["hkv"]
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 2
    s["pool"] = torch.empty(pages, hkv, _block(page, d), dtype=torch.uint8, device="cuda")
    parts = _parts(s["pool"], page, d)
    for values, params, offset in ((parts[0], parts[2], 1.0), (parts[1], parts[3], 0.0)):
        n, scale, zero = _quantise(normal(pages, page, hkv, d, offset=offset).transpose(1, 2).float())
        values.copy_(_pack(n))
        params.copy_(torch.stack([scale, zero], -1).flatten(-2))
    table, at = torch.zeros(len(kv), max(need), dtype=torch.int32), 0
    order = torch.randperm(pages, generator=g, device="cuda").int().cpu()
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    s["pages"] = table.cuda()
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    starts = [sum(qn[:i]) for i in range(len(qn) + 1)]
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["q"] = normal(starts[-1], hq, d)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(starts[-1], hq, dtype=torch.float32, device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms

def _rotate(x, table, positions, rot, inter, backward=False):
    """f32 [token][head][D] rotated by its tokens' angles."""
    cs = table[positions.long()][:, None]
    c, sn = cs[..., 0], cs[..., 1]
    if backward:
        sn = -sn
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    ya, yb = a * c - b * sn, b * c + a * sn
    y = torch.stack([ya, yb], -1).flatten(-2) if inter else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _quantise(x):
    """f32 [..., D] -> n uint8 [..., D], scale and zero bf16 [..., D/64]."""
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    zero, scale = low.bfloat16(), ((high - low) * (1.0 / 15.0)).bfloat16()
    n = ((x - zero.float()[..., None]) / scale.float()[..., None]).round()
    n = n.masked_fill(scale[..., None] == 0, 0.0).clamp(0, 15).to(torch.uint8)
    return n.flatten(-2), scale, zero


def _pack(n):
    return n[..., 0::2] | n[..., 1::2] << 4


def _unpack(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _parts(pool, page, d):
    """Views of the pool: K and V values [pages][heads][P][D/2], K and V parameters [pages][heads][P][D/64 * 2]."""
    v, p = page * d // 2, page * d // GROUP * 4
    cut = [0, v, 2 * v, 2 * v + p, 2 * v + 2 * p]
    a = [pool[..., i:j].unflatten(-1, (page, -1)) for i, j in zip(cut, cut[1:])]
    return a[0], a[1], a[2].view(torch.bfloat16), a[3].view(torch.bfloat16)


def _values(b, params):
    """f32 [..., D] of packed values and their parameters."""
    n = _unpack(b).float().unflatten(-1, (-1, GROUP))
    p = params.float().unflatten(-1, (-1, 2))
    return (p[..., 1:] + p[..., :1] * n).flatten(-2)


def _plain_append(s):
    c = s["case"]
    page, d = c["page"], c["d"]
    q = _rotate(s["q"].float(), s["table"], s["positions"], c["rot"], c["inter"]).bfloat16()
    k = _rotate(s["k"].float(), s["table"], s["positions"], c["rot"], c["inter"])
    parts = _parts(s["pool"], page, d)
    p, row = s["slots"].long() // page, s["slots"].long() % page
    for x, values, params in ((k, parts[0], parts[2]), (s["v"].float(), parts[1], parts[3])):
        n, scale, zero = _quantise(x)
        values[p, :, row] = _pack(n)
        params[p, :, row] = torch.stack([scale, zero], -1).flatten(-2)
    return {"q": q, "k": _values(parts[0][p, :, row], parts[2][p, :, row]).bfloat16(),
            "v": _values(parts[1][p, :, row], parts[3][p, :, row]).bfloat16()}


def _plain_attend(s):
    c = s["case"]
    page, d, hq, hkv, b = c["page"], c["d"], c["hq"], c["hkv"], c["batch"]
    parts, pages = _parts(s["pool"], page, d), s["pages"].long()
    k, v = (_values(x[pages], y[pages]).transpose(1, 2).flatten(2, 3) for x, y in
            ((parts[0], parts[2]), (parts[1], parts[3])))  # [sequence][KV head][key][D]
    starts, kv_len = s["q_start"].long(), s["kv_len"].long()
    qn = starts[1:] - starts[:-1]
    i = torch.arange(c["q"], device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)  # [sequence][query token]
    q = s["q"][row].float().unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ k.transpose(-1, -2)).unflatten(2, (hq // hkv, c["q"])) * d ** -0.5  # [sequence][KV head][group][token][key]
    j = torch.arange(k.shape[2], device="cuda")
    at = (kv_len - qn)[:, None] + i
    seen = (j < kv_len[:, None, None]).expand(b, c["q"], -1)
    if c["causal"]:
        seen = seen & (j <= at[..., None])
    if c["window"]:
        seen = seen & (j > at[..., None] - c["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = (x - m.masked_fill(m == -math.inf, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (hq // hkv, c["q"])) / total
    o = o.masked_fill(total == 0, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
    lse = (m + total.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
    own_row = i < qn[:, None]
    return {"out": o[own_row].bfloat16(), "lse": lse[own_row]}


# ---------------------------------------------------------------- the framework's calls

_engines = {}


def _engine(sage, d):
    """The engine and the attention's workspace that a serving process keeps for a head dim and stream."""
    stream = torch.cuda.current_stream()
    key = (d, stream.device_index, stream.cuda_stream)
    if key not in _engines:
        eng = sage.SageAttention(stream, d)
        _engines[key] = (eng, eng.kv4_workspace())
    return _engines[key]


def _own(s):
    sage = importlib.import_module("sota-papers-lab_b200")
    c = s["case"]
    d = c["d"]
    eng, ws = _engine(sage, d)
    if c["op"] == "rope":
        rot = sage.Rotary(s["table"], c["rot"], c["inter"])
        eng.rope(s["x"], s["out"], rot, s["positions"], backward=c["backward"])
        return s["out"]
    cache = sage.Kv4Cache(s["pool"], c["page"], d)
    if c["op"] == "append":
        rot = sage.Rotary(s["table"], c["rot"], c["inter"])
        eng.kv4_append(cache, s["k"], s["v"], s["slots"], rotary=rot, positions=s["positions"], q=s["q"],
                       q_out=s["q_out"])
        eng.kv4_read(cache, s["slots"], s["k_out"], s["v_out"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    eng.kv4_attend(ws, cache, s["q"], s["out"], s["pages"], s["kv_len"], q_start=s["q_start"], max_q=c["q"],
                   causal=c["causal"], window=c["window"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    if c["op"] == "rope":
        x = state["x"]
        return _rotate(x.float(), state["table"], state["positions"], c["rot"], c["inter"], c["backward"]).to(x.dtype)
    return _plain_append(state) if c["op"] == "append" else _plain_attend(state)


# ---------------------------------------------------------------- what the work cannot do without

def _visible(case):
    """Per sequence: (keys that any of its queries sees, pairs of query token and key)."""
    kv, qn = _lens(case)
    got = []
    for n, q in zip(kv, qn):
        first, pairs = n, 0
        for i in range(q):
            at = n - q + i
            high = at + 1 if case["causal"] else n
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            first = min(first, low)
            pairs += max(0, high - low)
        got.append((n - first, pairs))
    return got


def work(case):
    d = case["d"]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * d
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * n * size + case["tokens"] * (case["rot"] * 4 + 4), "flops": 3 * n * case["rot"] / d}
    if case["op"] == "append":
        t, hq, hkv = case["tokens"], case["hq"], case["hkv"]
        held = t * hkv * (d + d // GROUP * 8)
        return {"bytes": t * (hq + 2 * hkv) * d * 2 + t * hq * d * 2 + held + t * (case["rot"] * 4 + 8)
                + held + 2 * t * hkv * d * 2, "flops": t * (hq + 3 * hkv) * d * 3}
    seen = _visible(case)
    rows = sum(_lens(case)[1])
    return {"bytes": sum(k for k, _ in seen) * case["hkv"] * (d + d // GROUP * 8) + rows * case["hq"] * (4 * d + 4),
            "flops": 4 * sum(p for _, p in seen) * case["hq"] * d}


# ---------------------------------------------------------------- 64 bits

def _turned(x, case, positions, scaling, backward=False):
    """x rotated in 64 bits, as complex numbers times e^(i angle)."""
    f, m = _frequencies(case["rot"], scaling)
    turn = torch.polar(torch.full_like(f, m), f * positions.double()[:, None])[:, None]
    if backward:
        turn = turn.conj()
    y, r = x.double().clone(), case["rot"]
    i = torch.arange(r // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if case["inter"] else (i, i + r // 2)
    z = torch.complex(y[..., a], y[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _held(x):
    """The values that the cache stands for, of 64-bit rows."""
    x = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    zero = x.min(-1, keepdim=True).values
    scale = ((x.max(-1, keepdim=True).values - zero) / 15).float().bfloat16().double()
    zero = zero.float().bfloat16().double()
    return (zero + scale * torch.clamp(torch.round((x - zero) / scale), 0, 15)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s["x"], case, s["positions"], case["scaling"], case["backward"])
    if case["op"] == "append":
        return {"q": _turned(s["q"], case, s["positions"], "none"),
                "k": _held(_turned(s["k"], case, s["positions"], "none")), "v": _held(s["v"].double())}
    d, page, hq, hkv = case["d"], case["page"], case["hq"], case["hkv"]
    kv, qn = _lens(case)
    out, lse = torch.zeros(sum(qn), hq, d, dtype=torch.float64, device="cuda"), None
    lse = torch.full((sum(qn), hq), -math.inf, dtype=torch.float64, device="cuda")
    half = page * d // 2
    row = 0
    for i, (n, q) in enumerate(zip(kv, qn)):
        blocks = s["pool"][s["pages"][i, :-(-n // page)].long()]
        key = torch.arange(n, device="cuda")
        at = n - q + torch.arange(q, device="cuda")[:, None]
        hidden = (key > at) if case["causal"] else torch.zeros(q, n, dtype=torch.bool, device="cuda")
        if case["window"]:
            hidden = hidden | (key <= at - case["window"])
        for h in range(hkv):
            b = blocks[:, h]
            kv64 = []
            for part in range(2):
                raw = b[:, part * half:(part + 1) * half].reshape(-1, d // 2).int()
                wide = torch.empty(raw.shape[0], d, dtype=torch.float64, device="cuda")
                wide[:, 0::2], wide[:, 1::2] = raw % 16, raw // 16
                par = b[:, 2 * half:].reshape(b.shape[0], 2, page, d // GROUP, 4)[:, part].contiguous()
                par = par.view(torch.bfloat16).double().reshape(-1, d // GROUP, 2).repeat_interleave(GROUP, 1)
                kv64.append((par[..., 1] + par[..., 0] * wide)[:n])
            for e in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = s["q"][row:row + q, e].double() @ kv64[0].T / math.sqrt(d)
                x = torch.where(hidden, torch.full_like(x, -math.inf), x)
                lse[row:row + q, e] = torch.logsumexp(x, -1)
                out[row:row + q, e] = torch.nan_to_num(torch.softmax(x, -1)) @ kv64[1]
        row += q
    return {"out": out, "lse": lse}
