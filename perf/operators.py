"""Operators of an autoregressive token decoder, measured: their cases, inputs,
plain forms, work and 64-bit references.

A decoder that writes speech tokens from a text encoder's states runs, for
each layer and step: the queries' and keys' norms with the position rotation
(`qk_norm_rotary`), the keys and values into a cache of 8-bit codes
(`cache_append`), attention over that cache (`cache_attention`), attention
over the encoder's states (`cross_attention`); and at its end the penalties,
biases and grammar mask on the logits (`process_logits`).

Sizes: 12 heads of 64 are this framework's text encoder's (130 tokens the
benchmarked utterance, 26 frames a token); the others are generic.  B
sequences, T new tokens each, Hq query and Hk key/value heads of D values,
S encoder states, V entries of the vocabulary, L tokens of history.
"""
import functools
import importlib
import math

import numpy as np
import torch

own = False
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one sequence, heads of the text encoder's size: the latency of a step
        dict(name="rotary_step_f32", kind="rotary", B=1, T=1, Hq=12, Hk=12, D=64, R=64, inter=False,
             norm=True, dtype="f32", far=4000, factor=1.0),
        # prompts of a batch, queries and keys in one fused projection, positions scaled for a long context
        dict(name="rotary_prompt_f16", kind="rotary", B=4, T=4096, Hq=32, Hk=8, D=128, R=128, inter=False,
             norm=True, dtype="f16", far=131072, factor=8.0),
        # part of an 80-wide head rotated, neighbours paired, no norm, odd length, far positions
        dict(name="rotary_partial_f32", kind="rotary", B=2, T=1537, Hq=16, Hk=16, D=80, R=32, inter=True,
             norm=False, dtype="f32", far=1000000, factor=1.0),
        # one token of each of 32 sequences into partly filled blocks
        dict(name="append_step_f16", kind="append", B=32, T=1, Hk=8, D=128, block=64, dtype="f16", held=63),
        # prompts of odd length into blocks of 32
        dict(name="append_prompt_f32", kind="append", B=3, T=2051, Hk=12, D=64, block=32, dtype="f32", held=0),
        # a step of one short sequence
        dict(name="cache_step_f32", kind="cache", B=1, T=1, Hq=12, Hk=12, D=64, block=32, dtype="f32",
             longest=389, window=0),
        # a step of a serving batch over long, ragged contexts, four query heads a cached one
        dict(name="cache_step_long_f16", kind="cache", B=32, T=1, Hq=32, Hk=8, D=128, block=64, dtype="f16",
             longest=32768, window=0),
        # a chunk of new tokens over what is cached, itself included
        dict(name="cache_chunk_f16", kind="cache", B=2, T=1531, Hq=32, Hk=8, D=128, block=64, dtype="f16",
             longest=4099, window=0),
        # a step of four utterances over the text states of 130 tokens
        dict(name="cross_step_f32", kind="cross", B=4, T=1, S=130, Hq=12, Hk=12, D=64, dtype="f32", masked=False),
        # every frame of an utterance over its text states, teacher-forced
        dict(name="cross_frames_f32", kind="cross", B=2, T=3380, S=509, Hq=12, Hk=12, D=64, dtype="f32",
             masked=True),
        # a step of one sequence over a vocabulary of audio codes
        dict(name="logits_step", kind="logits", B=1, V=1025, L=350, dtype="f32"),
        # a serving batch over a large vocabulary
        dict(name="logits_batch", kind="logits", B=64, V=131072, L=4096, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every kind over its whole range, odd sizes among them."""
    kind = rng.choice(["rotary", "append", "cache", "cache", "cross", "cross", "logits"])
    dtype = rng.choice(["f32", "f16"])
    Hk = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([n for n in (1, 1, 2, 4, 7) if n * Hk <= 32])
    step = rng.random() < 0.5  # single tokens, as in serving, or longer runs of them
    if kind == "rotary":
        B = _log(rng, 1, 64) if step else rng.randint(1, 4)
        T = 1 if step else _log(rng, 2, 4096)
        D = rng.choice([64, 80, 96, 128, 256])
        return dict(kind=kind, B=B, T=T, Hq=Hk * group, Hk=Hk, D=D, R=rng.choice([D, D, 32]),
                    inter=rng.random() < 0.5, norm=rng.random() < 0.7, dtype=dtype,
                    far=_log(rng, T + 10, 1000000), factor=rng.choice([1.0, 4.0, 32.0]))
    if kind == "append":
        block = rng.choice([16, 32, 64, 128])
        return dict(kind=kind, B=_log(rng, 1, 64) if step else rng.randint(1, 4),
                    T=1 if step else _log(rng, 2, 3000), Hk=Hk, D=rng.choice([64, 96, 128]), block=block,
                    dtype=dtype, held=rng.randint(0, 3 * block))
    if kind == "cache":
        T = rng.choice([1, 1, 1, 2, 5]) if step else _log(rng, 6, 1500)
        longest = T + _log(rng, 1, 16000 if step else 2500)
        B = max(1, min(_log(rng, 1, 48) if step else rng.randint(1, 2), 400000 // longest))
        return dict(kind=kind, B=B, T=T, Hq=Hk * group, Hk=Hk, D=rng.choice([64, 96, 128]),
                    block=rng.choice([16, 32, 64, 128]), dtype=dtype, longest=longest,
                    window=rng.choice([0, 0, 0, 200, 1000]))
    if kind == "cross":
        return dict(kind=kind, B=_log(rng, 1, 32) if step else rng.randint(1, 2),
                    T=1 if step else _log(rng, 2, 3000), S=_log(rng, 1, 3000 if step else 1500), Hq=Hk * group,
                    Hk=Hk, D=rng.choice([64, 80, 128]), dtype=dtype, masked=rng.random() < 0.5)
    return dict(kind=kind, B=_log(rng, 1, 64), V=_log(rng, 50, 131072), L=_log(rng, 1, 4096), dtype=dtype)


# ------------------------------------------------------------------ prepare
def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _ints(g, lo, hi, shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)


def _turns(R, factor):
    """What each pair turns a position, in 2^64ths of a turn: base 10000, positions divided by `factor`."""
    return torch.tensor([int(10000.0 ** (-2.0 * i / R) / factor / (2 * math.pi) * 2.0 ** 64) for i in range(R // 2)],
                        dtype=torch.int64, device="cuda")


def _pool(need, most, g):
    """A pool with room for `most` pages a sequence, given out in any order, and the table of the `need` that each
    has; entries past a sequence's last page are -1."""
    pages = len(need) * most
    order = torch.randperm(pages, generator=g, device="cuda").cpu()
    table = torch.full((len(need), most), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return pages, table.cuda()


def _codes(g, shape):
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat, step = out.view(-1), 1 << 27
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        x = torch.randn(n, generator=g, device="cuda", dtype=torch.float16)
        flat[at:at + n] = x.mul_(34.0).round_().clamp_(-127.0, 127.0).to(torch.int8)
    return out


def _cache(case, pages, g):
    Hk, blk, D = case["Hk"], case["block"], case["D"]
    return dict(k=_codes(g, (pages, Hk, blk, D)), v=_codes(g, (pages, Hk, D, blk)),
                k_scale=torch.rand((pages, Hk), generator=g, device="cuda") * 0.02 + 0.02,
                v_scale=torch.rand((pages, Hk), generator=g, device="cuda") * 0.02 + 0.02)


def _rotary_state(c, g):
    B, T, Hq, Hk, D, t = c["B"], c["T"], c["Hq"], c["Hk"], c["D"], TYPES[c["dtype"]]
    qkv = _normal(g, (B, T, Hq + 2 * Hk, D), t, 1.5)
    starts = _ints(g, 0, c["far"] - T + 1, (B, 1))
    s = dict(q=qkv[:, :, :Hq], k=qkv[:, :, Hq:Hq + Hk], turns=_turns(c["R"], c["factor"]),
             positions=starts + torch.arange(T, dtype=torch.int32, device="cuda"), inter=c["inter"],
             amplitude=0.1 * math.log(c["factor"]) + 1.0)
    s["wq"], s["wk"] = ((1.0 + _normal(g, (D,), std=0.2), 1.0 + _normal(g, (D,), std=0.2)) if c["norm"]
                        else (None, None))
    return s


def _append_state(c, g):
    B, T, Hk, D, blk, t = c["B"], c["T"], c["Hk"], c["D"], c["block"], TYPES[c["dtype"]]
    starts = _ints(g, 0, c["held"] + 1, (B,))
    counts = _ints(g, max(1, T - T // 4), T + 1, (B,))
    need = [-(-int(n) // blk) for n in (starts + counts).cpu()]
    pages, table = _pool(need, -(-(c["held"] + T) // blk), g)
    return dict(_cache(c, pages, g), table=table, starts=starts, counts=counts,
                nk=_normal(g, (B, T, Hk, D), t), nv=_normal(g, (B, T, Hk, D), t))


def _cache_state(c, g):
    B, T, Hq, D, blk, t = c["B"], c["T"], c["Hq"], c["D"], c["block"], TYPES[c["dtype"]]
    lengths = _ints(g, max(T, c["longest"] // 2), c["longest"] + 1, (B,))
    lengths[0] = c["longest"]
    pages, table = _pool([-(-int(n) // blk) for n in lengths.cpu()], -(-c["longest"] // blk), g)
    return dict(_cache(c, pages, g), table=table, lengths=lengths, q=_normal(g, (B, T, Hq, D), t, 1.5),
                scale=1.0 / math.sqrt(D), window=c["window"])


def _cross_state(c, g):
    B, T, S, Hq, Hk, D, t = c["B"], c["T"], c["S"], c["Hq"], c["Hk"], c["D"], TYPES[c["dtype"]]
    kv = _normal(g, (B, S, 2, Hk, D), t)
    s = dict(q=_normal(g, (B, T, Hq, D), t, 1.5), k=kv[:, :, 0], v=kv[:, :, 1], scale=1.0 / math.sqrt(D),
             lengths=_ints(g, max(1, S // 2), S + 1, (B,)), mask=None)
    if c["masked"]:  # pauses and tags that a frame does not look at
        s["mask"] = torch.rand((B, S), generator=g, device="cuda") > 0.1
        s["mask"][:, 0] = True
    return s


def _logits_state(c, g):
    B, V, L = c["B"], c["V"], c["L"]
    u = torch.rand((B, L), generator=g, device="cuda")
    return dict(logits=_normal(g, (B, V), TYPES[c["dtype"]], 3.0),
                history=(u * u * u * V).to(torch.int32).clamp_(max=V - 1),  # common tokens come often
                history_lengths=_ints(g, 0, L + 1, (B,)),
                repetition=1.0 + torch.rand((B,), generator=g, device="cuda") * 0.5,
                presence=torch.rand((B,), generator=g, device="cuda"),
                frequency=torch.rand((B,), generator=g, device="cuda") * 0.3,
                bias=_normal(g, (V,), std=0.5),
                allowed=_ints(g, -2 ** 31, 2 ** 31, (B, (V + 31) // 32), torch.int64).to(torch.int32))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = globals()[f"_{case['kind']}_state"](case, g)
    torch.cuda.synchronize()
    return dict(s, kind=case["kind"])


# -------------------------------------------------------------- plain forms
def _norm_rotate(x, w, s):
    x32 = x.float()
    if w is not None:
        x32 = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS) * w
    half = s["turns"].numel()
    angle = s["positions"].double()[..., None] * (s["turns"].double() * (2 * math.pi / 2.0 ** 64))
    cos = (torch.cos(angle) * s["amplitude"]).float()[:, :, None]
    sin = (torch.sin(angle) * s["amplitude"]).float()[:, :, None]
    if s["inter"]:
        a, b = x32[..., 0:2 * half:2], x32[..., 1:2 * half:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x32[..., :half], x32[..., half:2 * half]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x32[..., 2 * half:]), -1).to(x.dtype)


def _rotary_plain(s):
    return [_norm_rotate(s["q"], s["wq"], s), _norm_rotate(s["k"], s["wk"], s)]


def _append_one(codes, scales, new, s, blk, tokens_last):
    """New rows into their pages (scale: the largest value's, never falling while a page fills), in place.  The
    quotients are formed in 64 bits: 32 could put one next to a half on its other side."""
    B, T = new.shape[:2]
    page_axis = s["table"].long()
    t = torch.arange(T, device="cuda")
    t = torch.where(t < s["counts"][:, None], t, 0)  # rows past a sequence's count repeat its first
    new = torch.gather(new.float(), 1, t[:, :, None, None].expand_as(new))
    p = s["starts"].long()[:, None] + t
    page = torch.gather(page_axis, 1, p // blk).reshape(-1)
    row = (p % blk).reshape(-1)
    rows = new.reshape(B * T, *new.shape[2:])
    top = torch.zeros_like(scales).index_reduce_(0, page, rows.abs().amax(-1), "amax")
    want = torch.where(top > 0, (top.double() / 127.0).float().clamp(min=2.0 ** -126), 0.0)
    first = torch.gather(page_axis, 1, (s["starts"].long() // blk)[:, None])[:, 0]
    held = s["starts"].long() % blk  # rows that the first page holds already
    before = torch.where((held > 0)[:, None], scales[first], 0.0)
    after = torch.maximum(before, want[first])
    ratio = torch.where(after > 0, before.double() / after, 0.0)
    old = codes[first]  # [B, Hk, rows, D], or [B, Hk, D, rows]
    place = torch.arange(blk, device="cuda")
    place = place[None, None, None, :] if tokens_last else place[None, None, :, None]
    codes[first] = torch.where(place < held[:, None, None, None],
                               torch.round(old * ratio[:, :, None, None]).to(torch.int8), old)
    scales[page] = want[page]
    scales[first] = after
    by = scales[page][..., None]
    q = torch.where(by > 0, torch.round(rows.double() / by).clamp(-127.0, 127.0), 0.0).to(torch.int8)
    if tokens_last:
        codes[page, :, :, row] = q
    else:
        codes[page, :, row] = q


def _append_plain(s):
    blk = s["k"].shape[2]
    _append_one(s["k"], s["k_scale"], s["nk"], s, blk, False)
    _append_one(s["v"], s["v_scale"], s["nv"], s, blk, True)
    return [s["k"].float() * s["k_scale"][:, :, None, None], s["k_scale"].clone(),
            s["v"].float() * s["v_scale"][:, :, None, None], s["v_scale"].clone()]


def _attend(q, k, v, seen, scale):
    """q [B, T, Hq, D], k [B, Hk, D, S], v [B, Hk, S, D], seen [B, 1 or T, S]; rows that see nothing are zeros."""
    B, T, Hq, D = q.shape
    Hk = k.shape[1]
    q32 = q.float().reshape(B, T, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    x = torch.matmul(q32, k).mul_(scale).reshape(B, Hk, Hq // Hk, T, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.reshape(B, Hk, -1, x.shape[-1]), v).reshape(B, Hk, Hq // Hk, T, D)
    y = torch.where(total > 0, y / total, 0.0)
    return y.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(q.dtype)


def _cache_plain(s):
    B, T = s["q"].shape[:2]
    Hk, blk, D = s["k"].shape[1:]
    page = s["table"].long().clamp(min=0)
    k = s["k"][page].float() * s["k_scale"][page][..., None, None]  # [B, pages, Hk, rows, D]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, Hk, D, -1)
    v = s["v"][page].float() * s["v_scale"][page][..., None, None]  # [B, pages, Hk, D, rows]
    v = v.permute(0, 2, 1, 4, 3).reshape(B, Hk, -1, D)
    at = torch.arange(page.shape[1] * blk, device="cuda")
    place = s["lengths"][:, None] - T + torch.arange(T, device="cuda")
    seen = at <= place[..., None]
    if s["window"]:
        seen = seen & (at > place[..., None] - s["window"])
    return _attend(s["q"], k, v, seen, s["scale"])


def _cross_plain(s):
    k = s["k"].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"].float().permute(0, 2, 1, 3).contiguous()
    seen = torch.arange(k.shape[-1], device="cuda") < s["lengths"][:, None]
    if s["mask"] is not None:
        seen = seen & s["mask"]
    return _attend(s["q"], k, v, seen[:, None], s["scale"])


def _logits_plain(s):
    B, V = s["logits"].shape
    L = s["history"].shape[1]
    live = (torch.arange(L, device="cuda") < s["history_lengths"][:, None]).float()
    count = torch.zeros((B, V), device="cuda").scatter_add_(1, s["history"].long(), live)
    x = s["logits"].float()
    rep = s["repetition"][:, None]
    x = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - torch.where(count > 0, s["presence"][:, None], 0.0)
    x = x + s["bias"]
    v = torch.arange(V, device="cuda")
    bit = (s["allowed"][:, v >> 5] >> (v & 31)) & 1
    return torch.where(bit != 0, x, -math.inf)


# ------------------------------------------------------- the framework's own
@functools.lru_cache
def _kk():
    return importlib.import_module("best-tts-godot_amd")


def _handles(kk, s):
    """The state's buffers as the framework's tensors (no copies), made once, as a program keeps them, and again where
    the state has got other buffers since."""
    made = s.get("handles")
    if made is None or not all(s[n] is x for n, x in made["of"]):
        of = [(n, x) for n, x in s.items() if isinstance(x, torch.Tensor)]
        made = {n: kk.DeviceTensor.from_array(x) for n, x in of}
        if "k_scale" in s:
            made["cache"] = kk.KVCache(*(made[n] for n in ("k", "k_scale", "v", "v_scale")))
        s["handles"] = dict(made, of=of)
    return s["handles"]


def _back(t):
    return torch.as_tensor(t, device="cuda")


def _own(s):
    kk = _kk()
    kk.init(0)
    if hasattr(kk, "use_stream"):  # torch's stream, so that a pass is in order with what torch does before and after it
        kk.use_stream(torch.cuda.current_stream().cuda_stream)
    h = _handles(kk, s)
    ops, kind = kk.ops, s["kind"]
    if kind == "rotary":
        q, k = ops.qk_norm_rotary(h["q"], h["k"], h["positions"], h["turns"], h.get("wq"), h.get("wk"), eps=EPS,
                                  interleaved=s["inter"], amplitude=s["amplitude"])
        return [_back(q), _back(k)]
    if kind == "append":
        cache = h["cache"]
        ops.cache_append(cache, h["nk"], h["nv"], h["table"], h["starts"], h["counts"])
        k, v = cache.values()
        return [_back(k), s["k_scale"], _back(v), s["v_scale"]]
    if kind == "cache":
        return _back(ops.cache_attention(h["q"], h["cache"], h["table"], h["lengths"], scale=s["scale"],
                                         window=s["window"]))
    if kind == "cross":
        return _back(ops.cross_attention(h["q"], h["k"], h["v"], h["lengths"], h.get("mask"), scale=s["scale"]))
    return _back(ops.process_logits(h["logits"], h["history"], h["history_lengths"], h["repetition"], h["presence"],
                                    h["frequency"], h["bias"], h["allowed"]))


def run(state):
    if own:
        return _own(state)
    return globals()[f"_{state['kind']}_plain"](state)


# --------------------------------------------------------------------- work
def _need(case):
    """Tokens that a cache case's sequences hold, on average (their lengths are drawn between half and whole)."""
    return case["B"] * 0.75 * case["longest"]


def work(case):
    c, kind = case, case["kind"]
    size = 2 if c["dtype"] == "f16" else 4
    if kind == "rotary":
        n = c["B"] * c["T"] * (c["Hq"] + c["Hk"]) * c["D"]
        return {"bytes": 2 * n * size + 4 * c["B"] * c["T"] + 4 * c["R"], "flops": 10 * n}
    if kind == "append":
        n = c["B"] * c["T"] * c["Hk"] * c["D"]
        held = c["B"] * -(-(c["held"] + c["T"]) // c["block"]) * c["block"] * c["Hk"] * c["D"]
        # rows in, codes out, and the pool's codes read and the values they stand for written
        return {"bytes": 2 * (n * size + n + 5 * held), "flops": 6 * n}
    if kind == "cache":
        rows = _need(c)
        if c["T"] == 1 and c["window"]:
            rows = min(rows, c["B"] * c["window"])
        pairs = c["T"] * (rows - c["B"] * (c["T"] - 1) / 2)
        if c["window"]:
            pairs = min(pairs, c["B"] * c["T"] * c["window"])
        return {"bytes": 2 * rows * c["Hk"] * c["D"] + 2 * size * c["B"] * c["T"] * c["Hq"] * c["D"],
                "flops": 4 * pairs * c["Hq"] * c["D"]}
    if kind == "cross":
        rows = c["B"] * (0.75 * c["S"])
        return {"bytes": 2 * size * (rows * c["Hk"] + c["B"] * c["T"] * c["Hq"]) * c["D"],
                "flops": 4 * c["T"] * rows * c["Hq"] * c["D"]}
    n = c["B"] * c["V"]
    return {"bytes": n * (size + 4) + n / 8 + 4 * c["V"] + 2 * c["B"] * c["L"], "flops": 6 * n}


# ------------------------------------------------------------------ 64 bits
def _exact_rotary(c, s):
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["D"] + EPS) * w.double()
        half = c["R"] // 2
        # the fraction of a turn in whole numbers: the position's product modulo 2^64
        part = (s["positions"].long()[..., None] * s["turns"]).double() * 2.0 ** -64
        turn = torch.polar(torch.full_like(part, s["amplitude"]), 2 * math.pi * part)[:, :, None]
        y = x.clone()
        first, second = (slice(0, c["R"], 2), slice(1, c["R"], 2)) if c["inter"] else (slice(0, half),
                                                                                      slice(half, c["R"]))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return out


def _exact_append(c, s):
    blk, out = c["block"], []
    starts, counts, table = s["starts"].tolist(), s["counts"].tolist(), s["table"].tolist()
    for name, new in (("k", s["nk"]), ("v", s["nv"])):
        codes = s[name].double().transpose(2, 3).clone() if name == "v" else s[name].double().clone()
        scales = s[name + "_scale"].double().clone()
        for b in range(c["B"]):
            at, end = starts[b], starts[b] + counts[b]
            while at < end:
                page, lo = table[b][at // blk], at % blk
                n = min(blk - lo, end - at)
                rows = new[b, at - starts[b]:at - starts[b] + n].double().transpose(0, 1)  # [Hk, n, D]
                want = (rows.abs().amax((1, 2)) / 127).float().double()  # a page holds its scale in 32 bits
                now = torch.maximum(scales[page], want) if lo else want
                if lo:
                    codes[page, :, :lo] = torch.round(codes[page, :, :lo] * (scales[page] / now)[:, None, None])
                codes[page, :, lo:lo + n] = torch.round(rows / now[:, None, None])
                scales[page] = now
                at += n
        values = codes * scales[:, :, None, None]
        out += [values.transpose(2, 3).contiguous() if name == "v" else values, scales]
    return out


def _exact_heads(q, k, v, seen, scale):
    """One sequence: q [T, Hq, D], k and v [S, Hk, D], seen [1 or T, S]."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for h in range(q.shape[1]):
        g = h // (q.shape[1] // k.shape[1])
        x = (q[:, h].double() @ k[:, g].double().T.contiguous()) * scale
        x = torch.where(seen, x, -math.inf)
        p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        out[:, h] = p @ v[:, g].double()
    return out


def _exact_cache(c, s):
    out, T, D = [], c["T"], c["D"]
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, :-(-n // c["block"])].long()
        k = s["k"][pages].double() * s["k_scale"][pages].double()[..., None, None]
        v = s["v"][pages].double() * s["v_scale"][pages].double()[..., None, None]
        k = k.transpose(1, 2).reshape(-1, c["Hk"], D)[:n]
        v = v.permute(0, 3, 1, 2).reshape(-1, c["Hk"], D)[:n]
        gap = torch.arange(n - T, n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        seen = (gap >= 0) & (gap < (s["window"] or n + 1))
        out.append(_exact_heads(s["q"][b], k, v, seen, s["scale"]))
    return torch.stack(out)


def _exact_cross(c, s):
    out = []
    for b, n in enumerate(s["lengths"].tolist()):
        seen = torch.ones((1, n), dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][b:b + 1, :n]
        out.append(_exact_heads(s["q"][b], s["k"][b, :n], s["v"][b, :n], seen, s["scale"]))
    return torch.stack(out)


def _exact_logits(c, s):
    x = s["logits"].double().cpu().numpy()
    history, lengths = s["history"].cpu().numpy(), s["history_lengths"].cpu().numpy()
    bits = np.unpackbits(s["allowed"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :c["V"]]
    rep, pres, freq = (s[n].double().cpu().numpy() for n in ("repetition", "presence", "frequency"))
    bias = s["bias"].double().cpu().numpy()
    for b in range(c["B"]):
        ids, n = np.unique(history[b, :lengths[b]], return_counts=True)
        y = x[b, ids]
        x[b, ids] = np.where(y > 0, y / rep[b], y * rep[b]) - freq[b] * n - pres[b]
        x[b] += bias
        x[b, bits[b] == 0] = -np.inf
    return x


def exact(case, seed):
    s = prepare(case, seed)
    return globals()[f"_exact_{case['kind']}"](case, s)
