"""Operators of a token decoder that serves many requests, measured: their
cases, inputs, plain forms, work and 64-bit references.

Around its layers a server runs, for each step: pages for the requests' new
tokens with their slots (`plan_pages`), the residual's addition with the norm,
into fp32 or fp16 or, ahead of an 8-bit product, into 8 bits with a scale a
token (`rms_norm`, `rms_norm_quant`), keys and values into a cache of 4-bit
codes (`cache4_append`), attention over that cache (`cache4_attention`), and at
its end a token from the logits (`sample`).

Sizes: 12 heads of 64, a width of 768 and 1025 audio codes are this framework's
text encoder's and decoder example's; the others are generic.  B sequences, T
new tokens each, Hq query and Hk key/value heads of D values, N the width of a
token, V entries of the vocabulary.
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
        # one token of four utterances between two layers: the latency of a step
        dict(name="norm_step_f32", kind="norm", rows=4, N=768, dtype="f32", quant=False, residual=True),
        # a batch of prompts ahead of an 8-bit product
        dict(name="norm_prompt_quant_f16", kind="norm", rows=8192, N=4096, dtype="f16", quant=True, residual=True),
        # a step of a serving batch: a page for the sequences that begin one
        dict(name="plan_step", kind="plan", B=32, T=1, block=64, held=32768, dtype="i64", short=False),
        # prompts of a batch, more than there are pages for
        dict(name="plan_prompt", kind="plan", B=64, T=4095, block=16, held=0, dtype="i64", short=True),
        # one token of each of 32 sequences into partly filled pages
        dict(name="append4_step_f16", kind="append4", B=32, T=1, Hk=8, D=128, block=64, dtype="f16", held=63),
        # prompts of odd length into pages of 32
        dict(name="append4_prompt_f32", kind="append4", B=3, T=2051, Hk=12, D=64, block=32, dtype="f32", held=0),
        # a step of one short sequence
        dict(name="attend4_step_f32", kind="attend4", B=1, T=1, Hq=12, Hk=12, D=64, block=32, dtype="f32",
             longest=389, window=0),
        # a step of a serving batch over long, ragged contexts, four query heads a cached one
        dict(name="attend4_step_long_f16", kind="attend4", B=32, T=1, Hq=32, Hk=8, D=128, block=64, dtype="f16",
             longest=32768, window=0),
        # a chunk of new tokens over what is cached, itself included
        dict(name="attend4_chunk_f16", kind="attend4", B=2, T=1531, Hq=32, Hk=8, D=128, block=64, dtype="f16",
             longest=4099, window=0),
        # the same of an fp32 model with a window and small pages
        dict(name="attend4_window_f32", kind="attend4", B=2, T=517, Hq=8, Hk=2, D=96, block=16, dtype="f32",
             longest=3001, window=1000),
        # a step of one utterance over a vocabulary of audio codes
        dict(name="sample_step", kind="sample", B=1, V=1025, dtype="f32", spread=3.0),
        # a serving batch over a large vocabulary
        dict(name="sample_batch", kind="sample", B=64, V=131072, dtype="f32", spread=3.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every kind over its whole range, odd sizes among them."""
    kind = rng.choice(["norm", "plan", "append4", "attend4", "attend4", "attend4", "sample"])
    dtype = rng.choice(["f32", "f16"])
    block = rng.choice([16, 32, 64, 128, 256])
    step = rng.random() < 0.5  # single tokens, as in serving, or longer runs of them
    if kind == "norm":
        N = rng.choice([64, 200, 512, 768, 1000, 2048, 4096, 5120, 7777, 8192, _log(rng, 32, 16384)])
        rows = _log(rng, 1, 64) if step else _log(rng, 2, min(16384, 33000000 // N))
        return dict(kind=kind, rows=rows, N=N, dtype=dtype, quant=rng.random() < 0.6, residual=rng.random() < 0.7)
    if kind == "plan":
        B = _log(rng, 1, 1024) if step else _log(rng, 1, 64)
        return dict(kind=kind, B=B, T=rng.choice([1, 1, 4]) if step else _log(rng, 2, 4095), block=block,
                    held=_log(rng, 1, 32768), dtype=rng.choice(["i32", "i64"]), short=rng.random() < 0.3)
    Hk = rng.choice([1, 2, 4, 8, 12])
    if kind == "append4":
        return dict(kind=kind, B=_log(rng, 1, 64) if step else rng.randint(1, 4),
                    T=1 if step else _log(rng, 2, 3000), Hk=Hk, D=rng.choice([64, 96, 128, 256]), block=block,
                    dtype=dtype, held=rng.randint(0, 2 * block))
    if kind == "attend4":
        group = rng.choice([n for n in (1, 1, 2, 4, 7) if n * Hk <= 32])
        T = rng.choice([1, 1, 1, 2, 5]) if step else _log(rng, 6, 1500)
        longest = T + _log(rng, 1, 16000 if step else 2500)
        B = max(1, min(_log(rng, 1, 48) if step else rng.randint(1, 2), 400000 // longest))
        return dict(kind=kind, B=B, T=T, Hq=Hk * group, Hk=Hk, D=rng.choice([64, 96, 128]), block=block, dtype=dtype,
                    longest=longest, window=rng.choice([0, 0, 0, 200, 1000]))
    return dict(kind=kind, B=_log(rng, 1, 64), V=_log(rng, 50, 131072), dtype=dtype,
                spread=rng.choice([0.5, 2.0, 3.0, 5.0]))


# ------------------------------------------------------------------ prepare
def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _ints(g, lo, hi, shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)


def _norm_state(c, g):
    t, shape = TYPES[c["dtype"]], (c["rows"], c["N"])
    x = _normal(g, shape, t)
    x *= torch.where(torch.rand(c["N"], generator=g, device="cuda") < 0.01, 20.0, 1.0).to(t)  # some channels stand out
    return dict(x=x, residual=_normal(g, shape, t, 2.0) if c["residual"] else None,
                weight=1.0 + _normal(g, (c["N"],), std=0.2), quant=c["quant"])


def _table(need, columns, g, pages=None):
    """A table with `need` [B] pages for each sequence, given out in any order from `pages` (None: just as many), -1
    behind them, and how many pages there are."""
    held = torch.arange(columns, device="cuda") < need[:, None]
    some = int(need.sum())
    pages = some if pages is None else pages
    order = torch.randperm(pages, generator=g, device="cuda")[:some].to(torch.int32)
    table = torch.full((need.numel(), columns), -1, dtype=torch.int32, device="cuda")
    table[held] = order
    return table, pages


def _plan_state(c, g):
    B, T, blk = c["B"], c["T"], c["block"]
    t = torch.int32 if c["dtype"] == "i32" else torch.int64
    starts = _ints(g, 0, c["held"] + 1, (B,), t)
    counts = _ints(g, max(1, T - T // 4), T + 1, (B,), t)
    table, pages = _table(-(-starts // blk), -(-(c["held"] + T) // blk), g)
    wanted = int((-(-(starts + counts) // blk) - -(-starts // blk)).sum())
    spare = max(1, wanted * 3 // 4 if c["short"] else wanted + B)
    taken = int(_ints(g, 0, 50, (1,)))  # pages at the list's begin that were given out before
    free = torch.randperm(taken + spare, generator=g, device="cuda").to(torch.int32) + pages
    return dict(table=table, starts=starts, counts=counts, free=free, T=T, block=blk,
                used=torch.tensor([taken], dtype=torch.int32, device="cuda"))


def _append4_state(c, g):
    B, T, Hk, D, blk, t = c["B"], c["T"], c["Hk"], c["D"], c["block"], TYPES[c["dtype"]]
    starts = _ints(g, 0, c["held"] + 1, (B, 1), torch.int64)
    counts = _ints(g, max(1, T - T // 4), T + 1, (B, 1), torch.int64)
    columns = -(-(c["held"] + T) // blk)
    table, pages = _table(-(-(starts + counts) // blk)[:, 0], columns, g, B * columns)
    at = torch.arange(T, device="cuda")
    place = torch.where(at < counts, starts + at, 0)
    slots = torch.gather(table.long(), 1, place // blk) * blk + place % blk
    codes, scales = (pages, Hk, blk, D // 2), (pages, Hk, blk, 2)
    return dict(k=torch.zeros(codes, dtype=torch.uint8, device="cuda"), k_scale=_normal(g, scales, torch.float16).abs_(),
                v=torch.zeros((pages, Hk, D // 2, blk), dtype=torch.uint8, device="cuda"),
                v_scale=_normal(g, scales, torch.float16).abs_(), slots=torch.where(at < counts, slots, -1),
                nk=_normal(g, (B, T, Hk, D), t, 1.5), nv=_normal(g, (B, T, Hk, D), t))


def _codes(g, shape):
    """Two 4-bit codes a byte, as a normal distribution's values have them."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    flat, step = out.view(-1), 1 << 26
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        x = torch.randn(2, n, generator=g, device="cuda", dtype=torch.float16)
        x = x.mul_(3.0).add_(7.5).round_().clamp_(0.0, 15.0).to(torch.uint8)
        flat[at:at + n] = x[0] | x[1] << 4
    return out


def _attend4_state(c, g):
    B, T, Hq, Hk, D, blk, t = c["B"], c["T"], c["Hq"], c["Hk"], c["D"], c["block"], TYPES[c["dtype"]]
    lengths = _ints(g, max(T, c["longest"] // 2), c["longest"] + 1, (B,))
    lengths[0] = c["longest"]
    table, pages = _table(-(-lengths // blk), -(-c["longest"] // blk), g)
    s = dict(k=_codes(g, (pages, Hk, blk, D // 2)), v=_codes(g, (pages, Hk, D // 2, blk)), table=table,
             lengths=lengths, q=_normal(g, (B, T, Hq, D), t, 1.5), scale=1.0 / math.sqrt(D), window=c["window"])
    for name in ("k_scale", "v_scale"):  # a step and a lowest value for each token and head
        step = torch.rand((pages, Hk, blk, 1), generator=g, device="cuda") * 0.1 + 0.3
        low = -step * (7.5 + _normal(g, (pages, Hk, blk, 1), std=0.5))
        s[name] = torch.cat((step, low), -1).half()
    return s


def _sample_state(c, g):
    B, V = c["B"], c["V"]
    logits = _normal(g, (B, V), std=c["spread"])
    logits[torch.rand((B, V), generator=g, device="cuda") < 0.1] = -math.inf  # what a grammar forbids
    logits[:, 0] = 0.0

    def rows(*choices):
        return torch.tensor(choices, device="cuda")[_ints(g, 0, len(choices), (B,), torch.int64)]
    return dict(logits=logits.to(TYPES[c["dtype"]]), uniforms=torch.rand((B,), generator=g, device="cuda"),
                temperature=rows(0.0, 0.6, 0.8, 1.0, 1.0, 1.3), top_k=rows(0, 0, 20, 50, 1000).int(),
                top_p=rows(1.0, 0.95, 0.9, 0.8), min_p=rows(0.0, 0.0, 0.05, 0.1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = globals()[f"_{case['kind']}_state"](case, g)
    torch.cuda.synchronize()
    return dict(s, kind=case["kind"])


# -------------------------------------------------------------- plain forms
def _norm_plain(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    if s["quant"]:
        # in 64 bits: 32 could put a quotient next to a half on its other side
        y = x.double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["weight"].double()
        top = y.abs().amax(-1, keepdim=True)
        scale = (top / 127.0).float()
        codes = torch.round(torch.where(top > 0, y * (127.0 / top), 0.0))
        out = [codes.float() * scale, scale]
    else:
        out = [(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"]).to(s["x"].dtype)]
    return out if s["residual"] is None else out + [x.to(s["x"].dtype)]


def _plan_plain(s):
    """A sequence whose new tokens need more pages than are left gets none, nor do those behind it that need some."""
    table, free, blk = s["table"], s["free"], s["block"]
    starts, counts, used = s["starts"].long(), s["counts"].long(), s["used"].long()
    have = (starts + blk - 1) // blk
    need = (starts + counts + blk - 1) // blk - have
    upto = torch.cumsum(need, 0)
    served = (need == 0) | (upto <= free.numel() - used)
    granted = torch.where(served, counts, 0)
    column = torch.arange(table.shape[1], device="cuda")
    nth = column - have[:, None]
    new = served[:, None] & (nth >= 0) & (nth < need[:, None])
    at = (used + upto - need)[:, None] + nth
    table.copy_(torch.where(new, free[at.clamp(0, free.numel() - 1)], table))
    t = torch.arange(s["T"], device="cuda")
    there = t < granted[:, None]
    place = torch.where(there, starts[:, None] + t, 0)
    slots = torch.gather(table, 1, place // blk).long() * blk + place % blk
    taken = torch.where(served & (need > 0), upto, 0).amax()
    return [torch.where(there, slots, -1), torch.where(there, place, -1).int(), (starts + granted).int(), granted.int(),
            table, (used + taken).int()]


def _append4_one(codes, scales, new, slots, tokens_last):
    blk = scales.shape[2]
    new = torch.nan_to_num(new.float().flatten(0, 1), nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    slots = slots.flatten()
    slots = torch.where(slots >= 0, slots, slots[0])  # (what is left out repeats the first)
    new = torch.where((slots == slots[0])[:, None, None], new[:1], new)
    low = new.amin(-1, keepdim=True).half()
    step = ((new.amax(-1, keepdim=True).double() - low.double()) / 15.0).float().half()
    code = torch.round((new.double() - low.double()) / torch.where(step > 0, step, 1.0).double()).clamp(0.0, 15.0)
    code = torch.where(step > 0, code, 0.0).to(torch.uint8)
    half = code.shape[-1] // 2
    code = code[..., :half] | code[..., half:] << 4
    page, row = slots // blk, slots % blk
    if tokens_last:
        codes[page, :, :, row] = code
    else:
        codes[page, :, row] = code
    scales[page, :, row] = torch.cat((step, low), -1)


def _values4(codes, scales, axis):
    """Codes and scales as the values that they stand for, a token's along `axis`."""
    both = torch.cat((codes & 15, codes >> 4), axis).float()
    step, low = (scales[..., i].float().unsqueeze(axis) for i in range(2))
    return both * step + low


def _append4_plain(s):
    _append4_one(s["k"], s["k_scale"], s["nk"], s["slots"], False)
    _append4_one(s["v"], s["v_scale"], s["nv"], s["slots"], True)
    return [_values4(s["k"], s["k_scale"], 3), _values4(s["v"], s["v_scale"], 2)]


def _attend4_plain(s):
    B, T, Hq, D = s["q"].shape
    Hk, blk = s["k"].shape[1:3]
    page = s["table"].long().clamp(min=0)
    k = _values4(s["k"][page], s["k_scale"][page], 4)  # [B, pages, Hk, rows, D]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, Hk, D, -1)
    v = _values4(s["v"][page], s["v_scale"][page], 3)  # [B, pages, Hk, D, rows]
    v = v.permute(0, 2, 1, 4, 3).reshape(B, Hk, -1, D)
    at = torch.arange(page.shape[1] * blk, device="cuda")
    place = s["lengths"][:, None] - T + torch.arange(T, device="cuda")
    seen = at <= place[..., None]
    if s["window"]:
        seen = seen & (at > place[..., None] - s["window"])
    q = s["q"].float().reshape(B, T, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    x = torch.matmul(q, k).mul_(s["scale"]).reshape(B, Hk, Hq // Hk, T, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    y = torch.matmul(x.reshape(B, Hk, -1, x.shape[-1]), v).reshape(B, Hk, Hq // Hk, T, D) / x.sum(-1, keepdim=True)
    return y.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype)


def _sample_plain(s):
    """In 64 bits: 32 could put a number next to a token's border on its other side."""
    V = s["logits"].shape[1]
    x, order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)  # ties: the lowest index first
    t, p, u, m = (s[n].double()[:, None] for n in ("temperature", "top_p", "uniforms", "min_p"))
    k = s["top_k"].long()[:, None]
    x = x.double()
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(V, device="cuda")
    w = torch.where((rank < torch.where(k > 0, k, V)) & ((rank == 0) | (t > 0)), w, 0.0)
    upto = torch.cumsum(w, -1)
    w = torch.where(((upto - w < p * upto[:, -1:]) | (p >= 1)) & (w >= m), w, 0.0)
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    at = (upto <= u * total).sum(-1, keepdim=True).clamp(max=V - 1)
    return [torch.gather(order, 1, at)[:, 0].int(), torch.log(torch.gather(w, 1, at) / total)[:, 0].float()]


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
            made["cache"] = kk.KVCache4(*(made[n] for n in ("k", "k_scale", "v", "v_scale")))
        s["handles"] = dict(made, of=of)
    return s["handles"]


def _back(t):
    return torch.as_tensor(t, device="cuda")


def _own(s):
    kk = _kk()
    kk.init(0)
    kk.use_stream(torch.cuda.current_stream().cuda_stream)  # in order with what torch does before and after it
    h = _handles(kk, s)
    ops, kind = kk.ops, s["kind"]
    if kind == "norm" and s["quant"]:
        codes, scale, *total = ops.rms_norm_quant(h["x"], h["weight"], h.get("residual"), EPS)
        return [_back(x) for x in (ops.dequantize(codes, scale), scale, *total)]
    if kind == "norm":
        y = ops.rms_norm(h["x"], h["weight"], h.get("residual"), EPS)
        return [_back(x) for x in (y if isinstance(y, tuple) else (y,))]
    if kind == "plan":
        slots, positions, lengths, granted, used = ops.plan_pages(h["table"], h["starts"], h["counts"], h["free"],
                                                                  h["used"], s["T"], s["block"])
        return [_back(slots), _back(positions), _back(lengths), _back(granted), s["table"], _back(used)]
    if kind == "append4":
        ops.cache4_append(h["cache"], h["nk"], h["nv"], h["slots"])
        return [_back(x) for x in h["cache"].values()]
    if kind == "attend4":
        return _back(ops.cache4_attention(h["q"], h["cache"], h["table"], h["lengths"], scale=s["scale"],
                                          window=s["window"]))
    return [_back(x) for x in ops.sample(h["logits"], h["uniforms"], h["temperature"], h["top_k"], h["top_p"],
                                         h["min_p"])]


def run(state):
    if own:
        return _own(state)
    return globals()[f"_{state['kind']}_plain"](state)


# --------------------------------------------------------------------- work
def work(case):
    c, kind = case, case["kind"]
    size = 2 if c["dtype"] == "f16" else 4
    if kind == "norm":
        n = c["rows"] * c["N"]
        moved = n * size * (3 if c["residual"] else 1) + 4 * c["N"]
        # 8 bits: the codes out, and read again for the values that they stand for
        return {"bytes": moved + ((1 + 1 + 4) * n + 4 * c["rows"] if c["quant"] else size * n), "flops": 6 * n}
    if kind == "plan":
        tokens, index = c["B"] * c["T"], 4 if c["dtype"] == "i32" else 8
        return {"bytes": c["B"] * (2 * index + 8) + tokens * 12 + 8 * (tokens // c["block"]), "flops": 4 * tokens}
    if kind == "append4":
        rows = c["B"] * c["T"] * c["Hk"]
        pool = c["B"] * -(-(c["held"] + c["T"]) // c["block"]) * c["block"] * c["Hk"]
        # rows in, codes out, and the pool's codes read and the values they stand for written
        return {"bytes": 2 * (rows * (c["D"] * size + c["D"] // 2 + 4) + pool * (c["D"] // 2 + 4 + 4 * c["D"])),
                "flops": 2 * rows * 8 * c["D"]}
    if kind == "attend4":
        rows = c["B"] * 0.75 * c["longest"]  # (lengths are drawn between half and whole)
        if c["T"] == 1 and c["window"]:
            rows = min(rows, c["B"] * c["window"])
        pairs = c["T"] * (rows - c["B"] * (c["T"] - 1) / 2)
        if c["window"]:
            pairs = min(pairs, c["B"] * c["T"] * c["window"])
        return {"bytes": 2 * rows * c["Hk"] * (c["D"] // 2 + 4) + 2 * size * c["B"] * c["T"] * c["Hq"] * c["D"],
                "flops": 4 * pairs * c["Hq"] * c["D"]}
    return {"bytes": c["B"] * (c["V"] * size + 28), "flops": 8 * c["B"] * c["V"]}


# ------------------------------------------------------------------ 64 bits
def _exact_norm(c, s):
    x = s["x"].double()
    if c["residual"]:
        x = x + s["residual"].double()
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["N"] + EPS) * s["weight"].double()
    if c["quant"]:
        top = y.abs().amax(-1, keepdim=True)
        y = [torch.round(y / top * 127) * (top / 127), top / 127]
    else:
        y = [y]
    return y + [x] if c["residual"] else y


def _exact_plan(c, s):
    blk, T = c["block"], c["T"]
    table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy()
    starts, counts, used = s["starts"].tolist(), s["counts"].tolist(), int(s["used"])
    slots, positions = np.full((c["B"], T), -1, np.int64), np.full((c["B"], T), -1, np.int32)
    left, full = len(free) - used, False
    for b in range(c["B"]):
        have = -(-starts[b] // blk)
        need = -(-(starts[b] + counts[b]) // blk) - have
        full = full or need > left
        if need and full:
            counts[b] = 0
            continue
        table[b, have:have + need] = free[used:used + need]
        used, left = used + need, left - need
        place = np.arange(starts[b], starts[b] + counts[b])
        positions[b, :counts[b]] = place
        slots[b, :counts[b]] = table[b, place // blk].astype(np.int64) * blk + place % blk
    return [slots, positions, np.array(starts, np.int32) + np.array(counts, np.int32), np.array(counts, np.int32),
            table, np.array([used], np.int32)]


def _exact_append4(c, s):
    out, blk = [], c["block"]
    slots = s["slots"].flatten()
    live = slots >= 0
    page, row = slots[live] // blk, slots[live] % blk
    for name, new in (("k", s["nk"]), ("v", s["nv"])):
        codes = s[name].double() if name == "k" else s[name].double().transpose(2, 3)
        values = torch.cat((codes % 16, torch.floor(codes / 16)), -1)
        values = values * s[name + "_scale"][..., :1].double() + s[name + "_scale"][..., 1:].double()
        x = new.double().flatten(0, 1)[live]
        low = x.amin(-1, keepdim=True).half().double()
        step = ((x.amax(-1, keepdim=True) - low) / 15).float().half().double()
        values[page, :, row] = low + step * torch.round((x - low) / step).clamp(0, 15)
        out.append(values if name == "k" else values.transpose(2, 3).contiguous())
    return out


def _exact_attend4(c, s):
    out, T, D, group = [], c["T"], c["D"], c["Hq"] // c["Hk"]

    def rows(codes, scales, n):  # [pages, Hk, rows, D / 2] of one sequence as [Hk, n, D]
        both = torch.cat((codes & 15, codes >> 4), -1).double()
        both = both * scales[..., :1].double() + scales[..., 1:].double()
        return both.transpose(0, 1).reshape(c["Hk"], -1, D)[:, :n]
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, :-(-n // c["block"])].long()
        k = rows(s["k"][pages], s["k_scale"][pages], n)
        v = rows(s["v"][pages].transpose(2, 3), s["v_scale"][pages], n)
        gap = torch.arange(n - T, n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        seen = (gap >= 0) & (gap < (s["window"] or n + 1))
        y = torch.zeros((T, c["Hq"], D), dtype=torch.float64, device="cuda")
        for h in range(c["Hq"]):
            x = (s["q"][b, :, h].double() @ k[h // group].T.contiguous()) * s["scale"]
            y[:, h] = torch.softmax(torch.where(seen, x, -math.inf), -1) @ v[h // group]
        out.append(y)
    return torch.stack(out)


def _exact_sample(c, s):
    x = s["logits"].double().cpu().numpy()
    t, k, p, m, u = (s[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "uniforms"))
    tokens, logs = np.zeros(c["B"], np.int32), np.zeros(c["B"])
    for b in range(c["B"]):
        order = np.argsort(-x[b], kind="stable")
        order = order[:1] if t[b] <= 0 else order[:int(k[b])] if k[b] > 0 else order
        w = np.exp((x[b, order] - x[b, order[0]]) / (t[b] if t[b] > 0 else 1.0))
        w /= w.sum()
        if p[b] < 1:
            w = w[:1 + np.searchsorted(np.cumsum(w), p[b])]
        w = w[w >= m[b] * w[0]]
        upto = np.cumsum(w)
        at = min(np.searchsorted(upto, u[b] * upto[-1], side="right"), len(w) - 1)
        tokens[b], logs[b] = order[at], np.log(w[at] / upto[-1])
    return [tokens, logs]


def exact(case, seed):
    s = prepare(case, seed)
    return globals()[f"_exact_{case['kind']}"](case, s)
