"""The operators of a cache kept in 8 bits and of drafted tokens, as they are measured: plain forms beside the framework's calls.

Four operators, in the order in which a serving step meets them:

``store``      keys rotated, keys and values rounded to 8 bits and written to their pages (`ops.rope_kv_store_q8`)
``attention``  single tokens, drafted tokens or portions of prompts over such pages (`ops.attention_q8`)
``load``       rows of such pages as ordinary numbers again (`ops.kv_load_q8`)
``verify``     drafted tokens accepted or replaced by the target's own (`ops.verify_drafts`)

A row of the cache is one token's key or value of one kv head: codes of 1 sign, 4 exponent and 3 mantissa bits, and one byte e
for the row, its numbers being code * 2^(e - 127).  The scale is the smallest power of two with which the row's largest
magnitude is at most 448, not below 2^-110, and 1 for a row of zeros.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# Layer sizes as bench.py's shapes have them: query heads, kv heads, head size, vocabulary.
SIZES = {"0.5B": (14, 2, 64, 151936), "1.5B": (12, 2, 128, 151936), "7B": (28, 4, 128, 152064)}
PAGE = 16
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a decode step of a few conversations: the projection comes as parts that are still to be summed
        dict(name="store, decode 8", op="store", size="0.5B", tokens=8, dtype="bf16", parts=7, page=PAGE),
        # a long prompt of a large model
        dict(name="store, prompt 2048", op="store", size="7B", tokens=2048, dtype="bf16", parts=0, page=PAGE),
        # decode steps: a few short conversations, where latency counts; a full batch; one very long context
        dict(name="attention, decode 8 x 530", op="attention", size="0.5B", requests=8, rows=1, past=529, ragged=0.2, window=0, page=PAGE),
        dict(name="attention, decode 32 x 4096", op="attention", size="7B", requests=32, rows=1, past=4095, ragged=0.1, window=0, page=PAGE),
        dict(name="attention, decode 1 x 100k", op="attention", size="7B", requests=1, rows=1, past=99999, ragged=0.0, window=0, page=64),
        # drafted tokens to be verified: five rows a request
        dict(name="attention, drafts 16 x 5", op="attention", size="1.5B", requests=16, rows=5, past=1700, ragged=0.3, window=0, page=PAGE),
        # a whole prompt, and portions of two prompts late in a long context with a sliding window
        dict(name="attention, prompt 2048", op="attention", size="0.5B", requests=1, rows=2048, past=0, ragged=0.0, window=0, page=PAGE),
        dict(name="attention, portions 2 x 1024", op="attention", size="7B", requests=2, rows=1024, past=7100, ragged=0.2, window=4096, page=32),
        # a conversation's rows read back, and a batch's contexts
        dict(name="load, 517 rows", op="load", size="0.5B", rows=517, dtype="bf16", page=PAGE),
        dict(name="load, 40000 rows", op="load", size="7B", rows=40000, dtype="f32", page=PAGE),
        # drafts with the draft model's probabilities at a temperature, and greedy ones of a full batch
        dict(name="verify, 8 x 5 sampled", op="verify", size="0.5B", requests=8, drafts=4, temperature=0.8, probs=True),
        dict(name="verify, 48 x 5 greedy", op="verify", size="7B", requests=48, drafts=4, temperature=0.0, probs=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("store", "attention", "attention", "attention", "load", "verify"))
    size = rng.choice(sorted(SIZES))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    if op == "store":
        parts = rng.choice((0, 0, rng.randint(2, 9)))
        return dict(op=op, size=size, tokens=_log(rng, 1, 128 if parts else 2048), parts=parts, page=page,
                    dtype="bf16" if parts else rng.choice(("bf16", "f32")))
    if op == "load":
        return dict(op=op, size=size, rows=_log(rng, 1, 40000), dtype=rng.choice(("bf16", "f32")), page=page)
    if op == "verify":
        temperature = rng.choice((0.0, round(rng.uniform(0.5, 1.5), 2)))
        return dict(op=op, size=size, requests=_log(rng, 1, 48), drafts=rng.randint(1, 4), temperature=temperature,
                    probs=temperature > 0 and rng.random() < 0.7)
    kind = rng.choice(("decode", "decode", "drafts", "portion"))
    window = rng.choice((0, 0, 0, _log(rng, 100, 4096)))
    ragged = round(rng.uniform(0.0, 0.6), 2)
    if kind == "decode":
        requests = _log(rng, 1, 48)
        return dict(op=op, size=size, requests=requests, rows=1, past=_log(rng, 1, 100000 // requests), ragged=ragged, window=window, page=page)
    if kind == "drafts":
        requests = _log(rng, 1, 24)
        return dict(op=op, size=size, requests=requests, rows=rng.randint(2, 9), past=_log(rng, 10, 60000 // requests), ragged=ragged,
                    window=window, page=page)
    requests = rng.randint(1, 3)
    return dict(op=op, size=size, requests=requests, rows=_log(rng, 20, 2048 // requests), past=rng.choice((0, _log(rng, 30, 4000))),
                ragged=ragged, window=window, page=page)


def _lengths(case):
    """(rows of each request, keys that each has held before): a little ragged, as a continuous batch is."""
    rng = random.Random(11)
    rows, past = [], []
    for _ in range(case["requests"]):
        rows.append(max(1, int(case["rows"] * (1 - case["ragged"] * rng.random()))) if case["rows"] > 9 else case["rows"])
        past.append(int(case["past"] * (1 - case["ragged"] * rng.random())))
    return rows, past


def _drafts(case):
    """Drafted tokens of each request: one request in four brings fewer."""
    rng = random.Random(13)
    return [case["drafts"] if rng.random() < 0.75 else rng.randint(0, case["drafts"]) for _ in range(case["requests"])]


# ------------------------------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------------------------------
def _rows(gen, shape, channels):
    """Rows as projections give them: normal, a few channels larger than the others."""
    x = torch.randn(shape, generator=gen, device="cuda")
    wide = torch.rand((channels,), generator=gen, device="cuda") < 0.05
    return x.view(-1, channels).mul_(torch.where(wide, 6.0, 1.0)).view(shape)


def _two_to(n):
    """2^n in 64 bits, from the exponent's own bits (a power function need not be exact)."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _encode(x):
    """Codes and scale bytes of rows [..., d] of 64-bit numbers."""
    top = x.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(top)
    power = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-110)
    power = torch.where(top == 0, torch.zeros_like(power), power)
    y = x * _two_to(-power).unsqueeze(-1)
    # steps of an eighth of the power of two below y, or of 2^-9 where that would be less
    step = _two_to(torch.frexp(y)[1].clamp(min=-5) - 4)
    y = torch.round(y / step) * step
    bad = ~torch.isfinite(x.float()).all(dim=-1)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(y), y).float().to(torch.float8_e4m3fn)
    return code, torch.where(bad, 255, power + 127).to(torch.uint8)


def _powers(byte):
    """2^(e - 127) in 32 bits, NaN for 255."""
    e = byte.to(torch.int32)
    return torch.where(e == 255, math.nan, (e << 23).view(torch.float32))


def _pool(gen, pages, n_kv, page, d):
    """Pages as earlier steps have left them."""
    out = {}
    for name in ("k", "v"):
        code, byte = _encode(_rows(gen, (pages, n_kv, page, d), d).double())
        out[name], out[name + "_scale"] = code, byte
    return out


def _table(gen, tokens, d):
    """(cos, sin) of the rows' angles, tokens at positions of a long context."""
    positions = torch.randint(0, 30000, (tokens, 1), generator=gen, device="cuda").double()
    angle = positions * torch.pow(1e6, -2.0 * torch.arange(d // 2, device="cuda").double() / d)
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n_q, n_kv, d, vocab = SIZES[case["size"]]
    s = dict(case, n_q=n_q, n_kv=n_kv, d=d)
    if case["op"] == "store":
        tokens, width, page = case["tokens"], (n_q + 2 * n_kv) * d, case["page"]
        pages = -(-tokens // page) + 2
        s.update(_pool(gen, pages, n_kv, page, d))
        x = _rows(gen, (tokens, width), width)
        s["bias"] = None
        if case["parts"]:
            s["qkv"] = torch.randn((case["parts"], tokens, width), generator=gen, device="cuda") * 0.5
            s["qkv"][0] += x
            s["bias"] = torch.randn((width,), generator=gen, device="cuda").to(torch.bfloat16)
        else:
            s["qkv"] = x.to(TYPES[case["dtype"]])
        s["table"] = _table(gen, tokens, d)
        s["slots"] = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].to(torch.int32)
    elif case["op"] == "load":
        pages = -(-case["rows"] // case["page"]) + 2
        s.update(_pool(gen, pages, n_kv, case["page"], d))
        # whole pages of a request, in the order in which it was given them
        order = torch.randperm(pages, generator=gen, device="cuda")
        s["slots"] = (order[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).reshape(-1)[: case["rows"]].to(torch.int32)
    elif case["op"] == "attention":
        rows, past = _lengths(case)
        page, held = case["page"], [r + p for r, p in zip(rows, past)]
        blocks = [-(-n // page) for n in held]
        pages = sum(blocks) + 3
        s.update(_pool(gen, pages, n_kv, page, d))
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(rows), max(blocks)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(blocks):
            table[b, :n] = order[at: at + n]
            at += n
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        integers = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        s.update(q=_rows(gen, (starts[-1], n_q * d), n_q * d).to(torch.bfloat16), block_table=table, q_start=integers(starts),
                 kv_len=integers(held), pos0=integers(past), q_lens=rows, max_kv_len=max(held), scale=1.0 / math.sqrt(d))
    else:
        counts = [n + 1 for n in _drafts(case)]
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        total = starts[-1]
        s["logits"] = torch.randn((total, vocab), generator=gen, device="cuda") * 2.5
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["temperature"] = s["seeds"] = s["positions"] = s["draft_probs"] = None
        if case["temperature"] > 0:
            B = case["requests"]
            s["temperature"] = torch.full((B,), case["temperature"], device="cuda")
            s["seeds"] = torch.randint(0, 1 << 31, (B,), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
            s["positions"] = torch.randint(1, 4000, (B,), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
            # the draft model is near the target
            near = s["logits"] / case["temperature"] + torch.randn((total, vocab), generator=gen, device="cuda") * 0.6
            probs = torch.softmax(near, dim=-1)
            if case["probs"]:
                s["draft_probs"] = probs
            s["drafts"] = torch.multinomial(probs, 1, generator=gen)[:, 0].to(torch.int32)
        else:
            other = torch.randint(0, vocab, (total,), generator=gen, device="cuda")
            s["drafts"] = torch.where(torch.rand((total,), generator=gen, device="cuda") < 0.8, s["logits"].argmax(dim=-1), other).to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------------------------------
def _plain_store(s):
    n_q, n_kv, d, page = s["n_q"], s["n_kv"], s["d"], s["page"]
    x = s["qkv"]
    if x.dim() == 3:
        x = (x.double().sum(dim=0) + s["bias"].double()).to(torch.bfloat16)
    kind, tokens = x.dtype, x.shape[0]
    x = x.double().view(tokens, n_q + 2 * n_kv, d)     # in 64 bits: a key next to the border of two codes takes the right one
    c, n = s["table"].double().unbind(dim=-1)
    c, n = c[:, None], n[:, None]
    lo, hi = x[:, : n_q + n_kv, : d // 2], x[:, : n_q + n_kv, d // 2:]
    turned = torch.cat((lo * c - hi * n, hi * c + lo * n), dim=-1)
    slots = s["slots"].long()
    at = (slots // page, slice(None), slots % page)
    for name, rows in (("k", turned[:, n_q:]), ("v", x[:, n_q + n_kv:])):
        code, byte = _encode(rows)
        s[name].view(torch.uint8)[at] = code.view(torch.uint8)
        s[name + "_scale"][at] = byte
    return turned[:, :n_q].to(kind).reshape(tokens, n_q * d)


def _plain_load(s):
    slots, out = s["slots"].long(), []
    at = (slots // s["page"], slice(None), slots % s["page"])
    for name in ("k", "v"):
        code = s[name].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        out.append((code * _powers(s[name + "_scale"][at]).unsqueeze(-1)).to(TYPES[s["dtype"]]))
    return tuple(out)


def _plain_attention(s):
    n_q, n_kv, d, page = s["n_q"], s["n_kv"], s["d"], s["page"]
    group, B, most = n_q // n_kv, len(s["q_lens"]), max(s["q_lens"])
    table = s["block_table"].long().clamp(min=0)

    def held(name):     # [requests, kv heads, keys, d]
        x = s[name][table].float() * _powers(s[name + "_scale"][table]).unsqueeze(-1)
        return x.transpose(1, 2).reshape(B, n_kv, -1, d)

    row = torch.arange(most, device="cuda")
    there = row < (s["q_start"][1:] - s["q_start"][:-1])[:, None]                        # [requests, most]
    at = (s["q_start"][:-1, None] + row).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][at].float().view(B, most, n_kv, group, d).permute(0, 2, 3, 1, 4).reshape(B, n_kv, group * most, d)
    scores = torch.matmul(q, held("k").transpose(2, 3)).mul_(s["scale"]).view(B, n_kv, group, most, -1)
    key = torch.arange(scores.shape[-1], device="cuda")
    pos = (s["pos0"][:, None] + row)[:, :, None]
    seen = (key <= pos) & (key < s["kv_len"][:, None, None])
    if s["window"]:
        seen &= key > pos - s["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    o = torch.matmul(scores.view(B, n_kv, group * most, -1), held("v")).view(B, n_kv, group, most, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(B, most, n_q * d)
    return o[there].to(torch.bfloat16)


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _uniform(h):
    return ((h >> 9).double() + 0.5) / 8388608.0


def _plain_verify(s):
    logits, starts = s["logits"], s["starts"].long()
    R, vocab, B = logits.shape[0], logits.shape[1], starts.numel() - 1
    row = torch.arange(R, device="cuda")
    req = torch.searchsorted(starts, row, right=True) - 1
    last = row == starts[1:][req] - 1
    draft = s["drafts"].long()
    if s["temperature"] is None:
        best = logits.argmax(dim=-1)
        taken = (draft == best) & ~last
        keys = p = None
    else:
        # probabilities in 64 bits: a token next to the border of being accepted goes the right way
        p = torch.softmax(logits.double() / s["temperature"][req, None].double(), dim=-1)
        keys = _mix(_mix((s["seeds"].long()[req] & 0xFFFFFFFF) ^ 0x9E3779B9) ^ (s["positions"].long()[req] + row - starts[req]))
        u = _uniform(_mix(keys ^ 0xFFFFFFFF))
        safe = draft.clamp(0, vocab - 1)[:, None]
        theirs = s["draft_probs"].gather(1, safe)[:, 0].double() if s["draft_probs"] is not None else torch.ones_like(u)
        taken = (u * theirs < p.gather(1, safe)[:, 0]) & ~last
    # a request's rows up to its first refusal
    refused = (~taken).long()
    before = refused.cumsum(0) - refused
    place = before - before[starts[:-1]][req]
    kept = (place == 0) & taken
    stop = starts[:-1] + torch.zeros(B, dtype=torch.long, device="cuda").index_add_(0, req, kept.long())     # the row that ends a request
    if s["temperature"] is None:
        new = best[stop]
    else:
        rest = p[stop]
        over = last[stop]
        if s["draft_probs"] is not None:
            less = (rest - s["draft_probs"][stop].double()).clamp(min=0)
        else:
            less = rest.scatter(1, draft[stop].clamp(0, vocab - 1)[:, None], 0.0)
        weight = torch.where((over | (less.amax(dim=-1) == 0))[:, None], rest, less)
        index = torch.arange(vocab, device="cuda")
        wait = -torch.log(_uniform(_mix((keys[stop, None] + index * 0x85EBCA6B) & 0xFFFFFFFF)))
        new = (weight / wait).argmax(dim=-1)
    tokens = torch.where(kept, draft, torch.full_like(draft, -1))
    tokens[stop] = new
    return tokens.to(torch.int32), (stop - starts[:-1] + 1).to(torch.int32)


def run(state):
    s = state
    if own:
        from llm_inference_lab_b200.kernels import ops
        if s["op"] == "verify":
            return ops.verify_drafts(s["logits"], s["drafts"], s["starts"], s["draft_probs"], s["temperature"], s["seeds"], s["positions"])
        pages = ops.QuantPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if s["op"] == "store":
            q = ops.rope_kv_store_q8(s["qkv"], s["table"], s["d"], s["slots"], pages, s["n_q"], s["n_kv"], s["d"], bias=s["bias"])
        elif s["op"] == "load":
            return ops.kv_load_q8(pages, s["slots"], TYPES[s["dtype"]])
        else:
            return ops.attention_q8(s["q"], pages, s["q_start"], s["kv_len"], s["pos0"], s["block_table"], len(s["q_lens"]), s["q_lens"],
                                    s["max_kv_len"], s["n_q"], s["n_kv"], s["d"], s["window"], s["scale"])
    elif s["op"] == "verify":
        return _plain_verify(s)
    elif s["op"] == "load":
        return _plain_load(s)
    elif s["op"] == "attention":
        return _plain_attention(s)
    else:
        q = _plain_store(s)
    # the store's outputs are the rotated queries and the pool, codes as the numbers that they stand for
    return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def work(case):
    n_q, n_kv, d, vocab = SIZES[case["size"]]
    row = 2 * d + 2                                  # a token's key and value of one kv head in the cache
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "store":
        width = (n_q + 2 * n_kv) * d
        came = width * (4 * case["parts"] if case["parts"] else size)
        return {"bytes": case["tokens"] * (came + n_q * d * size + n_kv * row + 4 * d + 4), "flops": case["tokens"] * (n_q + n_kv) * 3 * d}
    if case["op"] == "load":
        return {"bytes": case["rows"] * (n_kv * (row + 2 * d * size) + 4), "flops": case["rows"] * n_kv * 2 * d}
    if case["op"] == "verify":
        rows = sum(_drafts(case)) + case["requests"]
        return {"bytes": 4 * vocab * (rows + (case["requests"] if case["probs"] else 0)), "flops": 4 * vocab * rows}
    keys = pairs = total = 0
    for rows, past in zip(*_lengths(case)):
        reach = case["window"] or rows + past
        keys += rows + past - max(0, past - reach + 1)
        pairs += sum(min(reach, past + i + 1) for i in range(rows))
        total += rows
    return {"bytes": 4 * total * n_q * d + keys * n_kv * row, "flops": 4.0 * d * n_q * pairs}


# ------------------------------------------------------------------------------------------------------------------------
# The definition in 64 bits, for one request or one table look-up at a time
# ------------------------------------------------------------------------------------------------------------------------
def _numbers():
    """What the 127 codes without a sign stand for, ascending."""
    return torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64, device="cuda")


def _nearest(x):
    """(numbers of the codes, scale bytes) of rows [..., d]: the nearest code, of two equally near ones the even one."""
    numbers = _numbers()
    scale = torch.tensor([2.0 ** n for n in range(-110, 122)], dtype=torch.float64, device="cuda")
    at = torch.searchsorted(scale * 448.0, x.abs().amax(dim=-1).contiguous())
    at = torch.where(x.abs().amax(dim=-1) == 0, torch.full_like(at, 110), at)
    y = x.abs() / scale[at].unsqueeze(-1)
    up = torch.searchsorted(numbers, y.contiguous()).clamp(1, 126)
    below, above = numbers[up - 1], numbers[up]
    higher = (above - y < y - below) | ((above - y == y - below) & (up % 2 == 0))
    return torch.copysign(torch.where(higher, above, below), x), at + 17


def exact(case, seed):
    if case["op"] == "verify":
        return None     # whole numbers
    s = prepare(case, seed)
    n_q, n_kv, d, page = s["n_q"], s["n_kv"], s["d"], s["page"]
    power = torch.tensor([2.0 ** (e - 127) for e in range(255)] + [math.nan], dtype=torch.float64, device="cuda")
    value = lambda name: s[name].double() * power[s[name + "_scale"].long()].unsqueeze(-1)  # noqa: E731
    if case["op"] == "load":
        return tuple(value(n).transpose(1, 2).reshape(-1, n_kv, d)[s["slots"].long()] for n in ("k", "v"))
    if case["op"] == "store":
        x = s["qkv"].double()
        if x.dim() == 3:
            for part in x[1:]:
                x[0] += part
            x = (x[0] + s["bias"].double()).to(torch.bfloat16).double()
        heads = list(x.view(-1, n_q + 2 * n_kv, d).unbind(dim=1))
        turn = torch.view_as_complex(s["table"].double().contiguous())
        for h in range(n_q + n_kv):
            z = torch.complex(*heads[h].split(d // 2, dim=-1)) * turn
            heads[h] = torch.cat((z.real, z.imag), dim=-1)
        out = {"q": torch.cat(heads[:n_q], dim=-1)}
        slots = s["slots"].long()
        for name, first in (("k", n_q), ("v", n_q + n_kv)):
            pool = s[name].double().transpose(1, 2).reshape(-1, n_kv, d)
            scales = s[name + "_scale"].long().transpose(1, 2).reshape(-1, n_kv)
            pool[slots], scales[slots] = _nearest(torch.stack(heads[first: first + n_kv], dim=1))
            out[name] = pool.view(-1, page, n_kv, d).transpose(1, 2)
            out[name + "_scale"] = scales.view(-1, page, n_kv).transpose(1, 2).to(torch.uint8)
        return out
    k, v, outs = value("k"), value("v"), []
    for b, rows in enumerate(s["q_lens"]):
        first, past = int(s["q_start"][b]), int(s["pos0"][b])
        own_pages = s["block_table"][b][: -(-(rows + past) // page)].long()
        q = s["q"][first: first + rows].double().view(rows, n_q, d)
        o = torch.empty_like(q)
        distance = torch.arange(past, past + rows, device="cuda")[:, None] - torch.arange(rows + past, device="cuda")
        hidden = (distance < 0) | (distance >= (case["window"] or rows + past + 1))
        for h in range(n_q):
            kv = h // (n_q // n_kv)
            keys, values = (t[own_pages, kv].reshape(-1, d)[: rows + past] for t in (k, v))
            o[:, h] = torch.softmax((q[:, h] @ keys.T / math.sqrt(d)).masked_fill(hidden, -math.inf), dim=-1) @ values
        outs.append(o.view(rows, n_q * d))
    return torch.cat(outs)
