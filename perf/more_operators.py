"""Cases for timing the operators of a KV cache in 4 bits: what writes it, what reads it, and the tables that say where a step's rows lie.

A case is one call on the shapes of one step of one layer (sizes of ``ckpt.synthetic.SHAPES`` and of the benchmarks, random values):

* ``write``: the q | k | v rows of a projection: head norms, rotation, queries out in bf16, keys and values quantised into pages; then the pages that got rows,
  unpacked to bf16.
* ``decode``: one query row per sequence against the 4-bit pages.
* ``prompt``: packed query rows of sequences of different lengths, causal, against the 4-bit pages, which may hold more rows in front of them.
* ``tables``: positions, cache slots, block tables, query tiles and last rows of a step from the requests' lengths and page lists.

A cached row is ``D / 2`` bytes of codes (byte i: element 2 i in the low half, 2 i + 1 in the high one), then per block of 32 elements its step and its minimum, both fp16; a value is
``code * step + minimum``. The steps have 7 significant bits. Quantising is defined by its fp32 roundings
(1 / 15 and the reciprocal of a step among them), so that codes can be compared.

``run`` computes a case in elementary torch operations, or with ``own`` through the framework's calls. Sums of squares are in 64 bits, because the codes behind them change in steps.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 32
TILE = 64  # query rows of a tile
LIMIT = 472.0  # largest magnitude that is held
DEV = "cuda"


def _write(tokens, seqs, heads, kv, dim, rot, layout="halves", norm=True, far=4096, scaled=1.0):
    return {"op": "write", "tokens": tokens, "seqs": seqs, "heads": heads, "kv": kv, "dim": dim, "rot": rot, "layout": layout, "norm": norm, "far": far, "scaled": scaled}


def _decode(seqs, keys, spread, kv, group, dim, softcap=0.0, window=0):
    return {"op": "decode", "seqs": seqs, "keys": keys, "spread": spread, "kv": kv, "group": group, "dim": dim, "softcap": softcap, "window": window}


def _prompt(seqs, tokens, spread, prefix, kv, group, dim, softcap=0.0, window=0):
    return {"op": "prompt", "seqs": seqs, "tokens": tokens, "spread": spread, "prefix": prefix, "kv": kv, "group": group, "dim": dim, "softcap": softcap, "window": window}


def _tables(seqs, tokens, spread, cached, width):
    return {"op": "tables", "seqs": seqs, "tokens": tokens, "spread": spread, "cached": cached, "width": width}


def listed():
    return [
        # a single user's decode step, heads of the benchmark model (32 on 8 of 128, head norms): launch latency
        dict(_write(1, 1, 32, 8, 128, 128), name="write 1"),
        # a batch that decodes far behind its trained context: scaled angles, half of each head rotated, neighbouring pairs, narrow heads, an odd number of rows
        dict(_write(61, 61, 16, 4, 64, 32, "pairs", False, 131072, 8.0), name="write 61 partial"),
        # a full step of the scheduler: 8,192 prompt tokens in four prompts
        dict(_write(8192, 4, 32, 8, 128, 128), name="write 8192"),
        # a single conversation
        dict(_decode(1, 4000, 0, 8, 4, 128), name="decode 1x4000"),
        # the benchmark's decode step: 64 sequences behind prompts of 2048 tokens
        dict(_decode(64, 2176, 128, 8, 4, 128), name="decode 64x2176"),
        # sequences of very different length, narrow heads in groups of eight
        dict(_decode(16, 16000, 15500, 4, 8, 64), name="decode 16x16000 ragged"),
        # 128 streams with wide heads and soft-capped scores, as in the benchmark's shared-prefix workload
        dict(_decode(128, 1920, 256, 8, 2, 256, softcap=50.0), name="decode 128x1920 wide"),
        # a chat turn of odd length arrives alone
        dict(_prompt(1, 333, 0, 0, 8, 4, 128), name="prompt 333"),
        # a full step of long prompts
        dict(_prompt(4, 2048, 0, 0, 8, 4, 128), name="prompt 4x2048"),
        # short questions of different lengths behind long cached documents, narrow heads, a sliding window
        dict(_prompt(7, 301, 290, 5000, 4, 8, 64, window=4096), name="prompt 7x301 cached"),
        # tables of a decode step of 64 sequences
        dict(_tables(64, 1, 0, 2176, 80), name="tables 64x1"),
        # tables of a full prompt step of ragged prompts behind cached prefixes
        dict(_tables(32, 350, 187, 1536, 80), name="tables 32x350"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "decode", "prompt", "tables"))
    if op == "tables":
        tokens = _log(rng, 1, 4096)
        seqs = min(_log(rng, 1, 256), max(1, 8192 // tokens))
        cached = rng.randint(0, 8000)
        return _tables(seqs, tokens, rng.randint(0, tokens - 1), cached, -(-(cached + tokens) // PAGE) + rng.randint(0, 64))
    kv, dim = rng.choice((1, 2, 4, 6, 8)), rng.choice((64, 128, 256))
    if op == "write":
        heads = kv * rng.randint(1, 8)
        rot = rng.choice((dim, dim, dim // 2, dim // 4))
        tokens = _log(rng, 1, max(1, 8192 * 48 * 128 // ((heads + 2 * kv) * dim)))
        return _write(min(tokens, 8192), rng.randint(1, min(tokens, 8192, 64)), heads, kv, dim, rot, rng.choice(("halves", "halves", "pairs")), rng.random() < 0.5,
                      rng.choice((4096, 32768, 131072)), rng.choice((1.0, 1.0, 4.0, 8.0)))
    softcap, window = rng.choice((0.0, 0.0, 50.0)), rng.choice((0, 0, 0, 1000))
    if op == "decode":
        keys = _log(rng, 1, 32000)
        seqs = min(_log(rng, 1, 128), max(1, 64 * 2048 * 8 * 128 // (keys * kv * dim)))
        return _decode(seqs, keys, rng.randint(0, keys - 1), kv, rng.randint(1, 16), dim, softcap, window)
    tokens = _log(rng, 1, 2048)
    prefix = rng.choice((0, 0, rng.randint(1, 6000)))
    group = rng.choice((1, 2, 4, 8))
    per = lambda n: n * (prefix + n / 2 + 1) * kv * group * dim / (4 * 2048 * 1024 * 32 * 128)  # noqa: E731  (of the largest listed case)
    while per(tokens) > 1:
        tokens -= tokens // 3
    seqs = max(1, min(_log(rng, 1, 16), int(1 / per(tokens))))
    return _prompt(seqs, tokens, rng.randint(0, tokens - 1), prefix, kv, group, dim, softcap, window)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, most):
    """Lengths belong to the case, values to the seed: the first sequence is the longest."""
    rng = random.Random(7)
    return [most] + [most - rng.randint(0, case["spread"]) for _ in range(case["seqs"] - 1)]


def _page_lists(lens, g):
    """Pages in any order, as a pool that has been in use hands them out; page 0 is nobody's."""
    need = [-(-n // PAGE) for n in lens]
    order = (torch.randperm(sum(need), generator=g, device=DEV) + 1).to(torch.int32)
    return order, need


def _block_tables(lens, g):
    order, need = _page_lists(lens, g)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    return table, 1 + sum(need)


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=g)


def _row_bytes(dim):
    return dim // 2 + dim // 8


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to(DEV)


def _filled(g, pages, kv, dim, keys):
    """A cache as earlier steps have left it: unit values, and in keys a few columns of a head that are several times as large as the others."""
    cache = torch.empty(pages, kv, PAGE, _row_bytes(dim), dtype=torch.uint8, device=DEV)
    loud = 1.0 + 5.0 * (torch.rand(kv, 1, dim, generator=g, device=DEV) < 0.03)
    step = max(1, (1 << 25) // (kv * PAGE * dim))
    for at in range(0, pages, step):
        x = _normal(g, min(step, pages - at), kv, PAGE, dim)
        cache[at : at + step] = _pack(x.float() * loud if keys else x.float())
    return cache


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)
    s = {"case": case, "own": None}
    op = case["op"]
    if op == "tables":
        rng = random.Random(7)
        new = _lengths(case, case["tokens"])
        cached = [case["cached"] - rng.randint(0, case["cached"]) * (i > 0) for i in range(case["seqs"])]
        s["pages"], need = _page_lists([a + b for a, b in zip(cached, new)], g)
        s["page_start"] = _ints([sum(need[:i]) for i in range(len(need) + 1)])
        s["cached"], s["new"] = _ints(cached), _ints(new)
        s["start"] = s["cached"] + torch.randint(0, 100, (case["seqs"],), generator=g, device=DEV).to(torch.int32)  # (positions run ahead of rows in a shortened cache)
        s["tokens"], s["tiles"] = sum(new), sum(-(-n // TILE) for n in new)
        return s
    if op == "write":
        T, H, KV, D, half = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"] // 2
        s["qkv"] = _normal(g, T, (H + 2 * KV) * D)
        first = random.Random(7)
        new = [T // case["seqs"] + (i < T % case["seqs"]) for i in range(case["seqs"])]
        cached = [first.randint(0, 2 * PAGE) for _ in new]
        tables, pages = _block_tables([a + b for a, b in zip(cached, new)], g)
        positions, slots, touched = [], [], []
        for i, (a, n) in enumerate(zip(cached, new)):
            row = torch.arange(a, a + n, device=DEV)
            page = tables[i].long()[row // PAGE]
            slots.append(page * PAGE + row % PAGE)
            touched.append(tables[i, a // PAGE : -(-(a + n) // PAGE)])
            positions.append(row + first.randint(0, case["far"] - T - 3 * PAGE) if case["far"] > T + 3 * PAGE else row % case["far"])
        s["slots"], s["positions"], s["touched"] = torch.cat(slots), torch.cat(positions).to(torch.int32), torch.cat(touched)
        s["k"], s["v"] = (torch.zeros(pages, KV, PAGE, _row_bytes(D), dtype=torch.uint8, device=DEV) for _ in range(2))
        turn = torch.arange(case["far"], dtype=torch.float64, device=DEV).view(-1, 1) * (1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half) / case["scaled"])
        s["cos"], s["sin"] = torch.cos(turn).float(), torch.sin(turn).float()
        s["q_norm"], s["k_norm"] = ((1.0 + 0.1 * _normal(g, D, dtype=torch.float32)).to(torch.bfloat16) for _ in range(2)) if case["norm"] else (None, None)
        return s
    KV, G, D = case["kv"], case["group"], case["dim"]
    if op == "decode":
        lens = _lengths(case, case["keys"])
        rows = case["seqs"]
    else:
        new = _lengths(case, case["tokens"])
        lens = [n + (case["prefix"] if i % 3 != 1 else 0) for i, n in enumerate(new)]
        rows = sum(new)
        s["q_start"], s["q_len"] = _ints([sum(new[:i]) for i in range(len(new))]), _ints(new)
        s["q_len_host"] = new
        # (a step's query tiles are made once for all its layers)
        s["tiles"] = {n: (_ints([i for i, m in enumerate(new) for _ in range(0, m, n)]), _ints([t for m in new for t in range(0, m, n)])) for n in (64, 128, 256)}
    s["lens"] = lens
    s["tables"], pages = _block_tables(lens, g)
    s["ctx"] = _ints(lens)
    s["q"] = _normal(g, rows, KV * G * D)
    s["k"], s["v"] = _filled(g, pages, KV, D, True), _filled(g, pages, KV, D, False)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def _pack(x):
    """fp32 ``[..., D]`` -> bytes ``[..., row bytes]``."""
    b = x.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    low = (b.amin(-1) + 0.0).half()
    step = (b.amax(-1) - low.float()).clamp_min(0.0) * (1.0 / 15.0)
    up = ((step.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)
    step = torch.where(step < 2.0**-14, torch.ceil(step * 2.0**20) * 2.0**-20, up)
    c = torch.where(step.unsqueeze(-1) > 0, (b - low.float().unsqueeze(-1)) * (1.0 / step).unsqueeze(-1), 0.0).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    side = torch.stack((step.half(), low), -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat((c[..., 0::2] | (c[..., 1::2] << 4), side), -1)


def _unpack(rows, dim, dtype=torch.float32):
    """Bytes ``[..., row bytes]`` -> values ``[..., D]``."""
    codes = rows[..., : dim // 2]
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 32)).to(dtype)
    side = rows[..., dim // 2 :].contiguous().view(torch.float16).unflatten(-1, (-1, 2)).to(dtype)
    return (c * side[..., :1] + side[..., 1:]).flatten(-2)


def _plain_write(s):
    case = s["case"]
    T, H, KV, D, half = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"] // 2
    q, k, v = s["qkv"].float().view(T, H + 2 * KV, D).split((H, KV, KV), 1)
    if case["norm"]:
        norm = lambda x, w: x * (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)).float() * w.float()  # noqa: E731
        q, k = norm(q, s["q_norm"]), norm(k, s["k_norm"])
    at = s["positions"].long()
    c, n = s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)

    def turn(x):
        x = x.clone()
        a, b = (x[..., :half], x[..., half : 2 * half]) if case["layout"] == "halves" else (x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2])
        a0, b0 = a * c - b * n, b * c + a * n
        a.copy_(a0)
        b.copy_(b0)
        return x

    q, k = turn(q), turn(k)
    page, row = s["slots"] // PAGE, s["slots"] % PAGE
    s["k"][page, :, row] = _pack(k)
    s["v"][page, :, row] = _pack(v)
    t = s["touched"].long()
    return q.to(s["qkv"].dtype).view(T, H * D), _unpack(s["k"][t], D).to(s["qkv"].dtype), _unpack(s["v"][t], D).to(s["qkv"].dtype)


def _plain_scores(x, case, seen):
    x = x * case["dim"] ** -0.5
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    x = torch.where(seen, x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_decode(s):
    case = s["case"]
    B, KV, G, D, n = case["seqs"], case["kv"], case["group"], case["dim"], case["keys"]
    k, v = (_unpack(t[s["tables"].long()], D).transpose(1, 2).reshape(B, KV, -1, D)[:, :, :n] for t in (s["k"], s["v"]))
    at, ctx = torch.arange(n, device=DEV), s["ctx"].view(-1, 1, 1, 1)
    seen = (at < ctx) & (at >= ctx - case["window"]) if case["window"] else at < ctx
    p = _plain_scores(s["q"].view(B, KV, G, D).float() @ k.transpose(2, 3), case, seen)
    return (p @ torch.where((at < ctx.view(-1, 1, 1)).unsqueeze(-1), v, 0.0)).to(s["q"].dtype).view(B, KV * G * D)


def _plain_prompt(s):
    case = s["case"]
    KV, G, D = case["kv"], case["group"], case["dim"]
    out, at = [], 0
    for b, (n, new) in enumerate(zip(s["lens"], s["q_len_host"])):
        pages = s["tables"][b, : -(-n // PAGE)].long()
        q = s["q"][at : at + new].view(new, KV, G, D).float()
        last, key = torch.arange(n - new, n, device=DEV).view(-1, 1), torch.arange(n, device=DEV)
        seen = (key <= last) & (key > last - case["window"]) if case["window"] else key <= last
        heads = []
        for h in range(KV):
            k, v = (_unpack(t[pages, h].flatten(0, 1)[:n], D) for t in (s["k"], s["v"]))
            heads.append((_plain_scores(q[:, h].transpose(0, 1) @ k.T, case, seen) @ v).transpose(0, 1))
        out.append(torch.stack(heads, 1).flatten(1))
        at += new
    return torch.cat(out).to(s["q"].dtype)


def _plain_tables(s):
    case, T, N = s["case"], s["tokens"], s["tiles"]
    new, cached, start, first, pages = (s[n].long() for n in ("new", "cached", "start", "page_start", "pages"))
    seqs = torch.arange(case["seqs"], device=DEV)
    q_start = new.cumsum(0) - new
    b = seqs.repeat_interleave(new, output_size=T)
    off = torch.arange(T, device=DEV) - q_start[b]
    row = cached[b] + off
    slots = pages[first[b] + row // PAGE] * PAGE + row % PAGE
    col = torch.arange(case["width"], device=DEV)
    table = torch.where(col < (first[1:] - first[:-1]).view(-1, 1), pages[(first[:-1].view(-1, 1) + col).clamp_max(pages.shape[0] - 1)], 0)
    tiles = (new + TILE - 1) // TILE
    tile_seq = seqs.repeat_interleave(tiles, output_size=N)
    tile_q0 = (torch.arange(N, device=DEV) - (tiles.cumsum(0) - tiles)[tile_seq]) * TILE
    small = [t.to(torch.int32) for t in (start[b] + off, q_start, cached + new, table, tile_seq, tile_q0)]
    return {"positions": small[0], "slots": slots, "q_start": small[1], "ctx_len": small[2], "block_tables": small[3], "logits_rows": q_start + new - 1, "tile_seq": small[4],
            "tile_q0": small[5]}


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from deliverance_b200.ops.kv4 import decode_attention4, expand4, prefill_attention4, rope_kv4
        from deliverance_b200.ops.tables import step_tables

        if op == "write":
            q = rope_kv4(s["qkv"], s["positions"], s["slots"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], s["k"], s["v"], case["heads"], case["kv"], case["dim"], 1e-6,
                         rotate=case["layout"])
            return (q,) + tuple(expand4(s["k"], s["v"], s["touched"]))
        if op == "decode":
            return decode_attention4(s["q"], s["k"], s["v"], s["tables"], s["ctx"], case["kv"] * case["group"], case["dim"] ** -0.5, softcap=case["softcap"], window=case["window"])
        if op == "prompt":
            return prefill_attention4(s["q"], s["k"], s["v"], s["tables"], s["q_start"], s["q_len"], s["ctx"], case["kv"] * case["group"], case["dim"] ** -0.5,
                                      softcap=case["softcap"], window=case["window"], q_len_host=s["q_len_host"], ctx_len_host=s["lens"], tiles_for=s["tiles"].get)
        t = step_tables(s["pages"], s["page_start"], s["cached"], s["start"], s["new"], s["tokens"], case["width"], PAGE, TILE, s["tiles"])
        return {n: getattr(t, n) for n in ("positions", "slots", "q_start", "ctx_len", "block_tables", "logits_rows", "tile_seq", "tile_q0")}
    return {"write": _plain_write, "decode": _plain_decode, "prompt": _plain_prompt, "tables": _plain_tables}[op](s)


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    """Every input read once, every output written once; products over the visible keys."""
    op = case["op"]
    if op == "tables":
        rng = random.Random(7)
        new = _lengths(case, case["tokens"])
        cached = [case["cached"] - rng.randint(0, case["cached"]) * (i > 0) for i in range(case["seqs"])]
        pages = sum(-(-(a + b) // PAGE) for a, b in zip(cached, new))
        return {"bytes": 4.0 * pages + 16 * case["seqs"] + 12 * sum(new) + case["seqs"] * (16 + 4 * case["width"]) + 8 * sum(-(-n // TILE) for n in new), "flops": 0.0}
    KV, D = case["kv"], case["dim"]
    if op == "write":
        T, H = case["tokens"], case["heads"]
        pages = case["seqs"] * (1 + T / case["seqs"] / PAGE)
        return {"bytes": T * (4.0 * H * D + 4 * KV * D + 2 * KV * _row_bytes(D) + 4 * case["rot"] + 12) + pages * PAGE * KV * 2 * (_row_bytes(D) + 2 * D), "flops": 6.0 * T * (H + KV) * D}
    G = case["group"]
    if op == "decode":
        lens = [min(n, case["window"] or n) for n in _lengths(case, case["keys"])]
        return {"bytes": sum(lens) * KV * 2.0 * _row_bytes(D) + 4.0 * case["seqs"] * KV * G * D, "flops": 4.0 * sum(lens) * KV * G * D}
    new = _lengths(case, case["tokens"])
    bytes_, pairs = 0.0, 0
    for i, n in enumerate(new):
        before, w = case["prefix"] if i % 3 != 1 else 0, case["window"] or 1 << 30
        bytes_ += 4.0 * n * KV * G * D + min(before + n, w + n) * KV * 2.0 * _row_bytes(D)
        pairs += sum(min(before + j + 1, w) for j in range(n))
    return {"bytes": bytes_, "flops": 4.0 * pairs * KV * G * D}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _quantised(x):
    """The values that fp32 numbers become, block by block: 64-bit arithmetic, rounded to fp32 where the definition rounds."""
    b = torch.clamp(x.double(), -LIMIT, LIMIT).reshape(-1, 32)
    low = b.min(1, keepdim=True).values.half().double()
    step = ((b.max(1, keepdim=True).values - low).float().double().clamp_min(0.0) * torch.tensor(1.0 / 15.0).double().item()).float().double()
    frac, exp = torch.frexp(step)  # step = frac 2^exp, 1/2 <= frac < 1
    up = torch.ldexp(torch.ceil(frac * 128.0), (exp - 7).double())
    step = torch.where(step < 2.0**-14, torch.ceil(step * 2.0**20) / 2.0**20, up)
    inverse = (torch.ones_like(step) / step).float().double()
    c = torch.round(((b - low).float().double() * inverse).float().double()).clamp(0.0, 15.0)
    return torch.where(step > 0, c * step + low, low).view(x.shape)


def _exact_write(s, case):
    T, H, KV, D, half = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"] // 2
    rows = s["qkv"].view(T, H + 2 * KV, D)
    q, k = rows[:, :H].double(), rows[:, H : H + KV].double()
    f32 = lambda x: x.float().double()  # noqa: E731
    if case["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"].double()
        k = f32(f32(k * f32(1.0 / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6))) * s["k_norm"].double())
    where = s["positions"].long()
    c, n = s["cos"].double()[where][:, None], s["sin"].double()[where][:, None]
    i = torch.arange(half, device=DEV)
    first, second = (i, i + half) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
    a, b = q[..., first], q[..., second]
    q[..., first], q[..., second] = a * c - b * n, b * c + a * n
    a, b = k[..., first], k[..., second]
    k[..., first], k[..., second] = f32(f32(a * c) - f32(b * n)), f32(f32(b * c) + f32(a * n))
    out = [q.flatten(1)]
    for fresh in (k, rows[:, H + KV :].double()):
        held = torch.zeros(s["k"].shape[0] * PAGE, KV, D, dtype=torch.float64, device=DEV)
        held[s["slots"]] = _quantised(fresh)
        out.append(held.view(-1, PAGE, KV, D).transpose(1, 2)[s["touched"].long()])
    return tuple(out)


def _exact_rows(s, case, name, b):
    n = s["lens"][b]
    rows = s[name][s["tables"][b, : -(-n // PAGE)].long()].transpose(0, 1).flatten(1, 2)[:, :n]
    D = case["dim"]
    side = rows[..., D // 2 :].contiguous().view(torch.float16).double()
    out = torch.empty(*rows.shape[:2], D, dtype=torch.float64, device=DEV)
    out[..., 0::2], out[..., 1::2] = (rows[..., : D // 2] % 16).double(), (rows[..., : D // 2] // 16).double()
    return out * side[..., 0::2].repeat_interleave(32, -1) + side[..., 1::2].repeat_interleave(32, -1)


def _exact_attention(s, case):
    KV, G, D = case["kv"], case["group"], case["dim"]
    new = s.get("q_len_host") or [1] * case["seqs"]
    out, at = [], 0
    for b, (n, m) in enumerate(zip(s["lens"], new)):
        K, V = (_exact_rows(s, case, name, b) for name in ("k", "v"))
        q = s["q"][at : at + m].double().view(m, KV, G, D)
        hidden = torch.ones(m, n, dtype=torch.bool, device=DEV).tril(n - m).logical_not()
        if case["window"]:
            hidden |= torch.ones(m, n, dtype=torch.bool, device=DEV).tril(n - m - case["window"])
        part = torch.empty(m, KV, G, D, dtype=torch.float64, device=DEV)
        for h in range(KV):
            for i in range(G):
                x = torch.einsum("td,nd->tn", q[:, h, i], K[h]) / math.sqrt(D)
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                part[:, h, i] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ V[h]
        out.append(part.flatten(1))
        at += m
    return torch.cat(out)


def exact(case, seed):
    """From the definitions in 64 bits, sequence by sequence. Tables are whole numbers."""
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    return _exact_write(s, case) if case["op"] == "write" else _exact_attention(s, case)
