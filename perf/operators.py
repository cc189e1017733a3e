"""Cases for timing the operators that decide which rows of the cache live on: beam search and the bounded cache.

A case is one call on the shapes of one decode step (sizes of ``ckpt.synthetic.SHAPES`` and of the benchmarks, random values):

* ``select``: the best ``2 * beams`` continuations per request out of ``beams`` rows of logits each.
* ``reorder``: every beam takes over its parent's recurrent states and the filled rows of its last page, in all layers.
* ``attend``: one query row per sequence against the paged cache, with the attention weights of the keys added up per KV head.
* ``evict``: the rows with the largest weights and the newest ones move to the front, into other pages, in all layers.

``run`` computes a case in elementary torch operations, or with ``own`` through the framework's calls. Sums and comparisons of log-probabilities
are in 64 bits, because candidates of different beams are told apart by their log-sum-exp; the rest is in 32 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 32
DEV = "cuda"


def _select(requests, beams, vocab, masked=False, dtype="float32"):
    return {"op": "select", "requests": requests, "beams": beams, "vocab": vocab, "masked": masked, "dtype": dtype}


def _reorder(requests, beams, layers, kv, dim, state_layers=0, state=0):
    return {"op": "reorder", "requests": requests, "beams": beams, "layers": layers, "kv": kv, "dim": dim, "state_layers": state_layers, "state": state}


def _attend(seqs, keys, spread, kv, group, dim, softcap=0.0):
    return {"op": "attend", "seqs": seqs, "keys": keys, "spread": spread, "kv": kv, "group": group, "dim": dim, "softcap": softcap}


def _evict(seqs, rows, spread, keep, recent, layers, kv, dim):
    return {"op": "evict", "seqs": seqs, "rows": rows, "spread": spread, "keep": keep, "recent": recent, "layers": layers, "kv": kv, "dim": dim}


def listed():
    return [
        # one user's request with four beams, the vocabulary of the benchmark model: launch latency and how far one request spreads over the GPU
        dict(_select(1, 4, 151936), name="select 1x4"),
        # constrained decoding (a tool call's grammar lets few tokens through), an odd vocabulary: rows that start on any address
        dict(_select(7, 3, 50257, masked=True), name="select 7x3 guided"),
        # a full batch: 64 requests with four beams each
        dict(_select(64, 4, 151936), name="select 64x4"),
        # one request with four beams, the caches of the benchmark model (36 layers, 8 KV heads of 128)
        dict(_reorder(1, 4, 36, 8, 128), name="reorder 1x4"),
        # a batch on narrow caches (22 layers, 4 KV heads of 64), eight beams
        dict(_reorder(16, 8, 22, 4, 64), name="reorder 16x8"),
        # a decoder of attention and gated linear attention layers: fp32 states of 4 heads x 256 x 512 beside pages
        dict(_reorder(16, 4, 12, 4, 128, state_layers=12, state=4 * 256 * 512), name="reorder 16x4 states"),
        # a single conversation
        dict(_attend(1, 4000, 0, 8, 4, 128), name="attend 1x4000"),
        # the benchmark's decode step: 64 sequences behind prompts of 2048 tokens
        dict(_attend(64, 2176, 128, 8, 4, 128), name="attend 64x2176"),
        # sequences of very different length, narrow heads in groups of eight
        dict(_attend(16, 16000, 15500, 4, 8, 64), name="attend 16x16000 ragged"),
        # one conversation shortened from 1100 to 1024 rows in all 36 layers
        dict(_evict(1, 1100, 0, 1024, 256, 36, 8, 128), name="evict 1x1100"),
        # a batch that decoded up to 256 tokens beyond its limit; some sequences are still below it
        dict(_evict(16, 2304, 300, 2048, 256, 36, 8, 128), name="evict 16x2304"),
        # long prompts cut to a quarter
        dict(_evict(4, 30000, 5000, 8192, 1024, 8, 8, 128), name="evict 4x30000"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("select", "reorder", "attend", "evict"))
    if op == "select":
        beams, vocab = rng.choice((2, 3, 4, 5, 6, 8, 12, 16)), _log(rng, 1000, 262208)
        return _select(min(_log(rng, 1, 64), max(1, 64 * 4 * 151936 // (beams * vocab))), beams, vocab, rng.random() < 0.3, rng.choice(("float32", "float32", "bfloat16")))
    kv, dim = rng.choice((1, 2, 4, 6, 8)), rng.choice((64, 128, 256))
    if op == "reorder":
        beams, layers = rng.choice((2, 3, 4, 5, 8, 16)), rng.randint(1, 48)
        state_layers = rng.choice((0, 0, rng.randint(1, 24)))
        state = _log(rng, 1000, 500000) // 4 * 4 if state_layers else 0
        per = beams * (layers * 2 * kv * dim * PAGE * 2 + state_layers * state * 4)
        return _reorder(min(_log(rng, 1, 32), max(1, 1200000000 // per)), beams, layers, kv, dim, state_layers, state)
    if op == "attend":
        keys = _log(rng, 1, 32000)
        seqs = min(_log(rng, 1, 128), max(1, 64 * 2048 * 8 * 128 // (keys * kv * dim)))
        return _attend(seqs, keys, rng.randint(0, keys - 1), kv, rng.randint(1, 16), dim, rng.choice((0.0, 0.0, 50.0)))
    keep = _log(rng, 20, 9000)
    rows = keep + _log(rng, 1, 2 * keep)
    layers = rng.randint(1, 36)
    seqs = min(_log(rng, 1, 32), max(1, 16 * 2048 * 36 * 8 * 128 // (rows * layers * kv * dim)))
    return _evict(seqs, rows, rng.randint(0, rows - 1), keep, rng.randint(0, keep), layers, kv, dim)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, most):
    """Lengths belong to the case, values to the seed: the first sequence is the longest."""
    rng = random.Random(7)
    return [most] + [most - rng.randint(0, case["spread"]) for _ in range(case["seqs"] - 1)]


def _tables(lens, g, first=1):
    """Pages in any order, as a pool that has been in use hands them out; page 0 is nobody's."""
    need = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(need), generator=g, device=DEV) + first
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    return table, first + sum(need)


def _splits(seqs, kv):
    """Split-KV factor of decode attention, as the engine picks it: the smallest that fills two CTAs per SM evenly."""
    best, share = 1, 0.0
    for s in range(1, 33):
        n = max(1, seqs * kv) * s
        if n / (-(-n // 296) * 296) > share + 0.03:
            best, share = s, n / (-(-n // 296) * 296)
    return best


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=g)


def _allowed(g, rows, vocab):
    """Bit masks as a grammar gives them: a handful to a fifth of the tokens, one row in eight with a single one, one beam at a dead end."""
    share = torch.rand(rows, 1, generator=g, device=DEV).square() * 0.2
    bits = torch.rand(rows, vocab, generator=g, device=DEV) < share
    lone = torch.arange(rows, device=DEV) % 8 == 5
    bits[lone] = False
    bits[lone, vocab // 3] = True
    if rows > 2:
        bits[2] = False
    words = -(-vocab // 32)
    b = torch.nn.functional.pad(bits, (0, words * 32 - vocab)).view(rows, words, 32).to(torch.int64)
    packed = (b << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)
    s = {"case": case, "own": None}
    if case["op"] == "select":
        B, W, V = case["requests"], case["beams"], case["vocab"]
        # a model's logits: a broad bell and a few tokens that stand out; beams of one request go on from nearly the same text
        base = _normal(g, B, 1, V, dtype=torch.float32) * 2.5
        peaks = torch.randint(0, V, (B, 1, 24), generator=g, device=DEV)
        base.scatter_add_(2, peaks, 6.0 + 4.0 * torch.rand(B, 1, 24, generator=g, device=DEV))
        logits = (base + 0.7 * _normal(g, B, W, V, dtype=torch.float32)).view(B * W, V)
        s["logits"] = logits.to(getattr(torch, case["dtype"]))
        s["scores"] = -(torch.rand(B, W, generator=g, device=DEV) * 1.5).cumsum(1) - 3.0
        s["mask"] = _allowed(g, B * W, V) if case["masked"] else None
        return s
    if case["op"] == "reorder":
        B, W = case["requests"], case["beams"]
        s["pages"] = (torch.randperm(B * W, generator=g, device=DEV) + 1).view(B, W)
        s["slots"] = (torch.randperm(B * W, generator=g, device=DEV) + 1).view(B, W)
        s["parents"] = torch.randint(0, W, (B, W), generator=g, device=DEV)
        rng = random.Random(7)
        s["rows"] = torch.tensor([rng.randint(1, PAGE) for _ in range(B)], dtype=torch.int32, device=DEV)
        s["caches"] = _normal(g, 2 * case["layers"], 1 + B * W, case["kv"], PAGE, case["dim"])
        s["cache_list"] = list(s["caches"].unbind(0))
        s["states"] = _normal(g, case["state_layers"], 1 + B * W, case["state"], dtype=torch.float32)
        s["state_list"] = list(s["states"].unbind(0))
        return s
    if case["op"] == "attend":
        B, KV, G, D = case["seqs"], case["kv"], case["group"], case["dim"]
        lens = _lengths(case, case["keys"])
        s["tables"], pages = _tables(lens, g)
        s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["most"], s["splits"], s["even"] = max(lens), _splits(B, KV), 2 * max(lens) * B <= 3 * sum(lens)
        s["q"] = _normal(g, B, KV * G * D)
        s["k"], s["v"] = _normal(g, pages, KV, PAGE, D), _normal(g, pages, KV, PAGE, D)
        s["weights"] = torch.rand(1 + B, KV, -(-max(lens) // PAGE) * PAGE + PAGE, generator=g, device=DEV) * 0.5
        s["slots"] = torch.randperm(B, generator=g, device=DEV) + 1
        return s
    B, L, KV, D = case["seqs"], case["layers"], case["kv"], case["dim"]
    lens = _lengths(case, case["rows"])
    s["tables"], pages = _tables(lens, g)
    s["out_tables"], pages = _tables([min(n, case["keep"]) for n in lens], g, pages)
    s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["k"], s["v"] = _normal(g, L, pages, KV, PAGE, D), _normal(g, L, pages, KV, PAGE, D)
    s["k_list"], s["v_list"] = list(s["k"].unbind(0)), list(s["v"].unbind(0))
    # attention sums are far from even; a tenth of the keys were never looked at
    w = _normal(g, L, 1 + B, KV, -(-max(lens) // PAGE) * PAGE + PAGE, dtype=torch.float32).mul_(2.0).exp_()
    s["weights"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.1, 0.0, w)
    s["weight_list"] = list(s["weights"].unbind(0))
    s["slots"] = torch.randperm(B, generator=g, device=DEV) + 1
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def _bits(mask, vocab):
    return ((mask.unsqueeze(-1) >> torch.arange(32, device=mask.device)) & 1).bool().flatten(1)[:, :vocab]


def _plain_select(s):
    case = s["case"]
    B, W, V, k = case["requests"], case["beams"], case["vocab"], 2 * case["beams"]
    x = s["logits"].double()
    if s["mask"] is not None:
        x = torch.where(_bits(s["mask"], V), x, -math.inf)
    m = x.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    x = x - m
    logp = x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    total = (s["scores"].double().view(B * W, 1) + logp).view(B, W * V)
    total = torch.where(torch.isfinite(total), total, -math.inf)
    values, at = (t[:, :k] for t in torch.sort(total, dim=-1, descending=True, stable=True))
    none = torch.isinf(values)
    return values.float(), torch.where(none, -1, at // V), torch.where(none, -1, at % V)


def _plain_reorder(s):
    pages, slots, parents = s["pages"], s["slots"], s["parents"]
    filled = (torch.arange(PAGE, device=DEV) < s["rows"].view(-1, 1)).view(-1, 1, 1, PAGE, 1)
    c = s["caches"]
    c[:, pages] = torch.where(filled, c[:, pages.gather(1, parents)], c[:, pages])
    s["states"][:, slots] = s["states"][:, slots.gather(1, parents)]
    return c, s["states"]


def _plain_attend(s):
    case = s["case"]
    B, KV, G, D, n = case["seqs"], case["kv"], case["group"], case["dim"], s["most"]
    dense = [t[s["tables"].long()].transpose(1, 2).reshape(B, KV, -1, D)[:, :, :n].float() for t in (s["k"], s["v"])]
    x = s["q"].view(B, KV, G, D).float() @ dense[0].transpose(2, 3) * D**-0.5
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    there = (torch.arange(n, device=DEV) < s["ctx"].view(-1, 1)).view(B, 1, 1, n)
    x = torch.where(there, x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    s["weights"][s["slots"], :, :n] += p.sum(2)
    return (p @ torch.where(there.transpose(2, 3), dense[1], 0.0)).to(s["q"].dtype).view(B, KV * G * D), s["weights"]


def _plain_evict(s):
    case, tables, out, ctx = s["case"], s["tables"].long(), s["out_tables"].long(), s["ctx"].view(-1, 1, 1)
    keep, k, v = case["keep"], s["k"], s["v"]
    w = s["weights"][:, s["slots"]]
    place = torch.arange(w.shape[-1], device=DEV)
    key = torch.where(place < ctx, torch.where(place >= ctx - case["recent"], math.inf, w), -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    there = torch.arange(keep, device=DEV) < ctx.clamp_max(keep)
    order = torch.sort(torch.where(there, order, w.shape[-1]), dim=-1).values
    kept = torch.where(there, order, -1)
    layer, b, head, j = there.expand_as(order).nonzero(as_tuple=True)
    i = order[layer, b, head, j]
    source, target = tables[b, i // PAGE], out[b, j // PAGE]
    k[layer, target, head, j % PAGE] = k[layer, source, head, i % PAGE]
    v[layer, target, head, j % PAGE] = v[layer, source, head, i % PAGE]
    front = torch.where(there, w.gather(-1, order.clamp_max(w.shape[-1] - 1)), 0.0)
    front = torch.nn.functional.pad(front, (0, w.shape[-1] - keep)) if keep < w.shape[-1] else front[..., : w.shape[-1]]
    s["weights"][:, s["slots"]] = torch.where(place < ctx, front, w)
    return kept.to(torch.int32), s["ctx"].clamp_max(keep), k, v, s["weights"]


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from deliverance_b200.ops.beam import beam_reorder, beam_select
        from deliverance_b200.ops.evict import decode_attention_weighted, evict_keys

        if op == "select":
            return beam_select(s["logits"], s["scores"], 2 * case["beams"], mask=s["mask"])
        if op == "reorder":
            beam_reorder(s["parents"], states=s["state_list"], slots=s["slots"], caches=s["cache_list"], pages=s["pages"], rows=s["rows"])
            return s["caches"], s["states"]
        if op == "attend":
            o = decode_attention_weighted(s["q"], s["k"], s["v"], s["tables"], s["ctx"], case["kv"] * case["group"], case["dim"] ** -0.5, s["weights"], s["slots"],
                                          softcap=case["softcap"], splits=s["splits"], even=s["even"])
            return o, s["weights"]
        kept, lens = evict_keys(s["k_list"], s["v_list"], s["weight_list"], s["tables"], s["ctx"], s["slots"], case["keep"], case["recent"], out_tables=s["out_tables"])
        return kept, lens, s["k"], s["v"], s["weights"]
    return {"select": _plain_select, "reorder": _plain_reorder, "attend": _plain_attend, "evict": _plain_evict}[op](s)


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    """Every input read once, every output written once. Reorder: expected distinct parents read and beams that do not stay written."""
    if case["op"] == "select":
        rows, V = case["requests"] * case["beams"], case["vocab"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": rows * V * size + (rows * (-(-V // 32)) * 4 if case["masked"] else 0) + case["requests"] * case["beams"] * (4 + 2 * 20), "flops": rows * V * 4.0}
    if case["op"] == "reorder":
        B, W = case["requests"], case["beams"]
        rng = random.Random(7)
        filled = sum(rng.randint(1, PAGE) for _ in range(B))
        per_beam = 2 * case["layers"] * case["kv"] * case["dim"] * 2 * filled / B + case["state_layers"] * case["state"] * 4
        moved, read = W * (1 - 1 / W), W * (1 - (1 - 1 / W) ** W)
        return {"bytes": B * per_beam * (moved + read), "flops": 0.0}
    if case["op"] == "attend":
        keys, KV, G, D = sum(_lengths(case, case["keys"])), case["kv"], case["group"], case["dim"]
        return {"bytes": keys * KV * (4.0 * D + 8) + 4.0 * case["seqs"] * KV * G * D, "flops": 4.0 * keys * KV * G * D}
    lens, L, KV, D = _lengths(case, case["rows"]), case["layers"], case["kv"], case["dim"]
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": L * KV * (kept * (8.0 * D + 4) + 8.0 * sum(lens)), "flops": 0.0}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_select(s, case):
    """The values; which candidates they belong to is a matter of order."""
    B, W, V, k = case["requests"], case["beams"], case["vocab"], 2 * case["beams"]
    values = []
    for b in range(B):
        rows = s["logits"][b * W : (b + 1) * W].double()
        if s["mask"] is not None:
            rows = rows.masked_fill(~_bits(s["mask"][b * W : (b + 1) * W], V), -math.inf)
        best = (torch.log_softmax(rows, -1) + s["scores"][b].double()[:, None]).nan_to_num(-math.inf, -math.inf, -math.inf)
        values.append(best.flatten().topk(k).values)
    return torch.stack(values), None, None


def _exact_reorder(s, case):
    caches, states = s["caches"].clone(), s["states"].clone()
    pages, slots, parents, rows = (s[n].tolist() for n in ("pages", "slots", "parents", "rows"))
    for b in range(case["requests"]):
        for j, p in enumerate(parents[b]):
            caches[:, pages[b][j], :, : rows[b]] = s["caches"][:, pages[b][p], :, : rows[b]]
            states[:, slots[b][j]] = s["states"][:, slots[b][p]]
    return caches, states


def _exact_attend(s, case):
    KV, G, D = case["kv"], case["group"], case["dim"]
    weights, out = s["weights"].double(), []
    slots = s["slots"].tolist()
    for b, n in enumerate(s["ctx"].tolist()):
        pages = s["tables"][b, : -(-n // PAGE)].long()
        K, V = (t[pages].permute(1, 0, 2, 3).reshape(KV, -1, D)[:, :n].double() for t in (s["k"], s["v"]))
        x = torch.einsum("kgd,knd->kgn", s["q"][b].double().view(KV, G, D), K) / math.sqrt(D)
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        p = torch.softmax(x, -1)
        weights[slots[b], :, :n] += p.sum(1)
        out.append(torch.einsum("kgn,knd->kgd", p, V).flatten())
    return torch.stack(out), weights


def _exact_evict(s, case):
    keep, recent, KV = case["keep"], case["recent"], case["kv"]
    k, v, weights = s["k"], s["v"], s["weights"]
    slots = s["slots"].tolist()
    for b, n in enumerate(s["ctx"].tolist()):
        m, w = min(n, keep), weights[:, slots[b], :, :n].clone()
        chosen = torch.ones_like(w, dtype=torch.bool)
        if n > keep:
            old = w[..., : n - recent]
            if keep > recent:
                edge = old.kthvalue(old.shape[-1] - (keep - recent) + 1, dim=-1, keepdim=True).values
                tie = old == edge
                room = keep - recent - (old > edge).sum(-1, keepdim=True)
                chosen[..., : n - recent] = (old > edge) | (tie & (tie.cumsum(-1) <= room))
            else:
                chosen[..., : n - recent] = False
        rows = chosen.nonzero()[:, -1].view(case["layers"], KV, m)
        to, fro = s["out_tables"][b].long(), s["tables"][b].long()
        for layer in range(case["layers"]):
            for t in (k[layer], v[layer]):
                mine = t[fro].transpose(0, 1).flatten(1, 2).gather(1, rows[layer].unsqueeze(-1).expand(-1, -1, t.shape[-1]))
                for at in range(0, m, PAGE):
                    part = mine[:, at : at + PAGE]
                    t[to[at // PAGE], :, : part.shape[1]] = part
        weights[:, slots[b], :, :n] = 0.0
        weights[:, slots[b], :, :m] = w.gather(-1, rows)
    return None, None, k, v, weights


def exact(case, seed):
    """From the definitions in 64 bits, request by request. Copies have no rounding: they are exact in their own type."""
    s = prepare(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s, case)
