"""Decode attention that adds up its keys' weights, and the eviction that goes by them, against plain statements in 64 bits. On the CPU and, on a GPU
box, on the CUDA kernels."""
import math

import pytest
import torch

from deliverance_b200 import ops
from deliverance_b200.ops.evict import decode_attention_weighted, evict_keys

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, F32 = torch.bfloat16, torch.float32
P = 32


def tables_for(lens, first=1, extra=0):
    need = [-(-n // P) for n in lens]
    order = (torch.randperm(sum(need)) + first).to(torch.int32)
    t = torch.zeros(len(lens), max(max(need), 1) + extra, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at : at + n]
        at += n
    return t, first + sum(need)


def dense(cache, table, n):
    return cache[table[: -(-n // P)].long()].permute(1, 0, 2, 3).reshape(cache.shape[1], -1, cache.shape[3])[:, :n].double()


def plain_attention(q, k, v, table, lens, KV, scale, softcap, window):
    """fp64 outputs [B, H * D] and per sequence the probabilities summed over a KV head's query heads, [KV, n]."""
    B, D = q.shape[0], k.shape[3]
    out, sums = torch.zeros(B, q.shape[1], dtype=torch.float64), []
    for b, n in enumerate(lens):
        K, V = dense(k, table[b], n), dense(v, table[b], n)
        s = q[b].double().view(KV, -1, D) @ K.transpose(1, 2) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if window and n > window:
            s[:, :, : n - window] = -math.inf
        p = torch.softmax(s, -1) if n else s
        sums.append(p.sum(1))
        out[b] = (p @ V).flatten()
    return out, sums


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("KV,G", [(1, 1), (2, 4), (3, 5), (1, 16), (8, 8)])
@pytest.mark.parametrize("lens,splits", [([1], 1), ([33, 0, 1, 500], 1), ([700, 31, 32], 8), ([3001, 2], 32), ([64] * 70, 3)])
def test_weighted_attention_matches_plain(device, D, KV, G, lens, splits):
    if device == "cpu" and sum(lens) * KV * G * D > 3e7:
        pytest.skip("large for the CPU")
    run_attention(device, D, KV, G, lens, splits, 0.0, 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("softcap,window", [(50.0, 0), (0.5, 0), (0.0, 100), (50.0, 17)])
def test_weighted_attention_softcap_window(device, D, softcap, window):
    run_attention(device, D, 2, 2, [777, 16, 100, 101], 6, softcap, window)


def run_attention(device, D, KV, G, lens, splits, softcap, window, capacity=None, extra=1, even=False):
    B, H = len(lens), KV * G
    table, pages = tables_for(lens, extra=extra)
    q = torch.randn(B, H * D).to(BF16)
    k, v = torch.randn(pages, KV, P, D).to(BF16), torch.randn(pages, KV, P, D).to(BF16)
    # what lies behind a sequence's end must not matter
    for b, n in enumerate(lens):
        if n % P:
            k[table[b, n // P].long(), :, n % P :] = math.nan
            v[table[b, n // P].long(), :, n % P :] = math.nan
    cap = capacity or max(lens) + 7
    start = torch.rand(B + 2, KV, cap)
    slots = torch.randperm(B) + 1
    to = lambda t: t.to(device)  # noqa: E731
    w = to(start.clone())
    ctx = torch.tensor(lens, dtype=torch.int32)
    scale = D**-0.5
    out = decode_attention_weighted(to(q), to(k), to(v), to(table), to(ctx), H, scale, w, to(slots), softcap, window, splits, even)
    if device == "cuda":
        ops.check_status(0)
    want, sums = plain_attention(q, k, v, table, lens, KV, scale, softcap, window)
    out, w = out.cpu().double(), w.cpu().double()
    # Output: probabilities rounded to bf16 (2^-8 of each, against sum p |v| <= max |v|) and the result's own rounding; fp32 in between is far below.
    for b, n in enumerate(lens):
        top = float(dense(v, table[b], n).abs().max()) if n else 0.0
        assert (out[b] - want[b]).abs().max() <= 2**-8 * (want[b].abs().max() + top) + 1e-6, b
    # Weights: a score s = scale * q.k carries D + 2 fp32 roundings of at most sum |q k| * scale (here below 5 sqrt(D) for normal values), exp and __expf 2^-22 + 2^-23 |s|, the sum over n
    # probabilities and heads n * 2^-24 at the worst; relative to the probability. The addition rounds to 2^-24 of the entry.
    expect = start.double()
    for b, n in enumerate(lens):
        m = min(n, cap)
        expect[slots[b], :, :m] += sums[b][:, :m]
    for b, n in enumerate(lens):
        m = min(n, cap)
        slack = 5 * math.sqrt(D) * (D + 2) * 2**-24 + 64 * 2**-23 + n * 2**-24
        d = (w[slots[b], :, :m] - expect[slots[b], :, :m]).abs()
        assert (d <= sums[b][:, :m] * slack + expect[slots[b], :, :m] * 2**-23).all(), (b, float(d.max()))
        assert torch.equal(w[slots[b], :, m:], start[slots[b], :, m:].double())
    for s in range(B + 2):
        if s not in slots.tolist():
            assert torch.equal(w[s], start[s].double())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,splits", [([9000], 30), ([4001, 4000], 18), ([40, 33], 5), ([1], 2), ([0, 0], 3)])
def test_weighted_attention_of_like_lengths(device, D, lens, splits):
    run_attention(device, D, 2, 4, lens, splits, 0.0, 0, even=True)
    run_attention(device, D, 1, 3, lens, splits, 30.0, 700, even=True)


@pytest.mark.parametrize("device", DEVICES)
def test_weights_shorter_than_the_sequence(device):
    run_attention(device, 64, 2, 4, [300, 90, 129], 4, 0.0, 0, capacity=100)
    run_attention(device, 128, 1, 2, [300, 90, 129], 1, 0.0, 0, capacity=129, extra=40)


@pytest.mark.parametrize("device", DEVICES)
def test_weights_add_up_over_steps(device):
    """Ten steps on one cache: every step adds one per query head in all; strided query rows."""
    KV, G, D, n = 2, 3, 64, 210
    table, pages = tables_for([n, n - 50])
    k, v = torch.randn(pages, KV, P, D).to(BF16).to(device), torch.randn(pages, KV, P, D).to(BF16).to(device)
    w = torch.zeros(3, KV, 256, device=device)
    for i in range(10):
        q = torch.randn(2, KV * G * D + 64).to(BF16).to(device)[:, 2 : 2 + KV * G * D]
        decode_attention_weighted(q, k, v, table.to(device), torch.tensor([n, n - 50], dtype=torch.int32, device=device), KV * G, 0.125, w,
                                  torch.tensor([2, 1], device=device), splits=1 + i % 4)
    total = w.double().sum(-1).cpu()
    assert (total[1:] - 10 * G).abs().max() < 10 * G * 1e-5 and float(total[0].abs().max()) == 0
    assert float(w[2, :, n:].abs().max()) == 0 and float(w[1, :, n - 50 :].abs().max()) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_scratch_slot_adds_nothing(device):
    """Padded rows of a captured step share slot 0."""
    KV, D = 1, 64
    k, v = torch.randn(3, KV, P, D).to(BF16).to(device), torch.randn(3, KV, P, D).to(BF16).to(device)
    w = torch.zeros(2, KV, 64, device=device)
    decode_attention_weighted(torch.randn(3, D).to(BF16).to(device), k, v, torch.tensor([[1], [0], [0]], dtype=torch.int32, device=device),
                              torch.tensor([20, 1, 1], dtype=torch.int32, device=device), 1, 0.125, w, torch.tensor([1, 0, 0], device=device))
    assert float(w[0].abs().max()) == 0 and abs(float(w[1].sum()) - 1) < 1e-5
    if device == "cuda":
        ops.check_status(0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("slots", [[1, 1], [1, 9], [-1, 1]])
def test_bad_slots_are_reported(device, slots):
    KV, D = 1, 64
    k, v = torch.randn(3, KV, P, D).to(BF16).to(device), torch.randn(3, KV, P, D).to(BF16).to(device)
    w = torch.zeros(3, KV, 64, device=device)
    args = (torch.randn(2, D).to(BF16).to(device), k, v, torch.tensor([[1], [2]], dtype=torch.int32, device=device), torch.tensor([20, 10], dtype=torch.int32, device=device))
    with pytest.raises((IndexError, RuntimeError)):
        decode_attention_weighted(*args, 1, 0.125, w, torch.tensor(slots, device=device))
        ops.check_status(0)
    if device == "cuda":  # the good one counted, the bad one did not
        assert abs(float(w.sum()) - 1) < 1e-5
    kept_w = w.clone()
    with pytest.raises((IndexError, RuntimeError)):
        evict_keys([k], [v], [w], args[3], args[4], torch.tensor(slots, device=device), 5, 2)
        ops.check_status(0)
    bad = [s for s in range(3) if s not in slots]
    assert torch.equal(w[bad], kept_w[bad])


# ---------------------------------------------------------------------------------------------------------------- eviction
def plain_evict(w, n, keep, recent):
    """Rows kept of one head: fp64 weights [n]."""
    if n <= keep:
        return list(range(n))
    old = sorted(range(n - recent), key=lambda i: (math.isnan(w[i]), -w[i] if not math.isnan(w[i]) else 0.0, i))[: keep - recent]
    return sorted(old) + list(range(n - recent, n))


def run_evict(device, lens, keep, recent, L=2, KV=2, D=64, DV=None, dtype=BF16, capacity=None, out="same", weights=None, shared=()):
    B = len(lens)
    table, pages = tables_for(lens, extra=1)
    target = table.clone()
    if out != "same":
        fresh, pages = tables_for([min(n, keep) for n in lens], pages)
        if out == "fresh":
            target = fresh
        else:  # the first pages are held by others, the rest are the sequence's own
            for b in range(B):
                for j in range(min(shared[b], fresh.shape[1])):
                    if j < -(-min(lens[b], keep) // P):
                        target[b, j] = fresh[b, j]
    k = [torch.randn(pages, KV, P, D).to(dtype) for _ in range(L)]
    v = [torch.randn(pages, KV, P, DV or D).to(dtype) for _ in range(L)]
    cap = capacity or max(lens) + 5
    w = weights if weights is not None else [torch.where(torch.rand(B + 2, KV, cap) < 0.3, 0.0, torch.randn(B + 2, KV, cap).exp()) for _ in range(L)]
    slots = torch.randperm(B) + 1
    to = lambda t: t.clone().to(device)  # noqa: E731
    K, V, Wt = [to(t) for t in k], [to(t) for t in v], [to(t) for t in w]
    kept, new = evict_keys(K, V, Wt, to(table), torch.tensor(lens, dtype=torch.int32).to(device), to(slots), keep, recent, None if out == "same" else to(target))
    if device == "cuda":
        ops.check_status(0)
    assert kept.dtype == torch.int32 and new.tolist() == [min(n, keep) for n in lens]
    kept = kept.cpu()
    for i in range(L):
        want_k, want_v, want_w = k[i].clone(), v[i].clone(), w[i].clone()
        for b, n in enumerate(lens):
            s, m = int(slots[b]), min(n, keep)
            for h in range(KV):
                full = w[i][s, h, : min(n, cap)].tolist() + [0.0] * (n - min(n, cap))
                rows = plain_evict(full, n, keep, recent)
                assert kept[i, b, h].tolist() == rows + [-1] * (keep - m), (i, b, h)
                for t, o in ((k[i], want_k), (v[i], want_v)):
                    for j, r in enumerate(rows):
                        o[target[b, j // P].long(), h, j % P] = t[table[b, r // P].long(), h, r % P]
                if n > keep:
                    c = min(n, cap)
                    want_w[s, h, :c] = torch.tensor(([full[r] for r in rows] + [0.0] * n)[:c])
        assert torch.equal(K[i].cpu(), want_k) and torch.equal(V[i].cpu(), want_v)
        assert torch.equal(torch.nan_to_num(Wt[i].cpu(), -5.0), torch.nan_to_num(want_w, -5.0))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,keep,recent", [([1], 1, 0), ([2], 1, 0), ([2], 1, 1), ([0, 5, 70], 33, 8), ([100, 64, 65, 63], 64, 64), ([100, 97], 96, 0), ([513, 512, 3], 200, 31), ([1500], 1030, 100)])
@pytest.mark.parametrize("out", ["same", "fresh", "mixed"])
def test_evict_matches_plain(device, lens, keep, recent, out):
    run_evict(device, lens, keep, recent, out=out, shared=[i % 3 for i in range(1, 1 + len(lens))])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,DV,dtype", [(128, 128, BF16), (256, 64, BF16), (6, 6, BF16), (5, 3, BF16), (20, 20, F32), (5, 7, F32), (1032, 1032, F32), (2052, 20, F32)])
def test_evict_widths(device, D, DV, dtype):
    run_evict(device, [90, 200], 64, 10, L=1, D=D, DV=DV, dtype=dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_evict_ties_infinities_nan(device):
    """All weights equal, all zero, infinities of both signs, NaN, negative zero."""
    L, KV, n = 1, 2, 700
    for fill in (0.0, 1.5, math.nan):
        run_evict(device, [n], 300, 20, L=L, KV=KV, weights=[torch.full((3, KV, n), fill)])
    w = torch.randn(3, KV, n)
    w[:, :, ::3] = math.nan
    w[:, :, 1::7] = math.inf
    w[:, :, 2::5] = -math.inf
    w[:, :, 4::9] = 0.0
    w[:, :, 5::9] = -0.0
    for keep in (50, 350, 600, 699):
        run_evict(device, [n], keep, 20, L=L, KV=KV, weights=[w])


@pytest.mark.parametrize("device", DEVICES)
def test_evict_beyond_the_capacity(device):
    run_evict(device, [400, 90, 150], 120, 30, capacity=100)
    run_evict(device, [400, 90, 150], 64, 30, capacity=150)


@pytest.mark.parametrize("device", DEVICES)
def test_evict_many_layers(device):
    run_evict(device, [70], 40, 10, L=100, KV=1, D=8)


@pytest.mark.gpu
def test_evict_long_sequences():
    """More rows than the selection holds in registers; offsets of rows far into a page table."""
    run_evict("cuda", [9000, 4097], 4000, 500, L=1, KV=1, D=8)
    run_evict("cuda", [2561, 2560], 1001, 0, L=1, KV=1, D=8)
    run_evict("cuda", [10241, 20000], 5000, 4999, L=1, KV=1, D=8)
    run_evict("cuda", [40000, 100], 10000, 17, L=1, KV=1, D=8)
    run_evict("cuda", [40000], 39999, 17, L=1, KV=1, D=8, weights=[torch.zeros(3, 1, 40000)])
    for n in (2560, 9000, 30001):  # ties over many rows of a thread: few values, one value
        run_evict("cuda", [n], n // 3, n // 7, L=1, KV=2, D=8, weights=[torch.randint(0, 3, (3, 2, n)).float()])
        run_evict("cuda", [n], n - 1, 0, L=1, KV=1, D=8, weights=[torch.full((3, 1, n), 0.25)])
        run_evict("cuda", [n], n // 2, 5, L=1, KV=1, D=8, capacity=n // 2 + 77)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    KV, D = 2, 64
    k, w = torch.zeros(4, KV, P, D, dtype=BF16, device=device), torch.zeros(3, KV, 64, device=device)
    v = k.clone()
    t, n, s = torch.ones(1, 2, dtype=torch.int32, device=device), torch.tensor([40], dtype=torch.int32, device=device), torch.ones(1, dtype=torch.int64, device=device)
    q = torch.zeros(1, 4 * D, dtype=BF16, device=device)
    for bad in (lambda: evict_keys([], [], [], t, n, s, 8, 2), lambda: evict_keys([k], [v], [w], t, n, s, 8, 9), lambda: evict_keys([k], [v], [w], t, n, s, 0, 0),
                lambda: evict_keys([k], [k], [w], t, n, s, 8, 2), lambda: evict_keys([k], [v], [w[:, :1]], t, n, s, 8, 2), lambda: evict_keys([k], [v], [w.double()], t, n, s, 8, 2),
                lambda: evict_keys([k], [v], [w], t.long(), n, s, 8, 2), lambda: evict_keys([k], [v], [w], t, n, s.int(), 8, 2),
                lambda: evict_keys([k], [v], [w], t, n, s, 8, 2, t[0]), lambda: decode_attention_weighted(q, k, v, t, n, 4, 0.1, w[0], s),
                lambda: decode_attention_weighted(q, k, v, t, n, 4, 0.1, w, s.int()), lambda: decode_attention_weighted(q, k, v, t, n, 4, 0.1, w.half(), s)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    if device == "cuda":
        for bad in (lambda: evict_keys([k], [v], [w], t, n, s, 40, 2, t[:, :1]), lambda: decode_attention_weighted(q.float(), k, v, t, n, 4, 0.1, w, s),
                    lambda: decode_attention_weighted(torch.zeros(1, 34 * D, dtype=BF16, device=device), k, v, t, n, 34, 0.1, w, s), lambda: decode_attention_weighted(q, k, v, t.cpu(), n, 4, 0.1, w, s)):
            with pytest.raises(RuntimeError):
                bad()
    with pytest.raises((IndexError, RuntimeError)):  # a page outside the cache: left out, and reported
        evict_keys([k], [v], [w], torch.tensor([[1, 7]], dtype=torch.int32, device=device), n, s, 38, 2)
        ops.check_status(0)


# ---------------------------------------------------------------------------------------------------------------- together
def run_together(device, steps=24, W=3, L=2, KV=2, G=4, D=64, keep=40, recent=10):
    """Beams of one request on a bounded cache, operator by operator: every step writes a row per beam, attends and adds weights in all layers, selects, reorders pages, weights
    and a recurrent state; every eight steps all beams are shortened into pages of their own. Returns everything that can be compared."""
    from deliverance_b200.ops.beam import beam_reorder, beam_select

    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    to = lambda t: t.to(device)  # noqa: E731
    pool = 64
    k, v = ([to(rnd(pool, KV, P, D).to(BF16)) for _ in range(L)] for _ in range(2))
    weights = [to(torch.zeros(W + 1, KV, 160)) for _ in range(L)]
    state = to(rnd(W + 1, 50))
    n, free = 70, list(range(pool - 1, 0, -1))
    shared = [free.pop() for _ in range(n // P)]
    pages = [shared + [free.pop()] for _ in range(W)]
    slots = to(torch.arange(1, W + 1))
    for layer in range(L):  # all beams start with the same rows
        for j in range(1, W):
            k[layer][pages[j][-1]] = k[layer][pages[0][-1]]
            v[layer][pages[j][-1]] = v[layer][pages[0][-1]]
    scores, picked, kept_rows = torch.tensor([[0.0, -0.5, -1.0]]), [], []
    for step in range(steps):
        if n % P == 0:
            for pg in pages:
                pg.append(free.pop())
        for layer in range(L):
            for pg in pages:
                k[layer][pg[n // P], :, n % P] = to(rnd(KV, D).to(BF16))
                v[layer][pg[n // P], :, n % P] = to(rnd(KV, D).to(BF16))
        n += 1
        table = torch.zeros(W, 8, dtype=torch.int32)
        for j, pg in enumerate(pages):
            table[j, : len(pg)] = torch.tensor(pg)
        ctx = torch.full((W,), n, dtype=torch.int32)
        outs = [decode_attention_weighted(to(rnd(W, KV * G * D).to(BF16)), k[i], v[i], to(table), to(ctx), KV * G, D**-0.5, weights[i], slots, splits=1 + step % 5) for i in range(L)]
        values, parents, tokens = beam_select(to(rnd(W, 1000) * 3), to(scores), 2 * W)
        picked.append((parents.cpu(), tokens.cpu()))
        par = parents[:, :W].contiguous()
        full = n // P
        lists = [pages[p][:full] for p in par[0].tolist()]
        tails = torch.tensor([[pg[full] if n % P else 0 for pg in pages]])
        beam_reorder(par, states=weights + [state], slots=slots.view(1, -1), caches=k + v if n % P else (), pages=to(tails) if n % P else None,
                     rows=to(torch.tensor([n % P], dtype=torch.int32)) if n % P else None)
        pages = [a + pg[full:] for a, pg in zip(lists, pages)]
        scores = values[:, :W].cpu()
        if step % 8 == 7:
            table = torch.zeros(W, 8, dtype=torch.int32)
            out = torch.zeros(W, 2, dtype=torch.int32)
            fresh = [[free.pop(), free.pop()] for _ in range(W)]
            for j, pg in enumerate(pages):
                table[j, : len(pg)] = torch.tensor(pg)
                out[j] = torch.tensor(fresh[j])
            kept, lens = evict_keys(k, v, weights, to(table), to(ctx), slots, keep, recent, to(out))
            assert lens.tolist() == [keep] * W
            kept_rows.append(kept.cpu())
            pages, n = fresh, keep
    if device == "cuda":
        ops.check_status(0)
    return picked, kept_rows, [t.cpu() for t in weights], state.cpu(), [dense(t.cpu(), torch.tensor(pg), n) for t in k + v for pg in pages], [o.cpu().float() for o in outs]


def test_operators_together_on_the_cpu():
    picked, kept, weights, state, rows, outs = run_together("cpu")
    assert len(kept) == 3 and all((r[:, :, :, 1:] > r[:, :, :, :-1]).all() for r in kept)
    # what a row has gathered since it came is at most one per query head and step
    assert all(float(w.max()) <= 4 * 24 and float(w[:, :, 40:].abs().max()) == 0 for w in weights)


@pytest.mark.gpu
def test_operators_together():
    a, b = run_together("cpu"), run_together("cuda")
    for (p, t), (q, u) in zip(a[0], b[0]):
        assert torch.equal(p, q) and torch.equal(t, u)
    assert all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    for x, y in zip(a[2], b[2]):
        # (24 steps of the tolerance that a step has against 64 bits, on either side)
        assert (x - y).abs().max() <= 2 * 24 * 4 * (5 * 8 * 66 * 2**-24 + 64 * 2**-23 + 100 * 2**-24)
    assert torch.equal(a[3], b[3]) and all(torch.equal(x, y) for x, y in zip(a[4], b[4]))
    assert all((x - y).abs().max() <= 2**-8 * (x.abs().max() + 6) + 2**-8 * x.abs().max() for x, y in zip(a[5], b[5]))


@pytest.mark.gpu
def test_captured_and_replayed():
    """Attention, eviction and reordering in two captured graphs, replayed in turn, against the same calls made one by one; on a stream of their own too."""
    from deliverance_b200.ops.beam import beam_reorder

    def world(seed):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        table, pages = tables_for([100, 77])
        s = dict(k=rnd(pages, 2, P, 64).to(BF16).cuda(), v=rnd(pages, 2, P, 64).to(BF16).cuda(), w=torch.rand(3, 2, 128, generator=g).cuda(), q=rnd(2, 512).to(BF16).cuda(),
                 table=table.cuda(), ctx=torch.tensor([100, 77], dtype=torch.int32).cuda(), short=torch.tensor([50, 50], dtype=torch.int32).cuda(), slots=torch.tensor([2, 1]).cuda(),
                 parents=torch.tensor([[1, 1]]).cuda(), rows=torch.tensor([18], dtype=torch.int32).cuda())
        s["tails"] = s["table"][:, 1].long().view(1, 2).contiguous()
        return s

    def work(s):
        o = decode_attention_weighted(s["q"], s["k"], s["v"], s["table"], s["ctx"], 8, 0.125, s["w"], s["slots"], splits=4)
        kept, _ = evict_keys([s["k"]], [s["v"]], [s["w"]], s["table"], s["ctx"], s["slots"], 50, 9)
        beam_reorder(s["parents"], [s["w"]], s["slots"].view(1, 2), [s["k"], s["v"]], s["tails"], s["rows"])
        return [o, kept, s["k"], s["v"], s["w"]]

    want, graphs = [], []
    for seed in (1, 2):
        torch.manual_seed(seed)
        a = world(seed)
        torch.manual_seed(seed)
        b = world(seed)
        steps = [[t.clone() for t in work(a)] for _ in range(3)]
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            got = work(b)
        want.append(steps)
        graphs.append((g, got, b))  # (a graph reads its inputs where they are)
    for i in range(3):
        for (g, got, _), steps in zip(graphs, want):
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(got, steps[i]):
                assert torch.equal(x, y)
    side = torch.cuda.Stream()
    torch.manual_seed(1)
    c = world(1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work(c)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want[0][0]))
    ops.check_status(0)


@pytest.mark.gpu
def test_outputs_and_workspaces_stay_inside_their_guards():
    from deliverance_b200.ops.beam import beam_select

    ops.set_bounds_check(True)
    try:
        for lens, splits, D, KV, G in (([700, 31, 32, 0], 8, 64, 2, 5), ([64] * 40, 1, 128, 1, 16), ([500], 40, 256, 2, 1)):
            run_attention("cuda", D, KV, G, lens, splits, 0.0, 0)
        run_evict("cuda", [513, 512, 3], 200, 31)
        run_evict("cuda", [9000, 40], 4000, 31, L=1, KV=1, D=8)
        for B, W, V, k in ((1, 1, 7, 7), (2, 3, 4097, 6), (3, 5, 50257, 64)):
            beam_select(torch.randn(B * W, V).cuda(), torch.zeros(B, W).cuda(), k)
        torch.cuda.synchronize()
        ops.check_guards()
    finally:
        ops.set_bounds_check(False)


@pytest.mark.parametrize("device", DEVICES)
def test_evict_length_beyond_the_table(device):
    k, w = torch.zeros(4, 1, P, 8, dtype=BF16, device=device), torch.zeros(3, 1, 64, device=device)
    with pytest.raises((IndexError, RuntimeError)):
        evict_keys([k], [k.clone()], [w], torch.ones(1, 1, dtype=torch.int32, device=device), torch.tensor([40], dtype=torch.int32, device=device), torch.ones(1, dtype=torch.int64, device=device), 8, 2)
        ops.check_status(0)


# ---------------------------------------------------------------------------------------------------------------- engine
def tiny_model(tmp, device="cpu", family="llama", **over):
    from deliverance_b200.ckpt.loader import WeightLoader
    from deliverance_b200.ckpt.tiny import write_tiny_model
    from deliverance_b200.config import load_config
    from deliverance_b200.models.transformer import DecoderModel

    d = str(tmp / f"{family}_{device}")
    write_tiny_model(d, family, seed=5, std=0.25, **over)
    return DecoderModel(load_config(d), device).load(WeightLoader(d))


def engine_of(model, keep=0, recent=8, every=16, capacity=0, pages=256, **kw):
    from deliverance_b200.engine.engine import Engine, EngineConfig
    from deliverance_b200.kv.paged import KvCacheSettings

    kv = KvCacheSettings(keep_tokens=keep, keep_recent=recent, keep_every=every, keep_capacity=capacity)
    e = Engine(model, EngineConfig(num_pages=pages, max_batch_tokens=64, max_seqs=kw.pop("max_seqs", 8), kv=kv, **kw))
    e.eos_ids = frozenset()
    return e


def params_of(n, **kw):
    from deliverance_b200.params import GeneratorParameters

    return GeneratorParameters(max_tokens=n, **kw)


def plain_bounded(model, prompt, steps, keep, recent, every, cap):
    """Greedy decoding on a bounded cache, token by token in fp64: per layer and KV head a list of rows with the keys' weights."""
    c = model.cfg
    H, KV, D = c.num_heads, c.num_kv_heads, c.head_dim
    cos, sin = model.cos.double(), model.sin.double()
    rows = [[[[], [], []] for _ in range(KV)] for _ in model.layers]  # keys, values, weights
    norm = lambda x, w: x * torch.rsqrt(x.pow(2).mean() + c.norm_eps) * w.double()  # noqa: E731

    def rotate(x, pos):
        a, b = x[..., : D // 2], x[..., D // 2 :]
        return torch.cat([a * cos[pos] - b * sin[pos], b * cos[pos] + a * sin[pos]], -1)

    def feed(token, pos, weigh):
        h = model.embed[token].double()
        for i, lw in enumerate(model.layers):
            qkv = lw.qkv.w.double() @ norm(h, lw.input_norm)
            q = rotate(qkv[: H * D].view(KV, H // KV, D), pos)
            k = rotate(qkv[H * D : (H + KV) * D].view(KV, D), pos)
            v = qkv[(H + KV) * D :].view(KV, D)
            out = []
            for j in range(KV):
                ks, vs, ws = rows[i][j]
                ks.append(k[j]), vs.append(v[j]), ws.append(0.0)
                p = torch.softmax(q[j] @ torch.stack(ks).T * c.scale, -1)
                out.append(p @ torch.stack(vs))
                if weigh:
                    for t, x in enumerate(p.sum(0).tolist()[:cap]):
                        ws[t] += x
            h = h + lw.o.w.double() @ torch.stack(out).flatten()
            gu = lw.gate_up.w.double() @ norm(h, lw.pre_ff_norm)
            g, u = gu.chunk(2)
            h = h + lw.down.w.double() @ (torch.nn.functional.silu(g) * u)
        return model.lm_head.w.double() @ norm(h, model.final_norm)

    for pos, token in enumerate(prompt):
        z = feed(token, pos, False)
    tokens, seen, evictions = [int(z.argmax())], 0, 0
    while len(tokens) < steps:
        n = len(rows[0][0][0])
        if n > keep and (seen >= every or n >= cap):
            evictions += 1
            for layer in rows:
                for head in layer:
                    stay = plain_evict([x if t < cap else 0.0 for t, x in enumerate(head[2])], n, keep, recent)
                    head[:] = [[part[t] for t in stay] for part in head]
            seen = 0
        z = feed(tokens[-1], len(prompt) + len(tokens) - 1, True)
        seen += 1
        tokens.append(int(z.argmax()))
    return tokens, evictions


@pytest.mark.parametrize("n,steps,keep,recent,every,cap", [(10, 60, 24, 8, 16, 0), (100, 50, 40, 0, 7, 0), (40, 70, 33, 33, 20, 0), (90, 40, 64, 10, 16, 96), (150, 30, 50, 20, 12, 64), (5, 20, 64, 8, 4, 0)])
def test_engine_bounded_cache_matches_plain(tmp_path, n, steps, keep, recent, every, cap):
    model = tiny_model(tmp_path)
    prompt = [(7 * i * i + 3 * i + 11) % 200 + 3 for i in range(n)]
    want, evictions = plain_bounded(model, prompt, steps, keep, recent, every, cap or 10**6)
    e = engine_of(model, keep, recent, every, cap)
    got = e.generate(prompt, params_of(steps))
    assert got.token_ids == want and e.metrics.get("evictions", 0) == evictions
    e.kv.audit([])
    assert sorted(e.kv.free_weight_slots) == list(range(1, 9))
    if evictions:
        assert want != engine_of(model).generate(prompt, params_of(steps)).token_ids, "nothing that was dropped mattered: the comparison would prove little"


def test_engine_bounded_cache_off_until_needed(tmp_path):
    """Sequences below the limit answer as without one."""
    model = tiny_model(tmp_path)
    prompts = [[(5 * i * i + k) % 200 + 3 for i in range(k + 3)] for k in (0, 30, 61)]
    want = [r.token_ids for r in engine_of(model).generate_batch(prompts, params_of(20))]
    e = engine_of(model, 128)
    assert [r.token_ids for r in e.generate_batch(prompts, params_of(20))] == want and "evictions" not in e.metrics


def run_mixed(e, prompts, steps):
    """Requests that arrive while others run."""
    rs = []
    for i, p in enumerate(prompts):
        rs.append(e.add_request(p, params_of(steps + i)))
        for _ in range(3):
            e.step()
    e.run()
    return [r.output for r in rs]


@pytest.mark.parametrize("lookahead", [False, "force"])
def test_engine_bounded_cache_in_batches(tmp_path, lookahead):
    """Shared prefixes stay what they are; sequences of a batch are shortened each at its time; pages go back."""
    model = tiny_model(tmp_path)
    head = [(3 * i * i + 5) % 200 + 3 for i in range(96)]
    prompts = [head + [k + 3, 2 * k + 9] for k in range(4)] + [head[:40], head]
    alone = [engine_of(model, 48, 16, 10).generate(p, params_of(40 + i)).token_ids for i, p in enumerate(prompts)]
    e = engine_of(model, 48, 16, 10, lookahead=lookahead)
    assert run_mixed(e, prompts, 40) == alone
    e.kv.audit([])
    assert e.metrics["evictions"] > 10 and len(e.kv.free_weight_slots) == 8
    assert run_mixed(e, prompts, 40) == alone  # (cached prefixes still hold what they held)
    e.kv.prefix.clear()
    assert e.kv.allocator.available() == e.kv.num_pages - 1


def test_engine_bounded_cache_under_pressure(tmp_path):
    """A small pool: sequences are preempted and shortened, requests of all kinds still end, nothing is lost."""
    model = tiny_model(tmp_path)
    e = engine_of(model, 40, 8, 5, pages=17)
    rs = [e.add_request([(i * i + 7 * k) % 200 + 3 for i in range(60 + k)], params_of(60)) for k in range(5)]
    e.run()
    assert all(len(r.output) == 60 for r in rs)
    e.kv.audit([])
    assert len(e.kv.free_weight_slots) == 8
    r = e.add_request(list(range(3, 63)), params_of(50))
    for _ in range(5):
        e.step()
    e.reset()
    e.kv.audit([])
    assert len(e.kv.free_weight_slots) == 8 and r.weight_slot == -1


def test_engine_bounded_cache_refusals(tmp_path):
    model = tiny_model(tmp_path)
    for bad in (dict(keep=10, recent=11), dict(keep=10, recent=-1), dict(keep=10, every=0), dict(keep=100, capacity=100)):
        with pytest.raises(ValueError):
            engine_of(model, **bad)
    for family in ("gemma2", "granitemoehybrid"):
        with pytest.raises(ValueError):
            engine_of(tiny_model(tmp_path, family=family), 64)


@pytest.mark.parametrize("device", DEVICES)
def test_engine_beams_on_a_bounded_cache(tmp_path, device):
    """Beam search keeps whole caches; requests before and after it are shortened. Both engines hold the prompt's full page before the compared runs: a prompt
    that starts from cached rows takes other roundings in bf16 than one that is computed in one piece."""
    from deliverance_b200.params import GeneratorParameters

    over = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64) if device == "cuda" else {}
    model = tiny_model(tmp_path, device, "qwen3" if over else "llama", **over)
    prompt = [(7 * i * i + 3 * i + 11) % 200 + 3 for i in range(50)]
    p = GeneratorParameters(max_tokens=30, num_beams=3)
    whole, e = engine_of(model), engine_of(model, 40)
    whole.generate(prompt, params_of(1))
    want = [r.token_ids for r in whole.generate_beams([prompt], p)[0]]
    e.generate(prompt, params_of(1))
    first = e.generate(prompt, params_of(40)).token_ids
    assert [r.token_ids for r in e.generate_beams([prompt], p)[0]] == want
    assert e.generate(prompt, params_of(40)).token_ids == first
    e.kv.audit([])


def test_engine_bounded_cache_and_beams_under_tensor_parallelism(tmp_path):
    """Two ranks as threads: each shortens its own KV heads and takes the same beams; the tokens are those of one rank."""
    import threading

    from deliverance_b200.ckpt.loader import WeightLoader
    from deliverance_b200.ckpt.tiny import write_tiny_model
    from deliverance_b200.config import load_config
    from deliverance_b200.models.transformer import DecoderModel
    from deliverance_b200.parallel.context import InProcessCollectives, InProcessGroup, TensorParallelContext

    d = str(tmp_path / "tp")
    write_tiny_model(d, "llama", seed=5, std=0.25)
    prompt = [(7 * i * i + 3 * i + 11) % 200 + 3 for i in range(50)]

    def run(ctx, out, i):
        try:
            e = engine_of(DecoderModel(load_config(d), "cpu", tp=ctx).load(WeightLoader(d)), 30, 8, 9)
            out[i] = (e.generate(prompt, params_of(40)).token_ids, [r.token_ids for r in e.generate_beams([prompt], params_of(12, num_beams=3))[0]], e.metrics["evictions"])
        except Exception as x:  # noqa: BLE001
            out[i] = x

    single, out, group = [None], [None, None], InProcessGroup(2, timeout=60)
    run(TensorParallelContext(), single, 0)
    ts = [threading.Thread(target=run, args=(TensorParallelContext(r, 2, InProcessCollectives(group, r)), out, r)) for r in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not isinstance(out[0], Exception), out[0]
    assert out[0] == out[1] == single[0] and single[0][2] > 2


@pytest.mark.gpu
@pytest.mark.parametrize("D,KV", [(64, 2), (128, 1)])
def test_engine_bounded_cache_on_the_gpu(tmp_path, D, KV):
    """Captured steps one step ahead, captured steps and plain launches give the same tokens; the pool stays small."""
    model = tiny_model(tmp_path, "cuda", "qwen3", hidden_size=256, num_attention_heads=4, num_key_value_heads=KV, head_dim=D, vocab_size=512)
    head = [(3 * i * i + 5) % 200 + 3 for i in range(96)]
    prompts = [head + [k + 3, 2 * k + 9] for k in range(4)] + [head[:40], head]
    outs = []
    for kw in (dict(), dict(lookahead=False), dict(cuda_graphs=False)):
        e = engine_of(model, 48, 16, 10, **kw)
        outs.append(run_mixed(e, prompts, 60))
        ops.check_status(0)
        e.kv.audit([])
        assert e.metrics["evictions"] > 10
    # (batches of other sizes run other kernels, whose roundings differ: the schedules here are the same but for the step that lookahead settles late)
    assert outs[1] == outs[2]
    assert sum(a == b for x, y in zip(outs[0], outs[1]) for a, b in zip(x, y)) >= 0.5 * sum(map(len, outs[1]))


def shared_head(lens, head=64):
    """Prompts that begin alike."""
    h = [(3 * i * i + 5) % 200 + 3 for i in range(head)]
    return [h + [(7 * i + 11 * k) % 200 + 3 for i in range(n - head)] for k, n in enumerate(lens)]


@pytest.mark.parametrize("lookahead", [False, "force"])
@pytest.mark.parametrize("lens,keep,every,pages,steps", [([92, 84, 81], 83, 8, 8, 60), ([80, 68, 85], 92, 11, 7, 120), ([75, 81, 86], 86, 10, 7, 40), ([66, 95, 95, 70], 64, 3, 9, 40)])
def test_engine_bounded_cache_replaces_shared_pages_in_a_small_pool(tmp_path, lens, keep, every, pages, steps, lookahead):
    """The pages that replace shared ones come out of the pool that the step's new rows need too: both are counted before the step, and younger sequences make room."""
    model = tiny_model(tmp_path)
    e = engine_of(model, keep, 8, every, pages=pages, lookahead=lookahead)
    rs = [e.add_request(p, params_of(steps)) for p in shared_head(lens)]
    e.run()
    assert [(len(r.output), r.error) for r in rs] == [(steps, None)] * len(rs)
    e.kv.audit([])
    assert e.metrics["evictions"] > 2 and len(e.kv.free_weight_slots) == 8


def test_engine_bounded_cache_one_sequence_fills_the_pool(tmp_path):
    """Shared with nothing but cached prefixes, in a pool that its rows fill: cached prefixes give way."""
    model = tiny_model(tmp_path)
    for lookahead in (False, "force"):
        e = engine_of(model, 90, 8, 6, pages=4, lookahead=lookahead)  # three pages for 90 to 96 rows
        prompt = shared_head([80])[0]
        first = e.generate(prompt, params_of(60))
        assert len(first.token_ids) == 60 and e.metrics["evictions"] > 5
        e.kv.audit([])
        assert e.generate(prompt, params_of(60)).token_ids == first.token_ids
        assert first.token_ids == engine_of(model, 90, 8, 6).generate(prompt, params_of(60)).token_ids


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("at", [2, 23, 60, 61, 66])
def test_engine_bounded_cache_preempted_and_resumed(tmp_path, device, at):
    """A preempted sequence goes on as if nothing had happened: what was weighed and dropped cannot be rebuilt from its tokens. Where decoding fits, resuming fits."""
    over = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64) if device == "cuda" else {}
    model = tiny_model(tmp_path, device, "qwen3" if over else "llama", **over)
    prompt = shared_head([60])[0]
    lookahead = True if device == "cuda" else "force"
    for la, pages in ((False, 256), (lookahead, 256), (False, 4), (lookahead, 4)):
        alone = engine_of(model, 40, 8, 5, lookahead=la).generate(prompt, params_of(120)).token_ids
        e = engine_of(model, 40, 8, 5, lookahead=la, pages=pages)
        r = e.add_request(prompt, params_of(120))
        while len(r.output) < at:
            e.step()
        e._drain()
        e._preempt(r)
        assert not r.pages and r.weight_slot == -1
        e.kv._weights.fill_(7.0), [t.fill_(3.0) for t in e.kv.k + e.kv.v]
        e.kv.prefix.clear()
        e.run()
        assert r.output == alone and r.error is None and r.saved is None
        e.kv.audit([])
        r = e.add_request(prompt, params_of(120))
        while len(r.output) < at:
            e.step()
        e._drain()
        e._preempt(r)
        e.abort(r)
        assert r.saved is None and len(e.kv.free_weight_slots) == 8
        e.run()


def pressed(seed):
    import random

    rng = random.Random(seed)
    lens = [rng.choice([64, 96]) + rng.randint(1, 40) for _ in range(rng.randint(2, 4))]
    every, steps = rng.randint(3, 16), rng.randint(30, 80)
    keep = rng.randint(33, 100)
    recent = rng.randint(0, keep)
    # a sequence holds what its prompt and its first steps make or what it keeps and is weighed on, and a page more
    pages = 2 + max(-(-(max(max(lens), keep) + every + 1) // P) + 1, -(-(max(lens) + 1) // P) + 1) + rng.randint(0, 4)
    return shared_head(lens), keep, recent, every, steps, pages, rng.choice([False, "force"]), rng.choice([0, 0, 2])


@pytest.mark.parametrize("seed", range(24))
def test_engine_bounded_cache_answers_do_not_depend_on_the_pool(tmp_path, seed):
    prompts, keep, recent, every, steps, pages, lookahead, interleave = pressed(seed)
    model = tiny_model(tmp_path)
    alone = [engine_of(model, keep, recent, every).generate(p, params_of(steps)).token_ids for p in prompts]
    e = engine_of(model, keep, recent, every, pages=pages, lookahead=lookahead, decode_interleave=interleave)
    rs = [e.add_request(p, params_of(steps)) for p in prompts]
    e.run()
    assert [r.error for r in rs] == [None] * len(rs) and [r.output for r in rs] == alone
    e.kv.audit([])
    assert len(e.kv.free_weight_slots) == 8


def test_engine_bounded_cache_knows_unlike_lengths(tmp_path):
    """A captured step of a bounded cache is one for unlike lengths where weighted attention is launched otherwise for them, which is also where plain attention is not."""
    from deliverance_b200.ops.evict import by_length

    model = tiny_model(tmp_path)
    e, plain = engine_of(model, 64), engine_of(model)
    ragged = lambda n: [1000] * (n - 1) + [30000]  # noqa: E731
    seen = set()
    for B in (1, 2, 4, 8, 16, 32, 64, 128):
        room, splits = ops.decode_room(B, model.n_heads, model.n_kv, model.cfg.head_dim), e._splits(B)
        matters = by_length(splits, B, model.n_heads, model.n_kv, model.cfg.head_dim)
        assert e._even([700] * B) and (B < 4 or e._even(ragged(B)) == (not matters))
        assert matters == (room <= 32 or splits > room) and (B < 4 or plain._even(ragged(B)) == (splits <= room))
        seen.add((matters, splits <= room))
    assert (True, True) in seen and (False, True) in seen


@pytest.mark.gpu
def test_engine_bounded_cache_captures_unlike_lengths(tmp_path):
    """Sixteen sequences, one much longer: the step of that bucket is launched by a plan, and answers as plain launches do."""
    from deliverance_b200.ops.evict import by_length

    model = tiny_model(tmp_path, "cuda", "qwen3", hidden_size=256, num_attention_heads=8, num_key_value_heads=4, head_dim=64, vocab_size=512)
    assert by_length(9, 16, 8, 4, 64)
    prompts = [shared_head([40 + k])[0] for k in range(15)] + shared_head([215])
    outs = []
    for kw in (dict(lookahead=False), dict(cuda_graphs=False)):
        e = engine_of(model, 200, 16, 10, max_seqs=16, **kw)
        outs.append([r.token_ids for r in e.generate_batch(prompts, params_of(30))])
        ops.check_status(0)
    assert outs[0] == outs[1] and e.metrics["evictions"] > 1
    e = engine_of(model, 200, 16, 10, max_seqs=16)
    e.generate_batch(prompts, params_of(30))
    assert -16 in e._graphs


@pytest.mark.gpu
def test_weighted_attention_on_a_given_workspace():
    """Scores in a workspace of the caller's, used by one call after another: the same bits as with the call's own; one that is too small is refused."""
    from deliverance_b200.ops.evict import score_room

    table, pages = tables_for([700, 33, 500], extra=3)
    k, v = torch.randn(pages, 2, P, 64).to(BF16).cuda(), torch.randn(pages, 2, P, 64).to(BF16).cuda()
    ctx, slots, table = torch.tensor([700, 33, 500], dtype=torch.int32).cuda(), torch.tensor([3, 1, 2]).cuda(), table.cuda()
    room = score_room(3, 8, table.shape[1] * P, 650)
    assert room == 3 * 8 * 656
    scores = torch.full((room + 64,), math.nan, device="cuda")
    a, b = torch.rand(4, 2, 650).cuda(), None
    b = a.clone()
    for splits in (1, 6, 3):
        q = torch.randn(3, 512).to(BF16).cuda()
        x = decode_attention_weighted(q, k, v, table, ctx, 8, 0.125, a, slots, splits=splits)
        y = decode_attention_weighted(q, k, v, table, ctx, 8, 0.125, b, slots, splits=splits, scores=scores)
        assert torch.equal(x, y) and torch.equal(a, b) and scores[room:].isnan().all()
    for bad in (scores[: room - 1], scores.half(), scores.cpu(), scores[1:]):
        with pytest.raises(RuntimeError):
            decode_attention_weighted(q, k, v, table, ctx, 8, 0.125, b, slots, scores=bad)
    ops.check_status(0)


@pytest.mark.gpu
def test_engine_bounded_cache_keeps_one_workspace(tmp_path):
    """Steps captured for several batch sizes, of like and unlike lengths, over a context of 131,072: one workspace of 268 MB for all of them, allocated with the cache."""
    model = tiny_model(tmp_path, "cuda", "qwen3", hidden_size=256, num_attention_heads=8, num_key_value_heads=4, head_dim=64, vocab_size=512, max_position_embeddings=131072)
    e = engine_of(model, 200, 16, 10, max_seqs=64, capacity=131072)
    assert e.kv.key_scores.numel() * 4 == 64 * 8 * 131072 * 4
    torch.cuda.synchronize()
    before = torch.cuda.memory_reserved()
    e.generate_batch([shared_head([40 + k % 8])[0] for k in range(60)] + shared_head([400]), params_of(12))
    e.generate_batch([shared_head([40 + k])[0] for k in range(30)], params_of(4))
    assert {64, 32} <= {abs(b) for b in e._graphs}
    torch.cuda.synchronize()
    # (what the steps keep for themselves: activations, split outputs, block tables of 4,096 pages per row)
    assert torch.cuda.memory_reserved() - before < 200 << 20


@pytest.mark.gpu
def test_weights_of_more_rows_than_an_int_counts_are_refused():
    k = torch.zeros(2, 1, P, 64, dtype=BF16, device="cuda")
    w = torch.empty(1, 1, 2**31, device="cuda")  # (never touched)
    with pytest.raises(RuntimeError, match="out of range"):
        decode_attention_weighted(torch.zeros(1, 64, dtype=BF16, device="cuda"), k, k.clone(), torch.ones(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda"), 1, 0.1, w,
                                  torch.zeros(1, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,KV,G", [(64, 2, 4), (128, 2, 4), (256, 1, 2), (64, 1, 16)])
@pytest.mark.parametrize("lens,splits,even,extra", [([3001, 2, 700], 32, False, 1), ([9000], 30, True, 1), ([4001, 4000], 18, True, 60), ([40, 2500, 300], 1, False, 1), ([9000, 31, 5], 32, False, 200)])
def test_weighted_attention_outputs_value_by_value(device, D, KV, G, lens, splits, even, extra):
    """Long sequences of like keys have outputs far smaller than their values, so each output is held to its own sum of p |v|. A probability is rounded to bf16 (2^-8 of it) and is off by
    what its score is (as a weight is, numerator and denominator: twice), the result is rounded once more (2^-8 of it); sums in fp32 add n * 2^-24 of the sum of magnitudes."""
    if device == "cpu" and sum(lens) * KV * G * D > 3e7:
        pytest.skip("large for the CPU")
    B, H, n = len(lens), KV * G, max(lens)
    table, pages = tables_for(lens, extra=extra)
    q, k, v = torch.randn(B, H * D).to(BF16), torch.randn(pages, KV, P, D).to(BF16), torch.randn(pages, KV, P, D).to(BF16)
    to = lambda t: t.to(device)  # noqa: E731
    ctx = torch.tensor(lens, dtype=torch.int32)
    out = decode_attention_weighted(to(q), to(k), to(v), to(table), to(ctx), H, D**-0.5, torch.zeros(B + 1, KV, n, device=device), to(torch.arange(1, B + 1)), 0.0, 0, splits, even).cpu().double()
    want, _ = plain_attention(q, k, v, table, lens, KV, D**-0.5, 0.0, 0)
    size, _ = plain_attention(q, k, v.abs(), table, lens, KV, D**-0.5, 0.0, 0)
    # (D + 2 roundings of a score, each 2^-24 of the sum of its magnitudes at most; the exponential as in run_attention)
    heads = k.abs().float().permute(1, 0, 2, 3).reshape(KV, -1, D).transpose(1, 2)
    score = float((q.abs().float().view(B, KV, G, D).permute(1, 0, 2, 3).reshape(KV, -1, D) @ heads).max()) * D**-0.5 * (D + 2) * 2**-24 + 64 * 2**-23
    bound = (2**-8 + 2 * score + 2 * n * 2**-24) * size + 2**-8 * want.abs()
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() / bound).max())
    long = lens.index(n)
    assert bound[long].mean() < 0.4 * want[long].abs().mean()  # (an output of zeros is found)


def bounded_logits(model, prompt, tokens, recorded, keep, recent, every, rounded=False):
    """64-bit decoding of given tokens on a bounded cache that keeps, at its own times, the rows that were recorded ([layers, KV, keep] each); "own": those that its weights say, None: all.
    Returns the logits after the prompt and after every token, the rows kept and, for each eviction, what their old rows weigh, as a part of what the heaviest ones would. ``model``: of the CPU,
    its weights rounded to bf16 as the GPU's are. ``rounded``: every vector between two products is rounded to bf16 as well."""
    c = model.cfg
    H, KV, D = c.num_heads, c.num_kv_heads, c.head_dim
    w16 = lambda t: t.to(BF16).double()  # noqa: E731
    r16 = w16 if rounded else lambda t: t
    cos, sin = model.cos.double(), model.sin.double()
    layers = [(w16(lw.qkv.w), w16(lw.o.w), w16(lw.gate_up.w), w16(lw.down.w), w16(lw.input_norm), w16(lw.pre_ff_norm)) for lw in model.layers]
    rows = [[[torch.zeros(0, D, dtype=torch.float64), torch.zeros(0, D, dtype=torch.float64), torch.zeros(0, dtype=torch.float64)] for _ in range(KV)] for _ in layers]
    norm = lambda x, w: r16(x * torch.rsqrt(x.pow(2).mean() + c.norm_eps) * w)  # noqa: E731
    embed, head, last = w16(model.embed), w16(model.lm_head.w), w16(model.final_norm)

    def rotate(x, pos):
        a, b = x[..., : D // 2], x[..., D // 2 :]
        return r16(torch.cat([a * cos[pos] - b * sin[pos], b * cos[pos] + a * sin[pos]], -1))

    def feed(token, pos, weigh):
        h = embed[token]
        for i, (qkv_w, o_w, gu_w, down_w, n1, n2) in enumerate(layers):
            qkv = r16(qkv_w @ norm(h, n1))
            q, k, v = rotate(qkv[: H * D].view(KV, H // KV, D), pos), rotate(qkv[H * D : (H + KV) * D].view(KV, D), pos), qkv[(H + KV) * D :].view(KV, D)
            out = []
            for j in range(KV):
                r = rows[i][j]
                r[0], r[1], r[2] = torch.cat([r[0], k[j : j + 1]]), torch.cat([r[1], v[j : j + 1]]), torch.cat([r[2], torch.zeros(1, dtype=torch.float64)])
                p = torch.softmax(q[j] @ r[0].T * c.scale, -1)
                out.append(r16(r16(p) @ r[1]))
                if weigh:
                    r[2] += p.sum(0)
            h = r16(h + r16(o_w @ torch.stack(out).flatten()))
            g, u = r16(gu_w @ norm(h, n2)).chunk(2)
            h = r16(h + r16(down_w @ r16(torch.nn.functional.silu(g) * u)))
        return head @ norm(h, last)

    for pos, token in enumerate(prompt):
        z = feed(token, pos, False)
    logits, parts, kept, seen = [z], [], [], 0
    for i, token in enumerate(tokens):
        n = rows[0][0][0].shape[0]
        if recorded is not None and n > keep and seen >= every:
            best = [[plain_evict(r[2].tolist(), n, keep, recent) for r in layer] for layer in rows]
            kept.append(best if recorded == "own" else recorded[len(kept)].tolist())
            part = 1.0
            for layer, mine, heaviest in zip(rows, kept[-1], best):
                for r, stay, most in zip(layer, mine, heaviest):
                    assert len(stay) == keep and sorted(set(stay)) == stay and stay[keep - recent :] == list(range(n - recent, n))
                    part = min(part, float(r[2][stay[: keep - recent]].sum() / r[2][most[: keep - recent]].sum()))
                    r[:] = [x[stay] for x in r]
            parts.append(part)
            seen = 0
        logits.append(feed(token, len(prompt) + i, True))
        seen += 1
    return torch.stack(logits), [torch.tensor(x) for x in kept], parts


def away(a, b):
    return ((a - b).norm(dim=1) / b.norm(dim=1)).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("H,KV", [(4, 2), (4, 4), (2, 1)])
@pytest.mark.parametrize("lookahead", [False, True])
def test_engine_bounded_cache_logits_against_64_bits(tmp_path, monkeypatch, H, KV, lookahead):
    """The logits of every decode step on the GPU against a 64-bit decoder that is fed the same tokens and drops the same rows, which are held to be the heaviest by its own weights. How far
    roundings to bf16 carry is computed, not guessed: the same decoder with every vector between two products rounded, dropping what its own weights say, against the exact one that drops
    the same. The GPU rounds in other places of the same kind: three times that is allowed. What is kept weighs 95 % of the heaviest rows at least: the rounded decoder loses 0 to 1.5 % here,
    keeping the oldest rows instead 28 to 56 % in the worst eviction."""
    from deliverance_b200.engine import engine as module

    over = dict(hidden_size=256, num_attention_heads=H, num_key_value_heads=KV, vocab_size=512)
    gpu, cpu = tiny_model(tmp_path, "cuda", **over), tiny_model(tmp_path, "cpu", **over)
    keep, recent, every, steps = 48, 16, 10, 70
    e = engine_of(gpu, keep, recent, every, lookahead=lookahead)
    recorded, seen = [], []
    evict, greedy = module.evict_keys, e._greedy

    def record_evict(*a):
        got = evict(*a)
        recorded.append(got[0][:, 0].cpu())
        return got

    def record_logits(z):
        seen.append(z.float().cpu().double())
        return greedy(z)

    monkeypatch.setattr(module, "evict_keys", record_evict)
    e._greedy = record_logits
    prompt = [(7 * i * i + 3 * i + 11) % 200 + 3 for i in range(40)]
    tokens = e.generate(prompt, params_of(steps)).token_ids
    got = torch.cat(seen)[:steps]  # (a step ahead of the last token computes one more)
    run = lambda rows, **kw: bounded_logits(cpu, prompt, tokens[:-1], rows, keep, recent, every, **kw)  # noqa: E731
    want, kept, parts = run(recorded)
    assert len(kept) == len(recorded) >= 5
    bits16, own, _ = run("own", rounded=True)
    exact, _, own_parts = run(own)
    noise = away(bits16, exact)
    assert away(got, want) <= 3 * noise, (away(got, want), noise)
    assert min(parts) >= 0.95 and min(own_parts) >= 0.95, (parts, own_parts)
    whole, _, _ = run(None)
    assert away(whole, want) > 3 * noise  # (what was dropped shows)


def test_engine_bounded_cache_padding_is_not_unlike(tmp_path):
    """Like sequences in a bucket that is not full take the step for like ones, where the split is by number in both; an unlike one among them does not."""
    from deliverance_b200.ops.evict import by_length

    model = tiny_model(tmp_path)
    e, seen = engine_of(model, 64), 0
    for B in (8, 16, 32, 64):
        room, splits = ops.decode_room(B, model.n_heads, model.n_kv, model.cfg.head_dim), e._splits(B)
        if splits <= room and by_length(splits, B, model.n_heads, model.n_kv, model.cfg.head_dim):
            n, seen = B // 2 + 1, seen + 1
            assert e._even([700] * n + [1] * (B - n)) and not e._even([700] * (n - 1) + [20000] + [1] * (B - n))
    assert seen
