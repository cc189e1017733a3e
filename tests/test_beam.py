"""Beam search operators against plain statements in 64 bits, and beam search through the engine. On the CPU and, on a GPU box, on the CUDA kernels."""
import math

import pytest
import torch

from deliverance_b200 import ops
from deliverance_b200.ops.beam import MAX_BEAMS, MAX_CANDIDATES, beam_reorder, beam_select

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16 = torch.float32, torch.bfloat16
INF = math.inf


def pack(bits):
    rows, V = bits.shape
    words = -(-V // 32)
    b = torch.nn.functional.pad(bits, (0, words * 32 - V)).view(rows, words, 32).to(torch.int64)
    p = (b << torch.arange(32)).sum(-1)
    return torch.where(p >= 1 << 31, p - (1 << 32), p).to(torch.int32)


def plain_values(logits, scores, bits=None, softcap=0.0, inv_scale=1.0):
    """fp64 [B, W * V]: the value of every candidate, -inf where there is none."""
    B, W = scores.shape
    out = []
    for r, row in enumerate(logits.double()):
        z = row * inv_scale
        z = softcap * torch.tanh(z / softcap) if softcap else z
        z = torch.where(row == -INF, -INF, z)
        if bits is not None:
            z = torch.where(bits[r], z, -INF)
        s = float(scores[r // W, r % W])
        if not math.isfinite(s) or z.isnan().any() or (z == INF).any() or (z == -INF).all():
            out.append(torch.full_like(z, -INF))
        else:
            m = z.max()
            out.append(s + (z - m) - (z - m).exp().sum().log())
    return torch.stack(out).view(B, -1)


def check(got, values, V, tol):
    """Each returned candidate has the value that belongs to its place, and where neighbours are further apart than the tolerance it is that very candidate."""
    got = [t.cpu() for t in got]
    k = got[0].shape[1]
    want, at = torch.sort(values, dim=-1, descending=True, stable=True)
    for b in range(values.shape[0]):
        n = int((want[b, :k] > -INF).sum())
        assert (got[1][b, n:] == -1).all() and (got[2][b, n:] == -1).all() and (got[0][b, n:] == -INF).all()
        flat = got[1][b, :n] * V + got[2][b, :n]
        assert (got[2][b, :n] >= 0).all() and (got[2][b, :n] < V).all() and len(set(flat.tolist())) == n
        for j in range(n):
            w = float(want[b, j])
            assert abs(float(got[0][b, j]) - w) <= tol + abs(w) * 2**-24, (b, j)
            assert abs(float(values[b, flat[j]]) - w) <= 2 * tol
            apart = (j == 0 or want[b, j - 1] - w > 2 * tol) and (j + 1 >= want.shape[1] or w - want[b, j + 1] > 2 * tol)
            if apart:
                assert int(flat[j]) == int(at[b, j])


# The logarithm of the sum of exponentials. A term exp(d), d = logit - maximum, is off by 2^-24 |d| (difference), 2^-23 |d| (product with log2 e and that constant) and
# 2^-22 (base-two exponential), relative; weighted with the probabilities, |d| is at most the logarithm of V (13), so 2^-22 + 13 * 1.5 * 2^-23. Up to 16 additions in fp32
# and three factors expf (2^-23 each); the rest is in 64 bits.
LSE = 2**-22 + 19.5 * 2**-23 + 16 * 2**-24 + 3 * 2**-23


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,W,V,k", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 33, 6), (1, 4, 4095, 8), (3, 2, 4096, 64), (1, 32, 4097, 64), (5, 5, 12289, 10), (2, 4, 50257, 8), (1, 16, 151936, 32)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_matches_plain(device, B, W, V, k, dtype):
    logits = (torch.randn(B * W, V) * 4).to(dtype)
    scores = -torch.rand(B, W) * 5
    got = beam_select(logits.to(device), scores.to(device), k)
    assert got[0].dtype == F32 and got[1].dtype == torch.int64 and got[2].dtype == torch.int64
    check(got, plain_values(logits, scores), V, LSE)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 2), (0, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_rows_on_any_address(device, offset, pad, dtype):
    """Rows of a wider buffer that start on any element; what lies around them is larger than every logit."""
    B, W, V, k = 2, 3, 5003, 6
    logits = (torch.randn(B * W, V) * 3).to(dtype)
    scores = -torch.rand(B, W)
    wide = torch.full((B * W * (V + pad) + 16,), 1e4, dtype=dtype, device=device)
    view = wide[offset : offset + B * W * (V + pad)].view(B * W, V + pad)[:, :V]
    view.copy_(logits)
    check(beam_select(view, scores.to(device), k), plain_values(logits, scores), V, LSE)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("softcap,inv_scale", [(30.0, 1.0), (0.0, 0.125), (5.0, 2.0)])
def test_select_softcap_scale_mask(device, softcap, inv_scale):
    B, W, V, k = 2, 4, 3001, 8
    logits, scores = torch.randn(B * W, V) * 6, -torch.rand(B, W)
    bits = torch.rand(B * W, V) < 0.1
    bits[1] = False  # a beam at a dead end
    bits[2] = False
    bits[2, 2999] = True
    logits[3, ::2] = -INF
    tol = LSE + softcap * 2**-20  # (a quotient, tanhf and a product, 4 * 2^-23 each way of at most softcap)
    got = beam_select(logits.to(device), scores.to(device), k, pack(bits).to(device), softcap, inv_scale)
    check(got, plain_values(logits, scores, bits, softcap, inv_scale), V, tol)


@pytest.mark.parametrize("device", DEVICES)
def test_select_ties_go_to_the_lowest(device):
    """Beams with the same row and score, rows of one value, long runs of the maximum: order of beam, then token."""
    row = torch.randint(-2, 3, (9001,)).float()
    for rows in (torch.zeros(3, 9001), row.expand(3, -1).contiguous(), torch.full((3, 20000), -7.5)):
        V = rows.shape[1]
        v, p, t = (x.cpu() for x in beam_select(rows.to(device), torch.zeros(1, 3).to(device), 64))
        want = torch.sort(rows.flatten(), descending=True, stable=True).indices[:64]
        assert torch.equal(p[0] * V + t[0], want)
        assert (v[0, 1:] <= v[0, :-1]).all()
    zeros = torch.tensor([[-1.0, -0.0, 0.0, -0.0, 0.0]])  # equal
    assert beam_select(zeros.to(device), torch.zeros(1, 1).to(device), 4)[2][0].tolist() == [1, 2, 3, 4]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_select_sorted_rows(device, order):
    """Every tile of a rising row beats all before it, and within one the best lie side by side."""
    V = 40000
    row = torch.arange(V).float() * 1e-3
    rows = torch.stack([row, row + 5]) if order == "rising" else torch.stack([row, row]).flip(1)
    scores = torch.tensor([[-1.0, -1.5]])
    check(beam_select(rows.to(device), scores.to(device), 64), plain_values(rows, scores), V, LSE)


@pytest.mark.parametrize("device", DEVICES)
def test_select_without_candidates(device):
    """Dead beams, empty masks, NaN, infinities, and logits of the type's lowest value."""
    V, low = 1000, torch.finfo(F32).min
    logits = torch.randn(8, V)
    logits[0] = -INF
    logits[1, 500] = math.nan
    logits[2, 3] = INF
    logits[4] = low  # uniform
    logits[5] = low
    logits[5, 7] = 2.0  # certain
    scores = torch.tensor([[-1.0, -1.0], [-1.0, -2.0], [-1.0, -3.0], [-INF, math.nan]])
    got = [t.cpu() for t in beam_select(logits.to(device), scores.to(device), 8)]
    assert (got[2][0] == -1).all() and (got[0][0] == -INF).all() and (got[1][3] == -1).all()
    assert (got[1][1] == 1).all()
    assert got[1][2].tolist()[0] == 1 and got[2][2].tolist()[0] == 7 and float(got[0][2, 0]) == -3.0
    assert got[1][2].tolist()[1:] == [0] * 7 and got[2][2].tolist()[1:] == list(range(7))
    assert abs(float(got[0][2, 1]) - (-1 - math.log(V))) < 1e-5
    empty = beam_select(logits[:0].to(device), torch.zeros(0, 3).to(device), 2)
    assert [tuple(t.shape) for t in empty] == [(0, 2)] * 3


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 7, 100])
def test_select_split_count_changes_nothing(splits):
    logits, scores = torch.randn(6, 30011).cuda() * 3, -torch.rand(2, 3).cuda()
    one = ops.require_ext().beam_select(logits, scores, 12, splits=splits)
    two = beam_select(logits, scores, 12)
    assert torch.equal(one[1], two[1]) and torch.equal(one[2], two[2]) and float((one[0] - two[0]).abs().max()) <= 2 * LSE + 2**-20


@pytest.mark.gpu
def test_select_in_graphs_and_streams():
    """Two captured graphs replayed in turn, and a call on another stream, give what a call of their own gives."""
    outs, graphs, inputs = [], [], []
    for seed in (1, 2):
        x = torch.randn(8, 20000, generator=torch.Generator().manual_seed(seed)).cuda()
        s = -torch.rand(2, 4, generator=torch.Generator().manual_seed(seed)).cuda()
        beam_select(x, s, 8)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(beam_select(x, s, 8))
        graphs.append(g)
        inputs.append((x, s))
    for _ in range(3):
        for g in graphs:
            g.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [beam_select(x, s, 8) for x, s in inputs]
    torch.cuda.synchronize()
    for o, p, (x, s) in zip(outs, other, inputs):
        for a, b, c in zip(o, p, beam_select(x, s, 8)):
            assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.parametrize("device", DEVICES)
def test_select_refusals(device):
    x, s = torch.randn(6, 10).to(device), torch.zeros(2, 3).to(device)
    for bad in (lambda: beam_select(x[:5], s, 4), lambda: beam_select(x, s, 0), lambda: beam_select(x, s, 31), lambda: beam_select(x, s, MAX_CANDIDATES + 1),
                lambda: beam_select(torch.randn(2 * (MAX_BEAMS + 1), 10).to(device), torch.zeros(2, MAX_BEAMS + 1).to(device), 4), lambda: beam_select(x, s.flatten(), 4),
                lambda: beam_select(x, s, 4, inv_scale=0.0), lambda: beam_select(x, s, 4, softcap=-1.0)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    if device == "cuda":
        for bad in (lambda: beam_select(x.half(), s, 4), lambda: beam_select(x, s.double(), 4), lambda: beam_select(x, s.cpu(), 4), lambda: beam_select(x.t().contiguous().t(), s, 4),
                    lambda: beam_select(x, s, 4, torch.zeros(6, 1, dtype=torch.int64, device=device)), lambda: beam_select(x, s, 4, torch.zeros(5, 1, dtype=torch.int32, device=device))):
            with pytest.raises(RuntimeError):
                bad()


# ---------------------------------------------------------------------------------------------------------------- reordering
def plain_reorder(t, index, parents, rows=None):
    new = t.clone()
    for b in range(parents.shape[0]):
        for j in range(parents.shape[1]):
            p = int(parents[b, j])
            if 0 <= p < parents.shape[1]:
                d, s = int(index[b, j]), int(index[b, p])
                if rows is None:
                    new[d] = t[s]
                else:
                    new[d, :, : int(rows[b])] = t[s, :, : int(rows[b])]
    return new


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,W", [(1, 1), (1, 2), (3, 4), (2, 5), (1, 8), (4, 11), (2, 32)])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F32), (6, BF16), (5, F32), (3, BF16)])
def test_reorder_matches_plain(device, B, W, D, dtype):
    n = B * W + 3
    caches = [torch.randn(n, kv, 32, D).to(dtype) for kv in (1, 3)]
    states = [torch.randn(n, 3, D).to(dtype), torch.randn(n, 700, D).to(dtype)]
    pages = (torch.randperm(n - 1)[: B * W] + 1).view(B, W)
    slots = (torch.randperm(n - 1)[: B * W] + 1).view(B, W)
    parents = torch.randint(-1, W, (B, W))
    rows = torch.randint(0, 33, (B,)).to(torch.int32)
    rows[0] = 17
    mine = [t.clone().to(device) for t in caches], [t.clone().to(device) for t in states]
    to = lambda t: t.to(device)  # noqa: E731
    beam_reorder(to(parents), mine[1] + [mine[1][0]], to(slots), mine[0] + [None], to(pages), to(rows))
    for got, t in zip(mine[0], caches):
        assert torch.equal(got.cpu(), plain_reorder(t, pages, parents, rows))
    for got, t in zip(mine[1], states):
        assert torch.equal(got.cpu(), plain_reorder(t, slots, parents))
    beam_reorder(to(parents), caches=mine[0], pages=to(pages))  # whole pages
    for got, t in zip(mine[0], caches):
        assert torch.equal(got.cpu(), plain_reorder(plain_reorder(t, pages, parents, rows), pages, parents))


@pytest.mark.parametrize("device", DEVICES)
def test_reorder_many_layers(device):
    """More tensors than one launch takes, of different widths."""
    shapes = [(9, 2, 32, 64 if i % 3 else 128) for i in range(130)]
    caches = [torch.randn(s).to(BF16) for s in shapes]
    pages, parents, rows = torch.tensor([[3, 1, 7, 5], [2, 8, 4, 6]]), torch.tensor([[1, 0, 3, 3], [2, 2, 0, 9]]), torch.tensor([31, 1], dtype=torch.int32)
    got = [t.clone().to(device) for t in caches]
    beam_reorder(parents.to(device), caches=got, pages=pages.to(device), rows=rows.to(device))
    for a, t in zip(got, caches):
        assert torch.equal(a.cpu(), plain_reorder(t, pages, parents, rows))


@pytest.mark.parametrize("device", DEVICES)
def test_reorder_refusals(device):
    t, i = torch.zeros(4, 2, 32, 8, device=device), torch.zeros(1, 2, dtype=torch.int64, device=device)
    for bad in (lambda: beam_reorder(i, [t]), lambda: beam_reorder(i, [t], i.int()), lambda: beam_reorder(i.flatten(), [t], i.flatten()), lambda: beam_reorder(i, caches=[t[0]], pages=i),
                lambda: beam_reorder(i, caches=[t], pages=i, rows=torch.zeros(2, dtype=torch.int32, device=device)),
                lambda: beam_reorder(torch.zeros(1, 33, dtype=torch.int64, device=device), [t], torch.zeros(1, 33, dtype=torch.int64, device=device))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    with pytest.raises((IndexError, RuntimeError)):  # a slot outside: left out, and reported
        beam_reorder(torch.tensor([[1, 0]], device=device), [t], torch.tensor([[1, 4]], device=device))
        ops.check_status(0)
