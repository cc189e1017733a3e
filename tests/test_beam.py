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


@pytest.mark.gpu
def test_select_ties_over_many_groups():
    """One value everywhere, in more groups than are listed; the same with a masked start; two beams of which the second is behind."""
    for W, V, dtype in ((8, 20000, F32), (5, 60001, BF16)):
        rows = torch.full((W, V), 3.25, dtype=dtype).cuda()
        _, p, t = (x.cpu() for x in beam_select(rows, torch.zeros(1, W).cuda(), 64))
        assert (p == 0).all() and t[0].tolist() == list(range(64))
        bits = torch.ones(W, V, dtype=torch.bool)
        bits[0] = False
        bits[1, : V - 10] = False
        _, p, t = (x.cpu() for x in beam_select(rows, torch.tensor([[0.0, -12.0] + [-1.0] * (W - 2)]).cuda(), 64, pack(bits).cuda()))
        # ten tokens of the second beam at a tenth each beat V of the others only if -12 - log 10 > -1 - log V, which it does not
        assert (p == 2).all() and t[0].tolist() == list(range(64))


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


# ---------------------------------------------------------------------------------------------------------------- engine
def tiny_model(tmp, family, device="cpu", **over):
    from deliverance_b200.ckpt.loader import WeightLoader
    from deliverance_b200.ckpt.tiny import write_tiny_model
    from deliverance_b200.config import load_config
    from deliverance_b200.models.transformer import DecoderModel

    d = str(tmp / family)
    write_tiny_model(d, family, seed=11, std=over.pop("std", 0.2), **over)
    cfg = load_config(d)
    if family == "fopivik":
        from deliverance_b200.models.fopivik import FopivikModel as Model
    elif family == "gevovik":
        from deliverance_b200.models.gevovik import GevovikModel as Model
    else:
        Model = DecoderModel
    return Model(cfg, device).load(WeightLoader(d))


def engine_of(model, **kw):
    from deliverance_b200.engine.engine import Engine, EngineConfig
    from deliverance_b200.kv.paged import KvCacheSettings

    kv = kw.pop("kv", None) or KvCacheSettings()
    return Engine(model, EngineConfig(num_pages=kw.pop("pages", 256), max_batch_tokens=kw.pop("chunk", 64), kv=kv, max_seqs=kw.pop("max_seqs", 16), **kw))


def params_of(**kw):
    from deliverance_b200.params import GeneratorParameters

    return GeneratorParameters(**kw)


def plain_beams(model, prompt, W, steps, eos, lp):
    """Beam search by its definition: every hypothesis is run from the start at every step."""
    from deliverance_b200.params import FinishReason

    def logp(tokens):
        e = engine_of(model)
        r = e.open_replay()
        z = e.replay_step([(r, tokens, [len(tokens) - 1])])[0].double()
        return torch.log_softmax(z, -1)

    alive, ended = [(0.0, [])], []
    for n in range(1, steps + 1):
        cand = []
        for w, (score, toks) in enumerate(alive):
            for v, x in enumerate((logp(prompt + toks) + score).tolist()):
                cand.append((-x, w, v))
        cand = sorted(cand)[: 2 * W]
        nxt = []
        for rank, (x, w, v) in enumerate(cand):
            if v in eos or n == steps:
                if rank < W:
                    ended.append((-x / n**lp, alive[w][1] + [v], FinishReason.STOP_TOKEN if v in eos else FinishReason.MAX_TOKENS))
            elif len(nxt) < W:
                nxt.append((-x, alive[w][1] + [v]))
        ended = sorted(ended, key=lambda h: -h[0])[:W]
        alive = nxt
        if not alive or (len(ended) >= W and max(s for s, _ in alive) / n**lp <= ended[-1][0]):
            break
    return ended


@pytest.mark.parametrize("family,n,W,steps,lp,eos", [("llama", 5, 3, 6, 1.0, ()), ("llama", 31, 4, 5, 0.0, (7, 9)), ("llama", 32, 2, 4, 2.0, (3,)), ("qwen3", 63, 3, 4, 1.0, ()),
                                                      ("granitemoehybrid", 20, 3, 5, 1.0, ()), ("fopivik", 33, 2, 4, 1.0, ()), ("gevovik", 30, 3, 5, 1.0, ())])
def test_engine_beams_match_plain(tmp_path, family, n, W, steps, lp, eos):
    model = tiny_model(tmp_path, family)
    prompt = [(7 * i * i + 3 * i + 11) % 200 + 3 for i in range(n)]
    if eos:  # end tokens that come up: the likeliest continuations of the plain search without any
        eos = tuple({h[1][k] for h in plain_beams(model, prompt, W, steps, (), lp)[:2] for k in (2,)})
    want = plain_beams(model, prompt, W, steps, eos, lp)
    e = engine_of(model)
    e.eos_ids = frozenset(eos)
    free = e.kv.allocator.available()
    got = e.generate_beams([prompt], params_of(num_beams=W, max_tokens=steps, length_penalty=lp))[0]
    assert [r.token_ids for r in got] == [h[1] for h in want]
    assert [r.finish_reason for r in got] == [h[2] for h in want]
    # fp32 models, run in other orders: logits differ by rounding (2^-24 of sums of hundreds of terms of order one)
    assert max(abs(r.score - h[0]) for r, h in zip(got, want)) < 1e-3
    assert got[0].prompt_tokens == n and not e.running and not e.waiting
    e.kv.audit([])
    e.kv.prefix.clear()
    assert e.kv.allocator.available() == free
    if e.hybrid:
        assert len(e.kv.free_slots) == 16


def test_engine_beams_in_batches_and_repeats(tmp_path):
    """Prompts of one call share steps, some end before others; cached prefixes and other requests in between change nothing."""
    model = tiny_model(tmp_path, "llama")
    prompts = [[(5 * i * i + k * i + 2 * k + 1) % 200 + 3 for i in range(n)] for k, n in enumerate((3, 40, 64, 33, 70))]
    p = params_of(num_beams=3, max_tokens=20)
    e = engine_of(model, max_seqs=7)  # two prompts at a time
    alone = [engine_of(model).generate_beams([q], p)[0] for q in prompts]
    both = e.generate_beams(prompts, p)
    e.generate(prompts[1], params_of(max_tokens=4))
    again = e.generate_beams(prompts[::-1], p)[::-1]
    for a, b, c in zip(alone, both, again):
        assert [r.token_ids for r in a] == [r.token_ids for r in b] == [r.token_ids for r in c]
    e.kv.audit([])
    greedy = [r.token_ids for r in engine_of(model).generate_batch(prompts, params_of(max_tokens=20))]
    assert [engine_of(model).generate(q, p).token_ids for q in prompts] == [a[0].token_ids for a in alone]
    assert [r.token_ids for r in engine_of(model).generate_batch(prompts, p)] == [a[0].token_ids for a in alone]
    assert len(greedy) == 5


def test_beam_search_through_the_model_api(tmp_path):
    """Text in, ranked texts out; the first one is what ``generate`` answers."""
    from deliverance_b200.api import CausalLanguageModel
    from deliverance_b200.tokenizer.auto import AutoTokenizer

    model = tiny_model(tmp_path, "llama")
    clm = CausalLanguageModel(model, engine_of(model), AutoTokenizer.from_pretrained(str(tmp_path / "llama")), "t")
    p = params_of(num_beams=3, max_tokens=8)
    hyps = clm.generate_beams("Why is the sky blue?", p)
    best = clm.generate("Why is the sky blue?", p)
    assert best.token_ids == hyps[0].token_ids and best.text == hyps[0].text and best.score == hyps[0].score
    assert [r.score for r in hyps] == sorted([r.score for r in hyps], reverse=True) and all(isinstance(r.text, str) for r in hyps)
    assert [r.token_ids for r in clm.generate_many(["Why is the sky blue?", "Hi"], p)][0] == best.token_ids
    with pytest.raises(ValueError):
        clm.generate("Hi", p, on_event=lambda *a: None)
    with pytest.raises(ValueError):
        clm.submit("Hi", p)


def test_engine_beams_refusals(tmp_path):
    model = tiny_model(tmp_path, "llama")
    e = engine_of(model, pages=16, max_seqs=4)
    prompt = list(range(3, 40))
    for bad in (dict(num_beams=33), dict(num_beams=0), dict(num_beams=2, temperature=0.5), dict(num_beams=2, logprobs=True), dict(num_beams=2, stop_words=["x"]),
                dict(num_beams=2, guided_choice=["a"]), dict(num_beams=2, length_penalty=math.inf)):
        with pytest.raises(ValueError):
            e.generate_beams([prompt], params_of(max_tokens=4, **bad))
    with pytest.raises(ValueError):
        e.generate_beams([prompt], params_of(num_beams=5, max_tokens=4))  # more beams than places
    with pytest.raises(ValueError):
        e.add_request(prompt, params_of(num_beams=2))
    with pytest.raises(MemoryError):
        e.generate_beams([prompt], params_of(num_beams=4, max_tokens=200))
    with pytest.raises(ValueError):
        e.generate_beams([[]], params_of(num_beams=2, max_tokens=4))
    e.add_request(prompt, params_of(max_tokens=4))
    with pytest.raises(RuntimeError):
        e.generate_beams([prompt], params_of(num_beams=2, max_tokens=4))
    e.run()
    e.kv.audit([])
    assert len(e.generate_beams([prompt], params_of(num_beams=2, max_tokens=4))[0]) == 2
    e.kv.audit([])


@pytest.mark.gpu
@pytest.mark.parametrize("family,over", [("qwen3", dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64)), ("granitemoehybrid", dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64, mamba_d_head=64, mamba_n_heads=8)),
                                         ("qwen3", dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128))])
def test_engine_beams_on_the_gpu(tmp_path, family, over):
    """Captured steps and steps launched one by one give the same hypotheses, and their scores are those of the CPU model for these tokens."""
    cpu, gpu = tiny_model(tmp_path, family, **over), tiny_model(tmp_path, family, "cuda", **over)
    prompts = [[(7 * i * i + 3 * i + k) % 200 + 3 for i in range(n)] for k, n in enumerate((31, 64, 90))]
    p = params_of(num_beams=4, max_tokens=40)
    got = []
    for graphs in (True, False):
        e = engine_of(gpu, cuda_graphs=graphs)
        got.append(e.generate_beams(prompts, p))
        e.kv.audit([])
    assert [[r.token_ids for r in h] for h in got[0]] == [[r.token_ids for r in h] for h in got[1]]
    for prompt, hyps in zip(prompts, got[0]):
        assert hyps[0].score >= hyps[-1].score and len({tuple(r.token_ids) for r in hyps}) == 4
        e = engine_of(cpu)
        r = e.open_replay()
        toks = prompt + hyps[0].token_ids
        z = torch.log_softmax(e.replay_step([(r, toks, list(range(len(prompt) - 1, len(toks) - 1)))]).double(), -1)
        want = float(z.gather(1, torch.tensor(hyps[0].token_ids).view(-1, 1)).sum()) / len(hyps[0].token_ids)
        # bf16 activations over a few layers: a log-probability is off by some hundredths, here their mean over 40 tokens
        assert abs(hyps[0].score - want) < 0.1


@pytest.mark.parametrize("bad", [math.nan, INF])
def test_engine_beams_without_a_finite_continuation(tmp_path, bad):
    """A model that returns no numbers: the error says so, and nothing is lost. Hypotheses that ended before stand."""
    model = tiny_model(tmp_path, "llama")
    e, prompt = engine_of(model), list(range(3, 40))
    p = params_of(num_beams=3, max_tokens=6)
    want = e.generate_beams([prompt], p)[0]
    forward, calls = model.forward, []

    def broken(batch, kv):
        calls.append(1)
        z = forward(batch, kv)
        return torch.full_like(z, bad) if len(calls) > good else z

    model.forward = broken
    for good in (0, 1, 3):
        for call in (lambda: e.generate(prompt, p), lambda: e.generate_batch([prompt], p), lambda: e.generate_beams([prompt], p)):
            calls.clear()
            with pytest.raises(RuntimeError, match="logits are NaN"):
                call()
            assert not e.has_work()
            e.kv.audit([])
    first = want[0].token_ids[0]  # ends at the first step, as the others of its candidates do not
    e.eos_ids, good = frozenset([first]), 1
    calls.clear()
    assert [r.token_ids for r in e.generate_beams([prompt], p)[0]] == [[first]]
    model.forward, e.eos_ids = forward, frozenset()
    assert [r.token_ids for r in e.generate_beams([prompt], p)[0]] == [r.token_ids for r in want]


@pytest.mark.parametrize("lp", [1000.0, -2000.0, 33.0, math.nan, -INF])
def test_length_penalty_out_of_range_is_refused_at_once(tmp_path, lp):
    e = engine_of(tiny_model(tmp_path, "llama"))
    with pytest.raises(ValueError, match="length_penalty"):
        e.generate_beams([list(range(3, 40))], params_of(num_beams=2, max_tokens=9, length_penalty=lp))
    assert e.metrics["prefill_steps"] == 0


@pytest.mark.parametrize("lp", [32.0, -32.0])
def test_length_penalty_at_its_ends(tmp_path, lp):
    """The longest hypotheses, or the shortest, rank first, with finite scores; powers of the longest contexts are in range too."""
    model = tiny_model(tmp_path, "llama")
    e, prompt = engine_of(model), [(7 * i * i + 3 * i + 11) % 200 + 3 for i in range(31)]
    p = params_of(num_beams=4, max_tokens=5, length_penalty=lp)
    e.eos_ids = frozenset({h[1][2] for h in plain_beams(model, prompt, 4, 5, (), 0.0)[:2]})
    got = e.generate_beams([prompt], p)[0]
    assert [(r.score, r.token_ids) for r in got] == sorted([(r.score, r.token_ids) for r in got], key=lambda h: -h[0]) and all(math.isfinite(r.score) and r.score < 0 for r in got)
    assert (1 << 20) ** lp > 0 and math.isfinite(1e9 / (1 << 20) ** lp)


def test_beam_search_over_many_prompts_shares_its_steps(tmp_path):
    """``generate_many`` is one search over all prompts: as many decode steps as the longest takes, and the answers of one prompt after another."""
    from deliverance_b200.api import CausalLanguageModel
    from deliverance_b200.tokenizer.auto import AutoTokenizer

    model = tiny_model(tmp_path, "llama")
    tok = AutoTokenizer.from_pretrained(str(tmp_path / "llama"))
    prompts, p = ["Why is the sky blue?", "Hi", list(range(3, 40))], params_of(num_beams=3, max_tokens=8)
    one, many = (CausalLanguageModel(model, engine_of(model), tok, "t") for _ in range(2))
    one.engine.eos_ids = many.engine.eos_ids = frozenset()
    alone = [one.generate(q, p) for q in prompts]
    got = many.generate_many(prompts, p)
    assert [(r.token_ids, r.text) for r in got] == [(r.token_ids, r.text) for r in alone]
    assert max(abs(r.score - a.score) for r, a in zip(got, alone)) < 1e-3  # (fp32 in other orders)
    assert many.engine.metrics["decode_steps"] == 7 and one.engine.metrics["decode_steps"] == 21
    assert many.generate_many([], p) == []


def test_beam_search_has_no_session(tmp_path):
    """A session names a request's events, of which a search has none: refused like a callback for them, not left aside."""
    from deliverance_b200.api import CausalLanguageModel
    from deliverance_b200.tokenizer.auto import AutoTokenizer

    model = tiny_model(tmp_path, "llama")
    clm = CausalLanguageModel(model, engine_of(model), AutoTokenizer.from_pretrained(str(tmp_path / "llama")), "t")
    for kw in (dict(session="s"), dict(on_event=lambda *a: None)):
        with pytest.raises(ValueError):
            clm.generate("Hi", params_of(num_beams=3, max_tokens=8), **kw)
    assert clm.engine.metrics["prefill_steps"] == 0 and clm.generate("Hi", params_of(max_tokens=2), session="s").generated_tokens == 2


def test_all_prompts_are_checked_before_the_first_search(tmp_path):
    model = tiny_model(tmp_path, "llama")
    e, good = engine_of(model, pages=16, max_seqs=4), list(range(3, 40))
    p = params_of(num_beams=4, max_tokens=4)
    for bad, error in (([], ValueError), ([5, 10**6], ValueError), ([5] * 300, ValueError), (list(range(3, 163)), MemoryError)):
        with pytest.raises(error):
            e.generate_beams([good, bad], p if error is ValueError else params_of(num_beams=4, max_tokens=90))
        assert e.metrics["prefill_steps"] == 0 and not e.has_work()
        e.kv.audit([])
    assert len(e.generate_beams([good, good[:9]], p)) == 2


@pytest.mark.parametrize("device", DEVICES)
def test_select_values_beyond_fp32_are_no_candidates(device):
    """A masked place of the type's lowest value, scaled out of its range: a value that fp32 does not hold is none, and its place has no parent."""
    low = torch.finfo(F32).min
    for V, k in ((100, 8), (9000, 64)):
        logits = torch.full((2, V), low)
        logits[0, [3, V - 2]] = torch.tensor([2.0, 1.5])
        logits[1, 7] = 0.0
        scores = torch.tensor([[-1.0, -3.0]])
        # (the second token of the first beam: -1 - 2 - log(1 + e^-2) = -3.13 at a scale of 4, behind the second beam's -3; -1 - 0.75 - log(1 + e^-0.75) = -2.14 at 1.5)
        for inv_scale, parents, tokens in ((4.0, [0, 1, 0], [3, 7, V - 2]), (1.5, [0, 0, 1], [3, V - 2, 7])):
            v, p, t = (x.cpu()[0] for x in beam_select(logits.to(device), scores.to(device), k, inv_scale=inv_scale))
            assert p.tolist() == parents + [-1] * (k - 3) and t.tolist() == tokens + [-1] * (k - 3)
            assert v[:3].isfinite().all() and (v[3:] == -INF).all()
        # within the range they are candidates like any other
        v, p, t = (x.cpu()[0] for x in beam_select(logits.to(device), scores.to(device), k, inv_scale=0.5))
        assert t[:3].tolist() == [3, V - 2, 7] and p[3:].tolist() == [0] * (k - 3) and t[3:].tolist() == [j for j in range(V) if j not in (3, V - 2)][: k - 3] and v.isfinite().all()
