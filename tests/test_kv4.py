"""The KV cache in 4 bits (quantising write, unpacking, decode and prompt attention) and step tables against plain statements in 64 bits, on the CPU and, where there is a GPU, on the CUDA kernels."""
import math

import pytest
import torch

from deliverance_b200 import ops
from deliverance_b200.ops import ref
from deliverance_b200.ops.kv4 import decode_attention4, expand4, prefill_attention4, rope_kv4, row_bytes
from deliverance_b200.ops.tables import step_tables

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GPU = [pytest.param("cuda", marks=pytest.mark.gpu)]
BF16 = torch.bfloat16
HALF_STEP = torch.finfo(BF16).eps / 2


def done(device):
    if device == "cuda":
        ops.check_status()


def plain_block(x):
    """One block of 32 numbers by the definition, in Python: (codes, step, minimum)."""
    f32 = lambda v: torch.tensor(v, dtype=torch.float64).float().item()  # noqa: E731
    x = [min(max(float(v), -472.0), 472.0) for v in x]
    m = torch.tensor(min(x)).half().item()
    s0 = f32(max(f32(max(x) - m), 0.0) * f32(1 / 15))
    if s0 < 2.0**-14:
        s = math.ceil(s0 * 2**20) / 2**20
    else:
        frac, e = math.frexp(s0)
        s = math.ldexp(math.ceil(frac * 128), e - 7)
    codes = []
    for v in x:
        c = f32(f32(v - m) * f32(1 / s)) if s > 0 else 0.0
        codes.append(int(min(max(round(c), 0), 15)))  # (Python rounds halves to even, as rint does)
    return codes, s, m


def test_block_definition():
    for scale in (1e-6, 1e-5, 3e-4, 0.02, 1.0, 31.0, 2000.0):
        x = (torch.randn(40, 32) * scale).float()
        x[0] = 0.0
        x[1] = scale
        x[2, :16], x[2, 16:] = -0.0, 0.0
        x[3] = scale * torch.arange(32) / 31
        x[4, 0], x[4, 1] = math.inf, -math.inf
        rows = ref.kv4_pack(x)
        assert rows.shape == (40, row_bytes(32)) and row_bytes(128) == 80
        for r in range(40):
            codes, s, m = plain_block(x[r].tolist())
            packed = bytes(rows[r, :16].tolist())
            assert [packed[i // 2] >> (4 * (i % 2)) & 15 for i in range(32)] == codes
            side = rows[r, 16:].view(torch.float16)
            assert side[0].item() == s and side[1].item() == m and math.copysign(1.0, m or 1.0) == math.copysign(1.0, side[1].item() or 1.0)
        back = ref.kv4_unpack(rows)
        lo = x.clamp(-472, 472).amin(1, keepdim=True)
        step = rows[:, 16:18].view(torch.float16).float()
        # half a step, half a step of fp16 of the minimum (or of its smallest numbers), and the fp32 roundings of (x - m) / s, some 2^-22 of 15 steps
        assert ((back - x.clamp(-472, 472)).abs() <= step * (0.5 + 2.0**-18) + lo.abs() * 2.0**-11 + 2.0**-25).all()


def test_nan_makes_its_block_nan():
    x = torch.randn(3, 128)
    x[1, 70] = math.nan
    back = ref.kv4_unpack(ref.kv4_pack(x))
    assert torch.isnan(back[1, 64:96]).all() and not torch.isnan(back[1, :64]).any() and not torch.isnan(back[1, 96:]).any() and not torch.isnan(back[[0, 2]]).any()


def rotary(positions, half, far, mult=1.0):
    turn = torch.arange(far, dtype=torch.float64).view(-1, 1) * (1e4 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1)))
    return (torch.cos(turn) * mult).float(), (torch.sin(turn) * mult).float()


def exact_heads(x, w, eps, offset, cos, sin, positions, pairs):
    """fp64 [T, heads, D], element by element of a head."""
    x = x.double().clone()
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + eps) * (w.double() + offset)
    if cos is not None:
        y = x.clone()
        at = positions.clamp(0, cos.shape[0] - 1).long()
        for i in range(cos.shape[1]):
            a, b = (2 * i, 2 * i + 1) if pairs else (i, i + cos.shape[1])
            c, s = cos[at, i].double().view(-1, 1), sin[at, i].double().view(-1, 1)
            y[..., a] = x[..., a] * c - x[..., b] * s
            y[..., b] = x[..., b] * c + x[..., a] * s
        x = y
    return x


WRITES = [(D, H, KV, T, rotate, half, norm) for D, half in ((64, 32), (128, 64), (256, 128)) for H, KV, T in ((1, 1, 1), (6, 2, 37), (12, 3, 5))
          for rotate, norm in (("halves", True), ("pairs", False))] + [
    (64, 4, 1, 9, "halves", 5, True), (64, 4, 1, 9, "pairs", 5, False), (128, 4, 2, 9, "halves", 16, False), (128, 4, 2, 9, "halves", 20, True), (256, 2, 1, 9, "pairs", 33, True),
    (128, 4, 2, 9, "halves", 0, True), (128, 32, 8, 130, "halves", 64, True)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,H,KV,T,rotate,half,norm", WRITES)
def test_write_matches_plain(device, D, H, KV, T, rotate, half, norm):
    page, pages, eps, offset = 32 if D < 256 else 64, 2 + T // 16, 1e-5, 1.0 if T % 2 else 0.0
    wide = torch.randn(T, (H + 2 * KV) * D + 24).to(BF16)  # (rows further apart than they are long)
    wide[:, : H * D] *= 3
    qn, kn = (torch.randn(D).to(BF16), torch.randn(D).to(BF16)) if norm else (None, None)
    far = 300
    cos, sin = rotary(None, half, far, 1.2) if half else (None, None)
    positions = torch.randint(-2, far + 2, (T,), dtype=torch.int32)
    slots = torch.randperm(pages * page)[:T]
    if T > 3:
        slots[2] = -1
    start = torch.randint(0, 256, (2, pages, KV, page, row_bytes(D)), dtype=torch.uint8)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    x = to(wide)[:, : (H + 2 * KV) * D]
    before = x.clone()
    kc, vc = to(start[0].clone()), to(start[1].clone())
    q = rope_kv4(x, to(positions), to(slots), to(qn), to(kn), to(cos), to(sin), kc, vc, H, KV, D, eps, offset, rotate)
    done(device)
    assert torch.equal(x, before) and q.shape == (T, H * D) and q.dtype == BF16
    heads = wide[:, : (H + 2 * KV) * D].reshape(T, H + 2 * KV, D)
    want = exact_heads(heads[:, :H], qn, eps, offset, cos, sin, positions, rotate == "pairs").flatten(1)
    # one rounding to bf16, and before it fp32 roundings of some six products and sums no larger than 1.2 (|a| + |b|) of a pair
    size = 2.4 * exact_heads(heads[:, :H], qn, eps, offset, None, None, None, False).abs().amax(-1, keepdim=True).expand(T, H, D).flatten(1)
    assert ((q.cpu().double() - want).abs() <= want.abs() * HALF_STEP + size * 2.0**-21).all()
    # the cache: the same bytes as the plain statement, everything else as it was
    k64 = exact_heads(heads[:, H : H + KV], kn, eps, offset, cos, sin, positions, rotate == "pairs")
    k2, v2 = start[0].clone(), start[1].clone()
    ref.rope_kv4(wide[:, : (H + 2 * KV) * D], positions, slots, qn, kn, cos, sin, k2, v2, H, KV, D, eps, offset, rotate == "pairs")
    assert torch.equal(kc.cpu(), k2) and torch.equal(vc.cpu(), v2)
    for cache, old, fresh in ((kc, start[0], k64), (vc, start[1], heads[:, H + KV :].double())):
        flat, was = cache.cpu().transpose(1, 2).flatten(0, 1), old.transpose(1, 2).flatten(0, 1)
        written = slots[slots >= 0]
        rest = torch.ones(flat.shape[0], dtype=torch.bool)
        rest[written] = False
        assert torch.equal(flat[rest], was[rest])
        rows = flat[written]
        step = rows[..., D // 2 :].contiguous().view(torch.float16).float().unflatten(-1, (-1, 2))[..., 0].repeat_interleave(32, -1)
        x64 = fresh[slots >= 0].clamp(-472, 472)
        lo = x64.unflatten(-1, (-1, 32)).amin(-1).abs().repeat_interleave(32, -1)
        assert ((ref.kv4_unpack(rows).double() - x64).abs() <= step * (0.5 + 2.0**-18) + lo * 2.0**-11 + x64.abs().amax() * 2.0**-20).all()


@pytest.mark.parametrize("device", GPU)
def test_write_of_extremes_has_the_plain_bytes(device):
    D, H, KV, T = 128, 2, 2, 64
    x = torch.randn(T, H + 2 * KV, D) * 10.0 ** torch.randint(-7, 4, (T, 1, 1))
    x[5, 2:, 3], x[6, 2:, 9], x[7, 2:, 40], x[8], x[9] = math.nan, math.inf, -math.inf, 0.0, -0.0
    x = x.to(BF16).flatten(1)
    k, v = (torch.zeros(2, KV, 32, row_bytes(D), dtype=torch.uint8) for _ in range(2))
    kc, vc = k.to(device), v.to(device)
    slots, positions = torch.arange(T), torch.zeros(T, dtype=torch.int32)
    ref.rope_kv4(x, positions, slots, None, None, None, None, k, v, H, KV, D, 1e-6, 0.0, False)
    rope_kv4(x.to(device), positions.to(device), slots.to(device), None, None, None, None, kc, vc, H, KV, D, 1e-6)
    done(device)
    assert torch.equal(kc.cpu(), k) and torch.equal(vc.cpu(), v)


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("D,rotate,half", [(64, "halves", 32), (128, "halves", 64), (128, "halves", 32), (256, "pairs", 128), (128, "pairs", 21), (256, "halves", 24)])
def test_write_of_many_rows_has_the_plain_bytes(device, D, rotate, half):
    """Any operation that is contracted with another one shows in some thousand rows."""
    T, H, KV = 3000, 4, 2
    x, cos, sin = torch.randn(T, (H + 2 * KV) * D).to(BF16), *rotary(None, half, 5000)
    qn, kn = torch.randn(D).to(BF16), torch.randn(D).to(BF16)
    k, v = (torch.zeros(T // 32 + 1, KV, 32, row_bytes(D), dtype=torch.uint8) for _ in range(2))
    kc, vc = k.to(device), v.to(device)
    slots, positions = torch.randperm(T), torch.randint(0, 5000, (T,), dtype=torch.int32)
    q = ref.rope_kv4(x, positions, slots, qn, kn, cos, sin, k, v, H, KV, D, 1e-6, 0.0, rotate == "pairs")
    to = lambda t: t.to(device)  # noqa: E731
    got = rope_kv4(to(x), to(positions), to(slots), to(qn), to(kn), to(cos), to(sin), kc, vc, H, KV, D, 1e-6, 0.0, rotate)
    done(device)
    assert torch.equal(kc.cpu(), k) and torch.equal(vc.cpu(), v) and torch.equal(got.cpu(), q)


def random_cache(pages, KV, page, D, loud=True):
    x = torch.randn(pages, KV, page, D)
    if loud:
        x[..., :: 17] *= 6
    return ref.kv4_pack(x)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,KV,page", [(64, 3, 32), (128, 1, 96), (256, 2, 64)])
def test_expand_matches_plain(device, D, KV, page):
    k, v = random_cache(7, KV, page, D), random_cache(7, KV, page, D)
    for pages in ([3], [6, 0, 6, 1], []):
        want = [ref.kv4_unpack(t)[torch.tensor(pages, dtype=torch.long)] for t in (k, v)]
        for dtype in (torch.float32, BF16):
            got = expand4(k.to(device), v.to(device), torch.tensor(pages, dtype=torch.int32, device=device), dtype)
            done(device)
            for g, w in zip(got, want):
                assert g.dtype == dtype and torch.equal(g.cpu(), w.to(dtype))


def tables_for(lens, page, first=1, extra=0):
    need = [-(-n // page) for n in lens]
    order = (torch.randperm(sum(need)) + first).to(torch.int32)
    t = torch.zeros(len(lens), max(max(need), 1) + extra, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at : at + n]
        at += n
    return t, first + sum(need)


def plain_attention(q, k, v, table, lens, news, KV, scale, softcap, window, values=ref.kv4_unpack):
    """fp64 outputs, and what errors are measured by: sum of p |v|, and the largest sum of |q| |k| of a row."""
    D = k.shape[3] * 8 // 5
    out, mass, reach = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    row = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        if m == 0:
            continue
        pages = table[b, : -(-n // k.shape[2])].long()
        K, V = (values(t[pages]).transpose(0, 1).flatten(1, 2)[:, :n].double() for t in (k, v))
        Q = q[row : row + m].double().view(m, KV, -1, D).permute(1, 2, 0, 3)
        x = torch.einsum("kgtd,knd->kgtn", Q, K) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        last, j = torch.arange(n - m, n).view(-1, 1), torch.arange(n)
        hidden = j > last
        if window:
            hidden = hidden | (j <= last - window)
        if n:  # (without keys: zeros)
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            flat = lambda y: y.permute(2, 0, 1, 3).reshape(m, -1)  # noqa: E731
            out[row : row + m] = flat(torch.einsum("kgtn,knd->kgtd", p, torch.where(torch.isfinite(V), V, 0.0)))
            mass[row : row + m] = flat(torch.einsum("kgtn,knd->kgtd", p, torch.where(torch.isfinite(V), V, 0.0).abs()))
            size = torch.einsum("kgtd,knd->kgtn", Q.abs(), K.abs()).masked_fill(hidden, 0.0).amax(-1, keepdim=True) * scale
            reach[row : row + m] = flat(size.expand(*size.shape[:-1], D))
        row += m
    return out, mass, reach


def check_decode(got, q, k, v, table, lens, KV, scale, softcap, window):
    want, mass, reach = plain_attention(q, k, v, table, lens, [1] * len(lens), KV, scale, softcap, window)
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    # the result's rounding to bf16; of every probability one rounding to fp16 and the exponential's 2^-21 and 2^-22 of its argument, numerator and denominator; of a score, whose codes, steps and minima are exact, fp32 sums of 256 numbers
    # (products of tensor cores are cut off, not rounded: 2^-22 of the sum of magnitudes per addition would be 2^-14 at worst, and errs one way for all keys alike; 2^-17 is allowed)
    tol = want.abs() * HALF_STEP + mass * (2.0**-10 + reach * (2.0**-16 + 2.0**-20)) + 1e-30
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


def run_decode(device, D, KV, G, lens, softcap=0.0, window=0, page=32, extra=1, spoil=True, scale=None, mult=1.0):
    B, H = len(lens), KV * G
    table, pages = tables_for(lens, page, extra=extra)
    q = (torch.randn(B, H * D) * mult).to(BF16)
    k, v = random_cache(pages, KV, page, D), random_cache(pages, KV, page, D, False)
    if spoil:  # what lies behind a sequence's end or in front of its window must not matter, not even infinities and NaN
        for b, n in enumerate(lens):
            if n % page:
                k[table[b, n // page].long(), :, n % page :] = v[table[b, n // page].long(), :, n % page :] = 0xFE
            if window and n > window:
                for j in range(n - window):
                    k[table[b, j // page].long(), :, j % page] = v[table[b, j // page].long(), :, j % page] = 0x7D if j % 2 else 0xFE
    scale = scale or D**-0.5
    to = lambda t: t.to(device)  # noqa: E731
    got = decode_attention4(to(q), to(k), to(v), to(table), to(torch.tensor(lens, dtype=torch.int32)), H, scale, softcap, window)
    done(device)
    assert got.shape == q.shape and got.dtype == BF16
    check_decode(got, q, k, v, table, lens, KV, scale, softcap, window)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("KV,G", [(1, 1), (2, 4), (3, 5), (1, 16), (8, 8), (2, 9)])
@pytest.mark.parametrize("lens", [[1], [33, 0, 1, 500], [700, 31, 32], [3001, 2], [64] * 70, [0]])
def test_decode_matches_plain(device, D, KV, G, lens):
    if device == "cpu" and sum(lens) * KV * G * D > 3e7:
        pytest.skip("large for the CPU")
    run_decode(device, D, KV, G, lens)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G,softcap,window", [(2, 50.0, 0), (12, 0.5, 0), (2, 0.0, 100), (8, 50.0, 17), (3, 0.0, 1)])
def test_decode_softcap_window(device, D, G, softcap, window):
    run_decode(device, D, 2, G, [777, 16, 100, 101, 0, 1], softcap, window)


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("lens", [[40000], [20000, 1, 3, 500, 9000], [100 + 7 * i for i in range(130)], [1] * 300, [32] * 128, [5000] * 9, [31, 33] * 40])
@pytest.mark.parametrize("D,KV,G", [(128, 8, 4), (64, 1, 2), (256, 2, 16)])
def test_decode_work_split(device, lens, D, KV, G):
    run_decode(device, D, KV, G, lens, page=64 if len(lens) == 5 else 32, extra=0, spoil=len(lens) < 200)


@pytest.mark.parametrize("device", DEVICES)
def test_decode_sharp_and_large(device):
    run_decode(device, 128, 2, 4, [300, 65], mult=60.0)  # single keys take all the weight, scores of thousands
    run_decode(device, 128, 2, 4, [300, 65], mult=3e4, scale=1e-6)
    run_decode(device, 64, 1, 8, [200], mult=1e-30, scale=1e30)
    run_decode(device, 64, 1, 8, [200], mult=0.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_decode_scale_of_any_sign(device, scale):
    D, KV, G, lens = 128, 2, 3, [40, 1, 200]
    table, pages = tables_for(lens, 32)
    q, k, v = torch.randn(3, KV * G * D).to(BF16), random_cache(pages, KV, 32, D), random_cache(pages, KV, 32, D, False)
    to = lambda t: t.to(device)  # noqa: E731
    got = decode_attention4(to(q), to(k), to(v), to(table), to(torch.tensor(lens, dtype=torch.int32)), KV * G, scale)
    done(device)
    want, mass, reach = plain_attention(q, k, v, table, lens, [1] * 3, KV, scale, 0.0, 0)
    assert ((got.cpu().double() - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + reach.abs() * 2.0**-15) + 1e-30).all()


@pytest.mark.parametrize("device", DEVICES)
def test_decode_nan_stays_where_it_is(device):
    """A NaN in a query is its head's, one in a cached value its block's of the sequences that see it, and a misaligned or strided query is taken as it is."""
    D, KV, G, lens = 128, 2, 2, [100, 70, 33]
    table, pages = tables_for(lens, 32)
    wide = torch.randn(3, KV * G * D + 3).to(BF16)
    q = wide[:, 1 : 1 + KV * G * D]
    wide[1, 1 + D + 5] = math.nan  # head 1 of sequence 1
    k, x = random_cache(pages, KV, 32, D), torch.randn(pages, KV, 32, D)
    x[table[2, 0].long(), 1, 7, 40] = math.nan  # KV head 1 of sequence 2, block 1
    v = ref.kv4_pack(x)
    to = lambda t: t.to(device)  # noqa: E731
    got = decode_attention4(to(wide)[:, 1 : 1 + KV * G * D], to(k), to(v), to(table), to(torch.tensor(lens, dtype=torch.int32)), KV * G, D**-0.5).cpu().view(3, KV * G, 4, 32)
    done(device)
    bad = torch.zeros(3, KV * G, 4, 32, dtype=torch.bool)
    bad[1, 1] = True
    bad[2, 2:, 1] = True
    assert torch.equal(torch.isnan(got), bad)
    want, mass, reach = plain_attention(torch.nan_to_num(q), k, ref.kv4_pack(torch.nan_to_num(x)), table, lens, [1] * 3, KV, D**-0.5, 0.0, 0)
    err, tol = (got.double().flatten(1) - want).abs(), want.abs() * HALF_STEP + mass * (2.0**-10 + reach * 2.0**-15) + 1e-30
    assert (err <= tol)[~bad.flatten(1)].all()


@pytest.mark.parametrize("device", GPU)
def test_captured_calls_on_a_stream(device):
    """Writing, decode attention and tables in a captured graph, replayed with other lengths, pages and rows, beside calls on another stream."""
    D, H, KV, B, width = 128, 8, 2, 5, 12
    to = lambda t: t.to(device)  # noqa: E731
    cos, sin = (to(t) for t in rotary(None, 64, 400))
    kc, vc = (to(random_cache(B * width + 1, KV, 32, D, loud)) for loud in (True, False))
    qkv = torch.zeros(B, (H + 2 * KV) * D, dtype=BF16, device=device)
    pos, ctx = (torch.zeros(B, dtype=torch.int32, device=device) for _ in range(2))
    slots, table = torch.zeros(B, dtype=torch.int64, device=device), torch.zeros(B, width, dtype=torch.int32, device=device)

    def step(cache_k, cache_v):
        q = rope_kv4(qkv, pos, slots, None, None, cos, sin, cache_k, cache_v, H, KV, D, 1e-6)
        return q, decode_attention4(q, cache_k, cache_v, table, ctx, H, D**-0.5)

    slots.copy_(torch.arange(B))
    ctx.fill_(1)
    step(kc.clone(), vc.clone())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        q, out = step(kc, vc)
    side = torch.cuda.Stream()
    for lens in ([1, 1, 1, 1, 1], [300, 2, 33, 64, 384], [7, 384, 384, 1, 90]):
        pages = (torch.randperm(B * width) + 1).view(B, width).to(torch.int32)
        new = torch.tensor(lens) - 1
        qkv.copy_(torch.randn(qkv.shape))
        pos.copy_(new)
        ctx.copy_(torch.tensor(lens))
        table.copy_(pages)
        slots.copy_(pages.gather(1, (new // 32).view(-1, 1)).view(-1).long() * 32 + new % 32)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            apart = [step(kc.clone(), vc.clone())[1] for _ in range(3)]
        graph.replay()
        torch.cuda.synchronize()
        done(device)
        assert all(torch.equal(a, out) for a in apart)
        check_decode(out, q.cpu(), kc.cpu(), vc.cpu(), pages, lens, KV, D**-0.5, 0.0, 0)


def run_prefill(device, D, KV, G, news, befores, softcap=0.0, window=0, page=32):
    lens = [a + b for a, b in zip(news, befores)]
    H, T = KV * G, sum(news)
    table, pages = tables_for(lens, page, extra=1)
    q = torch.randn(T, H * D).to(BF16)
    k, v = random_cache(pages, KV, page, D, False), random_cache(pages, KV, page, D, False)
    for b, n in enumerate(lens):
        if n % page:
            k[table[b, n // page].long(), :, n % page :] = v[table[b, n // page].long(), :, n % page :] = 0xFE
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    start = [sum(news[:i]) for i in range(len(news))]
    got = prefill_attention4(q.to(device), k.to(device), v.to(device), table.to(device), i32(start), i32(news), i32(lens), H, D**-0.5, softcap, window)
    done(device)
    if device == "cpu":
        want, mass, reach = plain_attention(q, k, v, table, lens, news, KV, D**-0.5, softcap, window)
        tol = want.abs() * HALF_STEP + mass * (2.0**-16 + reach * 2.0**-16)
    else:  # keys and values in fp16, as the kernel behind reads them (2^-12 of a value, tested by itself): probabilities in fp16, numerator and denominator, fp32 sums as in decoding, the result in bf16
        want, mass, reach = plain_attention(q, k, v, table, lens, news, KV, D**-0.5, softcap, window, lambda t: ref.kv4_unpack(t, torch.float16))
        tol = want.abs() * HALF_STEP + mass * (2.0**-10 + reach * 2.0**-16)
    assert ((got.cpu().double() - want).abs() <= tol + 1e-30).all(), ((got.cpu().double() - want).abs() / (tol + 1e-30)).max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,KV,G", [(64, 2, 3), (128, 1, 4), (256, 2, 1)])
@pytest.mark.parametrize("news,befores", [([1], [0]), ([33, 5], [0, 70]), ([130, 1, 64], [3, 31, 0]), ([3, 0, 2], [0, 40, 9])])
def test_prefill_matches_plain(device, D, KV, G, news, befores):
    run_prefill(device, D, KV, G, news, befores)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("softcap,window,page", [(30.0, 0, 32), (0.0, 40, 64), (50.0, 7, 32), (0.0, 0, 96)])
def test_prefill_options(device, softcap, window, page):
    run_prefill(device, 64, 2, 2, [70, 40], [100, 0], softcap, window, page)


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("D,KV,G,news,befores", [(64, 4, 8, [600, 1, 129], [0, 64, 300]), (128, 8, 4, [257, 500], [40, 0]), (128, 8, 4, [128] * 4 + [1], [0] * 5), (128, 8, 4, [128] * 4, [0] * 4)])
def test_prefill_tile_heights(device, D, KV, G, news, befores, monkeypatch):
    """Calls on both sides of the rule on query tiles; a sequence has the same bits whichever height its call takes (its keys in one part)."""
    from deliverance_b200.ops import kv4

    run_prefill(device, D, KV, G, news, befores)
    monkeypatch.setattr(kv4, "_parts", lambda *args: 1)
    lens, H = [a + b for a, b in zip(news, befores)], KV * G
    table, pages = tables_for(lens, 32)
    k, v = (random_cache(pages, KV, 32, D, False).to(device) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q, start = torch.randn(sum(news), H * D, device=device).to(BF16), [sum(news[:i]) for i in range(len(news))]
    whole = prefill_attention4(q, k, v, table.to(device), i32(start), i32(news), i32(lens), H, D**-0.5)
    for b, (at, n) in enumerate(zip(start, news)):
        alone = prefill_attention4(q[at : at + n], k, v, table[b : b + 1].to(device), i32([0]), i32([n]), i32([lens[b]]), H, D**-0.5)
        assert torch.equal(alone, whole[at : at + n])
    done(device)


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("D,KV,G", [(64, 2, 3), (128, 1, 4), (256, 2, 1)])
@pytest.mark.parametrize("news,befores,softcap,window", [([1], [1023], 0.0, 0), ([1], [5000], 0.0, 0), ([33, 5], [2100, 70], 0.0, 0), ([130, 1, 64], [3, 4031, 0], 30.0, 0), ([3, 0, 2], [2000, 40, 9], 0.0, 0),
                                                         ([300], [3000], 0.0, 1500), ([129, 2], [100, 4000], 0.5, 1000), ([128], [1408], 0.0, 0), ([2000], [0], 0.0, 0)])
def test_prefill_in_parts(device, D, KV, G, news, befores, softcap, window):
    """Few query rows behind many keys: the keys are cut into parts."""
    from deliverance_b200.ops import kv4

    tiles = sum(-(-n // 128) for n in news) * KV * G
    assert kv4._parts(news, [a + b for a, b in zip(news, befores)], 128, KV * G, window) > 1 or 148 // tiles == 1  # (16 tiles of 6 heads are 96: whole)
    run_prefill(device, D, KV, G, news, befores, softcap, window)


@pytest.mark.parametrize("device", GPU)
def test_prefill_in_parts_captured(device):
    """Two captured calls with workspaces of their own, replayed in turn on two streams, with other tokens behind the same addresses."""
    KV, D, H, page, lens, news = 2, 64, 4, 32, [3000, 700], [40, 7]
    table, pages = tables_for(lens, page)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    k, v = (random_cache(pages, KV, page, D, False).to(device) for _ in range(2))
    rest = (k, v, table.to(device), i32([0, 40]), i32(news), i32(lens), H, 0.1)
    tiles = tuple(i32(t) for t in ops.prefill_tiles(news, 128))
    qs = [torch.randn(47, H * D).to(BF16).to(device) for _ in range(2)]
    run = lambda q: prefill_attention4(q, *rest, q_len_host=news, ctx_len_host=lens, tiles_for=lambda rows: tiles)  # noqa: E731
    run(qs[0])
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in qs]
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(q))
    for _ in range(3):
        for q in qs:
            q.copy_(torch.randn(47, H * D).to(BF16))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for q, out in zip(qs, outs):
            assert torch.equal(out, run(q))
    done(device)


@pytest.mark.parametrize("device", GPU)
def test_prefill_in_parts_keeps_nan(device):
    """A NaN block reaches the rows and heads that see it, whichever part holds it, and no others."""
    KV, D, H, page, lens = 2, 64, 4, 32, [4000]
    table, pages = tables_for(lens, page)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q = torch.randn(20, H * D).to(BF16).to(device)
    for cache, pos in ((0, 5), (0, 3000), (1, 5), (1, 2500), (0, 3990)):
        kv = [random_cache(pages, KV, page, D, False) for _ in range(2)]
        kv[cache][table[0, pos // page].long(), 1, pos % page, D // 2 :] = 0x7F
        got = prefill_attention4(q, kv[0].to(device), kv[1].to(device), table.to(device), i32([0]), i32([20]), i32(lens), H, 0.1).cpu().float().reshape(20, H, D)
        done(device)
        sees = torch.arange(20) + 3980 >= pos
        assert got[sees][:, 2:].isnan().all() and not got[:, :2].isnan().any()
        if cache == 0:
            assert not got[~sees].isnan().any()


def test_prefill_parts_rule():
    from deliverance_b200.ops.kv4 import _parts

    assert _parts([], [], 128, 4, 0) == 1 and _parts([1], [100], 128, 32, 0) == 1 and _parts([1], [10**6], 256, 32, 0) == 1
    assert _parts([100], [9000], 128, 32, 0) == 4 and _parts([200], [9000], 128, 32, 0) == 2 and _parts([300], [9000], 128, 32, 0) == 1
    assert _parts([1], [2**20], 128, 1, 0) == 32 and _parts([1], [2**20], 128, 1, 100) == 1 and _parts([0], [0], 128, 1, 0) == 1


@pytest.mark.parametrize("device", DEVICES)
def test_prefill_of_nothing(device):
    k = random_cache(2, 2, 32, 64).to(device)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
    q = torch.zeros(0, 256, dtype=BF16, device=device)
    assert prefill_attention4(q, k, k, i32(0, 1), i32(0), i32(0), i32(0), 4, 0.1).shape == (0, 256)
    assert prefill_attention4(q, k, k, i32(2, 1), i32(2), i32(2), i32(2), 4, 0.1).shape == (0, 256)
    done(device)


@pytest.mark.parametrize("device", GPU)
def test_prefill_ends_of_the_range(device):
    """Queries at both ends of bf16's range are as good as ordinary ones: their rows are scaled in front of fp16."""
    D, H, KV = 128, 4, 2
    table, pages = tables_for([90], 32)
    k, v = random_cache(pages, KV, 32, D), random_cache(pages, KV, 32, D, False)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q = torch.randn(50, H * D)
    for size, scale in ((1.0, 0.09), (1e30, 9e-32), (1e-30, 9e28)):
        x = (q * size).to(BF16)
        got = prefill_attention4(x.to(device), k.to(device), v.to(device), table.to(device), i32([0]), i32([50]), i32([90]), H, scale)
        done(device)
        want, mass, reach = plain_attention(x, k, v, table, [90], [50], KV, scale, 0.0, 0, lambda t: ref.kv4_unpack(t, torch.float16))
        assert ((got.cpu().double() - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + reach * 2.0**-16) + 1e-30).all()


@pytest.mark.parametrize("device", GPU)
def test_prefill_in_portions(device, monkeypatch):
    from deliverance_b200.ops import kv4

    monkeypatch.setattr(kv4, "EXPAND_PAGES_BYTES", 5 * 2 * 32 * 64 * 4)
    run_prefill(device, 64, 2, 2, [70, 40, 1, 9, 300], [100, 0, 20, 3, 0])


def plain_tables(pages, cached, start, new, width, page, tile):
    out = {n: [] for n in ("positions", "slots", "q_start", "ctx_len", "block_tables", "logits_rows", "tile_seq", "tile_q0")}
    row = 0
    for i, n in enumerate(new):
        out["q_start"].append(row)
        out["ctx_len"].append(cached[i] + n)
        out["logits_rows"].append(row + n - 1)
        out["block_tables"].append(pages[i] + [0] * (width - len(pages[i])))
        for j in range(n):
            out["positions"].append(start[i] + j)
            out["slots"].append(pages[i][(cached[i] + j) // page] * page + (cached[i] + j) % page)
        for t in range(0, n, tile):
            out["tile_seq"].append(i)
            out["tile_q0"].append(t)
        row += n
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new,page,tile", [([1], 32, 64), ([1] * 70, 32, 64), ([333, 1, 64, 65], 32, 64), ([5, 0, 0, 129, 0], 64, 32), ([0], 32, 64), ([3] * 1000, 96, 64), ([], 32, 64)])
def test_step_tables(device, new, page, tile):
    cached = [int(torch.randint(0, 200, ())) for _ in new]
    start = [c + int(torch.randint(0, 50, ())) for c in cached]
    need = [-(-(c + n) // page) + i % 3 for i, (c, n) in enumerate(zip(cached, new))]  # (some hold pages in reserve)
    order = (torch.randperm(sum(need)) + 1 + (1 << 28 if page == 96 else 0)).tolist()  # (slots beyond 32 bits)
    pages = [order[sum(need[:i]) : sum(need[: i + 1])] for i in range(len(new))]
    width, tiles = max(need + [0]) + 2, sum(-(-n // tile) for n in new)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    got = step_tables(i32(order), i32([sum(need[:i]) for i in range(len(new) + 1)]), i32(cached), i32(start), i32(new), sum(new), width, page, tile, tiles)
    done(device)
    want = plain_tables(pages, cached, start, new, width, page, tile)
    for name, t in got._asdict().items():
        dtype = torch.int64 if name in ("slots", "logits_rows") else torch.int32
        assert t.dtype == dtype and t.device.type == device
        assert torch.equal(t.cpu(), torch.tensor(want[name], dtype=dtype).reshape(t.shape)), name
    assert step_tables(i32(order), i32([sum(need[:i]) for i in range(len(new) + 1)]), i32(cached), i32(start), i32(new), sum(new), width, page).tile_seq.numel() == 0


BAD_TABLES = [
    dict(tokens=4),  # five rows
    dict(new=[2, -3]),
    dict(tiles=3),
    dict(width=1),
    dict(cached=[31, 33]),  # row 64 has no page
    dict(cached=[-1, 0]),
    dict(page_start=[0, 2, 9]),
    dict(page_start=[0, 3, 2]),
    dict(page_start=[-1, 1, 3]),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", BAD_TABLES)
def test_step_tables_reports(device, change):
    a = dict(pages=[4, 5, 6], page_start=[0, 1, 3], cached=[0, 30], start=[0, 30], new=[2, 3], tokens=5, width=2, tiles=2)
    a.update(change)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    call = lambda: step_tables(i32(a["pages"]), i32(a["page_start"]), i32(a["cached"]), i32(a["start"]), i32(a["new"]), a["tokens"], a["width"], 32, 64, a["tiles"])  # noqa: E731
    if device == "cpu":
        with pytest.raises(ValueError):
            call()
    else:
        got = call()
        with pytest.raises(RuntimeError, match="bad kernel arguments"):
            ops.check_status()
        ops.check_status()
        assert ((got.slots >= -1) & (got.slots < 7 * 32)).all() and ((got.block_tables >= 0) & (got.block_tables <= 6)).all()


def kv4_args(device, D=64, H=4, KV=2, T=3):
    to = lambda t: t.to(device)  # noqa: E731
    return dict(qkv=to(torch.randn(T, (H + 2 * KV) * D).to(BF16)), positions=to(torch.arange(T, dtype=torch.int32)), slots=to(torch.arange(T)), q_norm_w=to(torch.ones(D, dtype=BF16)),
                k_norm_w=to(torch.ones(D, dtype=BF16)), cos=to(torch.ones(9, D // 2)), sin=to(torch.zeros(9, D // 2)), k_cache=to(torch.zeros(2, KV, 32, row_bytes(D), dtype=torch.uint8)),
                v_cache=to(torch.zeros(2, KV, 32, row_bytes(D), dtype=torch.uint8)), H=H, KV=KV, D=D, eps=1e-6)


BAD_WRITES = [
    dict(rotate="thirds"), dict(D=96), dict(H=5), dict(KV=3), dict(cos=None), dict(k_norm_w=None), dict(positions=slice(0, 2)), dict(slots=slice(0, 2)), dict(slots=torch.int32),
    dict(k_cache=torch.int8), dict(v_cache=(2, 2, 32, 41)), dict(v_cache=(3, 2, 32, 40)), dict(cos=(9, 33), sin=(9, 33)), dict(sin=(8, 32)), dict(k_cache=(2, 2, 16, 40), v_cache=(2, 2, 16, 40)),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", BAD_WRITES)
def test_write_refuses(device, change):
    a = kv4_args(device)
    for name, c in change.items():
        t = a.get(name)
        a[name] = t[c] if isinstance(c, slice) else t.to(c) if isinstance(c, torch.dtype) else torch.zeros(c, dtype=t.dtype, device=device) if isinstance(c, tuple) else c
    with pytest.raises((ValueError, RuntimeError)):
        rope_kv4(**a)
    done(device)


@pytest.mark.parametrize("device", DEVICES)
def test_write_reports_slots_behind_the_cache(device):
    a = kv4_args(device)
    a["slots"] = torch.tensor([0, 64, 1 << 40], device=device)
    if device == "cpu":
        with pytest.raises(IndexError):
            rope_kv4(**a)
    else:
        rope_kv4(**a)
        with pytest.raises(RuntimeError, match="bad kernel arguments"):
            ops.check_status()
        assert (a["k_cache"][:, :, 1:] == 0).all() and a["k_cache"][0, :, 0].any()


def attention_args(device, B=2, D=64, KV=2, G=2):
    to = lambda t: t.to(device)  # noqa: E731
    return dict(q=to(torch.randn(B, KV * G * D).to(BF16)), k_cache=to(random_cache(4, KV, 32, D)), v_cache=to(random_cache(4, KV, 32, D)),
                block_tables=to(torch.tensor([[1, 2], [3, 0]], dtype=torch.int32)), ctx_lens=to(torch.tensor([40, 5], dtype=torch.int32)), H=KV * G, scale=0.1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", [dict(H=3), dict(H=8), dict(window=-1), dict(softcap=-1.0), dict(block_tables=torch.int64), dict(ctx_lens=slice(0, 1)), dict(block_tables=slice(0, 1)),
                                    dict(k_cache=slice(0, 3)), dict(v_cache=torch.int8)])
def test_decode_refuses(device, change):
    a = attention_args(device)
    for name, c in change.items():
        t = a.get(name)
        a[name] = t[c] if isinstance(c, slice) else t.to(c) if isinstance(c, torch.dtype) else c
    with pytest.raises((ValueError, RuntimeError)):
        decode_attention4(**a)
    done(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", [dict(block_tables=[[1, 9], [3, 0]]), dict(block_tables=[[1, -2], [3, 0]]), dict(ctx_lens=[65, 5]), dict(ctx_lens=[40, -1])])
def test_decode_reports_bad_tables(device, change):
    a = attention_args(device)
    for name, c in change.items():
        a[name] = torch.tensor(c, dtype=torch.int32, device=device)
    if device == "cpu":
        with pytest.raises((ValueError, IndexError)):
            decode_attention4(**a)
    else:
        assert decode_attention4(**a).shape == a["q"].shape
        with pytest.raises(RuntimeError, match="bad kernel arguments"):
            ops.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_expand_reports_pages_outside(device):
    k = random_cache(3, 1, 32, 64).to(device)
    for pages in ([0, 3], [-1]):
        pages = torch.tensor(pages, dtype=torch.int32, device=device)
        if device == "cpu":
            with pytest.raises(IndexError):
                expand4(k, k, pages)
        else:
            expand4(k, k, pages)
            with pytest.raises(RuntimeError, match="bad kernel arguments"):
                ops.check_status()
    with pytest.raises(ValueError):
        expand4(k, k, torch.zeros(1, dtype=torch.int32, device=device), torch.float64)


@pytest.mark.parametrize("device", GPU)
def test_prefill_reports(device):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    a = attention_args(device)
    q, rest = torch.randn(4, 256, device=device).to(BF16), (a["k_cache"], a["v_cache"])
    run = lambda table, news, lens, **kw: prefill_attention4(q, *rest, i32(table), i32([0, 3]), i32(news), i32(lens), 4, 0.1, **kw)  # noqa: E731
    with pytest.raises(ValueError):
        run([[1, 2], [3, 0]], [3, 2], [40, 5])
    with pytest.raises(ValueError):
        run([[1, 2], [3, 0]], [3, 1], [2, 5])
    run([[1, 7], [3, 0]], [3, 1], [40, 5])
    with pytest.raises(RuntimeError, match="bad kernel arguments"):
        ops.check_status()
    with pytest.raises(ValueError):
        run([[1, 2], [3, 0]], [3, 1], [70, 5])
    with pytest.raises(ValueError):
        prefill_attention4(q, *rest, i32([[1, 2], [3, 0]]), i32([0, 3]), i32([3, 1]), i32([40, 5]), 4, -0.1)
    run([[1, 2], [3, 0]], [3, 1], [40, 5], ctx_len_host=[30, 5])  # (one page where the device's lengths have two)
    with pytest.raises(RuntimeError, match="bad kernel arguments"):
        ops.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_operators_together(device):
    """Two prompts, one behind a cached prefix, then three decode steps: tables, write, attention, as a layer uses them; the attention against 64 bits over what the cache holds."""
    D, H, KV, page = 128, 8, 2, 32
    tol = lambda want, mass, reach: want.abs() * HALF_STEP + mass * (2.0**-10 + reach * 2.0**-16) + 1e-30  # noqa: E731
    to = lambda t: t.to(device)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    cos, sin = (to(t) for t in rotary(None, 32, 400))
    qn, kn = to(torch.randn(D).to(BF16)), to(torch.randn(D).to(BF16))
    kc, vc = to(random_cache(12, KV, page, D)), to(random_cache(12, KV, page, D, False))
    pages = [[3, 7, 1, 9, 4], [2, 11, 5]]
    cached, flat, first = [40, 0], i32(pages[0] + pages[1]), i32([0, 5, 8])
    for new in ([77, 50], [1, 1], [1, 1], [1, 1]):
        T = sum(new)
        t = step_tables(flat, first, i32(cached), i32(cached), i32(new), T, 6, page, 64, sum(-(-n // 64) for n in new))
        qkv = to(torch.randn(T, (H + 2 * KV) * D).to(BF16))
        q = rope_kv4(qkv, t.positions, t.slots, qn, kn, cos, sin, kc, vc, H, KV, D, 1e-6)
        if T > 2:
            got = prefill_attention4(q, kc, vc, t.block_tables, t.q_start, i32(new), t.ctx_len, H, D**-0.5)
        else:
            got = decode_attention4(q, kc, vc, t.block_tables, t.ctx_len, H, D**-0.5)
        done(device)
        lens = [a + b for a, b in zip(cached, new)]
        values = (lambda x: ref.kv4_unpack(x, torch.float16)) if device == "cuda" and T > 2 else ref.kv4_unpack
        want, mass, reach = plain_attention(q.cpu(), kc.cpu(), vc.cpu(), t.block_tables.cpu(), lens, new, KV, D**-0.5, 0.0, 0, values)
        assert ((got.cpu().double() - want).abs() <= tol(want, mass, reach)).all()
        v_new = qkv.view(T, H + 2 * KV, D)[:, H + KV :].cpu()
        held = vc.cpu().transpose(1, 2).flatten(0, 1)[t.slots.cpu()]
        assert torch.equal(held, ref.kv4_pack(v_new))
        cached = lens


@pytest.mark.parametrize("device", GPU)
def test_outputs_stay_inside_their_guard_areas(device):
    ops.set_bounds_check(True)
    try:
        for D, KV, G, lens in ((64, 2, 5, [700, 31, 32, 0]), (128, 1, 16, [64] * 40), (256, 2, 1, [5000])):
            run_decode(device, D, KV, G, lens)
        run_prefill(device, 64, 2, 3, [33, 5], [0, 70])
        run_prefill(device, 128, 1, 2, [5], [3], page=96)
        run_prefill(device, 128, 1, 2, [5], [3000])
        test_expand_matches_plain(device, 128, 1, 96)
        test_step_tables(device, [5, 0, 0, 129, 0], 64, 32)
        test_write_matches_plain(device, 128, 6, 2, 37, "halves", 64, True)
        test_write_matches_plain(device, 64, 4, 1, 9, "halves", 5, True)
        torch.cuda.synchronize()
        ops.check_guards()
    finally:
        ops.set_bounds_check(False)


# ---------------------------------------------------------------------------------------------------------------- engine
HEADS = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64)


def tiny_model(tmp, device="cpu", family="llama", **over):
    from deliverance_b200.ckpt.loader import WeightLoader
    from deliverance_b200.ckpt.tiny import write_tiny_model
    from deliverance_b200.config import load_config
    from deliverance_b200.models.transformer import DecoderModel

    d = str(tmp / f"{family}_{device}_{len(list(tmp.iterdir()))}")
    write_tiny_model(d, family, seed=5, std=0.25, **over)
    return DecoderModel(load_config(d), device).load(WeightLoader(d))


def engine_of(model, bits=4, pages=256, **kw):
    from deliverance_b200.engine.engine import Engine, EngineConfig
    from deliverance_b200.kv.paged import KvCacheSettings

    kv = KvCacheSettings(bits=bits, **kw.pop("kv", {}))
    e = Engine(model, EngineConfig(num_pages=pages, max_batch_tokens=kw.pop("max_batch_tokens", 64), max_seqs=kw.pop("max_seqs", 8), kv=kv, **kw))
    e.eos_ids = frozenset()
    return e


def params_of(n, **kw):
    from deliverance_b200.params import GeneratorParameters

    return GeneratorParameters(max_tokens=n, **kw)


def prompt_of(n, k=0):
    return [(7 * i * i + 3 * i + 11 + k) % 200 + 3 for i in range(n)]


def plain_greedy(model, prompt, steps, held):
    """Greedy decoding token by token in fp64; ``held``: what the cache makes of a key or value."""
    c = model.cfg
    H, KV, D = c.num_heads, c.num_kv_heads, c.head_dim
    cos, sin = model.cos.double(), model.sin.double()
    rows = [[[[], []] for _ in range(KV)] for _ in model.layers]
    norm = lambda x, w: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + c.norm_eps) * w.double()  # noqa: E731

    def rotate(x, pos):
        a, b = x[..., : D // 2], x[..., D // 2 :]
        return torch.cat([a * cos[pos] - b * sin[pos], b * cos[pos] + a * sin[pos]], -1)

    def feed(token, pos):
        h = model.embed[token].double()
        for i, lw in enumerate(model.layers):
            qkv = lw.qkv.w.double() @ norm(h, lw.input_norm)
            q, k, v = qkv[: H * D].view(KV, H // KV, D), qkv[H * D : (H + KV) * D].view(KV, D), qkv[(H + KV) * D :].view(KV, D)
            if lw.q_norm is not None:
                q, k = norm(q, lw.q_norm), norm(k, lw.k_norm)
            q, k, out = rotate(q, pos), rotate(k, pos), []
            for j in range(KV):
                ks, vs = rows[i][j]
                ks.append(held(k[j])), vs.append(held(v[j]))
                out.append(torch.softmax(q[j] @ torch.stack(ks).T * c.scale, -1) @ torch.stack(vs))
            h = h + lw.o.w.double() @ torch.stack(out).flatten()
            g, u = (lw.gate_up.w.double() @ norm(h, lw.pre_ff_norm)).chunk(2)
            h = h + lw.down.w.double() @ (torch.nn.functional.silu(g) * u)
        return model.lm_head.w.double() @ norm(h, model.final_norm)

    for pos, token in enumerate(prompt):
        z = feed(token, pos)
    tokens = [int(z.argmax())]
    while len(tokens) < steps:
        z = feed(tokens[-1], len(prompt) + len(tokens) - 1)
        tokens.append(int(z.argmax()))
    return tokens


@pytest.mark.parametrize("family,n,steps", [("llama", 10, 40), ("llama", 100, 20), ("qwen3", 40, 30)])
def test_engine_matches_plain(tmp_path, family, n, steps):
    model = tiny_model(tmp_path, family=family, **HEADS)
    held = lambda x: ref.kv4_unpack(ref.kv4_pack(x.float())).double()  # noqa: E731
    want = plain_greedy(model, prompt_of(n), steps, held)
    e = engine_of(model)
    assert e.generate(prompt_of(n), params_of(steps)).token_ids == want
    e.kv.audit([])
    assert want != plain_greedy(model, prompt_of(n), steps, lambda x: x), "the cache's rounding changed nothing: the comparison would prove little"


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("family,over", [("llama", {}), ("qwen3", {}), ("gemma2", {}), ("qwen3", dict(hidden_size=512, head_dim=128)), ("llama", dict(num_attention_heads=16, num_key_value_heads=1, hidden_size=1024))])
def test_engine_schedules_agree(tmp_path, device, family, over):
    """Sequences answer the same alone and together, with prompts whole and in portions, from cached prefixes, and after a preemption."""
    model = tiny_model(tmp_path, device, family, **{**HEADS, **over})
    prompts = [prompt_of(n, k) for k, n in enumerate((70, 5, 33, 90))]
    one = [engine_of(model, max_batch_tokens=4096).generate(p, params_of(60)).token_ids for p in prompts]
    if device == "cpu":  # (on a GPU products of other shapes round otherwise; there the rows of one schedule are compared below)
        e = engine_of(model, max_batch_tokens=32)
        assert [r.token_ids for r in e.generate_batch(prompts, params_of(60))] == one
        e = engine_of(model, pages=12)
        assert [r.token_ids for r in e.generate_batch(prompts, params_of(60))] == one and e.metrics.get("preemptions", 0) > 0
        e.kv.audit([])
    e = engine_of(model, max_batch_tokens=4096)
    first = e.generate(prompts[3], params_of(60))
    again = e.generate(prompts[3], params_of(60))
    assert first.token_ids == one[3] and again.prefix_hit_tokens > 0
    if device == "cpu":
        assert again.token_ids == one[3]
    assert len(e.kv.k[0].shape) == 4 and e.kv.k[0].dtype == torch.uint8 and e.kv.k[0].shape[3] == row_bytes(model.cfg.head_dim)
    done(device)


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("family,over", [("llama", {}), ("qwen3", dict(hidden_size=512, head_dim=128)), ("gemma2", {})])
def test_engine_captured_steps_agree(tmp_path, device, family, over):
    """Decode steps from captured graphs, with and without lookahead, and launched one by one give the same tokens: the attention's shares depend on the lengths alone."""
    model = tiny_model(tmp_path, device, family, **{**HEADS, **over})
    prompts = [prompt_of(n, k) for k, n in enumerate((70, 5, 33))]
    got = [[r.token_ids for r in engine_of(model, **kw).generate_batch(prompts, params_of(40))] for kw in ({}, {"lookahead": False}, {"cuda_graphs": False, "lookahead": False})]
    assert got[0] == got[1]
    assert [len(x) for x in got[2]] == [40, 40, 40]
    done(device)


@pytest.mark.parametrize("device", GPU)
def test_engine_steps_match_prompts(tmp_path, device):
    """Logits of a decode step against those of the same tokens as one prompt: the cache holds the same rows up to steps that fall otherwise, because projections of one row and of many round otherwise."""
    model = tiny_model(tmp_path, device, "qwen3", **{**HEADS, "hidden_size": 512, "head_dim": 128})
    e = engine_of(model, max_batch_tokens=4096, kv={"enabled": False})
    tokens = prompt_of(80)
    a, b = e.open_replay(), e.open_replay()
    whole = e.replay_step([(a, tokens, list(range(80)))])
    parts = [e.replay_step([(b, tokens[:40], list(range(40)))])]
    parts += [e.replay_step([(b, [t], [0])]) for t in tokens[40:]]
    parts = torch.cat(parts)
    # bf16 activations differ by roundings between the two, and codes in some places by one step: the logits by a few per cent of their spread
    err, spread = (whole - parts).double().square().mean().sqrt(), whole.double().std()
    assert err < 0.1 * spread
    assert torch.equal(whole[:1], parts[:1]) or err < 0.1 * spread


@pytest.mark.parametrize("device", DEVICES)
def test_engine_beams(tmp_path, device):
    model = tiny_model(tmp_path, device, "llama", **HEADS)
    e = engine_of(model)
    best = e.generate(prompt_of(37), params_of(12, num_beams=3))
    assert len(best.token_ids) == 12
    e.kv.audit([])
    if device == "cpu":
        assert e.generate(prompt_of(37), params_of(12, num_beams=1)).token_ids == engine_of(model).generate(prompt_of(37), params_of(12)).token_ids
    done(device)


def test_engine_disk_tier(tmp_path):
    model = tiny_model(tmp_path, **HEADS)
    prompt = prompt_of(70)
    for compression in ("NONE", "LZ4"):
        e = engine_of(model)
        disk = e.kv.attach_disk(str(tmp_path / compression), compression=compression)
        want = e.generate(prompt, params_of(10)).token_ids
        e.kv.prefix.clear()
        assert disk.metrics["disk_writes"] > 0
        got = e.generate(prompt, params_of(10))
        assert got.token_ids == want and got.prefix_hit_tokens > 0 and disk.metrics["disk_hits"] == 1
        # an engine whose cache has other rows does not find them
        other = engine_of(model, bits=16)
        other.kv.attach_disk(str(tmp_path / compression), compression=compression)
        assert other.generate(prompt, params_of(10)).prefix_hit_tokens == 0
    with pytest.raises(ValueError):
        engine_of(model).kv.attach_disk(str(tmp_path / "x"), compression="MSE_TURBOQUANT")


def test_engine_refuses(tmp_path):
    from deliverance_b200.api import AutoModelForCausalLM
    from deliverance_b200.ckpt.tiny import write_tiny_model
    from deliverance_b200.kv.paged import KvCacheSettings, PagedKVCache

    model = tiny_model(tmp_path, **HEADS)
    for kw in (dict(bits=8), dict(kv=dict(keep_tokens=64))):
        with pytest.raises(ValueError):
            engine_of(model, **kw)
    for family in ("gpt2", "fatotar"):
        d = str(tmp_path / family)
        write_tiny_model(d, family, seed=5)
        with pytest.raises(ValueError, match="4 bits"):
            AutoModelForCausalLM.new_builder(d).with_device("cpu").with_kv_cache_settings(KvCacheSettings(bits=4)).build()
    with pytest.raises(ValueError):
        engine_of(tiny_model(tmp_path, hidden_size=64, num_attention_heads=4, num_key_value_heads=2, head_dim=16))
    layout = model.kv_layout()
    assert PagedKVCache.bytes_per_page(layout, 32, torch.bfloat16) * 5 == PagedKVCache.bytes_per_page(layout, 32, torch.bfloat16, 4) * 16
    with pytest.raises(ValueError):
        PagedKVCache.bytes_per_page(dict(layout, head_dim=80), 32, torch.bfloat16, 4)


def test_server_key(tmp_path):
    from deliverance_b200.server.config import load_server_config

    p = tmp_path / "x.properties"
    p.write_text("deliverance.kv.bits=4\n")
    assert load_server_config(str(p)).kv_settings().bits == 4


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("kind", ["prompts", "decode", "mixed", "one"])
def test_batches_made_there(device, kind):
    """A batch whose tables a kernel makes is the host's, field by field."""
    from deliverance_b200.models.batch import make_batch

    new = {"prompts": [100, 1, 17, 300], "decode": [1] * 9, "mixed": [1, 1, 40], "one": [1]}[kind]
    seqs, page = [], 1
    for i, n in enumerate(new):
        start = int(torch.randint(0, 90, ()))
        held = -(-(start + n) // 32) + i % 2
        seqs.append({"tokens": torch.randint(0, 999, (n,)).tolist(), "start": start + 5 * i, "cached": start, "pages": list(range(page, page + held)), "prev": i - 1, "state_slot": i, "key_slot": i + 1})
        page += held
    for width in (None, 40):
        a, b = make_batch(seqs, 32, "cpu", width), make_batch(seqs, 32, device, width)
        done(device)
        for name in ("token_ids", "positions", "slots", "q_start", "q_len", "ctx_len", "block_tables", "logits_rows", "tile_seq", "tile_q0", "state_slots", "prev_ids", "key_slots"):
            x, y = getattr(a, name), getattr(b, name)
            assert (x is None) == (y is None), name
            if x is not None:
                assert y.is_cuda and x.dtype == y.dtype and torch.equal(x, y.cpu()), name
        for name in ("is_decode", "decode_even", "q_len_host", "ctx_len_host"):
            assert getattr(a, name) == getattr(b, name)
        assert a.rows_apart() == b.rows_apart() if a.is_decode else b.host_tables is None
    with pytest.raises(ValueError):
        make_batch([dict(seqs[0], pages=[])], 32, device)


# ---------------------------------------------------------------------------------------------------------------- ends of the operators
PARTS = """
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>
#include "kv4_parts.h"
using namespace dlv;
int main() {
  srand(7);
  for (int round = 0; round < 4000; ++round) {
    const int KV = 1 + rand() % 8, B = 1 + rand() % 40, ctas = 1 + rand() % (round % 3 ? 12 : 1024), workers = ctas * kKv4Warps, near = rand() % 9, pairs = B * KV;
    std::vector<int> n(B), front(B + 1, 0);
    for (int b = 0; b < B; ++b) {
      n[b] = rand() % 4 ? rand() % (round % 2 ? 9 : 400) : 0;
      front[b + 1] = front[b] + n[b];
    }
    const Kv4Shares shares(front[B] * KV, workers);
    const long long room = kv4_decode_parts(ctas, pairs, near);
    std::set<long long> places;
    for (int pair = 0; pair < pairs; ++pair) {
      const int b = pair / KV, h = pair % KV;
      const Kv4Parts p(shares, front[b] * KV + h * n[b], n[b]);
      if (n[b] == 0 && p.parts != 0) return 1;
      const bool whole = p.parts == 1 && !p.j0;  // seen whole by one warp, which writes the result and no part
      for (int i = 0; i < p.parts && !whole; ++i) {  // every part has a place of its own
        const long long at = kv4_place(pairs, near, pair, i, p.maker(i));
        if (at < 0 || at >= room || !places.insert(at).second) return 2;
      }
      const int counts[] = {p.parts, 0, -1, 1, near + 1, 1 << 30, 0x7fffffff, 0x3f800000, -0x7fffffff - 1};
      for (int count : counts) {  // what the second launch reads, whatever stands where the count should be
        for (int i = 0; i < near; ++i)
          if (kv4_place(pairs, near, pair, i, 0) >= room) return 3;
        for (int i = count < near ? count : near; i >= 0 && i < p.most(count); ++i) {
          const long long at = kv4_place(pairs, near, pair, i, p.maker(i));
          if (at < 0 || at >= room) return 4;
        }
      }
      if (p.most(p.parts) != p.parts) return 5;
    }
  }
  puts("ok");
}
"""


def test_decode_parts_stay_in_their_workspace(tmp_path):
    """The places of partial results, from the header that the kernels use: different ones, and inside the workspace even for a count that no warp has written."""
    import os
    import shutil
    import subprocess

    from deliverance_b200.ops import build

    if shutil.which("g++") is None:
        pytest.skip("no g++")
    (tmp_path / "parts.cpp").write_text(PARTS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", build.CSRC, str(tmp_path / "parts.cpp"), "-o", str(tmp_path / "parts")], check=True, timeout=120)
    assert subprocess.run([str(tmp_path / "parts")], capture_output=True, text=True, timeout=120, env=dict(os.environ)).stdout == "ok\n"


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("D,news,befores", [(64, [3, 200], [90, 40]), (128, [150, 7], [3000, 10]), (256, [2, 2], [10, 30])])
def test_prefill_reports_other_lengths(device, D, news, befores):
    """Lengths on the device that are not the host's, beyond the tables and below zero, are reported; the kernels stay inside tables and rows, and the next call is as good as any."""
    KV, H, page, lens = 2, 4, 32, [a + b for a, b in zip(news, befores)]
    table, pages = tables_for(lens, page)
    k, v = random_cache(pages, KV, page, D, False).to(device), random_cache(pages, KV, page, D, False).to(device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q, start, width = torch.randn(sum(news), H * D, device=device).to(BF16), [0, news[0]], table.shape[1]
    call = lambda ctx, new=news: prefill_attention4(q, k, v, table.to(device), i32(start), i32(new), i32(ctx), H, D**-0.5, q_len_host=news, ctx_len_host=lens)  # noqa: E731
    want = call(lens)
    done(device)
    ops.set_bounds_check(True)
    try:
        for ctx in ([lens[0], width * page + 999], [2**31 - 1, lens[1]], [-5, lens[1]], [0, 0], [lens[0], -(2**31)]):
            call(ctx)
            with pytest.raises(RuntimeError, match="bad kernel arguments"):
                ops.check_status()
        for new in ([news[0], news[1] + 4000], [lens[0] + 1, news[1]], [-1, news[1]], [news[0], 2**31 - 1]):
            call(lens, new)
            with pytest.raises(RuntimeError, match="bad kernel arguments"):
                ops.check_status()
        torch.cuda.synchronize()
        ops.check_guards()
    finally:
        ops.set_bounds_check(False)
    assert torch.equal(call(lens), want)
    done(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,KV,G,lens,first,count", [
    (128, 2, 2, [4000], 64, 512), (128, 2, 2, [4000], 3968, 32), (128, 2, 2, [4000], 0, 4000), (64, 1, 3, [20000], 4096, 2048),  # one sequence, cut into many shares
    (128, 2, 2, [4000], 256, 256), (128, 8, 4, [2176] * 64, 0, 128), (128, 8, 4, [2176] * 64, 0, 384), (128, 8, 4, [2176] * 64, 1792, 384), (128, 8, 4, [2176] * 64, 0, 544), (128, 8, 4, [2176] * 64, 1088, 1088), (64, 4, 8, [3000, 100] * 8, 512, 1024), (256, 2, 12, [3000, 7, 900] * 4, 64, 800),  # many pairs
])
@pytest.mark.parametrize("cache", ["keys", "values"])
def test_decode_keeps_nan_whatever_the_shares(device, D, KV, G, lens, first, count, cache):
    """Runs of rows without a number, long enough for whole shares of the work to hold nothing else: the heads that see them are NaN, all others are what they are without them."""
    if device == "cpu" and sum(lens) * KV * G * D > 5e7:
        pytest.skip("large for the CPU")
    table, pages = tables_for(lens, 32)
    H, q = KV * G, torch.randn(len(lens), KV * G * D).to(BF16)
    k, v = random_cache(pages, KV, 32, D), random_cache(pages, KV, 32, D, False)
    to = lambda t: t.to(device)  # noqa: E731
    call = lambda: decode_attention4(to(q), to(k), to(v), to(table), to(torch.tensor(lens, dtype=torch.int32)), H, D**-0.5).cpu().view(len(lens), KV, G * D)  # noqa: E731
    clean = call()
    hit = [b for b, n in enumerate(lens) if b % 3 == 0 and first + count <= n]
    for b in hit:
        for j in range(first, first + count):
            (k if cache == "keys" else v)[table[b, j // 32].long(), KV - 1, j % 32, D // 2 :] = 0x7E  # (steps and minima that are no numbers)
    got = call()
    done(device)
    bad = torch.zeros(len(lens), KV, dtype=torch.bool)
    bad[hit, KV - 1] = True
    assert hit and got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,news,befores,softcap", [(64, [70, 3], [100, 0], 0.0), (128, [5], [2000], 0.0), (256, [40], [9], 30.0)])
def test_prefill_of_zero_rows_at_small_scales(device, D, news, befores, softcap):
    """Query rows of zeros, and scales that take scores below the smallest numbers: every visible key counts alike, those that are not visible not at all."""
    KV, H, page, lens = 2, 4, 32, [a + b for a, b in zip(news, befores)]
    table, pages = tables_for(lens, page)
    k, v = random_cache(pages, KV, page, D, False), random_cache(pages, KV, page, D, False)
    to, i32 = lambda t: t.to(device), lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q = torch.randn(sum(news), H, D)
    q[:, ::2] = 0.0
    q = q.flatten(1).to(BF16)
    for scale in (1e-8, 1e-20, 1e-37):
        got = prefill_attention4(to(q), to(k), to(v), to(table), i32([0, news[0]][: len(news)]), i32(news), i32(lens), H, scale, softcap).cpu().double()
        done(device)
        want, mass, _ = plain_attention(q, k, v, table, lens, news, KV, scale, softcap, 0)
        # the result's rounding, values and probabilities in fp16 (half a step each; numerator and denominator)
        assert ((got - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-11 + 2.0**-10) + 2.0**-24).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,news,befores,window,page", [(64, [70, 1], [200, 300], 40, 32), (128, [5], [2000], 100, 96), (128, [20, 0, 33], [700, 40, 0], 7, 64), (256, [150], [333], 64, 32), (64, [300], [1000], 1, 32)])
def test_prefill_in_front_of_a_window(device, D, news, befores, window, page):
    """What stands in rows that no query row's window reaches does not matter, not even infinities and NaN."""
    KV, H, lens = 2, 6, [a + b for a, b in zip(news, befores)]
    table, pages = tables_for(lens, page)
    k, v = random_cache(pages, KV, page, D, False), random_cache(pages, KV, page, D, False)
    to, i32 = lambda t: t.to(device), lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q, start = torch.randn(sum(news), H * D).to(BF16), [sum(news[:i]) for i in range(len(news))]
    call = lambda: prefill_attention4(to(q), to(k), to(v), to(table), i32(start), i32(news), i32(lens), H, D**-0.5, 0.0, window).cpu()  # noqa: E731
    clean = call()
    want, mass, reach = plain_attention(q, k, v, table, lens, news, KV, D**-0.5, 0.0, window)
    # the result's rounding; keys, values and probabilities in fp16 (a key's half step reaches the exponent; numerator and denominator)
    assert ((clean.double() - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + 2.0**-11 + reach * (2.0**-10 + 2.0**-16)) + 2.0**-24).all()
    for b, (n, m) in enumerate(zip(lens, news)):
        for j in range(n - m + 1 - window if m else n):
            k[table[b, j // page].long(), :, j % page] = v[table[b, j // page].long(), :, j % page] = 0x7D if j % 2 else 0xFE
    assert torch.equal(call(), clean)
    done(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [1, 4])
def test_prefill_takes_query_rows_as_they_lie(device, rows):
    """Rows of any distance (none: the same row again) and alignment, a single one too."""
    KV, H, D, page = 2, 4, 64, 32
    table, pages = tables_for([40 + rows], page)
    to, i32 = lambda t: t.to(device), lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    k, v = to(random_cache(pages, KV, page, D)), to(random_cache(pages, KV, page, D, False))
    wide = to(torch.randn(rows, H * D + 3).to(BF16))
    call = lambda q: prefill_attention4(q, k, v, to(table), i32([0]), i32([rows]), i32([40 + rows]), H, 0.1)  # noqa: E731
    same = wide[:1, : H * D].contiguous()
    for q in (wide[:, : H * D], wide[:, 1 : 1 + H * D], same.expand(rows, -1), torch.randn(H * D, rows, device=device).to(BF16).t()):
        assert torch.equal(call(q), call(q.clone(memory_format=torch.contiguous_format)))
    done(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", [dict(ctx_lens=[70, 5]), dict(ctx_lens=[2, 5]), dict(ctx_lens=[40, -1]), dict(q_len=[3, 2]), dict(q_len=[5, -1]), dict(ctx_lens=[40, 5, 5]), dict(block_tables=[[1, 2]]),
                                    dict(block_tables=torch.int64), dict(ctx_lens=torch.int64), dict(H=3), dict(H=8), dict(window=-1), dict(softcap=-1.0), dict(scale=0.0), dict(scale=math.nan), dict(k_cache=slice(0, 3))])
def test_prefill_refuses(device, change):
    """The same calls on the CPU and on a GPU, before anything is computed."""
    a = attention_args(device, B=4)
    a.update(q_start=torch.tensor([0, 3], dtype=torch.int32, device=device), q_len=torch.tensor([3, 1], dtype=torch.int32, device=device))
    assert prefill_attention4(**a).shape == a["q"].shape
    for name, c in change.items():
        a[name] = a[name].to(c) if isinstance(c, torch.dtype) else a[name][c] if isinstance(c, slice) else torch.tensor(c, dtype=torch.int32, device=device) if isinstance(c, list) else c
    with pytest.raises((ValueError, RuntimeError)):
        prefill_attention4(**a)
    done(device)


def test_prefill_raises_on_the_cpu():
    a = attention_args("cpu", B=4)
    a.update(q_start=torch.tensor([0, 3], dtype=torch.int32), q_len=torch.tensor([3, 1], dtype=torch.int32))
    for change in (dict(q_len_host=[2, 2]), dict(ctx_len_host=[40, 6]), dict(q_start=torch.tensor([0, 2], dtype=torch.int32))):
        with pytest.raises(ValueError):
            prefill_attention4(**{**a, **change})
    for table in ([[1, 9], [3, 0]], [[1, -2], [3, 0]]):
        with pytest.raises(IndexError):
            prefill_attention4(**{**a, "block_tables": torch.tensor(table, dtype=torch.int32)})


@pytest.mark.parametrize("device", GPU)
def test_prefill_in_portions_captured(device, monkeypatch):
    """Portions take the tiles that the caller has (nothing is copied from the host: such a call can be captured), and their keys in parts where they have few tiles."""
    from deliverance_b200.ops import kv4

    KV, D, H, page, news, befores = 2, 64, 4, 32, [70, 0, 40, 1, 300], [100, 50, 0, 2000, 5]
    lens = [a + b for a, b in zip(news, befores)]
    table, pages = tables_for(lens, page)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    k, v = (random_cache(pages, KV, page, D, False) for _ in range(2))
    start = [sum(news[:i]) for i in range(len(news))]
    args = (k.to(device), v.to(device), table.to(device), i32(start), i32(news), i32(lens), H, 0.1)
    tiles, asked = {rows: tuple(i32(t) for t in ops.prefill_tiles(news, rows)) for rows in (128, 256)}, []
    run = lambda q: prefill_attention4(q, *args, q_len_host=news, ctx_len_host=lens, tiles_for=lambda rows: asked.append(rows) or tiles[rows])  # noqa: E731
    q = torch.randn(sum(news), H * D).to(BF16).to(device)
    monkeypatch.setattr(kv4, "EXPAND_PAGES_BYTES", 20 * KV * page * D * 4)
    seen, rule = [], kv4._parts
    monkeypatch.setattr(kv4, "_parts", lambda *a: seen.append(rule(*a)) or seen[-1])
    run(q)
    torch.cuda.synchronize()
    assert asked and max(seen) > 1 and len(seen) > 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(q)
    for _ in range(2):
        q.copy_(torch.randn(q.shape))
        graph.replay()
        torch.cuda.synchronize()
        want, mass, reach = plain_attention(q.cpu(), k, v, table, lens, news, KV, 0.1, 0.0, 0)
        assert ((out.cpu().double() - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + 2.0**-11 + reach * (2.0**-10 + 2.0**-16)) + 2.0**-24).all()
    done(device)


@pytest.mark.parametrize("compression", ["NONE", "LZ4", "DEFLATE", "MSE_TURBOQUANT"])
def test_snapshots_hold_the_rows_as_they_are(compression):
    from deliverance_b200.kv.paged import KvCacheSettings, PagedKVCache
    from deliverance_b200.kv.turboquant import restore_pages, snapshot_pages

    layout = dict(layer_kinds=["full"] * 2, kv_heads=2, head_dim=64)
    a, b = (PagedKVCache(layout, 8, "cpu", torch.float32, KvCacheSettings(bits=4)) for _ in range(2))
    for t in a.k + a.v:
        t.copy_(random_cache(8, 2, 32, 64))
    if compression == "MSE_TURBOQUANT":  # (a codec for numbers: bytes do not come back)
        with pytest.raises(ValueError, match="4-bit"):
            snapshot_pages(a, [5, 2], 40, compression)
        return
    restore_pages(b, snapshot_pages(a, [5, 2], 40, compression), [3, 7])
    for s, t in zip(a.k + a.v, b.k + b.v):
        assert torch.equal(t[3], s[5]) and torch.equal(t[7, :, :8], s[2, :, :8])


# what else decoders have around their attention: biases, local and global layers, recurrent layers, experts
FAMILIES = [("qwen2", {}), ("gemma3_text", {}), ("mixtral", {}), ("qwen3_moe", {}), ("granitemoehybrid", dict(mamba_n_heads=16))]


def replayed(e, tokens, cuts):
    """Logits of all positions, ``tokens`` fed in portions of the given sizes and the rest one by one."""
    r, out, at = e.open_replay(), [], 0
    for n in list(cuts) + [1] * (len(tokens) - sum(cuts)):
        out.append(e.replay_step([(r, tokens[at : at + n], list(range(n)))]))
        at += n
    return torch.cat(out)


@pytest.mark.parametrize("family,over", FAMILIES)
def test_engine_families(tmp_path, family, over):
    """A prompt whole, in portions, and token by token. (Tokens alone prove nothing here: fp32 sums of other lengths move a number by 2^-23 of its size, which now and then falls on the other side of a code's
    border; a step is a fifteenth of a block's range, and what it moves in the logits is a few per cent of their spread.)"""
    model = tiny_model(tmp_path, family=family, **{**HEADS, **over})
    assert model.supports_kv4()
    e, tokens = engine_of(model, max_batch_tokens=4096, kv={"enabled": False}), prompt_of(110)
    whole, portions, single = (replayed(e, tokens, cuts) for cuts in ([110], [33, 60], [1]))
    assert all(k is None or k.dtype == torch.uint8 for k in e.kv.k)
    rms = lambda x: x.double().square().mean().sqrt()  # noqa: E731
    assert rms(whole - portions) < 0.05 * rms(whole) and rms(whole - single) < 0.05 * rms(whole)
    assert rms(whole - replayed(engine_of(model, 16, max_batch_tokens=4096, kv={"enabled": False}), tokens, [110])) > 1e-3 * rms(whole)  # (fp32 noise is 1e-5)
    e = engine_of(model)
    first = e.generate(prompt_of(90), params_of(12))
    again = e.generate(prompt_of(90), params_of(12))
    assert len(first.token_ids) == 12 and again.prefix_hit_tokens > 0
    e.kv.audit([])


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("family,over", [f for f in FAMILIES if f[0] not in ("mixtral", "qwen3_moe")])
def test_engine_families_match_the_cpu(tmp_path, device, family, over):
    """Logits of a prompt, of a portion behind it and of decode steps against the plain forms in fp32 of the same checkpoint."""
    got, tokens = {}, prompt_of(100)
    for d in ("cpu", device):
        model = tiny_model(tmp_path, d, family, **{**HEADS, **over})
        for bits in (16, 4):
            got[d, bits] = replayed(engine_of(model, bits, max_batch_tokens=4096, kv={"enabled": False}), tokens, [60, 20]).double()
    # A number lies within 7.5 steps s of its block's middle. Rounded to bf16 it is off by up to 7.5 s 2^-8 = 0.03 s, and so are the roundings in front of it: with probability 0.03 or so it gets another code, s away,
    # which makes sqrt(0.03) s = 0.17 s in the mean square, where quantising itself makes s / sqrt(12) = 0.29 s. Hence: off by less than what bf16 makes without codes, and what quantising makes, together.
    err = lambda a, b: (got[a] - got[b]).square().mean(1).sqrt().mean()  # noqa: E731
    assert err((device, 4), ("cpu", 4)) < err((device, 16), ("cpu", 16)) + err(("cpu", 16), ("cpu", 4))
    done(device)


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("family,over", [("llama", {}), ("qwen3", dict(hidden_size=512, head_dim=128)), ("gemma2", {})])
def test_captured_steps_have_the_logits_of_single_launches(tmp_path, device, family, over):
    """The two divide the keys of decode attention otherwise (by the widest block table there can be, and by the batch's own), so that they agree up to roundings, and codes by a step where those decide."""
    model = tiny_model(tmp_path, device, family, **{**HEADS, **over})
    rows = []
    for graphs in (True, False):
        e = engine_of(model, max_batch_tokens=4096, kv={"enabled": False}, cuda_graphs=graphs)
        open_, parts = [e.open_replay() for _ in range(3)], []
        texts = [prompt_of(n + 30, k) for k, n in enumerate((70, 5, 133))]
        e.replay_step([(r, t[:-30], []) for r, t in zip(open_, texts)])
        for i in range(-30, 0):
            parts.append(e.replay_step([(r, [t[i]], [0]) for r, t in zip(open_, texts)]))
        rows.append(torch.stack(parts))
        assert (e.metrics["graph_replays"] > 0) == graphs
    err, spread = (rows[0] - rows[1]).double().square().mean(-1).sqrt(), rows[0].double().std()
    assert err.mean() < 0.05 * spread
    assert (rows[0][:, 0] - rows[1][:, 1]).double().square().mean(-1).sqrt().mean() > 0.5 * spread  # (those of another sequence)
    done(device)


def adapter_of(tmp, model):
    import json
    import os

    from deliverance_b200.ckpt.lora import lora_names
    from deliverance_b200.ckpt.safetensors_io import write_safetensors

    c, tensors = model.cfg, {}
    shapes = {"q_proj": c.num_heads * c.head_dim, "k_proj": c.num_kv_heads * c.head_dim, "v_proj": c.num_kv_heads * c.head_dim}
    for i in range(c.num_layers):
        for proj, n in shapes.items():
            a, b = lora_names(f"model.layers.{i}.self_attn.{proj}.weight")
            tensors[a], tensors[b] = torch.randn(4, model.embed.shape[1]) * 0.2, torch.randn(n, 4) * 0.2
    os.makedirs(tmp)
    write_safetensors(os.path.join(tmp, "adapter_model.safetensors"), tensors)
    with open(os.path.join(tmp, "adapter_config.json"), "w") as f:
        json.dump({"r": 4, "lora_alpha": 8, "target_modules": list(shapes)}, f)
    return tmp


def test_engine_lora(tmp_path):
    """Queries, keys and values with an adapter's share: swapped in, the same as merged into the weights."""
    from deliverance_b200.api import AutoModelForCausalLM
    from deliverance_b200.kv.paged import KvCacheSettings

    model = tiny_model(tmp_path, **HEADS)
    d, settings = str(next(tmp_path.iterdir())), KvCacheSettings(bits=4)
    adapter = adapter_of(str(tmp_path / "adapter"), model)
    build = lambda b: b.with_device("cpu").with_kv_cache_settings(settings).build()  # noqa: E731
    base, merged = build(AutoModelForCausalLM.new_builder(d)), build(AutoModelForCausalLM.new_builder(d).with_lora_adapter(adapter))
    prompt, p = prompt_of(40), params_of(20)
    plain, want = base.generate(prompt, p).token_ids, merged.generate(prompt, p).token_ids
    assert base.engine.kv.bits == merged.engine.kv.bits == 4
    base.activate_lora(base.register_lora(adapter))
    assert base.generate(prompt, p).token_ids == want != plain
    base.activate_lora(None)
    assert base.generate(prompt, p).token_ids == plain


@pytest.mark.parametrize("family", ["llama", "qwen3", "gemma2"])
def test_engine_tensor_parallel(tmp_path, family):
    """Two ranks with a KV head each in 4 bits answer as one with both."""
    import threading

    from deliverance_b200.ckpt.loader import WeightLoader
    from deliverance_b200.config import load_config
    from deliverance_b200.models.transformer import DecoderModel, TensorParallelContext
    from deliverance_b200.parallel.context import InProcessCollectives, InProcessGroup

    one = tiny_model(tmp_path, family=family, **HEADS)
    d = str(next(tmp_path.iterdir()))
    prompts = [prompt_of(40), prompt_of(7, 1)]
    want = [r.token_ids for r in engine_of(one).generate_batch(prompts, params_of(20))]
    group, got = InProcessGroup(2, timeout=60), [None, None]

    def rank(r):
        try:
            model = DecoderModel(load_config(d), "cpu", tp=TensorParallelContext(r, 2, InProcessCollectives(group, r))).load(WeightLoader(d))
            e = engine_of(model)
            assert e.kv.k[0].shape[1] == 1 and e.kv.k[0].dtype == torch.uint8
            got[r] = [x.token_ids for x in e.generate_batch(prompts, params_of(20))]
        except Exception as e:  # noqa: BLE001
            got[r] = e

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert got[0] == got[1] == want, got


@pytest.mark.parametrize("device", GPU)
@pytest.mark.parametrize("D,KV,G,news,befores,softcap", [(64, 2, 3, [33, 5], [2100, 70], 0.0), (128, 8, 4, [257, 500], [40, 0], 0.0), (128, 1, 4, [130, 1, 64], [3, 4031, 0], 30.0), (256, 2, 1, [70, 300], [0, 900], 0.0)])
def test_prefill_against_what_the_cache_holds(device, D, KV, G, news, befores, softcap):
    """Against 64 bits over the cached values themselves: fp16 keys and values count as the kernels' errors."""
    lens, H = [a + b for a, b in zip(news, befores)], KV * G
    table, pages = tables_for(lens, 32)
    k, v = random_cache(pages, KV, 32, D), random_cache(pages, KV, 32, D, False)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q, start = torch.randn(sum(news), H * D).to(BF16), [sum(news[:i]) for i in range(len(news))]
    got = prefill_attention4(q.to(device), k.to(device), v.to(device), table.to(device), i32(start), i32(news), i32(lens), H, D**-0.5, softcap).cpu().double()
    done(device)
    want, mass, reach = plain_attention(q, k, v, table, lens, news, KV, D**-0.5, softcap, 0)
    # the result in bf16; probabilities and values in fp16 (half a step each, 2^-11; probabilities in numerator and denominator); a key in fp16 moves its score by 2^-11 of sum |q| |k| (numerator and denominator), fp32 sums as in decoding
    assert ((got - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + 2.0**-11 + reach * (2.0**-10 + 2.0**-16)) + 2.0**-24).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,news,befores", [(64, [70, 3], [100, 0]), (128, [5], [2000]), (256, [130, 1], [9, 0])])
def test_prefill_that_is_not_causal(device, D, news, befores):
    KV, H, page, lens = 2, 4, 32, [a + b for a, b in zip(news, befores)]
    table, pages = tables_for(lens, page)
    k, v = random_cache(pages, KV, page, D), random_cache(pages, KV, page, D, False)
    to, i32 = lambda t: t.to(device), lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    q = torch.randn(sum(news), H * D).to(BF16)
    got = prefill_attention4(to(q), to(k), to(v), to(table), i32([0, news[0]][: len(news)]), i32(news), i32(lens), H, D**-0.5, causal=False).cpu().double()
    done(device)
    # every query row sees all keys, as the last row of its sequence does
    seq = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news))
    want, mass, reach = plain_attention(q, k, v, table[seq], [lens[b] for b in seq.tolist()], [1] * len(seq), KV, D**-0.5, 0.0, 0)
    assert ((got - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + 2.0**-11 + reach * (2.0**-10 + 2.0**-16)) + 2.0**-24).all()


@pytest.mark.parametrize("device", GPU)
def test_caches_beyond_32_bits(device):
    """Rows whose bytes lie more than 2^32 behind the first ones: write, decode and prompt attention, unpacking."""
    D, H, KV, page, lens = 128, 16, 8, 32, [90, 33]
    pages = 2**32 // (KV * page * row_bytes(D)) + 40
    kc, vc = (torch.zeros(pages, KV, page, row_bytes(D), dtype=torch.uint8, device=device) for _ in range(2))
    far = [[pages - 1, pages - 7, pages - 3], [pages - 2, pages - 9]]
    table = torch.tensor([far[0], far[1] + [0]], dtype=torch.int32)
    slots = torch.tensor([far[b][j // page] * page + j % page for b, n in enumerate(lens) for j in range(n)])
    T, at = sum(lens), [0, lens[0]]
    x, i32 = torch.randn(T, (H + 2 * KV) * D).to(BF16), lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    q = rope_kv4(x.to(device), torch.zeros(T, dtype=torch.int32, device=device), slots.to(device), None, None, None, None, kc, vc, H, KV, D, 1e-6).cpu()
    done(device)
    assert torch.equal(q, x[:, : H * D]) and not kc[: pages - 9].any() and not vc[: pages - 9].any()
    k, v = kc[pages - 9 :].cpu(), vc[pages - 9 :].cpu()
    near = torch.where(table > 0, table - (pages - 9), 0)
    for cache, cols in ((k, x.view(T, -1, D)[:, H : H + KV]), (v, x.view(T, -1, D)[:, H + KV :])):
        rows = torch.cat([cache[near[b].long()].transpose(1, 2).flatten(0, 1)[:n] for b, n in enumerate(lens)])
        assert torch.equal(rows, ref.kv4_pack(cols))
    whole = prefill_attention4(q.to(device), kc, vc, table.to(device), i32(at), i32(lens), i32(lens), H, D**-0.5).cpu().double()
    want, mass, reach = plain_attention(q, k, v, near, lens, lens, KV, D**-0.5, 0.0, 0)
    assert ((whole - want).abs() <= want.abs() * HALF_STEP + mass * (2.0**-10 + 2.0**-11 + reach * (2.0**-10 + 2.0**-16)) + 2.0**-24).all()
    last = q[[lens[0] - 1, T - 1]]
    got = decode_attention4(last.to(device), kc, vc, table.to(device), i32(lens), H, D**-0.5)
    check_decode(got, last, k, v, near, lens, KV, D**-0.5, 0.0, 0)
    for a, b in zip(expand4(kc, vc, i32([pages - 1, pages - 9]), torch.float32), (k, v)):
        assert torch.equal(a.cpu(), ref.kv4_unpack(b[[8, 0]]))
    done(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,KV", [(1, 1), (3, 2), (50, 4), (600, 8)])
def test_decode_without_keys(device, B, KV):
    k = random_cache(3, KV, 32, 64).to(device)
    q = torch.randn(B, KV * 2 * 64, device=device).to(BF16)
    zero = torch.zeros(B, dtype=torch.int32, device=device)
    assert (decode_attention4(q, k, k, torch.zeros(B, 9, dtype=torch.int32, device=device), zero, KV * 2, 0.1) == 0).all()
    assert decode_attention4(q[:0], k, k, torch.zeros(0, 9, dtype=torch.int32, device=device), zero[:0], KV * 2, 0.1).shape == (0, KV * 128)
    done(device)


@pytest.mark.parametrize("device", GPU)
def test_batches_made_there_of_odd_entries(device):
    """Entries without tokens, tokens in a tensor, pages in reserve, many sequences: the host's batch, field by field."""
    from deliverance_b200.models.batch import make_batch

    one = lambda n, start, pages, **kw: {"tokens": [(7 * i) % 99 for i in range(n)], "start": start, "pages": pages, **kw}  # noqa: E731
    cases = [
        [one(0, 5, [3]), one(4, 0, [9, 2])],
        [one(0, 0, []), one(0, 0, [])],
        [one(3, 0, [1])] * 9000,  # (more than the kernel takes: made on the host)
        [one(2, 62, [4, 5, 6, 7, 8]), one(1, 0, [1])] * 2000,
        [dict(one(0, 0, [2, 3]), tokens=torch.arange(40, dtype=torch.int64)), dict(one(0, 7, [5], cached=3), tokens=torch.tensor([8, 9]))],
    ]
    for seqs in cases:
        a, b = make_batch(seqs, 32, "cpu"), make_batch(seqs, 32, device)
        done(device)
        for name in ("token_ids", "positions", "slots", "q_start", "q_len", "ctx_len", "block_tables", "logits_rows", "tile_seq", "tile_q0"):
            x, y = getattr(a, name), getattr(b, name)
            assert (x is None) == (y is None) and (x is None or (x.dtype == y.dtype and torch.equal(x, y.cpu()))), name
        assert (a.is_decode, a.q_len_host, a.ctx_len_host) == (b.is_decode, b.q_len_host, b.ctx_len_host)
    for seqs, kw in (([one(40, 0, [1])], {}), ([one(4, 0, [1, 2, 3])], {"max_pages": 2})):
        for d in ("cpu", device):
            with pytest.raises((ValueError, RuntimeError)):
                make_batch(seqs, 32, d, **kw)
    done(device)


@pytest.mark.parametrize("device", GPU)
def test_prefill_portions_without_rows(device, monkeypatch):
    """Sequences without new tokens that fill portions of their own."""
    from deliverance_b200.ops import kv4

    monkeypatch.setattr(kv4, "EXPAND_PAGES_BYTES", 8 * 2 * 32 * 64 * 4)
    run_prefill(device, 64, 2, 2, [0, 5, 0, 0, 130], [400, 300, 700, 0, 20])
    run_prefill(device, 64, 2, 2, [0, 0], [400, 300])
