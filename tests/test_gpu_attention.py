"""Append to a paged cache and causal attention of ragged batches on the GPU,
against the formulas in 64 bits (attention_cases.py derives the tolerances)."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")
from attention_cases import HALF_STEP, SENTINEL, TYPES, Batch, reference  # noqa: E402

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (28, 4, 128), (4, 4, 128), (64, 1, 64), (9, 3, 64)]


@pytest.fixture(autouse=True)
def healthy(cuda, qmv):
    qmv.device_status(clear=True)
    yield
    assert qmv.device_status(clear=True) == 0


# ------------------------------------------------------------------ append

def _append_reference(b, base):
    """(q, k) turned, in 64 bits, and the position of every token."""
    pos = torch.cat([torch.arange(kv - n, kv) for n, kv in zip(b.new, b.kv)]).cuda()
    d = b.d

    def turn(x, heads):
        x = x[:b.used].double().view(b.used, heads, 2, d // 2)
        if base == 0.0:
            return x.reshape(b.used, heads, d)
        angle = pos.double()[:, None] * base ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        return torch.cat([x[:, :, 0] * c - x[:, :, 1] * s, x[:, :, 0] * s + x[:, :, 1] * c], -1)

    return turn(b.q, b.heads), turn(b.k, b.kv_heads), pos


def _near(got, want, size, u):
    """The product's rounding in f32 (four operations on terms up to size, and
    the sine's own 2^-22) and the rounding to the type, f16 subnormals too."""
    tol = u * want.abs() + 6 * 2.0 ** -23 * size + (2.0 ** -25 if u > 2.0 ** -20 else 0.0) + 2.0 ** -140
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS[:3])
@pytest.mark.parametrize("layout,page", [("position", 16), ("head", 64)])
def test_append(qmv, t, heads, kv_heads, d, layout, page):
    b = Batch(qmv, t, heads, kv_heads, d, [1, 17, 0, 5, 100], [1, 40, 0, 3000, 131], page=page, layout=layout, pad=2, poison=False)
    keys, values = b.keys.clone(), b.values.clone()
    k_out = torch.full((b.tokens, kv_heads * d), SENTINEL, dtype=b.dtype, device="cuda")
    qmv.paged_append(b.cache, b.batch(), b.id, heads, b.q, b.ld, b.k, b.ld, b.v, b.ld, 1e6, b.out, heads * d, k_out, kv_heads * d)
    torch.cuda.synchronize()
    q, k, _ = _append_reference(b, 1e6)
    size_q, size_k = (torch.cat([torch.hypot(*x[:b.used].double().view(b.used, -1, 2, d // 2).unbind(2))] * 2, -1) for x in (b.q, b.k))
    u, uc = HALF_STEP[t], HALF_STEP["bf16" if t == "bf16" else "f16"]
    _near(b.out[:b.used].view_as(q), q, size_q, u)
    _near(k_out[:b.used].view_as(k), k, size_k, u)
    assert torch.all(b.out[b.used:] == SENTINEL) and torch.all(k_out[b.used:] == SENTINEL)
    at = 0
    for s, (n, kv) in enumerate(zip(b.new, b.kv)):
        got, old = b.get(b.keys, s, kv), b.get(keys, s, kv)
        assert torch.equal(got[:kv - n], old[:kv - n])
        _near(got[kv - n:], k[at:at + n], size_k[at:at + n], uc)
        gv, ov = b.get(b.values, s, kv), b.get(values, s, kv)
        assert torch.equal(gv[:kv - n], ov[:kv - n])
        assert torch.equal(gv[kv - n:], b.v[at:at + n].view(n, kv_heads, d).to(gv.dtype))
        # nothing else of the cache changed
        b.put(b.keys, s, torch.arange(kv, device="cuda"), old)
        b.put(b.values, s, torch.arange(kv, device="cuda"), ov)
        at += n
    assert torch.equal(b.keys, keys) and torch.equal(b.values, values)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_append_without_rotation_copies(qmv, t):
    b = Batch(qmv, t, 6, 2, 64, [3, 2], [20, 2], poison=False)
    b.rows[0, :8] = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-7, 7.0, -7.0]).to(b.dtype)
    qmv.paged_append(b.cache, b.batch(), b.id, 6, b.q, b.ld, b.k, b.ld, b.v, b.ld, 0.0, b.out, 6 * 64)
    torch.cuda.synchronize()
    assert torch.equal(b.out[:5].view(torch.int32 if t == "f32" else torch.int16)[:, 1:], b.q.contiguous().view(torch.int32 if t == "f32" else torch.int16)[:, 1:])
    assert torch.equal(b.get(b.keys, 0, 20)[17:], b.k[:3].view(3, 2, 64).to(b.keys.dtype))


def test_append_in_place_and_without_queries(qmv):
    b = Batch(qmv, "f32", 4, 2, 64, [5, 7], [9, 7], poison=False)
    q, k, _ = _append_reference(b, 1e4)
    before = b.rows.clone()
    qmv.paged_append(b.cache, b.batch(), b.id, 4, None, 0, b.k, b.ld, b.v, b.ld, 1e4)
    torch.cuda.synchronize()
    assert torch.equal(b.rows, before)
    qmv.paged_append(b.cache, b.batch(), b.id, 4, b.q, b.ld, b.k, b.ld, b.v, b.ld, 1e4, b.q, b.ld, b.k, b.ld)
    torch.cuda.synchronize()
    assert float((b.q.double().view_as(q) - q).abs().max()) < 1e-5 and float((b.k.double().view_as(k) - k).abs().max()) < 1e-5
    assert torch.equal(b.v, before[:, 6 * 64:])


def test_append_far_positions(qmv):
    """The angle of position 2,000,000 is as exact as that of the first."""
    b = Batch(qmv, "f32", 2, 2, 128, [3], [2_000_000], page=256, poison=False)
    qmv.paged_append(b.cache, b.batch(), b.id, 2, b.q, b.ld, b.k, b.ld, b.v, b.ld, 10000.0, b.out, 256)
    torch.cuda.synchronize()
    # 64-bit angles lose 2^-53 * 2e6 / 2 pi turns themselves: 4e-11
    q, _, _ = _append_reference(b, 10000.0)
    _near(b.out[:3].view_as(q), q, torch.full_like(q, 8.0), 2.0 ** -24)


def test_append_skips_negative_positions(qmv):
    b = Batch(qmv, "f16", 2, 1, 64, [4], [2], poison=False)
    keys = b.keys.clone()
    qmv.paged_append(b.cache, b.batch(), b.id, 2, b.q, b.ld, b.k, b.ld, b.v, b.ld, 0.0, b.out, 128)
    torch.cuda.synchronize()
    assert torch.all(b.out[:2] == SENTINEL) and torch.equal(b.out[2:4], b.q[2:4])
    assert torch.equal(b.get(b.values, 0, 2), b.v[2:4].view(2, 1, 64))
    b.put(b.keys, 0, torch.arange(2, device="cuda"), b.get(keys, 0, 2))
    assert torch.equal(b.keys, keys)


# --------------------------------------------------------------- attention

LENGTHS = [[1], [2, 1, 1], [127], [128], [129, 1], [0, 63, 0, 64, 65, 0], [300, 5, 511, 17], [700]]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_packed(qmv, t, heads, kv_heads, d, lengths):
    b = Batch(qmv, t, heads, kv_heads, d, lengths, pad=3, seed=len(lengths), joint=heads != 9)
    b.run_packed()
    b.check(True)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS[:2])
def test_packed_long(qmv, t, heads, kv_heads, d):
    b = Batch(qmv, t, heads, kv_heads, d, [2500, 33, 1, 4001, 900])
    b.run_packed()
    b.check(True)


DECODE = [
    ([1], [1]), ([1], [16]), ([1], [17]), ([1], [1280]), ([1, 1, 1], [5, 700, 64]), ([1] * 40, [1 + 37 * i for i in range(40)]),
    ([1, 0, 1], [300, 50, 0]), ([2, 3, 1], [200, 3, 1000]), ([5] * 7, [5, 100, 2000, 31, 32, 33, 1024]),
]
CHUNKS = [
    ([16], [16]), ([40], [41]), ([100, 1, 30], [100, 1500, 800]), ([300], [2000]), ([1, 128, 7, 1], [900, 129, 8, 1]), ([64, 64], [64, 65]),
]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("case", range(len(DECODE) + len(CHUNKS)))
def test_paged(qmv, t, heads, kv_heads, d, case):
    new, kv = (DECODE + CHUNKS)[case]
    page, layout = [(16, "position"), (32, "head"), (64, "position"), (128, "head"), (256, "position")][case % 5]
    b = Batch(qmv, t, heads, kv_heads, d, new, kv, page=page, layout=layout, pad=case % 3, seed=case)
    b.run_paged()
    b.check(False)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 256])
def test_paged_long_decode(qmv, t, page):
    b = Batch(qmv, t, 28, 4, 128, [1, 1], [20011, 3], page=page)
    b.run_paged()
    b.check(False)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
def test_paged_chunk_over_a_long_cache(qmv, t, heads, kv_heads, d):
    """Few tiles over many keys: every tile is cut into dozens of shares."""
    b = Batch(qmv, t, heads, kv_heads, d, [45, 1], [20011, 9000], page=64, layout="head")
    b.run_paged()
    b.check(False)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_many_sequences(qmv, t):
    """More sequences than a CTA has threads, empty ones among them."""
    new = [(i * 7) % 5 for i in range(900)]
    kv = [n + (i * 13) % 40 if i % 11 else n for i, n in enumerate(new)]
    for hint in (1, 1000):
        b = Batch(qmv, t, 4, 2, 64, new, kv, page=16)
        b.run_paged(max_query=hint)
        torch.cuda.synchronize()
        for s in list(range(0, 900, 37)) + [896, 897, 898, 899]:
            a = sum(new[:s])
            if new[s]:
                k, v = b.kv_of(s, False)
                want, tol = reference(b.q[a:a + new[s]].double().view(new[s], 4, 64), k, v, 0.125, t)
                assert bool(((b.out[a:a + new[s]].double().view_as(want) - want).abs() <= tol).all()), (hint, s)
        assert not torch.any(b.out == SENTINEL)
    b = Batch(qmv, t, 4, 2, 64, new)
    b.run_packed()
    torch.cuda.synchronize()
    for s in range(0, 900, 37):
        a = sum(new[:s])
        if new[s]:
            k, v = b.kv_of(s, True)
            want, tol = reference(b.q[a:a + new[s]].double().view(new[s], 4, 64), k, v, 0.125, t)
            assert bool(((b.out[a:a + new[s]].double().view_as(want) - want).abs() <= tol).all()), s
    assert not torch.any(b.out == SENTINEL)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 60])
def test_output_rows_apart(qmv, t, new):
    """Output rows on 16-byte boundaries only, with room between them that
    stays as it was."""
    b = Batch(qmv, t, 6, 2, 64, [new, 2], [new + 90, 77])
    extra = 4 if t == "f32" else 8
    wide = torch.full((b.tokens, 6 * 64 + extra), SENTINEL, dtype=b.dtype, device="cuda")
    qmv.paged_attention(b.cache, b.batch(new), b.id, 6, b.q, b.ld, wide, 6 * 64 + extra)
    torch.cuda.synchronize()
    assert torch.all(wide[:, 6 * 64:] == SENTINEL)
    b.out.copy_(wide[:, :6 * 64])
    b.check(False)
    qmv.packed_attention(b.id, 6, 2, 64, b.start, 2, b.tokens, b.q, b.ld, b.k, b.ld, b.v, b.ld, wide, 6 * 64 + extra)
    torch.cuda.synchronize()
    assert torch.all(wide[:, 6 * 64:] == SENTINEL)
    b.out.copy_(wide[:, :6 * 64])
    b.check(True)


def test_offsets_past_32_bits(qmv):
    """Pages 2^31 elements apart, positions and heads with room between them."""
    hk, d, page, apart = 2, 64, 16, 2 ** 31 + 64
    size = apart + page * (hk * (d + 8) + 24) + 64
    keys, values = (torch.zeros(size, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = qmv.PagedCache(keys, values, 30, hk, d, page, 2, apart, hk * (d + 8) + 24, d + 8)
    view = [x.as_strided((2, page, hk, d), (apart, hk * (d + 8) + 24, d + 8, 1)) for x in (keys, values)]
    for new in (1, 20):
        b = Batch(qmv, "bf16", 8, hk, d, [new], [32], page=page)
        order = [1, 0]
        b.table[0, :2] = torch.tensor(order, dtype=torch.int32)
        qmv.paged_append(cache, b.batch(), b.id, 8, b.q, b.ld, b.k, b.ld, b.v, b.ld, 0.0)
        at = torch.arange(32 - new, 32, device="cuda")
        for x, rows in zip(view, (b.k, b.v)):
            assert torch.equal(x[torch.tensor(order, device="cuda")[at // page], at % page], rows[:new].view(new, hk, d))
            x.copy_(torch.randn(x.shape, device="cuda"))
        for hint in (1, 1000):
            b.out.fill_(SENTINEL)
            qmv.paged_attention(cache, b.batch(hint), b.id, 8, b.q, b.ld, b.out, 8 * d)
            torch.cuda.synchronize()
            k, v = (x[order].reshape(32, hk, d).double() for x in view)
            want, tol = reference(b.q[:new].double().view(new, 8, d), k, v, 0.125, "bf16")
            assert bool(((b.out[:new].double().view_as(want) - want).abs() <= tol).all()), (new, hint)


@pytest.mark.parametrize("hint", [1, 1000])
def test_max_query_is_only_a_hint(qmv, hint):
    b = Batch(qmv, "bf16", 14, 2, 64, [70, 1, 20], [300, 77, 20])
    b.run_paged(max_query=hint)
    b.check(False)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,kv", [([3, 1], [1, 0]), ([50, 20], [30, 0]), ([2], [0])])
def test_rows_without_keys_are_zero(qmv, t, new, kv):
    b = Batch(qmv, t, 14, 2, 64, new, kv)
    b.run_paged()
    torch.cuda.synchronize()
    at = 0
    for s, (n, m) in enumerate(zip(new, kv)):
        assert torch.all(b.out[at:at + n - m] == 0)
        at += n
    assert torch.isfinite(b.out).all()
    b.check(False)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.01, 3.0])
def test_scale(qmv, t, scale):
    """A flat and a peaked softmax."""
    b = Batch(qmv, t, 8, 2, 64, [1, 200, 1], [900, 333, 50])
    b.run_paged(scale=scale)
    b.check(False, scale=scale)
    b = Batch(qmv, t, 8, 2, 64, [200, 3])
    b.run_packed(scale=scale)
    b.check(True, scale=scale)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_masked_places_may_hold_anything(qmv, t, what):
    """A token's NaN or infinite key and value reach itself and later tokens of
    its sequence, nothing else."""
    b = Batch(qmv, t, 14, 2, 64, [90, 150, 40], pad=5)
    b.rows[90 + 70, 14 * 64:] = what  # k and v of token 70 of sequence 1
    b.rows[90 + 149, 16 * 64:] = -what  # v alone
    b.run_packed()
    torch.cuda.synchronize()
    out = b.out[:b.used].double()
    assert torch.isfinite(out[:90 + 70]).all() and torch.isfinite(out[240:280]).all()
    for s, (a, n) in enumerate([(0, 90), (90, 70), (240, 40)]):
        k, v = (x[a:a + n].view(n, 2, 64).double() for x in (b.k, b.v))
        want, tol = reference(b.q[a:a + n].double().view(n, 14, 64), k, v, 0.125, t)
        assert bool(((out[a:a + n].view_as(want) - want).abs() <= tol).all())
    assert torch.isnan(out[90 + 70:240]).any(-1).all()
    # the same in the cache: the last positions, seen by the last tokens only
    b = Batch(qmv, t, 14, 2, 64, [30, 1], [400, 100])
    b.put(b.values, 0, torch.tensor([390], device="cuda"), torch.full((1, 2, 64), what, dtype=b.values.dtype, device="cuda"))
    b.run_paged()
    torch.cuda.synchronize()
    out = b.out.double()
    assert torch.isfinite(out[:20]).all() and torch.isfinite(out[30]).all()
    assert not torch.isfinite(out[20:30]).any()
    k, v = b.kv_of(0, False)
    want, tol = reference(b.q[:20].double().view(20, 14, 64), k[:390], v[:390], 0.125, t)
    assert bool(((out[:20].view_as(want) - want).abs() <= tol).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lengths", [[700, 1500], [130, 65, 1029]], ids=str)
def test_not_a_number_from_a_token_on(qmv, t, lengths):
    """What a NaN token leaves behind it: tokens that are NaN all over, behind
    tokens that are not; and a value with one NaN element, which reaches that
    column only."""
    b = Batch(qmv, t, 14, 2, 64, lengths)
    at = b.used - lengths[-1]
    b.rows[at + 400:b.used] = math.nan
    b.v[at - 40, 5] = math.nan
    b.v[at + 3, 64 + 7] = math.nan
    b.run_packed()
    b.check(True)
    assert torch.isnan(b.out[at + 400:b.used]).all()
    assert torch.isfinite(b.out[at + 40:at + 400, :7 * 64]).all()
    assert int(torch.isnan(b.out[at + 40:at + 400, 7 * 64:]).sum()) == 360 * 7


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_large_and_small_magnitudes(qmv, t):
    """Scores of hundreds (one weight is 1, the rest vanish) and tiny ones."""
    for f in (30.0, 1e-3):
        b = Batch(qmv, t, 8, 2, 128, [70, 1, 9], [500, 300, 9], poison=False)
        b.rows[:, :8 * 128] *= f
        b.run_paged()
        b.check(False)
        b.run_packed()
        b.check(True)


# ----------------------------------------------- together, graphs, streams

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_prompt_chunk_and_decode_together(qmv, t):
    """Prompts enter through append and packed attention, a second chunk and
    three single tokens through append and paged attention: each step equals
    attention over the whole sequence so far."""
    heads, kv_heads, d, base = 14, 2, 64, 1e6
    first, second = [37, 1, 120], [20, 64, 5]
    total = [a + c + 3 for a, c in zip(first, second)]
    b = Batch(qmv, t, heads, kv_heads, d, first, first, page=16, layout="head")
    n = len(first)
    pages = [-(-x // 16) for x in total]
    width = max(pages)
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    order = torch.randperm(sum(pages), device="cuda").to(torch.int32)
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    dt, tid = TYPES[t]
    ct, cid = TYPES["bf16" if t == "bf16" else "f16"]
    keys, values = (torch.full((sum(pages), kv_heads, 16, d), math.nan, dtype=ct, device="cuda") for _ in range(2))
    cache = qmv.PagedCache(keys, values, cid, kv_heads, d, 16, sum(pages), kv_heads * 16 * d, d, 16 * d)
    cached = [0] * n
    for step, new in enumerate([first, second, [1] * n, [1] * n, [1] * n]):
        g = torch.Generator(device="cuda").manual_seed(step)
        rows = torch.randn(sum(new), (heads + 2 * kv_heads) * d, generator=g, device="cuda").to(dt)
        ld = rows.shape[1]
        q, k, v = rows[:, :heads * d], rows[:, heads * d:(heads + kv_heads) * d], rows[:, (heads + kv_heads) * d:]
        cached = [a + c for a, c in zip(cached, new)]
        start = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32, device="cuda")
        length = torch.tensor(cached, dtype=torch.int32, device="cuda")
        batch = qmv.PagedBatch(start, length, table, n, sum(new), width, max(new))
        out = torch.empty(sum(new), heads * d, dtype=dt, device="cuda")
        qmv.paged_append(cache, batch, tid, heads, q, ld, k, ld, v, ld, base, q, ld, k, ld)
        if step == 0:
            qmv.packed_attention(tid, heads, kv_heads, d, start, n, sum(new), q, ld, k, ld, v, ld, out, heads * d)
        else:
            qmv.paged_attention(cache, batch, tid, heads, q, ld, out, heads * d)
        torch.cuda.synchronize()
        at = 0
        for s in range(n):
            pos = torch.arange(cached[s], device="cuda")
            page = table[s].long()[pos // 16]
            ks, vs = keys.transpose(1, 2)[page, pos % 16].double(), values.transpose(1, 2)[page, pos % 16].double()
            assert torch.isfinite(ks).all() and torch.isfinite(vs).all()
            if step == 0:
                ks, vs = (x[at:at + new[s]].reshape(new[s], kv_heads, d).double() for x in (k, v))
            want, tol = reference(q[at:at + new[s]].reshape(new[s], heads, d).double(), ks, vs, 0.125, t)
            assert bool(((out[at:at + new[s]].double().view_as(want) - want).abs() <= tol).all()), (step, s)
            at += new[s]


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 50])
def test_captured_graph_follows_new_lengths(qmv, t, new):
    """A captured append + attention is replayed after lengths grow."""
    b = Batch(qmv, t, 14, 2, 64, [new, new], [900, 700])
    stream = torch.cuda.Stream()
    b.run_paged(stream=stream.cuda_stream)
    b.run_packed(stream=stream.cuda_stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    packed_out = torch.full_like(b.out, SENTINEL)
    with torch.cuda.graph(graph, stream=stream):
        s = torch.cuda.current_stream().cuda_stream
        b.run_paged(stream=s)
        b.run_packed(stream=s, out=packed_out)
    for kv in ([new, new + 1], [900, 700], [333, 512]):
        b.kv = kv
        b.length.copy_(torch.tensor(kv, dtype=torch.int32))
        b.out.fill_(SENTINEL)
        packed_out.fill_(SENTINEL)
        graph.replay()
        b.check(False)
        keep, b.out = b.out, packed_out
        b.check(True)
        b.out = keep


def test_two_streams_at_once(qmv):
    """Calls in flight together do not share scratch."""
    bs = [Batch(qmv, "bf16", 14, 2, 64, [1, 1], [5000 + i, 4000 - 7 * i], page=64, seed=i) for i in range(2)]
    cs = [Batch(qmv, "f16", 8, 2, 128, [200 + i], [1500 + i], page=32, seed=i) for i in range(2)]
    ss = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for b, c, s in zip(bs, cs, ss):
            b.run_paged(stream=s.cuda_stream)
            c.run_paged(stream=s.cuda_stream)
    for b in bs + cs:
        b.check(False)


def test_two_threads_at_once(qmv):
    """Calls from two host threads, each on its own stream."""
    packed, paged = Batch(qmv, "bf16", 14, 2, 64, [300, 700]), Batch(qmv, "f16", 32, 8, 128, [1] * 9, [900] * 9, seed=1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    failures = []

    def work(b, run, stream):
        try:
            for _ in range(50):
                run(stream=stream.cuda_stream)
        except Exception as e:  # noqa: BLE001 - handed to the test's thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=a) for a in ((packed, packed.run_packed, streams[0]), (paged, paged.run_paged, streams[1]))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    packed.check(True)
    paged.check(False)


def test_same_inputs_same_bits(qmv):
    for b in (Batch(qmv, "bf16", 28, 4, 128, [1, 1, 1], [5000, 300, 9], page=64), Batch(qmv, "f32", 14, 2, 64, [150, 9], [1400, 700])):
        b.run_paged()
        first = b.out.clone()
        for _ in range(5):
            b.out.fill_(0)
            b.run_paged()
            assert torch.equal(b.out, first)


def test_host_memory_is_refused(qmv):
    b = Batch(qmv, "f16", 2, 1, 64, [3])
    host = torch.zeros(3, 128, dtype=torch.float16)
    with pytest.raises(qmv.QmvError, match="device memory"):
        b.run_packed(out=host)


@pytest.mark.parametrize("which", ["keys", "values", "query_start", "length", "page_table", "q", "k", "v", "q_out", "k_out"])
def test_host_memory_is_refused_wherever_it_is_passed(qmv, which):
    """Every pointer is looked at before the launch; nothing runs."""
    b = Batch(qmv, "f16", 2, 1, 64, [3])
    host = torch.zeros(4096, dtype=torch.float16)
    cache, batch, at = b.cache, b.batch(), {n: host if n == which else x for n, x in dict(q=b.q, k=b.k, v=b.v, q_out=b.q, k_out=b.k).items()}
    if hasattr(cache.c, which):
        cache = qmv.PagedCache(*(host if which == n else x for n, x in (("keys", b.keys), ("values", b.values))), b.cache_id, 1, 64, b.page, b.count,
                               b.page * 64, 64, 64)
    elif hasattr(batch.c, which):
        meta = {n: host if n == which else x for n, x in dict(query_start=b.start, length=b.length, page_table=b.table).items()}
        batch = qmv.PagedBatch(**meta, sequences=1, tokens=b.tokens, max_pages=b.width)
    with pytest.raises(qmv.QmvError, match=which + " is not device memory"):
        qmv.paged_append(cache, batch, b.id, 2, at["q"], b.ld, at["k"], b.ld, at["v"], b.ld, 1e4, at["q_out"], b.ld, at["k_out"], b.ld)
    if which in ("keys", "values", "query_start", "length", "page_table", "q"):
        with pytest.raises(qmv.QmvError, match=which + " is not device memory"):
            qmv.paged_attention(cache, batch, b.id, 2, at["q"], b.ld, b.out, 128)
    if which in ("q", "k", "v", "query_start"):
        with pytest.raises(qmv.QmvError, match=("start" if which == "query_start" else which) + " is not device memory"):
            qmv.packed_attention(b.id, 2, 1, 64, host if which == "query_start" else b.start, 1, b.tokens, at["q"], b.ld, at["k"], b.ld, at["v"], b.ld, b.out, 128)


# --------------------------------------------- lengths about a half block

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (32, 8, 128), (2, 2, 128), (64, 1, 64)])
@pytest.mark.parametrize("paged", [False, True])
def test_lengths_about_half_a_block(qmv, t, heads, kv_heads, d, paged):
    """Tiles whose last block of 128 keys ends about its half."""
    if paged:
        b = Batch(qmv, t, heads, kv_heads, d, [40, 33, 34, 50, 17, 64, 40], [63, 64, 65, 191, 192, 193, 320], page=32, layout="head")
        b.run_paged(max_query=64)
    else:
        b = Batch(qmv, t, heads, kv_heads, d, [1, 63, 64, 65, 127, 128, 129, 191, 192, 193, 257], pad=5)
        b.run_packed()
    b.check(not paged)


# ----------------------------------------------------- metadata out of range

@pytest.mark.parametrize("new", [1, 40])
def test_metadata_out_of_range_is_reported(qmv, new):
    """A length beyond the table leaves its sequence out; a page index that
    does not exist is not followed; others are computed."""
    b = Batch(qmv, "bf16", 14, 2, 64, [new, new, new], [100, 200, 300])
    b.length[1] = b.width * b.page + 1
    b.run_paged()
    torch.cuda.synchronize()
    assert qmv.device_status(clear=True) == 32
    assert torch.all(b.out[new:2 * new] == SENTINEL)
    b.check(False, skip=(1,))
    b = Batch(qmv, "bf16", 14, 2, 64, [new, new, new], [100, 200, 300])
    page = int(b.table[1, 3])
    for bad in (-1, b.count, 2 ** 31 - 1):
        b.table[1, 3] = bad
        b.run_paged()
        torch.cuda.synchronize()
        assert qmv.device_status(clear=True) == 32
        b.table[1, 3] = page
        b.check(False, skip=(1,))
    b.table[1, 12] = -5  # positions 192.., the last page
    qmv.paged_append(b.cache, b.batch(), b.id, 14, b.q, b.ld, b.k, b.ld, b.v, b.ld, 1e4)
    torch.cuda.synchronize()
    assert qmv.device_status(clear=True) == 32
