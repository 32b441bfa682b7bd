"""How exact attention is on inputs whose rows, weights or values differ widely
in magnitude: the root of the mean square error against a model of it, which a
lost part of an operand passes by far (the worst-case bounds of
attention_cases.py do not notice one).

Per output element, with A = sum_j w_j |v_j|, o the output and n the row's keys:
 * weights and values meet in parts that hold 22 bits each: 2^-22 A twice;
 * a score is summed over 3 D / 16 steps of 16 products, each of which rounds
   the sum so far by up to 2^-23 of it.  The sum is of the size of
   c_j = scale sqrt(sum_e (q_e k_je)^2), and the steps are independent, so a
   score is off by sqrt(3 D / 16) 2^-23 c_j, and a normalised weight by twice
   that at most: sqrt(3 D / 16) 2^-22 (sum_j w_j c_j) A.  (A score that is one
   exact product has no such error.)
 * a weight is 2^e_j, e_j <= 0 its score behind the row's largest one in log2,
   rounded to f32: off by 2^-24 |e_j| at most, so the weight by ln 2 times that
   of itself, and the output by ln 2 2^-24 sum_j w_j |e_j| |v_j|.  (Beside a sink
   of 2^60 times their weight that is 2.5e-6 A, for exact scores too.)
 * the output is summed over 48 steps each 128 keys at most, each of which
   rounds the sum so far, of the size of o: sqrt(48 n / 128) 2^-23 |o|.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from attention_cases import Batch, reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def healthy(cuda, qmv):
    qmv.device_status(clear=True)
    yield
    assert qmv.device_status(clear=True) == 0


def model(q, k, v, scale, one_product=()):
    """(out, A, modelled error / A), 64 bits; one_product: keys whose scores are
    one exact product."""
    n, heads, d = q.shape
    keys, kv_heads = k.shape[0], k.shape[1]
    live = torch.arange(keys, device=q.device)[None, :] <= torch.arange(n, device=q.device)[:, None] + keys - n
    out, mass, err = (torch.zeros(n, heads, d, dtype=torch.float64, device=q.device) for _ in range(3))
    for a in range(heads):
        h = a // (heads // kv_heads)
        w = torch.softmax(torch.where(live, scale * (q[:, a] @ k[:, h].T), -math.inf), -1)
        out[:, a], mass[:, a] = w @ v[:, h], w @ v[:, h].abs()
        c = scale * ((q[:, a] ** 2) @ (k[:, h] ** 2).T).sqrt()
        for j in one_product:
            c[:, j] = 0.0
        score = math.sqrt(3 * d / 16) * 2.0 ** -22 * (w * c).sum(-1, keepdim=True)
        steps = (48 * live.sum(-1, keepdim=True).double() / 128).sqrt() * 2.0 ** -23
        behind = (w * torch.log2(w / w.amax(-1, keepdim=True)).clamp_min(-1e4).abs()) @ v[:, h].abs() / mass[:, a].clamp_min(1e-300)
        part = (out[:, a].abs() / mass[:, a].clamp_min(1e-300)) * steps
        err[:, a] = (2 * 2.0 ** -44 + score ** 2 + part ** 2 + (math.log(2.0) * 2.0 ** -24 * behind) ** 2).sqrt()
    return out, mass, err


def rms_of(b, packed, one_product=()):
    """Worst ratio of the measured to the modelled root mean square error of a
    sequence's columns."""
    torch.cuda.synchronize()
    worst, a = 0.0, 0
    for s, n in enumerate(b.new):
        k, v = b.kv_of(s, packed)
        q = b.q[a:a + n].double().view(n, b.heads, b.d)
        out, mass, err = model(q, k, v, 1.0 / math.sqrt(b.d), one_product)
        got = b.out[a:a + n].double().view_as(out)
        a += n
        assert torch.isfinite(got).all()
        use = mass > 0
        assert torch.equal(got[~use], out[~use])
        rel = torch.where(use, (got - out) / mass.clamp_min(1e-300), 0.0)
        err = torch.where(use, err, 0.0)
        # of a column over all rows and heads, so that one bad column shows
        ratio = rel.square().mean((0, 1)).sqrt() / err.square().mean((0, 1)).sqrt().clamp_min(2.0 ** -22)
        worst = max(worst, float(ratio.max()))
    return worst


# -------------------------------------------------- values of f32 prompts

@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e10, 1e30])
@pytest.mark.parametrize("token", [2, 127, 300, 511])
def test_one_large_value_reaches_its_column_only(qmv, heads, kv_heads, d, size, token):
    """One element of one value row is large: the other columns, that token's
    own too, and the earlier tokens are as exact as without it."""
    b = Batch(qmv, "f32", heads, kv_heads, d, [512, 40])
    b.v[token, 5] = size
    b.run_packed()
    b.check(True)
    assert rms_of(b, True) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("what", ["as they are", "small", "tiny", "large", "rows apart", "elements apart"])
def test_values_of_any_size(qmv, heads, kv_heads, d, what):
    b = Batch(qmv, "f32", heads, kv_heads, d, [700, 65, 1, 130])
    g = torch.Generator(device="cuda").manual_seed(1)
    if what in ("small", "tiny", "large"):
        b.v.mul_({"small": 2.0 ** -74, "tiny": 1e-30, "large": 1e35}[what])
    elif what == "rows apart":
        b.v.mul_(torch.exp2(torch.randint(-40, 41, (b.tokens, 1), generator=g, device="cuda").float()))
    elif what == "elements apart":
        b.v.mul_(torch.exp2(torch.randint(-30, 31, b.v.shape, generator=g, device="cuda").float()))
    b.run_packed()
    b.check(True)
    assert rms_of(b, True) <= 1.0


# ------------------------------------------------------- a sink's neighbours

def sink_batch(qmv, t, heads, kv_heads, d, log2_weight, new=(20, 1), kv=(1000, 9000), packed=False):
    """The first key has 2^log2_weight times a middling key's weight and a value
    of 0, so that the output is made of small weights.  Its score is one exact
    product: channel 0 of every query is 4, of every other key 0."""
    b = Batch(qmv, t, heads, kv_heads, d, new, new if packed else kv, poison=False)
    b.rows[:, 0:heads * d:d] = 4.0
    size = log2_weight * math.log(2.0) * math.sqrt(d) / 4.0
    first = torch.zeros(1, kv_heads, d, dtype=b.dtype if packed else b.keys.dtype, device="cuda")
    first[:, :, 0] = size
    if packed:
        b.k[:, ::d] = 0.0
        at = 0
        for n in new:
            b.k[at], b.v[at] = first.view(-1), 0.0
            at += n
    else:
        (b.keys if b.layout == "position" else b.keys.transpose(1, 2))[..., 0] = 0.0
        for s in range(len(new)):
            b.put(b.keys, s, torch.tensor([0], device="cuda"), first)
            b.put(b.values, s, torch.tensor([0], device="cuda"), torch.zeros_like(first))
    return b


@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("log2_weight", [12, 16, 20, 24])
@pytest.mark.parametrize("hint", [1, 1000])
def test_small_weights_beside_a_sink(qmv, heads, kv_heads, d, log2_weight, hint):
    """f32 over f16 pages: the weights' pairs reach down to 2^-24 of the largest."""
    b = sink_batch(qmv, "f32", heads, kv_heads, d, log2_weight)
    b.run_paged(max_query=hint)
    b.check(False)
    assert rms_of(b, False, one_product=(0,)) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("log2_weight", [12, 24, 60])
def test_small_weights_of_prompts(qmv, heads, kv_heads, d, log2_weight):
    b = sink_batch(qmv, "f32", heads, kv_heads, d, log2_weight, new=(700, 130), packed=True)
    b.run_packed()
    b.check(True)
    assert rms_of(b, True, one_product=(0,)) <= 1.0


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("log2_weight", [12, 20, 26])
@pytest.mark.parametrize("hint", [1, 1000])
def test_small_weights_in_16_bits(qmv, t, heads, kv_heads, d, log2_weight, hint):
    b = sink_batch(qmv, t, heads, kv_heads, d, log2_weight, new=(20, 1, 5), kv=(1000, 9000, 40))
    b.run_paged(max_query=hint)
    b.check(False)
    b = sink_batch(qmv, t, heads, kv_heads, d, log2_weight, new=(300, 30), packed=True)
    b.run_packed()
    b.check(True)


# ------------------------------------------------------------ wide groups

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (27, 3), (16, 1), (33, 1), (126, 2), (64, 1)])
def test_wide_groups_of_heads_at_128(qmv, t, heads, kv_heads):
    for new, kv in (([1, 2, 1], [700, 65, 3]), ([40, 3, 129], [41, 600, 300])):
        b = Batch(qmv, t, heads, kv_heads, 128, new, kv, page=32, layout="head", pad=2)
        for hint in (1, 1000):
            b.out.fill_(123.0)
            b.run_paged(max_query=hint)
            b.check(False)
    b = Batch(qmv, t, heads, kv_heads, 128, [150, 1, 5, 64], pad=1)
    b.run_packed()
    b.check(True)


@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("exponent", [-111, -99, 60, 111])
def test_queries_and_keys_of_any_size(qmv, heads, kv_heads, d, exponent):
    """Queries that are tiny and keys that are large, or the other way: powers of
    two that cancel in the scores change nothing."""
    b = Batch(qmv, "f32", heads, kv_heads, d, [300, 65, 1], poison=False)
    b.q.mul_(2.0 ** exponent)
    b.k.mul_(2.0 ** -exponent)
    b.run_packed()
    b.check(True)
    assert rms_of(b, True) <= 1.0


# ------------------------------------------------- sums over many keys in f32

def _rows_near(b, packed, s, rows):
    """Some rows of sequence s: the norm of their error against that of the row.

    With values about 1 the sums all have one sign, so that additions that cut
    towards zero show: they cost 2^-24 of the sum each, 2^-13 over 16000 keys in
    steps of 16.  What is allowed: 2^-21 for weights and values in parts; a
    product of 64 keys by itself, 4 additions of its large parts and 20 of parts
    that are 2^-7 of them, each cut by 2^-23 of the sum so far, (4 + 20 2^-7) 2^-23;
    the sum of the products, rounded by half of 2^-23 each, independently:
    sqrt(n / 16) 2^-24 (decode adds one for each 16 keys); the scores as in
    model()."""
    torch.cuda.synchronize()
    k, v = b.kv_of(s, packed)
    a, n = sum(b.new[:s]), b.new[s]
    worst = 0.0
    for r in rows:
        keys = k.shape[0] - n + r + 1
        q = b.q[a + r:a + r + 1].double().view(1, b.heads, b.d)
        out, _, _ = model(q, k[:keys], v[:keys], 1.0 / math.sqrt(b.d))
        c = ((q ** 2).mean() * (k[:keys] ** 2).mean()).sqrt()  # a middling c_j of model()
        bound = 2.0 ** -21 + (4 + 20 * 2.0 ** -7) * 2.0 ** -23 + math.sqrt(keys / 16) * 2.0 ** -24 + math.sqrt(3 * b.d / 16) * 2.0 ** -22 * float(c)
        got = b.out[a + r:a + r + 1].double().view_as(out)
        worst = max(worst, float((got - out).norm() / out.norm()) / bound)
    return worst


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 2, 64), (16, 2, 128)])
def test_sums_of_long_prompts(qmv, heads, kv_heads, d):
    b = Batch(qmv, "f32", heads, kv_heads, d, [16384])
    b.v.mul_(0.25).add_(1.0)
    b.run_packed()
    assert _rows_near(b, True, 0, [0, 100, 999, 4000, 8100, 12345, 16383]) <= 1.0


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 2, 64), (16, 2, 128)])
def test_sums_of_chunks_over_long_contexts(qmv, heads, kv_heads, d):
    b = Batch(qmv, "f32", heads, kv_heads, d, [2048], [32768], page=64, poison=False)
    b.values.mul_(0.25).add_(1.0)
    b.run_paged()
    assert _rows_near(b, False, 0, [0, 5, 1000, 2047]) <= 1.0


@pytest.mark.parametrize("d", [64, 128])
def test_sums_of_decode_over_long_contexts(qmv, d):
    """Enough sequences that no CTA's part of one is short."""
    b = Batch(qmv, "f32", 16, 8, d, [1] * 64, [16000] * 62 + [1000, 100], page=64, poison=False)
    b.values.mul_(0.25).add_(1.0)
    b.run_paged()
    for s in (0, 30, 62, 63):
        assert _rows_near(b, False, s, [0]) <= 1.0
