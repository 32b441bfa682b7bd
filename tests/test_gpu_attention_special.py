"""Attention where many keys or values are not finite, and where rows have to be
computed again without masked keys."""
import math

import pytest

torch = pytest.importorskip("torch")
from attention_cases import SENTINEL, Batch, reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def healthy(cuda, qmv):
    qmv.device_status(clear=True)
    yield
    assert qmv.device_status(clear=True) == 0


def fill_keys(b, s, first, last, what):
    at = torch.arange(first, last, device="cuda")
    b.put(b.keys, s, at, torch.full((last - first, b.kv_heads, b.d), what, dtype=b.keys.dtype, device="cuda"))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("first,last", [(0, 3000), (2000, 6000), (7000, 7900)])
def test_a_share_whose_keys_are_all_nan(qmv, t, heads, kv_heads, d, hint, first, last):
    """A cut tile's share that meets nothing but NaN scores: every row that sees
    them is NaN, however the shares are joined."""
    b = Batch(qmv, t, heads, kv_heads, d, [20, 3], [8000, 100], page=64)
    fill_keys(b, 0, first, last, math.nan)
    b.run_paged(max_query=hint)
    b.check(False)
    assert torch.isnan(b.out[:20]).all() and torch.isfinite(b.out[20:23]).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_a_prompt_whose_keys_are_nan_for_long(qmv, t):
    """The same over packed rows; queries and values are fine."""
    b = Batch(qmv, t, 2, 2, 64, [40, 6000])
    b.k[40 + 1000:40 + 4000] = math.nan
    b.run_packed()
    b.check(True)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("blocks", [2, 4, 5])
def test_nan_keys_that_fill_whole_shares_only(qmv, t, d, hint, blocks):
    """NaN keys from one border of 128 keys to another, wherever the shares'
    borders lie: also where each share has either NaN scores only or none."""
    b = Batch(qmv, t, 2, 1, d, [3], [8000], page=128)
    keys = b.get(b.keys, 0, 8000).clone()
    at = torch.arange(8000, device="cuda")
    for first in range(0, 62 - blocks):
        b.put(b.keys, 0, at, keys)
        fill_keys(b, 0, 128 * first, 128 * (first + blocks), math.nan)
        b.run_paged(max_query=hint)
        assert torch.isnan(b.out[:3]).all(), first


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hint", [1, 1000])
def test_keys_of_weight_zero_that_fill_whole_shares(qmv, t, hint):
    """Scores of minus infinity: their keys weigh nothing, and a NaN value of
    theirs still is one (0 times NaN), as it is where the keys stand among others."""
    b = Batch(qmv, t, 2, 1, 64, [3], [8000], page=128)
    b.rows[:, 0:128:64] = 2.0
    keys, values = (b.get(x, 0, 8000).clone() for x in (b.keys, b.values))
    at = torch.arange(8000, device="cuda")
    for first in range(0, 58, 3):
        gone = slice(128 * first, 128 * (first + 4))
        k, v = keys.clone(), values.clone()
        k[gone, :, 0] = -math.inf
        b.put(b.keys, 0, at, k)
        b.put(b.values, 0, at, values)
        b.run_paged(max_query=hint)
        b.check(False)
        assert torch.isfinite(b.out[:3]).all()
        v[gone, 0, 5] = math.nan
        b.put(b.values, 0, at, v)
        b.run_paged(max_query=hint)
        nan = torch.isnan(b.out[:3].view(3, 2, 64))
        assert nan[:, :, 5].all() and int(nan.sum()) == 6, first


def test_rows_computed_again_outlast_no_wait(qmv):
    """A masked NaN in the last value of a long context: the last rows of each
    head are computed again, 32 a warp at about 11 us for 32 of 260,000 keys,
    2.9 s in all, which is more than the 2 s after which the other warps of a CTA
    give a wait up.  The pairs of tiles that the CTA has behind them are right
    all the same."""
    new, kv = 9728, 260_000
    b = Batch(qmv, "f16", 8, 8, 128, [new], [kv], page=256, poison=False)
    b.run_paged()
    torch.cuda.synchronize()
    assert qmv.device_status() == 0
    clean = b.out.clone()
    b.put(b.values, 0, torch.tensor([kv - 1], device="cuda"), torch.full((1, 8, 128), math.nan, dtype=torch.float16, device="cuda"))
    b.out.fill_(SENTINEL)
    b.run_paged()
    torch.cuda.synchronize()
    assert qmv.device_status() == 0
    assert torch.equal(b.out[:new - 256], clean[:new - 256])
    assert torch.isfinite(b.out[:new - 1]).all() and torch.isnan(b.out[new - 1]).all()
    k, v = b.kv_of(0, False)
    want, tol = reference(b.q[new - 40:new - 1].double().view(39, 8, 128), k[:-1], v[:-1], 1.0 / math.sqrt(128), "f16")
    assert bool(((b.out[new - 40:new - 1].double().view_as(want) - want).abs() <= tol).all())
