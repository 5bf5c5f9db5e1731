"""Attention over the 4-bit cache within what its roundings are worth by weight.

A row's error is held to the root of the sum of squares of every rounding's
half step, each times the weight that it enters with: roundings of different
keys are independent, so this is sqrt(3) times what they are expected to make.
A value that has next to no weight adds nothing to the bound, however large."""
import math

import numpy as np
import pytest

import kv4_ref as R
import q3t
from test_gpu_kv4 import HALF, Setup, attend_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

H16 = 2.0 ** -11  # half a step of f16, relative to the value


def weighed(q, S, scale, window, prompt, pool=None):
    """(out, square of the bound) [T, heads, D] in float64 on the GPU.  prompt: whose roundings, None for either's."""
    k_all, v_all, _, v_s = (torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in
                            R.unpack(S.pool if pool is None else pool, S.D))
    q = q.double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    group = q.shape[1] // S.kvh
    for s, n in enumerate(S.kv):
        rows = slice(int(S.q_start[s]), int(S.q_start[s + 1]))
        pos = torch.arange(n - S.new[s], n, device="cuda")[:, None]
        at = [S.slot(s, p) for p in range(n)]
        pg, sl = (torch.tensor([x[i] for x in at], device="cuda") for i in range(2))
        key = torch.arange(n, device="cuda")[None, :]
        see = (key <= pos) & ((key > pos - window) if window else True) & (pg >= 0) & (pg < S.P)
        pg = pg.clamp(0, S.P - 1)
        for h in range(q.shape[1]):
            x, k, v = q[rows, h], k_all[pg, h // group, sl], v_all[pg, h // group, sl]
            digits = 15 * v_s[pg, h // group, sl]
            y = (x @ k.T * scale).masked_fill(~see, -math.inf)
            w = torch.softmax(y, -1)
            o = w @ v
            # scores: exponents and their largest in 32 bits, to 2^-22 of each; for prompts K in 11 bits
            y0 = y.masked_fill(~see, 0.0).abs()
            ds = ((y0 + y0.amax(-1, keepdim=True) + 32) * 2.0 ** -22) ** 2
            if prompt is not False:
                ds = ds + (scale * H16) ** 2 * (x * x) @ (k * k).T
            e = w * w * ds
            sq = e @ (v * v) - 2 * o * (e @ v) + o * o * e.sum(-1, keepdim=True)
            # weights in 11 bits, for prompts values too; for decoding the weight is of the digits, at most 15 of them
            kept = 0 if prompt is False else 2 * v * v
            sq = sq + H16 ** 2 * ((w * w) @ (kept if prompt else kept + digits * digits))
            # the smallest weights: f16 has steps of 2^-24, 2^-21 of the row's largest weight times value
            sq = sq + n * (2.0 ** -21 * (w * v.abs().amax(-1)).amax(-1, keepdim=True)) ** 2
            # values in f16 next to a larger one of the same key (16 keys where none is 2^10 times another)
            sq = sq + n * (2.0 ** -29 * (w * v.abs().amax(-1)).amax(-1, keepdim=True)) ** 2
            out[rows, h], bound[rows, h] = o, sq
    return out, bound


def check_weighed(got, q, S, window=0, scale=None, prompt=True, pool=None):
    ref, sq = weighed(q, S, S.D ** -0.5 if scale is None else scale, window, prompt, pool)
    err = got.double() - ref
    assert torch.isfinite(got).all()
    # the output's own rounding; and over all of a head's rows, roundings of different elements do not add up
    whole = ((HALF * ref) ** 2 + sq).sum((0, 2)).sqrt()
    assert (err.norm(dim=(0, 2)) <= whole).all(), (err.norm(dim=(0, 2)) / whole).max()
    # an element: six deviations of the sum of its roundings (a rounding's is its half step over sqrt(3))
    each = HALF * ref.abs() + 6 / math.sqrt(3) * sq.sqrt() + 1e-37
    assert (err.abs() <= each).all(), (err.abs() / each).max()


SHAPES = [  # D, kvh, group, new, past, window
    (128, 1, 2, [600], [0], 0),
    (128, 2, 2, [140], [700], 0),
    (128, 2, 2, [20], [1500], 0),
    (128, 1, 3, [100, 9, 60], [300, 900, 0], 150),
    (64, 2, 4, [70, 10, 33], [450, 17, 5], 0),
    (64, 1, 8, [40], [1100], 333),
]


@pytest.mark.parametrize("D, kvh, group, new, past, window", SHAPES)
@pytest.mark.parametrize("workspace", [64 << 10, q3t.KV4_WORKSPACE])
def test_prompts(D, kvh, group, new, past, window, workspace, monkeypatch):
    """Ordinary values, tiles whole and with their keys divided."""
    monkeypatch.setattr(q3t, "KV4_WORKSPACE", workspace)
    S = Setup(D, kvh, new, past)
    q = attend_case(S, group)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q, window=window), q, S, window)


@pytest.mark.parametrize("D, kvh, group, new, past, window", [
    (128, 2, 2, [1, 1, 2, 1], [700, 31, 2000, 4], 0), (64, 2, 4, [1, 1], [900, 77], 0), (128, 1, 5, [1, 3], [3000, 60], 100),
    (64, 1, 12, [1], [4000], 0)])
def test_decoding(D, kvh, group, new, past, window):
    S = Setup(D, kvh, new, past)
    q = attend_case(S, group)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q, window=window), q, S, window, prompt=False)


def test_prompts_with_missing_pages():
    S = Setup(128, 2, [90, 40, 3], [200, 1000, 300])
    q = attend_case(S, 2)
    S.table[0, [1, 3, 15]] = -1
    S.table[1, 4:60] = S.P + 7
    S.table[2, 2] = -9
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=None)


@pytest.mark.parametrize("hints", [None, (0, 0), (1, 1)])
def test_chunks_beside_decoding(hints):
    g = np.random.default_rng(3)
    new = [int(n) for n in g.choice([1, 1, 1, 2, 0, 19, 33], 40)]
    past = [int(n) for n in g.integers(0, 700, 40)]
    S = Setup(128, 2, new, past)
    q = attend_case(S, 2)
    cache, batch = S.on_gpu(*(hints or ()))
    for window in (0, 200):
        check_weighed(cache.attend(batch, q, window=window), q, S, window, prompt=None)


def outlier_case(D, new, past, times, at, score, seed=0, group=2):
    """Keys at positions `at` have values `times` the others' and, for every query, scores about `score` beside the
    others' few."""
    S = Setup(D, 1, [new], [past], seed=seed)
    g, n = S.rng, S.kv[0]
    k, v = (g.standard_normal((1, n, D)).astype(np.float32) for _ in range(2))
    x = g.standard_normal((S.T, group, D)).astype(np.float32)
    x[..., 0] = 8.0
    k[0, at, 0] = score / (8 * D ** -0.5)
    v[0, at] *= np.float32(times)
    S.fill([k], [v])
    return S, torch.from_numpy(x).cuda().bfloat16()


# where the large values are: next to keys that have weight, in a page of their own, at the end of every page (rows of
# a prompt before such a key must not see it, and share a page with it)
PLACES = {"one": lambda n: [21], "page": lambda n: list(range(32, 48)), "ends": lambda n: list(range(15, n, 16))}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(120, 90), (24, 1000), (300, 0)])
@pytest.mark.parametrize("where", PLACES)
@pytest.mark.parametrize("power", [9, 12, 16, 20, 26, 60])
def test_prompts_with_large_values_of_no_weight(D, new, past, where, power):
    S, q = outlier_case(D, new, past, 2.0 ** power, PLACES[where](new + past), -90.0)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(120, 90), (24, 1000)])
@pytest.mark.parametrize("power", [12, 20, 40])
def test_prompts_with_large_values_of_little_weight(D, new, past, power):
    """Weight times value is that of the other keys, so both count."""
    S, q = outlier_case(D, new, past, 2.0 ** power, [21, 60, 61], -power * math.log(2))
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(120, 90), (24, 1000)])
@pytest.mark.parametrize("power", [-12, -30, -60])
def test_prompts_with_small_values_of_most_weight(D, new, past, power):
    """One key has nearly all the weight and next to no value: the others' values, by their small weights, are the
    result."""
    S, q = outlier_case(D, new, past, 2.0 ** power, [3], 12.0)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S)
    S, q = outlier_case(D, new, past, 0.0, [3], 12.0)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S)


DECODING = [(1, 200), (1, 9000), (3, 700)]  # a warp's, many CTAs' and a few rows of which the last key is the last row's


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", DECODING)
@pytest.mark.parametrize("where", [*PLACES, "last"])
@pytest.mark.parametrize("power", [12, 20, 30, 40, 100])
def test_decoding_with_large_values_of_no_weight(D, new, past, where, power):
    n = new + past
    S, q = outlier_case(D, new, past, 2.0 ** power, [n - 1] if where == "last" else PLACES[where](n), -120.0)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", DECODING)
@pytest.mark.parametrize("power", [12, 40, 80, -12, -60])
def test_decoding_with_weight_and_size_apart(D, new, past, power):
    """Large values of little weight, that count as much as the others; small values, or none, of most weight."""
    S, q = outlier_case(D, new, past, 2.0 ** power, [21, 60, 61], -power * math.log(2) if power > 0 else 12.0)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=False)
    S, q = outlier_case(D, new, past, 0.0, [3], 12.0)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(1, 200), (1, 9000), (24, 1000)])
@pytest.mark.parametrize("low, high", [(-100, 100), (100, -100), (-90, 20)])
def test_sizes_that_grow_and_shrink_along_the_cache(D, new, past, low, high):
    """Parts of a row's keys whose values are hundreds of powers of two apart: each counts by its weight."""
    S = Setup(D, 1, [new], [past])
    g, n = S.rng, S.kv[0]
    k, v = (g.standard_normal((1, n, D)) for _ in range(2))
    v *= 2.0 ** np.round(np.linspace(low, high, n))[None, :, None]
    S.fill([k.astype(np.float32)], [v.astype(np.float32)])
    q = torch.from_numpy(g.standard_normal((S.T, 2, D)).astype(np.float32)).cuda().bfloat16()
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=new > 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(1, 200), (1, 9000), (24, 1000)])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 120, -(2.0 ** -90)])
def test_constant_values(D, new, past, size):
    """Groups without a scale: digits of zeros, and the zero is the value."""
    S = Setup(D, 1, [new], [past])
    g, n = S.rng, S.kv[0]
    k = g.standard_normal((1, n, D)).astype(np.float32)
    S.fill([k], [np.full((1, n, D), size, np.float32)])
    q = torch.from_numpy(g.standard_normal((S.T, 2, D)).astype(np.float32)).cuda().bfloat16()
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=new > 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(120, 90), (24, 1000), (300, 0)])
@pytest.mark.parametrize("where", PLACES)
@pytest.mark.parametrize("power", [9, 16, 30, 40, 90])
def test_prompts_with_large_keys_that_rows_do_not_see_or_score_low(D, new, past, where, power):
    """A key of large dims beside ordinary ones in its page: rows in front of it do not see it, rows behind it score it
    far below the others."""
    S, q = outlier_case(D, new, past, 1.0, PLACES[where](new + past), -2.0 ** power)
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [(1, 200), (1, 9000), (3, 900), (24, 1000), (300, 0)])
@pytest.mark.parametrize("spread", [True, False])
def test_values_near_the_largest(D, new, past, spread):
    """Groups of -3.2e38 .. 3.2e38, whose scale times 15 leaves 32 bits, or of 3.2e38 alone, which many keys sum up."""
    S = Setup(D, 1, [new], [past])
    g, n = S.rng, S.kv[0]
    v = 3.2e38 * (g.uniform(-1, 1, (1, n, D)) if spread else np.ones((1, n, D)))
    S.fill([g.standard_normal((1, n, D)).astype(np.float32)], [v.astype(np.float32)])
    q = torch.from_numpy((3 * g.standard_normal((S.T, 2, D))).astype(np.float32)).cuda().bfloat16()
    cache, batch = S.on_gpu()
    check_weighed(cache.attend(batch, q), q, S, prompt=new * 2 > 16)
