"""What an append stores behind norm and rotation, digit for digit: every digit,
scale and zero, and every bf16 query, equals the definition in 32 bits (norm's
factor and the angles in 64), each product and sum rounded by itself.

Angles of two 64-bit computations differ by about 2^-52 of themselves, 2e-11
at position 100,000, so one cosine in some thousand rounds to another 32-bit
number there, and a digit, with a border in some millions of such numbers,
changes once in 10^9 or so: none of these cases' 10^5."""
import numpy as np
import pytest

import kv4_ref as R
import q3t
from test_gpu_kv4 import EPS, Setup

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F = np.float32


def normed(x, gamma):
    if gamma is None:
        return x
    r = (1.0 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + EPS)).astype(F)
    return x * r * gamma


def rotated(x, pos, freqs, layout, amplitude):
    n = len(freqs)
    angle = np.asarray(pos, np.float64)[:, None] * freqs
    c, s = ((f(angle) * np.float64(F(amplitude))).astype(F)[:, None] for f in (np.cos, np.sin))
    x = x.copy()
    a, b = ((slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    u, w = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = u * c - w * s, w * c + u * s
    return x


@pytest.mark.parametrize("D, group, rope", [
    (128, 2, dict(theta=1e6)),
    (128, 1, dict(theta=1e6, layout="interleaved")),
    (128, 2, dict(rotary_dim=72, scaling="linear", factor=3.0)),
    (128, 1, dict(scaling="bands", factor=32.0, low=1.0, high=32.0, amplitude=1.34375)),
    (64, 4, dict(rotary_dim=32, layout="interleaved", scaling="linear", factor=4.0)),
    (64, 1, dict(rotary_dim=24)),
])
@pytest.mark.parametrize("new, past", [([70, 45], [99_000, 7]), ([1, 3, 1], [131_000, 5, 40_001])])
@pytest.mark.parametrize("dtype, norm", [(torch.bfloat16, True), (torch.float32, True), (torch.float32, False)])
def test_digits_behind_norm_and_rotation(D, group, rope, new, past, dtype, norm):
    kvh = 2
    S = Setup(D, kvh, new, past)
    cache, batch = S.on_gpu()
    g = S.rng
    rows = torch.from_numpy((g.standard_normal((S.T, (group + 2) * kvh, D)) * 1.5 + 0.4).astype(F)).cuda().to(dtype)
    x = rows.float().cpu().numpy()
    gq, gk = (1 + 0.3 * g.standard_normal((2, D))).astype(F) if norm else (None, None)
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    q, k, v = rows[:, :group * kvh], rows[:, group * kvh:-kvh], rows[:, -kvh:]
    q_out = cache.append(batch, k, v, q=q, rope=q3t.Rope(D, **rope), q_gamma=dev(gq), k_gamma=dev(gk), eps=EPS)

    kw = {a: float(F(b)) if isinstance(b, float) else b for a, b in rope.items()
          if a in ("scaling", "factor", "low", "high")}
    f = R.frequencies(rope.get("rotary_dim", D), float(F(rope.get("theta", 1e4))), **kw)
    pos = [p for _, _, p in S.places()]
    turn = lambda a, gamma: rotated(normed(a, gamma), pos, f, rope.get("layout", "half"), rope.get("amplitude", 1.0))  # noqa: E731
    qx, kx, vx = turn(x[:, :group * kvh], gq), turn(x[:, group * kvh:-kvh], gk), x[:, -kvh:]
    assert torch.equal(q_out.cpu(), torch.from_numpy(qx).bfloat16())
    pool = S.d_pool.cpu().numpy()
    kb, ks, vb, vs, sc = R.block_tables(D)
    half = pool.view(np.uint16)
    at = [(row, *S.slot(s, p)) for row, s, p in S.places()]
    for src, byte, shift, o in ((kx, kb, ks, 0), (vx, vb, vs, 2)):
        n, scale, zero = R.quantise(src)
        for row, pg, c in at:
            np.testing.assert_array_equal(pool[pg][:, byte[c]] >> shift[c] & 15, n[row])
            np.testing.assert_array_equal(half[pg][:, sc[c, ::32] + o], R.bf16_bits(scale[row]))
            np.testing.assert_array_equal(half[pg][:, sc[c, ::32] + o + 1], R.bf16_bits(zero[row]))
