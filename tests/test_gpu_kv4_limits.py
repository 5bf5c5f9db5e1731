"""The 4-bit key/value cache operators at the ends of what their arguments may
be: the widest groups, windows, lengths and scales."""
import numpy as np
import pytest

import kv4_ref as R
import q3t
from test_gpu_kv4 import HALF, Setup, attend_case, check_attend

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("D, group", [(128, 2100), (64, 4200), (128, 17)])
def test_attend_of_groups_wider_than_a_launch_lists(D, group):
    """Without hints the rows of one token are more than the decoding kernel lists, and every sequence is a prompt."""
    S = Setup(D, 1, [1, 2], [300, 40])
    q = attend_case(S, group)
    cache, batch = S.on_gpu(0, 0)
    check_attend(cache.attend(batch, q), q, S, 0, key_bits=11)


@pytest.mark.parametrize("new, kv", [([60, 300, 30], [25, 20, 0]), ([6, 1, 3], [3, 1, 0]), ([5, 70], [1, 40])])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3])
@pytest.mark.parametrize("hints", [True, False])
def test_attend_of_padding_under_the_widest_windows(new, kv, window, hints):
    """A window beyond every position is none, for rows that share a unit or a tile with ones in front of position 0."""
    S = Setup(128, 2, new, [0] * len(new))
    q = attend_case(S, 2)
    S.kv = kv
    cache, batch = S.on_gpu(*(() if hints else (0, 0)))
    out = cache.attend(batch, q, window=window)
    assert torch.equal(out, cache.attend(batch, q))
    check_attend(out, q, S, 0, key_bits=11)


@pytest.mark.parametrize("new, past", [([1, 1], [40, 21]), ([30, 1], [70, 5])])
@pytest.mark.parametrize("scale, rows", [(1e-20, 1.0), (-1e-38, 1.0), (1e35, 1e-35), (-3e37, 1e-37), (1e-36, 1e36)])
def test_attend_of_extreme_scales(new, past, scale, rows):
    """Scales near both ends of 32 bits, over rows of zeros and ones whose scores come out ordinary or as nothing."""
    S = Setup(128, 1, new, past)
    q = attend_case(S, 2) * rows
    q[-1, 0] = 0
    q[0, 1] = 0
    cache, batch = S.on_gpu()
    out = cache.attend(batch, q, scale=scale)
    check_attend(out, q, S, 0, scale=float(np.float32(scale)), key_bits=11)


@pytest.mark.parametrize("kv", [-(2 ** 31), -(2 ** 31) + 5, -7])
@pytest.mark.parametrize("new", [[2, 1], [30, 40]])
def test_lengths_below_zero_are_padding(kv, new):
    """Every row is in front of position 0: an append skips it, attend and read give zeros."""
    S = Setup(128, 2, new, [40, 30])
    q = attend_case(S, 2)
    S.kv = [kv, kv]
    cache, batch = S.on_gpu(0, 0)
    before = S.d_pool.clone()
    k, v = (torch.randn(S.T, 2, 128, device="cuda") for _ in range(2))
    q_out = torch.full_like(q, 3.0)
    cache.append(batch, k, v, q=q.float(), q_out=q_out)
    assert torch.equal(S.d_pool, before) and (q_out == 3.0).all()
    assert all((t == 0).all() for t in cache.read(batch))
    for window in (0, 5):
        assert (cache.attend(batch, q, window=window) == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_read_of_values_near_the_largest(D, dtype):
    """Of -3.2e38 .. 3.2e38 in one group 15 steps are 6.4e38, beyond 32 bits, but no value that is kept is."""
    S = Setup(D, 2, [33], [5])
    cache, batch = S.on_gpu()
    x = torch.from_numpy((3.2e38 * S.rng.uniform(-1, 1, (2, S.T, 2, D))).astype(np.float32)).cuda().to(dtype)
    x[..., ::32], x[..., 1::32] = -3.2e38, 3.2e38
    cache.append(batch, *x)
    kc, vc, _, _ = R.unpack(S.d_pool.cpu().numpy(), D)
    for got, stored in zip(cache.read(batch), (kc, vc)):
        got = got.double().cpu().numpy()
        for row, s, p in S.places():
            pg, c = S.slot(s, p)
            ref = stored[pg, :, c]
            assert (np.abs(got[row] - ref) <= HALF * np.abs(ref) + 2.0 ** -22 * 3.2e38).all()
