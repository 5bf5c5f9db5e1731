"""The 4-bit key/value cache entries without a GPU: every refusal happens on
the host before any CUDA call, the rotary frequencies are host code, and the
64-bit restatement that the GPU tests compare with is held to its own
definition."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R
import q3t

INVALID = q3t.INVALID_INPUT


def cache(**kw):
    d = dict(device=0, num_kv_heads=8, head_dim=128, table_rows=4, table_stride=16, num_pages=64, pool=1 << 20,
             page_table=1 << 20)
    d.update(kw)
    return q3t.KV4CacheView(**d)


def batch(**kw):
    d = dict(num_seqs=2, num_tokens=4, max_q_len=0, max_kv_len=0, q_start=1 << 20, kv_len=1 << 20, table_row=None)
    d.update(kw)
    return q3t.KV4BatchView(**d)


def rows(**kw):
    d = dict(dtype=1, num_heads=16, q=1 << 20, k=1 << 20, v=1 << 20, q_stride=4096, k_stride=4096, v_stride=4096,
             q_gamma=None, k_gamma=None, eps=1e-6, q_out=1 << 20, q_out_stride=2048)
    d.update(kw)
    return q3t.KV4Rows(**d)


def rope(**kw):
    d = dict(rotary_dim=128, layout=0, scaling=0, original=4096, theta=1e6, factor=1.0, low=1.0, high=4.0,
             amplitude=1.0)
    d.update(kw)
    return q3t.RopeView(**d)


def call_append(c=None, b=None, r=None, p=None):
    ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
    return q3t.lib().q3t_kv4_append(ref(c), ref(b), ref(r), ref(p), None)


BAD_CACHE = [dict(head_dim=96), dict(head_dim=0), dict(num_kv_heads=0), dict(num_kv_heads=1025), dict(num_pages=0),
             dict(num_pages=1 << 31), dict(table_rows=0), dict(table_stride=-1), dict(pool=None), dict(page_table=None),
             dict(pool=(1 << 20) + 8), dict(table_stride=(1 << 20) + 1)]
BAD_BATCH = [dict(num_seqs=-1), dict(num_seqs=(1 << 20) + 1), dict(num_tokens=-1), dict(num_tokens=(1 << 28) + 1),
             dict(max_q_len=-1), dict(max_kv_len=-5), dict(q_start=None), dict(kv_len=None)]
BAD_ROWS = [dict(dtype=2), dict(num_heads=-1), dict(k=None), dict(v=None), dict(q=None), dict(q_out=None),
            dict(k_stride=1023), dict(v_stride=0), dict(q_stride=2047), dict(q_out_stride=2047), dict(k=(1 << 20) + 1),
            dict(dtype=0, v=(1 << 20) + 2), dict(k_gamma=1 << 20, eps=float("nan")), dict(q_gamma=1 << 20, eps=-1.0)]
BAD_ROPE = [dict(rotary_dim=136), dict(rotary_dim=-8), dict(rotary_dim=12), dict(layout=2), dict(scaling=3),
            dict(theta=0.0), dict(theta=float("inf")), dict(amplitude=float("nan")), dict(scaling=1, factor=0.0),
            dict(scaling=1, factor=float("inf")), dict(scaling=2, low=4.0, high=4.0), dict(scaling=2, original=0)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_cache_is_refused(bad):
    L = q3t.lib()
    assert call_append(cache(**bad), batch(), rows()) == INVALID
    assert L.q3t_kv4_attend(C.byref(cache(**bad)), C.byref(batch()), 16, 1 << 20, 2048, 0.1, 0, 1 << 20, 2048, 1 << 21, 1 << 22, None) == INVALID
    assert L.q3t_kv4_read(C.byref(cache(**bad)), C.byref(batch()), 1 << 20, 1024, 1 << 20, 1024, None) == INVALID
    assert L.q3t_last_error()


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_bad_batch_is_refused(bad):
    L = q3t.lib()
    assert call_append(cache(), batch(**bad), rows()) == INVALID
    assert L.q3t_kv4_attend(C.byref(cache()), C.byref(batch(**bad)), 16, 1 << 20, 2048, 0.1, 0, 1 << 20, 2048, 1 << 21, 1 << 22, None) == INVALID
    assert L.q3t_kv4_read(C.byref(cache()), C.byref(batch(**bad)), 1 << 20, 1024, 1 << 20, 1024, None) == INVALID


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_bad_rows_are_refused(bad):
    assert call_append(cache(), batch(), rows(**bad)) == INVALID


@pytest.mark.parametrize("bad", BAD_ROPE)
def test_bad_rope_is_refused(bad):
    assert call_append(cache(), batch(), rows(), rope(**bad)) == INVALID
    assert q3t.lib().q3t_rope_freqs(C.byref(rope(**bad)), (C.c_double * 64)()) == INVALID


def test_rotation_wider_than_the_head_is_refused():
    assert call_append(cache(head_dim=64), batch(), rows(), rope(rotary_dim=128)) == INVALID
    with pytest.raises(q3t.Q3TError):
        q3t.Rope(64, rotary_dim=72)


@pytest.mark.parametrize("heads, q, qs, scale, window, out, os_", [
    (0, 1 << 20, 2048, 0.1, 0, 1 << 20, 2048), (12, 1 << 20, 2048, 0.1, 0, 1 << 20, 2048),
    (16, None, 2048, 0.1, 0, 1 << 20, 2048), (16, 1 << 20, 2047, 0.1, 0, 1 << 20, 2048),
    (16, 1 << 20, 2048, float("nan"), 0, 1 << 20, 2048), (16, 1 << 20, 2048, 0.1, -1, 1 << 20, 2048),
    (16, 1 << 20, 2048, 0.1, 0, None, 2048), (16, 1 << 20, 2048, 0.1, 0, 1 << 20, 100),
    (16, (1 << 20) + 1, 2048, 0.1, 0, 1 << 20, 2048)])
def test_bad_attend_is_refused(heads, q, qs, scale, window, out, os_):
    assert q3t.lib().q3t_kv4_attend(C.byref(cache()), C.byref(batch()), heads, q, qs, scale, window, out, os_,
                                    1 << 21, 1 << 22, None) == INVALID


@pytest.mark.parametrize("ws, size", [(None, 1 << 22), (1 << 21, (64 << 10) - 1), (1 << 21, 0), ((1 << 21) + 8, 1 << 22)])
def test_bad_workspace_is_refused(ws, size):
    assert q3t.lib().q3t_kv4_attend(C.byref(cache()), C.byref(batch()), 16, 1 << 20, 2048, 0.1, 0, 1 << 20, 2048, ws,
                                    size, None) == INVALID


def test_null_structs_and_read_without_outputs_are_refused():
    L = q3t.lib()
    assert call_append(None, batch(), rows()) == INVALID
    assert call_append(cache(), None, rows()) == INVALID
    assert call_append(cache(), batch(), None) == INVALID
    assert L.q3t_kv4_read(C.byref(cache()), C.byref(batch()), None, 1024, None, 1024, None) == INVALID
    assert L.q3t_kv4_read(C.byref(cache()), C.byref(batch()), 1 << 20, 1023, None, 0, None) == INVALID
    assert L.q3t_rope_freqs(None, (C.c_double * 64)()) == INVALID
    assert L.q3t_rope_freqs(C.byref(rope()), None) == INVALID


def test_empty_batches_need_no_gpu():
    L = q3t.lib()
    for b in (batch(num_seqs=0, q_start=None, kv_len=None), batch(num_tokens=0)):
        assert call_append(cache(), b, rows(q=None, k=None, v=None, q_out=None)) == q3t.OK
        assert L.q3t_kv4_attend(C.byref(cache()), C.byref(b), 16, None, 0, 0.1, 0, None, 0, None, 0, None) == q3t.OK
        assert L.q3t_kv4_read(C.byref(cache()), C.byref(b), None, 0, None, 0, None) == q3t.OK


@pytest.mark.parametrize("rot, theta, kw", [
    (128, 1e6, {}), (64, 1e4, {}), (16, 500.0, {}), (0, 1e4, {}), (64, 1e4, dict(scaling="linear", factor=4.0)),
    (128, 1e6, dict(scaling="bands", factor=8.0, low=1.0, high=4.0, original=8192)),
    (96, 1e4, dict(scaling="bands", factor=32.0, low=1.0, high=32.0, original=4096))])
def test_rope_frequencies(rot, theta, kw):
    got = q3t.Rope(128, rotary_dim=rot, theta=theta, **kw).freqs()
    ref = R.frequencies(rot, theta, **kw)
    assert got.shape == ref.shape
    # a power, a division and a blend in 64 bits: a few roundings of 2^-53
    np.testing.assert_allclose(got, ref, rtol=2.0 ** -49, atol=0)
    if kw.get("scaling") == "bands":  # the fastest dims are kept, the slowest slowed down by the whole factor
        plain = R.frequencies(rot, theta)
        assert got[0] == plain[0] and got[-1] == pytest.approx(plain[-1] / kw["factor"], rel=1e-12)


@pytest.mark.parametrize("D", [64, 128])
def test_every_byte_of_a_block_belongs_to_one_token(D):
    """The layout has no gap and no overlap: each nibble is one (token, dim), each scale entry one (token, group)."""
    kb, ks, vb, vs, sc = R.block_tables(D)
    nibbles = np.concatenate([(kb * 2 + ks // 4).ravel(), (vb * 2 + vs // 4).ravel()])
    assert sorted(nibbles) == list(range(2 * 16 * D))
    owner = {}
    for table in (kb, vb):
        for c in range(16):
            for b in table[c]:
                assert owner.setdefault(int(b), c) == c
    assert sorted(set(sc.ravel())) == list(range(8 * D, 10 * D, 4))
    for c in range(16):
        assert len(set(sc[c])) == D // 32 and all(len(set(sc[c, j:j + 32])) == 1 for j in range(0, D, 32))


def test_quantisation_error_is_within_its_bound():
    """|n s + z - x| <= s / 2: the zero never exceeds the minimum, so nothing clamps below, and a scale rounded down
    (by 2^-8 at most) puts the maximum at 15.06 s, where the clamp costs 0.06 s.  Without a scale what is left is
    the zero's own step, 2^-7."""
    g = np.random.default_rng(3)
    x = np.concatenate([g.standard_normal((50, 128)), 100 + g.standard_normal((50, 128)),
                        g.standard_normal((50, 128)) * 10.0 ** g.uniform(-20, 20, (50, 1)),
                        np.zeros((1, 128)), np.full((1, 128), -7.3)]).astype(np.float32)
    n, s, z = R.quantise(x)
    assert n.max() <= 15
    back = n.reshape(len(x), 4, 32) * s[..., None].astype(np.float64) + z[..., None]
    err = np.abs(back - x.reshape(len(x), 4, 32))
    lo = x.reshape(len(x), 4, 32).min(-1)
    assert (z <= lo).all()
    bound = s * 0.5 + np.where(s == 0, np.abs(lo) * 2.0 ** -7, 0)
    assert (err <= bound[..., None] * (1 + 1e-6)).all()
