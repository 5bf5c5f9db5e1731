"""The 4-bit key/value cache operators (q3t_kv4_append / attend / read) against
the 64-bit restatement in kv4_ref.py."""
import numpy as np
import pytest

import kv4_ref as R
import q3t

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EPS = 1e-6
HALF = 2.0 ** -8  # half a step of bf16, relative to the value


class Setup:
    """Pools, tables and a batch with `past` keys in front of each sequence's `new` tokens."""

    def __init__(self, D, kvh, new, past, seed=0, spare=3, stride_extra=1, table_row=None, device="cuda"):
        self.D, self.kvh, self.new, self.past = D, kvh, new, past
        g = self.rng = np.random.default_rng([seed, D, kvh, sum(new), sum(past)])
        B = len(new)
        self.kv = [n + p for n, p in zip(new, past)]
        pages = [-(-k // 16) for k in self.kv]
        self.P = sum(pages) + spare
        perm = g.permutation(self.P)
        rows = B if table_row is None else max(table_row) + 1
        self.table = g.integers(0, self.P, (rows, max(pages + [1]) + stride_extra)).astype(np.int32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b if table_row is None else table_row[b], :n] = perm[at:at + n]
            at += n
        self.q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.T = int(self.q_start[-1])
        self.pool = g.integers(0, 256, (self.P, kvh, 20 * D)).astype(np.uint8)  # stale bytes, NaN scales among them
        self.table_row, self.device = table_row, device

    def places(self):
        return R.places(self.q_start, np.array(self.kv))

    def slot(self, s, pos):
        return self.table[s if self.table_row is None else self.table_row[s], pos // 16], pos % 16

    def fill(self, k, v):
        """Puts f32 keys and values [kvh, n, D] of every sequence into the pool, in numpy."""
        kb, ks, vb, vs, sc = R.block_tables(self.D)
        half = self.pool.view(np.uint16)
        for s, n in enumerate(self.kv):
            for src, byte, shift, o in ((k[s], kb, ks, 0), (v[s], vb, vs, 2)):
                dig, scale, zero = R.quantise(src)
                for pos in range(n):
                    pg, c = self.slot(s, pos)
                    for h in range(self.kvh):
                        low = shift[c] == 0
                        blk = self.pool[pg, h]
                        blk[byte[c][low]] = (blk[byte[c][low]] & 0xf0) | dig[h, pos][low]
                        blk[byte[c][~low]] = (blk[byte[c][~low]] & 0x0f) | (dig[h, pos][~low] << 4)
                        half[pg, h, sc[c, ::32] + o] = R.bf16_bits(scale[h, pos])
                        half[pg, h, sc[c, ::32] + o + 1] = R.bf16_bits(zero[h, pos])

    def on_gpu(self, max_q=None, max_kv=None, tokens=None):
        dev = self.device
        self.d_pool = torch.from_numpy(self.pool).to(dev)
        self.d_table = torch.from_numpy(self.table).to(dev)
        cache = q3t.KV4Cache(self.d_pool, self.d_table, self.kvh, self.D)
        row = None if self.table_row is None else torch.tensor(self.table_row, dtype=torch.int32, device=dev)
        batch = q3t.KV4Batch(torch.from_numpy(self.q_start).to(dev),
                             torch.tensor(self.kv, dtype=torch.int32, device=dev),
                             self.T if tokens is None else tokens, table_row=row,
                             max_q=max(self.new) if max_q is None else max_q,
                             max_kv=max(self.kv) if max_kv is None else max_kv)
        return cache, batch


def rows_of(rng, T, heads, D, dtype, pad=0, bias=0.0):
    """(float64 values, device rows [T, heads, D] whose token stride is padded)."""
    x = (rng.standard_normal((T, heads, D)) * 1.5 + bias).astype(np.float32)
    buf = torch.zeros(T, heads * D + pad, device="cuda", dtype=dtype)
    buf[:, :heads * D] = torch.from_numpy(x.reshape(T, -1)).to("cuda").to(dtype)
    t = buf[:, :heads * D].unflatten(1, (heads, D))
    return t.double().cpu().numpy(), t


# ----------------------------------------------------------------------------
# append
# ----------------------------------------------------------------------------
APPEND = [  # D, kvh, group, new, past, dtype, norm, rope kwargs, row padding
    (128, 8, 2, [1], [0], torch.float32, True, dict(theta=1e6), 0),
    (128, 8, 2, [1, 1, 1], [5, 15, 16], torch.bfloat16, True, dict(theta=1e6), 0),
    (128, 2, 2, [16, 32, 17], [0, 16, 3], torch.bfloat16, False, dict(theta=1e4), 8),
    (128, 3, 5, [7, 0, 40, 1], [9, 4, 0, 31], torch.float32, True, dict(layout="interleaved"), 1),
    (64, 4, 1, [33, 1, 15], [0, 100, 1], torch.float32, False, dict(rotary_dim=32, layout="interleaved"), 0),
    (64, 1, 8, [100], [13], torch.bfloat16, True, dict(rotary_dim=24), 3),
    (128, 1, 1, [19], [100_003], torch.bfloat16, False, dict(rotary_dim=64, scaling="bands", factor=32.0, high=32.0,
                                                             amplitude=1.25), 0),
    (64, 2, 4, [9, 8], [70_000, 8], torch.float32, False, dict(scaling="linear", factor=3.0), 2),
    (128, 2, 0, [20], [12], torch.bfloat16, False, None, 0),
    (128, 20, 1, [5], [3], torch.bfloat16, False, dict(rotary_dim=0), 0),
    (128, 2, 2, [70, 40], [3, 100], torch.bfloat16, True, dict(theta=1e6), 0),
    (64, 3, 2, [64], [7], torch.float32, True, dict(layout="interleaved", rotary_dim=48), 0),
    (128, 1, 3, [45], [0], torch.float32, False, None, 1),
    (64, 2, 1, [35, 100], [60, 0], torch.bfloat16, False, dict(), 2),
    (128, 2, 1, [50, 33], [0, 1], torch.bfloat16, True, dict(rotary_dim=72), 0),
    (64, 1, 2, [3, 0, 18], [2, 0, 40], torch.float32, True, dict(rotary_dim=8), 0),
]


@pytest.mark.parametrize("D, kvh, group, new, past, dtype, norm, rp, pad", APPEND)
def test_append_matches_definition(D, kvh, group, new, past, dtype, norm, rp, pad):
    S = Setup(D, kvh, new, past)
    cache, batch = S.on_gpu()
    heads = kvh * group
    kx, k = rows_of(S.rng, S.T, kvh, D, dtype, pad, bias=0.7)
    vx, v = rows_of(S.rng, S.T, kvh, D, dtype, pad)
    qx, q = rows_of(S.rng, S.T, heads, D, dtype, pad) if heads else (None, None)
    gq, gk = (1 + 0.3 * S.rng.standard_normal((2, D))).astype(np.float32) if norm else (None, None)
    dg = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
    rope = None if rp is None else q3t.Rope(D, **rp)
    before = S.d_pool.clone()
    q_out = cache.append(batch, k, v, q=q, rope=rope, q_gamma=dg(gq), k_gamma=dg(gk), eps=EPS)
    k_rd, v_rd = cache.read(batch)
    torch.cuda.synchronize()

    pos = np.array([p for _, _, p in S.places()])
    def turned(x, gamma):
        x = R.rms_norm(x, None if gamma is None else gamma.astype(np.float64), EPS)
        if rp is None:
            return x
        kw = {a: b for a, b in rp.items() if a not in ("rotary_dim", "layout", "amplitude", "theta")}
        f = R.frequencies(rp.get("rotary_dim", D), rp.get("theta", 1e4), **kw)
        return R.rotate(x, pos, f, rp.get("layout", "half"), rp.get("amplitude", 1.0))
    kt, vt = turned(kx, gk), vx
    # 32-bit steps in front of the rounding: norm, gamma, two products and a sum of values up to the row's largest
    noise = lambda x: 8 * 2.0 ** -24 * np.abs(x).max(-1, keepdims=True)  # noqa: E731
    if heads:
        qt = turned(qx, gq)
        assert q_out.dtype == torch.bfloat16
        assert (np.abs(q_out.double().cpu().numpy() - qt) <= HALF * np.abs(qt) + noise(qt)).all()

    kc, vc, k_s, v_s = R.unpack(S.d_pool.cpu().numpy(), D)
    for row, s, p in S.places():
        pg, c = S.slot(s, p)
        for stored, scale, x in ((kc, k_s, kt), (vc, v_s, vt)):
            sc = scale[pg, :, c]
            rng_ = np.ptp(x[row].reshape(kvh, -1, 32), axis=-1).repeat(32, -1)
            low = np.abs(x[row].reshape(kvh, -1, 32).min(-1)).repeat(32, -1)
            # scale = (range + the zero's rounding) / 15, itself within half a step
            assert (sc <= (rng_ + 2.0 ** -7 * low) / 15 * (1 + HALF) + 1e-6).all()
            assert (np.abs(stored[pg, :, c] - x[row]) <= sc * 0.5 * (1 + 1e-5) + noise(x[row])).all()
        # the read gives the stored values, rounded once (and n s + z itself in 32 bits)
        for got, stored in ((k_rd, kc), (v_rd, vc)):
            ref = stored[pg, :, c]
            assert (np.abs(got[row].double().cpu().numpy() - ref) <= HALF * np.abs(ref) + 2.0 ** -22 * np.abs(ref).max()).all()

    # every byte that belongs to no appended token is as it was
    kb, _, vb, _, scx = R.block_tables(D)
    mine = torch.zeros_like(before, dtype=torch.bool).cpu().numpy()
    for _, s, p in S.places():
        pg, c = S.slot(s, p)
        at = np.concatenate([kb[c], vb[c], (2 * scx[c, ::32, None] + np.arange(8)).ravel()])
        mine[pg][:, at] = True
    same = (S.d_pool == before).cpu().numpy()
    assert same[~mine].all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new, past", [([16, 5, 37], [0, 11, 16]), ([64, 33], [0, 5])])
def test_append_without_rotation_stores_exact_digits(D, new, past):
    """Nothing precedes the quantisation, so every digit, scale and zero equals the definition's in 32 bits."""
    S = Setup(D, 3, new, past)
    cache, batch = S.on_gpu()
    g = S.rng
    x = (g.standard_normal((2, S.T, 3, D)) * 10.0 ** g.uniform(-6, 6, (2, S.T, 3, 1))).astype(np.float32)
    x[0, 0] = 0.0
    x[0, 1] = -7.3
    x[0, 2] = 3.3e38 * np.sign(g.standard_normal((3, D)))
    x[0, 3] = 1e-41
    x[1, 4] = 100 + 1e-3 * g.standard_normal((3, D))
    x[1, 5, :, ::2] = -0.0
    x[1, 6] = np.abs(x[1, 6])
    k, v = torch.from_numpy(x).cuda()
    cache.append(batch, k, v)
    pool = S.d_pool.cpu().numpy()
    kb, ks, vb, vs, sc = R.block_tables(D)
    half = pool.view(np.uint16)
    for src, byte, shift, o in ((x[0], kb, ks, 0), (x[1], vb, vs, 2)):
        n, scale, zero = R.quantise(src)
        for row, s, p in S.places():
            pg, c = S.slot(s, p)
            np.testing.assert_array_equal(pool[pg][:, byte[c]] >> shift[c] & 15, n[row])
            np.testing.assert_array_equal(half[pg][:, sc[c, ::32] + o], R.bf16_bits(scale[row]))
            np.testing.assert_array_equal(half[pg][:, sc[c, ::32] + o + 1], R.bf16_bits(zero[row]))


@pytest.mark.parametrize("new", [[9], [48]])
def test_append_norm_of_extreme_rows(new):
    """Rows whose squares 32 bits do not hold, rows of zeros, and q_out = q."""
    S = Setup(128, 2, new, [0])
    cache, batch = S.on_gpu()
    x = S.rng.standard_normal((S.T, 6, 128)) * 10.0 ** S.rng.choice([-35, -25, -12, 0, 12, 25, 35], (S.T, 6, 1))
    x[1] = 0
    x[2, :, 5] = 1e30  # one element far above the rest
    rows = torch.from_numpy(x).cuda().bfloat16()
    x = rows.double().cpu().numpy()
    gamma = (1 + 0.3 * S.rng.standard_normal(128)).astype(np.float32)
    g = torch.from_numpy(gamma).cuda()
    q, k, v = rows[:, :2].clone(), rows[:, 2:4], rows[:, 4:]
    for eps in (0.0, 1e-6):
        ref = R.rms_norm(x, gamma.astype(np.float64), eps) if eps else R.rms_norm(
            np.where(x == 0, np.nan, x), gamma.astype(np.float64), eps)  # 0 / 0 is no number
        ref = np.where(np.isnan(x * ref), np.nan, ref) if eps else ref
        mine = q.clone()
        out = cache.append(batch, k, v, q=mine, q_gamma=g, k_gamma=g, eps=eps, q_out=mine)
        assert out.data_ptr() == mine.data_ptr()
        got, want = mine.double().cpu().numpy(), ref[:, :2]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        # norm and gamma: two 32-bit roundings, the factor's own, and the bf16's; below 2^-126 steps are 2^-133
        err = np.abs(got - want) - (HALF + 2.0 ** -21) * np.abs(want) - 2.0 ** -133
        assert np.nanmax(err) <= 0


@pytest.mark.parametrize("B", [33, 129, 600])
def test_many_sequences(B):
    """More sequences than a warp, a CTA and one launch of attend look through at a time, some without rows."""
    g = np.random.default_rng(B)
    new = [int(x) for x in g.choice([0, 1, 1, 1, 2, 20], B)]
    past = [int(x) for x in g.integers(0, 40, B)]
    S = Setup(64, 2, new, past)
    q = attend_case(S, 2)
    cache, batch = S.on_gpu()
    check_attend(cache.attend(batch, q), q, S, 0)
    cache, batch = S.on_gpu(0, 0)
    check_attend(cache.attend(batch, q, window=9), q, S, 9)
    k, v = (torch.from_numpy(S.rng.standard_normal((S.T, 2, 64)).astype(np.float32)).cuda() for _ in range(2))
    cache.append(batch, k, v)
    kc, vc, _, _ = R.unpack(S.d_pool.cpu().numpy(), 64)
    got = [t.double().cpu().numpy() for t in cache.read(batch)]
    for x, y, stored, src in zip(got, range(2), (kc, vc), (k, v)):
        ref = np.stack([stored[S.slot(s, p)[0], :, S.slot(s, p)[1]] for _, s, p in S.places()])
        assert (np.abs(x - ref) <= HALF * np.abs(ref) + 2.0 ** -22 * np.abs(ref).max()).all()
        # and what is stored are the rows: within half a scale, which is at most (range + 2^-7 of the smallest) / 15
        src = src.double().cpu().numpy()
        step = (np.ptp(src.reshape(S.T, 2, 2, 32), axis=-1) * 1.02 + 0.04) / 15
        assert (np.abs(ref - src) <= 0.5 * step.repeat(32, -1) * (1 + 2.0 ** -6)).all()


def test_values_that_are_not_finite_read_back_as_nan():
    S = Setup(128, 2, [18], [0])
    cache, batch = S.on_gpu()
    x = S.rng.standard_normal((2, 18, 2, 128)).astype(np.float32)
    x[0, 3, 1, 40] = np.nan
    x[0, 17, 0, 0] = np.inf
    x[1, 5, 0, 127] = -np.inf
    cache.append(batch, *torch.from_numpy(x).cuda())
    k, v = (t.float().cpu().numpy() for t in cache.read(batch))
    bad = ~np.isfinite(x.reshape(2, 18, 2, 4, 32)).all(-1).repeat(32, -1).reshape(x.shape)
    np.testing.assert_array_equal(np.isnan(np.stack([k, v])), bad)
    # such a key hides behind the causal mask: rows before it do not see it, rows from it on are NaN
    q = torch.randn(18, 4, 128, device="cuda").bfloat16()
    out = cache.attend(batch, q).float().cpu().numpy()
    nan = np.isnan(out)
    assert not nan[:3].any() and nan[3:, 2:].all()  # key 3 of kv head 1: query heads 2 and 3
    assert not nan[:5, :2].any() and nan[17:, :2].all()
    assert nan[5:17, :2, 96:].all() and not nan[5:17, :2, :96].any()  # one group of a value


def test_rows_without_a_page_are_dropped():
    """Table entries outside the pool, rows past the table, negative positions: nothing is written for them, attend
    does not see them, read gives zeros, and the queries still come."""
    S = Setup(128, 2, [40, 10, 6], [0, 60, 0])
    S.kv[2] = 4  # two rows at negative positions
    S.table[0, 1] = -3
    S.table[1, 3] = S.P
    S.table[1, 4] = 1 << 30
    cache, batch = S.on_gpu()
    before = S.d_pool.clone()
    x = S.rng.standard_normal((2, S.T, 2, 128)).astype(np.float32)
    q = torch.randn(S.T, 4, 128, device="cuda")
    q_out = torch.full((S.T, 4, 128), 9.0, device="cuda").bfloat16()
    cache.append(batch, *torch.from_numpy(x).cuda(), q=q, q_out=q_out)
    skipped = [50, 51]
    kept = [i for i in range(S.T) if i not in skipped]
    assert torch.equal(q_out[kept], q[kept].bfloat16()) and (q_out[skipped] == 9.0).all()
    k, v = cache.read(batch)
    gone = list(range(16, 32)) + list(range(40, 50)) + skipped
    assert (k[gone] == 0).all() and (v[gone] == 0).all() and (k[[0, 15, 32, 39, 52, 55]] != 0).any(-1).all()
    kc, vc, _, _ = R.unpack(S.d_pool.cpu().numpy(), 128)
    used = {int(S.table[0, 0]), int(S.table[0, 2]), int(S.table[2, 0])}
    rest = [p for p in range(S.P) if p not in used]
    assert torch.equal(S.d_pool[rest], before[rest])
    qa = torch.randn(S.T, 4, 128, device="cuda").bfloat16()
    # the second sequence's pages 0..2 hold stale bytes: give its table no page at all
    S.d_table[1] = -1
    table = S.table.copy()
    table[1] = -1
    out = cache.attend(batch, qa).double().cpu().numpy()
    ref, big = R.attend(qa.double().cpu().numpy(), kc, vc, table, S.q_start, S.kv, 128 ** -0.5)
    assert (out[40:50] == 0).all() and (out[skipped] == 0).all()
    assert (np.abs(out - ref) <= HALF * np.abs(ref) + 2.0 ** -10 * big).all()


# ----------------------------------------------------------------------------
# attend
# ----------------------------------------------------------------------------
ATTEND = [  # D, kvh, group, new, past, window, hints
    (128, 2, 2, [1], [0], 0, True),
    (128, 8, 2, [1, 1, 1, 1], [15, 16, 17, 200], 0, True),
    (128, 1, 1, [1], [1000], 0, True),
    (128, 2, 2, [1, 1], [700, 31], 100, True),
    (128, 2, 2, [1, 5, 0, 33, 1], [40, 0, 7, 64, 300], 0, True),
    (128, 2, 2, [1, 5, 0, 33, 1], [40, 0, 7, 64, 300], 0, False),
    (128, 2, 3, [3, 2], [10, 250], 1, True),
    (128, 1, 8, [1, 1], [90, 513], 0, True),
    (128, 1, 16, [2, 1], [90, 48], 16, True),
    (64, 2, 1, [1, 1], [5, 333], 0, True),
    (64, 4, 4, [1, 1, 1], [0, 64, 129], 33, True),
    (64, 2, 8, [4, 1], [100, 17], 0, True),
    (64, 1, 5, [50], [0], 0, False),
    (128, 2, 2, [1, 2], [9, 40], 0, False),
    (64, 2, 1, [1], [3], 0, False),
    (128, 2, 2, [150], [0], 0, True),
    (128, 2, 2, [129, 64], [37, 500], 48, True),
    (64, 2, 2, [200], [33], 0, True),
    (128, 3, 1, [77], [0], 0, True),
    (64, 1, 12, [30], [250], 70, True),
    (128, 1, 8, [1, 1], [5000, 90], 0, True),
    (128, 2, 5, [1, 1, 1], [3000, 2, 800], 0, True),
    (64, 1, 12, [1], [4000], 0, True),
    (128, 2, 3, [2, 1, 0, 3], [900, 1500, 4, 60], 333, True),
]


def attend_case(S, group, scale_up=1.0):
    g = S.rng
    bias = 2.0 * g.standard_normal((S.kvh, 1, S.D)) * (g.random((S.kvh, 1, S.D)) < 0.1)
    k = [(g.standard_normal((S.kvh, n, S.D)) * scale_up + bias).astype(np.float32) for n in S.kv]
    v = [g.standard_normal((S.kvh, n, S.D)).astype(np.float32) for n in S.kv]
    S.fill(k, v)
    q = torch.from_numpy((1.3 * g.standard_normal((S.T, S.kvh * group, S.D))).astype(np.float32)).cuda().bfloat16()
    return q


def check_attend(out, q, S, window, scale=None, pool=None, key_bits=None):
    kc, vc, _, _ = R.unpack(S.pool if pool is None else pool, S.D)
    scale = S.D ** -0.5 if scale is None else scale
    ref, big = R.attend(q.double().cpu().numpy(), kc, vc, S.table, S.q_start, S.kv, scale, window, S.table_row)
    got = out.double().cpu().numpy()
    if key_bits:
        # keys in key_bits: a score is off by half a step of every product, its weight by e to that, and the weights'
        # sum too
        rows, k = np.abs(q.double().cpu().numpy()), np.abs(kc)
        pg = sorted({S.slot(s, p)[0] for s, n in enumerate(S.kv) for p in range(n)} & set(range(S.P)))
        most = np.nan_to_num(k[pg], nan=0).transpose(0, 2, 1, 3).reshape(-1, S.kvh, S.D)
        group = rows.shape[1] // S.kvh
        sums = np.stack([(most[:, h // group] @ rows[:, h].T).max(0) for h in range(rows.shape[1])], 1)
        big = big * (1 + 2 * abs(scale) * sums[..., None] * 2.0 ** -key_bits / (3 * 2.0 ** -11))
    # the output's own rounding, and weights and values in 11 bits: three half steps of 2^-11 on what they weigh
    # (a weight p s of the value, or the value and the weight; and the scores' 32-bit steps far below that)
    bound = HALF * np.abs(ref) + 3 * 2.0 ** -11 * big + 1e-30
    worst = (np.abs(got - ref) / bound).max()
    assert worst <= 1, worst


@pytest.mark.parametrize("D, kvh, group, new, past, window, hints", ATTEND)
def test_attend_matches_definition(D, kvh, group, new, past, window, hints):
    S = Setup(D, kvh, new, past)
    q = attend_case(S, group)
    cache, batch = S.on_gpu(*(() if hints else (0, 0)))
    check_attend(cache.attend(batch, q, window=window), q, S, window)


PROMPTS = [  # D, kvh, group, new, past, window, spread of the values
    (128, 1, 2, [600], [0], 0, 1.0),           # rows of several tiles, each with its own number of keys
    (128, 2, 2, [140], [700], 0, 1.0),         # both halves of a tile, its keys divided
    (128, 2, 2, [20], [1500], 0, 1.0),         # few rows on many keys
    (128, 1, 3, [100, 9, 60], [300, 900, 0], 150, 1.0),
    (64, 2, 4, [70, 1, 33], [450, 17, 5], 0, 1.0),
    (64, 1, 8, [40], [1100], 333, 1.0),
    (128, 1, 2, [200], [100], 0, 1e5),         # values and keys that later rows see are far larger
    (64, 1, 2, [18, 30], [900, 2], 0, 1e5),
]


@pytest.mark.parametrize("D, kvh, group, new, past, window, spread", PROMPTS)
@pytest.mark.parametrize("workspace", [64 << 10, q3t.KV4_WORKSPACE])
def test_attend_of_prompts(D, kvh, group, new, past, window, spread, workspace, monkeypatch):
    """Tiles of 256 rows on the tensor cores, whole (no room for parts) and with their keys divided."""
    monkeypatch.setattr(q3t, "KV4_WORKSPACE", workspace)
    S = Setup(D, kvh, new, past)
    q = attend_case(S, group)
    if spread > 1:
        g = S.rng
        grow = [spread ** np.linspace(-1, 0, n)[None, :, None] for n in S.kv]
        ks, vs = ([(g.standard_normal((kvh, n, D)) * w).astype(np.float32) for n, w in zip(S.kv, grow)] for _ in range(2))
        for v, n, p in zip(vs, new, past):
            v[:, (p + n // 2) | 15] *= 1e5  # the last key of a page, which the rows before it share
        S.fill(ks, vs)
    cache, batch = S.on_gpu()
    check_attend(cache.attend(batch, q, window=window), q, S, window, key_bits=11)
    a = cache.attend(batch, q, window=window)
    assert torch.equal(a, cache.attend(batch, q, window=window))


def test_attend_of_a_prompt_with_keys_that_are_no_numbers():
    """Rows behind such a key are NaN (of a value: its group), rows before it and outside their window are not."""
    S = Setup(128, 1, [300], [40])
    q = attend_case(S, 2)
    _, _, _, _, sc = R.block_tables(128)
    half = S.pool.view(np.uint16)
    for pos, what in ((200, 0), (250, 2)):  # K's scale of group 1, V's of group 2
        pg, c = S.slot(0, pos)
        half[pg, 0, sc[c, 32 * (1 + (what > 0))] + what] = 0x7fc0
    cache, batch = S.on_gpu()
    nan = np.isnan(cache.attend(batch, q).float().cpu().numpy())
    assert not nan[:160].any() and nan[160:].all()
    nan = np.isnan(cache.attend(batch, q, window=30).float().cpu().numpy())
    assert not nan[:160].any() and nan[160:190].all() and not nan[190:210].any() and not nan[240:].any()
    assert nan[210:240, :, 64:96].all() and not nan[210:240, :, :64].any() and not nan[210:240, :, 96:].any()


@pytest.mark.parametrize("window", [0, 7])
def test_attend_of_prompts_with_padding_in_front(window):
    """Rows at negative positions see nothing and give zeros: some of a tile's, all of one, all of a sequence."""
    S = Setup(128, 2, [60, 300, 30], [0, 0, 0])
    q = attend_case(S, 2)
    S.kv = [25, 20, 0]
    cache, batch = S.on_gpu()
    out = cache.attend(batch, q, window=window)
    assert (out[:35] == 0).all() and (out[60:340] == 0).all() and (out[360:] == 0).all()
    check_attend(out, q, S, window, key_bits=11)


def test_attend_of_a_prompt_with_missing_pages():
    S = Setup(128, 2, [90, 40], [200, 1000])
    q = attend_case(S, 2)
    S.table[0, [0, 3, 15]] = -1
    S.table[1, 4:60] = S.P + 7
    cache, batch = S.on_gpu()
    check_attend(cache.attend(batch, q), q, S, 0, key_bits=11)
    S.table[:] = -5
    cache, batch = S.on_gpu()
    assert (cache.attend(batch, q) == 0).all()


@pytest.mark.parametrize("new, group", [([2, 1], 2), ([20, 3], 2), ([1, 1], 16)])
def test_attend_of_lengths_far_past_the_table(new, group):
    """Positions that no table entry stands for hold no keys, up to the largest lengths there are."""
    # every table entry is a page of written keys: stale bytes are numbers up to 3e38, whose scores 32 bits do not hold
    S = Setup(128, 2, new, [96 - n for n in new], stride_extra=0)
    q = attend_case(S, group)
    S.kv = [100_000 + n for n in new]
    cache, batch = S.on_gpu(0, 0)
    out = cache.attend(batch, q)
    keys = S.table.shape[1] * 16
    kc, vc, _, _ = R.unpack(S.pool, 128)
    end = np.array([keys + n for n in new])  # every row sees the whole table
    ref, big = R.attend(q.double().cpu().numpy(), kc, vc, S.table, S.q_start, end, 128 ** -0.5)
    assert (np.abs(out.double().cpu().numpy() - ref) <= HALF * np.abs(ref) + 2.0 ** -9 * big).all()
    S.kv = [2 ** 31 - 1, 2 ** 31 - 17]
    cache, batch = S.on_gpu(0, 0)
    assert torch.equal(cache.attend(batch, q), out)
    assert torch.equal(cache.attend(batch, q, window=2 ** 31 - 1), out)
    assert (cache.attend(batch, q, window=1000) == 0).all()
    k, v = (torch.zeros(S.T, 2, 128, device="cuda") for _ in range(2))
    before = S.d_pool.clone()
    assert torch.equal(cache.append(batch, k, v, q=q.float()), q)  # the queries come all the same
    assert torch.equal(S.d_pool, before)
    assert all((t == 0).all() for t in cache.read(batch))


def test_attend_of_a_prompt_in_a_graph_next_to_eager_calls():
    """A captured prompt keeps its own parts: eager calls between replays do not disturb it."""
    S = Setup(128, 2, [30], [1200])
    q = attend_case(S, 2)
    cache, batch = S.on_gpu()
    ref = cache.attend(batch, q)
    once, twice = torch.empty_like(q), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(batch, q, out=once)
        cache.attend(batch, once, out=twice)  # on the parts' memory again
    ref2 = cache.attend(batch, ref)
    for _ in range(3):
        once.zero_()
        graph.replay()
        assert torch.equal(cache.attend(batch, q), ref)
        torch.cuda.synchronize()
        assert torch.equal(once, ref) and torch.equal(twice, ref2)


def test_attend_hints_do_not_change_what_is_computed():
    """max_q and max_kv below the truth choose another launch, not another result."""
    S = Setup(128, 2, [1, 19, 70], [300, 30, 0])
    q = attend_case(S, 2)
    for hints in ((1, 1), (2, 500), (1, 100_000), (70, 16)):
        cache, batch = S.on_gpu(*hints)
        check_attend(cache.attend(batch, q), q, S, 0)


def test_attend_long_cache_and_sharp_scores():
    """Keys split over many CTAs, with a few scores far above the rest and value scales that grow along the cache."""
    S = Setup(128, 1, [1], [4999])
    g = S.rng
    k = g.standard_normal((1, 5000, 128)).astype(np.float32)
    v = (g.standard_normal((1, 5000, 128)) * 10.0 ** np.linspace(-6, 3, 5000)[None, :, None]).astype(np.float32)
    qv = g.standard_normal((1, 2, 128)).astype(np.float32)
    k[0, 7] = 4 * qv[0, 0]
    k[0, 4100] = 3 * qv[0, 1]
    S.fill([k], [v])
    q = torch.from_numpy(qv).cuda().bfloat16()
    cache, batch = S.on_gpu()
    check_attend(cache.attend(batch, q), q, S, 0)
    check_attend(cache.attend(batch, q, scale=0.0), q, S, 0, scale=0.0)
    check_attend(cache.attend(batch, q, scale=-0.5), q, S, 0, scale=-0.5)


@pytest.mark.parametrize("D", [64, 128])
def test_attend_averages_of_very_many_keys(D):
    """80,000 keys that weigh about alike, for the whole GPU and (hints far too low) for one CTA: the average is some
    hundredths of the values, and keeps its own digits."""
    n = 80_000
    S = Setup(D, 1, [n], [0], spare=0)
    cache, batch = S.on_gpu()
    k, v = (torch.from_numpy(S.rng.standard_normal((n, 1, D)).astype(np.float32)).cuda() for _ in range(2))
    cache.append(batch, k, v)
    pool = S.d_pool.cpu().numpy()
    q = torch.from_numpy(S.rng.standard_normal((1, 2, D)).astype(np.float32)).cuda().bfloat16()
    kc, vc, _, _ = R.unpack(pool, D)
    for max_kv in (n, 1):
        one = q3t.KV4Batch(torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                           torch.tensor([n], dtype=torch.int32, device="cuda"), 1, max_q=1, max_kv=max_kv)
        got = cache.attend(one, q).double().cpu().numpy()
        ref, _ = R.attend(q.double().cpu().numpy(), kc, vc, S.table, [0, 1], [n], D ** -0.5)
        # a bf16 half step, and every key's weight p s rounded by half a step of 11 bits: independent, so together no
        # more of the sum of independent values than each of its own
        assert np.linalg.norm(got - ref) <= (HALF + 3 * 2.0 ** -11) * np.linalg.norm(ref)


def test_attend_extreme_queries_and_values():
    """Queries of zeros, tiny and large ones in one row, tiny and large value scales."""
    S = Setup(64, 1, [6], [40])
    g = S.rng
    k = [g.standard_normal((1, 46, 64)).astype(np.float32) * 1e-3]
    v = [(g.standard_normal((1, 46, 64)) * 1e-30).astype(np.float32)]
    v[0][0, 20:] *= 1e25
    S.fill(k, v)
    qv = g.standard_normal((6, 3, 64)).astype(np.float32)
    qv[0] = 0
    qv[1] *= 1e-30
    qv[2] *= 1e4
    qv[3, :, ::2] *= 1e-20
    q = torch.from_numpy(qv).cuda().bfloat16()
    cache, batch = S.on_gpu()
    check_attend(cache.attend(batch, q), q, S, 0)


@pytest.mark.parametrize("pad_q, pad_o", [(0, 0), (8, 16), (1, 3), (4, 0)])
def test_attend_row_strides(pad_q, pad_o):
    S = Setup(128, 2, [1, 3], [50, 20])
    q = attend_case(S, 2)
    H, D = q.shape[1:]
    qs = torch.zeros(S.T, H * D + pad_q, device="cuda", dtype=torch.bfloat16)
    qs[:, :H * D] = q.reshape(S.T, -1)
    os_ = torch.full((S.T + 2, H * D + pad_o), 5.0, device="cuda", dtype=torch.bfloat16)
    cache, batch = S.on_gpu()
    out = os_[:S.T, :H * D].unflatten(1, (H, D))
    cache.attend(batch, qs[:, :H * D].unflatten(1, (H, D)), out=out)
    check_attend(out, q, S, 0)
    assert (os_[S.T:] == 5.0).all() and (os_[:, H * D:] == 5.0).all()


def test_rows_behind_the_last_sequence_stay():
    S = Setup(128, 2, [2, 1], [30, 4])
    q = attend_case(S, 2)
    cache, batch = S.on_gpu(tokens=S.T + 5)
    q = torch.cat([q, torch.full((5, 4, 128), float("nan"), device="cuda").bfloat16()])
    out = torch.full_like(q, 3.0)
    cache.attend(batch, q, out=out)
    assert (out[S.T:] == 3.0).all()
    check_attend(out[:S.T], q[:S.T], S, 0)
    k = torch.full((S.T + 5, 2, 128), 3.0, device="cuda").bfloat16()
    v = k.clone()
    before = S.d_pool.clone()
    cache.read(batch, k=k, v=v)
    assert (k[S.T:] == 3.0).all() and (v[S.T:] == 3.0).all()
    qo = torch.full_like(q, 3.0)
    cache.append(batch, k, v, q=q, q_out=qo)
    assert (qo[S.T:] == 3.0).all()
    touched = {S.slot(s, p)[0] for _, s, p in S.places()}
    rest = [p for p in range(S.P) if p not in touched]
    assert torch.equal(S.d_pool[rest], before[rest])


def test_table_row_and_shared_pages():
    """Two sequences read one table row (a shared prefix), a third another."""
    S = Setup(128, 2, [1, 1, 1], [64, 64, 10], table_row=[2, 0, 3])
    q = attend_case(S, 2)
    S.table_row = [2, 2, 3]
    cache, batch = S.on_gpu()
    check_attend(cache.attend(batch, q), q, S, 0)


def test_results_repeat_bit_for_bit():
    S = Setup(128, 2, [1, 1, 40], [900, 33, 100])
    q = attend_case(S, 2)
    cache, batch = S.on_gpu()
    a = cache.attend(batch, q)
    for _ in range(3):
        assert torch.equal(a, cache.attend(batch, q))


# ----------------------------------------------------------------------------
# together, as a program runs them
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("D, group, layout", [(128, 2, "half"), (64, 4, "interleaved")])
def test_prompt_then_tokens_equals_one_long_prompt(D, group, layout):
    """A prompt appended and attended in one call, and then token by token, give the same rows as the whole sequence
    in one call; both against attention over the stored values."""
    kvh, n, m = 2, 45, 6
    rope = q3t.Rope(D, layout=layout)
    g = np.random.default_rng(5)
    x = lambda h: torch.from_numpy(g.standard_normal((n + m, h, D)).astype(np.float32)).cuda().bfloat16()  # noqa: E731
    k, v, q = x(kvh), x(kvh), x(kvh * group)

    whole = Setup(D, kvh, [n + m], [0])
    cache, batch = whole.on_gpu()
    q_all = cache.append(batch, k, v, q=q, rope=rope)
    out = cache.attend(batch, q_all)
    check_attend(out, q_all, whole, 0, pool=whole.d_pool.cpu().numpy())

    steps = Setup(D, kvh, [n + m], [0])
    cache, _ = steps.on_gpu()
    at = 0
    for count in [n] + [1] * m:
        b = q3t.KV4Batch(torch.tensor([0, count], dtype=torch.int32, device="cuda"),
                         torch.tensor([at + count], dtype=torch.int32, device="cuda"), count, max_q=count)
        qr = cache.append(b, k[at:at + count], v[at:at + count], q=q[at:at + count], rope=rope)
        assert torch.equal(qr, q_all[at:at + count])
        o = cache.attend(b, qr).double()
        ref = out[at:at + count].double()
        # both are within three half steps of 2^-11 on the values and a bf16 half step of the same attention
        assert ((o - ref).abs() <= 2 * HALF * ref.abs() + 6 * 2.0 ** -11 * 6.0).all()
        at += count
    used = whole.table[0, :-(-(n + m) // 16)]
    for i, pg in enumerate(used):
        full = min(16, n + m - 16 * i)
        kb, _, vb, _, sc = R.block_tables(D)
        at = np.concatenate([np.concatenate([kb[c], vb[c], (2 * sc[c, ::32, None] + np.arange(8)).ravel()])
                             for c in range(full)])
        np.testing.assert_array_equal(whole.d_pool[pg].cpu().numpy()[:, at],
                                      steps.d_pool[steps.table[0, i]].cpu().numpy()[:, at])


def test_graph_replay_with_changed_lengths():
    """A step captured once is replayed with new lengths, rows and page tables in the same buffers."""
    D, kvh, B = 128, 2, 3
    S = Setup(D, kvh, [1, 1, 1], [20, 100, 47])
    q = attend_case(S, 2)
    cache, _ = S.on_gpu()
    q_start = torch.from_numpy(S.q_start).cuda()
    kv_len = torch.tensor(S.kv, dtype=torch.int32, device="cuda")
    batch = q3t.KV4Batch(q_start, kv_len, B, max_q=1, max_kv=128)
    rope = q3t.Rope(D)
    k, v = (torch.randn(B, kvh, D, device="cuda") for _ in range(2))
    qr, out = torch.empty_like(q), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        cache.append(batch, k, v, q=q.float(), rope=rope, q_out=qr)
        cache.attend(batch, qr, out=out)
    side.synchronize()
    qf = q.float()
    with torch.cuda.graph(graph):
        cache.append(batch, k, v, q=qf, rope=rope, q_out=qr)
        cache.attend(batch, qr, out=out)
    for turn in range(3):
        k.normal_()
        v.normal_()
        qf.normal_()
        kv_len.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        S.kv = [int(x) for x in kv_len.cpu()]
        check_attend(out, qr, S, 0, pool=S.d_pool.cpu().numpy())
        eager_q = cache.append(batch, k, v, q=qf, rope=rope)
        assert torch.equal(eager_q, qr) and torch.equal(cache.attend(batch, eager_q), out)


def test_two_streams_at_once():
    """Calls on two caches from two streams do not meet: nothing is shared between calls."""
    sets = []
    for seed in (1, 2):
        S = Setup(128, 2, [1, 40], [1500, 60], seed=seed)
        q = attend_case(S, 2)
        sets.append((S, q, S.on_gpu(), torch.cuda.Stream()))
    ref = [c.attend(b, q) for _, q, (c, b), _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (_, q, (c, b), st) in enumerate(sets):
            with torch.cuda.stream(st):
                got[i].append(c.attend(b, q))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, ref[i]) for x in got[i])


def test_python_refusals():
    S = Setup(128, 2, [2], [3])
    q = attend_case(S, 2)
    cache, batch = S.on_gpu()
    k = torch.zeros(2, 2, 128, device="cuda")
    bad = [
        lambda: cache.attend(batch, q.float()),
        lambda: cache.attend(batch, q[:1]),
        lambda: cache.attend(batch, q.cpu()),
        lambda: cache.attend(batch, q[:, :3]),
        lambda: cache.attend(batch, q.transpose(1, 2)),
        lambda: cache.append(batch, k, k.bfloat16()),
        lambda: cache.append(batch, k.half(), k.half()),
        lambda: cache.append(batch, k, k, k_gamma=torch.ones(64, device="cuda")),
        lambda: cache.append(batch, k, k, k_gamma=torch.ones(128)),
        lambda: cache.read(batch, k=torch.empty(3, 2, 128, device="cuda").bfloat16()),
        lambda: q3t.KV4Cache(S.d_pool, S.d_table.long(), 2, 128),
        lambda: q3t.KV4Cache(S.d_pool, S.d_table, 4, 128),
        lambda: q3t.KV4Cache(S.d_pool.cpu(), S.d_table.cpu(), 2, 128),
        lambda: q3t.KV4Batch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1),
        lambda: q3t.KV4Batch(torch.zeros(3, dtype=torch.int32, device="cuda"),
                             torch.zeros(1, dtype=torch.int32, device="cuda"), 1),
        lambda: q3t.Rope(128, layout="other"),
    ]
    for f in bad:
        with pytest.raises(q3t.Q3TError) as e:
            f()
        assert e.value.status == q3t.INVALID_INPUT
    assert cache.attend(batch, q).shape == q.shape  # and the cache still works


def test_empty_calls():
    S = Setup(128, 2, [0, 0], [20, 0])
    S.kv = [20, 0]
    cache, batch = S.on_gpu(1, 20)
    e = torch.empty(0, 2, 128, device="cuda")
    assert cache.append(batch, e, e) is None
    assert cache.attend(batch, torch.empty(0, 4, 128, device="cuda").bfloat16()).shape == (0, 4, 128)
    k, v = cache.read(batch)
    assert k.shape == v.shape == (0, 2, 128)
