"""The talker on a 4-bit key/value cache (q3t_session_start_kv4,
q3t_batch_create_kv4) against a float64 restatement of its decoder layer whose
cached keys and values pass through the 4-bit definition.

The talker has one layer here, full size otherwise: its keys then come from
inputs that both sides hold exactly, so both pick the same digits but for
values on a border (a few in a million, as f32 and f64 differ there), and what
is left is the tolerance of the other talker parity tests.  Past a first layer
the two sides' inputs differ by bf16 rounding flips, and a share of digits with
them, which no tolerance on logits tells from a fault."""
import numpy as np
import pytest

import kv4_ref as R
import q3t
import synthetic as S

pytestmark = pytest.mark.gpu

ATOL, RTOL = 2e-2, 1e-2


def assert_close(gpu, ref, what):
    gpu, ref = np.asarray(gpu, np.float64), np.asarray(ref, np.float64)
    bound = max(ATOL, RTOL * np.abs(ref).max())
    worst = np.abs(gpu - ref).max()
    assert worst <= bound, f"{what}: max err {worst:.3e} > {bound:.3e}"
    rel = np.linalg.norm(gpu - ref) / max(np.linalg.norm(ref), 1e-30)
    assert rel <= RTOL, f"{what}: relative L2 error {rel:.3e}"


def bf(x):
    return S.bf16_round(np.array(x, np.float32)).astype(np.float64)


def stored(x):
    n, s, z = R.quantise(x.astype(np.float32))
    return (n.reshape(*s.shape, 32) * s[..., None].astype(np.float64) + z[..., None]).reshape(x.shape)


class Layer4:
    """One decoder layer, the final norm and codec_head in float64 over a 4-bit cache."""

    def __init__(self, cfg, w):
        self.c, self.w = cfg.talker, w
        self.k, self.v = [], []  # [position][n_kv][head_dim], as stored

    def get(self, name):
        return np.asarray(self.w[f"talker.model.layers.0.{name}.weight"], np.float64)

    def norm(self, x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.eps) * g

    def forward(self, x):
        """(logits, hidden) of input rows x appended to the cache."""
        c = self.c
        x = np.asarray(x, np.float64)
        T, D, pos = len(x), c.head_dim, len(self.k) + np.arange(len(x))
        h = bf(self.norm(x, self.get("input_layernorm")))
        q, k, v = (h @ self.get(f"self_attn.{n}_proj").T for n in "qkv")
        f = R.frequencies(D, c.theta)
        q = bf(R.rotate(self.norm(q.reshape(T, -1, D), self.get("self_attn.q_norm")), pos, f, "half"))
        k = R.rotate(self.norm(k.reshape(T, -1, D), self.get("self_attn.k_norm")), pos, f, "half")
        self.k += list(stored(k))
        self.v += list(stored(v.reshape(T, -1, D)))
        K, V = np.array(self.k), np.array(self.v)
        out = np.zeros((T, c.n_heads, D))
        for i, p in enumerate(pos):
            for hd in range(c.n_heads):
                g = hd * c.n_kv // c.n_heads
                s = K[:p + 1, g] @ q[i, hd] / np.sqrt(D)
                e = np.exp(s - s.max())
                out[i, hd] = e @ V[:p + 1, g] / e.sum()
        x = x + bf(out.reshape(T, -1)) @ self.get("self_attn.o_proj").T
        h = bf(self.norm(x, self.get("post_attention_layernorm")))
        g, u = h @ self.get("mlp.gate_proj").T, h @ self.get("mlp.up_proj").T
        x = x + bf(g / (1 + np.exp(-g)) * u) @ self.get("mlp.down_proj").T
        hid = self.norm(x, np.asarray(self.w["talker.model.norm.weight"], np.float64))
        return bf(hid) @ np.asarray(self.w["talker.codec_head.weight"], np.float64).T, hid


@pytest.fixture(scope="module")
def small():
    cfg = S.TalkerConfig().small(talker_layers=1, predictor_layers=1)
    w = S.make_talker_weights(cfg, seed=0)
    model = q3t.Model(cfg, w, kv_pages=2048, max_active=8)
    yield cfg, w, model
    model.close()


@pytest.mark.parametrize("prompt_len", [1, 16, 70, 300])
def test_session_prompt_and_steps(small, prompt_len):
    cfg, w, model = small
    prompt, trailing, pad = S.synthetic_talker_inputs(cfg, prompt_len, seed=prompt_len)
    sess = model.session(prompt, trailing, pad, max_new_tokens=4, first_logits=True, kv_bits=4)
    twin = Layer4(cfg, w)
    logits, _ = twin.forward(prompt)
    assert_close(sess.first_logits, logits[-1], "prompt logits")
    g = np.random.default_rng(prompt_len)
    for step in range(3):
        emb = g.standard_normal(cfg.talker.hidden).astype(np.float32)
        got, hid = sess.decode_embeds(emb)
        logits, ref_hid = twin.forward(emb[None])
        assert_close(got, logits[0], f"logits of step {step}")
        assert_close(hid, ref_hid[0], f"hidden of step {step}")
    sess.close()


def frame_input(cfg, w, codes, extra):
    """The talker's next input row: the frame's code embeddings plus the trailing row (infer/mod.rs:343-383)."""
    x = np.asarray(w["talker.model.codec_embedding.weight"], np.float32)[codes[0]].astype(np.float32)
    for q in range(1, cfg.n_groups):
        x = x + np.asarray(w[f"talker.code_predictor.model.codec_embedding.{q - 1}.weight"], np.float32)[codes[q]]
    return x + extra


def test_batch_mixes_prompts_and_frames(small):
    """Eight slots: requests of different prompt lengths admitted over time, prompts in chunks beside decode tokens,
    every frame's logits against the restatement."""
    cfg, w, model = small
    lens, frames = [5, 100, 16, 260, 1, 33, 64, 17, 40], 6
    b = model.batch(max_active=8, kv_bits=4)
    reqs = []
    for i, n in enumerate(lens):
        prompt, trailing, pad = S.synthetic_talker_inputs(cfg, n, seed=100 + i)
        codes = S.teacher_codes(frames, seed=100 + i)
        first = np.zeros(cfg.talker.vocab, np.float32)
        rid = b.submit(prompt, trailing, pad, frames, forced=codes, first_logits=first)
        twin = Layer4(cfg, w)
        reqs.append(dict(rid=rid, twin=twin, codes=codes, first=first, trailing=trailing, pad=pad, frames=0,
                         ref_first=twin.forward(prompt)[0][-1]))
    for _ in range(60):
        before = [b.poll(r["rid"])[1] for r in reqs]
        b.step()
        for r, n in zip(reqs, before):
            state, done, _ = b.poll(r["rid"])
            if done == n:
                continue
            assert done == n + 1
            x = frame_input(cfg, w, r["codes"][n], r["trailing"][n] if n < len(r["trailing"]) else r["pad"])
            logits, _ = r["twin"].forward(x[None])
            if done < frames:  # a finished request left the frame
                assert_close(b.logits(r["rid"])[0], logits[0], f"request {r['rid']} frame {n}")
            r["frames"] = done
        if b.pending() == (0, 0):
            break
    for r in reqs:
        assert b.poll(r["rid"])[0] == 2 and r["frames"] == frames
        assert_close(r["first"], r["ref_first"], f"request {r['rid']} first logits")
        got, _, _ = b.take(r["rid"])
        np.testing.assert_array_equal(got, r["codes"].T)
    b.close()


def test_cache_saved_and_loaded(small):
    """load_kv quantises, read_kv gives what the digits stand for; a bf16 session gives the bits back."""
    cfg, w, model = small
    c = cfg.talker
    g = np.random.default_rng(4)
    k, v = (S.bf16_round(g.standard_normal((c.n_layers, c.n_kv, 53, c.head_dim)).astype(np.float32)) for _ in range(2))
    prompt, trailing, pad = S.synthetic_talker_inputs(cfg, 3)
    for bits in (16, 4):
        s = model.session(prompt, trailing, pad, max_new_tokens=4, kv_bits=bits)
        s.load_kv(S.bf16_bits(k), S.bf16_bits(v), 53)
        got = s.read_kv()
        for a, x in zip(got, (k, v)):
            ref = x if bits == 16 else stored(x).astype(np.float32)
            np.testing.assert_array_equal(a, S.bf16_bits(ref.copy()))
        # 54 positions after a step, and too small a buffer is refused
        s.decode_embeds(np.ones(c.hidden, np.float32))
        assert s.read_kv()[0].shape[2] == 54
        L = q3t.lib()
        buf = np.zeros(16, np.uint16).ctypes.data_as(q3t.C.POINTER(q3t.C.c_uint16))
        assert L.q3t_session_read_kv(s.h, buf, buf, 53, None) == q3t.INVALID_INPUT
        assert L.q3t_session_read_kv(s.h, buf, None, 54, None) == q3t.INVALID_INPUT
        s.close()


def test_session_continues_from_a_saved_cache(small):
    """A prompt's 4-bit cache saved and loaded into another 4-bit session: the next step matches attention over the
    saved values quantised once more."""
    cfg, w, model = small
    prompt, trailing, pad = S.synthetic_talker_inputs(cfg, 80, seed=9)
    a = model.session(prompt, trailing, pad, max_new_tokens=4, kv_bits=4)
    k, v = a.read_kv()
    a.close()
    b = model.session(prompt[:1], trailing, pad, max_new_tokens=4, kv_bits=4)
    b.load_kv(k, v, 80)
    twin = Layer4(cfg, w)
    val = lambda x: stored(R.bf16_value(x).reshape(x.shape)[0].transpose(1, 0, 2))  # noqa: E731
    twin.k, twin.v = list(val(k)), list(val(v))
    emb = np.random.default_rng(1).standard_normal(cfg.talker.hidden).astype(np.float32)
    got, _ = b.decode_embeds(emb)
    assert_close(got, twin.forward(emb[None])[0][0], "step on the loaded cache")
    b.close()


def test_pool_exhaustion_fails_one_request(small):
    cfg, w, _ = small
    model = q3t.Model(cfg, w, kv_pages=4, max_active=2)
    prompt, trailing, pad = S.synthetic_talker_inputs(cfg, 30, seed=3)
    s = model.session(prompt, trailing, pad, max_new_tokens=60, kv_bits=4)
    with pytest.raises(q3t.Q3TError) as e:
        for _ in range(60):
            s.step()
    assert e.value.status == q3t.OUT_OF_PAGES
    s.close()
    with pytest.raises(q3t.Q3TError) as e:
        model.session(prompt, trailing, pad, max_new_tokens=4, kv_bits=8)
    assert e.value.status == q3t.INVALID_INPUT
    model.close()


def test_eager_and_graph_frames_agree(small, monkeypatch):
    cfg, w, model = small
    out = []
    for graphs in ("1", "0"):
        monkeypatch.setenv("Q3T_GRAPHS", graphs)
        prompt, trailing, pad = S.synthetic_talker_inputs(cfg, 40, seed=6)
        s = model.session(prompt, trailing, pad, max_new_tokens=5, kv_bits=4)
        rows = [s.step_forced(c)[1] for c in S.teacher_codes(4, seed=6)]
        out.append(np.array(rows))
        s.close()
    np.testing.assert_array_equal(out[0], out[1])
