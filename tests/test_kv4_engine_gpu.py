"""The engine with per-head q / k norms, rotation by halves and a 4-bit KV cache against a 64-bit model of the same file
(kv4_ref's definitions), teacher-forced so that every step's logits are compared on the same history.

The engine's keys and values come from a 32-bit projection, so one in some ten thousand lies close enough to the border
of two codes to take the other: half a step each way around the exact value. The tolerance, 4e-3 of the largest logit,
leaves room for that (a flipped key moves one score of about a hundred by a step, 0.3 of its spread, of one of 64 or
128 dims: 0.3 / 8 on a weight of 1 / 100, 4e-4 of an output, at most a few times over 2 layers) and is a tenth of what
the rounding to 4 bits itself moves the logits by."""
import ctypes

import numpy as np
import pytest

import kv4_ref
import vsl_testlib

pytestmark = pytest.mark.gpu

TINY = dict(hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=4, intermediate_size=688, vocab_size=4096,
            max_position_embeddings=2048, rope_theta=10000.0, rms_eps=1e-5, dtype=0)
SMALL = dict(hidden_size=1024, num_layers=2, num_heads=8, num_kv_heads=2, intermediate_size=2816, vocab_size=2048,
             max_position_embeddings=4096, rope_theta=500000.0, rms_eps=1e-5, dtype=1)


class Model:
    """The token loop in 64 bits over a GGUF file's weights."""

    def __init__(self, vsl, path, cfg, kv4, halves, window):
        self.c, self.kv4, self.halves, self.window = cfg, kv4, halves, window
        self.lib, h = vsl.engine_lib(), ctypes.c_void_p()
        vsl.check(self.lib.vsl_gguf_open(str(path).encode(), ctypes.byref(h)), self.lib)
        self.h = h
        self.hd = cfg["hidden_size"] // cfg["num_heads"]

    def w(self, name, *shape):
        out = np.empty(int(np.prod(shape)), np.float32)
        n = self.lib.vsl_gguf_read_f32(self.h, name.encode(), out.ctypes.data_as(ctypes.c_void_p), out.size)
        if n == -30:
            return None
        assert n == out.size
        return out.reshape(shape).astype(np.float64)

    def norm(self, x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(self.c["rms_eps"]))) * g

    def logits(self, ids):
        """Logits after every token, one causal pass."""
        c, hd = self.c, self.hd
        d, nq, nkv, F, V = (c[k] for k in ("hidden_size", "num_heads", "num_kv_heads", "intermediate_size", "vocab_size"))
        S = len(ids)
        cos, sin = kv4_ref.tables(S, hd, c["rope_theta"])
        x = self.w("token_embd.weight", V, d)[ids]
        for l in range(c["num_layers"]):
            def t(n, *s):
                return self.w(f"blk.{l}.{n}.weight", *s)

            n = self.norm(x, t("attn_norm", d))
            qkv = np.concatenate([n @ t("attn_q", nq * hd, d).T, n @ t("attn_k", nkv * hd, d).T, n @ t("attn_v", nkv * hd, d).T], 1)
            q, k, v = kv4_ref.append(qkv, nq, nkv, hd, 0, t("attn_q_norm", hd), t("attn_k_norm", hd), c["rms_eps"], self.halves,
                                     cos, sin)
            if self.kv4:
                k, v = (kv4_ref.values(*kv4_ref.quantize(a)) for a in (k, v))
            elif c["dtype"] == 1:
                k, v = (a.astype(np.float16).astype(np.float64) for a in (k, v))
            a = kv4_ref.attend(q, k, v, 0, 1 / np.sqrt(hd), self.window).reshape(S, nq * hd)
            x = x + a @ t("attn_o", d, nq * hd).T
            n = self.norm(x, t("ffn_norm", d))
            g, u = n @ t("ffn_gate", F, d).T, n @ t("ffn_up", F, d).T
            x = x + (g / (1 + np.exp(-g)) * u) @ t("ffn_down", d, F).T
        return self.norm(x, self.w("output_norm.weight", d)) @ self.w("output.weight", V, d).T

    def close(self):
        self.lib.vsl_gguf_close(self.h)


CASES = [  # configuration, q / k norms, 4-bit cache, halves, window, prompt, steps, engine options
    (TINY, True, False, False, None, 20, 12, {}),
    (TINY, True, True, True, None, 37, 20, {}),
    (TINY, False, False, True, None, 9, 6, {}),
    (TINY, False, True, False, (16, 4, 24), 40, 12, {}),
    (SMALL, True, True, False, None, 150, 12, dict(prefill_chunk=64)),
    (SMALL, True, False, True, None, 70, 6, {}),
    (SMALL, False, True, True, (40, 8, 64), 130, 10, dict(prefill_chunk=48)),
    (SMALL, False, True, False, None, 61, 6, dict(batched_prefill=False)),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_engine(vsl, tmp_path, case):
    cfg, qk_norm, kv4, halves, window, n_prompt, steps, opts = CASES[case]
    rng = np.random.default_rng(case)
    path = tmp_path / "m.gguf"
    # weights of twice the usual spread, so that attention is not flat
    vsl.write_synthetic_gguf(path, cfg, seed=case, init_std=0.04, qk_norm=qk_norm)
    prompt, forced = rng.integers(0, cfg["vocab_size"], n_prompt), rng.integers(0, cfg["vocab_size"], steps)
    m = Model(vsl, path, cfg, kv4, halves, window)
    ref = m.logits(np.concatenate([prompt, forced[:-1]]))[n_prompt - 1:]
    m.close()
    hd = cfg["hidden_size"] // cfg["num_heads"]
    got = []
    for graph in (True, False):
        with vsl.Engine(path, kv_capacity=200, kv4=kv4, rope_halves=halves, window=window, use_graph=graph, **opts) as e:
            toks, lg = e.generate_ids(prompt, steps, return_logits=True, forced=forced)
            dt = vsl.VSL_DT_KV4 if kv4 else cfg["dtype"]
            assert e.kv_bytes() == 2 * cfg["num_layers"] * vsl.hip().vsl_kv_cache_bytes(dt, cfg["num_kv_heads"], 200, hd)
            got.append(lg)
            again = e.generate_ids(prompt, steps, return_logits=True, forced=forced)[1]  # over the first run's cache
            assert np.array_equal(again, lg)
            for op in range(6):
                assert e.time_op(op, 1) > 0
    assert np.array_equal(*got)
    scale = np.abs(ref).max()
    assert np.abs(got[0] - ref).max() <= 4e-3 * scale
    assert np.array_equal(toks, got[0].argmax(1))


def test_engine_refuses_partial_norms(vsl, tmp_path):
    """A file with query / key norms in one layer only is not opened."""
    path = tmp_path / "m.gguf"
    vsl.write_synthetic_gguf(path, TINY, qk_norm=True)
    data = path.read_bytes()
    assert data.count(b"blk.1.attn_k_norm.weight") == 1
    path.write_bytes(data.replace(b"blk.1.attn_k_norm.weight", b"blk.1.attn_k_nurm.weight"))
    with pytest.raises(vsl.VslError):
        vsl.Engine(path)
