"""Performance cases of a token step's operators for models whose rotation is scaled, partial or restarts
with each packed document, whose scores are capped or biased by distance, and whose users sample by
temperature, top-k, top-p and min-p.

  tables   cos / sin tables of scaled rotary frequencies (vsl_rope_tables)
  append   rotation of part of each head and cache append of S prompt rows, rotary positions given row by
           row (vsl_rope_part_append)
  token    the same for the one row of a decode step (vsl_rope_part_append_decode)
  decode   attention of one position with a tanh cap, a distance bias and a range of keys (vsl_attn_decode_mods)
  prompt   the same for S prompt rows, each with its own range of keys (vsl_attn_prefill_mods)
  sample   one token for each row of logits (vsl_sample_rows)

Formulas.
  tables   f_j = theta^(-2j / rot) / ff_j for j < rot / 2 (ff: a file's own factors), then
             linear  f_j / factor
             llama3  with n_j = orig f_j / (2 pi) turns over the first context: f_j where n_j > high, f_j /
                     factor where n_j < low, between them a mix of both, s = (n_j - low) / (high - low) of f_j
             yarn    a mix, r_j of f_j / factor: r_j = (j - a) / max(b - a, 0.001) within 0..1, a = floor(c(high)),
                     b = ceil(c(low)), both within 0..rot - 1, c(n) = rot ln(orig / (2 pi n)) / (2 ln theta)
           cos, sin of p f_j, times the scale m (yarn: 0.1 ln(factor) + 1)
  append   the pairs (2i, 2i + 1) or (i, i + rot / 2) of the first rot dims turned by the tables' row of the row's
           rotary position; q out, k and v into the caches at pos0 + s
  decode, prompt
           s_k = scale q.k, capped: c tanh(s_k / c), then - slope_h |p - k|; softmax over the row's range of keys
           [begin, end) (without ranges: 0..p), a row without keys gives zeros
  sample   w_i = exp((l_i - max l) / T).  Kept: the first top_k tokens by logit (ties: lower index first); of those,
           in that order, the shortest run whose weights reach top_p of their sum; of those, w_i >= min_p.  The token
           is the first one, by index, whose running sum of kept weights exceeds u times their total.  T <= 0: the
           first maximum.  The other output is the token's share of the kept weights.

listed() names the cases, draw() gives more of the same ranges, prepare() makes a case's inputs on the GPU
from a seed, run() is one pass (`own`: the framework's calls, else plain torch in 32 bits, angles and
sampling weights in 64), exact() the same outputs in 64 bits, work() the bytes and operations of a pass.
"""
import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32
SPLITS = 32    # the engine's attention splits
ACT = 1.28     # spread of q, k, v: 0.02 * sqrt(4096) of a normalised input

# The repository's model configurations: query / KV heads, head_dim, RoPE theta.
GEOM = {
    "tiny": dict(nq=4, nkv=4, hd=64, theta=10000.0),
    "gqa3": dict(nq=6, nkv=2, hd=128, theta=500000.0),
    "1b": dict(nq=32, nkv=8, hd=64, theta=10000.0),
    "8b": dict(nq=32, nkv=8, hd=128, theta=500000.0),
    "70b": dict(nq=64, nkv=8, hd=128, theta=500000.0),
}
# Scalings of the rotary frequencies: kind, factor, first context, low and high turns.
SCALING = {
    "none": dict(type=0, factor=1.0, orig=0.0, low=0.0, high=0.0),
    "linear": dict(type=1, factor=4.0, orig=0.0, low=0.0, high=0.0),
    "llama3": dict(type=2, factor=8.0, orig=8192.0, low=1.0, high=4.0),
    "yarn": dict(type=3, factor=16.0, orig=4096.0, low=1.0, high=32.0),
}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the tables of the 8B model's 32768 positions, long-context scaling by turns
        dict(name="tables_8b_llama3", kind="tables", rot=128, rows=32768, pos0=0, theta=500000.0, scaling="llama3"),
        # the tables of a model that turns half of each 128-dim head, 131072 positions by yarn
        dict(name="tables_half_yarn", kind="tables", rot=64, rows=131072, pos0=0, theta=10000.0, scaling="yarn"),
        # one decode step's row of the 8B model, half of each head turned: launch bound
        dict(name="token_8b_half", kind="token", geom="8b", rot=64, pos=777, cap=4096, halves=True, kv="f16"),
        # a 2048-row chunk of packed documents (rotary positions restart), a quarter of each head turned, the engine's split q
        dict(name="append_8b_2048_packed", kind="append", geom="8b", rot=32, rows=2048, pos0=6144, cap=32768, halves=True,
             packed=True, kv="f16", q="f16x2"),
        # decode attention of a tiny model early in a generation, distance bias instead of rotation: the smallest call
        dict(name="decode_tiny_bias", kind="decode", geom="tiny", pos=40, begin=0, cap=2048, kv="f16", softcap=0.0, slopes=True),
        # capped scores at the end of the 8B model's 32768-position cache
        dict(name="decode_8b_capped", kind="decode", geom="8b", pos=32000, begin=0, cap=32768, kv="f16", softcap=50.0, slopes=False),
        # a short chat turn (odd length) behind 3001 cached positions, capped scores
        dict(name="prompt_8b_45_capped", kind="prompt", geom="8b", rows=45, pos0=3001, cap=4096, q="f16x2", softcap=50.0,
             slopes=False, mask="causal"),
        # 512 rows of packed documents of the 1B model, distance bias, single-plane q
        dict(name="prompt_1b_512_packed", kind="prompt", geom="1b", rows=512, pos0=0, cap=4096, q="f16", softcap=0.0,
             slopes=True, mask="packed"),
        # the last 2048-row chunk of an 8192-token prompt of the 8B model, capped scores, the engine's split q
        dict(name="prompt_8b_2048_capped", kind="prompt", geom="8b", rows=2048, pos0=6144, cap=32768, q="f16x2", softcap=30.0,
             slopes=False, mask="causal"),
        # one step of a chat with the engine's default parameters (temperature 0.7, top-k 40, top-p 0.9)
        dict(name="sample_1x32000", kind="sample", rows=1, vocab=32000, dtype="f32", params="default", spread=2.5),
        # one row of a large vocabulary by top-p alone
        dict(name="sample_1x131072_nucleus", kind="sample", rows=1, vocab=131072, dtype="f32", params="nucleus", spread=2.5),
        # a serving batch, every row with its own parameters
        dict(name="sample_64x131072_mixed", kind="sample", rows=64, vocab=131072, dtype="f32", params="mixed", spread=2.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed kinds' ranges; none costs more than the largest listed one."""
    kind = rng.choice(["tables", "append", "token", "decode", "decode", "prompt", "prompt", "sample", "sample"])
    if kind == "tables":
        return dict(kind=kind, rot=2 * rng.randint(5, 64), rows=_log(rng, 500, 65536), pos0=rng.choice([0, 0, 4097, 500000]),
                    theta=rng.choice([10000.0, 500000.0]), scaling=rng.choice(["none", "linear", "llama3", "yarn"]))
    if kind == "sample":
        rows, vocab = _log(rng, 1, 48), rng.choice([4096, 32000, _log(rng, 1000, 160000)])
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "f32", "f16"]),
                    params=rng.choice(["default", "nucleus", "mixed", "mixed"]), spread=rng.choice([1.0, 2.5, 5.0]))
    if kind in ("append", "token"):
        geom = rng.choice(["tiny", "gqa3", "8b", "70b"])
        hd, cap = GEOM[geom]["hd"], 4096
        case = dict(kind=kind, geom=geom, rot=2 * rng.randint(4, hd // 2), cap=cap, halves=rng.random() < 0.5,
                    kv=rng.choice(["f16", "f16", "f32"]))
        if kind == "token":
            return dict(case, pos=_log(rng, 3, cap - 2))
        rows = _log(rng, 2, 1200)
        return dict(case, rows=rows, pos0=rng.choice([0, _log(rng, 3, cap - rows)]), packed=rng.random() < 0.5,
                    q=rng.choice(["f32", "f16", "f16x2"]))
    geom = rng.choice(["tiny", "gqa3", "1b", "8b", "8b", "70b"])
    cap = 2048 if geom == "tiny" else 32768 if rng.random() < 0.4 else 4096
    case = dict(kind=kind, geom=geom, cap=cap, softcap=rng.choice([0.0, 30.0, 50.0, 50.0]), slopes=rng.random() < 0.4)
    if kind == "decode":
        pos = _log(rng, 3, cap - 2)
        return dict(case, pos=pos, begin=rng.choice([0, 0, pos // 3]), kv=rng.choice(["f16", "f16", "f16", "f32"]))
    rows = _log(rng, 2, {"tiny": 1024, "70b": 768}.get(geom, 1536))
    pos0 = 0 if rng.random() < 0.5 else _log(rng, 3, min(cap - rows, 6144))
    return dict(case, rows=rows, pos0=pos0, q=rng.choice(["f16", "f16x2", "f16x2"]), mask=rng.choice(["causal", "packed", "prefix"]))


def _bounds(case):
    """(begin, end) of the keys of each prompt row, as numpy; a row of padding has none."""
    S, p0 = case["rows"], case["pos0"]
    s = np.arange(S)
    begin, end = np.zeros(S, np.int64), p0 + s + 1
    if case["mask"] == "packed":  # documents of 150 to 260 rows, the first goes on from the cache; the last rows are padding
        at, step = 0, 150 + S % 37
        while at < S:
            n = min(step, S - at)
            begin[at:at + n] = 0 if at == 0 else p0 + at
            at, step = at + n, 150 + (step * 7) % 111
        pad = S // 40
        if pad:
            begin[S - pad:] = end[S - pad:] = 0
    elif case["mask"] == "prefix":  # the first third of the rows sees itself whole, both ways
        end = np.maximum(end, p0 + S // 3)
    return begin, end


def _positions(case):
    """Rotary positions of packed documents' rows."""
    s = np.arange(case["rows"])
    return s % 611 if case["packed"] else case["pos0"] + s


def work(case):
    """Bytes read and written once and operations of one pass."""
    kind = case["kind"]
    if kind == "tables":
        n = case["rows"] * (case["rot"] // 2)
        return {"bytes": 8 * n, "flops": 20 * n}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "f16" else 4) + 28 * case["rows"], "flops": 20 * n}
    g = GEOM[case["geom"]]
    nq, nkv, hd = g["nq"], g["nkv"], g["hd"]
    eb = 4 if case.get("kv") == "f32" else 2
    if kind in ("append", "token"):
        S = case.get("rows", 1)
        qb = {"f32": 4, "f16": 2, "f16x2": 4}[case.get("q", "f32")]
        angles = min(S, 611) if case.get("packed") else S
        return {"bytes": S * (4 * (nq + 2 * nkv) * hd + qb * nq * hd + eb * 2 * nkv * hd) + 4 * angles * case["rot"],
                "flops": 3 * S * (nq + nkv) * case["rot"]}
    if kind == "decode":
        n = case["pos"] + 1 - case["begin"]
        return {"bytes": eb * 2 * nkv * hd * n + 8 * nq * hd, "flops": 4 * nq * hd * n}
    begin, end = _bounds(case)
    S, pairs = case["rows"], int((end - begin).sum())
    seen = np.zeros(int(end.max()) + 1, np.int64)
    full = end > begin
    np.add.at(seen, begin[full], 1)
    np.add.at(seen, end[full], -1)
    keys = int((np.cumsum(seen) > 0).sum())
    qb = 2 * nq * hd * (2 if case["q"] == "f16x2" else 1)
    return {"bytes": 4 * nkv * hd * keys + S * (qb + 2 * nq * hd), "flops": 4 * nq * hd * pairs}


# ---------------------------------------------------------------------------------------------
# inputs, made from the seed alone
# ---------------------------------------------------------------------------------------------
def _rand(r, *shape, std=1.0):
    return torch.randn(shape, generator=r, device=DEV, dtype=F32) * std


def _tables(case, g, rows):
    j = torch.arange(case["rot"] // 2, device=DEV, dtype=F64)
    a = torch.arange(rows, device=DEV, dtype=F64)[:, None] * g["theta"] ** (-2.0 * j / case["rot"])
    return a.cos().float(), a.sin().float()


def _row_params(case, rng):
    """[rows, 4]: temperature, top-k, top-p, min-p (as float64; top-k whole)."""
    rows, kind = case["rows"], case["params"]
    p = np.zeros((rows, 4))
    if kind == "default":
        p[:] = (0.7, 40, 0.9, 0.0)
    elif kind == "nucleus":
        p[:] = (1.0, 0, 0.95, 0.0)
    else:  # users of one batch: greedy, all filters, single ones, none
        choices = [(0.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (1.2, 0, 1.0, 0.05), (0.8, 200, 0.95, 0.02),
                   (1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (1.5, 1000, 0.8, 0.0)]
        for i in range(rows):
            p[i] = choices[int(rng.integers(len(choices)))]
    return p


def _inputs(case, seed):
    kind = case["kind"]
    r = torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + 17) & 0x7FFFFFFF)
    rng = np.random.default_rng([int(seed) & 0x7FFFFFFF, 5])
    t = {}
    if kind == "tables":
        # a file's factors: near 1 where a pair turns fast, up to several times that where it turns slowly
        n = case["rot"] // 2
        t["ff"] = 1.0 + _rand(r, n).abs() * torch.linspace(0, 4, n, device=DEV)
        return None, t
    if kind == "sample":
        t["logits"] = _rand(r, case["rows"], case["vocab"], std=case["spread"]).to(F16 if case["dtype"] == "f16" else F32)
        p = _row_params(case, rng).astype(np.float32)
        packed = p.copy()
        packed[:, 1] = p[:, 1].astype(np.int32).view(np.float32)  # top_k is a whole number in the struct
        t["params"] = torch.from_numpy(packed).to(DEV)
        t["u"] = torch.rand(case["rows"], generator=r, device=DEV, dtype=F32)
        return None, t
    g = GEOM[case["geom"]]
    nq, nkv, hd, cap = g["nq"], g["nkv"], g["hd"], case["cap"]
    if kind in ("append", "token"):
        S = case.get("rows", 1)
        t["qkv"] = _rand(r, S, (nq + 2 * nkv) * hd, std=ACT)
        t["cos"], t["sin"] = _tables(case, g, cap)
        t["kc"], t["vc"] = (torch.zeros((nkv, cap, hd), device=DEV, dtype=F32 if case["kv"] == "f32" else F16) for _ in range(2))
        if kind == "append" and case["packed"]:
            t["positions"] = torch.from_numpy(_positions(case).astype(np.int32)).to(DEV)
        return g, t
    n = case["pos"] + 1 if kind == "decode" else case["pos0"] + case["rows"]
    kvt = F32 if case.get("kv") == "f32" else F16
    t["kc"], t["vc"] = (torch.zeros((nkv, cap, hd), device=DEV, dtype=kvt) for _ in range(2))
    t["kc"][:, :n] = _rand(r, nkv, n, hd).to(kvt)
    t["vc"][:, :n] = _rand(r, nkv, n, hd, std=ACT).to(kvt)
    t["slopes"] = 2.0 ** (-8.0 * torch.arange(1, nq + 1, device=DEV, dtype=F32) / nq) if case["slopes"] else None
    spread = 3.0  # scores of a few units, as trained models have; the cap bends the largest
    if kind == "decode":
        t["q"] = _rand(r, nq * hd, std=spread)
        t["ranges"] = torch.tensor([[case["begin"], 0x7FFFFFFF]], device=DEV, dtype=I32) if case["begin"] else None
    else:
        q = _rand(r, case["rows"], nq * hd, std=spread)
        hi = q.to(F16)
        t["q"] = torch.stack([hi, (q - hi.float()).to(F16)]) if case["q"] == "f16x2" else hi[None].clone()
        t["ranges"] = None
        if case["mask"] != "causal":
            t["ranges"] = torch.from_numpy(np.stack(_bounds(case), 1).astype(np.int32)).to(DEV)
    return g, t


class _State:
    def __init__(self, case, g, t):
        self.case, self.g, self.t, self.call, self.args, self.out, self.hold = case, g, t, None, None, None, None


def prepare(case, seed):
    return _State(case, *_inputs(case, seed))


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------
def _package():
    name = "vulkan_symbiote_loader_amd"  # the package's folder name has dashes
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join("vulkan-symbiote-loader_amd", "__init__.py"))
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _empty(*shape, dtype=F32):
    return torch.empty(shape, device=DEV, dtype=dtype)


def _bind(st):
    """The call of a pass, with the buffers and the control block that a user's program keeps."""
    vsl = _package()
    H, case, g, t, kind = vsl.hip(), st.case, st.g, st.t, st.case["kind"]
    if kind == "tables":
        s = SCALING[case["scaling"]]
        scaling = vsl.RopeScaling(type=s["type"], theta=case["theta"], factor=s["factor"], orig_ctx=s["orig"], low=s["low"],
                                  high=s["high"], mscale=0.0)
        cos, sin = (_empty(case["rows"], case["rot"] // 2) for _ in range(2))
        st.call, st.out = H.vsl_rope_tables, {"cos": cos, "sin": sin}
        args = (case["rot"], case["pos0"], case["rows"], ctypes.byref(scaling), t["ff"], cos, sin, None)
        st.hold = scaling
    elif kind == "sample":
        rows, V = t["logits"].shape
        tokens, probs = _empty(rows, dtype=I32), _empty(rows)
        n = H.vsl_sample_rows_ws_bytes(rows, V)
        ws = _empty(n, dtype=torch.uint8)
        dt = vsl.VSL_DT_F16 if case["dtype"] == "f16" else vsl.VSL_DT_F32
        st.call, st.out = H.vsl_sample_rows, {"tokens": tokens, "probs": probs}
        args = (t["logits"], dt, rows, V, V, t["params"], t["u"], tokens, probs, ws, n, None)
    else:
        nq, nkv, hd, cap = g["nq"], g["nkv"], g["hd"], case["cap"]
        kvdt = vsl.VSL_DT_F32 if case.get("kv") == "f32" else vsl.VSL_DT_F16
        qdt = {"f16": vsl.VSL_DT_F16, "f16x2": vsl.VSL_DT_F16X2, "f32": vsl.VSL_DT_F32}[case.get("q", "f32")]
        rope = vsl.ROPE_HALVES if case.get("halves") else vsl.ROPE_PAIRS
        ctrl = torch.tensor([case.get("pos", 0), 0, 0, 0, 1 << 30, 0, cap, 0], device=DEV, dtype=I32)
        scale = 1.0 / math.sqrt(hd)
        if kind == "append":
            S, p0 = case["rows"], case["pos0"]
            q = _empty(2 if case["q"] == "f16x2" else 1, S, nq * hd, dtype=F32 if case["q"] == "f32" else F16)
            st.call = H.vsl_rope_part_append
            args = (t["qkv"], S, nq, nkv, hd, case["rot"], rope, p0, t.get("positions"), t["cos"], t["sin"], cap, q, qdt,
                    t["kc"], t["vc"], kvdt, cap, None)
            # the remainder plane of a split q holds what the first one's rounding dropped
            st.out = {"q": q[0], "k": t["kc"][:, p0:p0 + S], "v": t["vc"][:, p0:p0 + S]}
        elif kind == "token":
            p, q = case["pos"], _empty(nq * hd)
            st.call = H.vsl_rope_part_append_decode
            args = (t["qkv"], nq, nkv, hd, case["rot"], rope, None, t["cos"], t["sin"], cap, q, t["kc"], t["vc"], kvdt, cap,
                    ctrl, None)
            st.out = {"q": q, "k": t["kc"][:, p:p + 1], "v": t["vc"][:, p:p + 1]}
        else:
            mods = vsl.AttnMods(softcap=case["softcap"], slopes=t["slopes"].data_ptr() if case["slopes"] else None,
                                ranges=t["ranges"].data_ptr() if t["ranges"] is not None else None)
            st.hold = mods
            if kind == "decode":
                po, pml, attn = _empty(nq * SPLITS * hd), _empty(nq * SPLITS * 2), _empty(nq * hd)
                st.call = H.vsl_attn_decode_mods
                args = (t["q"], t["kc"], t["vc"], kvdt, nq, nkv, hd, cap, scale, SPLITS, po, pml, attn, ctrl,
                        ctypes.byref(mods), None)
            else:
                S, p0 = case["rows"], case["pos0"]
                attn = _empty(S, nq * hd, dtype=F16)
                n = H.vsl_attn_prefill_mods_ws_bytes(S, p0, nq, nkv, hd)
                ws = _empty(max(n, 16), dtype=torch.uint8)
                st.call = H.vsl_attn_prefill_mods
                args = (t["q"], qdt, t["kc"], t["vc"], S, p0, nq, nkv, hd, cap, scale, attn, vsl.VSL_DT_F16,
                        ctypes.byref(mods), ws, n, None)
            st.out = {"attn": attn}
    st.hold = (st.hold, args)
    st.args = tuple(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _plain_tables(case, t):
    rot, s = case["rot"], SCALING[case["scaling"]]
    j = torch.arange(rot // 2, device=DEV, dtype=F64)
    f = case["theta"] ** (-2.0 * j / rot) / t["ff"].double()
    m = 1.0
    if case["scaling"] == "linear":
        f = f / s["factor"]
    elif case["scaling"] == "llama3":
        mix = ((s["orig"] * f / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        f = mix * f + (1 - mix) * f / s["factor"]
    elif case["scaling"] == "yarn":
        def dim(n):
            return rot * math.log(s["orig"] / (2 * math.pi * n)) / (2 * math.log(case["theta"]))
        a, b = (min(max(x, 0), rot - 1) for x in (math.floor(dim(s["high"])), math.ceil(dim(s["low"]))))
        mix = ((j - a) / max(b - a, 0.001)).clamp(0, 1)
        f = mix * f / s["factor"] + (1 - mix) * f
        m = 0.1 * math.log(s["factor"]) + 1
    a = (case["pos0"] + torch.arange(case["rows"], device=DEV, dtype=F64))[:, None] * f
    return {"cos": (a.cos() * m).float(), "sin": (a.sin() * m).float()}


def _plain_append(case, g, t):
    nq, nkv, hd, rot = g["nq"], g["nkv"], g["hd"], case["rot"]
    S, p0 = t["qkv"].shape[0], case["pos0"] if case["kind"] == "append" else case["pos"]
    y = t["qkv"].view(S, nq + 2 * nkv, hd)
    if case.get("packed"):
        cos, sin = t["cos"][t["positions"].long()][:, None], t["sin"][t["positions"].long()][:, None]
    else:
        cos, sin = t["cos"][p0:p0 + S, None], t["sin"][p0:p0 + S, None]
    x, rest = y[:, :nq + nkv, :rot], y[:, :nq + nkv, rot:]
    if case["halves"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:]
        x = torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        x = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)
    kvt = t["kc"].dtype
    q, k, v = x[:, :nq].flatten(1), x[:, nq:].transpose(0, 1).to(kvt), y[:, nq + nkv:].transpose(0, 1).to(kvt)
    t["kc"][:, p0:p0 + S], t["vc"][:, p0:p0 + S] = k, v
    if case["kind"] == "token":
        return {"q": q.flatten(), "k": k, "v": v}
    return {"q": q if case["q"] == "f32" else q.to(F16), "k": k, "v": v}


def _plain_attention(case, g, t):
    nq, nkv, hd = g["nq"], g["nkv"], g["hd"]
    decode = case["kind"] == "decode"
    S, p0 = (1, case["pos"]) if decode else (case["rows"], case["pos0"])
    n = p0 + S
    q = (t["q"] if decode else t["q"].float().sum(0)).view(S, nq, hd)
    K, V = t["kc"][:, :n].float(), t["vc"][:, :n].float()
    p, k = p0 + torch.arange(S, device=DEV)[:, None], torch.arange(n, device=DEV)
    if t["ranges"] is None:
        keep = k <= p
    else:
        keep = (k >= t["ranges"][:, :1]) & (k < t["ranges"][:, 1:])
    s = q.transpose(0, 1).reshape(nkv, nq // nkv * S, hd) @ K.transpose(1, 2) * (1.0 / math.sqrt(hd))
    s = s.view(nq, S, n)
    if case["softcap"]:
        s = case["softcap"] * (s / case["softcap"]).tanh()
    if case["slopes"]:
        s = s - t["slopes"][:, None, None] * (p - k).abs()
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - top.clamp(min=-1e30)).exp()
    o = (e.view(nkv, nq // nkv * S, n) @ V).view(nq, S, hd) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.transpose(0, 1)
    return {"attn": o.flatten() if decode else o.flatten(1).to(F16)}


def _plain_sample(t):
    l = t["logits"].double()
    rows, V = l.shape
    T, p, mp = (t["params"][:, i:i + 1].double() for i in (0, 2, 3))
    k = t["params"][:, 1].contiguous().view(I32).long()[:, None]
    k = torch.where(k == 0, V, k).clamp(max=V)
    greedy = T <= 0
    k = torch.where(greedy, 1, k)
    w = ((l - l.amax(1, keepdim=True)) / torch.where(greedy, 1.0, T)).exp()
    order = l.sort(dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    ws = torch.where(torch.arange(V, device=DEV) < k, ws, 0.0)
    before = ws.cumsum(1) - ws
    keep = (torch.arange(V, device=DEV) < k) & ((before < p * ws.sum(1, keepdim=True)) | (p >= 1)) & (ws >= mp)
    keep[:, 0] = True
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0.0)
    run_sum = w.cumsum(1)
    over = run_sum > t["u"].double()[:, None] * run_sum[:, -1:]
    token = torch.where(over, torch.arange(V, device=DEV), V).amin(1)
    prob = w.gather(1, token[:, None])[:, 0] / run_sum[:, -1]
    return {"tokens": token.to(I32), "probs": prob.float()}


def run(state):
    if own:
        if state.call is None:
            _bind(state)
        _package().check(state.call(*state.args))
        return state.out
    case, kind = state.case, state.case["kind"]
    if kind == "tables":
        return _plain_tables(case, state.t)
    if kind == "sample":
        return _plain_sample(state.t)
    return (_plain_append if kind in ("append", "token") else _plain_attention)(case, state.g, state.t)


# ---------------------------------------------------------------------------------------------
# the same outputs in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_tables(case, t):
    rot, s, kind = case["rot"], SCALING[case["scaling"]], case["scaling"]
    half = rot // 2
    freq, mag = np.empty(half), 1.0
    ff = t["ff"].cpu().numpy().astype(np.float64)
    ramp0 = ramp1 = 0.0
    if kind == "yarn":
        def at(turns):  # the pair that makes so many turns over the first context
            return rot * math.log(s["orig"] / (turns * 2 * math.pi)) / (2 * math.log(case["theta"]))
        ramp0 = min(max(math.floor(at(s["high"])), 0), rot - 1)
        ramp1 = min(max(math.ceil(at(s["low"])), 0), rot - 1)
        mag = 1.0 + 0.1 * math.log(s["factor"])
    for j in range(half):
        f = math.exp(-2.0 * j / rot * math.log(case["theta"])) / ff[j]
        if kind == "linear":
            f /= s["factor"]
        elif kind == "llama3":
            length = 2 * math.pi / f
            if length > s["orig"] / s["low"]:
                f /= s["factor"]
            elif length >= s["orig"] / s["high"]:
                a = (s["orig"] / length - s["low"]) / (s["high"] - s["low"])
                f = (1 - a) * f / s["factor"] + a * f
        elif kind == "yarn":
            a = min(max((j - ramp0) / max(ramp1 - ramp0, 0.001), 0.0), 1.0)
            f = f * (1 - a) + f / s["factor"] * a
        freq[j] = f
    p = torch.arange(case["pos0"], case["pos0"] + case["rows"], device=DEV, dtype=F64)
    angle = torch.outer(p, torch.from_numpy(freq).to(DEV))
    return {"cos": torch.cos(angle) * mag, "sin": torch.sin(angle) * mag}


def _exact_append(case, g, t):
    nq, nkv, hd, rot = g["nq"], g["nkv"], g["hd"], case["rot"]
    S = t["qkv"].shape[0]
    at = torch.from_numpy(_positions(case)).to(DEV) if case["kind"] == "append" else torch.tensor([case["pos"]], device=DEV)
    x = t["qkv"].to(F64).reshape(S, nq + 2 * nkv, hd).permute(1, 0, 2).clone()  # [heads, S, hd]
    c, s = t["cos"].to(F64)[at], t["sin"].to(F64)[at]
    i = torch.arange(rot // 2, device=DEV)
    one, two = (i, i + rot // 2) if case["halves"] else (2 * i, 2 * i + 1)
    for h in range(nq + nkv):
        y = x[h].clone()
        x[h][:, one] = y[:, one] * c - y[:, two] * s
        x[h][:, two] = y[:, two] * c + y[:, one] * s
    q = x[:nq].permute(1, 0, 2).reshape(S, nq * hd)
    return {"q": q.flatten() if case["kind"] == "token" else q, "k": x[nq:nq + nkv], "v": x[nq + nkv:]}


def _exact_attention(case, g, t):
    nq, nkv, hd = g["nq"], g["nkv"], g["hd"]
    if case["kind"] == "decode":
        S, p0, q = 1, case["pos"], t["q"].to(F64)
        begin, end = torch.tensor([case["begin"]], device=DEV), torch.tensor([p0 + 1], device=DEV)
    else:
        S, p0, q = case["rows"], case["pos0"], t["q"].to(F64).sum(0)
        begin, end = (torch.from_numpy(a).to(DEV) for a in _bounds(case))
    q = q.reshape(S, nq, hd).permute(1, 0, 2)
    n = p0 + S
    key = torch.arange(n, device=DEV)[None]
    hidden = (key < begin[:, None]) | (key >= end[:, None])
    none = (end <= begin)[:, None]
    far = (key - (p0 + torch.arange(S, device=DEV)[:, None])).abs().to(F64)
    out = torch.empty(S, nq, hd, device=DEV, dtype=F64)
    for h in range(nq):
        K, V = (t[c][h * nkv // nq, :n].to(F64) for c in ("kc", "vc"))
        s = q[h] @ K.T / math.sqrt(hd)
        if case["softcap"]:
            s = torch.tanh(s / case["softcap"]) * case["softcap"]
        if case["slopes"]:
            s = s - float(t["slopes"][h]) * far
        s = torch.where(hidden, torch.full_like(s, -math.inf), s)
        w = torch.where(none, torch.zeros_like(s), torch.softmax(s, 1))
        out[:, h] = w @ V
    return {"attn": out.flatten() if case["kind"] == "decode" else out.flatten(1)}


def _exact_sample(t):
    logits, u = t["logits"].cpu().numpy().astype(np.float64), t["u"].cpu().numpy().astype(np.float64)
    params = t["params"].cpu().numpy()
    ks = params[:, 1].copy().view(np.int32)
    tokens, probs = np.empty(len(logits), np.int32), np.empty(len(logits))
    for r, l in enumerate(logits):
        T, k, p, m = float(params[r, 0]), int(ks[r]), float(params[r, 2]), float(params[r, 3])
        order = np.lexsort((np.arange(l.size), -l))
        if T <= 0:
            tokens[r], probs[r] = order[0], 1.0
            continue
        order = order[:k] if k else order
        w = np.exp((l[order] - l[order[0]]) / T)
        if p < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))]
            w = w[:order.size]
        kept = np.sort(order[(w >= m) | (np.arange(order.size) == 0)])
        w = np.exp((l[kept] - l.max()) / T)
        c = np.cumsum(w)
        i = int(np.searchsorted(c, u[r] * c[-1], side="right"))
        tokens[r], probs[r] = kept[i], w[i] / c[-1]
    return {"tokens": torch.from_numpy(tokens).to(DEV), "probs": torch.from_numpy(probs).to(DEV)}


def exact(case, seed):
    g, t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "tables":
        return _exact_tables(case, t)
    if kind == "sample":
        return _exact_sample(t)
    return (_exact_append if kind in ("append", "token") else _exact_attention)(case, g, t)
