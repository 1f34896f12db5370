"""Performance cases of the 4-bit KV cache and of the query / key norms that write it.

The operators are the attention stage of a Llama-style decoder between the QKV projection and the O
projection, with the cache held in 4 bits (VSL_DT_KV4) and with an RMSNorm on every query and key head:

  rows     the append of S prompt rows: per-head norms of q and k, rotation, q out, k and v into the cache
           (vsl_qk_norm_rope_append), the appended rows read back as the values they stand for (vsl_kv4_read)
  decode   attention of one position over the cache (vsl_attn_decode, vsl_attn_decode_window)
  token    both for one decode step (vsl_qk_norm_rope_append_decode, then vsl_attn_decode), captured into a
           graph as the engine captures its steps, the new row read back
  prompt   causal attention of S prompt rows over the cache (vsl_attn_prefill_kv4)

The 4-bit form: 32 consecutive head dims of a position are a block with a step d (7 significant bits, at
least 2^-14) and a zero point z; the code n (0..15) stands for (n - z) d.  With lo = min(0, x), hi =
max(0, x) over the block: d = the smallest such number >= (hi - lo) / 15, z = rint(-lo / d), n =
clamp(rint(x / d) + z, 0, 15).  A cache of `cap` positions (rounded up to P, a multiple of 128) holds, from
its first byte, the codes and then, at a multiple of 256 bytes, the steps (binary16, z in the four low bits):
  K  codes [n_kv][P][hd / 8] words of 8 dims, steps [n_kv][P][hd / 32]
  V  codes [n_kv][P / 8][hd] words of 8 positions, steps [n_kv][P / 8][hd / 32][8]
with value e of a word's eight in the nibble e / 2 + 4 (e % 2).

listed() names the cases, draw() gives more of the same ranges, prepare() makes a case's inputs on the GPU
from a seed, run() is one pass (`own`: the framework's calls, else plain torch in 32 bits, the codes'
choice in 64), exact() the same outputs in 64 bits, work() the bytes and operations of a pass.
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
F16, F32, F64 = torch.float16, torch.float32, torch.float64
EPS = float(np.float32(1e-5))
SPLITS = 32                # the engine's attention splits
ACT = 1.28                 # spread of q, k, v: 0.02 * sqrt(4096) of a normalised input
WINDOW = (512, 16, 8192)   # the windowed mode's window, global tokens and threshold

# The repository's model configurations: query / KV heads, head_dim, RoPE theta.
GEOM = {
    "tiny": dict(nq=4, nkv=4, hd=64, theta=10000.0),
    "gqa3": dict(nq=6, nkv=2, hd=128, theta=500000.0),
    "1b": dict(nq=32, nkv=8, hd=64, theta=10000.0),
    "8b": dict(nq=32, nkv=8, hd=128, theta=500000.0),
    "70b": dict(nq=64, nkv=8, hd=128, theta=500000.0),
}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the attention stage of a tiny model's decode step early in a generation: launch bound, the smallest call
        dict(name="token_tiny", kind="token", geom="tiny", pos=40, cap=2048, norm=True, halves=False),
        # the same stage of the 8B model in the middle of its 512 generated tokens: the main decode workload
        dict(name="token_8b", kind="token", geom="8b", pos=777, cap=4096, norm=True, halves=False),
        # and deep in a long context, where a 4-bit cache counts
        dict(name="token_8b_long", kind="token", geom="8b", pos=20011, cap=32768, norm=True, halves=True),
        # decode attention of the 1B model after its 128-token prompt (head_dim 64)
        dict(name="decode_1b", kind="decode", geom="1b", pos=255, cap=4096, window=False),
        # decode attention at the end of an 8B model's 32768-position cache
        dict(name="decode_8b_long", kind="decode", geom="8b", pos=32000, cap=32768, window=False),
        # the windowed mode past its threshold: 16 global positions and the last 513
        dict(name="decode_8b_window", kind="decode", geom="8b", pos=20011, cap=32768, window=True),
        # a short chat turn (odd length) appended behind 13 cached positions: partial 8-position words at both ends
        dict(name="rows_8b_45", kind="rows", geom="8b", rows=45, pos0=13, cap=4096, kv="kv4", norm=True, halves=True, q="f16x2"),
        # a 512-token prompt of the 1B model with q / k norms and an fp16 cache
        dict(name="rows_1b_512_f16", kind="rows", geom="1b", rows=512, pos0=0, cap=4096, kv="f16", norm=True, halves=False,
             q="f16"),
        # the last 2048-row chunk of an 8192-token prompt of the 8B model
        dict(name="rows_8b_2048_at_6144", kind="rows", geom="8b", rows=2048, pos0=6144, cap=32768, kv="kv4", norm=True,
             halves=False, q="f16x2"),
        # prompt attention of a short chat turn (odd length)
        dict(name="prompt_8b_45", kind="prompt", geom="8b", rows=45, pos0=0, cap=4096, q="f16x2", window=False),
        # prompt attention of the 1B model's 512-token prompt, single-plane q
        dict(name="prompt_1b_512", kind="prompt", geom="1b", rows=512, pos0=0, cap=4096, q="f16", window=False),
        # prompt attention of the last 2048-row chunk of an 8192-token prompt, the engine's split q
        dict(name="prompt_8b_2048_at_6144", kind="prompt", geom="8b", rows=2048, pos0=6144, cap=32768, q="f16x2", window=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed kinds' ranges; none costs more than the largest listed one."""
    kind = rng.choice(["token", "token", "decode", "decode", "rows", "rows", "prompt", "prompt"])
    geom = rng.choice(["tiny", "gqa3", "1b", "8b", "8b", "70b"])
    cap = 2048 if geom == "tiny" else 32768 if rng.random() < 0.4 else 4096
    if kind in ("token", "decode"):
        case = dict(kind=kind, geom=geom, pos=_log(rng, 3, cap - 2), cap=cap)
        if kind == "decode":
            return dict(case, window=cap == 32768 and rng.random() < 0.3)
        return dict(case, norm=rng.random() < 0.8, halves=rng.random() < 0.5)
    rows = _log(rng, 2, {"tiny": 1024, "70b": 768}.get(geom, 1536))
    pos0 = 0 if rng.random() < 0.5 else _log(rng, 3, min(cap - rows, 6144))
    case = dict(kind=kind, geom=geom, rows=rows, pos0=pos0, cap=cap, q=rng.choice(["f16", "f16x2", "f16x2"]))
    if kind == "prompt":
        return dict(case, window=False)
    return dict(case, kv=rng.choice(["kv4", "kv4", "kv4", "f16"]), norm=rng.random() < 0.8, halves=rng.random() < 0.5)


def _attended(case):
    n = case["pos"] + 1
    return WINDOW[0] + WINDOW[1] + 1 if case.get("window") and n > WINDOW[2] else n


def work(case):
    """Bytes read and written once and operations of one pass."""
    g = GEOM[case["geom"]]
    nq, nkv, hd = g["nq"], g["nkv"], g["hd"]
    row4 = 2 * nkv * (hd // 2 + hd // 16)  # K and V of one position in 4 bits
    width, attn = (nq + 2 * nkv) * hd, 4 * nq * hd
    if case["kind"] in ("decode", "token"):
        n = _attended(case)
        w = {"bytes": row4 * n + 8 * nq * hd, "flops": attn * n}
        if case["kind"] == "token":
            w["bytes"] += 4 * width + 12 * hd + row4 + 4 * nkv * hd
            w["flops"] += 8 * width
        return w
    S, p0 = case["rows"], case["pos0"]
    qb = 2 * nq * hd * (2 if case["q"] == "f16x2" else 1)
    if case["kind"] == "rows":
        back = row4 + 4 * nkv * hd if case["kv"] == "kv4" else 0  # the rows read back as binary16
        row = row4 if case["kv"] == "kv4" else 4 * nkv * hd
        return {"bytes": S * (4 * width + 4 * hd + qb + row + back) + 8 * hd, "flops": 8 * S * width}
    return {"bytes": row4 * (p0 + S) + S * (qb + 2 * nq * hd), "flops": attn * (S * p0 + S * (S + 1) // 2)}


# ---------------------------------------------------------------------------------------------
# the 4-bit form in plain torch
# ---------------------------------------------------------------------------------------------
def _positions(cap):
    return (cap + 127) // 128 * 128


def _steps_at(nkv, cap, hd):
    """Byte offset of a cache's steps: the codes' bytes, rounded up to a multiple of 256."""
    return (nkv * _positions(cap) * hd // 2 + 255) // 256 * 256


def _cache_bytes(nkv, cap, hd):
    return _steps_at(nkv, cap, hd) + nkv * _positions(cap) * (hd // 32) * 2


def _quantize(x):
    """(codes, zero points, steps) of the blocks of x [..., hd], in 64 bits."""
    b = x.double().unflatten(-1, (-1, 32))
    lo, hi = b.amin(-1).clamp(max=0.0), b.amax(-1).clamp(min=0.0)
    low = (1 << 46) - 1  # the significand's bits below the seven kept
    d = ((((hi - lo) / 15.0).view(torch.int64) + low) & ~low).view(F64).clamp(min=2.0 ** -14)
    z = (-lo / d).round()
    n = ((b / d[..., None]).round() + z[..., None]).clamp(0, 15)
    return n.flatten(-2).long(), z.long(), d


def _values(n, z, d):
    """What codes stand for, exact in 32 bits."""
    return ((n.unflatten(-1, (-1, 32)) - z[..., None]).float() * d.float()[..., None]).flatten(-2)


def _words(n):
    """Codes [..., 8] as 32-bit words."""
    at = torch.tensor([4 * (e // 2 + 4 * (e % 2)) for e in range(8)], device=n.device)
    w = (n << at).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _pack(x, cap, is_v):
    """Rows x [n_kv, n, hd] of a cache of `cap` positions, as its bytes."""
    nkv, n, hd = x.shape
    P = _positions(cap)
    buf = torch.zeros(_cache_bytes(nkv, cap, hd), device=x.device, dtype=torch.uint8)
    at = _steps_at(nkv, cap, hd)
    codes = buf[:nkv * P * hd // 2].view(torch.int32)
    steps = buf[at:].view(torch.int16)
    if not n:
        return buf
    if n % 8:
        x = torch.cat([x, x.new_zeros(nkv, 8 - n % 8, hd)], 1)
    for h in range(nkv):
        c, z, d = _quantize(x[h])
        m = c.shape[0]
        s = (d.to(F16).view(torch.int16).long() | z).to(torch.int16)
        if is_v:
            codes.view(nkv, P // 8, hd)[h, :m // 8] = _words(c.view(m // 8, 8, hd).transpose(1, 2))
            steps.view(nkv, P // 8, hd // 32, 8)[h, :m // 8] = s.view(m // 8, 8, hd // 32).transpose(1, 2)
        else:
            codes.view(nkv, P, hd // 8)[h, :m] = _words(c.view(m, hd // 8, 8))
            steps.view(nkv, P, hd // 32)[h, :m] = s
    return buf


def _unpack(buf, n, nkv, cap, hd, is_v):
    """The first n rows of every head, [n_kv, n, hd] in 32 bits."""
    P, m = _positions(cap), (n + 7) // 8 * 8
    codes = buf[:nkv * P * hd // 2].view(torch.int32)
    steps = buf[_steps_at(nkv, cap, hd):].view(torch.int16)
    at = torch.tensor([4 * (e // 2 + 4 * (e % 2)) for e in range(8)], device=buf.device, dtype=torch.int32)
    if is_v:
        c = ((codes.view(nkv, P // 8, 1, hd)[:, :m // 8] >> at[:, None]) & 15).reshape(nkv, m, hd)
        s = steps.view(nkv, P // 8, hd // 32, 8)[:, :m // 8].transpose(2, 3).reshape(nkv, m, hd // 32)
    else:
        c = ((codes.view(nkv, P, hd // 8, 1)[:, :m] >> at) & 15).reshape(nkv, m, hd)
        s = steps.view(nkv, P, hd // 32)[:, :m]
    return _values(c, s & 15, (s & -16).view(F16))[:, :n]


# ---------------------------------------------------------------------------------------------
# inputs, made from the seed alone
# ---------------------------------------------------------------------------------------------
def _rand(r, *shape, std=1.0):
    return torch.randn(shape, generator=r, device=DEV, dtype=F32) * std


def _tables(g, cap):
    j = torch.arange(g["hd"] // 2, device=DEV, dtype=F64)
    a = torch.arange(cap, device=DEV, dtype=F64)[:, None] * g["theta"] ** (-2.0 * j / g["hd"])
    return a.cos().float(), a.sin().float()


def _inputs(case, seed):
    g = GEOM[case["geom"]]
    nq, nkv, hd, cap, kind = g["nq"], g["nkv"], g["hd"], case["cap"], case["kind"]
    r = torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + 17) & 0x7FFFFFFF)
    t = {}
    if kind in ("rows", "token"):
        t["qkv"] = _rand(r, case.get("rows", 1), (nq + 2 * nkv) * hd, std=ACT)
        t["gq"], t["gk"] = (1.0 + _rand(r, hd, std=0.1) if case["norm"] else None for _ in range(2))
        t["cos"], t["sin"] = _tables(g, cap)
    if kind == "rows":  # a cache whose earlier positions are not read
        if case["kv"] == "kv4":
            t["kc"], t["vc"] = (torch.zeros(_cache_bytes(nkv, cap, hd), device=DEV, dtype=torch.uint8) for _ in range(2))
        else:
            t["kc"], t["vc"] = (torch.zeros((nkv, cap, hd), device=DEV, dtype=F16) for _ in range(2))
        return g, t
    n = {"token": case.get("pos"), "decode": case.get("pos", 0) + 1, "prompt": case.get("pos0", 0) + case.get("rows", 0)}[kind]
    t["kc"] = _pack(_rand(r, nkv, n, hd), cap, False)  # keys as their norm leaves them
    t["vc"] = _pack(_rand(r, nkv, n, hd, std=ACT), cap, True)
    if kind == "decode":
        t["q"] = _rand(r, nq * hd)
    elif kind == "prompt":
        q = _rand(r, case["rows"], nq * hd)
        hi = q.to(F16)
        t["q"] = torch.stack([hi, (q - hi.float()).to(F16)]) if case["q"] == "f16x2" else hi[None].clone()
    return g, t


class _State:
    def __init__(self, case, g, t):
        self.case, self.g, self.t = case, g, t
        self.calls, self.hold, self.out, self.graph = [], [], None, None

    def add(self, fn, *args):
        self.calls.append((fn, tuple(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args)))
        self.hold.append(args)

    def __del__(self):
        if self.graph:
            torch.cuda.synchronize()
            _package().hip().vsl_graph_destroy(self.graph)


def _package():
    name = "vulkan_symbiote_loader_amd"  # the package's folder name has dashes
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join("vulkan-symbiote-loader_amd", "__init__.py"))
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _capture(vsl, st):
    """The calls so far as one graph, replayed on the default stream (a decode step is captured once)."""
    H, s, g = vsl.hip(), ctypes.c_void_p(), ctypes.c_void_p()
    torch.cuda.synchronize()
    vsl.check(H.vsl_stream_create(ctypes.byref(s)))
    vsl.check(H.vsl_graph_begin(s))
    for fn, args in st.calls:
        vsl.check(fn(*args, s))
    vsl.check(H.vsl_graph_end(s, ctypes.byref(g)))
    vsl.check(H.vsl_stream_sync(s))
    vsl.check(H.vsl_stream_destroy(s))
    st.graph = g


def _zeros(*shape, dtype=F32):
    return torch.zeros(shape, device=DEV, dtype=dtype)


def _bind(st):
    """The framework's calls of a pass, with the buffers and the control block that a user's program keeps."""
    vsl = _package()
    H, case, g, t = vsl.hip(), st.case, st.g, st.t
    nq, nkv, hd, cap, kind = g["nq"], g["nkv"], g["hd"], case["cap"], case["kind"]
    scale = 1.0 / math.sqrt(hd)
    qdt = {"f16": vsl.VSL_DT_F16, "f16x2": vsl.VSL_DT_F16X2}.get(case.get("q"))
    rope = vsl.ROPE_HALVES if case.get("halves") else vsl.ROPE_PAIRS
    st.out = {}
    if kind in ("token", "decode"):
        ctrl = torch.tensor([case["pos"], 0, 0, 0, 1 << 30, 0, cap, 0], device=DEV, dtype=torch.int32)
        po, pml, attn = _zeros(nq * SPLITS * hd), _zeros(nq * SPLITS * 2), _zeros(nq * hd)
        q = t["q"] if kind == "decode" else _zeros(nq * hd)
        if kind == "token":
            k, v = _zeros(nkv, 1, hd, dtype=F16), _zeros(nkv, 1, hd, dtype=F16)
            st.add(H.vsl_qk_norm_rope_append_decode, t["qkv"], nq, nkv, hd, t["gq"], t["gk"], EPS, rope, t["cos"], t["sin"],
                   q, t["kc"], t["vc"], vsl.VSL_DT_KV4, cap, ctrl)
            st.out.update(q=q, k=k, v=v)
        args = (q, t["kc"], t["vc"], vsl.VSL_DT_KV4, nq, nkv, hd, cap, scale, SPLITS, po, pml, attn, ctrl)
        if case.get("window"):
            st.add(H.vsl_attn_decode_window, *args, *WINDOW)
        else:
            st.add(H.vsl_attn_decode, *args)
        if kind == "token":
            st.add(H.vsl_kv4_read, t["kc"], t["vc"], nkv, cap, hd, case["pos"], 1, k, v, vsl.VSL_DT_F16)
        st.out["attn"] = attn
        _capture(vsl, st)
    elif kind == "rows":
        S, p0, kv4 = case["rows"], case["pos0"], case["kv"] == "kv4"
        q = _zeros(2 if case["q"] == "f16x2" else 1, S, nq * hd, dtype=F16)
        st.add(H.vsl_qk_norm_rope_append, t["qkv"], S, nq, nkv, hd, p0, t["gq"], t["gk"], EPS, rope, t["cos"], t["sin"], q,
               qdt, t["kc"], t["vc"], vsl.VSL_DT_KV4 if kv4 else vsl.VSL_DT_F16, cap, None)
        if kv4:
            k, v = _zeros(nkv, S, hd, dtype=F16), _zeros(nkv, S, hd, dtype=F16)
            st.add(H.vsl_kv4_read, t["kc"], t["vc"], nkv, cap, hd, p0, S, k, v, vsl.VSL_DT_F16, None)
        else:
            k, v = t["kc"][:, p0:p0 + S], t["vc"][:, p0:p0 + S]
        st.out.update(q=q[0], k=k, v=v)  # the remainder plane of a split q holds what the first one's rounding dropped
    else:
        out = _zeros(case["rows"], nq * hd, dtype=F16)
        st.add(H.vsl_attn_prefill_kv4, t["q"], qdt, t["kc"], t["vc"], case["rows"], case["pos0"], nq, nkv, hd, cap, scale, out,
               vsl.VSL_DT_F16, None)
        st.out["attn"] = out
    torch.cuda.synchronize()


def prepare(case, seed):
    g, t = _inputs(case, seed)
    st = _State(case, g, t)
    if own:
        _bind(st)
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _append(case, g, t, p0):
    """q [S, nq, hd], k and v [nkv, S, hd] after the norms and the rotation, in 64 bits (the codes' choice
    hangs on values next to a border)."""
    nq, nkv, hd = g["nq"], g["nkv"], g["hd"]
    S = t["qkv"].shape[0]
    y = t["qkv"].double().view(S, nq + 2 * nkv, hd)
    cos, sin = t["cos"][p0:p0 + S, None].double(), t["sin"][p0:p0 + S, None].double()

    def rotated(x, gain):
        if gain is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gain.double()
        if case["halves"]:
            a, b = x[..., :hd // 2], x[..., hd // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    q, k = rotated(y[:, :nq], t["gq"]), rotated(y[:, nq:nq + nkv], t["gk"])
    return q, k.transpose(0, 1), y[:, nq + nkv:].transpose(0, 1)


def _attend(case, g, q, K, V, p0):
    """Causal attention of q [S, nq, hd] at positions p0.. over the rows K, V [n_kv, n, hd], in 32 bits."""
    S, nq, hd = q.shape
    nkv, n = K.shape[:2]
    p, j = p0 + torch.arange(S, device=DEV)[:, None], torch.arange(n, device=DEV)
    keep = j <= p
    if case.get("window"):
        keep &= (p + 1 <= WINDOW[2]) | (j < WINDOW[1]) | (j >= p - WINDOW[0])
    s = q.transpose(0, 1).reshape(nkv, nq // nkv * S, hd) @ K.transpose(1, 2) * (1.0 / math.sqrt(hd))
    s = s.view(nq, S, n).masked_fill(~keep, -math.inf)
    e = (s - s.amax(-1, keepdim=True)).exp()
    o = (e.view(nkv, nq // nkv * S, n) @ V).view(nq, S, hd) / e.sum(-1, keepdim=True)
    return o.transpose(0, 1)


def _plain(st):
    case, g, t = st.case, st.g, st.t
    nq, nkv, hd, cap, kind = g["nq"], g["nkv"], g["hd"], case["cap"], case["kind"]

    def cached(n):
        return (_unpack(t[c], n, nkv, cap, hd, c == "vc") for c in ("kc", "vc"))

    if kind == "rows":
        q, k, v = _append(case, g, t, case["pos0"])
        if case["kv"] == "kv4":
            k, v = _values(*_quantize(k)), _values(*_quantize(v))
        return {"q": q.flatten(1).to(F16), "k": k.to(F16), "v": v.to(F16)}
    if kind == "token":
        q, k, v = _append(case, g, t, case["pos"])
        q, k, v = q.float(), _values(*_quantize(k)), _values(*_quantize(v))
        K, V = (torch.cat([x, y], 1) for x, y in zip(cached(case["pos"]), (k, v)))
        a = _attend(case, g, q, K, V, case["pos"])
        return {"q": q.flatten(), "k": k.to(F16), "v": v.to(F16), "attn": a.flatten()}
    if kind == "decode":
        a = _attend(case, g, t["q"].view(1, nq, hd), *cached(case["pos"] + 1), case["pos"])
        return {"attn": a.flatten()}
    q = t["q"].float().sum(0).view(-1, nq, hd)
    a = _attend(case, g, q, *cached(case["pos0"] + case["rows"]), case["pos0"])
    return {"attn": a.flatten(1).to(F16)}


def run(state):
    if not own:
        return _plain(state)
    vsl = _package()
    if state.graph is not None:
        vsl.check(vsl.hip().vsl_graph_launch(state.graph, None))
    else:
        for fn, args in state.calls:
            vsl.check(fn(*args))
    return state.out


# ---------------------------------------------------------------------------------------------
# the same outputs in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_block(x):
    """The values that the 4-bit form of x [..., hd] stands for, from its definition: the step is found
    as 64..127 times a power of two."""
    shape = x.shape
    b = x.reshape(-1, 32)
    top = torch.maximum(b.max(1).values, torch.zeros_like(b[:, 0]))
    bottom = torch.minimum(b.min(1).values, torch.zeros_like(b[:, 0]))
    need = (top - bottom) / 15
    frac, e = torch.frexp(need)               # need = frac 2^e, frac in [0.5, 1)
    step = torch.ldexp(torch.ceil(torch.ldexp(frac, torch.full_like(e, 7))), e - 7)
    step = torch.where(step < 2.0 ** -14, torch.full_like(step, 2.0 ** -14), step)[:, None]
    zero = torch.round(-bottom[:, None] / step)
    code = torch.round(b / step) + zero
    code = torch.where(code < 0, torch.zeros_like(code), torch.where(code > 15, torch.full_like(code, 15.0), code))
    return ((code - zero) * step).reshape(shape)


def _exact_cache(buf, nkv, cap, hd, n, is_v):
    """The first n rows [nkv, n, hd] of a cache's bytes in 64 bits, byte by byte."""
    P, at = _positions(cap), _steps_at(nkv, cap, hd)
    b = buf[:nkv * P * hd // 2].view(-1, 4)                              # a word's bytes: elements (0, 2), (4, 6), (1, 3), (5, 7)
    e = torch.empty(b.shape[0], 8, device=DEV, dtype=torch.uint8)
    for byte, (first, second) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
        e[:, first], e[:, second] = b[:, byte] % 16, b[:, byte] // 16
    s = buf[at:].view(torch.int16).to(torch.int32)
    z = s % 16
    d = (s - z).to(torch.int16).view(F16).double()
    out = torch.empty(nkv, n, hd, device=DEV, dtype=F64)
    for h in range(nkv):
        if is_v:
            c = e.view(nkv, P // 8, hd, 8)[h].permute(0, 2, 1).reshape(P, hd)[:n]
            zz, dd = (a.view(nkv, P // 8, hd // 32, 8)[h].permute(0, 2, 1).reshape(P, hd // 32)[:n] for a in (z, d))
        else:
            c = e.view(nkv, P, hd)[h, :n]
            zz, dd = (a.view(nkv, P, hd // 32)[h, :n] for a in (z, d))
        out[h] = (c.double() - zz.double().repeat_interleave(32, 1)) * dd.repeat_interleave(32, 1)
    return out


def exact(case, seed):
    g, t = _inputs(case, seed)
    nq, nkv, hd, cap, kind = g["nq"], g["nkv"], g["hd"], case["cap"], case["kind"]
    res = {}
    if kind in ("rows", "token"):
        S, p0 = t["qkv"].shape[0], case["pos0"] if kind == "rows" else case["pos"]
        x = t["qkv"].to(F64).reshape(S, nq + 2 * nkv, hd).permute(1, 0, 2).clone()   # [heads, S, hd]
        c, s = t["cos"].to(F64)[p0:p0 + S], t["sin"].to(F64)[p0:p0 + S]
        first = torch.arange(hd // 2, device=DEV) if case["halves"] else torch.arange(0, hd, 2, device=DEV)
        second = first + (hd // 2 if case["halves"] else 1)
        for h in range(nq + nkv):
            y, gain = x[h], t["gq"] if h < nq else t["gk"]
            if gain is not None:
                y = y * gain.to(F64) * torch.rsqrt((y * y).sum(1, keepdim=True) / hd + EPS)
            z = torch.empty_like(y)
            z[:, first] = y[:, first] * c - y[:, second] * s
            z[:, second] = y[:, second] * c + y[:, first] * s
            x[h] = z
        q, k, v = x[:nq], x[nq:nq + nkv], x[nq + nkv:]
        if kind == "token" or case["kv"] == "kv4":
            k, v = _exact_block(k), _exact_block(v)
        res = {"q": q.permute(1, 0, 2).reshape(S, nq * hd), "k": k, "v": v}
        if kind == "rows":
            return res
        K, V = (torch.cat([_exact_cache(t[n], nkv, cap, hd, p0, n == "vc"), w], 1) for n, w in (("kc", k), ("vc", v)))
        res["q"] = res["q"].flatten()
    else:
        S, p0 = case.get("rows", 1), case["pos"] if kind == "decode" else case["pos0"]
        q = (t["q"].to(F64).sum(0) if kind == "prompt" else t["q"].to(F64)).reshape(S, nq, hd).permute(1, 0, 2)
        K, V = (_exact_cache(t[n], nkv, cap, hd, p0 + S, n == "vc") for n in ("kc", "vc"))
    attn = torch.empty(S, nq, hd, device=DEV, dtype=F64)
    key, at = torch.arange(K.shape[1], device=DEV)[None], p0 + torch.arange(S, device=DEV)[:, None]
    hidden = key > at
    if case.get("window"):
        hidden |= (at >= WINDOW[2]) & (key >= WINDOW[1]) & (key < at - WINDOW[0])
    for h in range(nq):
        w = torch.softmax((q[h] @ K[h * nkv // nq].T / math.sqrt(hd)).masked_fill(hidden, -math.inf), 1)
        attn[:, h] = w @ V[h * nkv // nq]
    res["attn"] = attn.flatten() if kind in ("token", "decode") else attn.flatten(1)
    return res
