"""Operators of a transformer block with multi-axis rotary positions, differential attention and
norms on both sides of the block, as a program calls them: the cases, their inputs and the plain forms.

Device memory is torch's: the library takes device pointers, so a torch tensor's storage serves as input
or output of any call. The plain form computes in 32 bits (rotary angles in 64) from elementary torch
operations and rounds once; `own` makes the calls of the package instead.

The package's calls run on a stream of its runtime, which neither waits for torch's streams nor is waited for by them:
`prepare` waits for the device before and after it makes tensors, and a program that lets torch read a result, or drops a
state, waits for the device first (torch.cuda.synchronize). Passes over the same state follow each other.
"""
import ctypes
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one new row of each CFG arm, q and k heads at once: latency only
        _rope("rope_token", "f32", 2, 32, 64, (16, 24, 24), 1, 0, False),
        # the clip stream of 8 s at 8 frames a second with 16 x 16 patches, two arms: q and k heads
        # turned out of the wider q|k|v rows
        _rope("rope_video_f16", "f16", 32768, 32, 64, (16, 24, 24), 2, 1024, False),
        # halves instead of neighbours, wider heads, an odd row count, the tail of each head left as it is
        _rope("rope_half_bf16", "bf16", 4999, 24, 128, (32, 32, 48), 1, 0, True),
        # one block end of a few rows: latency only
        _norm("norm_rows_f32", 8, 1024, "f32", "f32", "f32", "rms", "rms", 4, True),
        # a fused block's end in the batch of eight prompts under CFG: f32 stream, f16 branch and operand
        _norm("norm_batch16", 6352, 1024, "f32", "f16", "f16", "rms", "ln", 397, True),
        # the video rows in a bf16 stream, modulated row by row
        _norm("norm_video_bf16", 32771, 2048, "bf16", "bf16", "bf16", "ln", "rms", 1, False),
        # joint rows of the 8 s clip under CFG, the unconditional arm's text padded
        _attn("diff_8s", "f16", 2, 397, 397, 8, 8, 64, False, True),
        # the 30 s clip, eight prompts under CFG
        _attn("diff_30s_b16", "bf16", 16, 1101, 1101, 8, 8, 64, False, False),
        # a long video context, an odd length
        _attn("diff_long", "f16", 1, 12289, 12289, 8, 8, 64, False, False),
        # causal prompts of unequal length with shared key and value heads, narrow maps
        _attn("diff_causal_gqa", "f16", 4, 2047, 2047, 16, 4, 32, True, True),
        # one new row against its cache: latency
        _attn("diff_token", "f16", 1, 1, 4099, 8, 8, 64, True, False),
        # one new row of 64 sequences against long caches of unequal length
        _attn("diff_cache", "bf16", 64, 1, 8192, 16, 4, 64, True, True),
    ]


def _rope(name, dtype, rows, nh, hd, dims, arms, pad, half):
    """pad: elements behind the turned heads in a row of x (v heads)"""
    return _named(name, {"op": "rope", "dtype": dtype, "rows": rows, "nh": nh, "hd": hd, "d0": dims[0], "d1": dims[1],
                         "d2": dims[2], "arms": arms, "pad": pad, "half": half})


def _norm(name, rows, H, x, f, y, post, pre, mod_rows, weights):
    return _named(name, {"op": "norm", "rows": rows, "H": H, "x": x, "f": f, "y": y, "post": post, "pre": pre,
                         "mod_rows": mod_rows, "weights": weights})


def _attn(name, dtype, B, Sq, Sk, nh, nkv, hd, causal, ragged):
    return _named(name, {"op": "attn", "dtype": dtype, "B": B, "Sq": Sq, "Sk": Sk, "nh": nh, "nkv": nkv, "hd": hd,
                         "causal": causal, "ragged": ragged})


def _named(name, case):
    return dict(case, name=name) if name else case


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "norm", "attn", "attn"])
    if op == "rope":
        dtype, hd = rng.choice(["f32", "f16", "bf16"]), rng.choice([32, 64, 80, 128])
        q = hd // 16
        a = 4 * rng.randint(1, q)
        b = 4 * rng.randint(1, q)
        arms = rng.choice([1, 2, 3])
        nh = rng.randint(2, 40)
        rows = arms * _log_int(rng, 1, min(32768, 60_000_000 // (nh * hd)) // arms)
        return _rope(None, dtype, rows, nh, hd, (a, b, 4 * rng.randint(0, (hd - a - b) // 4)), arms,
                     rng.choice([0, 0, hd * nh // 2, 24]), rng.random() < 0.5)
    if op == "norm":
        H = rng.choice([8 * _log_int(rng, 8, 512), _log_int(rng, 65, 4099)])
        rows = _log_int(rng, 1, min(32768, 64_000_000 // H))
        t = ["f32", "f16", "bf16"]
        return _norm(None, rows, H, rng.choice(t), rng.choice(t), rng.choice(t), rng.choice(["none", "rms", "ln"]),
                     rng.choice(["rms", "ln"]), rng.choice([1, _log_int(rng, 1, rows), rows]), rng.random() < 0.5)
    dtype, hd, causal, ragged = rng.choice(["f16", "bf16"]), rng.choice([32, 64, 64]), rng.random() < 0.5, rng.random() < 0.5
    nkv = rng.choice([1, 2, 4, 8])
    nh = nkv * rng.choice([1, 1, 2, 3, 4])
    B = rng.choice([1, 2, 2, 3, 4, 8, 16])
    if rng.random() < 0.4:   # a few new rows against a cache
        Sq = rng.choice([1, 1, 1, 2, 5, 16])
        Sk = _log_int(rng, 32, min(65536, 2_000_000 // (B * nkv)))
        return _attn(None, dtype, B, Sq, max(Sq, Sk), nh, nkv, hd, causal, ragged)
    Sk = _log_int(rng, 32, int(math.sqrt(500_000_000 // (B * nh))))
    return _attn(None, dtype, B, Sk if causal else _log_int(rng, 17, Sk), Sk, nh, nkv, hd, causal, ragged)


# ---------------------------------------------------------------- inputs

def _lengths(case):
    """(q_len, kv_len) of each sample: the same for every seed, so that work() can count them"""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    if not case["ragged"]:
        return [Sq] * B, [Sk] * B
    r = random.Random(1000003 * B + Sk)
    kv = [Sk] + [r.randint(max(1, Sk // 4), Sk) for _ in range(B - 1)]
    return ([Sq] * B if not case["causal"] or Sq < Sk else list(kv)), kv


def _inputs(case, seed):
    g = torch.Generator(DEV).manual_seed(1000003 * int(seed) + 29)

    def rn(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device=DEV, generator=g) * std + mean

    if case["op"] == "rope":   # positions of a (frame, y, x) grid, from a place of the seed's in a long video
        n = case["rows"] // case["arms"]
        r = torch.arange(n, device=DEV)
        start = int(torch.randint(0, 4000, (1,), device=DEV, generator=g))
        pos = torch.stack([start + r // 256, (r // 16) % 16, r % 16], 1).int().contiguous()
        return {"x": rn(case["rows"], case["nh"] * case["hd"] + case["pad"]).to(DT[case["dtype"]]), "pos": pos}
    if case["op"] == "norm":   # a residual stream that has grown over the blocks, small gates, weights near one
        rows, H = case["rows"], case["H"]
        i = {"x": rn(rows, H, std=3.0).to(DT[case["x"]]), "f": rn(rows, H, std=0.7).to(DT[case["f"]]),
             "mod": rn(-(-rows // case["mod_rows"]), 3 * H, std=0.2)}
        for n in ("post_w", "post_b", "pre_w", "pre_b"):
            kind = case[n.split("_")[0]]
            if case["weights"] and (kind == "ln" or kind == "rms" and n.endswith("w")):
                i[n] = rn(H, std=0.1, mean=1.0 if n.endswith("w") else 0.0)
        return i
    B, Sq, Sk, nh, nkv, hd, dt = (case[k] for k in ("B", "Sq", "Sk", "nh", "nkv", "hd", "dtype"))
    # rows after a per-head RMS norm with weights of about 1.3: scores of a few units; rows past a
    # length hold what an earlier use of the buffer left
    q = rn(B, Sq, 2 * nh, hd)
    q = 1.3 * q / q.square().mean(-1, keepdim=True).sqrt()
    k = rn(B, Sk, 2 * nkv, hd)
    k = 1.3 * k / k.square().mean(-1, keepdim=True).sqrt()
    ql, kl = _lengths(case)
    return {"q": q.reshape(B, Sq, 2 * nh * hd).to(DT[dt]), "k": k.reshape(B, Sk, 2 * nkv * hd).to(DT[dt]),
            "v": rn(B, Sk, 2 * nkv * hd).to(DT[dt]), "lam": rn(1, 4, hd, std=0.1),
            "w": rn(2 * hd, std=0.1, mean=1.0),
            "ql": torch.tensor(ql, device=DEV, dtype=torch.int32), "kl": torch.tensor(kl, device=DEV, dtype=torch.int32)}


LAMBDA_INIT, SCALES = 0.5, (0.9, 1.1)   # x_scale, f_scale of the block ends
BASES = (10000.0, 100.0, 100.0)
EPS = 1e-5


class Dev:
    """A torch tensor as the package's calls take a device array: pointer, size, shape."""

    def __init__(self, t):
        self.t = t
        self.p = ctypes.c_void_p(t.data_ptr())
        self.nbytes = t.numel() * t.element_size()
        self.shape = tuple(t.shape)


_kept = {}


def _package():
    import importlib
    if "tsn" not in _kept:
        _kept["tsn"] = importlib.import_module("thinksound-native_amd")
        _kept["rt"] = _kept["tsn"].Runtime(0)
    return _kept["tsn"], _kept["rt"]


class State:
    """What a program holds before the call: inputs, output buffers and the call's description."""

    def __init__(self, case, seed):
        self.case, self.i = case, _inputs(case, seed)
        i = self.i
        if case["op"] == "rope":
            self.out = {"y": torch.zeros(case["rows"], case["nh"] * case["hd"], device=DEV, dtype=i["x"].dtype)}
        elif case["op"] == "norm":
            self.out = {"x": torch.zeros_like(i["x"]), "y": torch.zeros(i["x"].shape, device=DEV, dtype=DT[case["y"]])}
        else:
            self.out = {"o": torch.zeros(case["B"], case["Sq"], 2 * case["nh"] * case["hd"], device=DEV, dtype=i["q"].dtype)}
        self.plan = _plan(case) if own else None
        self.d = {n: Dev(t) for n, t in i.items()}
        self.o = {n: Dev(t) for n, t in self.out.items()}


def _plan(case):
    tsn, _ = _package()
    code = {"f32": tsn.F32, "f16": tsn.F16, "bf16": tsn.BF16}
    if case["op"] == "rope":
        return tsn.rope_axes_spec(code[case["dtype"]], case["rows"], case["nh"], case["hd"],
                                  (case["d0"], case["d1"], case["d2"]), BASES, ldx=case["nh"] * case["hd"] + case["pad"],
                                  pos_rows=case["rows"] // case["arms"], half_split=case["half"])
    if case["op"] == "norm":
        kinds = {"none": tsn.NORM_NONE, "rms": tsn.NORM_RMS, "ln": tsn.NORM_LN}
        return tsn.gate_norm_spec(case["rows"], case["H"], code[case["x"]], code[case["f"]], code[case["y"]],
                                  post=kinds[case["post"]], pre=kinds[case["pre"]], x_scale=SCALES[0], f_scale=SCALES[1],
                                  chunks=3, mod_rows=case["mod_rows"], gate=2, shift=0, scale=1, post_eps=EPS, pre_eps=EPS)
    return tsn.diff_attn_spec(code[case["dtype"]], case["B"], case["Sq"], case["Sk"], case["nh"], case["nkv"], case["hd"],
                              causal=case["causal"], scale=case["hd"] ** -0.5, lambda_init=LAMBDA_INIT, eps=EPS)


def prepare(case, seed):
    torch.cuda.synchronize()   # a call on an earlier state may still be using memory that torch hands out again
    st = State(case, seed)
    torch.cuda.synchronize()   # inputs and cleared outputs are there before a call on another stream
    return st


def run(st):
    if own:
        rt, i, o, op = _kept["rt"], st.d, st.o, st.case["op"]
        if op == "rope":
            rt.rope_axes(st.plan, i["x"], i["pos"], o["y"])
        elif op == "norm":
            rt.gate_add_norm(st.plan, i["x"], i["f"], i["mod"], o["x"], o["y"], i.get("post_w"), i.get("post_b"),
                             i.get("pre_w"), i.get("pre_b"))
        else:
            rt.diff_attention(st.plan, i["q"], i["k"], i["v"], i["lam"], i["w"], i["ql"], i["kl"], o["o"])
        return st.out
    return {"rope": _plain_rope, "norm": _plain_norm, "attn": _plain_attn}[st.case["op"]](st)


# ---------------------------------------------------------------- the plain forms

def _angles(c, pos):
    """[rows][hd/2] angles in 64 bits; pairs behind the axes' own do not turn"""
    dims = (c["d0"], c["d1"], c["d2"])
    axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(dims, device=DEV) // 2)
    start = torch.tensor([0, dims[0], dims[0] + dims[1]], device=DEV) // 2
    dim, base = torch.tensor(dims, device=DEV).double(), torch.tensor(BASES, device=DEV).double()
    i = torch.arange(sum(dims) // 2, device=DEV) - start[axis]
    return pos.double()[:, axis] * base[axis] ** (-2.0 * i / dim[axis]), axis, i


def _pair_index(c, axis, i):
    """positions in a head of the two elements of each pair"""
    dims = torch.tensor((c["d0"], c["d1"], c["d2"]), device=DEV)
    start = torch.tensor((0, c["d0"], c["d0"] + c["d1"]), device=DEV)[axis]
    if c["half"]:
        return start + i, start + i + dims[axis] // 2
    return start + 2 * i, start + 2 * i + 1


def _plain_rope(st):
    c, x = st.case, st.i["x"]
    ang, axis, i = _angles(c, st.i["pos"])
    e0, e1 = _pair_index(c, axis, i)
    n = c["rows"] // c["arms"]
    v = x[:, :c["nh"] * c["hd"]].float().reshape(c["arms"], n, c["nh"], c["hd"])
    cs, sn = ang.cos().float()[None, :, None], ang.sin().float()[None, :, None]
    y = v.clone()
    x0, x1 = v[..., e0], v[..., e1]
    y[..., e0], y[..., e1] = x0 * cs - x1 * sn, x0 * sn + x1 * cs
    return {"y": y.reshape(c["rows"], -1).to(x.dtype)}


def _plain_norm_rows(kind, x, w, b):
    if kind == "none":
        return x
    if kind == "ln":
        x = x - x.mean(-1, keepdim=True)
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    y = y if w is None else y * w
    return y if b is None else y + b


def _plain_norm(st):
    c, i = st.case, st.i
    mod = i["mod"].repeat_interleave(c["mod_rows"], 0)[:c["rows"]]
    shift, scale, gate = mod.split(c["H"], 1)
    z = _plain_norm_rows(c["post"], i["f"].float(), i.get("post_w"), i.get("post_b"))
    x = SCALES[0] * i["x"].float() + SCALES[1] * gate * z
    y = _plain_norm_rows(c["pre"], x, i.get("pre_w"), i.get("pre_b")) * (1.0 + scale) + shift
    return {"x": x.to(i["x"].dtype), "y": y.to(DT[c["y"]])}


def _plain_attn(st):
    c, i = st.case, st.i
    B, Sq, Sk, nkv, G, hd = c["B"], c["Sq"], c["Sk"], c["nkv"], c["nh"] // c["nkv"], c["hd"]
    q = i["q"].float().reshape(B, Sq, nkv, G, 2, hd).permute(0, 2, 4, 3, 1, 5).reshape(B * nkv * 2, G * Sq, hd)
    k = i["k"].float().reshape(B, Sk, nkv, 2, hd).permute(0, 2, 3, 4, 1).reshape(B * nkv * 2, hd, Sk)
    v = i["v"].float().reshape(B, Sk, nkv, 2 * hd).permute(0, 2, 1, 3).reshape(B * nkv, Sk, 2 * hd)
    s = torch.bmm(q.contiguous(), k.contiguous()).mul_(hd ** -0.5).view(B, nkv, 2, G, Sq, Sk)
    row, key = torch.arange(Sq, device=DEV)[None, :, None], torch.arange(Sk, device=DEV)[None, None]
    ql, kl = i["ql"][:, None, None], i["kl"][:, None, None]
    last = torch.minimum(kl, row + kl - ql + 1) if c["causal"] else kl
    s.masked_fill_((key >= last)[:, None, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill(total == 0.0, 1.0))
    lam = i["lam"][0]
    lam = (lam[0] * lam[1]).sum().exp() - (lam[2] * lam[3]).sum().exp() + LAMBDA_INIT
    d = p[:, :, 0] - lam * p[:, :, 1]
    o = torch.bmm(d.reshape(B * nkv, G * Sq, Sk), v.contiguous()).view(B, nkv, G, Sq, 2 * hd)
    o = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * i["w"] * (1.0 - LAMBDA_INIT)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Sq, -1).to(i["q"].dtype)
    live = torch.arange(Sq, device=DEV)[None, :, None] < ql
    return {"o": torch.where(live, o, st.out["o"])}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    i = _inputs(case, seed)
    return {"rope": _exact_rope, "norm": _exact_norm, "attn": _exact_attn}[case["op"]](case, i)


def _exact_rope(c, i):
    """Each pair as a complex number times e^(i angle)."""
    n, hd = c["rows"] // c["arms"], c["hd"]
    x = i["x"][:, :c["nh"] * hd].double().reshape(c["arms"], n, c["nh"], hd)
    y, at = x.clone(), 0
    for a, dim in enumerate((c["d0"], c["d1"], c["d2"])):
        for p in range(dim // 2):
            t = i["pos"][:, a].double() * math.pow(BASES[a], -2.0 * p / dim)
            u, w = (at + p, at + p + dim // 2) if c["half"] else (at + 2 * p, at + 2 * p + 1)
            z = torch.complex(x[..., u], x[..., w]) * torch.polar(torch.ones_like(t), t)[None, :, None]
            y[..., u], y[..., w] = z.real, z.imag
        at += dim
    return {"y": y.reshape(c["rows"], -1)}


def _exact_norm(c, i):
    H = c["H"]
    at = torch.arange(c["rows"], device=DEV) // c["mod_rows"]

    def norm(kind, x, w, b):
        if kind == "ln":
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            x = (x - mean) * (var + EPS).rsqrt()
        elif kind == "rms":
            x = x * ((x * x).sum(-1, keepdim=True) / H + EPS).rsqrt()
        x = x if w is None else x * w.double()
        return x if b is None else x + b.double()

    m = i["mod"].double()
    z = norm(c["post"], i["f"].double(), i.get("post_w"), i.get("post_b"))
    x = z.mul_(m[:, 2 * H:][at]).mul_(SCALES[1]).add_(i["x"].double(), alpha=SCALES[0])
    y = norm(c["pre"], x, i.get("pre_w"), i.get("pre_b"))
    return {"x": x, "y": y + y * m[:, H:2 * H][at] + m[:, :H][at]}


def _exact_attn(c, i):
    """One head of one sample after the other, over the keys that a row sees."""
    B, Sq, nh, hd = c["B"], c["Sq"], c["nh"], c["hd"]
    G = nh // c["nkv"]
    ql, kl = _lengths(c)
    a = i["lam"][0].double()
    lam = math.exp(float(a[0] @ a[1])) - math.exp(float(a[2] @ a[3])) + LAMBDA_INIT
    out = torch.zeros(B, Sq, 2 * nh * hd, device=DEV, dtype=torch.float64)
    for b in range(B):
        n, m = ql[b], kl[b]
        if c["causal"]:
            hidden = torch.arange(m, device=DEV)[None] > torch.arange(n, device=DEV)[:, None] + (m - n)
        for h in range(nh):
            g = h // G
            maps = []
            for j in (0, 1):
                q = i["q"][b, :n, (2 * h + j) * hd:(2 * h + j + 1) * hd].double()
                k = i["k"][b, :m, (2 * g + j) * hd:(2 * g + j + 1) * hd].double()
                s = (q @ k.t().contiguous()) / math.sqrt(hd)
                if c["causal"]:
                    s.masked_fill_(hidden, -math.inf)
                maps.append(torch.nan_to_num(torch.softmax(s, -1), nan=0.0))
            o = maps[0].sub_(maps[1], alpha=lam) @ i["v"][b, :m, 2 * g * hd:2 * (g + 1) * hd].double()
            o = o * ((o * o).mean(-1, keepdim=True) + EPS).rsqrt()
            out[b, :n, 2 * h * hd:2 * (h + 1) * hd] = o * i["w"].double() * (1.0 - LAMBDA_INIT)
    return {"o": out}


# ---------------------------------------------------------------- work

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "rope":
        n = case["rows"] * case["nh"]
        turned = case["d0"] + case["d1"] + case["d2"]
        return {"bytes": 2 * n * case["hd"] * size[case["dtype"]] + 12 * (case["rows"] // case["arms"]), "flops": 3.0 * n * turned}
    if case["op"] == "norm":
        rows, H = case["rows"], case["H"]
        rw = 2 * size[case["x"]] + size[case["f"]] + size[case["y"]]
        return {"bytes": rows * H * rw + 12 * H * (-(-rows // case["mod_rows"])) + (8 * H if case["weights"] else 0),
                "flops": 16.0 * rows * H}
    ql, kl = _lengths(case)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    seen = 0
    for n, m in zip(ql, kl):
        if case["causal"]:   # row r sees m - n + r + 1 keys
            first = max(0, n - m)
            seen += (n - first) * (m - n + first + 1 + m) // 2
        else:
            seen += n * m
    # each sample's rows once; both maps' products and the difference's product with V
    return {"bytes": 2 * (4 * nh * hd * sum(ql) + 4 * nkv * hd * sum(kl)), "flops": 8.0 * hd * nh * seen}
