"""The serving path over a 4-bit KV cache, and the norm in front of its projections: attention of
new queries over the cache, the cache's append and read-back, and the RMS norm that adds the
residual and writes MX codes.

The cache holds E2M1 values (4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) in blocks of 32 along the
head dimension, one E8M0 scale to a block, K and V alike:
  codes  [B][Hkv][L][D/2]             element 2i in the low four bits of byte i, 2i + 1 in the high
  scales [B][Hkv][L/32][4][D/32][8]   token t of 32 at [t % 4][block][2 * (t / 4 % 4) + t / 16]
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mxfa():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "radiance-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mxfa
    return mxfa


# ---- cases ----------------------------------------------------------------------------------

def _attention(name, B, Hkv, group, D, Sq, L, **kw):
    c = dict(name=name, kind="attention", B=B, Hkv=Hkv, group=group, D=D, Sq=Sq, L=L, capacity=(L + 31) // 32 * 32,
             ragged=False, causal=True, window=0, softcap=0.0, f32=False)
    c.update(kw)
    return c


def listed():
    return [
        # A few short conversations on a small model: launches and latency.
        _attention("decode_d64_l300", 2, 2, 4, 64, 1, 300, ragged=True, capacity=512),
        # A full serving batch of the Llama-style shape (bench.py's decode): bound by HBM.
        _attention("decode_b64_l8192", 64, 8, 4, 128, 1, 8192),
        # One user with a very long document: a single sequence has to fill the card.
        _attention("decode_b1_l131072", 1, 8, 4, 128, 1, 131072),
        # Gemma-style decode, sequences of different lengths, fp32 O for the library's quantizers.
        _attention("decode_d256_window", 24, 8, 2, 256, 1, 7000, ragged=True, window=4096, softcap=50.0, f32=True,
                   capacity=8192),
        # Five drafted tokens of each sequence to verify.
        _attention("draft_q5_b16_l6001", 16, 8, 4, 128, 5, 6001, ragged=True, capacity=8192),
        # A chunk of a long prompt against the cache so far, its own tokens included.
        _attention("chunk_q1000_l16384", 1, 8, 4, 128, 1000, 16384),
        # One decode step's new tokens into the cache, each sequence at its own length.
        dict(name="append_step_b64", kind="append", B=64, Hkv=8, D=128, n=1, capacity=8192, ragged=True, f32=False),
        # Prompts of different lengths, padded to one, into the cache.
        dict(name="append_prompt_b4_n4096", kind="append", B=4, Hkv=8, D=128, n=4096, capacity=8192, ragged=True, f32=False),
        # A short stretch of one sequence's cache read back (a prefix handed to another consumer) ...
        dict(name="read_n100", kind="read", B=1, Hkv=8, D=128, n=100, capacity=1024, ragged=True, f32=True),
        # ... and whole caches of a batch.
        dict(name="read_b8_n8192", kind="read", B=8, Hkv=8, D=128, n=8192, capacity=8192, ragged=False, f32=False),
        # The norm before the projections of a decode batch, scales as mxfa.gemm reads them ...
        dict(name="norm_m64_k4096", kind="norm", rows=64, cols=4096, residual=True, f32=False, offset=0.0, gemm=True),
        # ... and of a prompt.
        dict(name="norm_m8192_k4096", kind="norm", rows=8192, cols=4096, residual=True, f32=False, offset=0.0, gemm=True),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(["attention"] * 6 + ["append"] * 2 + ["read"] * 2 + ["norm"] * 2)
    f32 = rng.random() < 0.3
    if kind == "norm":
        rows, cols = int(_log(rng, 1, 16384)), 32 * int(_log(rng, 8, 512))
        while rows * cols * (2 if f32 else 1) > 8192 * 4096:
            rows //= 2
        return dict(kind=kind, rows=rows, cols=cols, residual=rng.random() < 0.7, f32=f32,
                    offset=rng.choice([0.0, 0.0, 1.0]), gemm=rng.random() < 0.6)
    D = rng.choice([64, 128, 128, 256])
    Hkv, group = rng.choice([(8, 4), (8, 2), (4, 8), (16, 1), (2, 7), (1, 8), (2, 16), (1, 24)])
    B = int(_log(rng, 1, 64))
    ragged = rng.random() < 0.6
    if kind in ("append", "read"):
        n = int(_log(rng, 1, 8192))
        while B * Hkv * n * D * (2 if f32 else 1) > 4 * 8 * 4096 * 128:
            B, n = max(1, B // 2), max(1, n * 3 // 4)
        capacity = 32 * ((n + int(_log(rng, 1, 4096))) // 32 + 1)
        return dict(kind=kind, B=B, Hkv=Hkv, D=D, n=n, capacity=capacity, ragged=ragged, f32=f32)
    Sq = rng.choice([1, 1, 1, rng.randint(2, 8), int(_log(rng, 9, 2000))])
    L = max(Sq, int(_log(rng, 1, 131072)))
    while B * Hkv * L * D > 64 * 8 * 8192 * 128 or B * Hkv * group * Sq * L * D > 32 * 1000 * 16384 * 128:
        if B > 1:
            B //= 2
        elif Sq > 8:
            Sq //= 2
        else:
            L = L * 3 // 4
    return dict(kind=kind, B=B, Hkv=Hkv, group=group, D=D, Sq=Sq, L=L, capacity=32 * ((L + 31) // 32 + rng.choice([0, 5, 64])),
                ragged=ragged, causal=Sq == 1 or rng.random() < 0.85, window=rng.choice([0, 0, 4096]),
                softcap=rng.choice([0.0, 0.0, 50.0]), f32=f32)


def _lengths(c):
    """Keys of each sequence: one is full, an empty slot of the batch has none."""
    B, L = c["B"], c["L"]
    n = [max(1, L * (b + 1) // B) if c["ragged"] else L for b in range(B)]
    if c["ragged"] and B >= 8:
        n[0] = 0
    return n


def _starts(c):
    """Where each sequence's stretch of an append or a read begins, and how many of its tokens count."""
    B, n, room = c["B"], c["n"], c["capacity"] - c["n"]
    start = [room * (b + 1) // (B + 1) if c["ragged"] else room // 2 for b in range(B)]
    count = [max(1, n - n * b // (2 * B)) if c["ragged"] else n for b in range(B)]
    return start, count


# ---- the inputs ------------------------------------------------------------------------------

def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _quantize(x):
    """fp32 [..., D] -> (codes [..., D/2], scale codes [..., D/32]): the scale is 2 to the exponent of the
    block's largest magnitude, less 2; elements round half to even and stop at 6; a NaN counts as 0."""
    xb = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).reshape(*x.shape[:-1], -1, 32)
    amax = xb.abs().amax(-1, keepdim=True)
    e = torch.where(amax == math.inf, 125, torch.frexp(amax).exponent - 3).clamp(-127, 125)
    e = torch.where(amax == 0, -127, e)
    y = torch.ldexp(xb, -e)
    a = y.abs()
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = (mag + 8 * (y < 0).to(torch.uint8)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e[..., 0] + 127).to(torch.uint8)


def _make_cache(B, Hkv, D, capacity, used, g):
    """A cache of N(0, 1) keys and values, the keys with channels of unlike size; scales past `used` tokens are
    what was there before."""
    def half(channels):
        codes = torch.empty((B, Hkv, capacity, D // 2), dtype=torch.uint8, device=DEV)
        scales = torch.empty((B, Hkv, capacity // 32, 4, D // 32, 4, 2), dtype=torch.uint8, device=DEV)
        for b in range(B):
            x = _normal((Hkv, capacity, D), g) * channels
            codes[b], s = _quantize(x)
            # token 16 t + 4 i + k at [k][block][i][t]
            scales[b] = s.reshape(Hkv, capacity // 32, 2, 4, 4, D // 32).permute(0, 1, 4, 5, 3, 2)
        if used < capacity:
            scales[:, :, (used + 31) // 32:] = 127
        return codes, scales.reshape(B, Hkv, capacity // 32, 4, D // 32, 8)
    return (*half(torch.exp(0.5 * _normal((D,), g))), *half(1.0))


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dtype = torch.float32 if c["f32"] else torch.bfloat16
    if c["kind"] == "norm":
        rows, cols = c["rows"], c["cols"]
        return dict(kind="norm", c=c, x=_normal((rows, cols), g, dtype),
                    residual=(4.0 * _normal((rows, cols), g)).to(dtype) if c["residual"] else None,
                    weight=(1.0 - c["offset"] + 0.2 * _normal((cols,), g)).to(dtype))
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    s = dict(kind=c["kind"], c=c)
    if c["kind"] == "attention":
        lens = _lengths(c)
        order = torch.randperm(B, generator=g, device=DEV)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)[order]
        Hq, Sq = Hkv * c["group"], c["Sq"]
        # q as it leaves the fused projection: a slice of each token's q, k and v
        qkv = _normal((B, Sq, (Hq + 2 * Hkv) * D), g, torch.bfloat16)
        s["q"] = qkv[..., :Hq * D].view(B, Sq, Hq, D).transpose(1, 2)
        s["kv"] = _make_cache(B, Hkv, D, c["capacity"], c["L"], g)
        s["out"] = torch.empty((B, Sq, Hq, D), dtype=dtype, device=DEV)
    else:
        start, count = _starts(c)
        order = torch.randperm(B, generator=g, device=DEV)
        s["pos"] = torch.tensor(start, dtype=torch.int32, device=DEV)[order]
        s["kv"] = _make_cache(B, Hkv, D, c["capacity"], c["capacity"], g)
        if c["kind"] == "append":
            s["counts"] = torch.tensor(count, dtype=torch.int32, device=DEV)[order] if c["ragged"] else None
            kv = _normal((B, c["n"], 2, Hkv, D), g, dtype)
            s["new"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    if own:
        # the handle, the parameters and the workspace that a serving loop keeps between its calls
        mxfa = _mxfa()
        s["cache"] = mxfa.Kv4Cache.of(*s["kv"])
        if c["kind"] == "attention":
            s["p"] = mxfa.make_kv4_params(B, Hkv * c["group"], Hkv, c["Sq"], c["L"], D, max_len=c["capacity"],
                                          causal=c["causal"], window=c["window"], softcap=c["softcap"],
                                          o_fmt=mxfa.C_F32 if c["f32"] else mxfa.C_BF16)
            s["ws"] = torch.empty(mxfa.kv4_attention_plan(s["p"])[1], dtype=torch.uint8, device=DEV)
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    mxfa, c = _mxfa(), s["c"]
    if s["kind"] == "attention":
        mxfa.kv4_attention(s["p"], s["q"], s["cache"], kv_len=s["lens"], out=s["out"].transpose(1, 2), workspace=s["ws"])
        return s["out"]
    if s["kind"] == "norm":
        codes, scales, h = mxfa.rmsnorm_quantize(s["x"], s["weight"], eps=1e-6, residual=s["residual"],
                                                 weight_offset=c["offset"], gemm_scales=c["gemm"])
        return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), h if c["residual"] else None
    if s["kind"] == "append":
        s["cache"].append(*s["new"], pos=s["pos"], counts=s["counts"])
    return s["cache"].read(c["n"], pos=s["pos"], dtype=torch.float32 if c["f32"] else torch.bfloat16)


def _values(codes, scales):
    """fp32 values [..., n, D] of codes [..., n, D/2] and the scale codes [..., n, D/32] of the same tokens."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=DEV)
    x = torch.stack([levels[(codes & 15).long()], levels[(codes >> 4).long()]], -1)
    return torch.ldexp(x.reshape(*scales.shape, 32), scales.to(torch.int32)[..., None] - 127).flatten(-2)


def _token_order(scales):
    """[B][Hkv][L/32][4][D/32][8] -> [B][Hkv][L][D/32]"""
    B, H, blocks, _, nb, _ = scales.shape
    return scales.reshape(B, H, blocks, 4, nb, 4, 2).permute(0, 1, 2, 6, 5, 3, 4).reshape(B, H, 32 * blocks, nb)


def _run_plain(s):
    c = s["c"]
    if s["kind"] == "attention":
        return _plain_attention(s)
    if s["kind"] == "norm":
        return _plain_norm(s)
    dtype = torch.float32 if c["f32"] else torch.bfloat16
    k, ks, v, vs = s["kv"]
    B, n = c["B"], c["n"]
    at = s["pos"].long()[:, None] + torch.arange(n, device=DEV)                        # [B, n]
    rows = torch.arange(B, device=DEV)[:, None]
    where = (rows, slice(None), at // 32, at % 4, slice(None), 2 * (at // 4 % 4) + at // 16 % 2)
    got = []
    for i, (codes, scales) in enumerate(((k, ks), (v, vs))):
        if s["kind"] == "append":
            new, sc = _quantize(s["new"][i].float().transpose(1, 2))                   # [B, n, Hkv, ...]
            if s["counts"] is not None:
                live = (torch.arange(n, device=DEV) < s["counts"][:, None])[..., None, None]
                new = torch.where(live, new, codes[rows, :, at])
                sc = torch.where(live, sc, scales[where])
            codes[rows, :, at] = new
            scales[where] = sc
        got.append(_values(codes[rows, :, at], scales[where]).transpose(1, 2).to(dtype).contiguous())
    return tuple(got)


def _plain_attention(s):
    c = s["c"]
    B, Hkv, G, Sq, D = c["B"], c["Hkv"], c["group"], c["Sq"], c["D"]
    L = (c["L"] + 31) // 32 * 32
    k, ks, v, vs = s["kv"]
    K = _values(k[:, :, :L], _token_order(ks[:, :, :L // 32]))
    V = _values(v[:, :, :L], _token_order(vs[:, :, :L // 32]))
    q = s["q"].float().reshape(B, Hkv, G * Sq, D)
    x = torch.matmul(q, K.transpose(-1, -2).contiguous()) / math.sqrt(D)
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    lens, key = s["lens"].long()[:, None, None], torch.arange(L, device=DEV)
    at = lens - Sq + torch.arange(Sq, device=DEV)[:, None]                               # each query's position
    seen = (key < lens).expand(B, Sq, L)
    if c["causal"]:
        seen = seen & (key <= at)
    if c["window"]:
        seen = seen & (key > at - c["window"])
    x = x.reshape(B, Hkv, G, Sq, L).masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, G * Sq, L), V).reshape(B, Hkv, G, Sq, D) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.reshape(B, Hkv * G, Sq, D).transpose(1, 2))
    return s["out"]


def _plain_norm(s):
    c = s["c"]
    x = s["x"].float()
    h = None
    if c["residual"]:
        h = (x + s["residual"].float()).to(s["x"].dtype)
        x = h.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (s["weight"].float() + c["offset"])
    yb = y.reshape(c["rows"], -1, 32)
    amax = yb.abs().amax(-1, keepdim=True)
    e = torch.where(amax == 0, -127, (torch.frexp(amax).exponent - 9).clamp(-127, 127))
    z = torch.ldexp(yb, -e)
    z = torch.where(z.abs() < 2.0 ** -6, 0.0, z.clamp(-448.0, 448.0))
    scales = (e[..., 0] + 127).to(torch.uint8)
    scales = scales.t().contiguous() if c["gemm"] else scales
    return z.to(torch.float8_e4m3fn).reshape(c["rows"], c["cols"]), scales.view(torch.float8_e8m0fnu), h


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    c = case
    t = 4 if c["f32"] else 2
    if c["kind"] == "norm":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (t * (3 if c["residual"] else 1) + 33 / 32) + c["cols"] * t, "flops": 6.0 * n}
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if c["kind"] != "attention":
        new = sum(_starts(c)[1]) if c["kind"] == "append" else 0
        per = 2 * Hkv * D                                                       # elements of a token
        return {"bytes": per * (new * (t + 17 / 32) + B * c["n"] * (t + 17 / 32)), "flops": 2.0 * per * (new + B * c["n"])}
    Sq, keys, pairs = c["Sq"], 0, 0
    for n in _lengths(c):
        first, last = n, -1
        for i in range(Sq):
            at = n - Sq + i
            hi = min(n - 1, at) if c["causal"] else n - 1
            lo = max(0, at - c["window"] + 1) if c["window"] else 0
            if hi >= lo:
                pairs += hi - lo + 1
                first, last = min(first, lo), max(last, hi)
        keys += max(0, last - first + 1)
    Hq = Hkv * c["group"]
    return {"bytes": keys * Hkv * D * 2 * 17 / 32 + B * Hq * Sq * D * (2 + t), "flops": 4.0 * D * Hq * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------------

def _exact_values(codes, scales):
    """As _values, from the fields of each code: sign, two exponent bits, one mantissa bit."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int32)
    exponent, mantissa = (n >> 1) & 3, (n & 1).to(torch.float64)
    size = torch.where(exponent == 0, 0.5 * mantissa, (1.0 + 0.5 * mantissa) * 2.0 ** (exponent - 1).to(torch.float64))
    two = torch.repeat_interleave(2.0 ** (scales.to(torch.float64) - 127), 32, -1)
    return torch.where(n > 7, -size, size) * two


def _exact_round(y, bits, lowest):
    """y to `bits` bits after the leading one, half to even, steps no finer than those at 2^lowest."""
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** lowest))) - bits)
    return torch.round(y / step) * step


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "norm":
        x, h = s["x"].double(), None
        if c["residual"]:
            h = (x + s["residual"].double()).to(s["x"].dtype).double()           # what is stored is what is normed
            x = h
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (s["weight"].double() + c["offset"])
        y = y.reshape(c["rows"], -1, 32)
        two = 2.0 ** (torch.floor(torch.log2(y.abs().amax(-1))) - 8).clamp(min=-127)
        z = y / two[..., None]
        z = torch.where(z.abs() < 2.0 ** -6, 0.0, _exact_round(z, 3, -6).clamp(-448, 448))
        return z.reshape(c["rows"], c["cols"]), two.t() if c["gemm"] else two, h
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    k, ks, v, vs = s["kv"]
    out = []
    if c["kind"] != "attention":
        n, pos = c["n"], s["pos"].tolist()
        counts = [n if c["kind"] == "append" else 0] * B
        if c["kind"] == "append" and s["counts"] is not None:
            counts = s["counts"].tolist()
        for i, (codes, scales) in enumerate(((k, ks), (v, vs))):
            order, got = _token_order(scales), []
            for b in range(B):
                x = _exact_values(codes[b, :, pos[b]:pos[b] + n], order[b, :, pos[b]:pos[b] + n])
                if counts[b]:
                    new = s["new"][i][b, :, :counts[b]].double().reshape(Hkv, counts[b], -1, 32)
                    two = 2.0 ** (torch.floor(torch.log2(new.abs().amax(-1, keepdim=True))) - 2).clamp(-127, 125)
                    x[:, :counts[b]] = (_exact_round(new / two, 1, 0).clamp(-6, 6) * two).flatten(-2)
                got.append(x)
            out.append(torch.stack(got))
        return tuple(out)
    G, Sq = c["group"], c["Sq"]
    o = torch.zeros((B, Sq, Hkv * G, D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        up = (n + 31) // 32 * 32
        for head in range(Hkv if n else 0):
            K = _exact_values(k[b, head, :up], _token_order(ks[b:b + 1, head:head + 1, :up // 32])[0, 0])[:n]
            V = _exact_values(v[b, head, :up], _token_order(vs[b:b + 1, head:head + 1, :up // 32])[0, 0])[:n]
            q = s["q"][b, head * G:(head + 1) * G].double()                       # [G, Sq, D]
            x = torch.matmul(q.reshape(G * Sq, D), K.t().contiguous()).reshape(G, Sq, n) * D ** -0.5
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            at = torch.arange(n - Sq, n, device=DEV)[:, None]
            key = torch.arange(n, device=DEV)[None]
            hide = torch.zeros((Sq, n), dtype=torch.bool, device=DEV)
            if c["causal"]:
                hide |= key > at
            if c["window"]:
                hide |= key + c["window"] <= at
            w = torch.nan_to_num(torch.softmax(x.masked_fill(hide, -math.inf), -1))
            o[b, :, head * G:(head + 1) * G] = torch.matmul(w.reshape(G * Sq, n), V).reshape(G, Sq, D).transpose(0, 1)
    return o
