"""The 4-bit KV cache and the quantizing norm in 64 bits, from their definitions (numpy / torch on the host)."""
import math

import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
STEPS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])           # halfway points; ties go to the even code


def quantize(x):
    """fp32 [..., D] -> (codes 0..15 [..., D], scale codes [..., D/32])."""
    x = np.asarray(x, np.float32).astype(np.float64)
    x = np.where(np.isnan(x), 0.0, x)
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(np.isinf(amax), 125, np.where(amax == 0, -127, np.frexp(amax)[1] - 3))
    e = np.clip(e, -127, 125).astype(int)
    with np.errstate(over="ignore"):
        y = np.abs(np.ldexp(b, -e[..., None]))
    code = np.zeros(y.shape, np.uint8)
    for i, s in enumerate(STEPS):
        code += (y > s) | ((y == s) & (i % 2 == 1))
    code += 8 * np.signbit(b).astype(np.uint8)
    return code.reshape(x.shape), (e + 127).astype(np.uint8)


def values(codes, scales):
    """float64 values of codes 0..15 [..., D] and scale codes [..., D/32]."""
    c = np.asarray(codes)
    v = np.where(c >= 8, -LEVELS[c & 7], LEVELS[c & 7]).reshape(*c.shape[:-1], -1, 32)
    return np.ldexp(v, np.asarray(scales).astype(int)[..., None] - 127).reshape(c.shape)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def scale_place(t, block, nb):
    """Index of token t, block `block` in a head's flat scales."""
    return t // 32 * (32 * nb) + ((t % 4) * nb + block) * 8 + 2 * (t // 4 % 4) + t // 16 % 2


def scales_by_token(sc):
    """[B, H, L/32, 4, nb, 8] -> [B, H, L, nb]"""
    B, H, blocks, _, nb, _ = sc.shape
    flat = sc.reshape(B, H, -1)
    t = np.arange(32 * blocks)
    return flat[:, :, scale_place(t[:, None], np.arange(nb)[None], nb)]


def scales_in_cache(by_token):
    """The inverse: [B, H, L, nb] -> [B, H, L/32, 4, nb, 8]"""
    B, H, L, nb = by_token.shape
    out = np.empty((B, H, L * nb), np.uint8)
    out[:, :, scale_place(np.arange(L)[:, None], np.arange(nb)[None], nb)] = by_token
    return out.reshape(B, H, L // 32, 4, nb, 8)


def cache_values(codes, scales):
    """float64 [B, H, L, D] of a cache's tensors."""
    return values(unpack(np.asarray(codes)), scales_by_token(np.asarray(scales)))


def attention(q, K, V, lens, causal=True, q_pos0=None, window=0, scale=None, softcap=0.0):
    """(O, A, X, Y): O = softmax(S) V in 64 bits; A = sum p |v| / sum p (what a relative error of P can move O by);
    X = largest |score| in log2 units and Y = largest sum |q||k| * scale, log2 units, over what is visible.
    q [B, Hq, Sq, D], K and V [B, Hkv, L, D]; lens[b] keys; q_pos0 None: queries end at lens[b]."""
    B, Hq, Sq, D = q.shape
    G = Hq // K.shape[1]
    scale = scale or 1.0 / math.sqrt(D)
    O = torch.zeros(q.shape, dtype=torch.float64)
    A = torch.zeros_like(O)
    X = Y = 0.0
    q, K, V = (torch.as_tensor(t).double() for t in (q, K, V))
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        k, v = K[b, :, :n].repeat_interleave(G, 0), V[b, :, :n].repeat_interleave(G, 0)
        kt = k.transpose(1, 2).contiguous()
        s = torch.matmul(q[b], kt) * scale
        mag = torch.matmul(q[b].abs(), kt.abs()) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        at = (n - Sq if q_pos0 is None else q_pos0) + torch.arange(Sq)[:, None]
        key = torch.arange(n)[None]
        seen = torch.ones((Sq, n), dtype=torch.bool)
        if causal:
            seen &= key <= at
        if window:
            seen &= key + window > at
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(-1, keepdim=True)
        total = torch.where(total == 0, 1.0, total)
        O[b] = torch.matmul(p, v) / total
        A[b] = torch.matmul(p, v.abs()) / total
        if seen.any():
            X = max(X, float(s.masked_fill(~seen, 0).abs().max()) * math.log2(math.e))
            Y = max(Y, float((mag * seen).max()) * math.log2(math.e))
    return O, A, X, Y


def attention_bound(O, A, X, Y, D, keys, f32, rows, softcap=0.0):
    """How far a kernel's O may be, element by element.  With u = 2^-24: a score is a sum of D exact products added
    in fp32, off by at most D u Y; scaling, the reference exponent and the difference round three times at
    u max(X, 1) each, twice that range; tanh by exponentials is off by some 8 u of its cap.  P is then off by ln 2
    times that, by two steps of exp2 and by what its bf16 terms leave of it (2^-8 for each: three terms for fp32 O, for
    bf16 O two up to 32 rows of a KV head and one beyond), O
    by twice P's relative error of A (numerator and sum) and by `keys` roundings in each sum; then O is rounded."""
    u = 2.0 ** -24
    x = u * (D * Y + 6 * max(X, 1.0) + 8 * softcap * math.log2(math.e))
    p = math.log(2) * x + 4 * u + 2.0 ** -(8 * (3 if f32 else 2 if rows <= 32 else 1))
    return 2 * (p + (keys + 16) * u) * A + (u if f32 else 2.0 ** -8) * O.abs() + keys * 2.0 ** -126


def norm(x, weight, eps, residual=None, offset=0.0):
    """(y, h) in 64 bits; x, weight, residual: torch tensors of one type on the host."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    d = h.double()
    y = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    return y.numpy(), h


def r1_scale(amax):
    """Exponent of rule R1's E4M3 scale, floor(log2(amax)) - 8, at least -127."""
    with np.errstate(divide="ignore"):
        return np.where(amax == 0, -127, np.clip(np.frexp(amax)[1] - 1 - 8, -127, 127)).astype(int)


def r1_round(z):
    """E4M3 value of z by rule R1: 0 below 2^-6, three mantissa bits half to even, 448 at most."""
    a = np.abs(z)
    step = np.ldexp(1.0, np.frexp(np.maximum(a, 2.0 ** -6))[1] - 1 - 3)
    v = np.minimum(np.round(a / step) * step, 448.0)
    return np.where(a < 2.0 ** -6, 0.0, np.copysign(v, z))


def norm_delta(cols):
    """Relative error of an fp32 y: a square sum of at most cols / 256 + 8 sequential terms per thread and 10 more
    additions, halved by the root, and some eight roundings on the way to y, u = 2^-24 each."""
    return (cols / 256 + 8 + 10 + 8) * 2.0 ** -24
