"""The 4-bit KV cache on the GPU: append and read-back bit for bit against the rule in 64 bits, attention against
softmax(S) V in 64 bits within the error that its arithmetic can make (kv4ref.attention_bound)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4ref as R  # noqa: E402
import mxfa  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _hard_values(rng, shape):
    """Rows with what a block can hold: ordinary values, zeros of both signs, ties, subnormals, the largest and
    infinite values, NaN, magnitudes right at and around a power of two."""
    x = rng.standard_normal(shape).astype(np.float32)
    flat = x.reshape(-1, 32)
    n = len(flat)
    with np.errstate(over="ignore"):
        for i, r in enumerate(rng.permutation(n)[:max(12, n // 2)]):
            kind = i % 12
            if kind == 0:
                flat[r] = 0.0
            elif kind == 1:
                flat[r] = -0.0
            elif kind == 2:
                flat[r] = np.concatenate([R.STEPS, -R.STEPS, R.LEVELS, -R.LEVELS, [6.0, -6.0]])[:32] * np.float32(2.0 ** rng.integers(-20, 20))
            elif kind == 3:
                flat[r] *= np.float32(2.0 ** -135)
            elif kind == 4:
                flat[r] = np.float32(3.4e38) * rng.uniform(-1, 1, 32).astype(np.float32)
            elif kind == 5:
                flat[r, rng.integers(32)] = np.nan
            elif kind == 6:
                flat[r, rng.integers(32)] = np.inf if i % 2 else -np.inf
            elif kind == 7:
                flat[r] = np.nan
            elif kind == 8:
                flat[r] = np.clip(flat[r], -1, 1)
                flat[r, 3] = np.float32(8.0)
            elif kind == 9:
                flat[r] = np.clip(flat[r], -1, 1)
                flat[r, 3] = np.nextafter(np.float32(8.0), np.float32(0))
            elif kind == 10:
                flat[r] = np.float32(1e-44)
            else:
                flat[r] *= np.float32(2.0 ** rng.integers(-100, 100))
    return x


def _check_cache(cache, K, V, written, before):
    """Codes and scales of the written tokens are the rule's, all other bytes are what they were."""
    for x, codes, scales, (c0, s0), name in ((K, cache.k, cache.ks, before[0], "K"), (V, cache.v, cache.vs, before[1], "V")):
        want_c, want_s = R.quantize(x)
        got_c, got_s = R.unpack(codes.cpu().numpy()), R.scales_by_token(scales.cpu().numpy())
        c0, s0 = R.unpack(c0), R.scales_by_token(s0)
        full_c = np.where(written[:, None, :, None], want_c, c0)
        full_s = np.where(written[:, None, :, None], want_s, s0)
        assert np.array_equal(got_s, full_s), name
        assert np.array_equal(got_c, full_c), name


def _filled(B, H, D, L, seed):
    """A cache of random bytes (scales of moderate size)."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cache = mxfa.Kv4Cache(B, H, D, L)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=DEV, dtype=torch.uint8))
    for t in (cache.ks, cache.vs):
        t.copy_(torch.randint(120, 132, t.shape, generator=g, device=DEV, dtype=torch.uint8))
    return cache


def _bytes(cache):
    return ((cache.k.cpu().numpy(), cache.ks.cpu().numpy()), (cache.v.cpu().numpy(), cache.vs.cpu().numpy()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,D,L,n,layout", [
    (1, 1, 32, 32, 1, "dense"), (1, 2, 64, 64, 64, "dense"), (3, 2, 128, 96, 7, "fused"), (2, 3, 256, 64, 33, "fused"),
    (2, 1, 96, 128, 50, "tokens"), (5, 8, 128, 32, 1, "fused"), (1, 4, 160, 256, 200, "dense"),
])
def test_append_is_the_rule(B, H, D, L, n, layout, dtype):
    print(f"append B{B} H{H} D{D} L{L} n{n} {layout} {dtype}", flush=True)
    rng = np.random.default_rng(B * 1000 + D + n)
    K, V = (torch.from_numpy(_hard_values(rng, (B, H, n, D))).to(dtype) for _ in range(2))
    cache = _filled(B, H, D, L, 5)
    before = _bytes(cache)
    pos = rng.integers(0, L - n + 1, B).astype(np.int32)
    counts = rng.integers(0, n + 1, B).astype(np.int32)
    counts[0] = n
    if layout == "fused":                       # inside the rows of [B, n, (2 + 2 H) D]
        rows = torch.zeros((B, n, 2 + 2 * H, D), dtype=dtype)
        rows[:, :, 2:2 + H], rows[:, :, 2 + H:] = K.transpose(1, 2), V.transpose(1, 2)
        rows = rows.to(DEV)
        kd, vd = rows[:, :, 2:2 + H].transpose(1, 2), rows[:, :, 2 + H:].transpose(1, 2)
    elif layout == "tokens":                    # [n, B, H, D]
        kd, vd = (t.permute(2, 0, 1, 3).contiguous().to(DEV).permute(1, 2, 0, 3) for t in (K, V))
    else:
        kd, vd = K.to(DEV), V.to(DEV)
    cache.append(kd, vd, pos=_dev(pos), counts=_dev(counts))
    t = np.arange(L)[None]
    written = (t >= pos[:, None]) & (t < (pos + counts)[:, None])
    full = []
    for x in (K, V):
        a = np.zeros((B, H, L, D), np.float32)
        for b in range(B):
            a[b, :, pos[b]:pos[b] + n] = x[b].float().numpy()
        full.append(a)
    _check_cache(cache, *full, written, before)
    # read-back: exact in both types, wherever it starts
    want = [R.cache_values(*p) for p in _bytes(cache)]
    for out in (torch.float32, torch.bfloat16):
        got = cache.read(n, pos=_dev(pos), dtype=out)
        for g, w in zip(got, want):
            for b in range(B):
                assert np.array_equal(g[b].double().cpu().numpy(), w[b, :, pos[b]:pos[b] + n])


def test_append_and_read_skip_what_lies_outside():
    """Device-side positions outside the cache are skipped by append and read as 0; counts beyond n_new or below
    0 write n_new tokens or none."""
    B, H, D, L, n = 5, 2, 64, 64, 20
    rng = np.random.default_rng(3)
    K, V = (rng.standard_normal((B, H, n, D)).astype(np.float32) for _ in range(2))
    cache = _filled(B, H, D, L, 6)
    before = _bytes(cache)
    pos = np.array([-8, 60, 2 ** 31 - 5, -2 ** 31, 10], np.int32)
    counts = np.array([n, n, n, n, 2 ** 31 - 1], np.int32)
    cache.append(_dev(K), _dev(V), pos=_dev(pos), counts=_dev(counts))
    full = [np.zeros((B, H, L, D), np.float32) for _ in range(2)]
    written = np.zeros((B, L), bool)
    for b in range(B):
        for t in range(n):
            at = int(pos[b]) + t
            if 0 <= at < L:
                written[b, at] = True
                full[0][b, :, at], full[1][b, :, at] = K[b, :, t], V[b, :, t]
    _check_cache(cache, *full, written, before)
    got = cache.read(n, pos=_dev(pos), dtype=torch.float32)
    want = [R.cache_values(*p) for p in _bytes(cache)]
    for g, w in zip(got, want):
        g = g.double().cpu().numpy()
        for b in range(B):
            for t in range(n):
                at = int(pos[b]) + t
                assert np.array_equal(g[b, :, t], w[b, :, at] if 0 <= at < L else np.zeros((H, D)))
    cache.append(_dev(K), _dev(V), pos=_dev(np.zeros(B, np.int32)), counts=_dev(np.array([0, -1, -2 ** 31, 0, 0], np.int32)))
    _check_cache(cache, *full, written, before)


def test_append_at_length_advances_it_and_refuses_past_the_end():
    cache = mxfa.Kv4Cache(1, 2, 64, 64)
    x = torch.randn((1, 2, 40, 64), device=DEV)
    cache.append(x, x)
    cache.append(x[:, :, :24], x[:, :, :24])
    assert cache.length == 64
    with pytest.raises(mxfa.MxfaError):
        cache.append(x[:, :, :1], x[:, :, :1])
    K, _ = cache.read(64, dtype=torch.float32)
    want = R.values(*R.quantize(torch.cat([x, x[:, :, :24]], 2).cpu().numpy()))
    assert np.array_equal(K.double().cpu().numpy(), want)


def test_read_into_strided_rows():
    cache = _filled(2, 3, 128, 64, 8)
    rows = torch.full((2, 17, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    cache.read(17, pos=11, out=(rows[:, :, 1:4].transpose(1, 2), rows[:, :, 4:7].transpose(1, 2)))
    K, V = cache.read(17, pos=11)
    assert torch.equal(rows[:, :, 1:4], K.transpose(1, 2)) and torch.equal(rows[:, :, 4:7], V.transpose(1, 2))
    assert bool((rows[:, :, 0] == 7).all()) and bool((rows[:, :, 7] == 7).all())


# ---- attention -----------------------------------------------------------------------------------

def _problem(B, Hq, Hkv, Sq, D, L, lens, seed, amp=1.0):
    """(q bf16, cache of `lens` tokens, garbage behind them)"""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cache = _filled(B, Hkv, D, L, seed)
    K = torch.randn((B, Hkv, L, D), generator=g, device=DEV) * torch.exp(0.5 * torch.randn((D,), generator=g, device=DEV))
    V = torch.randn((B, Hkv, L, D), generator=g, device=DEV) + 0.3
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    # nothing that a scale can hold behind the last token of a sequence may matter
    for t in (cache.ks, cache.vs):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=DEV, dtype=torch.uint8) | 0xf0)
    cache.append(K, V, pos=torch.zeros(B, dtype=torch.int32, device=DEV), counts=lt)
    q = (amp * torch.randn((B, Hq, Sq, D), generator=g, device=DEV)).bfloat16()
    return q, cache, lt


def _want(q, cache, lens, p, uniform):
    K, V = (R.cache_values(*x) for x in _bytes(cache))
    return R.attention(q.cpu(), K, V, lens, causal=bool(p.causal), q_pos0=p.q_pos0 if uniform else None, window=p.window,
                       scale=p.softmax_scale, softcap=p.softcap)


def _check(got, want, p, keys, what=""):
    O, A, X, Y = want
    f32 = p.o_fmt == mxfa.C_F32
    assert got.dtype == (torch.float32 if f32 else torch.bfloat16)
    bound = R.attention_bound(O, A, X, Y, p.head_dim, keys, f32, p.num_q_heads // p.num_kv_heads * p.seq_q, p.softcap)
    err = (got.double().cpu() - O).abs()
    worst = float((err / bound).max())
    rel = float((got.double().cpu() - O).norm() / max(float(O.norm()), 1e-30))
    print(f"   {what} rel-L2 {rel:.2e}, worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0


ATTENTION = [
    # B, Hq, Hkv, Sq, D, L, lens, options
    (1, 1, 1, 1, 64, 32, [1], {}),
    (1, 4, 1, 1, 128, 32, [31], {}),
    (2, 8, 2, 1, 64, 320, [150, 300], {}),
    (3, 8, 2, 1, 128, 448, [0, 64, 430], {}),
    (2, 4, 2, 1, 256, 224, [65, 201], {}),
    (1, 14, 2, 1, 128, 160, [129], {}),                          # 7 heads to a KV head
    (1, 24, 1, 1, 128, 256, [255], {}),                          # more than a tile of heads
    (1, 64, 2, 1, 64, 96, [77], {}),
    (2, 8, 2, 5, 128, 352, [3, 333], {}),                        # drafted tokens; queries before position 0
    (1, 4, 4, 17, 64, 160, [150], {}),
    (2, 6, 2, 40, 128, 224, [40, 222], {}),
    (1, 4, 2, 130, 128, 288, [260], {}),
    (1, 4, 2, 129, 64, 160, [129], {}),                          # a whole prompt
    (1, 2, 1, 70, 256, 160, [160], {}),
    (2, 8, 2, 6, 128, 352, [2, 333], dict(causal=False)),
    (1, 4, 2, 100, 128, 288, [100], dict(causal=False)),
    (2, 8, 2, 1, 128, 544, [70, 540], dict(window=64)),
    (1, 4, 2, 200, 128, 544, [520], dict(window=33)),
    (1, 4, 2, 50, 64, 544, [520], dict(window=1)),
    (1, 2, 2, 150, 256, 416, [400], dict(window=100, softcap=50.0)),
    (2, 8, 2, 1, 128, 544, [70, 540], dict(softcap=20.0)),
    (1, 8, 2, 9, 64, 544, [541], dict(softcap=30.0, causal=False)),
    (1, 8, 2, 300, 128, 704, [700], {}),
    (2, 8, 2, 90, 64, 352, [0, 350], {}),                        # an empty slot
    (1, 4, 2, 60, 128, 96, [20], {}),                            # more queries than keys: rows without one
    (1, 4, 2, 60, 128, 96, [20], dict(causal=False, window=10)),
]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,D,L,lens,kw", ATTENTION)
def test_attention(B, Hq, Hkv, Sq, D, L, lens, kw, f32):
    print(f"attention B{B} Hq{Hq} Hkv{Hkv} Sq{Sq} D{D} L{L} lens {lens} {kw} f32 {f32}", flush=True)
    q, cache, lt = _problem(B, Hq, Hkv, Sq, D, L, lens, seed=Sq * 7 + D)
    p = mxfa.make_kv4_params(B, Hq, Hkv, Sq, max(max(lens), 1), D, L, o_fmt=mxfa.C_F32 if f32 else mxfa.C_BF16, **kw)
    got = mxfa.kv4_attention(p, q, cache, kv_len=lt)
    _check(got, _want(q, cache, lens, p, False), p, max(lens))
    again = mxfa.kv4_attention(p, q, cache, kv_len=lt)
    assert torch.equal(got, again)


@pytest.mark.parametrize("Sq,pos0,causal,window", [(1, 199, True, 0), (1, 50, True, 0), (8, 100, True, 40), (150, 50, True, 0),
                                                   (150, 400, True, 0), (20, 500, True, 64), (150, 0, False, 0)])
def test_attention_of_one_length(Sq, pos0, causal, window):
    """kv_len None: seq_k keys for everybody, queries from q_pos0 on (beyond the keys too, where a window may leave
    them none)."""
    q, cache, _ = _problem(2, 4, 2, Sq, 128, 224, [200, 200], seed=Sq + pos0)
    p = mxfa.make_kv4_params(2, 4, 2, Sq, 200, 128, 224, causal=causal, q_pos0=pos0, window=window)
    got = mxfa.kv4_attention(p, q, cache)
    _check(got, _want(q, cache, [200, 200], p, True), p, 200)


@pytest.mark.parametrize("B,Hq,Hkv,Sq,D,n,kw", [
    (1, 8, 2, 1, 128, 20000, {}), (1, 8, 2, 1, 64, 20001, dict(softcap=50.0)), (2, 4, 2, 1, 256, 9000, dict(window=4096)),
    (1, 8, 2, 3, 128, 20000, {}), (1, 8, 2, 50, 128, 9999, {}), (1, 4, 1, 200, 64, 9000, dict(window=3000)),
    (1, 2, 1, 100, 256, 6000, {}),
])
@pytest.mark.parametrize("f32", [False, True])
def test_attention_split_over_a_long_cache(B, Hq, Hkv, Sq, D, n, kw, f32):
    """Parts of the key range merged through the workspace; a sequence far shorter than seq_k leaves parts empty."""
    print(f"split B{B} Hq{Hq} Sq{Sq} D{D} n{n} {kw}", flush=True)
    L = (n + 31) // 32 * 32 + 64
    lens = [n] if B == 1 else [n, 40]
    q, cache, lt = _problem(B, Hq, Hkv, Sq, D, L, lens, seed=n + Sq, amp=1.5)
    p = mxfa.make_kv4_params(B, Hq, Hkv, Sq, n, D, L, o_fmt=mxfa.C_F32 if f32 else mxfa.C_BF16, **kw)
    shares, ws = mxfa.kv4_attention_plan(p)
    assert shares > 1
    # a workspace of garbage, larger than needed
    got = mxfa.kv4_attention(p, q, cache, kv_len=lt, workspace=torch.full((ws + 512,), 255, dtype=torch.uint8, device=DEV))
    _check(got, _want(q, cache, lens, p, False), p, n, f"{shares} shares")


@pytest.mark.parametrize("B,Hq,Hkv,Sq,D,n,kw,line", [
    (100, 2, 1, 1, 64, 1200, {}, False),                         # pieces of items, more tiles than a wave has lanes
    (80, 8, 4, 1, 64, 1900, {}, True),                           # a line of items cut into shares
    (40, 16, 8, 1, 128, 1900, dict(window=1700), True),
    (68, 8, 4, 9, 64, 1900, {}, True),                           # (two tiles of rows)
    (24, 16, 4, 66, 64, 3300, {}, True),                         # (tiled, three row tiles to a KV head)
    (34, 4, 2, 80, 256, 3300, dict(softcap=30.0), True),
])
def test_attention_of_many_items(B, Hq, Hkv, Sq, D, n, kw, line):
    """Ragged batches whose items are shared out over workgroups: lengths of 0, 1 and around a block's end, and one
    in four long, so that a share ends inside an item, holds many, or none."""
    print(f"many B{B} Hq{Hq} Hkv{Hkv} Sq{Sq} D{D} n{n} {kw}", flush=True)
    L = (n + 31) // 32 * 32
    rng = np.random.default_rng(B + Sq)
    lens = [int(x) for x in np.where(np.arange(B) % 4 == 1, rng.integers(n // 2, n + 1, B), rng.integers(0, 200, B))]
    lens[0], lens[2], lens[3], lens[4], lens[6], lens[-1] = 0, 1, 63, 64, 65, n
    q, cache, lt = _problem(B, Hq, Hkv, Sq, D, L, lens, seed=n + Sq, amp=1.5)
    p = mxfa.make_kv4_params(B, Hq, Hkv, Sq, n, D, L, **kw)
    shares, ws = mxfa.kv4_attention_plan(p)
    rows = Hq // Hkv * Sq
    slots = ws // (4 * (D + 2) * (16 if rows <= 16 else 32 if rows <= 32 else 128))
    assert shares > 1 and slots == (2 * shares if line else shares)
    full = torch.full((ws,), 255, dtype=torch.uint8, device=DEV)
    got = mxfa.kv4_attention(p, q, cache, kv_len=lt, workspace=full)
    _check(got, _want(q, cache, lens, p, False), p, n, f"{shares} shares")
    assert torch.equal(got, mxfa.kv4_attention(p, q, cache, kv_len=lt, workspace=full))
    # an empty batch but for its last sequence
    lens0 = [0] * (B - 1) + [n]
    lt0 = torch.tensor(lens0, dtype=torch.int32, device=DEV)
    last = mxfa.kv4_attention(p, q, cache, kv_len=lt0, workspace=full)
    assert not bool(last[:-1].any())
    _check(last, _want(q, cache, lens0, p, False), p, n, "the last alone")


def test_attention_lengths_are_clamped():
    q, cache, _ = _problem(3, 4, 2, 1, 128, 96, [96, 96, 96], seed=4)
    p = mxfa.make_kv4_params(3, 4, 2, 1, 90, 128, 96)
    got = mxfa.kv4_attention(p, q, cache, kv_len=torch.tensor([-5, 2 ** 31 - 1, 91], dtype=torch.int32, device=DEV))
    want = mxfa.kv4_attention(p, q, cache, kv_len=torch.tensor([0, 90, 90], dtype=torch.int32, device=DEV))
    assert torch.equal(got, want) and bool((got[0] == 0).all())


@pytest.mark.parametrize("Sq", [1, 6, 150])
@pytest.mark.parametrize("f32", [False, True])
def test_attention_strided_q_and_o(Sq, f32):
    """q inside the fused projection's rows and O as [B, Sq, Hq, D], with rows around it left alone."""
    B, Hq, Hkv, D, L = 2, 8, 2, 128, 352
    q, cache, lt = _problem(B, Hq, Hkv, Sq, D, L, [200, 350], seed=21)
    p = mxfa.make_kv4_params(B, Hq, Hkv, Sq, 350, D, L, o_fmt=mxfa.C_F32 if f32 else mxfa.C_BF16)
    want = mxfa.kv4_attention(p, q, cache, kv_len=lt)
    rows = torch.zeros((B, Sq, Hq + 2 * Hkv, D), dtype=torch.bfloat16, device=DEV)
    rows[:, :, :Hq] = q.transpose(1, 2)
    out = torch.full((B, Sq + 1, Hq + 1, D), 7.0, dtype=want.dtype, device=DEV)
    mxfa.kv4_attention(p, rows[:, :, :Hq].transpose(1, 2), cache, kv_len=lt, out=out[:, :Sq, :Hq].transpose(1, 2))
    assert torch.equal(out[:, :Sq, :Hq].transpose(1, 2), want)
    assert bool((out[:, Sq] == 7).all()) and bool((out[:, :, Hq] == 7).all())


@pytest.mark.parametrize("amp", [4.0, 400.0])
@pytest.mark.parametrize("Sq", [1, 40, 150])
def test_attention_of_extreme_scores(Sq, amp):
    """Scores of tens or thousands, growing along the cache (the reference exponent rises again and again), a row
    whose probability sits on one key, and values at both ends of the scale's range."""
    B, Hq, Hkv, D, L, n = 1, 4, 2, 128, 704, 700
    q, cache, lt = _problem(B, Hq, Hkv, Sq, D, L, [n], seed=31, amp=amp)
    ramp = torch.linspace(0.01, 12.0, n, device=DEV)[:, None]
    K = ramp * torch.sign(torch.randn((D,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)))
    V = torch.randn((1, Hkv, n, D), device=DEV)
    V[0, 0] *= 2.0 ** -100
    V[0, 1] *= 2.0 ** 100
    cache.append(K.expand(1, Hkv, n, D).contiguous(), V, pos=torch.zeros(1, dtype=torch.int32, device=DEV))
    for f32 in (False, True):
        p = mxfa.make_kv4_params(B, Hq, Hkv, Sq, n, D, L, o_fmt=mxfa.C_F32 if f32 else mxfa.C_BF16)
        got = mxfa.kv4_attention(p, q, cache, kv_len=lt)
        O, A, X, Y = _want(q, cache, [n], p, False)
        assert X > 10 * amp
        bound = R.attention_bound(O, A, X, Y, D, n, f32, Hq // Hkv * Sq)
        err = (got.double().cpu() - O).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("Sq", [2, 33, 140])
def test_hidden_tokens_do_not_matter(Sq):
    """Whatever lies where no query may look (behind the last token, before the window) leaves O as it is, bit
    for bit: NaN scales, random codes."""
    B, Hq, Hkv, D, L, lens = 2, 8, 2, 128, 480, [190, 401]
    q, cache, lt = _problem(B, Hq, Hkv, Sq, D, L, lens, seed=41)
    p = mxfa.make_kv4_params(B, Hq, Hkv, Sq, 401, D, L, window=100)
    got = mxfa.kv4_attention(p, q, cache, kv_len=lt)
    nb = D // 32
    t = np.arange(L)
    for codes, scales in ((cache.k, cache.ks), (cache.v, cache.vs)):
        c, s = codes.cpu().numpy().copy(), R.scales_by_token(scales.cpu().numpy())
        for b in range(B):
            hidden = (t >= lens[b]) | (t + 100 <= lens[b] - Sq)
            c[b][:, hidden] = 0x5a
            s[b][:, hidden] = 255
        codes.copy_(_dev(c))
        scales.copy_(_dev(R.scales_in_cache(s)))
        assert scales.shape[4] == nb
    assert torch.equal(mxfa.kv4_attention(p, q, cache, kv_len=lt), got)
    assert bool(torch.isfinite(got).all())


def test_nan_in_a_query_stays_in_its_row():
    q, cache, lt = _problem(1, 8, 2, 30, 128, 224, [222], seed=51)
    p = mxfa.make_kv4_params(1, 8, 2, 30, 222, 128, 224)
    want = mxfa.kv4_attention(p, q, cache, kv_len=lt)
    q[0, 3, 11, 5] = float("nan")
    q[0, 6, 2, 100] = float("inf")
    got = mxfa.kv4_attention(p, q, cache, kv_len=lt)
    bad = torch.zeros((8, 30), dtype=torch.bool, device=DEV)
    bad[3, 11] = bad[6, 2] = True
    assert bool(got[0][bad].isnan().all()) and torch.equal(got[0][~bad], want[0][~bad])


def test_offsets_past_32_bits():
    """A cache whose tensors pass 2^32 bytes and whose heads come near 2^31: the last tokens of the last head."""
    B, Hkv, D = 1, 3, 256
    L = (2 ** 31 - 1) // (D // 2) // 32 * 32
    cache = mxfa.Kv4Cache(B, Hkv, D, L)
    n = 70
    g = torch.Generator(device=DEV).manual_seed(61)
    K, V = (torch.randn((B, Hkv, n, D), generator=g, device=DEV) for _ in range(2))
    cache.append(K, V, pos=torch.tensor([L - n], dtype=torch.int32, device=DEV))
    got_k, got_v = cache.read(n, pos=L - n, dtype=torch.float32)
    kv = [R.values(*R.quantize(x.cpu().numpy())) for x in (K, V)]
    assert np.array_equal(got_k.double().cpu().numpy(), kv[0]) and np.array_equal(got_v.double().cpu().numpy(), kv[1])
    for Sq in (1, 40):
        q = torch.randn((B, 2 * Hkv, Sq, D), generator=g, device=DEV).bfloat16()
        p = mxfa.make_kv4_params(B, 2 * Hkv, Hkv, Sq, L, D, L, window=30)
        got = mxfa.kv4_attention(p, q, cache, kv_len=torch.tensor([L], dtype=torch.int32, device=DEV))
        want = R.attention(q.cpu(), *kv, [n], window=30)
        _check(got, want, p, 30, f"Sq {Sq}")


def test_refusals_of_tensors():
    cache = mxfa.Kv4Cache(2, 2, 128, 64)
    x = torch.zeros((2, 2, 3, 128), device=DEV)
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)
    bad = [
        lambda: cache.append(x.cpu(), x), lambda: cache.append(x, x.bfloat16()), lambda: cache.append(x[:, :1], x),
        lambda: cache.append(x.half(), x.half()), lambda: cache.append(x, x, pos=pos.long()), lambda: cache.append(x, x, pos=pos[:1]),
        lambda: cache.append(x, x, pos=pos.cpu()), lambda: cache.append(x, x, counts=torch.zeros(4, dtype=torch.int32, device=DEV)[::2]),
        lambda: cache.append(x.transpose(2, 3).contiguous().transpose(2, 3), x),
        lambda: cache.append(torch.zeros((2, 2, 3, 130), device=DEV)[..., 1:129], x),     # rows off their alignment
        lambda: cache.append(torch.zeros((2, 2, 3, 130), device=DEV)[..., :128], x),
        lambda: cache.append(torch.zeros(128, device=DEV).expand(2, 2, 3, 128), x),
        lambda: cache.read(60, pos=5), lambda: cache.read(3, pos=-1), lambda: cache.read(3, out=(x, x[:1])),
        lambda: cache.read(3, out=(x[:, :, :1].expand(2, 2, 3, 128), x)),
        lambda: cache.read(3, dtype=torch.float32, out=(x.bfloat16(), x.bfloat16())),
        lambda: mxfa.Kv4Cache.of(cache.k, cache.ks[:1], cache.v, cache.vs), lambda: mxfa.Kv4Cache.of(cache.k, cache.ks, cache.v[:, :, :32], cache.vs),
    ]
    p = mxfa.make_kv4_params(2, 4, 2, 1, 64, 128, 64)
    q = torch.zeros((2, 4, 1, 128), dtype=torch.bfloat16, device=DEV)
    o = torch.zeros((2, 4, 1, 128), dtype=torch.bfloat16, device=DEV)
    bad += [
        lambda: mxfa.kv4_attention(p, q.float(), cache), lambda: mxfa.kv4_attention(p, q[:1], cache),
        lambda: mxfa.kv4_attention(p, q, cache, out=o.float()), lambda: mxfa.kv4_attention(p, q, cache, kv_len=pos.long()),
        lambda: mxfa.kv4_attention(p, q, cache, out=o[:, :1].expand(2, 4, 1, 128)),
        lambda: mxfa.kv4_attention(p, q, cache, workspace=torch.zeros(4, device=DEV)),
        lambda: mxfa.kv4_attention(mxfa.make_kv4_params(2, 4, 2, 1, 64, 128, 96), q, cache),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(mxfa.MxfaError):
            f()
            print("not refused:", i)
    assert cache.length == 0 and not bool(cache.k.any())


def test_refusals_of_places_and_counts():
    cache = mxfa.Kv4Cache(2, 2, 128, 64)
    x = torch.zeros((2, 2, 3, 128), device=DEV)
    for f in (lambda: cache.append(x, x, counts=torch.ones(2, dtype=torch.int32, device=DEV)),   # (no common length then)
              lambda: cache.read(3, pos=1 << 32), lambda: cache.read(-1), lambda: cache.read((1 << 32) + 1),
              lambda: mxfa.Kv4Cache.of(cache.k[0], cache.ks, cache.v, cache.vs), lambda: mxfa.Kv4Cache.of(None, None, None, None)):
        with pytest.raises(mxfa.MxfaError):
            f()
    assert cache.length == 0


def test_what_a_call_allocates_belongs_to_its_stream(monkeypatch):
    """Outputs and workspaces come from the stream that the call runs on, handle or object."""
    q, cache, lt = _problem(1, 8, 2, 1, 128, 4128, [4096], seed=3)
    p = mxfa.make_kv4_params(1, 8, 2, 1, 4096, 128, 4128)
    assert mxfa.kv4_attention_plan(p)[1] > 0
    w = torch.ones(128, device=DEV)
    x = torch.randn((5, 128), device=DEV)
    calls = [lambda s: mxfa.kv4_attention(p, q, cache, kv_len=lt, stream=s), lambda s: cache.read(7, stream=s)[0],
             lambda s: mxfa.rmsnorm_quantize(x, w, residual=x, stream=s)[0]]
    want = [f(None) for f in calls]
    torch.cuda.synchronize()
    side, seen, empty = torch.cuda.Stream(), [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (seen.append(torch.cuda.current_stream().cuda_stream), empty(*a, **k))[1])
    for f, y in zip(calls, want):
        for s in (side, side.cuda_stream):
            seen.clear()
            got = f(s)
            assert seen and set(seen) == {side.cuda_stream}
            side.synchronize()
            assert torch.equal(got, y)


def test_graph_and_streams():
    """A decode step over device-side lengths, captured once and replayed while the lengths grow, with eager calls
    of the same kind on another stream in between, equals the eager steps."""
    B, Hq, Hkv, D, L = 3, 8, 2, 128, 2048
    start = [1000, 3, 1900]
    q0, cache, lt = _problem(B, Hq, Hkv, 1, D, L, start, seed=71)
    steps = 4
    g = torch.Generator(device=DEV).manual_seed(72)
    rows = torch.randn((steps, B, 1, Hq + 2 * Hkv, D), generator=g, device=DEV).bfloat16()
    p = mxfa.make_kv4_params(B, Hq, Hkv, 1, L, D, L)
    shares, ws_bytes = mxfa.kv4_attention_plan(p)
    assert shares > 1

    def make():
        c = mxfa.Kv4Cache.of(cache.k.clone(), cache.ks.clone(), cache.v.clone(), cache.vs.clone())
        return dict(c=c, pos=lt.clone(), x=torch.empty_like(rows[0]), o=torch.empty((B, 1, Hq, D), dtype=torch.bfloat16, device=DEV),
                    ws=torch.empty(ws_bytes, dtype=torch.uint8, device=DEV))

    def step(s):
        x = s["x"].transpose(1, 2)
        s["c"].append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], pos=s["pos"])
        s["pos"].add_(1)
        mxfa.kv4_attention(p, x[:, :Hq], s["c"], kv_len=s["pos"], out=s["o"].transpose(1, 2), workspace=s["ws"])

    eager, want = make(), []
    for i in range(steps):
        eager["x"].copy_(rows[i])
        step(eager)
        want.append(eager["o"].clone())
    K, V = (R.cache_values(*x) for x in _bytes(eager["c"]))
    final = R.attention(rows[-1][:, :, :Hq].transpose(1, 2).cpu(), K, V, [n + steps for n in start])
    _check(want[-1].transpose(1, 2), final, p, L)

    s = make()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s)
    torch.cuda.synchronize()
    other, want_other = make(), []
    for i in range(steps):
        s["x"].copy_(rows[i])
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other["x"].copy_(rows[i])
            step(other)
        torch.cuda.synchronize()
        want_other.append(other["o"].clone())
        assert torch.equal(s["o"], want[i]) and torch.equal(other["o"], want[i]), i
    for a, b in zip(_bytes(s["c"]), _bytes(eager["c"])):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("graph", [False, True])
def test_a_decode_step_of_a_layer(graph):
    """Norm, fused projection, append, attention and output projection of one layer for a batch at different
    lengths, as a serving loop runs them, against the same in 64 bits: each stage from the inputs that the
    library's own previous stage gave it."""
    B, Hq, Hkv, D, E, L = 16, 8, 2, 64, 512, 256
    g = torch.Generator(device=DEV).manual_seed(81)
    lens = [int(v) for v in torch.randint(1, 200, (B,), generator=g, device=DEV)]
    _, cache, lt = _problem(B, Hq, Hkv, 1, D, L, lens, seed=82)
    x = torch.randn((B, E), generator=g, device=DEV).bfloat16()
    res = torch.randn((B, E), generator=g, device=DEV).bfloat16()
    w = (1 + 0.1 * torch.randn((E,), generator=g, device=DEV)).bfloat16()
    N = (Hq + 2 * Hkv) * D

    def weights(k, n):
        c, sc = mxfa.quantize_rows(torch.randn((n, k), generator=g, device=DEV) / math.sqrt(k))
        return c.t().contiguous(), sc.t().contiguous()
    wqkv, wo = weights(E, N), weights(Hq * D, E)
    p = mxfa.make_kv4_params(B, Hq, Hkv, 1, L, D, L, o_fmt=mxfa.C_F32)
    ws = torch.empty(mxfa.kv4_attention_plan(p)[1], dtype=torch.uint8, device=DEV)
    pos = lt.clone()
    o = torch.empty((B, 1, Hq, D), device=DEV)
    kept = {}

    def step():
        a, asc, h = mxfa.rmsnorm_quantize(x, w, residual=res, gemm_scales=True)
        qkv = mxfa.gemm(a, asc, *wqkv, c_fmt=mxfa.C_BF16)
        r = qkv.view(B, 1, Hq + 2 * Hkv, D).transpose(1, 2)
        cache.append(r[:, Hq:Hq + Hkv], r[:, Hq + Hkv:], pos=pos)
        kv = pos + 1
        mxfa.kv4_attention(p, r[:, :Hq], cache, kv_len=kv, out=o.transpose(1, 2), workspace=ws)
        oc, osc = mxfa.quantize_rows(o.view(B, Hq * D))
        y = mxfa.gemm(oc, osc.t().contiguous(), *wo, c_fmt=mxfa.C_BF16)
        kept.update(a=a, asc=asc, h=h, qkv=qkv, oc=oc, osc=osc, y=y, kv=kv)

    step()
    if graph:
        first = {k: v.clone() for k, v in kept.items()}
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            step()
        for _ in range(3):
            o.zero_()
            cg.replay()
            torch.cuda.synchronize()
            for k, v in kept.items():
                assert torch.equal(v, first[k]), k
            (x.float() @ x.float().t()).sum().item()            # work of others in between
    torch.cuda.synchronize()
    e4m3 = lambda c: c.view(torch.float8_e4m3fn).double().cpu()  # noqa: E731
    deq = lambda c, s: e4m3(c) * torch.repeat_interleave(torch.ldexp(torch.ones((), dtype=torch.float64), s.cpu().int() - 127), 32, 1)  # noqa: E731
    A = deq(kept["a"], kept["asc"].t())
    want, h = R.norm(x.cpu(), w.cpu(), 1e-6, residual=res.cpu())
    assert torch.equal(kept["h"].cpu(), h)
    # E4M3 with a floor scale: an element is off by at most 1/8 of itself (saturation) or 2^-6 of its block's scale
    assert np.all(np.abs(A.numpy() - want) <= 0.13 * np.abs(want) + 2.0 ** -14 * np.abs(want).max())
    qkv = A @ deq(wqkv[0].t().contiguous(), wqkv[1].t()).t()
    # the matrix unit cuts each of 8 products to 2^-13 of the largest: 2^-10 of the sum of magnitudes, and bf16's half step
    mag = A.abs() @ deq(wqkv[0].t().contiguous(), wqkv[1].t()).t().abs()
    got = kept["qkv"].double().cpu()
    assert bool(((got - qkv).abs() <= 2.0 ** -8 * qkv.abs() + 2.0 ** -10 * mag).all())
    r = kept["qkv"].view(B, 1, Hq + 2 * Hkv, D).transpose(1, 2).cpu()
    K, V = (R.cache_values(*c) for c in _bytes(cache))
    for i, (cv, new) in enumerate(((K, r[:, Hq:Hq + Hkv]), (V, r[:, Hq + Hkv:]))):
        vals = R.values(*R.quantize(new.float().numpy()))
        for b in range(B):
            assert np.array_equal(cv[b, :, lens[b]], vals[b, :, 0])
    _check(o.transpose(1, 2), R.attention(r[:, :Hq], K, V, [n + 1 for n in lens]), p, 201)
    Y = deq(kept["oc"], kept["osc"])
    Wo = deq(wo[0].t().contiguous(), wo[1].t()).t()
    assert bool(((kept["y"].double().cpu() - Y @ Wo).abs() <= 2.0 ** -8 * (Y @ Wo).abs() + 2.0 ** -10 * (Y.abs() @ Wo.abs())).all())
