"""The 8-bit cache and its rotation on the GPU, against plain implementations
(tests/q8_ref.py).  Every bound below follows from the formats:

rotation   one rounding of the output's type, and for each pair of length r an
           angle held to 2^-24 half turns and cosines to two units: 4e-7 r
write      codes and scales equal the definition's, bit for bit
read       equal to code * scale rounded once
attention  half a unit of the output's type; softmax weights in 16 bits: 2^-11
           of sum p|v| (2^-25 of the largest |v| for each weight below the
           normal range); scores summed in 32 bits: 2^-19 of the largest
           sum |q k| in each exponent, for the weight and for the sum
"""
import ctypes as C

import numpy as np
import pytest
import torch

import q8_ref as R
import spb200

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _batch(new, kv, seq=None, max_new=None, max_kv=None):
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    return spb200.Q8Batch(_i32(cu), _i32(kv), cu[-1], max(new) if max_new is None else max_new,
                          max(kv) if max_kv is None else max_kv, None if seq is None else _i32(seq))


# -------------------------------------------------------------- rotation --

ROPE = [
    # tokens, heads of q and k, hd, rot, sections, pairing, interleave, ladder
    (1, 1, 1, 64, 64, [32], "adjacent", False, False),
    (5, 32, 8, 128, 128, [16, 24, 24], "adjacent", False, False),
    (77, 7, 3, 128, 128, [16, 24, 24], "halves", False, True),
    (130, 5, 1, 256, 192, [40, 28, 28], "halves", True, False),
    (33, 4, 2, 80, 48, [10, 0, 7, 7], "adjacent", True, True),
    (300, 28, 4, 64, 48, [24], "halves", False, False),
    (1000, 2, 2, 512, 512, [128, 128], "adjacent", True, False),
]


@pytest.mark.parametrize("case", ROPE, ids=[str(i) for i in range(len(ROPE))])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope_matches_formula(cuda, case, dtype, inverse):
    T, hq, hk, hd, rot, sections, pairing, inter, ladder = case
    rng = np.random.default_rng(5)
    pos = rng.integers(-1000, 200000, (len(sections), T)).astype(np.int32)
    plan = spb200.RopeAxes(hd, sections, pairing=pairing, interleave=inter, axis_ladder=ladder, theta=1e4)
    xs = [torch.from_numpy(rng.standard_normal((T, h, hd))).to(R.DTYPES[dtype]).cuda() for h in (hq, hk)]
    got = plan.apply(torch.from_numpy(pos).cuda(), *xs, inverse=inverse)
    for x, y in zip(xs, got):
        x = x.double().cpu().numpy()
        want = R.rope(x, pos, sections, rot, pairing, inter, ladder, 1e4, -1.0 if inverse else 1.0)
        half = rot // 2
        if pairing == "adjacent":
            r = np.repeat(np.hypot(x[..., 0:rot:2], x[..., 1:rot:2]), 2, -1)
        else:
            r = np.tile(np.hypot(x[..., :half], x[..., half:rot]), 2)
        tol = R.EPS[dtype] * np.abs(want)
        tol[..., :rot] += 4e-7 * r + (2.0 ** -25 if dtype == "f16" else 0.0)
        off = np.abs(y.double().cpu().numpy() - want)
        assert (off <= tol).all(), float((off - tol).max())


def test_rope_in_place_strided_and_one_half(cuda):
    """A fused projection's rows turned in place; keys alone; another stream."""
    T, hq, hk, hd = 19, 6, 2, 128
    qkv = torch.randn(T, hq + 2 * hk, hd, device="cuda", dtype=torch.float16)
    pos = torch.randint(0, 5000, (3, T), device="cuda", dtype=torch.int32)
    plan = spb200.RopeAxes(hd, [16, 24, 24], pairing="halves")
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    v = qkv[:, hq + hk:].clone()
    want = plan.apply(pos, q.contiguous(), k.contiguous())
    only, alone = plan.apply(pos, None, k.contiguous())
    assert only is None and torch.equal(alone, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    plan.apply(pos, q, k, q_out=q, k_out=k, stream=side)
    side.synchronize()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, hq + hk:], v)


def test_rope_gradient(cuda):
    """The inverse is the transpose: <R x, g> = <x, R^-1 g>, and it agrees with
    differences of the loss along random directions."""
    T, h, hd = 11, 3, 64
    plan = spb200.RopeAxes(hd, [8, 12, 12], interleave=True)
    pos = torch.randint(0, 9000, (3, T), device="cuda", dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, gy, d = (torch.randn(T, h, hd, device="cuda", generator=g) for _ in range(3))
    gx = plan.apply(pos, gy, None, inverse=True)[0]

    def loss(z):
        return (plan.apply(pos, z, None)[0].double() * gy.double()).sum().item()
    step = 2.0 ** -3            # the loss is linear: a large step only rounds less
    numeric = (loss(x + step * d) - loss(x - step * d)) / (2 * step)
    exact = (gx.double() * d.double()).sum().item()
    size = gy.double().norm().item() * (x.double().norm().item() / step + d.double().norm().item())
    assert abs(numeric - exact) <= 4e-7 * size


def test_rope_factors_and_empty(cuda):
    T, hd = 6, 64
    ff = np.linspace(0.05, 8.0, hd // 2).astype(np.float32)      # below 1/(2 pi): more than a turn for each step
    plan = spb200.RopeAxes(hd, [hd // 2], freq_factors=ff.tolist())
    pos = np.array([[0, 1, 7, 1000, 123456, 2 ** 31 - 1]], np.int32)
    x = torch.randn(T, 2, hd, device="cuda")
    got = plan.apply(torch.from_numpy(pos).cuda(), x, None)[0].double().cpu().numpy()
    want = R.rope(x.double().cpu().numpy(), pos, [hd // 2], hd, "adjacent", False, False, 1e4, factors=ff.astype(np.float64))
    # 64-bit angles themselves are off by 2^-53 of up to 2^31 / 0.05 radians
    assert np.abs(got - want).max() <= 2e-5
    empty = torch.empty(0, 2, hd, device="cuda")
    assert plan.apply(torch.empty(1, 0, dtype=torch.int32, device="cuda"), empty, None)[0].shape[0] == 0


# ---------------------------------------------------------- write and read --

def _fill(cache, seed, scale_sigma=0.3):
    """Random codes and scales everywhere; returns them on the CPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    got = []
    for which in (0, 1):
        c, s = cache.slab(which), cache.scales(which)
        x = torch.randn(c.shape, generator=g, device="cuda") * (40.0 if cache.fmt == "int8" else 60.0)
        x *= torch.empty(1, 1, cache.n_heads_kv, 1, cache.head_dim, device="cuda").log_normal_(0, 0.3, generator=g)
        c.view(torch.uint8).copy_(R.code(x.cpu(), cache.fmt).view(c.shape))
        s.copy_(torch.empty(s.shape, device="cuda").log_normal_(-3.5, scale_sigma, generator=g))
        got += [c.view(torch.uint8).cpu(), s.cpu()]
    return got


WRITES = [
    # hd, heads, block, [(start, n), ...] one for each sequence
    (64, 1, 16, [(0, 1)]),
    (64, 3, 16, [(15, 1), (16, 1), (17, 30), (0, 0)]),
    (128, 8, 64, [(0, 200), (63, 2), (70, 1), (64, 64), (127, 129)]),
    (128, 2, 128, [(5, 300), (300, 5)]),
    (256, 2, 32, [(31, 33), (32, 32), (1, 1)]),
    (256, 4, 128, [(100, 156)]),
]


@pytest.mark.parametrize("case", WRITES, ids=[str(i) for i in range(len(WRITES))])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write_matches_definition(cuda, case, fmt, dtype):
    hd, H, B, spans = case
    n = len(spans)
    cache = spb200.Q8Cache(hd, 2, H, 512, n_seqs=n, fmt=fmt, block_tokens=B)
    want = _fill(cache, 7)
    new, kv = [m for _, m in spans], [s + m for s, m in spans]
    g = torch.Generator().manual_seed(11)
    x = [torch.randn(sum(new), H, hd, generator=g) * s for s in (3.0, 0.4)]      # the first makes old scales grow
    x = [t.to(R.DTYPES[dtype]) for t in x]
    cache.write_kv_tokens(1, _batch(new, kv), x[0].cuda(), x[1].cuda())
    assert cache.status() == 0
    for which in (0, 1):
        codes, scales = want[2 * which], want[2 * which + 1]
        at = 0
        for i, (s, m) in enumerate(spans):
            for h in range(H):
                R.write(codes[1, i, h], scales[1, i, h], x[which][at:at + m, h].float(), s, B, fmt)
            at += m
        assert torch.equal(cache.scales(which).cpu(), scales)
        assert torch.equal(cache.slab(which).view(torch.uint8).cpu(), codes)
        # and the definition in 64 bits: half a step, or half a unit of the code
        at = 0
        for i, (s, m) in enumerate(spans):
            y = x[which][at:at + m].double().transpose(0, 1)
            sc = scales[1, i].double().repeat_interleave(B, -1)[:, s:s + m, None]
            off = (R.values(codes[1, i], fmt)[:, s:s + m].double() * sc - y).abs()
            step = sc / 2 if fmt == "int8" else torch.maximum(y.abs() * 2.0 ** -4, sc * 2.0 ** -10)
            # the reciprocal's and the product's roundings, and the scale's, are relative to the value
            assert (off <= step + y.abs() * 2.0 ** -22).all()
            at += m


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_odd_values(cuda, fmt):
    """Zeros, infinities, NaN, tiny and huge values; a block is never left without a scale."""
    hd, B = 64, 16
    x = torch.zeros(5 * B, 1, hd)
    x[B:2 * B] = torch.randn(B, 1, hd)
    x[B, 0, :3] = torch.tensor([float("inf"), -float("inf"), float("nan")])
    x[2 * B:3 * B] = torch.randn(B, 1, hd) * 1e-30
    x[3 * B:4 * B] = torch.randn(B, 1, hd) * 1e38
    x[4 * B:] = float("inf")
    cache = spb200.Q8Cache(hd, 1, 1, 5 * B, fmt=fmt, block_tokens=B)
    cache.write_kv_tokens(0, _batch([5 * B], [5 * B]), x.cuda(), None)
    codes, scales = torch.zeros(128, hd, dtype=torch.uint8), torch.zeros(8)
    R.write(codes, scales, x[:, 0], 0, B, fmt)
    assert torch.equal(cache.scales(0).cpu()[0, 0, 0], scales)
    got = cache.slab(0)[0, 0, 0].view(torch.uint8).cpu()
    assert torch.equal(R.values(got, fmt), R.values(codes, fmt))
    assert torch.isfinite(R.values(got, fmt)).all()
    assert not cache.slab(1).view(torch.uint8).any()          # no values were given: that half is untouched


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_token_by_token_and_rollback(cuda, fmt):
    """Appended one by one, and begun again after some tokens were taken back."""
    hd, H, B = 128, 2, 32
    cache = spb200.Q8Cache(hd, 1, H, 128, fmt=fmt, block_tokens=B)
    codes, scales = torch.zeros(H, 128, hd, dtype=torch.uint8), torch.zeros(H, 128 // B)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(60, H, hd, generator=g) * torch.linspace(0.2, 4.0, 60)[:, None, None]
    for p, n in [(i, 1) for i in range(40)] + [(33, 4), (36, 1), (37, 20)]:
        cache.write_kv_tokens(0, _batch([n], [p + n]), x[:n].cuda() * (1 + p / 10), x[:n].cuda())
        for h in range(H):
            R.write(codes[h], scales[h], x[:n, h] * (1 + p / 10), p, B, fmt)
    assert torch.equal(cache.scales(0)[0, 0].cpu(), scales)
    assert torch.equal(cache.slab(0)[0, 0].view(torch.uint8).cpu(), codes)


def test_write_sequence_ids_strides_stream(cuda):
    """Entries name their sequences; k and v are slices of a fused projection;
    the cache's stream is not the current one."""
    hd, H = 64, 2
    side = torch.cuda.Stream()
    cache = spb200.Q8Cache(hd, 1, H, 128, n_seqs=7, block_tokens=16, stream=side)
    qkv = torch.randn(9, 3 * H, hd, device="cuda", dtype=torch.bfloat16)
    k, v = qkv[:, H:2 * H], qkv[:, 2 * H:]
    b = _batch([2, 0, 7], [2, 50, 27], seq=[5, 0, 3])
    side.wait_stream(torch.cuda.current_stream())
    cache.write_kv_tokens(0, b, k, v)
    out = torch.empty(7, H, hd, device="cuda")
    cache.read_kv_tokens(1, 0, 3, 20, out)
    side.synchronize()
    flat = spb200.Q8Cache(hd, 1, H, 128, n_seqs=7, block_tokens=16)
    flat.write_kv_tokens(0, b, k.contiguous(), v.contiguous())
    torch.cuda.synchronize()
    for which in (0, 1):
        assert torch.equal(cache.slab(which), flat.slab(which)) and torch.equal(cache.scales(which), flat.scales(which))
    step = cache.scales(1)[0, 3, :, 1]
    assert ((out - v[2:].float()).abs() <= step[None, :, None] * 0.5001).all()
    assert not cache.slab(0)[0, [0, 1, 2, 4, 6]].any()


@pytest.mark.parametrize("hd,H,B,start,n", [(64, 1, 16, 0, 1), (64, 5, 16, 13, 77), (128, 8, 64, 100, 412),
                                            (256, 3, 128, 127, 2), (256, 1, 32, 0, 512)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read_matches_definition(cuda, hd, H, B, start, n, fmt, dtype):
    cache = spb200.Q8Cache(hd, 2, H, 512, n_seqs=2, fmt=fmt, block_tokens=B)
    got = _fill(cache, 3)
    for which in (0, 1):
        out = torch.empty(n, H, hd, device="cuda", dtype=R.DTYPES[dtype])
        cache.read_kv_tokens(which, 1, 1, start, out)
        c, s = got[2 * which][1, 1], got[2 * which + 1][1, 1]
        want = (R.values(c, fmt) * s.repeat_interleave(B, -1)[..., None])[:, start:start + n]
        assert torch.equal(out.cpu(), want.transpose(0, 1).to(R.DTYPES[dtype]))


def test_views_keep_their_cache(cuda):
    """A slab or scale view outlives the handle it was taken from."""
    import gc
    import weakref
    cache = spb200.Q8Cache(64, 1, 1, 128)
    alive, codes, scales = weakref.ref(cache), cache.slab(0), cache.scales(1)
    del cache
    gc.collect()
    assert alive() is not None
    del codes
    gc.collect()
    assert alive() is not None
    del scales
    gc.collect()
    assert alive() is None


# --------------------------------------------------------------- attention --

def _check_attn(cache, fills, layer, q, new, kv, seq, out, lse, scale, causal, window):
    kc, ks, vc, vs = fills
    B, H, hd = cache.block_tokens, cache.n_heads_kv, cache.head_dim
    G = q.shape[1] // H
    dtype = {torch.float16: "f16", torch.bfloat16: "bf16"}[q.dtype]
    q, out = q.double().cpu().numpy(), out.double().cpu().numpy()
    lse = None if lse is None else lse.double().cpu().numpy()
    at = 0
    for i, (m, n) in enumerate(zip(new, kv)):
        s = i if seq is None else seq[i]
        for h in range(H):
            k, v = (((R.values(c[layer, s, h, :n], cache.fmt).double()
                      * x[layer, s, h].double().repeat_interleave(B)[:n, None])).numpy() for c, x in ((kc, ks), (vc, vs)))
            rows = slice(h * G, h * G + G)
            pos = np.arange(n - m, n)
            want, wl, pv, size = R.attend(q[at:at + m, rows], k, v, pos, scale, causal, window)
            got = out[at:at + m, rows]
            vmax = np.abs(v).max(initial=0.0)
            tol = (R.EPS[dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -18 * (1 + size)) * pv + n * 2.0 ** -25 * vmax
                   + (2.0 ** -25 if dtype == "f16" else 0.0))
            off = np.abs(got - want)
            if dtype == "f16":          # past fp16's largest value the output is infinite
                past = np.abs(want) + tol >= 65520.0
                assert (np.abs(got[past]) >= 65504.0 - tol[past]).all() and (np.sign(got[past]) == np.sign(want[past])).all()
                off = np.where(past, 0.0, off)
            assert (off <= tol).all(), (i, h, float((off / np.maximum(tol, 1e-30)).max()))
            if lse is not None:
                gl = lse[at:at + m, rows]
                assert np.array_equal(np.isneginf(gl), np.isneginf(wl))
                ok = np.isfinite(wl)
                assert (np.abs(gl[ok] - wl[ok]) <= 2.0 ** -18 * (1 + size)).all()
        at += m


def _run_attn(hd, H, G, B, fmt, dtype, new, kv, causal=True, window=0, seq=None, max_seq=None, layer=0, n_layers=1,
              strided=False, garbage=True, scale=None, want_lse=True, max_new=None, max_kv=None, n_seqs=None):
    n_seqs = n_seqs or len(kv)
    cache = spb200.Q8Cache(hd, n_layers, H, max_seq or max(max(kv), 1), n_seqs=n_seqs, fmt=fmt, block_tokens=B)
    fills = _fill(cache, 17)
    if garbage:                 # what lies past a sequence's end must not matter
        for i, n in enumerate(kv):
            s = i if seq is None else seq[i]
            for which in (0, 1):
                cache.slab(which).view(torch.uint8)[:, s, :, n:] = 0x7f
                cache.scales(which)[:, s, :, (n + B - 1) // B:] = float("nan")
    g = torch.Generator(device="cuda").manual_seed(23)
    T = sum(new)
    if strided:
        q = torch.randn(T, H * G + 2 * H, hd, generator=g, device="cuda").to(R.DTYPES[dtype])[:, :H * G]
        out = torch.zeros(T, H * G + 8, hd, device="cuda", dtype=R.DTYPES[dtype])[:, :H * G]
    else:
        q = torch.randn(T, H * G, hd, generator=g, device="cuda").to(R.DTYPES[dtype])
        out = torch.full_like(q, 7.0)
    lse = torch.full((T, H * G), 7.0, device="cuda") if want_lse else None
    scale = scale if scale is not None else 2.0 / np.sqrt(hd)
    b = _batch(new, kv, seq, max_new, max_kv)
    cache.attn(layer, b, q, out=out, lse=lse, logit_scale=scale, causal=causal, window=window)
    assert cache.status() == 0
    _check_attn(cache, fills, layer, q, new, kv, seq, out, lse, scale, causal, window)
    first = out.clone()
    for _ in range(2):          # the same bits again: no order of arrival in the results
        cache.attn(layer, b, q, out=out, lse=lse, logit_scale=scale, causal=causal, window=window)
        assert torch.equal(out, first)
    return cache, q, out


SHAPES = [
    # hd, H, G, B, new, kv, window
    (128, 2, 4, 64, [1], [1], 0),
    (128, 2, 4, 64, [1, 1, 1], [1, 17, 300], 0),
    (128, 1, 1, 16, [1, 1], [15, 16], 0),
    (128, 8, 4, 32, [1], [2049], 0),
    (64, 4, 8, 16, [4, 1, 3], [4, 1000, 131], 0),
    (64, 2, 3, 128, [2, 5], [129, 77], 0),
    (256, 2, 8, 128, [1, 2], [600, 63], 0),
    (256, 1, 2, 16, [3], [3], 0),
    (128, 1, 16, 64, [1, 2], [700, 5], 0),
    (128, 1, 31, 64, [1], [200], 0),
    (64, 1, 128, 64, [1], [333], 0),
    (128, 2, 4, 64, [64], [64], 0),
    (128, 2, 4, 64, [100, 7, 33], [100, 407, 33], 0),
    (128, 1, 1, 16, [257], [600], 0),
    (64, 2, 2, 32, [130, 1], [400, 400], 0),
    (256, 1, 4, 64, [70], [300], 0),
    (256, 2, 1, 128, [129, 128], [129, 500], 0),
    (128, 2, 4, 64, [90], [700], 65),
    (64, 1, 4, 16, [40, 1], [300, 500], 1),
    (256, 1, 2, 32, [50, 3], [333, 200], 17),
    (128, 1, 5, 128, [1], [1000], 100),
    (128, 1, 4, 64, [300], [300], 5000),
]


@pytest.mark.parametrize("case", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("fmt,dtype", [("int8", "f16"), ("e4m3", "bf16")])
def test_attn_matches_formula(cuda, case, fmt, dtype):
    hd, H, G, B, new, kv, window = case
    _run_attn(hd, H, G, B, fmt, dtype, new, kv, window=window)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fmt,dtype", [("int8", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("new", [[1, 2, 0, 1], [130, 3, 0, 40]])
def test_attn_not_causal(cuda, hd, fmt, dtype, new):
    _run_attn(hd, 2, 2, 32, fmt, dtype, new, [200, 5, 9, 333], causal=False)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("many", [False, True])
def test_attn_empty_rows(cuda, hd, many):
    """Entries without positions, without tokens, and with more tokens than positions."""
    new = [3, 0, 2, 1] if not many else [80, 0, 50, 1]
    kv = [0, 40, 1, 0] if not many else [0, 40, 20, 3]
    _, _, out = _run_attn(hd, 2, 4, 16, "int8", "f16", new, kv)
    assert not out[:new[0]].any()
    _run_attn(hd, 2, 4, 16, "e4m3", "bf16", new, kv, causal=False)


@pytest.mark.parametrize("new", [[1, 3, 1], [1, 40, 70]])
def test_attn_sequences_strides_layers(cuda, new):
    _run_attn(128, 2, 4, 32, "int8", "f16", new, [100, 260, 70], seq=[4, 0, 2], n_seqs=6, max_seq=300, layer=2,
              n_layers=3, strided=True, want_lse=False)


@pytest.mark.parametrize("new", [[1, 1], [2, 100]])
def test_attn_loose_bounds(cuda, new):
    """max_new and max_kv may be larger than what the batch has."""
    _run_attn(128, 2, 4, 32, "e4m3", "f16", new, [333, 150], max_seq=2000, max_new=500, max_kv=2048)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 100])
def test_attn_scales_far_apart(cuda, fmt, new):
    """A first block that takes most of the weight but has tiny values, a block of
    zeros, and blocks whose scales span 2^-40 .. 2^12: every weight counts in the sum."""
    hd, H, B, n = 128, 1, 16, 160
    cache = spb200.Q8Cache(hd, 1, H, n, fmt=fmt, block_tokens=B)
    fills = _fill(cache, 5)
    for c, s in ((0, [0, 1]), (1, [2, 3])):
        fills[s[1]][0, 0, 0, :10] = torch.tensor([2.0 ** -12, 0.03, 0.02, 0.05, 0.01, 2.0 ** -40, 0.03, 0.02, 2.0 ** -20, 0.04])
        if c == 0:
            fills[s[1]][0, 0, 0, :10] = 0.02
        else:
            fills[s[0]][0, 0, 0, 5 * B:6 * B] = 0
            fills[s[1]][0, 0, 0, 9] = 2.0 ** 12
        cache.slab(c).view(torch.uint8).copy_(fills[s[0]])
        cache.scales(c).copy_(fills[s[1]])
    for end in (B, 5 * B + 3, 6 * B, 9 * B, n):
        for scale in (0.0, 0.05, 2.0):
            m = min(new, end)
            q = torch.randn(m, 4, hd, device="cuda", dtype=torch.float16)
            out, lse = torch.empty_like(q), torch.empty(m, 4, device="cuda")
            cache.attn(0, _batch([m], [end]), q, out=out, lse=lse, logit_scale=scale)
            _check_attn(cache, fills, 0, q, [m], [end], None, out, lse, scale, True, 0)


@pytest.mark.parametrize("new", [1, 100])
def test_attn_large_and_small_queries(cuda, new):
    """bf16 queries far outside fp16's range, rows of zeros, large logits."""
    hd, n = 128, 300
    cache = spb200.Q8Cache(hd, 1, 1, n, fmt="int8", block_tokens=64)
    fills = _fill(cache, 9)
    q = torch.randn(new, 4, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    q[:, 0] *= 1e20
    q[:, 1] *= 1e-20
    q[:, 2] = 0
    q = q.to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(new, 4, device="cuda")
    for head, scale in ((0, 3e-21), (1, 3e19), (2, 1.0), (3, 20.0)):
        cache.attn(0, _batch([new], [n]), q, out=out, lse=lse, logit_scale=scale)
        one = q[:, head:head + 1]
        _check_attn(cache, fills, 0, one, [new], [n], None, out[:, head:head + 1], lse[:, head:head + 1], scale, True, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [[1, 1], [33, 1]])
def test_attn_long(cuda, fmt, new):
    """Tens of thousands of positions: the split rows and their join."""
    _run_attn(128, 2, 4, 64, fmt, "f16", new, [40000, 9000], scale=1.0 / np.sqrt(128))


def test_attn_past_32_bits(cuda):
    """The last layer of a cache whose slabs are over 4 GiB each."""
    hd, L, H, S = 128, 9, 8, 65536
    cache = spb200.Q8Cache(hd, L, H, S, n_seqs=8, block_tokens=64)
    assert cache.slab(0).numel() > 2 ** 32
    q = torch.randn(70, 8, hd, device="cuda", dtype=torch.float16)
    k, v = (torch.randn(200, H, hd, device="cuda", dtype=torch.float16) for _ in range(2))
    b = _batch([200], [S], seq=[7])
    cache.write_kv_tokens(L - 1, b, k, v)
    small = spb200.Q8Cache(hd, 1, H, 256, block_tokens=64)
    small.write_kv_tokens(0, _batch([200], [256]), k, v)
    for m in (1, 70):
        got = cache.attn(L - 1, _batch([m], [S], seq=[7]), q[:m], logit_scale=0.1, window=100)
        want = small.attn(0, _batch([m], [256]), q[:m], logit_scale=0.1, window=100)
        # the same sums in other splits
        assert ((got.float() - want.float()).abs() <= 2.0 ** -9).all()
    out, ref = torch.empty(150, H, hd, device="cuda"), torch.empty(150, H, hd, device="cuda")
    cache.read_kv_tokens(0, L - 1, 7, S - 150, out)
    small.read_kv_tokens(0, 0, 0, 256 - 150, ref)
    assert torch.equal(out, ref)


def test_attn_stream_and_graph(cuda):
    """On another stream, and replayed from a graph with other lengths."""
    hd, H = 128, 2
    cache = spb200.Q8Cache(hd, 1, H, 1024, fmt="e4m3", block_tokens=64)
    _fill(cache, 4)
    q = torch.randn(1, 8, hd, device="cuda", dtype=torch.float16)
    kv, cu = _i32([1000]), _i32([0, 1])
    b = spb200.Q8Batch(cu, kv, 1, 1, 1024)
    want = {}
    for n in (1000, 37):
        kv.fill_(n)
        want[n] = cache.attn(0, b, q, logit_scale=0.1).clone()
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.attn(0, b, q, out=out, logit_scale=0.1, stream=side)
    for n in (37, 1000, 37):
        kv.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[n])


def test_bad_entries_are_skipped(cuda):
    """Lengths out of range are found by the kernels: those entries are skipped and reported."""
    hd, H = 64, 1
    cache = spb200.Q8Cache(hd, 1, H, 128, n_seqs=4, block_tokens=16)
    k = torch.randn(8, H, hd, device="cuda", dtype=torch.float16)
    for kv, cu, seq in (([2, 1], [0, 2, 4], None),              # two new tokens, one position
                        ([2, 300], [0, 2, 4], None),            # past the cache's end
                        ([2, -1], [0, 2, 4], None),
                        ([2, 3], [0, 2, 9], None),              # past the packed tokens
                        ([2, 3], [0, 2, 1], None),              # descending
                        ([2, 3], [0, 2, 4], [0, 4])):           # no such sequence
        b = spb200.Q8Batch(_i32(cu), _i32(kv), 8, 4, 128, None if seq is None else _i32(seq))
        cache.write_kv_tokens(0, b, k, k)
        assert cache.status(clear=True) == 1
        assert cache.slab(0)[0, 0].any() and not cache.slab(0)[0, 1:].any()
        if kv[1] != 1:
            out = torch.full((8, 2, hd), 7.0, device="cuda", dtype=torch.float16)
            q = torch.randn(8, 2, hd, device="cuda", dtype=torch.float16)
            cache.attn(0, b, q, out=out, logit_scale=0.1)
            assert cache.status(clear=True) == 1
            assert (out[:2] != 7.0).any() and (out[2:] == 7.0).all()
    assert cache.status() == 0


def test_refusals(cuda):
    L = spb200.lib()
    cache = spb200.Q8Cache(128, 2, 2, 256, n_seqs=2)
    x = torch.zeros(4, 2, 128, device="cuda", dtype=torch.float16)
    q = torch.zeros(4, 8, 128, device="cuda", dtype=torch.float16)
    b = _batch([2, 2], [2, 2])
    p, st = x.data_ptr(), q.data_ptr()
    arg, uns = spb200.SP_ERR_ARG, spb200.SP_ERR_UNSUPPORTED
    w, a, r = L.sp_cuda_q8_write_kv_tokens, L.sp_cuda_q8_attn, L.sp_cuda_q8_read_kv_tokens
    qc = cache._ref
    assert w(qc, 2, b.ref, p, p, 0, 1) == arg                     # layer
    assert w(qc, -1, b.ref, p, p, 0, 1) == arg
    assert w(qc, 0, b.ref, p + 2, p, 0, 1) == arg                 # alignment
    assert w(qc, 0, b.ref, p, p, 260, 1) == arg
    assert w(qc, 0, b.ref, p, p, 128, 1) == arg                   # stride
    assert w(qc, 0, b.ref, p, p, 0, 3) == arg                     # type
    assert w(qc, 0, None, p, p, 0, 1) == arg
    assert w(None, 0, b.ref, p, p, 0, 1) == arg
    assert w(C.byref(spb200.SpQ8Cache()), 0, b.ref, p, p, 0, 1) == arg
    assert "not initialised" in spb200.last_error()[1]
    assert w(qc, 0, b.ref, None, None, 0, 1) == 0                 # nothing to write
    for field, value in (("n_seqs", 3), ("n_seqs", -1), ("n_tokens", -1), ("max_new", -1), ("max_kv", 257), ("d_cu", None),
                         ("d_kv_len", None)):
        bad = spb200.SpQ8Batch.from_buffer_copy(b.b)
        setattr(bad, field, value)
        assert w(qc, 0, C.byref(bad), p, p, 0, 1) == arg, field
        assert a(qc, 0, C.byref(bad), st, 0, 8, 1, 1.0, 1, 0, st, 0, None, None) == arg, field
    assert a(qc, 0, b.ref, st, 0, 8, 0, 1.0, 1, 0, st, 0, None, None) == uns     # fp32 queries
    assert a(qc, 0, b.ref, st, 0, 7, 1, 1.0, 1, 0, st, 0, None, None) == arg     # heads
    assert a(qc, 0, b.ref, st, 0, 258, 1, 1.0, 1, 0, st, 0, None, None) == arg
    assert a(qc, 0, b.ref, st, 0, 8, 1, float("nan"), 1, 0, st, 0, None, None) == arg
    assert a(qc, 0, b.ref, st, 0, 8, 1, 1.0, 0, 5, st, 0, None, None) == arg     # window without causal
    assert a(qc, 0, b.ref, st, 0, 8, 1, 1.0, 1, -1, st, 0, None, None) == arg
    assert a(qc, 0, b.ref, st + 8, 0, 8, 1, 1.0, 1, 0, st, 0, None, None) == arg
    assert a(qc, 0, b.ref, st, 1028, 8, 1, 1.0, 1, 0, st, 0, None, None) == arg
    assert a(qc, 0, b.ref, None, 0, 8, 1, 1.0, 1, 0, st, 0, None, None) == arg
    assert r(qc, 2, 0, 0, 0, 1, p, 1) == arg
    assert r(qc, 0, 0, 2, 0, 1, p, 1) == arg
    assert r(qc, 0, 0, 0, 255, 2, p, 1) == arg
    assert r(qc, 0, 0, 0, -1, 2, p, 1) == arg
    assert r(qc, 0, 0, 0, 0, 1, p + 4, 1) == arg
    assert r(qc, 0, 0, 0, 0, 0, None, 1) == 0
    plan = spb200.RopeAxes(128, [64])
    f = L.sp_cuda_rope_axes
    assert f(plan._ref, st, 4, st, 0, 8, None, 0, None, 0, 0, None, 0, 1, 0, None) == arg     # no output
    assert f(plan._ref, st, 4, st, 0, 8, st, 2048, None, 0, 0, None, 0, 1, 0, None) == arg    # in place, two strides
    assert f(plan._ref, st, 4, st + 4, 0, 8, st, 0, None, 0, 0, None, 0, 1, 0, None) == arg
    assert f(plan._ref, None, 4, st, 0, 8, st, 0, None, 0, 0, None, 0, 1, 0, None) == arg
    assert f(plan._ref, st, 4, st, 0, 8, st, 0, None, 0, 0, None, 0, 5, 0, None) == arg
    assert f(plan._ref, st, 4, st, 0, 8, st, 4, None, 0, 0, None, 0, 1, 0, None) == arg
    with pytest.raises(ValueError):
        cache.attn(0, b, q[:, :, :64])
    with pytest.raises(ValueError):
        cache.write_kv_tokens(0, b, x[:2], x[:2])
    with pytest.raises(RuntimeError):
        spb200.Q8Cache(96, 1, 1, 128)
    with pytest.raises(RuntimeError):
        spb200.Q8Cache(128, 1, 1, 128, block_tokens=48)
    torch.cuda.synchronize()


@pytest.mark.parametrize("hd,H,G,fmt", [(256, 2, 8, "e4m3"), (128, 2, 4, "int8"), (64, 3, 2, "e4m3")])
def test_attn_many_tiles_again_and_again(cuda, hd, H, G, fmt):
    """Long chunks of several entries: runs that end and begin inside units, the
    roles of the many-row kernel far apart.  Every pass gives the same bits and
    no wait runs out."""
    new, kv = [301, 1, 700, 95], [3000, 2500, 5000, 95]
    cache, q, first = _run_attn(hd, H, G, 64, fmt, "f16", new, kv, scale=1.0 / np.sqrt(hd))
    b = _batch(new, kv)
    for _ in range(40):
        out = cache.attn(0, b, q, logit_scale=1.0 / np.sqrt(hd))
        assert torch.equal(out, first)
    assert cache.status() == 0


@pytest.mark.parametrize("most", [1, 40])
def test_attn_many_entries(cuda, most):
    """More entries than a CTA has threads, of many lengths, some of them empty,
    through both kernels."""
    new = [(0, 1, most, 1, (i * 7) % most + 1)[i % 5] for i in range(601)]
    kv = [n + (i * 13) % 90 for i, n in enumerate(new)]
    _run_attn(64, 1, 2, 16, "int8", "f16", new, kv, max_seq=144)


@pytest.mark.parametrize("most", [1, 40])
def test_write_many_entries(cuda, most):
    n, hd, B = 601, 64, 16
    new = [(0, 1, most, 1, (i * 7) % most + 1)[i % 5] for i in range(n)]
    at = [(i * 13) % 90 for i in range(n)]
    cache = spb200.Q8Cache(hd, 1, 1, 144, n_seqs=n, fmt="e4m3", block_tokens=B)
    want = _fill(cache, 7)
    g = torch.Generator().manual_seed(11)
    x = [torch.randn(sum(new), 1, hd, generator=g) * s for s in (3.0, 0.4)]
    cache.write_kv_tokens(0, _batch(new, [a + m for a, m in zip(at, new)]), x[0].cuda(), x[1].cuda())
    assert cache.status() == 0
    for which in (0, 1):
        codes, scales = want[2 * which], want[2 * which + 1]
        row = 0
        for i, (s, m) in enumerate(zip(at, new)):
            R.write(codes[0, i, 0], scales[0, i, 0], x[which][row:row + m, 0], s, B, "e4m3")
            row += m
        assert torch.equal(cache.scales(which).cpu(), scales)
        assert torch.equal(cache.slab(which).view(torch.uint8).cpu(), codes)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new,kv", [(1, 700), (3, 90), (100, 700)])
def test_attn_nan_queries_stay_in_their_rows(cuda, fmt, new, kv):
    """A query row with a NaN has NaN for its output and lse; the others are as they should be."""
    hd, G = 128, 4
    cache = spb200.Q8Cache(hd, 1, 1, kv, fmt=fmt, block_tokens=64)
    fills = _fill(cache, 17)
    q = torch.randn(new, G, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).half()
    q[new // 2, 1, 77] = float("nan")
    out, lse = torch.empty_like(q), torch.empty(new, G, device="cuda")
    cache.attn(0, _batch([new], [kv]), q, out=out, lse=lse, logit_scale=0.1)
    assert cache.status() == 0
    assert torch.isnan(out[new // 2, 1]).all() and torch.isnan(lse[new // 2, 1])
    for head in (0, 2, 3):
        _check_attn(cache, fills, 0, q[:, head:head + 1], [new], [kv], None, out[:, head:head + 1], lse[:, head:head + 1],
                    0.1, True, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_example_runs(cuda, fmt):
    """The example: rotation, write, attention over prompts and a graph of single tokens."""
    import importlib.util
    from pathlib import Path
    at = Path(__file__).resolve().parent.parent / "shannon-prime-llama_b200" / "examples" / "q8_layers.py"
    spec = importlib.util.spec_from_file_location("q8_layers", at)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    # the output's own rounding (2^-11) and the weights' (2^-11)
    assert mod.main(["--layers", "2", "--steps", "5", "--fmt", fmt]) <= 2.0 ** -10
