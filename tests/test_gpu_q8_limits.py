"""The 8-bit tier on the GPU at the ends of what it accepts.  Bounds are those
of test_gpu_q8.py."""
import numpy as np
import pytest
import torch

import q8_ref as R
import spb200
from test_gpu_q8 import _batch, _check_attn, _fill, _run_attn

pytestmark = pytest.mark.gpu


# ------------------------------------------- logits that rise late and far --

@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fmt,dtype", [("int8", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [2, 40])
@pytest.mark.parametrize("zeros", [False, True])
def test_attn_one_key_far_above(cuda, hd, fmt, dtype, causal, new, zeros):
    """Ordinary logits, then one key 2^100 to 2^500 times the others' weight, at
    each position mod 32 (a sequence for each) past the first tiles; `zeros`: after
    values whose blocks have the smallest scale, as a write of zeros leaves them."""
    H, G, B, n, seqs = 1, 4, 64, 600, 32
    cache = spb200.Q8Cache(hd, 1, H, n, n_seqs=seqs, fmt=fmt, block_tokens=B)
    kc, ks, vc, vs = _fill(cache, 31)
    g = torch.Generator().manual_seed(8)
    u = torch.randint(0, 2, (hd,), generator=g).float() * 2 - 1
    kc.copy_(R.code(torch.randn(kc.shape, generator=g) * 2.5, fmt).view(kc.shape))
    ks.fill_(2.0 ** -7)
    for i in range(seqs):
        kc[0, i, 0, 256 + 32 * (i % 8) + i] = R.code(112.0 * u, fmt)
    if zeros:
        vc[:, :, :, :256] = 0
        vs[:, :, :, :256 // B] = 2.0 ** -40
    for which, c, s in ((0, kc, ks), (1, vc, vs)):
        cache.slab(which).view(torch.uint8).copy_(c)
        cache.scales(which).copy_(s)
    q = u + 0.25 * torch.randn(seqs * new, G, hd, generator=g)
    q = q.to(R.DTYPES[dtype]).cuda()
    out, lse = torch.empty_like(q), torch.empty(seqs * new, G, device="cuda")
    b = _batch([new] * seqs, [n] * seqs)
    for rise in (100, 130, 200, 256, 300, 500):
        scale = rise * np.log(2.0) / (112.0 * hd / 128)
        cache.attn(0, b, q, out=out, lse=lse, logit_scale=scale, causal=causal)
        assert cache.status() == 0
        _check_attn(cache, (kc, ks, vc, vs), 0, q, [new] * seqs, [n] * seqs, None, out, lse, scale, causal, 0)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 100])
def test_attn_scales_far_apart_other_dims(cuda, hd, fmt, new):
    """Blocks of V whose scales span 2^-40 .. 2^12, one of zeros: every weight counts in the sum."""
    B, n = 16, 160
    cache = spb200.Q8Cache(hd, 1, 1, n, fmt=fmt, block_tokens=B)
    fills = _fill(cache, 5)
    fills[1][0, 0, 0, :10] = 0.02
    fills[3][0, 0, 0, :10] = torch.tensor([2.0 ** -12, 0.03, 0.02, 0.05, 0.01, 2.0 ** -40, 0.03, 0.02, 2.0 ** -20, 2.0 ** 12])
    fills[2][0, 0, 0, 5 * B:6 * B] = 0
    for c in (0, 1):
        cache.slab(c).view(torch.uint8).copy_(fills[2 * c])
        cache.scales(c).copy_(fills[2 * c + 1])
    for end in (B, 5 * B + 3, 6 * B, 9 * B, n):
        for scale in (0.0, 0.05, 2.0):
            m = min(new, end)
            q = torch.randn(m, 4, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(end)).half()
            out, lse = torch.empty_like(q), torch.empty(m, 4, device="cuda")
            cache.attn(0, _batch([m], [end]), q, out=out, lse=lse, logit_scale=scale)
            _check_attn(cache, fills, 0, q, [m], [end], None, out, lse, scale, True, 0)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("new", [1, 100])
def test_attn_large_and_small_queries_other_dims(cuda, hd, new):
    """bf16 queries far outside fp16's range, rows of zeros, logits far apart along the sequence."""
    n = 700
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
        _check_attn(cache, fills, 0, q[:, head:head + 1], [new], [n], None, out[:, head:head + 1], lse[:, head:head + 1],
                    scale, True, 0)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("new,kv", [(3, 90), (100, 700)])
def test_attn_nan_queries_other_dims(cuda, hd, new, kv):
    """A query row with a NaN has NaN for its output and lse; the others are as they should be."""
    cache = spb200.Q8Cache(hd, 1, 1, kv, fmt="e4m3", block_tokens=64)
    fills = _fill(cache, 17)
    q = torch.randn(new, 4, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).half()
    q[new // 2, 1, 33] = float("nan")
    out, lse = torch.empty_like(q), torch.empty(new, 4, device="cuda")
    cache.attn(0, _batch([new], [kv]), q, out=out, lse=lse, logit_scale=0.1)
    assert cache.status() == 0
    assert torch.isnan(out[new // 2, 1]).all() and torch.isnan(lse[new // 2, 1])
    for head in (0, 2, 3):
        _check_attn(cache, fills, 0, q[:, head:head + 1], [new], [kv], None, out[:, head:head + 1], lse[:, head:head + 1],
                    0.1, True, 0)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fmt,dtype", [("int8", "f16"), ("e4m3", "bf16")])
def test_attn_maximum_rises_inside_a_tile(cuda, hd, fmt, dtype):
    """A key 2^9 to 2^11.5 times the others' weight, then, up to 63 positions on, one that
    takes nearly all of it and has no value: what the first one leaves in the output
    is its weight rounded at most twice to fp16 (2^-11 of it, or 2^-25 of the largest)."""
    seqs, H, G, B, n, new = 32, 8, 4, 64, 600, 40       # more tiles than CTAs by far: runs of many tiles
    cache = spb200.Q8Cache(hd, 1, H, n, n_seqs=seqs, fmt=fmt, block_tokens=B)
    g = torch.Generator().manual_seed(12)
    u = torch.randint(0, 2, (hd,), generator=g).float() * 2 - 1
    kc, vc = torch.zeros(seqs, H, cache.max_seq_len, hd), torch.zeros(seqs, H, cache.max_seq_len, hd)
    for i in range(seqs):
        first = 256 + (5 * i) % 32
        kc[i, :, first], kc[i, :, 256 + 32 + (3 * i) % 32] = 64.0 * u, 112.0 * u
        vc[i, :, first] = torch.randint(1, 8, (H, hd), generator=g).float() * 16
    for which, c, s in ((0, kc, 2.0 ** -7), (1, vc, 2.0 ** -5)):
        cache.slab(which).view(torch.uint8).copy_(R.code(c, fmt).view(1, *c.shape))
        cache.scales(which).fill_(s)
    q = (u + 0.25 * torch.randn(seqs * new, H * G, hd, generator=g)).to(R.DTYPES[dtype]).cuda()
    out, lse = torch.empty_like(q), torch.empty(seqs * new, H * G, device="cuda")
    qd = q.double().view(seqs, new, H, G, hd)
    raw = torch.einsum("stkgd,sknd->stkgn", qd, kc[:, :, :n].double().cuda() * 2.0 ** -7)
    seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - new, n, device="cuda")[:, None]
    for rise in (9.0, 10.0, 10.7, 11.5):
        scale = rise * np.log(2.0) / (64.0 * hd / 128)
        cache.attn(0, _batch([new] * seqs, [n] * seqs), q, out=out, lse=lse, logit_scale=scale)
        assert cache.status() == 0
        z = torch.where(seen[None, :, None, None], raw * scale, -torch.inf)
        want = torch.einsum("stkgn,sknd->stkgd", torch.softmax(z, -1), vc[:, :, :n].double().cuda() * 2.0 ** -5).reshape(out.shape)
        size = (qd.abs().sum(-1).max() * 112 * 2.0 ** -7 * scale).item()
        tol = (R.EPS[dtype] + 2 * 2.0 ** -11 + 2.0 ** -18 * (1 + size)) * want.abs() + 2 * 2.0 ** -25 * 7 * 16 * 2.0 ** -5
        off = (out.double() - want).abs()
        assert (off <= tol).all(), (rise, (off / tol).max().item())
        assert ((lse.double() - torch.logsumexp(z, -1).reshape(lse.shape)).abs() <= 2.0 ** -18 * (1 + size)).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fmt,dtype", [("int8", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("new", [2, 40])
def test_attn_logits_past_32_bit_resolution(cuda, hd, fmt, dtype, new):
    """Logits of 1e7 to 1e30, whose neighbours are whole numbers of powers of two apart: the key
    that is far above the others, at each position mod 32, is the output."""
    H, G, B, n, seqs = 1, 4, 64, 600, 32
    cache = spb200.Q8Cache(hd, 1, H, n, n_seqs=seqs, fmt=fmt, block_tokens=B)
    kc, ks, vc, vs = _fill(cache, 31)
    g = torch.Generator().manual_seed(8)
    u = torch.randint(0, 2, (hd,), generator=g).float() * 2 - 1
    kc.copy_(R.code(torch.randn(kc.shape, generator=g) * 2.5, fmt).view(kc.shape))
    ks.fill_(2.0 ** -7)
    at = [32 * (5 * i % 17) + i for i in range(seqs)]
    for i, j in enumerate(at):
        kc[0, i, 0, j] = R.code(112.0 * u, fmt)
    for which, c, s in ((0, kc, ks), (1, vc, vs)):
        cache.slab(which).view(torch.uint8).copy_(c)
        cache.scales(which).copy_(s)
    q = u + 0.25 * torch.randn(seqs * new, G, hd, generator=g)
    q = q.to(R.DTYPES[dtype])
    out, lse = torch.empty(seqs * new, G, hd, device="cuda", dtype=q.dtype), torch.empty(seqs * new, G, device="cuda")
    for causal in (True, False):
        for size in (1e7, 1e8, 1e9, 1e12, 1e30):
            scale = size / (112.0 * hd / 128)
            cache.attn(0, _batch([new] * seqs, [n] * seqs), q.cuda(), out=out, lse=lse, logit_scale=scale, causal=causal)
            assert cache.status() == 0
            for i, j in enumerate(at):
                rows = slice(i * new, i * new + new)
                want = R.values(vc[0, i, 0, j], fmt).double() * vs[0, i, 0, j // B].double()
                off = (out[rows].double().cpu() - want).abs()
                # the output's rounding, the weight's, and the sum's reciprocal
                assert (off <= (R.EPS[dtype] + 2.0 ** -11 + 2.0 ** -20) * want.abs() + 2.0 ** -25).all(), (size, i)
                z = q[rows].double() @ (R.values(kc[0, i, 0, j], fmt).double() * 2.0 ** -7) * scale
                # the scale's, the factors' and the sum's roundings
                assert ((lse[rows].double().cpu() - z).abs() <= 2.0 ** -19 * z.abs()).all(), (size, i)


# -------------------------------------------------------- windows and tokens --

@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 257, 256])
@pytest.mark.parametrize("new,kv", [([5, 2, 1], [2, 2, 0]), ([90, 3, 60], [20, 250, 256])])
def test_attn_windows_past_the_cache(cuda, hd, window, new, kv):
    """The widest windows, with tokens before the first position."""
    _run_attn(hd, 1, 4, 16, "int8", "f16", new, kv, window=window, max_seq=256)


def test_attn_rows_past_32_bits_are_refused(cuda):
    """Entries that may have 2^31 rows; a loose bound on an entry's tokens is no such claim."""
    cache = spb200.Q8Cache(64, 1, 1, 256)
    q = torch.randn(4, 128, 64, device="cuda", dtype=torch.float16)
    p, call = q.data_ptr(), spb200.lib().sp_cuda_q8_attn
    for tokens, most, rc in ((2 ** 30, 2 ** 30, spb200.SP_ERR_ARG), (2 ** 24, 2 ** 31 - 1, spb200.SP_ERR_ARG), (4, 2 ** 31 - 1, 0)):
        b = spb200.Q8Batch(torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.tensor([9], dtype=torch.int32, device="cuda"),
                           tokens, most, 256)
        assert call(cache._ref, 0, b.ref, p, 0, 128, 1, 1.0, 1, 0, p, 0, None, None) == rc, (tokens, most)
    assert cache.status() == 0


# ------------------------------------------------------------------- streams --

@pytest.mark.parametrize("which", ["rope", "attn"])
def test_new_outputs_are_memory_of_their_stream(cuda, which):
    """An output that a call allocates is written on the call's stream: it is neither
    memory that the current stream may still be using nor given out again while
    either stream is busy with it."""
    T, hd = 37, 64
    x = torch.randn(T, 3, hd, device="cuda", dtype=torch.float16)
    pos = torch.zeros(1, T, dtype=torch.int32, device="cuda")
    rope, cache = spb200.RopeAxes(hd, [32]), spb200.Q8Cache(hd, 1, 3, 128)
    batch = _batch([T], [T])

    def call(**kw):
        return rope.apply(pos, x, None, **kw)[0] if which == "rope" else cache.attn(0, batch, x, **kw)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for stream, current in ((side, torch.cuda.default_stream()), (side, other), (None, other)):
        with torch.cuda.stream(current):
            old = torch.empty_like(x)
            at = old.data_ptr()
            del old
            y = call(stream=stream)                 # not what the current stream has just given back
            assert y.data_ptr() != at
            at = y.data_ptr()
            del y
            z = torch.empty_like(x)                 # nor is it the current stream's to give out
            assert z.data_ptr() != at
            y = call(stream=stream)
            current.wait_stream(stream or torch.cuda.default_stream())
            at = y.data_ptr()
            torch.cuda._sleep(20000000)             # about 10 ms
            w = y.clone()
            del y
            y = call(stream=stream)                 # the copy of the last one has not run yet
            assert y.data_ptr() != at
            torch.cuda.synchronize()
            assert torch.equal(w, y)


# ------------------------------------------------------------------ gradients --

@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope_autograd(cuda, pairing, inverse):
    """The gradient of q and k (slices of one projection) against autograd through the
    formula in 64 bits, and against differences of the loss."""
    T, hq, hk, hd, rot = 23, 5, 2, 64, 48
    plan = spb200.RopeAxes(hd, [8, 8, 8], pairing=pairing, rot_dim=rot)
    g = torch.Generator(device="cuda").manual_seed(6)
    pos = torch.randint(0, 9000, (3, T), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn(T, hq + hk, hd, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(T, hq + hk, hd, generator=g, device="cuda")

    def loss(z):
        q, k = plan.apply(pos, z[:, :hq], z[:, hq:], inverse=inverse)
        return (torch.cat([q, k], 1).double() * w.double()).sum()
    grad, = torch.autograd.grad(loss(x), x)
    # the formula, its cosines as constants
    f = torch.tensor([float(np.float32(10000.0 ** (-2.0 * i / rot))) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    axis = torch.arange(3, device="cuda").repeat_interleave(8)
    a = (pos[axis].double().t() * f)[:, None] * (-1.0 if inverse else 1.0)
    z = x.detach().double().requires_grad_()
    u, v = (z[..., 0:rot:2], z[..., 1:rot:2]) if pairing == "adjacent" else (z[..., :rot // 2], z[..., rot // 2:rot])
    lo, hi = u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()
    y = torch.stack([lo, hi], -1).flatten(-2) if pairing == "adjacent" else torch.cat([lo, hi], -1)
    want, = torch.autograd.grad((torch.cat([y, z[..., rot:]], -1) * w.double()).sum(), z)
    # each element is a rotation of a pair of w: its rounding and the cosines' (4e-7 of the pair's length)
    assert ((grad.double() - want).abs() <= 6e-7 * (w.double().abs().amax() * 2 ** 0.5)).all()
    d = torch.randn(x.shape, generator=g, device="cuda")
    step = 2.0 ** -3            # the loss is linear: a large step only rounds less
    with torch.no_grad():
        numeric = ((loss(x + step * d) - loss(x - step * d)) / (2 * step)).item()
    size = w.double().norm().item() * (x.detach().double().norm().item() / step + d.double().norm().item())
    assert abs(numeric - (grad.double() * d.double()).sum().item()) <= 4e-7 * size


def test_rope_autograd_shapes_and_streams(cuda):
    """One half alone, a half without a gradient, a gradient expanded from one number,
    a second derivative, another stream, and nothing kept without gradients."""
    T, hd = 9, 64
    plan = spb200.RopeAxes(hd, [32])
    pos = torch.arange(T, dtype=torch.int32, device="cuda")[None]
    x = torch.randn(T, 3, hd, device="cuda", requires_grad=True)
    k = torch.randn(T, 1, hd, device="cuda")
    back = plan.apply(pos, torch.ones_like(k), None, inverse=True)[0].expand(T, 3, hd)
    for q, kk in ((x, None), (None, x), (x, k), (k, x)):
        y = plan.apply(pos, q, kk)
        mine = y[0] if q is x else y[1]
        assert mine.requires_grad and not any(o.requires_grad for o in y if o is not None and o is not mine)
        grad, = torch.autograd.grad(mine.sum(), x)
        assert torch.equal(grad, back)
    y = plan.apply(pos, x, None)[0]
    grad, = torch.autograd.grad(y.square().sum(), x, create_graph=True)      # 2 x, whose own derivative is 2
    again, = torch.autograd.grad(grad.sum(), x)
    assert ((again - 2.0).abs() <= 2e-6 * 4).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grad, = torch.autograd.grad(plan.apply(pos, x, None, stream=side)[0].sum(), x)
    side.synchronize()
    assert torch.equal(grad, back)
    with torch.no_grad():
        assert not plan.apply(pos, x, None)[0].requires_grad
    assert not plan.apply(pos, x.detach(), None)[0].requires_grad
