"""What the 8-bit tier's binding refuses before anything is launched.  No GPU:
tensors in main memory stand in for tensors of a card."""
import pytest
import torch


class OnCard:
    """A tensor that says it lies on card 0; nothing is launched on it."""

    is_cuda = True

    def __init__(self, t, device=0):
        self.t, self.device = t, torch.device("cuda", device)

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.device.index


def _cache(hd=64, heads=2):
    """A Q8Cache that has its shape and no memory."""
    import spb200
    c = object.__new__(spb200.Q8Cache)
    c.qc = spb200.SpQ8Cache()
    c.head_dim, c.n_heads_kv, c.fmt, c.stream, c.device = hd, heads, "int8", None, 0
    c._ref = None

    def launched(*a):
        raise AssertionError("the call reached the library")
    c._write = c._read = c._attn = launched
    return c


def _batch(n_tokens):
    import spb200
    b = object.__new__(spb200.Q8Batch)
    b._keep, b.n_tokens, b.ref, b.device = (), n_tokens, None, 0
    return b


@pytest.fixture(autouse=True)
def current_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def _rope():
    import spb200
    r = spb200.RopeAxes(64, [32])

    def launched(*a):
        raise AssertionError("the call reached the library")
    r._call = launched
    return r, OnCard(torch.zeros(1, 5, dtype=torch.int32))


def _one(heads=2, dtype=torch.float16):
    """Five tokens that are one token's memory."""
    return OnCard(torch.zeros(1, heads, 64, dtype=dtype).expand(5, heads, 64))


def _all(heads=2, dtype=torch.float16):
    return OnCard(torch.zeros(5, heads, 64, dtype=dtype))


def test_tokens_that_share_memory_are_refused(built_lib):
    """A tensor expanded over its tokens has less memory than its shape says."""
    rope, pos = _rope()
    cache, batch = _cache(), _batch(5)
    overlapping = OnCard(torch.zeros(600, dtype=torch.float16).as_strided((5, 2, 64), (64, 64, 1)))
    for bad in (_one(), overlapping):
        for call in (lambda: rope.apply(pos, bad, None, q_out=_all()), lambda: rope.apply(pos, None, bad, k_out=_all()),
                     lambda: rope.apply(pos, _all(), None, q_out=bad), lambda: rope.apply(pos, None, _all(), k_out=bad),
                     lambda: cache.write_kv_tokens(0, batch, bad, None), lambda: cache.write_kv_tokens(0, batch, None, bad),
                     lambda: cache.write_kv_tokens(0, batch, bad, bad), lambda: cache.attn(0, batch, bad, out=_all()),
                     lambda: cache.attn(0, batch, _all(), out=bad), lambda: cache.read_kv_tokens(0, 0, 0, 0, bad)):
            with pytest.raises(ValueError):
                call()


def test_one_token_may_be_expanded(built_lib):
    """One token has all the memory it needs, whatever its stride."""
    import spb200.q8 as q8
    assert q8._rows(OnCard(torch.zeros(1, 1, 64).expand(1, 1, 64)), 1, 64, "x") == 0
    fused = OnCard(torch.zeros(5, 6, 64)[:, 2:4])
    assert q8._rows(fused, 2, 64, "x") == 6 * 64


def test_runs_of_more_tiles_than_32_bits_count(tmp_path):
    """The many-row attention's cut into runs (tests/c/q8_runs_check.cpp)."""
    import subprocess

    from conftest import PKG, ROOT, load_build_module
    b = load_build_module()
    exe = tmp_path / "q8_runs_check"
    subprocess.run([b.HOST_CXX, "-O1", "-std=c++17", "-Wall", "-Werror", f"-I{PKG / 'csrc'}",
                    str(ROOT / "tests" / "c" / "q8_runs_check.cpp"), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "ok\n"


def test_tensors_of_another_device_are_refused(built_lib):
    """Pointers of another card's memory are none of the kernels'."""
    import spb200
    rope, pos = _rope()
    cache, batch = _cache(), _batch(5)
    far, here = OnCard(_all().t, device=1), _all()
    lse = OnCard(torch.zeros(5, 2), device=1)
    other = _batch(5)
    other.device = 1
    out = OnCard(torch.zeros(5, 2, 64, dtype=torch.float16), device=1)
    for call in (lambda: rope.apply(pos, far, None, q_out=here), lambda: rope.apply(pos, here, None, q_out=far),
                 lambda: rope.apply(pos, None, far, k_out=here), lambda: rope.apply(pos, None, here, k_out=far),
                 lambda: rope.apply(OnCard(pos.t, device=1), far, None, q_out=far),
                 lambda: cache.write_kv_tokens(0, batch, far, far), lambda: cache.write_kv_tokens(0, batch, here, far),
                 lambda: cache.write_kv_tokens(0, batch, None, far), lambda: cache.write_kv_tokens(0, other, here, here),
                 lambda: cache.read_kv_tokens(0, 0, 0, 0, out), lambda: cache.attn(0, batch, far, out=here),
                 lambda: cache.attn(0, batch, here, out=far), lambda: cache.attn(0, other, here, out=here),
                 lambda: cache.attn(0, batch, here, out=here, lse=lse)):
        with pytest.raises(ValueError, match="device"):
            call()
    cu, kv = OnCard(torch.zeros(3, dtype=torch.int32)), OnCard(torch.zeros(2, dtype=torch.int32), device=1)
    with pytest.raises(ValueError, match="device"):
        spb200.Q8Batch(cu, kv, 4, 4, 4)
    with pytest.raises(AssertionError):          # the same on the right card reaches the library
        rope.apply(pos, here, here, q_out=here, k_out=here)
    with pytest.raises(AssertionError):
        cache.attn(0, batch, here, out=here, lse=OnCard(lse.t))


def test_rotation_that_would_lose_a_gradient_is_refused(built_lib):
    """With gradients wanted an output cannot be given; without them it can."""
    rope, pos = _rope()
    x = OnCard(torch.zeros(5, 2, 64, requires_grad=True))
    out = OnCard(torch.zeros(5, 2, 64))
    for call in (lambda: rope.apply(pos, x, None, q_out=out), lambda: rope.apply(pos, None, x, k_out=out),
                 lambda: rope.apply(pos, out, x, q_out=out, k_out=out), lambda: rope.apply(pos, x, None, q_out=x)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(AssertionError, match="reached"):
            call()


def test_refused_plan_is_no_plan(built_lib):
    """A plan whose frequencies were refused half-way, after one that was good."""
    import ctypes as C

    import spb200
    L, plan = spb200.lib(), spb200.SpRopeAxes()

    def init(factors):
        return L.sp_rope_axes_init(C.byref(plan), 64, 64, 0, 1, (C.c_int * 1)(32), 0, 1e4, (C.c_float * 32)(*factors))
    for bad in ([1.0] * 31 + [0.0], [1.0] * 20 + [1e-45] * 12, [float("inf")] + [1.0] * 31):
        assert init([1.0] * 32) == 0 and plan.head_dim == 64
        assert init(bad) == spb200.SP_ERR_ARG
        assert bytes(plan) == bytes(C.sizeof(plan))
        assert L.sp_cuda_rope_axes(C.byref(plan), None, 0, None, 0, 0, None, 0, None, 0, 0, None, 0, 1, 0, None) == spb200.SP_ERR_ARG
