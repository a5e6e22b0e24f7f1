"""The 8-bit K/V cache without a GPU: the 64-bit definition against torch's own e4m3, and what the entry points refuse."""
import ctypes as C

import pytest
import torch

import kv8_reference as R

OK, ERR_SHAPE, ERR_ALIGN = 0, -1, -2
P = C.c_void_p
FAKE = P(0x10000)            # 16-byte aligned, non-null, never dereferenced


def test_reference_grid_is_e4m3():
    codes = torch.arange(256, dtype=torch.uint8)
    v, t = R.values(codes), codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.isnan(v), torch.isnan(t)) and torch.equal(v[~torch.isnan(v)], t[~torch.isnan(t)])
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.05, 0.05, 5001), R.GRID.float(), ((R.GRID[1:] + R.GRID[:-1]) / 2).float()])
    assert torch.equal(R.to_grid(x.double()), x.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("a,s", [(448.0, 0), (449.0, 1), (1.75, -8), (1.7500001, -7), (1.0, -8), (0.0, -126), (3.0e38, 120), (1e-44, -126)])
def test_reference_scale(a, s):
    x = torch.tensor([[a, -a / 2, float("inf"), float("nan")]], dtype=torch.float32).double()
    assert float(R.shift(x, (1,))) == s


@pytest.fixture(scope="module")
def L():
    from libra_amd import _lib
    return _lib.lib()


def test_c_entry_points_refuse(L):
    def fill(**kw):
        a = dict(dict(ks=FAKE, lk=256, kc=FAKE, lc=256, vs=FAKE, lv=256, vc=FAKE, lw=256, codes=FAKE, scales=FAKE, B=2, S=8, H=2, cap=32,
                      block=16, start=None, st=None), **kw)
        return L.libra_kv8_fill(*a.values())
    assert fill(S=0) == OK and fill(B=0) == OK
    for bad in (dict(S=33), dict(S=-1), dict(B=-1), dict(H=0), dict(cap=40), dict(block=3), dict(block=0), dict(block=128, cap=128), dict(lk=128),
                dict(B=70000)):
        assert fill(**bad) == ERR_SHAPE, bad
    for bad in (dict(ks=None), dict(vc=P(0x10008)), dict(codes=P(0x10004)), dict(scales=None), dict(lc=260)):
        assert fill(**bad) == ERR_ALIGN, bad

    def append(**kw):
        a = dict(dict(ks=FAKE, lk=256, kc=FAKE, lc=256, vs=FAKE, lv=256, vc=FAKE, lw=256, codes=FAKE, scales=FAKE, B=2, H=2, cap=32, block=16,
                      slot=FAKE, st=None), **kw)
        return L.libra_kv8_append(*a.values())
    assert append(B=0) == OK and append(slot=None) == ERR_ALIGN and append(cap=33) == ERR_SHAPE and append(lw=255) == ERR_SHAPE

    def read(**kw):
        a = dict(dict(codes=FAKE, scales=FAKE, out=FAKE, ldo=256, bs=4096, B=2, H=2, cap=32, block=16, first=0, n=8, st=None), **kw)
        return L.libra_kv8_read(*a.values())
    assert read(n=0) == OK and read(first=25) == ERR_SHAPE and read(first=-1) == ERR_SHAPE and read(ldo=128) == ERR_SHAPE
    assert read(out=None) == ERR_ALIGN and read(ldo=257) == ERR_ALIGN

    ws = L.libra_bridge_attn_decode8_workspace_bytes(2, 2, 2048)

    def attn(**kw):
        a = dict(dict(q=FAKE, ldq=256, codes=FAKE, scales=FAKE, kf=FAKE, fs=2048, qf=FAKE, ln=FAKE, start=None, out=FAKE, ldo=256, B=2, H=2,
                      cap=2048, block=16, scale=0.1, ws=FAKE, wsb=ws, st=None), **kw)
        return L.libra_bridge_attn_decode8(*a.values())
    assert attn(B=0) == OK
    for bad in (dict(ldq=128), dict(ldo=128), dict(fs=2047), dict(cap=2047), dict(block=5), dict(H=-1)):
        assert attn(**bad) == ERR_SHAPE, bad
    for bad in (dict(q=None), dict(q=P(0x10008)), dict(kf=None), dict(qf=None), dict(ln=None), dict(out=None), dict(ws=P(0x10004)), dict(wsb=ws - 1),
                dict(ldq=260)):
        assert attn(**bad) == ERR_ALIGN, bad


    def rope(**kw):
        a = dict(dict(qkv=FAKE, ld=768, tb=FAKE, ldt=64, kl=FAKE, kv=FAKE, vl=FAKE, vv=FAKE, flag=FAKE, cos=FAKE, sin=FAKE, mp=64, B=2, pos=FAKE, ps=1,
                      H=2, codes=FAKE, scales=FAKE, cap=32, block=16, slot=FAKE, st=None), **kw)
        return L.libra_rope_bridge_pos_append8(*a.values())
    assert rope(B=0) == OK
    for bad in (dict(ld=512), dict(ldt=8), dict(ps=3), dict(cap=33), dict(block=6), dict(mp=0), dict(B=-2)):
        assert rope(**bad) == ERR_SHAPE, bad
    for bad in (dict(pos=None), dict(slot=None), dict(codes=None), dict(qkv=P(0x10008)), dict(cos=None), dict(ld=769)):
        assert rope(**bad) == ERR_ALIGN, bad


def test_log_probability_entry_points_refuse(L):
    def fwd(**kw):
        a = dict(dict(z=FAKE, ldz=100, rows=4, V=100, f32=0, t=FAKE, T=2, sub=0, lp=FAKE, st=FAKE, top=3, ids=FAKE, tlp=FAKE, s=None), **kw)
        return L.libra_token_logprobs(*a.values())
    assert fwd(rows=0) == OK
    for bad in (dict(V=0), dict(ldz=99), dict(T=65), dict(T=-1), dict(top=65), dict(top=101, V=100), dict(top=-1), dict(rows=-1)):
        assert fwd(**bad) == ERR_SHAPE, bad
    for bad in (dict(z=None), dict(z=P(0x10001)), dict(z=P(0x10002), f32=1), dict(t=None), dict(lp=None), dict(st=None), dict(ids=None), dict(tlp=None)):
        assert fwd(**bad) == ERR_ALIGN, bad

    def bwd(**kw):
        a = dict(dict(z=FAKE, ldz=100, rows=4, V=100, f32=0, t=FAKE, T=2, sub=0, st=FAKE, g=FAKE, ge=None, dz=FAKE, lddz=100, s=None), **kw)
        return L.libra_token_logprobs_bwd(*a.values())
    assert bwd(rows=0) == OK
    assert bwd(lddz=99) == ERR_SHAPE and bwd(V=0) == ERR_SHAPE
    for bad in (dict(dz=None), dict(dz=P(0x10001)), dict(st=None), dict(t=None), dict(z=None)):
        assert bwd(**bad) == ERR_ALIGN, bad


def test_cache_container_on_the_host():
    """KVCache dtype "fp8": buffers, capacity rounding, batch re-gather - no kernel involved."""
    from libra_amd import decoder_engine as DE
    c = DE.KVCache(3, 2, 21, 512, "cpu", dtype="fp8", block=16)
    assert len(c.layers) == 3 and tuple(c.layers[0][0].shape) == (4, 2, 4, 32, 128) and tuple(c.flag.shape) == (2, 32) and c.capacity == 21
    for i, (codes, scales) in enumerate(c.layers):
        codes.copy_(torch.arange(2, dtype=torch.uint8)[None, :, None, None, None].expand_as(codes) + i)
    c.start, c.graphs = torch.tensor([3, 5], dtype=torch.int32), {"x": 1}
    c.reorder(torch.tensor([1, 1, 0]))
    assert c.B == 3 and c.start.tolist() == [5, 5, 3] and not c.graphs
    assert [int(c.layers[2][0][0, b, 0, 0, 0]) for b in range(3)] == [3, 3, 2] and tuple(c.layers[0][1].shape) == (4, 3, 4, 2)
    assert c.nbytes() * 2 < DE.KVCache(3, 3, 32, 512, "cpu").nbytes() * 1.01
    with pytest.raises(ValueError):
        DE.KVCache(1, 1, 8, 128, "cpu", dtype="int8")
    with pytest.raises(ValueError):
        c.rows(0, 0, 1)


def test_host_wrappers_refuse_without_a_gpu():
    """Shapes, types and devices are judged before anything is launched."""
    from libra_amd import kernels as K
    codes, scales = K.kv8_alloc(2, 20, 3, "cpu", 16)
    assert tuple(codes.shape) == (4, 2, 3, 32, 128) and tuple(scales.shape) == (4, 2, 3, 2)         # capacity rounded up
    for block in (0, 3, 128, -1):
        with pytest.raises(ValueError):
            K.kv8_alloc(1, 8, 1, "cpu", block)
    assert K._kv8_geometry(codes, scales, "t") == (2, 3, 32, 16)
    for c, s in ((codes.view(torch.int8), scales), (codes[:, :, :, :31], scales), (codes[..., :64], scales), (codes, scales[:, :1]),
                 (codes, scales.transpose(0, 1)), (codes[0], scales), (codes, scales[..., :0])):
        with pytest.raises(ValueError):
            K._kv8_geometry(c, s, "t")
    rows = [torch.zeros(2, 384, dtype=torch.bfloat16) for _ in range(4)]
    with pytest.raises(ValueError):
        K.kv8_append(rows, codes, scales, torch.zeros(1, dtype=torch.int64))                        # host tensors
    with pytest.raises(ValueError):
        K.kv8_append(rows[:3], codes, scales, torch.zeros(1, dtype=torch.int64))


# ---- operands of the rotary + bridge launches: tensors of a device that is not there, a library that only records --------------------
ROPE = ("rope_bridge", "rope_bridge_pos", "rope_bridge_pos_append8")


def _rope_call(monkeypatch, name, N=2, H=2, **change):
    """The entry point on fake device tensors -> the name of the library call it made."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from libra_amd import kernels as K
    made = []

    class Library:
        def __getattr__(self, fn):
            return lambda *a: made.append(fn) or 0
    monkeypatch.setattr(K._lib, "lib", Library)
    monkeypatch.setattr(K, "_stream", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    bf, D = torch.bfloat16, H * 128
    with FakeTensorMode():
        e = lambda *s, dtype=bf, device="cuda": torch.empty(*s, dtype=dtype, device=device)  # noqa: E731
        a = dict(qkv=e(N, 3 * D), tb=e(N, 64), bk_l=e(D, 8), bk_v=e(D, 8), bv_l=e(D, 8), bv_v=e(D, 8), flag=e(N, dtype=torch.uint8),
                 cos=e(64, 128), sin=e(64, 128))
        a.update({k: v(e) for k, v in change.items() if k in a})
        if name == "rope_bridge":
            K.rope_bridge(*a.values(), 1, H)
        else:
            pos = change.get("positions", lambda e: e(N, dtype=torch.int32))(e)
            if name == "rope_bridge_pos":
                K.rope_bridge_pos(*a.values(), pos, H)
            else:
                K.rope_bridge_pos_append8(*a.values(), pos, H, e(4, N, H, 32, 128, dtype=torch.uint8), e(4, N, H, 2, dtype=torch.uint8),
                                          e(1, dtype=torch.int64))
    return made[-1]


@pytest.mark.parametrize("name", ROPE)
def test_rope_operands_are_taken(monkeypatch, name):
    assert _rope_call(monkeypatch, name) == "libra_" + name
    assert _rope_call(monkeypatch, name, qkv=lambda e: e(2, 3 * 256 + 64)[:, :768], tb=lambda e: e(2, 3 * 256 + 64)[:, 768:]) == "libra_" + name


@pytest.mark.parametrize("name", ROPE)
@pytest.mark.parametrize("what,bad", [
    ("flag", lambda e: e(1, dtype=torch.uint8)), ("flag", lambda e: e(2, dtype=torch.int64)), ("flag", lambda e: e(4, dtype=torch.uint8)[::2]),
    ("flag", lambda e: e(2, dtype=torch.uint8, device="cpu")),
    ("tb", lambda e: e(2, 8)), ("tb", lambda e: e(1, 64)),
    ("bk_l", lambda e: e(128, 8)), ("bk_v", lambda e: e(256, 4)), ("bv_l", lambda e: e(256, 8, dtype=torch.float32)), ("bv_v", lambda e: e(8, 256).t()),
    ("bk_l", lambda e: e(256, 8, device="cpu")),
    ("cos", lambda e: e(64, 64)), ("sin", lambda e: e(32, 128)), ("cos", lambda e: e(64, 128, dtype=torch.float32)), ("sin", lambda e: e(64, 128, device="cpu")),
    ("sin", lambda e: e(64, 256)[:, :128]), ("qkv", lambda e: e(2, 1024)[:, :640])])
def test_rope_operands_are_refused(monkeypatch, name, what, bad):
    """What the launch would read outside of: too few flags, weights or table rows, another type, another device."""
    with pytest.raises(ValueError):
        _rope_call(monkeypatch, name, **{what: bad})


@pytest.mark.parametrize("name", ROPE[1:])
@pytest.mark.parametrize("bad", [lambda e: e(1, dtype=torch.int32), lambda e: e(2, dtype=torch.int64), lambda e: e(2, dtype=torch.int32, device="cpu")])
def test_rope_positions_are_refused(monkeypatch, name, bad):
    with pytest.raises(ValueError):
        _rope_call(monkeypatch, name, positions=bad)


def test_one_row_of_any_stride_reaches_the_library(monkeypatch):
    """A batch of one row whose stride is 1 (what a transpose leaves): the library is told the row's width instead."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from libra_amd import kernels as K
    made = {}

    class Library:
        def __getattr__(self, fn):
            return lambda *a: made.update({fn: a}) or 0
    monkeypatch.setattr(K._lib, "lib", Library)
    monkeypatch.setattr(K, "_stream", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        u8, i32 = torch.uint8, torch.int32
        row = lambda n, **kw: e(n, 1, **kw).t()  # noqa: E731
        cache = e(4, 1, 2, 32, 128, dtype=u8), e(4, 1, 2, 2, dtype=u8)
        assert row(256).stride() == (1, 1)
        K.kv8_fill([row(256)] * 4, *cache, 1)
        K.kv8_append([row(256)] * 4, *cache, e(1, dtype=torch.int64))
        K.rope_bridge_pos_append8(row(768), row(16), *[e(256, 8)] * 4, e(1, dtype=u8), e(64, 128), e(64, 128), e(1, dtype=i32), 2, *cache, e(1, dtype=torch.int64))
        K.bridge_attn_decode8(row(256), *cache, row(32, dtype=u8), e(1, dtype=u8), e(1, dtype=i32), 0.1)
    assert made["libra_kv8_fill"][1:8:2] == made["libra_kv8_append"][1:8:2] == (256,) * 4
    assert made["libra_rope_bridge_pos_append8"][1:4:2] == (768, 16)
    assert (made["libra_bridge_attn_decode8"][1], made["libra_bridge_attn_decode8"][5]) == (256, 32)
