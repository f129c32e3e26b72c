"""The native host path (host/native.cpp) of heads normed and turned, of the cache in 8 bits and of drafted trees against the methods
of kernels.py, on the CPU: a library of recorders, compiled here from the header, takes what each passes."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from adrastea_amd import (DraftTree, GpuKernels, HeadNorm, PagedBatch, PagedCache, PagedCacheU8, Rotary, RotaryAxes, TensorLayout,
                          TensorView, _ffi, kernels)
from adrastea_amd.kernels import _NATIVE_STEP_CALLS, _bind_native
from adrastea_amd.tensor import _native
from test_native_sequences import SHIM

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ABI = _ffi.lib().adr_abi_version()
STEP_SHIM = SHIM.replace("template <class... A> static int record", """
static void put(float v) { put((double)v); }
static void put(const adr_paged_cache_u8& c) {
  put(c.key), put(c.key_scale), put(c.value), put(c.value_scale), put(c.pages), put(c.kv_heads), put(c.page_size), put(c.d);
  put(c.stride_kx), put(c.stride_ky), put(c.stride_kz), put(c.stride_kp), put(c.stride_vx), put(c.stride_vy), put(c.stride_vz);
  put(c.stride_vp), put(c.stride_ksy), put(c.stride_ksz), put(c.stride_ksp), put(c.stride_vsy), put(c.stride_vsz), put(c.stride_vsp);
}
static void put(const adr_rotary_axes& r) { put(r.turns), put(r.axis), put(r.dims), put(r.layout), put((double)r.magnitude), put(r.axes); }
static void put(const adr_head_norm& n) { put(n.weight), put((double)n.eps); }
static void put(const adr_draft_tree& t) { put(t.bits), put(t.words), put(t.pitch); }
template <class... A> static int record""") + "".join(f"RECORDED({name})\n" for name in _NATIVE_STEP_CALLS)


class Recorders:
    def __init__(self, path):
        self.so = C.CDLL(path)
        self.so.taken.restype = C.c_char_p
        self.addresses = []
        for name in _NATIVE_STEP_CALLS:
            at = getattr(self.so, "at_" + name)
            at.restype = C.c_void_p
            self.addresses.append(at())
            setattr(self, name, C.CFUNCTYPE(C.c_int, *getattr(_ffi.lib(), name).argtypes)(self.addresses[-1]))

    def taken(self):
        return self.so.taken().decode()


@pytest.fixture(scope="module")
def recorders(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no C++ compiler")
    if _native is None:
        pytest.skip("the native module is not built")
    where = tmp_path_factory.mktemp("recorders")
    (where / "shim.cpp").write_text(STEP_SHIM)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"), "-o", str(where / "shim.so"),
                    str(where / "shim.cpp")], check=True)
    return Recorders(str(where / "shim.so"))


@pytest.fixture
def both(recorders, monkeypatch):
    """A call through the native path and through the general one: what each passed on (None: refused)."""
    _native.bind(ABI, *[0] * 8, lambda: -1, lambda device: 0x1001 + device)   # (tensors of the host say device -1)
    _native.bind_sequences(*[0] * 4, torch.int32)
    _native.bind_step(*recorders.addresses, RotaryAxes, HeadNorm, PagedCacheU8, DraftTree)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(kernels, "_current_stream", lambda: 0x1000)
    k = GpuKernels.__new__(GpuKernels)
    k._lib, k._workspace = recorders, None

    def call(name, *args):
        rc = getattr(_native, name)(*args)
        native = recorders.taken()
        assert rc in (0, None) and (rc == 0) == (native != "")
        monkeypatch.setattr(kernels, "_native", None)
        try:
            getattr(k, name)(*args)
            general = recorders.taken()
        except (AssertionError, AttributeError, TypeError, ValueError, C.ArgumentError):
            general = None
        finally:
            monkeypatch.setattr(kernels, "_native", _native)
        return native or None, general
    yield call
    _bind_native()


def half(*dims):
    return torch.zeros(*dims, dtype=torch.float16)


def rows(heads, n, d, packed=False):
    return TensorView.of(half(heads, n, d)) if packed else TensorView.of(half(n, heads, d)).permute([1, 0, 2])


def cache(pages=6, heads=2, size=16, d=64):
    return PagedCache(TensorView.of(half(pages, size, heads, d)).permute([0, 2, 1, 3]), TensorView.of(half(pages, heads, size, d)))


def codes(pages=6, heads=2, size=16, d=64):
    k, v = (torch.zeros(pages, heads, size, d, dtype=torch.uint8) for _ in range(2))
    return PagedCacheU8(TensorView.of(k), TensorView.of(half(pages, size, heads)).permute([0, 2, 1]),
                        TensorView(torch.zeros(k.numel() + 32, dtype=torch.uint8), TensorLayout.row_major(v.shape), 32),
                        TensorView.of(half(pages, heads, size)))


def batch(sequences=3, width=4, pitch=None, hints=(5, 40)):
    table = torch.zeros(sequences, pitch or width, dtype=torch.int32)[:, :width]
    return PagedBatch(torch.zeros(sequences + 1, dtype=torch.int32), torch.zeros(sequences, dtype=torch.int32), table, *hints)


def rotary(axes=2, dims=64, layout=1):
    return RotaryAxes(torch.zeros(dims // 2, dtype=torch.float64), torch.zeros(dims // 2, dtype=torch.int32), axes, layout, 1.25)


def positions(axes, n, pitch=0):
    return torch.zeros(axes, n + pitch, dtype=torch.int32)[:, :n]


def norm(d=64):
    return HeadNorm(half(d), 1e-5)


ONE = Rotary(torch.zeros(32, dtype=torch.float64), 0, 1.0)


def test_both_ways_pass_the_same(both):
    p1 = torch.zeros(7, dtype=torch.int32)
    for args in ((rows(4, 7, 64), rows(4, 7, 64, True), positions(2, 7), rotary(), norm()), (rows(4, 7, 64), rows(4, 7, 64), p1, ONE, None),
                 (rows(4, 7, 64), rows(4, 7, 64), positions(3, 7, 5), rotary(3), norm()), (rows(1, 7, 64), TensorView.of(half(7, 64)), None, None, norm()),
                 (rows(4, 7, 64), rows(4, 7, 64), positions(1, 7), rotary(1), None), (rows(4, 7, 64), rows(4, 7, 64), p1, rotary(1), None)):
        native, general = both("norm_rotary_f16", *args)
        assert native == general and native is not None
    k, v, q, o = rows(2, 9, 64), rows(2, 9, 64, True), rows(8, 9, 64), rows(8, 9, 64, True)
    for name, c in (("append_norm_f16", cache()), ("append_u8", codes())):
        for rest in ((rotary(), o, q, positions(2, 9), norm(), norm()), (None, None, None, None, None, None), (ONE, o, q, None, None, norm()),
                     (rotary(3), None, None, positions(3, 9, 2), None, norm()), (ONE, o, q, torch.zeros(9, dtype=torch.int32), norm(), None)):
            native, general = both(name, c, batch(pitch=6), k, v, *rest)
            assert native == general and native is not None
    native, general = both("read_u8", k, v, codes(), batch())
    assert native == general and native is not None
    for s in (0.125, 1):
        native, general = both("attention_paged_u8", o, q, codes(), batch(1), s, 1.5, 1)
        assert native == general and native is not None
    for bits in (torch.zeros(9, 2, dtype=torch.int32), torch.zeros(9, 5, dtype=torch.int32)[:, :3]):
        for name, c in (("attention_tree_f16", cache()), ("attention_tree_u8", codes())):
            native, general = both(name, o, q, c, batch(), DraftTree(bits), 0.125, 1.0)
            assert native == general and native is not None


def test_what_one_refuses_the_other_does_not_take(both):
    k, q, o = rows(2, 9, 64), rows(8, 9, 64), rows(8, 9, 64)
    other = TensorView.of(torch.zeros(8, 9, 64, dtype=torch.float32))
    tree = DraftTree(torch.zeros(9, 2, dtype=torch.int32))
    for name, *args in (
            ("norm_rotary_f16", o, rows(8, 8, 64), None, None, None), ("norm_rotary_f16", o, q, positions(1, 9), rotary(2), None),
            ("norm_rotary_f16", o, q, positions(2, 8), rotary(2), None), ("norm_rotary_f16", o, q, torch.zeros(9, dtype=torch.int32), rotary(2), None),
            ("norm_rotary_f16", o, q, torch.zeros(2, 9, dtype=torch.int64), rotary(2), None), ("norm_rotary_f16", o, q, None, None, norm(32)),
            ("norm_rotary_f16", o, other, None, None, None), ("norm_rotary_f16", o, q, positions(4, 9).t()[:4].t(), rotary(2), None),
            ("append_u8", codes(), batch(), rows(2, 9, 32), rows(2, 9, 32), None, None, None, None, None, None),
            ("append_u8", codes(), batch(), k, rows(2, 8, 64), None, None, None, None, None, None),
            ("append_u8", codes(), batch(), k, k, None, None, q, None, None, None),
            ("append_norm_f16", cache(), batch(), k, k, None, o, rows(8, 8, 64), None, None, None),
            ("append_norm_f16", cache(), batch(), k, k, rotary(), None, None, positions(3, 9), None, None),
            ("append_norm_f16", cache(), batch(), k, k, None, None, None, None, None, norm(60)),
            ("read_u8", k, rows(2, 8, 64), codes(), batch()), ("read_u8", q, o, codes(), batch()),
            ("attention_paged_u8", o, q, codes(d=32), batch(), 0.1, 1.0, 1), ("attention_paged_u8", other, q, codes(), batch(), 0.1, 1.0, 1),
            ("attention_tree_f16", o, q, cache(), batch(), DraftTree(torch.zeros(8, 2, dtype=torch.int32)), 0.1, 1.0),
            ("attention_tree_u8", o, rows(8, 8, 64), codes(), batch(), tree, 0.1, 1.0)):
        native, general = both(name, *args)
        assert native is None and general is None, (name, args)


def test_objects_of_other_kinds_are_refused(both):
    """A cache of codes where one of 16 bits is asked for (its codes would be read as halves, twice as far), several axes where one
    is, and objects that only have attributes of the same names, such as a norm of a model with weights of 32 bits."""
    k, q, o, tree = rows(2, 9, 64), rows(8, 9, 64), rows(8, 9, 64), DraftTree(torch.zeros(9, 2, dtype=torch.int32))

    class Like:
        def __init__(self, of, **change):
            self.__dict__.update({n: getattr(of, n) for n in of.__dataclass_fields__}, **change)
    wide = torch.nn.RMSNorm(64, eps=1e-5)
    for name, *args in (
            ("attention_tree_f16", o, q, codes(), batch(), tree, 0.1, 1.0), ("attention_tree_u8", o, q, cache(), batch(), tree, 0.1, 1.0),
            ("attention_paged_u8", o, q, cache(), batch(), 0.1, 1.0, 1), ("read_u8", k, k, cache(), batch()),
            ("append_norm_f16", codes(), batch(), k, k, None, None, None, None, None, None),
            ("append_u8", cache(), batch(), k, k, None, None, None, None, None, None),
            ("append_u8", codes(), batch(), k, k, None, None, None, None, None, wide), ("norm_rotary_f16", o, q, None, None, wide),
            ("norm_rotary_f16", o, q, None, None, Like(norm(), weight=torch.zeros(64))),
            ("attention_paged_u8", o, q, Like(codes()), batch(), 0.1, 1.0, 1),
            ("attention_tree_f16", o, q, cache(), batch(), Like(tree, bits=torch.zeros(9, 2, dtype=torch.int64)), 0.1, 1.0)):
        native, general = both(name, *args)
        assert native is None and general is None, (name, args)


def test_calls_of_one_axis_and_16_bits_refuse_the_new_kinds(recorders, monkeypatch):
    """rotary_f16, append_f16 and attention_paged_f16 through the native path, bound to where a call would be seen."""
    at = recorders.addresses[0]
    _native.bind(ABI, *[0] * 8, lambda: -1, lambda device: 0x1001 + device)
    _native.bind_sequences(at, at, at, at, torch.int32)
    _native.bind_step(*recorders.addresses, RotaryAxes, HeadNorm, PagedCacheU8, DraftTree)
    k, q, o = rows(2, 9, 64), rows(8, 9, 64), rows(8, 9, 64)
    try:
        p = torch.zeros(9, dtype=torch.int32)
        assert _native.rotary_f16(o, q, p, rotary(1)) is None
        assert _native.append_f16(cache(), batch(), k, k, rotary(1), None, None, None) is None
        assert _native.append_f16(codes(), batch(), k, k, None, None, None, None) is None
        assert _native.attention_paged_f16(o, q, codes(), batch(), 0.1, 1.0, 1) is None
        assert recorders.taken() == ""
    finally:
        _bind_native()


@pytest.mark.parametrize("axes", [1, 3])
def test_one_row_has_no_stride(both, axes):
    """Positions and bits of one row, or of one word, whatever the stride that is not used."""
    one = torch.zeros(1, axes, dtype=torch.int32).t()
    native, general = both("norm_rotary_f16", rows(4, 1, 64), rows(4, 1, 64), one, rotary(axes), None)
    assert general is not None and native in (None, general)
    native, general = both("attention_tree_f16", rows(8, 9, 64), rows(8, 9, 64), cache(), batch(), DraftTree(torch.zeros(9, 4, dtype=torch.int32)[:, ::4]), 0.1,
                           1.0)
    assert general is not None and native in (None, general)
