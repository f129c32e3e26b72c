"""The native host path of the calls over several sequences (host/native.cpp) against the methods of kernels.py, on the
CPU: a library of recorders, compiled here from the header, stands in the place of the kernels and takes what each passes."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from adrastea_amd import GpuKernels, MatmulMask, PackedBatch, PagedBatch, PagedCache, Rotary, TensorLayout, TensorView, _ffi, kernels
from adrastea_amd.kernels import _NATIVE_SEQUENCE_CALLS, _bind_native
from adrastea_amd.tensor import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ABI = _ffi.lib().adr_abi_version()
SHIM = """
#include "adrastea_kernels.h"
#include <cstdio>
#include <string>
static std::string seen;
static void put(double v) { char b[40]; snprintf(b, sizeof b, "%.17g ", v); seen += b; }
static void put(const void* p) { char b[40]; snprintf(b, sizeof b, "%p ", p); seen += b; }
static void put(int32_t v) { seen += std::to_string(v) + " "; }
static void put(uint32_t v) { seen += std::to_string(v) + " "; }
static void put(int64_t v) { seen += std::to_string(v) + " "; }
static void put(const adr_paged_cache& c) {
  put(c.key), put(c.value), put(c.pages), put(c.kv_heads), put(c.page_size), put(c.d), put(c.stride_kx), put(c.stride_ky);
  put(c.stride_kz), put(c.stride_kp), put(c.stride_vx), put(c.stride_vy), put(c.stride_vz), put(c.stride_vp);
}
static void put(const adr_paged_batch& b) {
  put(b.row_offsets), put(b.lengths), put(b.table), put(b.sequences), put(b.table_width), put(b.table_pitch);
  put(b.longest_rows), put(b.longest);
}
static void put(const adr_packed_batch& b) {
  put(b.row_offsets), put(b.key_offsets), put(b.sequences), put(b.longest_rows), put(b.longest);
}
static void put(const adr_rotary& r) { put(r.turns), put(r.dims), put(r.layout), put((double)r.magnitude); }
template <class... A> static int record(const A&... a) { seen.clear(); (put(a), ...); return 0; }
template <class F> struct Recorder;
template <class... A> struct Recorder<int(A...)> { static int call(A... a) { return record(a...); } };
extern "C" const char* taken() { static std::string t; t.swap(seen), seen.clear(); return t.c_str(); }
#define RECORDED(name) \\
  extern "C" void* at_##name() { return (void*)&Recorder<decltype(name)>::call; }
RECORDED(adr_rotary_f16) RECORDED(adr_append_f16) RECORDED(adr_attention_paged_f16) RECORDED(adr_attention_packed_f16)
"""


class Recorders:
    """The stand-in library: its four functions with the signatures of the real one, and what they were last given."""

    def __init__(self, path):
        self.so = C.CDLL(path)
        self.so.taken.restype = C.c_char_p
        self.addresses = []
        for name in _NATIVE_SEQUENCE_CALLS:
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
    (where / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"), "-o", str(where / "shim.so"),
                    str(where / "shim.cpp")], check=True)
    return Recorders(str(where / "shim.so"))


@pytest.fixture
def both(recorders, monkeypatch):
    """A call through the native path and through the general one: what each passed on (None: refused)."""
    _native.bind(ABI, *[0] * 8, lambda: -1, lambda device: 0x1001 + device)   # (tensors of the host say device -1)
    _native.bind_sequences(*recorders.addresses, torch.int32)
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
        except (AssertionError, AttributeError, TypeError, C.ArgumentError):
            general = None
        finally:
            monkeypatch.setattr(kernels, "_native", _native)
        return native or None, general
    yield call
    _bind_native()


def half(*dims):
    return torch.zeros(*dims, dtype=torch.float16)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def rows(heads, n, d, packed=False):
    return TensorView.of(half(heads, n, d)) if packed else TensorView.of(half(n, heads, d)).permute([1, 0, 2])


def cache(pages=6, heads=2, size=16, d=64):
    return PagedCache(TensorView.of(half(pages, size, heads, d)).permute([0, 2, 1, 3]), TensorView.of(half(pages, heads, size, d)))


def batch(n=2, pages=4, wide=7, **hints):
    return PagedBatch(ints(*range(n + 1)), ints(*[9] * n), torch.zeros(n, wide, dtype=torch.int32)[:, :pages], **hints)


def rotary(d=64, layout=1, magnitude=1.3):
    return Rotary(torch.zeros(d // 2, dtype=torch.float64), layout, magnitude)


def same(outcome):
    native, general = outcome
    assert native is not None and native == general
    return native


@pytest.mark.parametrize("packed", [False, True])
def test_rotary(both, packed):
    seen = same(both("rotary_f16", rows(3, 5, 64), rows(3, 5, 64, packed), ints(*range(5)), rotary()))
    assert seen.split()[-9:] == ["3", "5", "64", "1", "192", "64", *(["1", "64", "320"] if packed else ["1", "192", "64"])]
    x = TensorView.of(half(5, 64))
    same(both("rotary_f16", x, x, ints(*range(5)), rotary(32, 0)))


def test_append(both):
    c, b, k, v, q, o = cache(), batch(longest_rows=1, longest=60), rows(2, 2, 64), rows(2, 2, 64, True), rows(6, 2, 64), rows(6, 2, 64)
    at = ints(4, 5)
    for args in ((rotary(), None, None, None), (None, None, None, None), (rotary(), o, q, None), (rotary(), o, q, at),
                 (None, q, q, at), (rotary(), None, None, at)):
        same(both("append_f16", c, b, k, v, *args))


@pytest.mark.parametrize("mask", [MatmulMask.CAUSAL, MatmulMask.NONE, 1])
def test_attention(both, mask):
    q, o = rows(6, 2, 64), rows(6, 2, 64, True)
    for b in (batch(), batch(wide=4, longest_rows=1, longest=33)):
        same(both("attention_paged_f16", o, q, cache(), b, 0.125, 1.0, mask))
    one = PagedBatch(ints(0, 2), ints(9), torch.zeros(1, 4, dtype=torch.int32))
    same(both("attention_paged_f16", o, q, cache(), one, 0.3, 2, mask))
    p = PackedBatch(ints(0, 1, 2), ints(0, 4, 9), 1, 5)
    same(both("attention_packed_f16", o, q, rows(2, 9, 64), rows(2, 9, 64, True), p, 0.125, 1.0, mask))
    x = TensorView.of(half(2, 64))
    same(both("attention_packed_f16", x, x, x, x, PackedBatch(ints(0, 2), ints(0, 2)), 0.125, 1.0, mask))


def test_what_one_refuses_the_other_refuses(both):
    q, o, c, b, at, r = rows(6, 2, 64), rows(6, 2, 64), cache(), batch(), ints(4, 5), rotary()
    k = rows(2, 2, 64)
    p = PackedBatch(ints(0, 1, 2), ints(0, 1, 2))
    refused = [("rotary_f16", rows(5, 2, 64), q, at, r), ("rotary_f16", o, q, ints(1, 2, 3), r), ("rotary_f16", o, q, at.long(), r),
               ("rotary_f16", o, q, ints(1, 2, 3, 4)[::2], r), ("rotary_f16", o, q, [1, 2], r), ("rotary_f16", o, q, None, r),
               ("rotary_f16", o, q, ints(1, 2).view(1, 2), r), ("rotary_f16", o, q, at, None), ("rotary_f16", o, "q", at, r),
               ("append_f16", c, b, rows(3, 2, 64), rows(3, 2, 64), r, None, None, None),
               ("append_f16", c, b, rows(2, 2, 32), rows(2, 2, 32), r, None, None, None),
               ("append_f16", c, b, k, rows(2, 3, 64), r, None, None, None), ("append_f16", c, b, k, k, r, o, None, None),
               ("append_f16", c, b, k, k, r, None, q, None), ("append_f16", c, b, k, k, r, rows(5, 2, 64), q, None),
               ("append_f16", c, b, k, k, r, rows(6, 3, 64), rows(6, 3, 64), None), ("append_f16", c, b, k, k, r, o, q, at.long()),
               ("append_f16", c, b, k, k, r, o, q, ints(1)), ("append_f16", c, None, k, k, r, o, q, at),
               ("append_f16", None, b, k, k, r, o, q, at), ("append_f16", c, p, k, k, r, o, q, at),
               ("attention_paged_f16", rows(5, 2, 64), q, c, b, 0.1, 1.0, 1), ("attention_paged_f16", o, q, cache(d=32), b, 0.1, 1.0, 1),
               ("attention_paged_f16", o, q, c, p, 0.1, 1.0, 1), ("attention_paged_f16", o, q, c, b, "0.1", "x", 1),
               ("attention_packed_f16", o, q, k, rows(2, 3, 64), p, 0.1, 1.0, 1),
               ("attention_packed_f16", o, q, rows(2, 2, 32), rows(2, 2, 32), p, 0.1, 1.0, 1),
               ("attention_packed_f16", rows(6, 1, 64), q, k, k, p, 0.1, 1.0, 1), ("attention_packed_f16", o, q, k, k, b, 0.1, 1.0, 1)]
    for name, *args in refused:
        try:
            outcome = both(name, *args)
        except ValueError:      # (float("x"))
            outcome = None, None
        assert outcome == (None, None), (name, args)


def test_memory_of_another_device(both):
    class Elsewhere:   # (a tensor as far as the calls look, of a device that is not the current one)
        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)

        def get_device(self):
            return 1

    def away(view):
        return TensorView(Elsewhere(view.storage), view.layout, view.offset)
    q, c, b, at, r = rows(2, 2, 64), cache(), batch(), ints(4, 5), rotary()
    p = PackedBatch(ints(0, 1, 2), ints(0, 1, 2))
    for name, *args in [("rotary_f16", away(q), q, at, r), ("rotary_f16", q, away(q), at, r), ("rotary_f16", q, q, Elsewhere(at), r),
                        ("rotary_f16", q, q, at, Rotary(Elsewhere(r.turns), 1, 1.0)),
                        ("append_f16", PagedCache(away(c.key), c.value), b, q, q, r, None, None, None),
                        ("append_f16", c, b, q, away(q), r, None, None, None), ("append_f16", c, b, q, q, r, q, q, Elsewhere(at)),
                        ("attention_paged_f16", q, q, PagedCache(c.key, away(c.value)), b, 0.1, 1.0, 1),
                        ("attention_paged_f16", q, q, c, PagedBatch(b.row_offsets, Elsewhere(b.lengths), b.table), 0.1, 1.0, 1),
                        ("attention_packed_f16", q, q, away(q), q, p, 0.1, 1.0, 1),
                        ("attention_packed_f16", q, q, q, q, PackedBatch(p.row_offsets, Elsewhere(p.key_offsets)), 0.1, 1.0, 1)]:
        assert both(name, *args) == (None, None), (name, args)
    same(both("rotary_f16", q, q, at, r))


FAR = 1 << 31


def spread(*strides, dims=(6, 2, 64), offset=0):
    return TensorView(half(6 * 2 * 64), TensorLayout(dims, strides), offset)


def test_strides_and_sizes_of_more_than_32_bits(both):
    """Neither path passes on what the C interface would take for another number."""
    q, o, c, b, at, r, k = rows(6, 2, 64), rows(6, 2, 64), cache(), batch(), ints(4, 5), rotary(), rows(2, 2, 64)
    p = PackedBatch(ints(0, 1, 2), ints(0, 1, 2))
    two = (2, 2, 64)
    for strides in ((FAR, 64, 1), ((1 << 32) + 64, 64, 1), (-FAR - 1, 64, 1), (128, FAR, 1), (128, 64, 1 << 33)):
        x, y = spread(*strides), spread(*strides, dims=two)
        for name, *args in [("rotary_f16", x, q, at, r), ("rotary_f16", o, x, at, r), ("append_f16", c, b, y, k, r, None, None, None),
                            ("append_f16", c, b, k, y, r, None, None, None), ("append_f16", c, b, k, k, r, o, x, None),
                            ("append_f16", c, b, k, k, r, x, q, at), ("attention_paged_f16", x, q, c, b, 0.1, 1.0, 1),
                            ("attention_paged_f16", o, x, c, b, 0.1, 1.0, 1), ("attention_packed_f16", o, q, y, k, p, 0.1, 1.0, 1),
                            ("attention_packed_f16", o, q, k, y, p, 0.1, 1.0, 1), ("attention_packed_f16", o, x, k, k, p, 0.1, 1.0, 1)]:
            with pytest.raises(ValueError):
                both(name, *args)
    long = spread(64, 64, 1, dims=(2, FAR, 64))   # (never read: its address is all that a call takes)
    with pytest.raises(ValueError):
        both("attention_packed_f16", o, q, long, long, p, 0.1, 1.0, 1)
    pages = TensorView(half(64), TensorLayout((FAR, 2, 16, 64), (2048, 1024, 64, 1)))
    with pytest.raises(ValueError):
        both("attention_paged_f16", o, q, PagedCache(pages, pages), b, 0.1, 1.0, 1)


def test_what_fits_is_passed_on(both):
    """The ends of 32 bits, strides that no element uses, and hints of any size."""
    q, c, b = rows(6, 2, 64), cache(), batch()
    for z in (FAR - 1, -FAR):
        assert str(z) in same(both("attention_paged_f16", spread(z, 64, 1), q, c, b, 0.1, 1.0, 1)).split()
    one = spread(1 << 40, 64, 1, dims=(1, 2, 64))
    assert both("rotary_f16", one, one, ints(1, 2), rotary())[1].split()[-6:] == ["1", "64", "0", "1", "64", "0"]
    seen = both("attention_paged_f16", q, q, c, batch(longest_rows=1 << 40, longest=1 << 31), 0.1, 1.0, 1)[1].split()
    assert seen.count(str(FAR - 1)) == 2


def test_sizes_of_a_workspace_have_32_bits():
    p = PackedBatch.__new__(PackedBatch)
    for args in ((1 << 32, 2, 50, 50, 64), (4, 2, 1 << 31, 50, 64), (4, 2, 50, (1 << 32) + 1, 64)):
        with pytest.raises(ValueError):
            kernels.attention_packed_workspace_bytes(p, *args)
    with pytest.raises(ValueError):
        kernels.attention_paged_workspace_bytes(None, None, 4, 1 << 31)


CPP = r"""
#include "adrastea_amd/host/kernels.hpp"
#include <cstdio>
using namespace adrastea;
static f16* const P = (f16*)4096;  // never read
static int wrong = 0;
template <typename F> static void refuses(const char* what, F f) {
  try { f(); } catch (const std::logic_error&) { return; } catch (const std::exception&) {}
  printf("passed on: %s\n", what), wrong++;
}
int main() {
  GpuKernels k;
  const size_t far = size_t(1) << 31, z[] = {far, (far << 1) + 64, (size_t)(-(long)far - 1)};
  const PagedCache cache{{P, TensorLayout::row_major({6, 2, 16, 64})}, {P, TensorLayout::row_major({6, 2, 16, 64})}};
  const PagedBatch batch{(const int32_t*)P, (const int32_t*)P, (const int32_t*)P, 2, 3, 3, 1, 48};
  const PackedBatch packed{(const int32_t*)P, (const int32_t*)P, 2, 1, 48};
  const Rotary none{nullptr, 0, ADR_ROTARY_HALVES, 1.0f};
  TensorView<f16> out(P, TensorLayout::row_major({4, 3, 64}));
  const TensorView<const f16> q(P, out.layout), kv(P, TensorLayout::row_major({2, 3, 64}));
  for (size_t s : z) {
    TensorView<f16> o(P, TensorLayout({4, 3, 64}, {s, 64, 1}));
    const TensorView<const f16> x(P, o.layout), y(P, TensorLayout({2, 3, 64}, {s, 64, 1})), v(P, TensorLayout({2, 3, 64}, {192, s, 1}));
    refuses("rotary, output", [&] { k.rotary_f16(o, q, (const int32_t*)P, none); });
    refuses("rotary, input", [&] { k.rotary_f16(out, x, (const int32_t*)P, none); });
    refuses("append, key", [&] { k.append_f16(cache, batch, y, kv, none); });
    refuses("append, value", [&] { k.append_f16(cache, batch, kv, v, none); });
    refuses("append, query", [&] { k.append_f16(cache, batch, kv, kv, none, &out, &x); });
    refuses("paged", [&] { k.attention_paged_f16(out, x, cache, batch, 0.1f); });
    refuses("packed", [&] { k.attention_packed_f16(out, q, y, kv, packed, 0.1f); });
    refuses("packed, values", [&] { k.attention_packed_f16(out, q, kv, v, packed, 0.1f); });
  }
  const TensorLayout pages({far, 2, 16, 64}, {2048, 1024, 64, 1});
  refuses("pages", [&] { PagedCache{{P, pages}, {P, pages}}.lower(); });
  const TensorView<const f16> one(P, TensorLayout({1, 3, 64}, {far, 64, 1}));   // (a stride that no element uses)
  if (GpuKernels::rows_of(one, "").z != 0) printf("unused stride\n"), wrong++;
  const TensorView<const f16> back(P, TensorLayout({2, 3, 64}, {(size_t)-192l, 64, 1}));
  if (GpuKernels::rows_of(back, "").z != -192) printf("negative stride\n"), wrong++;
  return wrong;
}
"""


def test_strides_and_sizes_through_the_host_mirror(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "sizes.cpp").write_text(CPP)
    lib = os.path.dirname(_ffi.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-I" + ROOT, "-o", str(tmp_path / "sizes"), str(tmp_path / "sizes.cpp"), "-L" + lib,
                    "-l:" + os.path.basename(_ffi.LIB_PATH), "-Wl,-rpath," + lib, "-Wl,--allow-shlib-undefined"], check=True)
    r = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64, torch.uint8, torch.int32])
def test_values_of_another_type(both, dtype):
    """Nothing but fp16 is read, or written, as fp16."""
    def other(view):
        return TensorView(torch.zeros(view.storage.shape, dtype=dtype), view.layout)
    q, c, b, at, r, k = rows(6, 2, 64), cache(), batch(), ints(4, 5), rotary(), rows(2, 2, 64)
    p = PackedBatch(ints(0, 1, 2), ints(0, 1, 2))
    for name, *args in [("rotary_f16", other(q), q, at, r), ("rotary_f16", q, other(q), at, r),
                        ("append_f16", c, b, other(k), k, r, None, None, None), ("append_f16", c, b, k, other(k), r, None, None, None),
                        ("append_f16", c, b, k, k, r, other(q), q, None), ("append_f16", c, b, k, k, r, q, other(q), None),
                        ("attention_paged_f16", other(q), q, c, b, 0.1, 1.0, 1), ("attention_paged_f16", q, other(q), c, b, 0.1, 1.0, 1),
                        ("attention_packed_f16", other(q), q, k, k, p, 0.1, 1.0, 1), ("attention_packed_f16", q, other(q), k, k, p, 0.1, 1.0, 1),
                        ("attention_packed_f16", q, q, other(k), k, p, 0.1, 1.0, 1), ("attention_packed_f16", q, q, k, other(k), p, 0.1, 1.0, 1)]:
        assert both(name, *args) == (None, None), (name, args)
    for pools in ((other(c.key), c.value), (c.key, other(c.value))):
        with pytest.raises(TypeError):
            PagedCache(*pools)


@pytest.mark.parametrize("dtype", [torch.int16, torch.uint16])
def test_bits_of_fp16(both, dtype):
    """fp16 kept as 16-bit integers, as the C interface has it, is taken by the general path."""
    x = TensorView(torch.zeros(2, 6, 64, dtype=dtype), TensorLayout((6, 2, 64), (64, 384, 1)))
    native, general = both("rotary_f16", x, x, ints(4, 5), rotary())
    assert native is None and general.split()[-9:] == ["6", "2", "64", "1", "384", "64", "1", "384", "64"]


def test_views_that_begin_inside_their_storage(both):
    """As query, key and value views of one projection are."""
    qkv = TensorView.of(half(2, 10, 64)).permute([1, 0, 2])
    q, k, v = qkv.take([6, -1, -1]), qkv.skip([6, 0, 0]).take([2, -1, -1]), qkv.skip([8, 0, 0])
    same(both("append_f16", cache(), batch(), k, v, rotary(), q, q, None))
    p = PackedBatch(ints(0, 1, 2), ints(0, 1, 2))
    seen = same(both("attention_packed_f16", q, q, k, v, p, 0.1, 1.0, 1)).split()
    assert [int(x, 16) - int(seen[2], 16) for x in seen[3:5]] == [6 * 64 * 2, 8 * 64 * 2]
