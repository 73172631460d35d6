"""CPU: the 4-bit cache's oracle against its definition, what its wrappers refuse and
pass on, and the C entry points' refusals."""
from __future__ import annotations

import ctypes as C
import math
import os

import pytest
import torch

from oracle import paged as OP
from tests.paged_fp4_inputs import E8M0, FP4, cache4, pages
from tests.paged_inputs import TYPES, cache, tables
from tests.test_paged_wrappers import Reached, on_cpu  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "scope_amd", "libscope_amd.so")
needs_lib = pytest.mark.skipif(not os.path.exists(LIB), reason="libscope_amd.so not built")


# ---- the oracle ---------------------------------------------------------------------
def groups(dtype):
    """Groups of 32 that reach every rule: ties, carries of the scale, the type's ends, zeros, infinities, NaN."""
    t, g = TYPES[dtype], torch.Generator().manual_seed(1)
    big = torch.finfo(t).max
    rows = [torch.zeros(32), -torch.zeros(32), torch.full((32,), big), torch.full((32,), torch.finfo(t).smallest_normal),
            torch.full((32,), torch.finfo(t).smallest_normal / 4), torch.linspace(-big, big, 32)]
    for top in (6.0, 6.98, 7.0, 7.02, 8.0, 4.0, 3.5, 5.0, 1.75, 1.7421875):
        x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.26, 0.24, 0.74, 0.76, 2.49, 2.51, 4.9, 5.1] * 2).clamp(max=top)
        x[16:] *= -1
        x[3] = top
        rows += [x, x * 2.0 ** -9, x * 2.0 ** 12 if dtype == "fp16" else x * 2.0 ** 120]
    rows += [torch.randn(32, generator=g) * 2.0 ** e for e in range(-30, 15, 3)]
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.randn(32, generator=g)
        x[17] = bad
        rows.append(x)
    return torch.stack(rows).to(t)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_the_tensor_form_is_the_definition(dtype):
    x = groups(dtype)
    q, s = OP.quantise(x)
    for row, bytes_, byte in zip(x, q, s):
        codes, e = OP.quantise_group(row)
        assert byte.item() == e
        assert [b for pair in bytes_.tolist() for b in (pair % 16, pair // 16)] == codes


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_no_value_is_off_by_more_than_half_a_step(dtype):
    """Where the scale is not at an end: half of the grid's step around each value, and the largest by half of its own."""
    g = torch.Generator().manual_seed(2)
    x = (torch.randn((4000, 32), generator=g) * 2.0 ** torch.randint(-8, 8, (4000, 1), generator=g)).to(TYPES[dtype])
    q, s = OP.quantise(x)
    back, unit = OP.e2m1_values(q, s), 2.0 ** (s.double() - 127)
    z = back.abs() / unit
    step = torch.where(z < 2, 0.5, torch.where(z < 4, 1.0, 2.0))
    assert bool(((back - x.double()).abs() <= step / 2 * unit).all())
    assert bool((x.double().abs().amax(-1, keepdim=True) / unit <= 7).all())
    # what the values stand for, written once more, is itself
    again = OP.quantise(back.to(TYPES[dtype]))
    assert torch.equal(OP.e2m1_values(*again), back)


def test_values_of_every_byte():
    b = torch.arange(256, dtype=torch.uint8).reshape(16, 16)
    v = OP.e2m1_values(b, torch.full((16, 1), 127 + 3, dtype=torch.uint8))
    assert v[0, 3].item() == 0.0 and v[1, :6].tolist() == [0.0, 4.0, 4.0, 4.0, 8.0, 4.0][:6]
    assert v[15, 30:].tolist() == [-48.0, -48.0] and v[7, 30:].tolist() == [-48.0, 48.0]
    assert bool(torch.isnan(OP.e2m1_values(b, torch.full((16, 1), 255, dtype=torch.uint8))).all())


# ---- the wrappers -------------------------------------------------------------------
def call_of(ops, c, **kw):
    return ops.paged_decode_attn(c["q"], c["k_pages"], c["v_pages"], c["table"], c["lens"], scale=0.1, k_scale=c["k_scale"],
                                 v_scale=c["v_scale"], **kw)


@needs_lib
def test_calls_reach_their_entry_points(on_cpu):  # noqa: F811
    ops = on_cpu
    c = cache4([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    kw = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])
    with pytest.raises(Reached) as e:
        call_of(ops, c)
    assert e.value.args[0] == "scope_paged_decode_attn_fp4"
    with pytest.raises(Reached) as e:
        ops.paged_append(kv, kv, c["k_pages"], c["v_pages"], c["table"], c["lens"], **kw)
    assert e.value.args[0] == "scope_paged_append_fp4"
    for dtype in (None, torch.bfloat16, torch.float16):
        with pytest.raises(Reached) as e:
            ops.paged_read(c["k_pages"], c["v_pages"], c["table"], c["lens"], rows=2, dtype=dtype, **kw)
        assert e.value.args[0] == "scope_paged_read"


def test_scales_that_do_not_fit_are_refused(on_cpu):  # noqa: F811
    ops = on_cpu
    c = cache4([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    P, bad = c["k_pages"].shape[0], []
    bad += [None, c["k_scale"].view(torch.uint8), torch.ones(2), c["k_scale"][:, :, :, :1], c["k_scale"][:, :1], c["k_scale"][1:]]
    bad.append(c["k_scale"].view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(E8M0) if P else None)
    for s in bad:
        for name in ("k_scale", "v_scale"):
            with pytest.raises(RuntimeError, match="float8_e8m0fnu"):
                call_of(ops, dict(c, **{name: s}))
    d = cache([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    with pytest.raises(RuntimeError, match="scale"):
        call_of(ops, dict(d, k_scale=c["k_scale"], v_scale=c["v_scale"]))
    with pytest.raises(RuntimeError, match="one shape and type"):
        call_of(ops, dict(c, v_pages=c["v_pages"][:, :, :, :16]))
    with pytest.raises(RuntimeError, match="one shape and type"):
        call_of(ops, dict(c, v_pages=d["v_pages"]))
    with pytest.raises(RuntimeError, match="bfloat16 or float16 rows"):
        call_of(ops, dict(c, q=c["q"].float()))
    kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="expanded"):
        ops.paged_append(kv, kv, c["k_pages"], c["v_pages"], c["table"], c["lens"], k_scale=c["k_scale"],
                         v_scale=c["v_scale"][:1].expand(P, -1, -1, -1))
    with pytest.raises(RuntimeError, match="k and v must be"):
        ops.paged_append(kv[:, :, :32], kv[:, :, :32], c["k_pages"], c["v_pages"], c["table"], c["lens"], k_scale=c["k_scale"],
                         v_scale=c["v_scale"])


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "k_scale", "v_scale"])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_rows_are_not_written_into_expanded_tensors(on_cpu, name, dim):  # noqa: F811
    """Any of them, along any dimension; one of a single element is no expansion."""
    ops = on_cpu
    kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    of = dict(Hq=4, Hkv=2, D=64, bs=16)

    def call(c, kv=kv):
        ops.paged_append(kv, kv, c["k_pages"], c["v_pages"], c["table"], c["lens"], k_scale=c["k_scale"], v_scale=c["v_scale"])

    for c in (cache4([40, 5], **of),) + ((cache([40, 5], **of),) if name.endswith("pages") else ()):
        with pytest.raises(RuntimeError, match="expanded|contiguous in a page's head"):
            call(dict(c, **{name: c[name].narrow(dim, 0, 1).expand(c[name].shape)}))
    c = cache4([5, 0], Hq=1, Hkv=1, D=64, bs=16)
    one = {n: c[n][:1] for n in ("k_pages", "v_pages", "k_scale", "v_scale")}
    one[name] = one[name][0, 0][None, None].expand(1, 1, -1, -1)
    with pytest.raises(Reached):
        call(dict(c, **one), kv[:, :1])


def test_reads_that_do_not_fit_are_refused(on_cpu):  # noqa: F811
    ops = on_cpu
    c = cache([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    args = [c[k] for k in ("k_pages", "v_pages", "table", "lens")]
    cu = torch.tensor([0, 3, 7])
    for rows in (3, -1, 2 ** 31):
        with pytest.raises(RuntimeError, match="rows="):
            ops.paged_read(*args, rows=rows)
    with pytest.raises(RuntimeError, match="rows="):
        ops.paged_read(*args, rows=2 ** 31, cu=cu)
    with pytest.raises(RuntimeError, match="float16"):
        ops.paged_read(*args, rows=7, cu=cu, dtype=torch.float16)
    for kw in (dict(cu=cu[:2]), dict(cu=cu.float()), dict(cu=cu, first=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="must be int32 or int64"):
            ops.paged_read(*args, rows=1, **kw)
    with pytest.raises(Reached):
        ops.paged_read(*args, rows=7, cu=cu, first=2 ** 40)


def test_a_gradient_that_reaches_the_rows_raises(on_cpu, monkeypatch):  # noqa: F811
    ops = on_cpu
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    c = cache([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    kp = c["k_pages"].clone().requires_grad_()
    k, v = ops.paged_read(kp, c["v_pages"], c["table"], c["lens"], rows=2)
    for x in (k, v):
        with pytest.raises(RuntimeError, match="paged_read is not differentiable"):
            x.float().sum().backward()
    with torch.no_grad():
        assert not any(x.requires_grad for x in ops.paged_read(kp, c["v_pages"], c["table"], c["lens"], rows=2))


@needs_lib
@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
@pytest.mark.parametrize("fp8", [True, False])
def test_a_gradient_that_reaches_the_scales_raises(on_cpu, monkeypatch, name, fp8):  # noqa: F811
    """The results of e4m3 and 4-bit pages are products with their scales."""
    ops = on_cpu
    monkeypatch.setattr(ops, "_launch", lambda *a: None)
    of = dict(Hq=4, Hkv=2, D=64, bs=16)
    c = cache([40, 5], fp8=True, **of) if fp8 else cache4([40, 5], **of)
    c[name] = c[name].clone().requires_grad_()
    kw = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])
    for who, call in (("paged_read", lambda: ops.paged_read(c["k_pages"], c["v_pages"], c["table"], c["lens"], rows=2, **kw)),
                      ("paged_decode_attn", lambda: call_of(ops, c))):
        for x in call():
            with pytest.raises(RuntimeError, match=f"{who} is not differentiable"):
                x.float().sum().backward()
        with torch.no_grad():
            assert not any(x.requires_grad for x in call())


@pytest.fixture()
def held(monkeypatch):
    """A cache of three sequences of 40, 0 and 7 rows on the CPU, and what its reads pass on: (rows, first, cu)."""
    from scope_amd import PagedKVCache, ops

    monkeypatch.setattr(ops, "paged_append", lambda *a, **kw: None)
    monkeypatch.setattr(ops, "paged_read", lambda *a, rows, cu, first, **kw: (rows, first.tolist(), cu.tolist()))
    c = PagedKVCache(pages=9, sequences=3, max_len=64, kv_heads=1, head_dim=64, page_size=16, device="cpu")
    x = torch.zeros((47, 1, 64), dtype=torch.bfloat16)
    c.append(x, x, [40, 0, 7])
    return c


def test_a_cache_is_read_from_one_number_on(held):
    assert held.read() == held.read(first=0) == (47, [0, 0, 0], [0, 40, 40, 47])
    rows, first, cu = held.read(first=5)
    assert (rows, cu) == (37, [0, 35, 35, 37]) and (first[0], first[2]) == (5, 5)
    for f in ([5, 0, 5], torch.tensor([5, 0, 5])):
        assert held.read(first=f) == (37, [5, 0, 5], [0, 35, 35, 37])
    for f in (torch.tensor(2), 2):
        rows, first, cu = held.read([3, 0, 5], f)
        assert (rows, cu) == (8, [0, 3, 3, 8]) and (first[0], first[2]) == (2, 2)
    for f in (-1, [0, -1, 0], [0, 0], []):
        with pytest.raises(ValueError, match="are not held"):
            held.read(first=f)


def test_a_cache_read_from_behind_its_rows_gives_none(held):
    for far in (40, 2 ** 31, 2 ** 63):
        assert held.read(first=far) == (0, [0, 0, 0], [0, 0, 0, 0])
        assert held.read([2, 0, 0], [38, far, far]) == (2, [38, 0, 0], [0, 2, 2, 2])


def test_what_a_captured_call_of_the_cache_says(held, monkeypatch):
    """read changes nothing on the host, the others do."""
    class OnGPU:
        is_cuda = True

    held.table = OnGPU()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="read goes by the lengths on the host"):
        held.read()
    for call, name in ((lambda: held.reserve([1, 1, 1]), "reserve"), (lambda: held.evict(1), "evict"), (lambda: held.release(0), "release")):
        with pytest.raises(RuntimeError, match=f"{name} changes lengths or pages on the host"):
            call()


def test_no_cpu_path():
    from scope_amd import ops

    c = cache4([40, 5], Hq=4, Hkv=2, D=64, bs=16)
    kv = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    kw = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])
    for call in (lambda: call_of(ops, c), lambda: ops.paged_append(kv, kv, c["k_pages"], c["v_pages"], c["table"], c["lens"], **kw),
                 lambda: ops.paged_read(c["k_pages"], c["v_pages"], c["table"], c["lens"], rows=2, **kw)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# ---- the C entry points (their pointers are never followed) ---------------------------
def c_cache(**kw):
    from scope_amd import _lib

    f = dict(B=2, Hkv=2, D=64, bs=16, MP=4, type=0, fp8=0, P=9, k_sp=1024, k_sh=512, k_sr=32, v_sp=1024, v_sh=512, v_sr=32)
    f.update(kw)
    return _lib.PagedCache(**f)


@needs_lib
@pytest.mark.parametrize("bad,text", [(dict(D=96), "head dim"), (dict(bs=24), "page size"), (dict(type=2), "unknown type"), (dict(B=0), "bad sizes"),
                                      (dict(B=65536), "bad sizes"), (dict(Hkv=4097), "bad sizes"), (dict(P=0), "bad sizes"),
                                      (dict(MP=2 ** 27), "table row"), (dict(k_sr=24), "16-byte"), (dict(v_sp=8), "16-byte")])
def test_c_refusals_of_the_cache(bad, text):
    from scope_amd import _lib

    lib, one, c, z = _lib.load(), C.c_void_p(64), c_cache(**bad), _lib.PagedScales(64, 32, 64, 32)
    calls = [lambda: lib.scope_paged_append_fp4(C.byref(c), C.byref(z), 1, one, 0, 0, one, 0, 0, None, one, one, one, one, one, one, None),
             lambda: lib.scope_paged_read(C.byref(c), C.byref(z), 1, None, one, one, None, one, one, one, one, one, one, None),
             lambda: lib.scope_paged_decode_attn_fp4(C.byref(c), C.byref(z), 2, 0, 1.0, one, 0, 0, one, one, one, one, one, one, None, None,
                                                     None, None, one, one, one, None)]
    for call in calls:
        assert call() == -1 and text in lib.scope_last_error().decode(), lib.scope_last_error()


@needs_lib
def test_c_refusals_of_the_rest():
    from scope_amd import _lib

    lib, one, odd, c = _lib.load(), C.c_void_p(64), C.c_void_p(72), c_cache()
    z = _lib.PagedScales(64, 32, 64, 32)

    def refused(rc, text):
        assert rc == -1 and text in lib.scope_last_error().decode(), (rc, lib.scope_last_error())

    def append(c=C.byref(c), z=C.byref(z), N=1, k=one, k_sn=0, cu=None, table=one, ks=one, kp=one):
        return lib.scope_paged_append_fp4(c, z, N, k, k_sn, 0, one, 0, 0, cu, table, one, ks, one, kp, one, None)

    def read(c=C.byref(c), z=C.byref(z), N=1, cu=None, lens=one, ks=one, kp=one, k=one):
        return lib.scope_paged_read(c, z, N, cu, one, lens, None, ks, one, kp, one, k, one, None)

    def attend(c=C.byref(c), z=C.byref(z), Hq=2, maxkv=0, q=one, ks=one, idx=None, work=one, kp=one):
        return lib.scope_paged_decode_attn_fp4(c, z, Hq, maxkv, 1.0, q, 0, 0, kp, one, ks, one, one, one, None, None, idx, None, work,
                                               one, one, None)

    for f in (append, read, attend):
        refused(f(c=None), "null cache")
        refused(f(ks=None), "null scales")
        refused(f(ks=odd), "scales of a page's head")
        refused(f(z=C.byref(_lib.PagedScales(64, 24, 64, 32))), "scales of a page's head")
        refused(f(kp=None), "null pages")
    refused(append(z=None), "null scales")
    refused(attend(z=None), "null scales")
    for f in (append, read):
        refused(f(N=-1), "rows")
        refused(f(N=2 ** 31, cu=one), "rows")
        refused(f(N=3), "need cu")
        assert f(N=0) == 0
    refused(append(k=None), "null pointer")
    refused(append(k=odd), "16-byte")
    refused(append(k_sn=12), "16-byte")
    refused(append(table=None), "null pointer")
    refused(read(lens=None), "null pointer")
    refused(read(k=odd), "16-byte")
    refused(attend(Hq=3), "multiple")
    refused(attend(q=None), "null pointer")
    refused(attend(q=odd), "16-byte")
    refused(attend(idx=one), "come together")


@needs_lib
def test_struct_layout():
    import subprocess
    import tempfile

    from scope_amd import _lib

    text = '#include <stdio.h>\n#include <stddef.h>\n#include "%s/include/scope_amd.h"\nint main(void) { printf("%%zu %%zu", ' \
           'sizeof(scope_paged_scales), offsetof(scope_paged_scales, v_sh)); return 0; }' % ROOT
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "a.c"), os.path.join(d, "a")
        open(src, "w").write(text)
        subprocess.run(["gcc", "-std=c11", src, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [C.sizeof(_lib.PagedScales), _lib.PagedScales.v_sh.offset]


def test_rows_of_a_wavefront():
    """Every row is of one wavefront, its chunks fill the lanes, and the grid holds them all."""
    import subprocess
    import tempfile

    code = r'''
#include <stdio.h>
#include "%s/scope_amd/csrc/paged_plan.h"
using namespace scope;
int main() {
  const int64_t rows[] = {1, 2, 63, 64, 8191, 8192, 70000, (int64_t)1 << 27, ((int64_t)1 << 31) - 1};
  const int chunks[] = {8, 16, 24, 48, 64, 80, 128, 1024, 4096 * 32};
  for (int64_t N : rows)
    for (int c : chunks) {
      const int r = moved_rows(N, c);
      if (r < append_rows(N) || r > 64 || (r < 64 && (int64_t)r * c < 64)) return 1;
      if ((N + 4 * r - 1) / (4 * r) * 256 > kGridItems) return 2;
      if ((int64_t)r * c > INT32_MAX) return 3;
    }
  int b = 7;
  const int32_t cu[] = {0, 3, 3, 10};
  if (row_position(cu, nullptr, 3, 4, &b) != 1 || b != 2) return 4;
  if (row_position(nullptr, nullptr, 3, 2, &b) != 0 || b != 2) return 5;
  if (row_position(cu, nullptr, 3, 10, &b) != -1) return 6;
  return 0;
}''' % ROOT
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "a.cc"), os.path.join(d, "a")
        open(src, "w").write(code)
        subprocess.run(["g++", "-std=c++17", src, "-o", exe], check=True)
        assert subprocess.run([exe]).returncode == 0


def test_the_pieces_of_a_batch_have_slots():
    """The pieces that the attention's wavefronts find over 4-bit pages are no more than the slots that the host laid
    out, cover every tile once, and are as many as the device holds where the batch is large."""
    import random
    import subprocess
    import tempfile

    code = r'''
#include <stdio.h>
#include <stdlib.h>
#include "%s/scope_amd/csrc/paged_plan.h"
using namespace scope;
int main(int argc, char** argv) {
  // lines of B Hkv Hq D bs MP resident, then B lengths and B first positions
  int B, Hkv, Hq, D, bs, MP, resident, line = 0;
  while (scanf("%%d %%d %%d %%d %%d %%d %%d", &B, &Hkv, &Hq, &D, &bs, &MP, &resident) == 7) {
    ++line;
    int* lens = (int*)malloc(4 * B);
    int* first = (int*)malloc(4 * B);
    for (int b = 0; b < B; ++b) if (scanf("%%d", lens + b) != 1) return 1;
    for (int b = 0; b < B; ++b) if (scanf("%%d", first + b) != 1) return 1;
    const SplitSizes s = split_sizes(B, Hkv, D, bs, MP, Hq, 0);
    const int cols = Hkv * ((Hq / Hkv + 15) / 16);
    const int64_t cap = (int64_t)MP * bs;
    int64_t total = 0, pieces = 0;
    int lo;
    for (int b = 0; b < B; ++b) total += seq_tiles(lens[b], first[b], cap, &lo);
    const int w = pieces_wanted4(total, cols, B, resident), n = w < s.pieces ? w : s.pieces;
    if (n < 1) return 2;
    const int64_t piece = piece_tiles(total, n, kPieceTiles, piece_turn(D));
    for (int b = 0; b < B; ++b) {
      const int tiles = seq_tiles(lens[b], first[b], cap, &lo), m = seq_pieces(tiles, piece);
      int at = lo;
      for (int i = 0; i < m; ++i) {
        int t0, t1;
        piece_range(lo, tiles, m, i, &t0, &t1);
        if (t0 != at || t1 < t0) return 3;
        at = t1;
      }
      if (at != lo + tiles) return 4;
      if (m > 1 && !s.split) return 5;
      if (m > s.pieces + 1 && B == 1) return 6;
      pieces += m;
    }
    if (pieces > s.slots) { printf("line %%d: %%lld pieces, %%d slots\\n", line, (long long)pieces, s.slots); return 7; }
    // (as many as start together, one more a sequence, unless they would be longer than 120 tiles)
    if (B == 1 && total > 12LL * resident / cols && total < 100LL * resident / cols && resident >= 2 * cols && s.pieces >= resident / cols &&
        pieces * 2 < resident / cols) return 8;
    free(lens);
    free(first);
  }
  return line == 400 ? 0 : 9;
}''' % ROOT
    rng = random.Random(5)
    lines = []
    for _ in range(400):
        B = rng.choice([1, 1, 2, 7, 63, 64, 65, 300])
        Hkv, G = rng.choice([1, 2, 4, 8, 64, 600]), rng.choice([1, 4, 8, 16, 17, 40])
        bs, D = rng.choice([16, 32, 128, 256]), rng.choice([64, 128, 256])
        MP = max(1, int(2 ** rng.uniform(0, 13)))
        lens = [rng.choice([rng.randint(-3, MP * bs + 5), int(MP * bs * rng.random() ** 4)]) for _ in range(B)]
        first = [rng.choice([0, -2, rng.randint(0, MP * bs)]) for _ in range(B)]
        lines.append(f"{B} {Hkv} {Hkv * G} {D} {bs} {MP} {rng.choice([512, 768, 1024])}\n{' '.join(map(str, lens))}\n{' '.join(map(str, first))}\n")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "a.cc"), os.path.join(d, "a")
        open(src, "w").write(code)
        subprocess.run(["g++", "-std=c++17", src, "-o", exe], check=True)
        r = subprocess.run([exe], input="".join(lines), text=True, capture_output=True)
        assert r.returncode == 0, (r.returncode, r.stdout)
