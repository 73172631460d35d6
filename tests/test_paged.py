"""CPU: the paged cache's plan (which pieces a batch is cut into, where a row goes,
which page a block has) compiled for the host, the entry points' refusals, and the
oracle against closed forms.  No kernel runs here."""
from __future__ import annotations

import ctypes as C
import math
import os
import random
import subprocess

import pytest
import torch

from oracle import paged as OP
from tests.paged_inputs import cache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "scope_amd", "libscope_amd.so")
needs_lib = pytest.mark.skipif(not os.path.exists(LIB), reason="libscope_amd.so not built")

PLAN = r'''
#include "%s/scope_amd/csrc/paged_plan.h"
using namespace scope;
extern "C" {
int tiles(int64_t len, int64_t first, int64_t cap, int* lo) { return seq_tiles(len, first, cap, lo); }
int64_t piece(int64_t total, int pieces, int least, int turn) { return piece_tiles(total, pieces, least, turn); }
int pieces(int tiles, int64_t piece) { return seq_pieces(tiles, piece); }
void range(int lo, int tiles, int n, int i, int* t) { piece_range(lo, tiles, n, i, t, t + 1); }
int64_t page(const int32_t* row, int MP, int64_t lb, int64_t P) { return block_page(row, MP, lb, P); }
int64_t position(const int32_t* cu, const int32_t* lens, int B, int64_t i, int* b) { return row_position(cu, lens, B, i, b); }
}
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PLAN % ROOT)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    i64, p = C.c_int64, C.c_void_p
    for name, res, args in (("tiles", C.c_int, [i64, i64, i64, p]), ("piece", i64, [i64, C.c_int, C.c_int, C.c_int]),
                            ("pieces", C.c_int, [C.c_int, i64]), ("range", None, [C.c_int] * 4 + [p]),
                            ("page", i64, [p, C.c_int, i64, i64]), ("position", i64, [p, p, C.c_int, i64, p])):
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    return lib


@pytest.mark.parametrize("seed", range(40))
def test_every_tile_is_in_one_piece(plan, seed):
    """Batches of ragged lengths: the pieces cover each sequence's tiles once, fit
    their slots, and are at most a piece long; the tiles hold the seen positions."""
    r = random.Random(seed)
    B = r.choice([1, 1, 2, 3, 64, 65, 200])
    cap = r.choice([16, 4096, 131072, 2 ** 31 - 16])
    want = r.choice([1, 2, 128, 1024])
    least = r.choice([1, 8, 16])
    seqs = []
    for _ in range(B):
        n = r.choice([0, 1, -5, cap, cap + 9, 2 ** 31 - 1, r.randint(0, cap), int(cap ** r.random())])
        f = r.choice([0, 0, -7, n, n - 1, r.randint(0, cap), 2 ** 31 - 1])
        lo = C.c_int()
        t = plan.tiles(n, f, cap, C.byref(lo))
        end, first = min(max(n, 0), cap), max(f, 0)
        if first >= end:
            assert t == 0
        else:
            assert lo.value * 32 <= first < lo.value * 32 + 32 and (lo.value + t - 1) * 32 < end <= (lo.value + t) * 32
        seqs.append((lo.value, t))
    total = sum(t for _, t in seqs)
    turn = r.choice([1, 4])
    c = plan.piece(total, want, least, turn)
    assert c >= least and (c == least or c % turn == 0)
    slots = 0
    for lo, t in seqs:
        n = plan.pieces(t, c)
        assert 1 <= n <= max(want, 1)
        at = lo
        for i in range(n):
            got = (C.c_int * 2)()
            plan.range(lo, t, n, i, got)
            assert got[0] == at and got[0] <= got[1] <= lo + t and got[1] - got[0] <= max(c, 1)
            at = got[1]
        assert at == lo + t
        slots += n
    assert slots <= want + B and slots <= B * -(-(-(-cap // 32)) // least)


def test_list_pieces_cover_every_list(plan):
    """Lists share their pieces' length (that of a full list)."""
    for cap in (1, 2, 9, 36, 64, 1000, 33333):
        for n in (1, 2, 3, 7, 128):
            at = 0
            for i in range(n):
                got = (C.c_int * 2)()
                plan.range(0, cap, n, i, got)
                assert got[0] == at <= got[1] <= cap
                at = got[1]
            assert at == cap


def test_bad_pages_are_no_pages(plan):
    row = (C.c_int32 * 6)(0, 4, 5, -1, -2 ** 31, 2 ** 31 - 1)
    assert [plan.page(row, 6, i, 5) for i in range(-1, 7)] == [-1, 0, 4, -1, -1, -1, -1, -1]
    assert plan.page(row, 6, 2 ** 31 + 1, 5) == -1 and plan.page(row, 6, -2 ** 31, 5) == -1


def test_rows_find_their_sequence(plan):
    """Ordinary offsets, empty sequences, rows of none; offsets that decrease stay inside the batch."""
    lens = (C.c_int32 * 4)(10, 20, 30, 40)
    cu = (C.c_int32 * 5)(2, 5, 5, 9, 11)
    b = C.c_int()
    got = []
    for i in range(13):
        pos = plan.position(cu, lens, 4, i, C.byref(b))
        got.append((pos, b.value if pos >= 0 else None))
    assert got == [(-1, None)] * 2 + [(10, 0), (11, 0), (12, 0), (30, 2), (31, 2), (32, 2), (33, 2), (40, 3), (41, 3)] + [(-1, None)] * 2
    assert plan.position(None, lens, 4, 2, C.byref(b)) == 30 and b.value == 2
    r = random.Random(1)
    for _ in range(300):
        bad = (C.c_int32 * 5)(*[r.randint(-2 ** 31, 2 ** 31 - 1) for _ in range(5)])
        plan.position(bad, lens, 4, r.randint(0, 2 ** 31 - 1), C.byref(b))
        assert 0 <= b.value < 4


# ---- the oracle -----------------------------------------------------------------------
def test_oracle_attention_is_a_softmax_over_what_is_seen():
    c = cache([40, 7], Hq=4, Hkv=2, D=64, bs=16, seed=1)
    r = OP.decode_attn(c["q"], c["k_pages"], c["v_pages"], c["table"], c["lens"], scale=0.1, first=torch.tensor([3, 0]))
    for b, (lo, hi) in enumerate(((3, 40), (0, 7))):
        pages = c["table"][b, :-(-hi // 16)].long()
        k, v = (x[pages].transpose(0, 1).reshape(2, -1, 64)[:, lo:hi].double() for x in (c["k_pages"], c["v_pages"]))
        q = c["q"][b].double().reshape(2, 2, 64)
        p = torch.softmax(0.1 * q @ k.transpose(1, 2), -1)
        assert torch.allclose((p @ v).reshape(4, 64), r["out"][b], atol=1e-12)
        assert torch.allclose(r["weights"][b].sum(-1), torch.full((2,), 2.0, dtype=torch.float64))


def test_oracle_eviction_and_penalties_by_hand():
    table = torch.tensor([[5, 6, -1, 7, 8]], dtype=torch.int32)
    mass = torch.tensor([[[0.3, 0.1, 0.0, 0.1, 9.0]]])
    new, freed, n = OP.evict(table, mass, torch.tensor([5 * 16 - 2]), torch.tensor([2]), bs=16)
    assert new.tolist() == [[5, -1, -1, -1, 8]] and freed.tolist() == [[6, 7, -1, -1, -1]] and n.tolist() == [2]
    new, freed, n = OP.evict(table, mass, torch.tensor([33]), torch.tensor([0]), bs=16, window=1, n_global=1)
    assert new.tolist() == [[5, -1, -1, 7, 8]] and n.tolist() == [1]
    z = OP.penalties(torch.tensor([[2.0, -2.0, 1.0, 4.0]]), torch.tensor([[0, 1, 0, 9]]), torch.tensor([3]), repetition=2.0,
                     presence=0.5, frequency=0.25, temperature=0.5, bias=torch.tensor([0.0, 0.0, 1.0, 0.0]), mask=torch.tensor([7]))
    assert z.tolist() == [[(1.0 - 0.5 - 0.5) * 2, (-4.0 - 0.25 - 0.5) * 2, 4.0, -math.inf]]


# ---- refusals --------------------------------------------------------------------------
@needs_lib
def test_library_refuses_before_any_launch():
    """Bad sizes at the C boundary: an error code and its message, with pointers that are never followed."""
    from scope_amd import _lib

    lib = _lib.load()
    one = C.c_void_p(16)
    good = dict(B=2, Hkv=2, D=128, bs=64, MP=4, type=0, fp8=0, P=8, k_sp=2 * 64 * 128, k_sh=64 * 128, k_sr=128, v_sp=2 * 64 * 128,
                v_sh=64 * 128, v_sr=128)

    def attn(word, Hq=4, maxkv=0, q=one, q_sb=512, num=None, idx=None, work=one, pages=one, **kw):
        c = _lib.PagedCache(**{**good, **kw})
        rc = lib.scope_paged_decode_attn(C.byref(c), Hq, maxkv, 0.1, q, q_sb, 128, pages, pages, None, None, one, one, None, num, idx,
                                         None, work, one, one, None)
        assert rc == -1 and word in lib.scope_last_error().decode(), lib.scope_last_error()

    for word, kw in (("head dim", dict(D=96)), ("page size", dict(bs=48)), ("page size", dict(bs=512)), ("type", dict(type=2)),
                     ("bad sizes", dict(B=0)), ("bad sizes", dict(B=65536)), ("bad sizes", dict(Hkv=0)), ("bad sizes", dict(P=0)),
                     ("table row", dict(MP=0)), ("table row", dict(MP=2 ** 25)), ("aligned", dict(k_sr=132)),
                     ("table row", dict(MP=2 ** 27 - 1, bs=16)),  # 2^26 tiles, 64 of which pass 32 bits
                     ("aligned", dict(v_sp=4)), ("aligned", dict(fp8=1, k_sr=136)), ("aligned", dict(pages=C.c_void_p(8))),
                     ("null pages", dict(pages=None)), ("multiple", dict(Hq=3)), ("multiple", dict(Hq=0)),
                     ("multiple", dict(Hq=65536)), ("kv_num", dict(num=one)), ("kv_num", dict(idx=one, maxkv=3)),
                     ("kv_num", dict(num=one, idx=one)), ("kv_num", dict(maxkv=3)), ("kv_num", dict(num=one, idx=one, maxkv=2 ** 26)),
                     ("null pointer", dict(q=None)), ("null pointer", dict(work=None, MP=4096)), ("aligned", dict(q_sb=516)),
                     ("aligned", dict(q=C.c_void_p(24))), ("aligned", dict(work=C.c_void_p(8)))):
        attn(word, **kw)

    def append(word, N=2, k=one, k_sn=256, cu=None, **kw):
        c = _lib.PagedCache(**{**good, **kw})
        rc = lib.scope_paged_append(C.byref(c), N, k, k_sn, 128, one, 256, 128, cu, one, one, None, None, one, one, None)
        assert rc == -1 and word in lib.scope_last_error().decode(), lib.scope_last_error()

    for word, kw in (("rows", dict(N=-1)), ("need cu", dict(N=3)), ("null pointer", dict(k=None)), ("aligned", dict(k_sn=260)),
                     ("aligned", dict(k=C.c_void_p(4))), ("head dim", dict(D=80))):
        append(word, **kw)
    c = _lib.PagedCache(**good)
    assert lib.scope_paged_append(C.byref(c), 0, None, 0, 0, None, 0, 0, None, None, None, None, None, one, one, None) == 0

    def evict(word, B=1, Hkv=1, MP=4, bs=16, window=1, n_global=0, table=one):
        rc = lib.scope_paged_evict(B, Hkv, MP, bs, window, n_global, table, one, one, one, one, one, one, None)
        assert rc == -1 and word in lib.scope_last_error().decode(), lib.scope_last_error()

    for word, kw in (("bad sizes", dict(B=0)), ("bad sizes", dict(MP=65537)), ("bad sizes", dict(MP=0)), ("bad sizes", dict(bs=0)),
                     ("bad sizes", dict(Hkv=0)), ("window", dict(window=0)), ("window", dict(n_global=-1)), ("null pointer", dict(table=None))):
        evict(word, **kw)

    def penalise(word, logits=one, **kw):
        p = _lib.PenaltyParams(**{**dict(B=1, type=2, V=100, T=5, repetition=1.0, temperature=1.0), **kw})
        rc = lib.scope_logit_penalties(C.byref(p), logits, one, one, *[None] * 8, one, None)
        assert rc == -1 and word in lib.scope_last_error().decode(), lib.scope_last_error()

    for word, kw in (("sizes", dict(B=0)), ("sizes", dict(B=70000)), ("sizes", dict(V=0)), ("sizes", dict(T=-1)),
                     ("sizes", dict(V=2 ** 31)), ("type", dict(type=3)), ("null pointer", dict(logits=None))):
        penalise(word, **kw)
    # the workspace of sizes that no call takes: none, and no division by them
    assert lib.scope_paged_attn_workspace_bytes(None, 4, 0, 0) == 0
    for bad in (dict(B=0), dict(MP=0), dict(bs=0), dict(D=0), dict(Hkv=0), dict(Hkv=3), dict(B=-1), dict(MP=-2)):
        c = _lib.PagedCache(**{**good, **bad})
        assert lib.scope_paged_attn_workspace_bytes(C.byref(c), 4, 9, 1) == 0
    c = _lib.PagedCache(**good)
    assert lib.scope_paged_attn_workspace_bytes(C.byref(c), 0, 9, 1) == lib.scope_paged_attn_workspace_bytes(C.byref(c), 4, -1, 1) == 0
    assert lib.scope_paged_attn_workspace_bytes(C.byref(c), 4, 9, 1) > 0


@pytest.fixture()
def on_cpu(monkeypatch):
    """The wrappers' own checks, with the device check and the library left out: a
    call that passes them ends at the library's name."""
    from scope_amd import ops

    class Reached(Exception):
        pass

    def reached(*a):
        raise Reached

    monkeypatch.setattr(ops, "_gpu", lambda who, *ts: torch.device("cpu"))
    monkeypatch.setattr(ops, "_launch", reached)
    monkeypatch.setattr(ops, "query", lambda *a: 16)
    return ops, Reached


def test_cpu_tensors_are_refused():
    from scope_amd import ops

    c = cache([20], Hq=2, Hkv=1, D=64, bs=16)
    args = [c[k] for k in ("q", "k_pages", "v_pages", "table", "lens")]
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_decode_attn(*args, scale=0.1)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_append(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, 1, 64).bfloat16(), *args[1:])
    with pytest.raises(RuntimeError, match="GPU"):
        ops.paged_evict(c["table"], torch.zeros(1, 1, c["table"].shape[1]), c["lens"], 1, bs=16)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.logit_penalties(torch.zeros(8), torch.zeros(3, dtype=torch.int64), 3)


def test_attention_wrapper_refusals(on_cpu):
    ops, Reached = on_cpu
    c = cache([20, 5], Hq=4, Hkv=2, D=64, bs=16)
    f8 = cache([20, 5], Hq=4, Hkv=2, D=64, bs=16, fp8=True)

    def call(src=c, **kw):
        d = {**src, "scale": 0.1, **kw}
        return ops.paged_decode_attn(d.pop("q"), d.pop("k_pages"), d.pop("v_pages"), d.pop("table"), d.pop("lens"), **d)

    MP = c["table"].shape[1]
    num, idx = torch.ones(2, 2, dtype=torch.int32), torch.zeros(2, 2, 3, dtype=torch.int32)
    for src, ok in ((c, {}), (f8, {}), (c, dict(kv_num=num, kv_idx=idx, mass=torch.zeros(2, 2, MP), first=torch.tensor([0, 1]))),
                    (c, dict(lens=torch.tensor([3, 4])))):
        with pytest.raises(Reached):
            call(src, **ok)
    for src, bad in ((c, dict(q=c["q"].float())), (c, dict(q=c["q"].half())), (c, dict(q=c["q"][:, :3])), (c, dict(q=c["q"][:1])),
                     (c, dict(q=c["q"][0])), (c, dict(q=c["q"][:, :0])), (c, dict(q=c["q"][..., ::2].repeat(1, 1, 2).transpose(1, 2).contiguous().transpose(1, 2))),
                     (c, dict(v_pages=c["v_pages"][:, :1])), (c, dict(k_pages=c["k_pages"].float(), v_pages=c["v_pages"].float())),
                     (c, dict(v_pages=f8["v_pages"])), (c, dict(k_scale=torch.ones(2))), (f8, dict(k_scale=torch.ones(1))),
                     (f8, dict(v_scale=torch.ones(2).half())), (c, dict(table=c["table"].long())), (c, dict(table=c["table"][:, ::2])),
                     (c, dict(table=c["table"][0])), (c, dict(lens=torch.ones(3, dtype=torch.int32))), (c, dict(lens=torch.ones(2))),
                     (c, dict(first=torch.ones(1, dtype=torch.int32))), (c, dict(kv_num=num)), (c, dict(kv_idx=idx)),
                     (c, dict(kv_num=num[:1], kv_idx=idx)), (c, dict(kv_num=num, kv_idx=idx.float())), (c, dict(kv_num=num.float(), kv_idx=idx)), (c, dict(kv_num=num, kv_idx=idx[0])), (c, dict(kv_num=num, kv_idx=idx[..., :0])),
                     (c, dict(mass=torch.zeros(2, 2, MP + 1))), (c, dict(mass=torch.zeros(2, 2, MP).double())),
                     (c, dict(mass=torch.zeros(2, 2, 2 * MP)[..., ::2]))):
        with pytest.raises(RuntimeError, match="paged_decode_attn"):
            call(src, **bad)


def test_integers_past_32_bits_stay_on_their_side(on_cpu):
    """A limit of 2^40 or the largest int64 for "none": not the 0 or -1 of its low 32 bits."""
    ops, _ = on_cpu
    x = torch.tensor([2 ** 40, -2 ** 40, 2 ** 63 - 1, -2 ** 63, 2 ** 31, -2 ** 31 - 1, 7, -7])
    want = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 7, -7]
    assert ops._ints("x", "x", x, 8, x.device).tolist() == ops._sat32(x[None])[0].tolist() == want
    y = torch.stack((x, x), 1)[:, 0]  # a column
    assert ops._ints("x", "y", y, 8, x.device).tolist() == want
    z = torch.arange(16, dtype=torch.int32)[::2]
    assert ops._ints("x", "z", z, 8, z.device).is_contiguous() and ops._sat32(z).tolist() == list(range(0, 16, 2))


def test_append_and_evict_wrapper_refusals(on_cpu):
    ops, Reached = on_cpu
    c = cache([20, 5], Hq=4, Hkv=2, D=64, bs=16)
    x = torch.zeros(2, 2, 64).bfloat16()

    def append(k=x, v=x, **kw):
        d = {**c, **kw}
        ops.paged_append(k, v, d["k_pages"], d["v_pages"], d["table"], d["lens"], cu=kw.get("cu"), k_scale=kw.get("k_scale"))

    for ok in ({}, dict(cu=torch.tensor([0, 1, 2]))):
        with pytest.raises(Reached):
            append(**ok)
    for bad in (dict(k=x.half(), v=x.half()), dict(k=x[:1]), dict(v=x.half()), dict(k=x[..., :32], v=x[..., :32]), dict(k=x[0], v=x[0]),
                dict(k=x.transpose(0, 2).contiguous().transpose(0, 2)), dict(cu=torch.tensor([0, 2])), dict(cu=torch.tensor([0.0, 1, 2])),
                dict(k_pages=c["k_pages"][:1].expand(4, -1, -1, -1), v_pages=c["v_pages"][:4]), dict(k_scale=torch.ones(2)),
                dict(lens=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="paged_append"):
            append(**bad)
    MP = c["table"].shape[1]
    mass = torch.zeros(2, 2, MP)

    def evict(table=c["table"], mass=mass, lens=c["lens"], budget=1, **kw):
        ops.paged_evict(table, mass, lens, budget, bs=16, **kw)

    for ok in ({}, dict(budget=torch.tensor([1, 2])), dict(out=c["table"])):
        with pytest.raises(Reached):
            evict(**ok)
    for bad in (dict(table=c["table"].long()), dict(mass=mass[..., :1]), dict(mass=mass.half()), dict(mass=mass[0]), dict(mass=mass.transpose(0, 1)[:, :, :]
                .contiguous().transpose(0, 1)), dict(lens=c["lens"][:1]), dict(budget=torch.tensor([1])), dict(out=c["table"].long()),
                dict(out=c["table"][:1]), dict(window=0), dict(window=-2 ** 32 + 5), dict(n_global=-1), dict(n_global=-2 ** 32)):
        with pytest.raises(RuntimeError, match="paged_evict"):
            evict(**bad)


def test_penalty_wrapper_refusals(on_cpu):
    ops, Reached = on_cpu
    z, t = torch.zeros(2, 70), torch.zeros(2, 9, dtype=torch.int64)

    def call(z=z, t=t, lens=3, **kw):
        ops.logit_penalties(z, t, lens, **kw)

    for ok in ({}, dict(z=z[0], t=t[0]), dict(lens=torch.tensor([1, 2])), dict(repetition=torch.ones(2), first=torch.tensor([0, 1])),
               dict(bias=torch.zeros(70), mask=torch.zeros(2, 3, dtype=torch.int32)), dict(out=z), dict(t=t[:, :0])):
        with pytest.raises(Reached):
            call(**ok)
    for bad in (dict(z=z.double()), dict(z=z.T), dict(z=z[None]), dict(z=z[:, :0]), dict(t=t[:1]), dict(t=t.float()), dict(t=t[:, ::2]),
                dict(lens=torch.tensor([1, 2, 3])), dict(lens=torch.tensor([1.0, 2.0])), dict(bias=torch.zeros(69)),
                dict(bias=torch.zeros(70).half()), dict(bias=torch.zeros(3, 70)), dict(mask=torch.zeros(2, 2, dtype=torch.int32)),
                dict(mask=torch.zeros(2, 3, dtype=torch.int64)), dict(out=z[:1]), dict(out=z.half()), dict(out=z[:1].expand(2, 70)),
                dict(repetition=torch.ones(3)), dict(first=torch.tensor([1])), dict(n_prompt=torch.tensor([1, 2, 3]))):
        with pytest.raises(RuntimeError, match="logit_penalties"):
            call(**bad)
    for bad in (dict(repetition=0.0), dict(repetition=-1.0), dict(temperature=0.0), dict(temperature=math.nan), dict(presence=math.inf),
                dict(frequency=math.nan)):
        with pytest.raises(ValueError, match="logit_penalties"):
            call(**bad)


def test_struct_layouts_match_the_header(tmp_path):
    from scope_amd._lib import PagedCache, PenaltyParams

    header = os.path.join(ROOT, "include", "scope_amd.h")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    structs = {"scope_paged_cache": PagedCache, "scope_penalty_params": PenaltyParams}
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls in structs.values():
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


# ---- the cache's bookkeeping -------------------------------------------------------------
def test_cache_takes_and_returns_pages():
    from scope_amd import PagedKVCache

    c = PagedKVCache(pages=6, sequences=2, max_len=80, kv_heads=1, head_dim=64, page_size=16, device="cpu")
    assert c.table.shape == (2, 5) and c.free_pages == 6
    c.reserve([17, 0])
    assert c.table.tolist() == [[0, 1, -1, -1, -1], [-1] * 5] and c.free_pages == 4
    c._len[0] = 17
    c.reserve([15, 1])  # to the end of its second page: only the other sequence needs one
    assert c.table.tolist() == [[0, 1, -1, -1, -1], [2, -1, -1, -1, -1]]
    c._len = [32, 1]
    with pytest.raises(RuntimeError, match="5 pages needed, 3 free"):
        c.reserve([48, 32])
    assert c.free_pages == 3 and c.table.tolist()[0] == [0, 1, -1, -1, -1]  # nothing was taken
    with pytest.raises(RuntimeError, match="81 positions of 80"):
        c.reserve([49, 0])
    with pytest.raises(ValueError, match="rows"):
        c.reserve([1])
    with pytest.raises(ValueError, match="rows"):
        c.reserve([1, -1])
    c.mass.fill_(1.0)
    c.release(0)
    assert c.free_pages == 5 and c.length(0) == 0 and c.table.tolist()[0] == [-1] * 5 and c.mass[0].sum() == 0 and c.mass[1].sum() > 0
    c.reserve([1, 0])
    assert c.table[0, 0] == 0  # the lowest of its own first
    with pytest.raises(ValueError, match="announced"):
        c.append(torch.zeros(2, 1, 64).bfloat16(), torch.zeros(2, 1, 64).bfloat16(), rows=[1, 0])
    with pytest.raises(RuntimeError, match="GPU"):
        c.append(torch.zeros(2, 1, 64).bfloat16(), torch.zeros(2, 1, 64).bfloat16())
    with pytest.raises(ValueError, match="at least 1"):
        PagedKVCache(pages=0, sequences=1, max_len=1, kv_heads=1, head_dim=64, device="cpu")
