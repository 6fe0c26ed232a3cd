"""The C entries of a step of drafted tokens refuse what they cannot do before they launch anything (no GPU is needed for that), and the host packs their
arguments as the structures lie in memory."""
import ctypes as C
import shutil
import subprocess

import pytest

from spite_b200.kernels import build, cuda

SOME = 1 << 20                 # an address that is never looked at
BAD, UNSUPPORTED = -1, -2


def entry(library, name, *argtypes):
    f = getattr(build.load(library), name)
    f.argtypes = argtypes
    return f


TREE = dict(q=SOME, out=SOME, num_heads=4, window_kind=0, window_size=0, scale=1.0, has_sink=0, sink=0.0, sinks=0, slopes=0, gates=0, by_head=0, softcap=0.0,
            bias=0, runs=0, bias_len=0, positions=SOME, seg=SOME, table=SOME, width=4, tokens=0, kv=SOME, v_offset=4096, pages=2, page=64, kv_heads=2, size=64,
            key_scale=0, cu=SOME, sets=SOME, segments=1, words=1)


@pytest.mark.parametrize("change,status", [
    (dict(), 0), (dict(q=0), BAD), (dict(kv=0), BAD), (dict(positions=0), BAD), (dict(seg=0), BAD), (dict(table=0), BAD), (dict(cu=0), BAD), (dict(sets=0), BAD),
    (dict(num_heads=3), BAD), (dict(kv_heads=0), BAD), (dict(words=0), BAD), (dict(segments=0), BAD), (dict(tokens=-1), BAD), (dict(width=0), BAD),
    (dict(window_kind=3), BAD), (dict(window_kind=2), BAD), (dict(bias=SOME), BAD), (dict(size=0), BAD), (dict(page=0), BAD)])
def test_tree_attention(change, status):
    call = cuda._TREE_CALL.pack(*{**TREE, **change}.values())
    plain = entry("attention_tree", "spite_tree_attention", C.c_int, C.c_char_p, C.c_void_p, C.c_longlong, C.c_int, C.c_int, C.c_void_p)
    tc = entry("attention_tree_tc", "spite_tree_attention_tc", C.c_char_p, C.c_int, C.c_void_p, C.c_longlong, C.c_void_p)
    assert plain(0, call, None, 0, 1, 64, None) == status
    assert tc(call, 148, SOME, 1 << 40, None) == status


def test_tree_attention_limits():
    pack = lambda **kw: cuda._TREE_CALL.pack(*{**TREE, **kw}.values())
    plain = entry("attention_tree", "spite_tree_attention", C.c_int, C.c_char_p, C.c_void_p, C.c_longlong, C.c_int, C.c_int, C.c_void_p)
    tc = entry("attention_tree_tc", "spite_tree_attention_tc", C.c_char_p, C.c_int, C.c_void_p, C.c_longlong, C.c_void_p)
    assert plain(0, pack(size=257), None, 0, 1, 64, None) == UNSUPPORTED
    assert plain(2, pack(tokens=5), None, 0, 1, 64, None) == BAD                       # a type that there is not
    assert plain(0, pack(tokens=5), None, 0, 2, 64, None) == BAD                       # shares without a place for them
    assert plain(0, pack(tokens=5), SOME, 5 * 4 * 2 * 68 - 1, 2, 64, None) == BAD
    assert plain(0, pack(), None, 0, 33, 64, None) == BAD and plain(0, pack(), None, 0, 1, 0, None) == BAD
    for kw in (dict(size=32), dict(page=32), dict(num_heads=258), dict(key_scale=SOME), dict(v_offset=0), dict(v_offset=4), dict(q=SOME + 8), dict(pages=1 << 30)):
        assert tc(pack(**kw), 148, SOME, 1 << 40, None) == UNSUPPORTED
    assert tc(pack(), 148, SOME, 148 * (4 * 66 * 128 + 4) - 1, None) == BAD and tc(pack(), 0, SOME, 1 << 40, None) == BAD
    assert tc(pack(tokens=1 << 30, width=1 << 20), 148, SOME, 1 << 40, None) == UNSUPPORTED        # (a line of work beyond 32 bits)


LAYOUT = dict(tables=SOME, held=SOME, free=SOME, n_free=SOME, slots=SOME, lengths=SOME, new=SOME, parents=0, block=SOME, cu=SOME, positions=SOME, seg=SOME,
              slot_map=SOME, sets=0, status=SOME, rows=4, width=8, pages=10, requests=2, out_width=8, tokens=16, n_parents=0, words=0, page=16, kind=0, size=0)


@pytest.mark.parametrize("change,status", [
    *[({n: 0}, BAD) for n in ("tables", "held", "slots", "lengths", "new", "block", "cu", "status", "positions", "seg", "slot_map", "free", "n_free", "rows", "width",
                              "requests", "out_width", "page", "pages")],
    (dict(tokens=-1), BAD), (dict(kind=3), BAD), (dict(kind=1), BAD), (dict(sets=SOME), BAD), (dict(parents=SOME, n_parents=-1), BAD),
    (dict(requests=4097), UNSUPPORTED), (dict(rows=(1 << 16) + 1), UNSUPPORTED), (dict(words=33, sets=SOME), UNSUPPORTED), (dict(tokens=(1 << 20) + 1), UNSUPPORTED),
    (dict(width=(1 << 20) + 1), UNSUPPORTED)])
def test_layout_step(change, status):
    f = entry("drafts", "spite_layout_step", C.c_char_p, C.c_int, C.c_void_p)
    call = cuda._LAYOUT_CALL.pack(*{**LAYOUT, **change}.values())
    assert f(call, 0, None) == status


def test_layout_blocks():
    f = entry("drafts", "spite_layout_step", C.c_char_p, C.c_int, C.c_void_p)
    pack = lambda **kw: cuda._LAYOUT_CALL.pack(*{**LAYOUT, **kw}.values())
    assert f(pack(), 9, None) == BAD and f(pack(), -1, None) == BAD and f(pack(requests=513), 1, None) == UNSUPPORTED


ACCEPT = dict(tokens=SOME, parents=0, targets=SOME, cu=SOME, counts=SOME, path=SOME, emitted=SOME, slots=0, lengths=0, lengths_out=0, n=4, requests=1, depth=3, rows=0,
              n_groups=1)
GROUP = dict(kv=SOME, scales=0, slot_map=SOME, plane_bytes=4096, planes=2, caches=1, pages=2, heads=1, page=16, row=128)


@pytest.mark.parametrize("change,group,status", [
    *[({n: 0}, {}, BAD) for n in ("tokens", "targets", "cu", "counts", "path", "emitted", "requests", "depth")],
    (dict(n=-1), {}, BAD), (dict(lengths=SOME, rows=1), {}, BAD), (dict(lengths=SOME, lengths_out=SOME), {}, BAD), (dict(n_groups=-1), {}, BAD),
    *[({}, {n: 0}, BAD) for n in ("kv", "slot_map", "planes", "caches", "pages", "heads", "page", "row")],
    (dict(depth=1025), {}, UNSUPPORTED), (dict(n_groups=9), {}, UNSUPPORTED), ({}, dict(row=255), UNSUPPORTED)])
def test_accept_drafts(change, group, status):
    f = entry("drafts", "spite_accept_drafts", C.c_char_p, C.c_int, C.c_void_p)
    call = cuda._ACCEPT_CALL.pack(*{**ACCEPT, **change}.values(), cuda._ACCEPT_GROUP.pack(*{**GROUP, **group}.values()))
    assert f(call, 1, None) == status
    assert f(call, 0, None) in (BAD, status)


@pytest.mark.skipif(shutil.which("g++") is None or not build._nvcc(), reason="needs the CUDA toolkit")
def test_the_packed_arguments_are_the_structures(tmp_path):
    """Sizes and last fields, by the compiler."""
    source = tmp_path / "sizes.cu"
    source.write_text('#include "attention_tree.cuh"\n#include "drafts.cu"\n#include <cstdio>\n#include <cstddef>\n'
                      'int main() { printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(TreeCall), offsetof(TreeCall, x) + offsetof(TreeStep, n_words), '
                      'sizeof(LayoutParams), offsetof(LayoutParams, window_size), sizeof(AcceptParams), offsetof(AcceptParams, groups), sizeof(AcceptGroup)); }\n')
    subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", str(build.CSRC), "-o", str(tmp_path / "sizes"), str(source)], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    tree, layout, accept, group = (s.size for s in (cuda._TREE_CALL, cuda._LAYOUT_CALL, cuda._ACCEPT_CALL, cuda._ACCEPT_GROUP))
    assert got == [tree, tree - 4, layout, layout - 8, accept, accept - cuda._ACCEPT_GROUPS * group, group]
