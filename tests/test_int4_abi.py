"""CPU checks of the 4-bit cache's entry points: structs as the header lays them out, host-side refusals."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("struct,name", [("Int4Layout", "akv_int4_layout"), ("Int4Cache", "akv_int4_cache"),
                                         ("PageTable", "akv_page_table")])
def test_struct_matches_header(tmp_path, struct, name):
    from akv import _C
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    S = getattr(_C, struct)
    fields = [f[0] for f in S._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "akv_b200.h"\nint main(void){\n'
                   + f'printf("%zu\\n", sizeof({name}));\n'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "s"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(S)
    assert out[1:] == [getattr(S, f).offset for f in fields]


@pytest.mark.parametrize("packer,name,last", [("IO_ARGS", "akv_int4_io_args", "reserved"),
                                              ("ATTENTION_ARGS", "akv_int4_attention_args", "reserved"),
                                              ("VERIFY_ARGS", "akv_verify_args", "dtype")])
def test_packed_args_match_header(tmp_path, packer, name, last):
    """The packed argument structs have the header's size, and their last field its place."""
    from akv import _C
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "akv_b200.h"\nint main(void){\n'
                   f'printf("%zu %zu\\n", sizeof({name}), offsetof({name}, {last}));return 0;}}\n')
    exe = tmp_path / "s"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    size, off = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    S = getattr(_C, packer)
    assert (S.size, S.size - 4) == (size, off)


def test_layout():
    from akv import _C
    for d in (64, 128, 256):
        for g in (1, 2, 4):
            L = _C.int4_layout(d, d // g)
            assert (L.kc, L.vc, L.kp, L.vp, L.bytes) == (0, 16 * d, 32 * d, 32 * d + 128 * g, 32 * d + 256 * g)
            assert L.bytes % 16 == 0 and L.n_groups == g
    lib = _C.load()
    L = _C.Int4Layout()
    for d, g in ((96, 96), (128, 16), (128, 48), (0, 0), (512, 512)):
        assert lib.akv_int4_layout_init(d, g, ctypes.byref(L)) == -1
    assert lib.akv_int4_layout_init(128, 128, None) == -7
    assert _C.strerror(-9) != "unknown status"


def test_host_refusals():
    """Bad arguments come back as codes before anything is launched."""
    from akv import _C
    lib = _C.load()

    def cache(**kw):
        d = dict(pool=256, page_stride=8704, head_stride=4352, n_pages=4, table=256, table_stride=4, lens=256,
                 max_seqs=2, max_blocks=4, kv_heads=2, head_dim=128, group=128)
        d.update(kw)
        return ctypes.byref(_C.Int4Cache(*[d[f[0]] for f in _C.Int4Cache._fields_]))

    def append(c, k=256, dtype=0, R=1, M=1):
        return lib.akv_int4_append(_C.IO_ARGS.pack(0 if c is None else ctypes.addressof(c._obj), 0, 0, 0, k or 0, 0, 0,
                                                   0, 256, 0, 0, 0, 0, R, M, dtype, 0), None)

    assert append(None) == -7 and append(cache(pool=0)) == -7 and append(cache(), k=None) == -7
    assert append(cache(head_dim=96)) == -1 and append(cache(table_stride=3)) == -1 and append(cache(), R=-1) == -1
    assert append(cache(page_stride=8)) == -3 and append(cache(), k=257) == -3
    assert append(cache(), dtype=2) == -4 and append(cache(), R=70000) == -4
    assert append(cache(), R=0) == 0 and append(cache(), M=0) == 0

    need = lib.akv_int4_attention_workspace_bytes(1, 1, 4, 2, 128, 4)
    assert need > 0 and lib.akv_int4_attention_workspace_bytes(1, 1, 3, 2, 128, 4) == 0

    def attend(c, Hq=4, q=256, ws=256, n=need, dtype=0):
        return lib.akv_int4_attention(_C.ATTENTION_ARGS.pack(0 if c is None else ctypes.addressof(c._obj), 0, 0, q or 0,
                                                             0, 0, 0, 256, 0, 0, 0, 0, ws or 0, n, 0, 1, 1, Hq, dtype,
                                                             1.0, 0), None)

    assert attend(None) == -7 and attend(cache(), q=None) == -7 and attend(cache(), ws=None) == -7
    assert attend(cache(), Hq=3) == -1 and attend(cache(), ws=264) == -3 and attend(cache(), n=need - 1) == -8
    assert attend(cache(), dtype=2) == -4

    pt = _C.PageTable(256, 4, 256, 256, 256, 2, 4, 4)
    wb = lib.akv_pages_workspace_bytes(4, 2)

    def reserve(t, n=2, ws=256, nb=wb, layers=1, page=4352, granted=256):
        return lib.akv_pages_reserve(t, None, None, 1, n, granted, 256, layers, 0, page, ws, nb, None, None)

    t = ctypes.byref(pt)
    assert reserve(None) == -7 and reserve(t, granted=None) == -7 and reserve(t, n=2000) == -4 and reserve(t, n=-1) == -1
    assert reserve(t, nb=wb - 1) == -8 and reserve(t, page=8) == -3 and reserve(t, layers=0) == -1
    assert reserve(ctypes.byref(_C.PageTable(256, 4, 256, 256, 256, 2, 4, 0))) == -1
    assert lib.akv_pages_fork(t, None, 256, 1, None, None) == -7 and lib.akv_pages_fork(t, None, None, 0, None, None) == 0
    assert lib.akv_pages_truncate(t, None, None, -1, None, None) == -1
    assert lib.akv_pages_compact(t, 256, 1, 0, 4352, None, 256, wb, None, None) == -7
    assert lib.akv_pages_copy(256, 1, 0, 4352, 4, None, 256, 1, None, None) == -7

    def verify(target=256, K=2, V=10, dtype=2, B=1, tokens=256):
        return lib.akv_verify_draft(_C.VERIFY_ARGS.pack(target or 0, 0, 0, 256, 0, 0, tokens or 0, 0, 256, 256, 256, 256,
                                                        0, B, K, V, dtype), None)

    assert verify(target=None) == -7 and verify(tokens=None) == -7 and verify(V=0) == -1 and verify(K=-1) == -1
    assert verify(dtype=3) == -4 and verify(target=257) == -3 and verify(B=0) == 0 and verify(V=1 << 24) == -1
