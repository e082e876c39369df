"""CPU checks of the weight and eviction entries: structs as the header lays them out, host-side refusals."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("packer,name,last", [("WEIGH_ARGS", "akv_int4_weigh_args", "reserved"),
                                              ("EVICT_ARGS", "akv_int4_evict_args", "recent")])
def test_packed_args_match_header(tmp_path, packer, name, last):
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


def _table(**kw):
    from akv import _C
    d = dict(table=256, table_stride=4, lens=256, refs=256, free_bits=256, max_seqs=2, max_blocks=4, n_pages=4)
    d.update(kw)
    return _C.PageTable(*[d[f[0]] for f in _C.PageTable._fields_])


def test_weigh_refusals():
    from akv import _C
    lib = _C.load()

    need = lib.akv_int4_weigh_workspace_bytes(1, 64, 4, 2, 128, 128)
    assert need > 16 and lib.akv_int4_weigh_workspace_bytes(1, 1, 4, 2, 128, 128) == 16
    assert lib.akv_int4_weigh_workspace_bytes(1, 64, 3, 2, 128, 128) == 0

    def weigh(c=None, Hq=4, q=256, lse=256, w=256, stride=128, R=1, M=1, dtype=0, ws=0, nb=0, **kw):
        d = dict(pool=256, page_stride=8704, head_stride=4352, n_pages=4, table=256, table_stride=4, lens=256,
                 max_seqs=2, max_blocks=4, kv_heads=2, head_dim=128, group=128)
        d.update(kw)
        cache = _C.Int4Cache(*[d[f[0]] for f in _C.Int4Cache._fields_])
        return lib.akv_int4_weigh(_C.WEIGH_ARGS.pack(ctypes.addressof(cache) if c is None else c, 0, 0, q, 0, 0, 0, lse,
                                                     w, stride, ws, nb, 0, R, M, Hq, dtype, 1.0, 0), None)

    assert lib.akv_int4_weigh(None, None) == -7 and weigh(c=0) == -7
    assert weigh(q=0) == -7 and weigh(lse=0) == -7 and weigh(w=0) == -7 and weigh(pool=0) == -7
    assert weigh(Hq=3) == -1 and weigh(R=-1) == -1 and weigh(M=-1) == -1 and weigh(stride=127) == -1
    assert weigh(head_dim=96) == -1 and weigh(q=257) == -3 and weigh(lse=258) == -3 and weigh(w=257) == -3
    assert weigh(M=64) == -7 and weigh(M=64, ws=264, nb=need) == -3 and weigh(M=64, ws=256, nb=need - 1) == -8
    assert weigh(dtype=2) == -4 and weigh(R=0) == 0 and weigh(M=0) == 0 and weigh(M=1 << 29) == -4


def test_evict_refusals():
    from akv import _C
    lib = _C.load()
    need = lib.akv_int4_evict_workspace_bytes(1, 4, 4)
    assert need > 0 and lib.akv_int4_evict_workspace_bytes(0, 4, 4) == 0

    def evict(t=None, pool=256, page=8704, w=256, w_row=128, kept=256, ws=256, nb=need, n=1, layers=1, H=2, D=128,
              group=128, keep=8, first=0, recent=0, **kw):
        table = _table(**kw)
        return lib.akv_int4_evict(_C.EVICT_ARGS.pack(ctypes.addressof(table) if t is None else t, pool, 0, page, w, 0,
                                                     w_row, 0, kept, ws, nb, 0, n, layers, H, D, group, keep, first,
                                                     recent), None)

    assert lib.akv_int4_evict(None, None) == -7 and evict(t=0) == -7 and evict(pool=0) == -7 and evict(w=0) == -7
    assert evict(kept=0) == -7 and evict(ws=0) == -7 and evict(lens=0) == -7
    assert evict(keep=0) == -1 and evict(first=-1) == -1 and evict(recent=9) == -1 and evict(first=4, recent=5) == -1
    assert evict(n=-1) == -1 and evict(n=65536) == -1 and evict(layers=0) == -1 and evict(page=4352) == -1
    assert evict(w_row=127) == -1 and evict(D=96) == -1 and evict(max_blocks=0) == -1
    assert evict(pool=264) == -3 and evict(ws=264) == -3 and evict(w=258) == -3 and evict(nb=need - 1) == -8
    assert evict(max_blocks=(1 << 20) + 1, table_stride=1 << 21) == -4 and evict(n=0) == 0


def test_weight_helpers_refusals():
    from akv import _C
    lib = _C.load()
    t = _table()
    r = ctypes.byref(t)
    for f in (lib.akv_int4_weights_clear, lib.akv_int4_weights_fork):
        assert f(None, 256, 0, 128, 1, 256, 256, 1, None) == -7 and f(r, None, 0, 128, 1, 256, 256, 1, None) == -7
        assert f(r, 256, 0, 127, 1, 256, 256, 1, None) == -1 and f(r, 256, 0, 128, 0, 256, 256, 1, None) == -1
        assert f(r, 256, 0, 128, 1, 256, 256, -1, None) == -1 and f(r, 256, 0, 128, 1, 256, 256, 0, None) == 0
        assert f(r, 256, 0, 128, 1, 256, None, 1, None) == -7
