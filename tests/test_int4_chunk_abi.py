"""CPU checks of the chunk attention entry: host-side refusals."""
import ctypes


def test_host_refusals():
    """Bad arguments come back as codes before anything is launched."""
    from akv import _C
    lib = _C.load()
    need = lib.akv_int4_chunk_workspace_bytes(128)
    assert need > 0 and lib.akv_int4_chunk_workspace_bytes(96) == 0

    def call(c=None, Hq=4, q=256, out=256, ws=256, nb=need, dtype=1, R=1, M=64, **kw):
        d = dict(pool=256, page_stride=8704, head_stride=4352, n_pages=4, table=256, table_stride=4, lens=256,
                 max_seqs=2, max_blocks=4, kv_heads=2, head_dim=128, group=128)
        d.update(kw)
        cache = _C.Int4Cache(*[d[f[0]] for f in _C.Int4Cache._fields_])
        return lib.akv_int4_chunk_attention(
            _C.ATTENTION_ARGS.pack(ctypes.addressof(cache) if c is None else c, 0, 0, q, 0, 0, 0, out, 0, 0, 0, 0, ws, nb,
                                   0, R, M, Hq, dtype, 1.0, 0), None)

    assert lib.akv_int4_chunk_attention(None, None) == -7
    assert call(c=0) == -7 and call(q=0) == -7 and call(out=0) == -7 and call(ws=0) == -7 and call(pool=0) == -7
    assert call(Hq=3) == -1 and call(R=-1) == -1 and call(M=-1) == -1 and call(head_dim=96) == -1
    assert call(q=257) == -3 and call(ws=264) == -3 and call(page_stride=8) == -3
    assert call(dtype=2) == -4 and call(M=1 << 21) == -4 and call(nb=need - 1) == -8
    assert call(R=0) == 0 and call(M=0) == 0
