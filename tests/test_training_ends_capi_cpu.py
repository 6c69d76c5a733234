"""What the C entries of the embedding, the cross entropy without logits and the orthogonalised update refuse, before they touch a device."""
import ctypes as C

ONE = C.c_void_p(4096)
AT = lambda byte: C.c_void_p(4096 + byte)


def _lookup(lib, table=ONE, dtype=0, vocab=10, channels=8, ids=ONE, n=3, scale=1.0, padding=-1, out=ONE):
    return lib.pb_embedding_lookup(table, dtype, vocab, channels, ids, n, scale, padding, out, None)


def _lookup_bwd(lib, g=ONE, dtype=0, ids=ONE, n=3, vocab=10, channels=8, d=ONE, ws=ONE, size=1 << 30):
    return lib.pb_embedding_lookup_bwd(g, dtype, ids, n, vocab, channels, 1.0, -1, d, ws, size, None)


def test_embedding(built_lib):
    for name in ("table", "ids", "out"):
        assert _lookup(built_lib, **{name: None}) == 1, name
    for name in ("g", "ids", "d", "ws"):
        assert _lookup_bwd(built_lib, **{name: None}) == 1, name
    assert _lookup(built_lib, dtype=2) == 4 and _lookup_bwd(built_lib, dtype=-1) == 4
    for bad in (dict(vocab=0), dict(channels=0), dict(n=-1), dict(vocab=1 << 31), dict(channels=1 << 22), dict(n=1 << 29)):
        assert _lookup(built_lib, **bad) == 2 and _lookup_bwd(built_lib, **bad) == 2, bad
    assert _lookup(built_lib, n=1 << 28, channels=1 << 21) == 2
    assert _lookup(built_lib, table=AT(2)) == 9 and _lookup(built_lib, out=AT(1), dtype=1) == 9 and _lookup(built_lib, ids=AT(4)) == 9
    assert _lookup_bwd(built_lib, g=AT(2)) == 9 and _lookup_bwd(built_lib, d=AT(1), dtype=1) == 9 and _lookup_bwd(built_lib, ids=AT(4)) == 9 and _lookup_bwd(built_lib, ws=AT(16)) == 9
    need = built_lib.pb_embedding_lookup_bwd_workspace_size(3, 10, 8)
    assert need > 0 and _lookup_bwd(built_lib, size=need - 1) == 5
    assert built_lib.pb_embedding_lookup_bwd_workspace_size(3, 0, 8) == 0
    assert _lookup(built_lib, n=0, table=None, ids=None, out=None) == 0


def _xent(lib, x=ONE, outer=1, inner=4, so=0, si=8, depth=8, w=ONE, ld=16, by_word=0, vocab=16, t=ONE, smoothing=0.0, loss=ONE, lse=ONE, ws=ONE, size=1 << 40):
    return lib.pb_linear_xent(x, outer, inner, so, si, depth, w, ld, by_word, vocab, t, smoothing, loss, lse, ws, size, None)


def _xent_bwd(lib, x=ONE, outer=1, inner=4, so=0, si=8, depth=8, w=ONE, ld=16, by_word=0, vocab=16, t=ONE, smoothing=0.0, lse=ONE, g=ONE, dx=ONE, dw=ONE, ws=ONE, size=1 << 40):
    return lib.pb_linear_xent_bwd(x, outer, inner, so, si, depth, w, ld, by_word, vocab, t, smoothing, lse, g, dx, dw, ws, size, None)


def test_cross_entropy(built_lib):
    for name in ("x", "w", "t", "ws"):
        assert _xent(built_lib, **{name: None}) == 1 and _xent_bwd(built_lib, **{name: None}) == 1, name
    assert _xent(built_lib, loss=None) == 1 and _xent(built_lib, lse=None) == 1 and _xent_bwd(built_lib, lse=None) == 1 and _xent_bwd(built_lib, g=None) == 1
    for bad in (dict(outer=-1), dict(inner=-1), dict(so=-8), dict(si=-8), dict(depth=0), dict(vocab=0), dict(ld=15), dict(by_word=1, ld=7), dict(inner=1 << 25), dict(outer=1 << 13, inner=1 << 13),
                dict(smoothing=-0.1), dict(smoothing=1.1), dict(smoothing=float("nan")), dict(depth=1 << 21), dict(vocab=1 << 29, ld=1 << 29)):
        assert _xent(built_lib, **bad) == 2 and _xent_bwd(built_lib, **bad) == 2, bad
    for name, byte in (("x", 1), ("w", 1), ("t", 4), ("ws", 128), ("lse", 2)):
        assert _xent(built_lib, **{name: AT(byte)}) == 9 and _xent_bwd(built_lib, **{name: AT(byte)}) == 9, name
    assert _xent(built_lib, loss=AT(2)) == 9 and _xent_bwd(built_lib, g=AT(2)) == 9 and _xent_bwd(built_lib, dx=AT(1)) == 9 and _xent_bwd(built_lib, dw=AT(1)) == 9
    for backward, call in ((0, _xent), (1, _xent_bwd)):
        need = built_lib.pb_linear_xent_workspace_size(4, 8, ONE, 16, 0, 16, backward)
        assert need > 0 and call(built_lib, size=need - 1) == 5
        # a weight that lies off 16 bytes, or whose rows do, is copied: 8 rows of 16 more
        assert built_lib.pb_linear_xent_workspace_size(4, 8, AT(2), 16, 0, 16, backward) >= need + 8 * 16 * 2 and built_lib.pb_linear_xent_workspace_size(4, 8, ONE, 17, 0, 16, backward) >= need + 8 * 16 * 2
    assert built_lib.pb_linear_xent_workspace_size(4, 0, ONE, 16, 0, 16, 0) == 0
    assert _xent(built_lib, inner=0, x=None, t=None, loss=None, lse=None, ws=None) == 0
    assert _xent_bwd(built_lib, dx=None, dw=None) == 0                    # nothing is asked for


def _ortho(lib, g=ONE, dtype=0, batch=1, rows=200, cols=300, steps=5, co=(3.4445, -4.7750, 2.0315), eps=1e-7, out=ONE, ws=ONE, size=1 << 40):
    numbers = (C.c_float * (3 * max(1, steps if steps < 100 else 1)))(*(co * max(1, steps if steps < 100 else 1))) if co else None
    return lib.pb_orthogonalize(g, dtype, batch, rows, cols, steps, numbers, eps, out, ws, size, None)


def test_orthogonalized_update(built_lib):
    for name in ("g", "co", "out", "ws"):
        assert _ortho(built_lib, **{name: None}) == 1, name
    assert _ortho(built_lib, dtype=2) == 4
    for bad in (dict(batch=0), dict(rows=0), dict(cols=-1), dict(batch=65536), dict(rows=(1 << 24) + 1), dict(steps=0), dict(steps=65, co=(0.0, 0.0, 0.0)), dict(eps=-1.0), dict(eps=float("nan"))):
        assert _ortho(built_lib, **bad) == 2, bad
    assert _ortho(built_lib, g=AT(2)) == 9 and _ortho(built_lib, out=AT(1)) == 9 and _ortho(built_lib, ws=AT(64)) == 9
    need = built_lib.pb_orthogonalize_workspace_size(1, 200, 300)
    assert need > 0 and _ortho(built_lib, size=need - 1) == 5 and built_lib.pb_orthogonalize_workspace_size(1, 0, 3) == 0
    for far in ((9.0, 0.0, 0.0), (3.0, 40.0, -40.0), (float("inf"), 0.0, 0.0), (float("nan"),) * 3, (2.5, 0.0, 0.0)):
        assert _ortho(built_lib, co=far) == 8, far
    assert built_lib.pb_orthogonalize_workspace_size(7, 2048, 128) > 0 and _ortho(built_lib, rows=2048, cols=128, size=1) == 5
