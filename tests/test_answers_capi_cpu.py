"""What the C entries of the log probabilities and of the weights in 4 bits refuse, before they touch a device."""
import ctypes as C

ONE = C.c_void_p(4096)
ODD = C.c_void_p(4099)


def _scores(lib, z=ONE, dtype=0, outer=1, inner=4, so=0, si=8, vocab=8, tokens=ONE, n=1, top=2, lp=ONE, tl=ONE, tt=ONE, stats=ONE):
    return lib.pb_token_logprobs(z, dtype, outer, inner, so, si, vocab, tokens, n, top, lp, ONE, tl, tt, stats, None)


def test_scores(built_lib):
    assert _scores(built_lib, z=None) == 1 and _scores(built_lib, tokens=None) == 1 and _scores(built_lib, lp=None) == 1 and _scores(built_lib, tl=None) == 1 and _scores(built_lib, tt=None) == 1
    assert _scores(built_lib, dtype=2) == 4
    for bad in (dict(vocab=0), dict(vocab=1 << 31), dict(outer=-1), dict(inner=-1), dict(si=-8), dict(so=-8), dict(n=-1), dict(n=129), dict(top=-1), dict(top=9), dict(top=129, vocab=1000),
                dict(outer=1 << 20, inner=1 << 20)):
        assert _scores(built_lib, **bad) == 2, bad
    assert _scores(built_lib, z=ODD) == 9 and _scores(built_lib, stats=C.c_void_p(4100)) == 9
    assert _scores(built_lib, inner=0, z=None) == 0          # no rows: nothing to do


def _gradient(lib, stats=ONE, tt=ONE, top=2, entropy=ONE, g_entropy=ONE, dz=ONE, inner=4):
    return lib.pb_token_logprobs_bwd(ONE, 1, 1, inner, 0, 8, 8, ONE, 1, tt, top, stats, entropy, ONE, g_entropy, ONE, dz, None)


def test_gradient(built_lib):
    assert _gradient(built_lib, stats=None) == 1 and _gradient(built_lib, tt=None) == 1 and _gradient(built_lib, entropy=None) == 1 and _gradient(built_lib, dz=None) == 1
    assert _gradient(built_lib, dz=C.c_void_p(4100)) == 9 and _gradient(built_lib, stats=C.c_void_p(4100)) == 9
    assert _gradient(built_lib, inner=0, dz=None) == 0


def test_quantizer(built_lib):
    f, b = built_lib.pb_quantize_int4, built_lib.pb_dequantize_int4
    assert f(None, 0, 128, 16, 128, ONE, ONE, None, None) == 1 and f(ONE, 0, 128, 16, 128, None, ONE, None, None) == 1 and b(ONE, None, None, 128, 16, 128, ONE, 0, None) == 1
    assert f(ONE, 3, 128, 16, 128, ONE, ONE, None, None) == 4 and b(ONE, ONE, None, 128, 16, 128, ONE, 3, None) == 4
    assert f(ONE, 0, 128, 16, 48, ONE, ONE, None, None) == 3 and b(ONE, ONE, None, 128, 16, 256, ONE, 0, None) == 3
    assert f(ONE, 0, 0, 16, 128, ONE, ONE, None, None) == 2 and b(ONE, ONE, None, 128, -1, 128, ONE, 0, None) == 2
    assert f(ONE, 0, 128, 16, 128, ODD, ONE, None, None) == 9 and b(ODD, ONE, None, 128, 16, 128, ONE, 0, None) == 9
    assert f(ONE, 0, 128, 1 << 23, 128, ONE, ONE, None, None) == 8


def _product(lib, x=ONE, x_dtype=0, rows=2, depth=256, stride=256, q=ONE, scale=ONE, zero=None, group=64, cols=16, out=ONE, out_dtype=0):
    return lib.pb_int4_product(x, x_dtype, rows, depth, stride, q, scale, zero, group, cols, out, out_dtype, None)


def test_product(built_lib):
    for name in ("x", "q", "scale", "out"):
        assert _product(built_lib, **{name: None}) == 1
        assert _product(built_lib, **{name: ODD}) == 9
    assert _product(built_lib, zero=ODD) == 9
    assert _product(built_lib, x_dtype=2) == 4 and _product(built_lib, out_dtype=-1) == 4
    assert _product(built_lib, group=0) == 3
    for bad in (dict(rows=-1), dict(depth=0), dict(cols=0), dict(stride=-1), dict(depth=1 << 31), dict(cols=1 << 30), dict(depth=1 << 30, cols=1 << 29)):
        assert _product(built_lib, **bad) == 2, bad
    assert _product(built_lib, rows=0, x=None) == 0


def test_a_weights_parts_lie_where_a_lane_loads_them_from(built_lib):
    """Four scales of a group of 32 come as eight bytes, two of a group of 64 as four; the zero points of each are half of that."""
    at = lambda byte: C.c_void_p(4096 + byte)
    for byte in (2, 4, 6):
        assert _product(built_lib, scale=at(byte), group=32) == 9, byte
    assert _product(built_lib, scale=at(2), group=64) == 9 and _product(built_lib, scale=at(1), group=128) == 9
    for byte in (1, 2, 3):
        assert _product(built_lib, zero=at(byte), group=32) == 9, byte
    assert _product(built_lib, zero=at(1), group=64) == 9


def test_every_array_lies_at_its_types_bytes(built_lib):
    """Nothing reaches a kernel that would load or store across an element."""
    at = lambda byte: C.c_void_p(4096 + byte)
    f, b = built_lib.pb_quantize_int4, built_lib.pb_dequantize_int4
    assert f(at(2), 0, 128, 16, 128, ONE, ONE, None, None) == 9 and f(at(1), 1, 128, 16, 128, ONE, ONE, None, None) == 9 and f(ONE, 0, 128, 16, 128, ONE, at(1), None, None) == 9
    assert b(ONE, at(1), None, 128, 16, 128, ONE, 0, None) == 9 and b(ONE, ONE, None, 128, 16, 128, at(2), 0, None) == 9 and b(ONE, ONE, None, 128, 16, 128, at(1), 1, None) == 9
    for name, byte in (("z", 2), ("tokens", 4), ("lp", 2), ("tl", 2), ("tt", 4), ("stats", 4)):
        assert _scores(built_lib, **{name: at(byte)}) == 9, name
    assert built_lib.pb_token_logprobs(ONE, 0, 1, 4, 0, 8, 8, ONE, 1, 2, ONE, at(2), ONE, ONE, None, None) == 9          # the entropy
    arrays = dict(z=ONE, tokens=ONE, tt=ONE, stats=ONE, entropy=ONE, g_logprobs=ONE, g_entropy=ONE, g_top=ONE, dz=ONE)
    for name, byte in (("z", 1), ("tokens", 4), ("tt", 4), ("stats", 4), ("entropy", 2), ("g_logprobs", 2), ("g_entropy", 2), ("g_top", 2), ("dz", 8)):
        a = {**arrays, name: at(byte)}
        assert built_lib.pb_token_logprobs_bwd(a["z"], 1, 1, 4, 0, 8, 8, a["tokens"], 1, a["tt"], 2, a["stats"], a["entropy"], a["g_logprobs"], a["g_entropy"], a["g_top"], a["dz"], None) == 9, name
