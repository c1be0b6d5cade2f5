"""The single-token operators without a GPU: the C ABI refuses bad arguments before any launch, the Python entry points
refuse what the kernels cannot take, and rope_axes says which axis turns which frequency."""

from __future__ import annotations

import ctypes

import pytest
import torch

from jeff_b200 import _lib, kernels
from jeff_b200 import constants as C

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)   # not 16-byte aligned


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    from jeff_b200 import build

    build.build()
    return _lib.load()


def _tables(lib, **over):
    a = dict(b=4, free=P, free_count=8, stride=60, width=60, entry=50, page=32, fixed=0, tokens=4) | over
    return lib.jb_block_tables(P, P, a["b"], a["free"], a["free_count"], P, a["stride"], a["width"], a["entry"],
                               a["page"], a["fixed"], a["tokens"], P, P, P, P, P, None)


def _prep(lib, **over):
    a = dict(pr=P, w1=P, ldpr=5120, t=3, stride=3, kn=P, vn=P, kv=None, pages=0, page_bytes=0, layer=0, layers=0,
             slots=None) | over
    return lib.jb_attn_prep_axes(a["pr"], a["ldpr"], a["t"], a["w1"], P, P, P, a["stride"], 0, P, a["kn"], a["vn"], a["kv"],
                                 a["pages"], a["page_bytes"], a["layer"], a["layers"], a["slots"], None)


def _decode(lib, **over):
    a = dict(q=P, ldq=2048, pages=10, page_bytes=393216, layer=0, layers=6, stride=60, width=60, entry=50, b=2, heads=8,
             kv_heads=2, dim=256, pr=None, ldpr=0, ldy=2048) | over
    return lib.jb_decode_attention(a["q"], a["ldq"], P, a["pages"], a["page_bytes"], a["layer"], a["layers"], P,
                                   a["stride"], a["width"], a["entry"], P, a["b"], a["heads"], a["kv_heads"], a["dim"],
                                   1.0, a["pr"], a["ldpr"], P, a["ldy"], None, 0, None)


def _scan(lib, **over):
    a = dict(q=P, row=2048, tok=2048, b=2, n=5, heads=16, page_bytes=393216, per=6, first=0, stride=50, out=None,
             out_stride=0) | over
    return lib.jb_linear_scan(a["q"], a["row"], a["tok"], P, 2048, 2048, P, 2048, 2048, P, 0, 0, None, P, a["b"],
                              a["n"], a["heads"], P, 100, a["page_bytes"], a["per"], a["first"], P, a["stride"],
                              a["out"], a["out_stride"], None, 0, None)


def _step(lib, **over):
    a = dict(out=P, row=2048, per=6, first=0) | over
    return lib.jb_linear_step(P, a["row"], P, 2048, P, 2048, P, 16, None, P, 2, 16, P, 100, 393216, a["per"],
                              a["first"], P, 50, a["out"], 50, None)


@pytest.mark.parametrize(("call", "over", "says"), [
    (_tables, {"b": 0}, b"0 rows"),
    (_tables, {"tokens": 0}, b"0 tokens"),
    (_tables, {"free": None}, b"free list"),
    (_tables, {"free_count": -1}, b"free list"),
    (_tables, {"entry": 60}, b"entry 60"),
    (_tables, {"width": 61}, b"61 wide"),
    (_tables, {"page": 0}, b"pages of 0"),
    (_prep, {"t": 0}, b"t 0"),
    (_prep, {"ldpr": 5112}, b"ldpr 5112"),
    (_prep, {"ldpr": 5121}, b"ldpr 5121"),
    (_prep, {"pr": ODD}, b"aligned"),
    (_prep, {"w1": ODD}, b"aligned"),
    (_prep, {"vn": None}, b"keys and values"),
    (_prep, {"kn": None, "vn": None}, b"keys and values"),
    (_prep, {"kv": P, "pages": 4, "page_bytes": 393216, "layers": 6}, b"keys and values"),
    (_prep, {"kv": P, "slots": P, "pages": 4, "page_bytes": 393216, "layer": 6, "layers": 6}, b"layer 6 of 6"),
    (_prep, {"kv": P, "slots": P, "pages": 4, "page_bytes": 393200, "layers": 6}, b"does not fit"),
    (_decode, {"dim": 96}, b"heads of 96"),
    (_decode, {"heads": 9}, b"9 query heads"),
    (_decode, {"heads": 34}, b"at most 16"),
    (_decode, {"b": 0}, b"0 rows"),
    (_decode, {"layer": 6}, b"layer 6 of 6"),
    (_decode, {"page_bytes": 1024}, b"does not fit"),
    (_decode, {"entry": 61}, b"entry 61"),
    (_decode, {"stride": 59}, b"60 wide"),
    (_decode, {"ldq": 2044}, b"row strides"),
    (_decode, {"pr": P, "ldpr": 2048}, b"row strides"),
    (_decode, {"q": ODD}, b"aligned"),
    (_decode, {"heads": 8}, b"a scratch of 0 floats"),
    (_scan, {"n": 0}, b"0 tokens"),
    (_scan, {"heads": 0}, b"0 heads"),
    (_scan, {"tok": 2044}, b"multiples of 8"),
    (_scan, {"q": ODD}, b"aligned"),
    (_scan, {"n": 1000}, b"a scratch of 0 floats"),
    (_scan, {"per": 7}, b"7 heads per page"),
    (_scan, {"first": 285}, b"past the block table"),
    (_scan, {"out": P, "out_stride": 2}, b"past the block table"),
    (_step, {"out": None}, b"out_tables"),
    (_step, {"first": -16}, b"past the block table"),
])
def test_bad_arguments_are_refused_before_any_launch(lib, call, over, says) -> None:
    assert call(lib, **over) == -1
    assert says in lib.jb_last_error()


def test_block_tables_refuses_more_than_its_indices_hold(lib) -> None:
    for count in (2 ** 31 - 1, 0x7f000001):
        assert _tables(lib, tokens=count) == -1
        assert b"%d tokens" % count in lib.jb_last_error()
        assert _tables(lib, b=count) == -1
        assert b"%d rows" % count in lib.jb_last_error()


@pytest.mark.parametrize(("over", "says"), [
    ({"width": 2 ** 26, "stride": 2 ** 26, "entry": 0}, b"tables of 2147483648 tokens"),
    ({"width": 0x3f80002, "stride": 0x3f80002, "entry": 1}, b"tables of 2130706464 tokens"),
    ({"width": 0x3f80000, "stride": 0x3f80000, "entry": 0, "heads": 512, "kv_heads": 256, "dim": 64,
      "page_bytes": 2 ** 24, "ldq": 2 ** 15, "ldy": 2 ** 15}, b"256 key/value heads"),
    ({"heads": 2 ** 23, "kv_heads": 2 ** 20, "page_bytes": 2 ** 50}, b"2 rows of 8388608 heads of 256"),
    ({"b": 0x7f000001, "heads": 1, "kv_heads": 1}, b"2130706433 rows"),
])
def test_decode_attention_refuses_more_than_its_indices_hold(lib, over, says) -> None:
    assert _decode(lib, **over) == -1
    assert says in lib.jb_last_error()


def test_scratch_sizes(lib) -> None:
    """Two cut rows' flags and parts a share; a state and its decay for each of a long row's segments, which all run at once, and
    none for rows that stay whole."""
    assert lib.jb_decode_attention_scratch(8, 2, 256) == 2 * 148 * (2 + 4 * 258)
    assert lib.jb_decode_attention_scratch(34, 2, 256) == lib.jb_decode_attention_scratch(8, 0, 256) == 0
    for b, heads, n in ((1, 16, 1000), (2, 16, 8192), (1, 1, 100000), (100, 1, 4096)):
        floats = lib.jb_linear_scan_scratch(b, heads, n)
        count, rest = divmod(floats, b * heads * (128 * 128 + 1))
        assert rest == 0 and 2 <= count and b * heads * count <= 296
    for b, heads, n in ((1, 16, 1), (1, 16, 64), (64, 16, 128), (300, 1, 8192), (0, 16, 64)):
        assert lib.jb_linear_scan_scratch(b, heads, n) == 0


def test_no_scratch_size_for_heads_that_are_refused(lib) -> None:
    for heads, kv_heads, dim in ((9, 2, 256), (8, 2, 96), (8, 2, 32), (0, 2, 64), (1, 2, 64), (17, 1, 64)):
        assert lib.jb_decode_attention_scratch(heads, kv_heads, dim) == 0
        assert _decode(lib, heads=heads, kv_heads=kv_heads, dim=dim) == -1
    for dim in (64, 128, 256):
        assert lib.jb_decode_attention_scratch(16, 1, dim) > lib.jb_decode_attention_scratch(4, 2, dim) > 0


def test_rope_axes() -> None:
    def of(axes: int) -> list[int]:
        return [axes >> 2 * i & 3 for i in range(32)]

    assert of(kernels.rope_axes((32,))) == [0] * 32
    assert of(kernels.rope_axes((8, 12, 12))) == [0] * 8 + [1] * 12 + [2] * 12
    assert of(kernels.rope_axes((11, 11, 10), True)) == [i % 3 for i in range(32)]
    assert of(kernels.rope_axes((12, 10, 10), True)) == [i % 3 for i in range(30)] + [0, 0]
    assert of(kernels.rope_axes((0, 0, 0, 32))) == [3] * 32
    for bad in ((), (16, 15), (40, -8), (8, 8, 8, 4, 4)):
        with pytest.raises(ValueError, match="sections"):
            kernels.rope_axes(bad)


def _kv(pages: int = 3) -> torch.Tensor:
    return torch.zeros(pages, 6, 2, 32, 2, 256, dtype=torch.bfloat16)


def _decode_args() -> dict:
    return dict(q=torch.zeros(2, 8, 256, dtype=torch.bfloat16), kv=_kv(), tables=torch.zeros(2, 60, dtype=torch.int32),
                attn_layer=0, lengths=torch.zeros(2, dtype=torch.int32), kv_entry=50)


def _linear_args() -> dict:
    x = torch.zeros(2, 5, 16, 128, dtype=torch.bfloat16)
    return dict(q=x, k=x, v=x, g=torch.zeros(2, 5, 16), state=torch.zeros(4, 6, 128, 128),
                tables=torch.zeros(2, 50, dtype=torch.int32), layer=0)


def _tables_args() -> dict:
    i = torch.zeros(2, dtype=torch.int32)
    return dict(lengths=i, new=i, free=i, tables=torch.zeros(2, 60, dtype=torch.int32), kv_entry=50, tokens=4)


def _prep_args() -> dict:
    w = torch.ones(C.HD)
    return dict(pr=torch.zeros(3, C.ATTN_PROJ, dtype=torch.bfloat16), q_w1=w, k_w1=w, inv_freq=torch.ones(32),
                positions=torch.zeros(3, 3, dtype=torch.int32), axes=kernels.rope_axes((11, 11, 10)), kv=_kv(),
                slots=torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize(("entry", "args", "over", "says"), [
    (kernels.decode_attention, _decode_args, {}, "expected a CUDA tensor"),
    (kernels.decode_attention, _decode_args, {"q": torch.zeros(2, 8, 256)}, "q: expected torch.bfloat16"),
    (kernels.decode_attention, _decode_args, {"q": torch.zeros(2, 2048)}, "q: expected"),
    (kernels.linear_scan, _linear_args, {}, "expected a CUDA tensor"),
    (kernels.linear_scan, _linear_args, {"q": torch.zeros(2, 16, 128)}, "q: expected"),
    (kernels.linear_step, _linear_args, {}, "q: expected"),
    (kernels.block_tables, _tables_args, {}, "expected a CUDA tensor"),
    (kernels.block_tables, _tables_args, {"lengths": torch.zeros(2, 2, dtype=torch.int32)}, "lengths: expected"),
    (kernels.attn_prep_axes, _prep_args, {}, "expected a CUDA tensor"),
    (kernels.attn_prep_axes, _prep_args, {"pr": torch.zeros(3, 100)}, "pr: expected"),
])
def test_entry_points_refuse(entry, args, over, says) -> None:
    with pytest.raises(ValueError, match=says):
        entry(**(args() | over))
