"""The block norm's spec as the ops pack it is hsmoe_block_norm_spec as ctypes lays it out (no GPU needed)."""
import ctypes

import pytest
import torch

from home_seek_amd import _lib, ops

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,stream,weights,gates", ((BF16, F32, BF16, F32), (F32, BF16, BF16, BF16), (BF16, BF16, F32, BF16),
                                                       (BF16, BF16, BF16, F32)))
def test_packed_as_the_struct(rows, stream, weights, gates):
    kinds = {BF16: _lib.OUT_BF16, F32: _lib.OUT_F32}
    f, post, pre = torch.zeros(3, 64, dtype=rows), torch.zeros(64, dtype=weights), torch.zeros(64, dtype=weights)
    for form, shape in ((_lib.GATE_CHANNEL, (64,)), (_lib.GATE_TOKEN, (3, 1)), (_lib.GATE_FULL, (3, 64))):
        packed, got, (a, b, g) = ops._block_norm_spec(f, stream, post, torch.zeros(shape, dtype=gates), pre)
        assert len(packed) == ctypes.sizeof(_lib.BlockNormSpec) and got == form
        s = _lib.BlockNormSpec.from_buffer_copy(packed)
        assert (s.post_w_dev, s.pre_w_dev, s.gate_dev) == (a.data_ptr(), b.data_ptr(), g.data_ptr())
        assert len({s.post_w_dev, s.pre_w_dev, s.gate_dev}) == 3
        assert (s.row_kind, s.stream_kind, s.weight_kind, s.gate_kind, s.gate_form) == (kinds[rows], kinds[stream], kinds[weights], kinds[gates], form)
    packed, form, _ = ops._block_norm_spec(f, stream, None, None, None)
    s = _lib.BlockNormSpec.from_buffer_copy(packed)
    assert (s.post_w_dev, s.pre_w_dev, s.gate_dev, s.gate_form, form) == (None, None, None, _lib.GATE_NONE, _lib.GATE_NONE)


def test_the_header_has_the_same_fields():
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "hsmoe.h").read_text()
    body = re.search(r"typedef struct \{([^}]*)\} hsmoe_block_norm_spec;", text).group(1)
    names = []
    for line in body.split(";"):
        pointer = re.match(r"\s*const void\*\s*(\w+)", line)
        if pointer:
            names.append((pointer.group(1), ctypes.c_void_p))
        elif line.strip():
            names += [(n.strip(), ctypes.c_int) for n in re.match(r"\s*int\s+(.*)", line, re.S).group(1).split(",")]
    assert names == _lib.BlockNormSpec._fields_
