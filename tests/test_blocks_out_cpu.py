"""Which blocks `quantize` writes a matrix into: the host's checks, on CPU tensors."""
import pytest

torch = pytest.importorskip("torch")

from gsx_amd import fields  # noqa: E402
from gsx_amd._lib import GsxHipError  # noqa: E402


def _blocks(rows, wide, words, cols):
    return fields.Blocks(torch.zeros(rows, wide, dtype=torch.uint8), torch.zeros(rows, words, dtype=torch.uint8), cols)


def _room(out, rows=3, cols=130):
    return fields._blocks_room(fields.Blocks, 128, 128, rows, cols, out, "cpu")


def test_room_for_whole_blocks(monkeypatch):
    monkeypatch.setattr(fields, "_device", lambda: -1)  # where CPU tensors say they live
    new, args = _room(None)
    assert new.values.shape == (3, 256) and new.exponents.shape == (3, 4) and new.cols == 130
    assert _room(new) == (new, args) and args == new.arguments()
    wide = fields.Blocks(torch.zeros(3, 512, dtype=torch.uint8)[:, 16:288], torch.zeros(3, 12, dtype=torch.uint8)[:, 4:9], 130)
    result, args = _room(wide)
    assert result is wide and args == (wide.values.data_ptr(), 512, wide.exponents.data_ptr(), 12)


@pytest.mark.parametrize("rows,wide,words,cols", [(2, 256, 4, 130), (3, 256, 4, 129), (3, 240, 4, 130), (3, 256, 3, 130)])
def test_refused(rows, wide, words, cols):
    with pytest.raises(GsxHipError):
        _room(_blocks(rows, wide, words, cols))


def test_refused_kinds():
    four = fields.Blocks4(torch.zeros(3, 256, dtype=torch.uint8), torch.zeros(3, 8, dtype=torch.uint8), 130)
    flat = fields.Blocks(torch.zeros(3, dtype=torch.uint8), torch.zeros(3, dtype=torch.uint8), 130)
    for out in (four, four.values, flat):
        with pytest.raises(GsxHipError):
            _room(out)
