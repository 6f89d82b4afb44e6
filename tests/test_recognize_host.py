"""What OcrEngine.recognize refuses before it touches a page or a device (no GPU needed)."""
import pytest

from pvlc_b200 import model as M


@pytest.mark.parametrize("beams", [0, -1, -4, 33])
def test_numbers_of_beams(beams):
    eng = M.OcrEngine.__new__(M.OcrEngine)
    with pytest.raises(ValueError, match="beams"):
        eng.recognize([], beams=beams)
    with pytest.raises(ValueError, match="beams"):
        eng.recognize([], beams=beams, length_penalty=2.0)
