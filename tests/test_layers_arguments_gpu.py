"""Arguments of the calls around the head that are refused in a way of their own."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [1 << 63, 1 << 64, 1 << 70, -(1 << 70), (1 << 64) + 5])
def test_a_first_id_beyond_every_word(cuda, lily, first):
    scratch = lily.SamplerScratch(1000, max_rows=1)
    logits = cuda.zeros((1, 1000), device="cuda")
    with pytest.raises(lily.LilyError, match="first_id") as e:
        scratch.adjust_logits(logits, first_id=first)
    assert e.value.code == lily.ERR_ARG
