"""The choice of a token at its edges, against its definition in 64 bits: min-p above 1 among
many equal logits, logits whose differences pass fp32's range."""
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("vocab", [300, 20000])
@pytest.mark.parametrize("settings", [dict(top_k=[7000] * 4), dict(top_p=[0.6] * 4), dict(top_k=[9000] * 4, top_p=[0.7] * 4), {}])
def test_min_p_that_only_the_first_of_the_largest_passes(vocab, settings):
    """Of equal largest logits min-p above 1 leaves the first alone, whichever way the row takes."""
    x = torch.zeros(4, vocab)
    x[1, 5:] = 1.0
    x[2, ::2] = -1.0
    x[3, :-3] = -2.0
    check(x, [0.1, 0.5, 0.9, 0.999], [1.0] * 4, min_p=[2.0, 1.5, 1.0 + 2.0 ** -20, 3.0], **settings)
    check(x, [0.1, 0.5, 0.9, 0.999], [1.0] * 4, min_p=[1.0] * 4, **settings)
