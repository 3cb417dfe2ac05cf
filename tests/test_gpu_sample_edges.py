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


@pytest.mark.parametrize("t", [5e37, 3e38])
def test_logits_whose_differences_pass_the_range(t):
    """Logits near either end of fp32, at temperatures as large: their differences do not fit fp32, their weights do."""
    g = torch.Generator().manual_seed(9)
    x = 3.3e38 * torch.sign(torch.rand(6, 3000, generator=g) - 0.5) * (0.9 + 0.1 * torch.rand(6, 3000, generator=g))
    x[0, ::3] = 0.0
    x[1, 100:] = -3.4e38
    x[2] = -3.4e38
    x[2, 7] = 3.4e38
    u = [0.05, 0.999, 0.99, 0.5, 0.7, 0.9]
    check(x, u, [t] * 6, [2000, 500, 40, 1600, 2500, 1400])
    check(x, u, [t] * 6, None, [0.99, 0.9, 0.9999, 0.999, 0.7, 0.5])
    check(x, u, [t] * 6, [1600] * 6, [0.999] * 6)


@pytest.mark.parametrize("u", [1.0, 7.0])
def test_the_last_kept_token_hardly_weighs(u):
    """Where no sum passes u of all, the last kept token is taken, also one of 2^-65 of the weights in a slice of its own."""
    x = torch.full((3, 20000), -100.0)
    x[:, 3] = 0.0
    x[0, 19000], x[1, 9000], x[2, 100] = -45.0, -45.0, -45.0
    check(x, [u] * 3, [1.0] * 3, [2] * 3)
    check(x, [u] * 3, [1.0] * 3, [3] * 3, [1.0] * 3)
    check(x, [u] * 3, [1.0] * 3)
