"""Rows, slots and logits more than 2^32 elements apart: the same kernels on the same
values give the same bits wherever those lie."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def apart(x, step):
    """x with `step` elements from one of its rows to the next."""
    room = torch.empty((x.shape[0] - 1) * step + x[0].numel(), dtype=x.dtype, device=x.device)
    y = room.as_strided(x.shape, (step, *x.stride()[1:]))
    return y.copy_(x)


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("takes 60 GB")
    yield
    torch.cuda.empty_cache()


def batch(new, slots):
    from inferno_hip import device as D
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    return D.StateBatch(ints(starts), ints(slots), starts[-1], kv_lens=ints([n if i % 2 else n + 7 for i, n in enumerate(new)]))


def test_the_convolution():
    from inferno_hip import device as D
    g = torch.Generator("cuda").manual_seed(1)
    new, slots = [1, 40, 3, 33], [36, 0, 20, 35]
    x = torch.randn(sum(new), 64, device="cuda", generator=g).bfloat16()
    w, state = torch.randn(64, 4, device="cuda", generator=g), torch.randn(37, 3, 64, device="cuda", generator=g)
    far = apart(x, 1 << 26), apart(state, 1 << 27)
    assert far[0].stride(0) * (sum(new) - 1) > 1 << 32 and far[1].stride(0) * 36 > 1 << 32
    b = batch(new, slots)
    assert torch.equal(D.short_conv(x, w, state, b), D.short_conv(far[0], w, far[1], b))
    assert torch.equal(state, far[1])


@pytest.mark.parametrize("new", [[1, 8, 3, 68, 1], [70, 3, 2, 1, 9]])
def test_the_delta_rule(new):
    from inferno_hip import device as D
    g = torch.Generator("cuda").manual_seed(2)
    K, H, dk, dv, T = 2, 4, 64, 32, sum(new)
    x = torch.randn(T, 2 * K * dk + H * dv, device="cuda", generator=g).bfloat16()
    ab, z = torch.randn(T, 2 * H, device="cuda", generator=g), torch.randn(T, H, dv, device="cuda", generator=g)
    state = torch.randn(35, H, dk, dv, device="cuda", generator=g)
    decay, dt, norm = -torch.rand(H, device="cuda"), torch.randn(H, device="cuda"), torch.rand(dv, device="cuda")
    b = batch(new, [34, 0, 33, 17, 1])

    def run(x, ab, z, state):
        q, k = (x[:, i * K * dk:(i + 1) * K * dk].unflatten(1, (K, dk)) for i in (0, 1))
        v = x[:, 2 * K * dk:].unflatten(1, (H, dv))
        return D.gated_delta(q, k, v, ab[:, :H], ab[:, H:], D.DeltaLayer(state, K, decay, dt, norm_w=norm), b, gate=z)

    far = apart(x, 1 << 26), apart(ab, 1 << 26), apart(z, 1 << 26), apart(state, 1 << 27)
    assert far[0].stride(0) * (T - 1) > 1 << 32 and far[3].stride(0) * 34 > 1 << 32
    assert torch.equal(run(x, ab, z, state), run(*far))
    assert torch.equal(state, far[3])


def test_sampling():
    from inferno_hip import device as D
    g = torch.Generator("cuda").manual_seed(3)
    n, vocab = 20, 40001
    l, u = 3 * torch.randn(n, vocab, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    far = apart(l, (1 << 28) + 1)
    assert far.stride(0) * (n - 1) > 1 << 32
    t = torch.linspace(0.5, 1.5, n, device="cuda")
    for kw in (dict(), dict(top_k=ints([50] * n), top_p=torch.full((n,), 0.9, device="cuda")),
               dict(min_p=torch.full((n,), 0.01, device="cuda"))):
        lp = [torch.zeros(n, device="cuda") for _ in range(2)]
        assert torch.equal(D.sample(l, u, temperature=t, logprobs=lp[0], **kw), D.sample(far, u, temperature=t, logprobs=lp[1], **kw))
        assert torch.equal(*lp)
