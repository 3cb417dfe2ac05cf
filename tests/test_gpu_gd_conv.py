"""The short convolution against its definition in 64 bits: lengths from none to over a
tile, sequences that begin and go on, every width and type, slices of wider rows,
slots that no sequence may touch."""
import pytest

import gd_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts_of(new, first=0):
    s = [first]
    for n in new:
        s.append(s[-1] + n)
    return s


def case(seed, new, begins, C, W, act, out_type, bias, first=0, pad=0, scale=1.0, wide=0):
    g = torch.Generator().manual_seed(seed)
    starts = starts_of(new, first)
    T, n = starts[-1] + pad, len(new)
    x = (scale * torch.randn(T, C + wide, generator=g)).to(act)
    slots = torch.randperm(n + 2, generator=g)[:n].tolist()
    state = scale * torch.randn(n + 2, W - 1, C, generator=g)
    for s, b in zip(slots, begins):
        if b:
            state[s] = float("nan")
    return dict(x=x, w=torch.randn(C, W, generator=g), bias=torch.randn(C, generator=g) if bias else None, state=state,
                new=new, begins=begins, slots=slots, starts=starts, out=torch.full((T, C), -7.0).to(out_type), wide=wide)


def check(c, silu=True):
    from inferno_hip import device as D
    C = c["w"].shape[0]
    lens = [n if b else n + 5 for n, b in zip(c["new"], c["begins"])]
    batch = D.StateBatch(ints(c["starts"]), ints(c["slots"]), c["x"].shape[0], kv_lens=ints(lens))
    state, out, flags = c["state"].cuda(), c["out"].cuda(), ints([0])
    x = c["x"].cuda()[:, c["wide"]:]
    D.short_conv(x, c["w"].cuda(), state, batch, bias=None if c["bias"] is None else c["bias"].cuda(), silu=silu, out=out,
                 flags=flags)
    y, held, tol = gd_plain.conv(c["x"][:, c["wide"]:], c["w"], c["bias"], silu, c["state"], c["new"], c["begins"], c["slots"],
                                 c["starts"], c["out"])
    got = out.cpu().double()
    assert bool(((got - y).abs() <= tol).all()), float(((got - y).abs() - tol).max())
    # a sequence without new tokens keeps even a slot of NaN
    assert torch.equal(state.cpu().double().nan_to_num(12345.0), held.nan_to_num(12345.0))
    assert int(flags.item()) == 0 and C == out.shape[1]


@pytest.mark.parametrize("act,out_type", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                          ("bf16", "f32")])
@pytest.mark.parametrize("W", [2, 3, 4, 8])
def test_lengths_and_types(W, act, out_type):
    print("[case]", W, act, out_type, flush=True)
    new = [1, 0, 2, 31, 32, 33, 7, 64, 100, 3]
    check(case(W, new, [i % 3 == 0 for i in range(len(new))], 1032, W, TYPES[act], TYPES[out_type], W % 2 == 0, first=3, pad=5))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_tiles_of_32_tokens(act):
    """From 1024 workgroups on; fewer take tiles of 16."""
    new = [15, 16, 17, 1, 31, 32, 33, 0, 32768, 65]
    check(case(21, new, [i % 2 == 0 for i in range(len(new))], 24, 4, TYPES[act], TYPES[act], True, first=2, pad=3))


@pytest.mark.parametrize("W", [5, 6, 7])
def test_other_widths_and_no_silu(W):
    check(case(W, [1, 70, W - 2], [False, True, False], 40, W, F32, F32, True), silu=False)


def test_one_channel_block_and_single_tokens():
    for C in (8, 2048):
        check(case(C, [1] * 70, [i % 5 == 0 for i in range(70)], C, 4, F32, F32, False, pad=2))


def test_rows_of_a_wider_projection():
    check(case(3, [5, 40], [False, True], 64, 4, F32, BF16, False, wide=72))
    check(case(4, [5, 40], [False, True], 64, 4, F16, F16, True, wide=8))


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_sizes_of_values(scale):
    c = case(8, [3, 34], [False, True], 16, 4, F32, F32, False, scale=scale)
    c["w"] *= 1e-3
    check(c, silu=scale < 1)


def test_slots_that_are_not_a_sequences_own():
    """A slot outside the pool, and one that an earlier sequence with new tokens has, are left out and reported; an
    earlier sequence without new tokens does not count."""
    from inferno_hip import _lib
    from inferno_hip import device as D
    x, w = torch.randn(12, 16, device="cuda"), torch.randn(16, 4, device="cuda")
    state = torch.randn(3, 3, 16, device="cuda")
    for slots, new, left_out in (([0, 1, 0], [4, 4, 4], [2]), ([0, 3, 1], [4, 4, 4], [1]), ([-1, 1, 2], [4, 4, 4], [0]),
                                 ([2, 2, 1], [0, 6, 6], [])):
        starts = starts_of(new)
        s, out, flags = state.clone(), torch.full((12, 16), -7.0, device="cuda"), ints([0])
        D.short_conv(x, w, s, D.StateBatch(ints(starts), ints(slots), 12), out=out, flags=flags)
        mine = [-1 if i in left_out else v for i, v in enumerate(slots)]
        y, held, tol = gd_plain.conv(x.cpu(), w.cpu(), None, True, state.cpu(), new, [False] * 3, mine, starts,
                                     torch.full((12, 16), -7.0))
        assert bool(((out.cpu().double() - y).abs() <= tol).all()) and torch.equal(s.cpu().double(), held)
        assert int(flags.item()) == (_lib.FLAG_STATE_SLOT if left_out else 0)


def test_ranges_that_do_not_fit_are_cut():
    from inferno_hip import _lib
    from inferno_hip import device as D
    x, w = torch.randn(6, 16, device="cuda"), torch.randn(16, 4, device="cuda")
    for starts, lens in (([0, 4, 9], None), ([-3, 4, 6], None), ([0, 5, 2], None), ([0, 3, 6], [2, 9])):
        out, flags = torch.full((8, 16), -7.0, device="cuda"), ints([0])
        D.short_conv(x, w, torch.zeros(2, 3, 16, device="cuda"), D.StateBatch(ints(starts), ints([0, 1]), 6,
                                                                              kv_lens=None if lens is None else ints(lens)),
                     out=out[:6], flags=flags)
        assert bool((out[6:] == -7).all()) and int(flags.item()) & _lib.FLAG_KV_LENGTH
