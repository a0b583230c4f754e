"""Rotary positions and norms with the rotation in one pass, against 64 bits."""
import math

import pytest
import torch

import primitiv_b200 as pb
from attention_lib import F32, MODES, rotary, store_rounding

pytestmark = pytest.mark.gpu
PAIRS, HALVES = pb.ROTARY_PAIRS, pb.ROTARY_HALVES


def inputs(shape, dtype, seed, ld_extra=0, shift=0):
    """[tokens, heads, head] with `ld_extra` more elements per token, starting `shift` elements into an allocation."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, h, d = shape
    ld = h * d + ld_extra
    flat = torch.randn(t * ld + shift + 64, device="cuda", generator=g).to(dtype)
    return flat[shift:].as_strided((t, h, d), (ld, d, 1)), ld


def turn_bound(x, dtype, amplitude):
    """Angles are right to 2^-25 of a turn (2 pi 2^-25 = 3.2 F32 2), sine and cosine to 2 units, products and the sum to one each."""
    store, tiny = store_rounding(dtype)
    size = abs(x).amax(-1, keepdim=True) * 2 * amplitude
    return size * 16 * F32 + store * size + tiny


# (tokens, heads, head, rot, layout, extra elements per token, offset of the first element)
SHAPES = [
    (1, 1, 2, 2, PAIRS, 0, 0), (1, 1, 1, 0, PAIRS, 0, 0), (3, 5, 64, 64, HALVES, 0, 0), (37, 3, 80, 20, HALVES, 0, 0),
    (37, 3, 80, 20, PAIRS, 7, 1), (129, 2, 128, 128, HALVES, 256, 0), (5, 40, 128, 32, PAIRS, 0, 0), (65, 7, 255, 254, HALVES, 1, 1),
    (9, 2, 256, 256, HALVES, 0, 2), (9, 2, 256, 250, PAIRS, 0, 0), (2, 3, 33, 6, HALVES, 0, 0), (4, 300, 16, 16, HALVES, 0, 0),
    (1000, 6, 48, 48, PAIRS, 48, 4), (7, 3, 96, 0, HALVES, 0, 0), (66, 2, 254, 252, HALVES, 0, 0), (64, 2, 250, 250, PAIRS, 0, 0),
]


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(ctx, mode, shape):
    t, h, d, rot, layout, extra, shift = shape
    code, dtype = MODES[mode][:2]
    x, ld = inputs((t, h, d), dtype, 1, extra, shift)
    positions = torch.randint(0, 1 << 20, (t,), device="cuda", dtype=torch.int32)
    freqs, amplitude = pb.rotary_frequencies(rot, 10000.0, "by_parts", 4.0, 512.0) if rot else ([], 1.0)
    f = torch.tensor(freqs + [0.0], device="cuda", dtype=torch.float64)
    angles = positions.double()[:, None] * f[:rot // 2]
    y = torch.full((t, h + 1, d), 7.0, device="cuda", dtype=dtype)
    ctx.rotary_fw(code, x.data_ptr(), y.data_ptr(), d, h, t, ld, (h + 1) * d, rot, layout, f.data_ptr(), amplitude, positions.data_ptr())
    want = rotary(x.double(), angles, amplitude, rot, layout)
    assert (abs(y[:, :h].double() - want) <= turn_bound(x.double(), dtype, amplitude)).all()
    assert (y[:, h:] == 7.0).all()
    assert torch.equal(y[:, :h][..., rot:], x[..., rot:])
    # gradient: the transposed map, added
    gx = torch.full((t, h, d), 0.5, device="cuda", dtype=dtype)
    ctx.rotary_bw(code, x.data_ptr(), gx.data_ptr(), d, h, t, ld, 0, rot, layout, f.data_ptr(), amplitude, positions.data_ptr(), accumulate=True)
    want = rotary(x.double(), angles, amplitude, rot, layout, back=True) + 0.5
    store = store_rounding(dtype)[0]
    assert (abs(gx.double() - want) <= turn_bound(x.double(), dtype, amplitude) + 0.5 * store + F32).all()
    # in place: the same bits
    once = torch.empty((t, h, d), device="cuda", dtype=dtype)
    ctx.rotary_fw(code, x.data_ptr(), once.data_ptr(), d, h, t, ld, 0, rot, layout, f.data_ptr(), amplitude, positions.data_ptr())
    ctx.rotary_fw(code, x.data_ptr(), x.data_ptr(), d, h, t, ld, ld, rot, layout, f.data_ptr(), amplitude, positions.data_ptr())
    assert torch.equal(once, x)


def test_positions_that_are_not_given_count_from_zero(ctx):
    t, h, d = 70, 3, 64
    x, ld = inputs((t, h, d), torch.float32, 2)
    f = torch.tensor(pb.rotary_frequencies(d)[0], device="cuda", dtype=torch.float64)
    a, b = torch.empty_like(x), torch.empty_like(x)
    at = torch.arange(t, device="cuda", dtype=torch.int32)
    ctx.rotary_fw(0, x.data_ptr(), a.data_ptr(), d, h, t, 0, 0, d, HALVES, f.data_ptr())
    ctx.rotary_fw(0, x.data_ptr(), b.data_ptr(), d, h, t, 0, 0, d, HALVES, f.data_ptr(), positions=at.data_ptr())
    assert torch.equal(a, b)


def test_far_positions_keep_their_precision(ctx):
    t, h, d = 4, 1, 8
    x = torch.ones((t, h, d), device="cuda")
    at = torch.tensor([4294967295 - (1 << 32), 2147483647, 16777217, 999999937], device="cuda", dtype=torch.int32)
    f = torch.tensor(pb.rotary_frequencies(d)[0], device="cuda", dtype=torch.float64)
    y = torch.empty_like(x)
    ctx.rotary_fw(0, x.data_ptr(), y.data_ptr(), d, h, t, 0, 0, d, PAIRS, f.data_ptr(), positions=at.data_ptr())
    pos = at.long() & 0xffffffff
    want = rotary(x.double(), pos.double()[:, None] * f, 1.0, d, PAIRS)
    # the angle itself, of 2^32 radians in 64 bits, is right to 2^32 2^-52
    assert (abs(y.double() - want) <= 2 * 16 * F32 + 2.0 ** -19).all()


def norm_reference(x, gq, gk, hq, angles, amplitude, rot, layout, eps, gy=None):
    x = x.double().clone().requires_grad_(gy is not None)
    heads = x.shape[1]
    gains = torch.stack([gq.double()] * hq + [gk.double()] * (heads - hq)).requires_grad_(gy is not None)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    if gy is None:
        return rotary(n * gains, angles, amplitude, rot, layout)
    g = rotary(gy.double(), angles, amplitude, rot, layout, back=True)
    gx, gg = torch.autograd.grad(n * gains, (x, gains), g)
    n, r, gains = n.detach(), r.detach(), gains.detach()
    # fp32 throughout: about ten roundings on terms of the size of the largest, and sums of `head` terms
    d = x.shape[-1]
    size = r * (abs(g).amax(-1, keepdim=True) * 2 * abs(gains).amax() * (1 + abs(n).amax(-1, keepdim=True) ** 2))
    e_gx = size * (32 + d / 8) * F32
    terms = abs(g).amax(-1, keepdim=True) * abs(n) * 2 * (32 + d / 8 + 64) * F32      # a sum's order: at most 64 roundings deep here
    return gx, gg[:hq].sum(0), gg[hq:].sum(0), e_gx, terms[:, :hq].sum((0, 1)), terms[:, hq:].sum((0, 1))


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rotary(ctx, mode, shape):
    t, h, d, rot, layout, extra, shift = shape
    hq = (h + 1) // 2
    code, dtype = MODES[mode][:2]
    store, tiny = store_rounding(dtype)
    x, ld = inputs((t, h, d), dtype, 3, extra, shift)
    gy, gld = inputs((t, h, d), dtype, 4, extra, shift)
    gain_q, gain_k = (1 + 0.3 * torch.randn(2, d, device="cuda")).to(dtype)
    positions = torch.randint(0, 1 << 20, (t,), device="cuda", dtype=torch.int32)
    freqs, amplitude = pb.rotary_frequencies(rot, 10000.0, "by_parts", 4.0, 512.0) if rot else ([], 1.0)
    f = torch.tensor(freqs + [0.0], device="cuda", dtype=torch.float64)
    angles, eps = positions.double()[:, None] * f[:rot // 2], 1e-5
    common = (rot, layout, f.data_ptr(), amplitude, positions.data_ptr(), eps)
    y = torch.empty((t, h, d), device="cuda", dtype=dtype)
    ctx.norm_rotary_fw(code, x.data_ptr(), gain_q.data_ptr(), gain_k.data_ptr(), y.data_ptr(), d, hq, h - hq, t, ld, 0, *common)
    want = norm_reference(x, gain_q, gain_k, hq, angles, amplitude, rot, layout, eps)
    size = abs(want).amax(-1, keepdim=True) * 2
    assert (abs(y.double() - want) <= size * ((32 + d / 8) * F32 + store) + tiny).all()

    gx, ggq, ggk, e_gx, e_q, e_k = norm_reference(x, gain_q, gain_k, hq, angles, amplitude, rot, layout, eps, gy)
    got, gq = torch.full((t, h, d), 0.25, device="cuda", dtype=dtype), torch.full((2, d), 0.5, device="cuda", dtype=dtype)
    scratch = torch.full((pb.NORM_ROTARY_SCRATCH,), float("nan"), device="cuda")
    for accumulate in (True, False):
        ctx.norm_rotary_bw(code, x.data_ptr(), gain_q.data_ptr(), gain_k.data_ptr(), gy.data_ptr(), got.data_ptr(), gq[0].data_ptr(),
                           gq[1].data_ptr(), scratch.data_ptr(), d, hq, h - hq, t, ld, gld, 0, *common, accumulate_x=accumulate,
                           accumulate_gain=accumulate)
        old_x, old_g = (0.25, 0.5) if accumulate else (0.0, 0.0)
        for value, exact, bound, old in ((got, gx, e_gx, old_x), (gq[0], ggq, e_q, old_g), (gq[1], ggk, e_k, old_g)):
            exact = exact + old
            assert (abs(value.double() - exact) <= bound + store * (abs(exact) + bound) + tiny + F32 * old).all()


def test_norm_gradient_against_differences(ctx):
    t, hq, hk, d = 21, 2, 1, 48
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, gy, dx = (torch.randn(t, hq + hk, d, device="cuda", generator=gen) for _ in range(3))
    gains, dg = 1 + 0.2 * torch.randn(2, d, device="cuda", generator=gen), torch.randn(2, d, device="cuda", generator=gen)
    f = torch.tensor(pb.rotary_frequencies(32)[0], device="cuda", dtype=torch.float64)
    angles = torch.arange(t, device="cuda").double()[:, None] * f
    gx, gg, scratch = torch.empty_like(x), torch.empty_like(gains), torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda")
    ctx.norm_rotary_bw(0, x.data_ptr(), gains[0].data_ptr(), gains[1].data_ptr(), gy.data_ptr(), gx.data_ptr(), gg[0].data_ptr(), gg[1].data_ptr(),
                       scratch.data_ptr(), d, hq, hk, t, 0, 0, 0, 32, PAIRS, f.data_ptr(), accumulate_x=False, accumulate_gain=False)

    def loss(step):
        g = gains.double() + step * dg.double()
        return (norm_reference(x.double() + step * dx.double(), g[0], g[1], hq, angles, 1.0, 32, PAIRS, 1e-6) * gy.double()).sum()
    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    mine = (gx.double() * dx.double()).sum() + (gg.double() * dg.double()).sum()
    size = abs(gx * dx).sum() + abs(gg * dg).sum()
    assert abs(slope - mine) <= 1e-6 * size      # 2^-20 of the terms' size for fp32, 1e-10 for the difference


def test_gain_sums_are_the_same_every_time_and_may_be_left_out(ctx):
    t, hq, hk, d = 5000, 3, 2, 64
    x, gy = (torch.randn(t, hq + hk, d, device="cuda").half() for _ in range(2))
    gain = torch.ones(d, device="cuda").half()
    f = torch.tensor(pb.rotary_frequencies(d)[0], device="cuda", dtype=torch.float64)
    scratch = torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda")
    runs = []
    for _ in range(3):
        gx, gg = torch.empty_like(x), torch.empty(2, d, device="cuda").half()
        ctx.norm_rotary_bw(2, x.data_ptr(), gain.data_ptr(), gain.data_ptr(), gy.data_ptr(), gx.data_ptr(), gg[0].data_ptr(), gg[1].data_ptr(),
                           scratch.data_ptr(), d, hq, hk, t, 0, 0, 0, d, HALVES, f.data_ptr(), accumulate_x=False, accumulate_gain=False)
        runs.append((gx, gg))
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))
    # neither gain's gradient wanted; and in place over gy
    ctx.norm_rotary_bw(2, x.data_ptr(), gain.data_ptr(), gain.data_ptr(), gy.data_ptr(), gy.data_ptr(), None, None, None, d, hq, hk, t, 0, 0, 0,
                       d, HALVES, f.data_ptr(), accumulate_x=False)
    assert torch.equal(gy, runs[0][0])


def test_no_tokens(ctx):
    g = torch.full((2, 8), 3.0, device="cuda")
    s = torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda")
    f = torch.zeros(4, device="cuda", dtype=torch.float64)
    args = (0, None, g.data_ptr(), g.data_ptr(), None, None, g[0].data_ptr(), g[1].data_ptr(), s.data_ptr(), 8, 1, 1, 0, 0, 0, 0, 8, 0, f.data_ptr())
    ctx.norm_rotary_bw(*args, accumulate_gain=True)
    assert (g == 3.0).all()
    ctx.norm_rotary_bw(*args, accumulate_gain=False)
    assert (g == 0.0).all()
    ctx.rotary_fw(0, None, None, 8, 2, 0, 0, 0, 8, 0, f.data_ptr())


def test_refusals(ctx):
    x, y = (torch.zeros(4, 2, 8, device="cuda") for _ in range(2))
    f = torch.zeros(4, device="cuda", dtype=torch.float64)
    g = torch.ones(8, device="cuda")
    X, Y, F, G = x.data_ptr(), y.data_ptr(), f.data_ptr(), g.data_ptr()
    cases = [
        (1001, lambda: ctx.rotary_fw(9, X, Y, 8, 2, 4, 0, 0, 8, 0, F)), (1001, lambda: ctx.rotary_fw(0, None, Y, 8, 2, 4, 0, 0, 8, 0, F)),
        (1001, lambda: ctx.rotary_fw(0, X, None, 8, 2, 4, 0, 0, 8, 0, F)), (1001, lambda: ctx.rotary_fw(0, X, Y, 0, 2, 4, 0, 0, 0, 0, F)),
        (1001, lambda: ctx.rotary_fw(0, X, Y, 8, 2, 4, 15, 0, 8, 0, F)), (1001, lambda: ctx.rotary_fw(0, X, Y, 8, 2, 4, 0, 15, 8, 0, F)),
        (1001, lambda: ctx.rotary_fw(0, X, Y, 8, 2, 4, 0, 0, 7, 0, F)), (1001, lambda: ctx.rotary_fw(0, X, Y, 8, 2, 4, 0, 0, 10, 0, F)),
        (1001, lambda: ctx.rotary_fw(0, X, Y, 8, 2, 4, 0, 0, 8, 2, F)), (1001, lambda: ctx.rotary_fw(0, X, Y, 8, 2, 4, 0, 0, 8, 0, None)),
        (1006, lambda: ctx.rotary_fw(0, X, Y, 258, 2, 4, 0, 0, 8, 0, F)), (1001, lambda: ctx.rotary_fw(0, X, X, 8, 2, 2, 16, 32, 8, 0, F)),
        (1001, lambda: ctx.rotary_bw(0, X, X, 8, 2, 4, 0, 0, 8, 0, F, accumulate=True)),
        (1001, lambda: ctx.norm_rotary_fw(0, X, None, G, Y, 8, 1, 1, 4, 0, 0, 8, 0, F)),
        (1001, lambda: ctx.norm_rotary_fw(0, X, G, None, Y, 8, 1, 1, 4, 0, 0, 8, 0, F)),
        (1001, lambda: ctx.norm_rotary_fw(0, X, G, G, Y, 8, 1, 1, 4, 0, 0, 8, 0, F, eps=math.nan)),
        (1001, lambda: ctx.norm_rotary_bw(0, X, G, G, Y, X, G, G, Y, 8, 1, 1, 4, 0, 0, 0, 8, 0, F)),
        (1001, lambda: ctx.norm_rotary_bw(0, X, G, G, Y, Y, G, G, None, 8, 1, 1, 4, 0, 0, 0, 8, 0, F, accumulate_x=False)),
    ]
    for code, call in cases:
        with pytest.raises(pb.B200Error) as e:
            call()
        assert e.value.code == code
    ctx.norm_rotary_fw(0, X, G, None, Y, 8, 2, 0, 4, 0, 0, 8, 0, F)      # no heads of keys: no gain for them


def test_heads_of_either_kind_may_be_missing(ctx):
    """All heads as queries, or all as keys: the same numbers, and the other gain's gradient is nothing."""
    t, h, d = 333, 5, 96
    gen = torch.Generator(device="cuda").manual_seed(30)
    x, gy = (torch.randn(t, h, d, device="cuda", generator=gen).half() for _ in range(2))
    gain = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).half()
    f = torch.tensor(pb.rotary_frequencies(d)[0], device="cuda", dtype=torch.float64)
    scratch, runs = torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda"), []
    for hq, hk in ((h, 0), (0, h)):
        y, gx, gg = torch.empty_like(x), torch.empty_like(x), torch.full((2, d), 9.0, device="cuda").half()
        gains = (gain.data_ptr(), None) if hq else (None, gain.data_ptr())
        ctx.norm_rotary_fw(2, x.data_ptr(), *gains, y.data_ptr(), d, hq, hk, t, 0, 0, d, PAIRS, f.data_ptr())
        ctx.norm_rotary_bw(2, x.data_ptr(), *gains, gy.data_ptr(), gx.data_ptr(), gg[0].data_ptr(), gg[1].data_ptr(), scratch.data_ptr(), d, hq, hk, t,
                           0, 0, 0, d, PAIRS, f.data_ptr(), accumulate_x=False, accumulate_gain=False)
        runs.append((y, gx, gg[0] if hq else gg[1]))
        assert ((gg[1] if hq else gg[0]) == 0).all()
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_offsets_that_pass_32_bits(ctx):
    """Tokens in rows of a megabyte and more, forward and backward: the same bits as from rows of their own."""
    t, h, d, ld = 4200, 3, 64, (1 << 20) + 8
    f = torch.tensor(pb.rotary_frequencies(d)[0], device="cuda", dtype=torch.float64)
    near = [inputs((t, h, d), torch.float16, seed)[0] for seed in (51, 52)]
    gains = (1 + 0.3 * torch.randn(2, d, device="cuda")).half()
    buffers = [torch.empty(t * ld, device="cuda", dtype=torch.float16) for _ in range(3)]
    assert buffers[0].numel() > 1 << 32
    far = [b.as_strided((t, h, d), (ld, d, 1)) for b in buffers]
    for a, b in zip(far, near):
        a.copy_(b)
    scratch = torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda")
    code, eps = MODES["fp16"][0], 1e-5

    def every(x, gy, out, at):
        got = []
        keep = lambda: got.append(out.contiguous().clone())
        ctx.rotary_fw(code, x.data_ptr(), out.data_ptr(), d, h, t, at, at, d, HALVES, f.data_ptr()), keep()
        ctx.rotary_bw(code, gy.data_ptr(), out.data_ptr(), d, h, t, at, at, d, PAIRS, f.data_ptr(), accumulate=False), keep()
        more = (d, HALVES, f.data_ptr(), 1.0, None, eps)
        ctx.norm_rotary_fw(code, x.data_ptr(), gains[0].data_ptr(), gains[1].data_ptr(), out.data_ptr(), d, 2, 1, t, at, at, *more), keep()
        sums = torch.zeros_like(gains)
        ctx.norm_rotary_bw(code, x.data_ptr(), gains[0].data_ptr(), gains[1].data_ptr(), gy.data_ptr(), out.data_ptr(), sums[0].data_ptr(),
                           sums[1].data_ptr(), scratch.data_ptr(), d, 2, 1, t, at, at, at, *more, accumulate_x=False), keep()
        return got + [sums]
    want = every(near[0], near[1], torch.zeros_like(near[0]), h * d)
    assert all(torch.equal(a, b) for a, b in zip(every(*far, ld), want))


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("head, rot, layout", [(64, 64, HALVES), (128, 32, PAIRS), (96, 96, HALVES), (34, 12, PAIRS), (33, 6, HALVES)])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_gains_off_every_boundary(ctx, mode, head, rot, layout, shift):
    """Gains that start anywhere in a buffer of parameters, beside x, y and gy on 16-byte boundaries: the bits that aligned gains give."""
    t, hq, hk = 37, 3, 2
    code, dtype = MODES[mode][:2]
    (x, _), (gy, _) = (inputs((t, hq + hk, head), dtype, seed) for seed in (71, 72))
    f = torch.tensor(pb.rotary_frequencies(rot)[0], device="cuda", dtype=torch.float64)
    aligned = [(1 + 0.3 * torch.randn(head, device="cuda")).to(dtype) for _ in range(2)]
    sums = torch.full((2 * head + 8,), 9.0, device="cuda", dtype=dtype)
    params = torch.full((2 * head + 8,), float("nan"), device="cuda", dtype=dtype)
    shifted = [params[shift:shift + head], params[shift + head + 1:shift + 2 * head + 1]]
    for a, b in zip(shifted, aligned):
        a.copy_(b)
    scratch, runs = torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda"), []
    for gains, gg in ((aligned, [torch.empty_like(a) for a in aligned]), (shifted, [sums[shift:shift + head], sums[shift + head + 1:shift + 2 * head + 1]])):
        y, gx = torch.empty_like(x), torch.empty_like(x)
        at, more = [g.data_ptr() for g in gains], (rot, layout, f.data_ptr())
        ctx.norm_rotary_fw(code, x.data_ptr(), *at, y.data_ptr(), head, hq, hk, t, 0, 0, *more)
        ctx.norm_rotary_bw(code, x.data_ptr(), *at, gy.data_ptr(), gx.data_ptr(), gg[0].data_ptr(), gg[1].data_ptr(), scratch.data_ptr(), head, hq, hk,
                           t, 0, 0, 0, *more, accumulate_x=False, accumulate_gain=False)
        runs.append([y, gx] + [g.clone() for g in gg])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert (sums[:shift] == 9.0).all() and sums[shift + head] == 9.0 and (sums[shift + 2 * head + 1:] == 9.0).all()


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("t, hq, hk, d, rot", [(1, 1, 1, 64, 64), (5, 3, 2, 64, 32), (67, 9, 1, 33, 6), (131, 5, 3, 128, 128)])
def test_an_epsilon_of_zero(ctx, mode, t, hq, hk, d, rot):
    """Blocks whose last tokens or heads do not exist, where x = 0 makes no infinite 1 / sqrt(0): nothing of them is in the sums."""
    code, dtype = MODES[mode][:2]
    store, tiny = store_rounding(dtype)
    (x, _), (gy, _) = (inputs((t, hq + hk, d), dtype, seed) for seed in (61, 62))
    gain_q, gain_k = (1 + 0.3 * torch.randn(2, d, device="cuda")).to(dtype)
    f = torch.tensor(pb.rotary_frequencies(rot)[0], device="cuda", dtype=torch.float64)
    angles = torch.arange(t, device="cuda").double()[:, None] * f
    gx, ggq, ggk, e_gx, e_q, e_k = norm_reference(x, gain_q, gain_k, hq, angles, 1.0, rot, PAIRS, 0.0, gy)
    got, gg, scratch = torch.empty_like(gx).to(dtype), torch.empty(2, d, device="cuda", dtype=dtype), torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda")
    ctx.norm_rotary_bw(code, x.data_ptr(), gain_q.data_ptr(), gain_k.data_ptr(), gy.data_ptr(), got.data_ptr(), gg[0].data_ptr(), gg[1].data_ptr(),
                       scratch.data_ptr(), d, hq, hk, t, 0, 0, 0, rot, PAIRS, f.data_ptr(), eps=0.0, accumulate_x=False, accumulate_gain=False)
    for value, exact, bound in ((got, gx, e_gx), (gg[0], ggq, e_q), (gg[1], ggk, e_k)):
        assert (abs(value.double() - exact) <= bound + store * (abs(exact) + bound) + tiny).all()


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("layout", [PAIRS, HALVES])
def test_angles_are_as_good_far_out_as_near_zero(ctx, layout, back):
    """fp32 at positions up to the last one, against angles reduced in exact arithmetic: the bound that holds near position 0."""
    from fractions import Fraction
    two_pi = 2 * Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    pos, rot = [0, 5, 16777217, 999999937, (1 << 32) - 1] + [(1 << 31) + i * 7158279 for i in range(300)], 32
    freqs = pb.rotary_frequencies(rot)[0]
    angles = torch.tensor([[float(p * Fraction(f) % two_pi) for f in freqs] for p in pos], device="cuda", dtype=torch.float64)
    x = torch.randn(len(pos), 3, 40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(81))
    at = torch.tensor([p - (1 << 32) if p >> 31 else p for p in pos], device="cuda", dtype=torch.int32)
    f, y = torch.tensor(freqs, device="cuda", dtype=torch.float64), torch.empty_like(x)
    if back:
        ctx.rotary_bw(0, x.data_ptr(), y.data_ptr(), 40, 3, len(pos), 0, 0, rot, layout, f.data_ptr(), positions=at.data_ptr(), accumulate=False)
    else:
        ctx.rotary_fw(0, x.data_ptr(), y.data_ptr(), 40, 3, len(pos), 0, 0, rot, layout, f.data_ptr(), positions=at.data_ptr())
    want = rotary(x.double(), angles, 1.0, rot, layout, back=back)
    # The angle in turns is rounded to 32 bits once, 2^-26 of a turn: 2 pi 2^-26 = 1.6 F32 of the pair's size; sine and cosine are right to
    # 2 units each (2 sqrt(2) F32 of the pair); a product and the sum round once (2 F32).
    pair = torch.view_as_complex(x[..., :rot].double().reshape(len(pos), 3, rot // 2, 2)).abs() if layout == PAIRS \
        else torch.hypot(x[..., :rot // 2].double(), x[..., rot // 2:rot].double())
    size = pair.repeat_interleave(2, -1) if layout == PAIRS else torch.cat((pair, pair), -1)
    assert (abs(y.double() - want)[..., :rot] <= size * 7 * F32).all()
    assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("t, hq, hk, d, rot, layout", [(20011, 2, 1, 32, 32, HALVES), (9001, 1, 1, 33, 6, PAIRS), (40003, 1, 2, 64, 16, PAIRS)])
def test_norm_gradients_over_many_tiles(ctx, mode, t, hq, hk, d, rot, layout):
    """More tokens than the blocks take at a time: a block goes from tile to tile, each with angles of its own."""
    code, dtype = MODES[mode][:2]
    store, tiny = store_rounding(dtype)
    (x, _), (gy, _) = (inputs((t, hq + hk, d), dtype, seed) for seed in (91, 92))
    gain_q, gain_k = (1 + 0.3 * torch.randn(2, d, device="cuda")).to(dtype)
    positions = torch.randint(0, 1 << 20, (t,), device="cuda", dtype=torch.int32)
    f = torch.tensor(pb.rotary_frequencies(rot)[0], device="cuda", dtype=torch.float64)
    gx, ggq, ggk, e_gx, e_q, e_k = norm_reference(x, gain_q, gain_k, hq, positions.double()[:, None] * f, 1.0, rot, layout, 1e-5, gy)
    got, gg, scratch = torch.empty_like(x), torch.empty(2, d, device="cuda", dtype=dtype), torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda")
    ctx.norm_rotary_bw(code, x.data_ptr(), gain_q.data_ptr(), gain_k.data_ptr(), gy.data_ptr(), got.data_ptr(), gg[0].data_ptr(), gg[1].data_ptr(),
                       scratch.data_ptr(), d, hq, hk, t, 0, 0, 0, rot, layout, f.data_ptr(), 1.0, positions.data_ptr(), 1e-5, accumulate_x=False,
                       accumulate_gain=False)
    # (the sums' bound takes 64 roundings one on another: at most 32 rows of heads in a thread here, 5 between lanes, 8 warps, 14 blocks, 32 lanes of those;
    # each is of a part of the sum, and the bound's terms are all of it, with a factor 2)
    for value, exact, bound in ((got, gx, e_gx), (gg[0], ggq, e_q), (gg[1], ggk, e_k)):
        assert (abs(value.double() - exact) <= bound + store * (abs(exact) + bound) + tiny).all()
