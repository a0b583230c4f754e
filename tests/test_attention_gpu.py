"""Attention over packed, padded and cached sequences, forward and backward, against 64 bits."""
import math

import pytest
import torch

import primitiv_b200 as pb
from attention_lib import MODES, attention

pytestmark = pytest.mark.gpu
NAN = float("nan")


def i32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


class Problem:
    """Sequences of (queries, keys) given as (first row, length) each; everything outside them holds NaN."""

    def __init__(self, mode, head, hq, hk, q_at, k_at, causal, seed=0, fused=False, gap=0, shift=0, scale=None, gy_size=1.0, size=1.0):
        self.mode, self.dtype = MODES[mode][:2]
        self.name, self.head, self.hq, self.hk, self.q_at, self.k_at, self.causal = mode, head, hq, hk, q_at, k_at, causal
        self.scale = 1 / math.sqrt(head) if scale is None else scale
        self.rows_q = max([a + n for a, n in q_at] + [0]) + gap
        self.rows_k = max([a + n for a, n in k_at] + [0]) + gap
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def make(rows, heads, at, times=1.0):
            t = torch.full((rows, heads, head), NAN, device="cuda")
            for first, n in at:
                t[first:first + n] = times * torch.randn(n, heads, head, device="cuda", generator=gen)
            flat = torch.full((rows * heads * head + shift,), NAN, device="cuda", dtype=self.dtype)
            flat[shift:] = t.to(self.dtype).flatten()
            return flat[shift:].view(rows, heads, head)
        if fused:
            qkv = make(self.rows_q, hq + 2 * hk, q_at, size)
            self.q, self.k, self.v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        else:
            self.q, self.k, self.v = make(self.rows_q, hq, q_at, size), make(self.rows_k, hk, k_at, size), make(self.rows_k, hk, k_at)
        self.gy = make(self.rows_q, hq, q_at, gy_size)
        self.y = torch.full((self.rows_q, hq, head), 7.0, device="cuda", dtype=self.dtype)
        self.lse = torch.full((hq, self.rows_q), 7.0, device="cuda")
        self.keep = []

    def plan(self, **more):
        fields = dict(head=self.head, heads_q=self.hq, heads_k=self.hk, rows_q=self.rows_q, rows_k=self.rows_k, q_ld=self.q.stride(0),
                      k_ld=self.k.stride(0), v_ld=self.v.stride(0), y_ld=self.y.stride(0), seqs=len(self.q_at), causal=int(self.causal),
                      scale=self.scale)
        for side, at, rows in (("q", self.q_at, self.rows_q), ("k", self.k_at, self.rows_k)):
            starts, lens = i32([a for a, _ in at] + [rows]), i32([n for _, n in at])
            self.keep += [starts, lens]
            fields[side + "_starts"], fields[side + "_lens"] = starts.data_ptr(), lens.data_ptr()
            fields["max_" + side] = max([n for _, n in at] + [1])
        fields.update(more)
        return pb.Attention(**fields)

    def forward(self, ctx, plan=None, stream=None, lse=True):
        ctx.attention_fw(self.mode, plan or self.plan(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.y.data_ptr(),
                         self.lse.data_ptr() if lse else None, stream=stream)

    def backward(self, ctx, plan=None, accumulate=False, start=NAN, stream=None):
        plan = plan or self.plan()
        self.scratch = torch.full((plan.bw_scratch_floats(),), NAN, device="cuda")
        if self.q.stride(0) != self.hq * self.head:
            g = torch.full((self.rows_q, self.hq + 2 * self.hk, self.head), start, device="cuda", dtype=self.dtype)
            self.gq, self.gk, self.gv = g[:, :self.hq], g[:, self.hq:self.hq + self.hk], g[:, self.hq + self.hk:]
        else:
            self.gq, self.gk, self.gv = (torch.full(t.shape, start, device="cuda", dtype=self.dtype) for t in (self.q, self.k, self.v))
        ctx.attention_bw(self.mode, plan, self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.y.data_ptr(), self.lse.data_ptr(),
                         self.gy.data_ptr(), self.gq.data_ptr(), self.gk.data_ptr(), self.gv.data_ptr(), self.scratch.data_ptr(),
                         accumulate=accumulate, stream=stream)

    def check(self, gradients=False, start=0.0):
        group = self.hq // self.hk
        if gradients:
            sums = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in (("gq", self.q), ("gk", self.k), ("gv", self.v))}
            tols = {n: torch.zeros_like(t) for n, t in sums.items()}
        outside = torch.ones(self.rows_q, dtype=torch.bool, device="cuda")
        for (q0, lq), (k0, lk) in zip(self.q_at, self.k_at):
            outside[q0:q0 + lq] = False
            for h in range(self.hq):
                kh = h // group
                val, tol = attention(self.q[q0:q0 + lq, h].double(), self.k[k0:k0 + lk, kh].double(), self.v[k0:k0 + lk, kh].double(), self.scale,
                                     self.causal, self.gy[q0:q0 + lq, h].double() if gradients else None, self.name)
                got, lse = self.y[q0:q0 + lq, h].double(), self.lse[h, q0:q0 + lq].double()
                off = abs(got - val["y"]) - tol["y"]
                assert lq == 0 or not (off > 0).any() and not got.isnan().any(), ("y", h, q0, off.max().item())
                seen = val["lse"] > -math.inf
                assert torch.equal(lse[~seen], val["lse"][~seen])
                assert (abs(lse - val["lse"])[seen] <= tol["lse"][seen]).all(), ("lse", abs(lse - val["lse"])[seen].max())
                if gradients:
                    sums["gq"][q0:q0 + lq, h], tols["gq"][q0:q0 + lq, h] = val["gq"], tol["gq"]
                    for n in ("gk", "gv"):
                        sums[n][k0:k0 + lk, kh] += val[n]
                        tols[n][k0:k0 + lk, kh] += tol[n]
        assert (self.y[outside] == 7.0).all() and (self.lse[:, outside] == 7.0).all()
        if gradients:
            half = 2.0 ** -11 if self.dtype == torch.float16 else 2.0 ** -23
            for n in sums:
                got = getattr(self, n).double()
                off = abs(got - (sums[n] + start)) - tols[n] - abs(start) * half - half * abs(start + sums[n]) * (start != 0)
                assert not got.isnan().any() and not (off > 0).any(), (n, off.max().item())


def packed(lengths, first=0, gap=0):
    at = []
    for n in lengths:
        at.append((first, n))
        first += n + gap
    return at


SELF = [  # head, heads of q, of k, lengths, causal, fused
    (64, 2, 2, [1], True, False), (64, 4, 2, [64, 1, 65, 0, 200], True, False), (128, 4, 1, [130, 257, 31], True, True),
    (128, 2, 2, [128, 384, 512], False, False), (80, 6, 2, [100, 3, 300], True, True), (32, 8, 8, [33, 129], False, True),
    (96, 7, 1, [77, 150], True, False), (256, 2, 1, [70, 129], True, False), (200, 2, 2, [65], False, True), (17, 3, 1, [40, 90], True, False),
    (1, 2, 1, [10, 70], False, False), (128, 14, 2, [5, 700], True, True), (64, 1, 1, [1025], True, False), (112, 3, 3, [255, 256], True, False),
]


@pytest.mark.parametrize("mode", ["fp16", "3xtf32", "tf32"])
@pytest.mark.parametrize("shape", SELF)
def test_packed_sequences(ctx, mode, shape):
    head, hq, hk, lengths, causal, fused = shape
    at = packed(lengths, first=3, gap=0 if fused else 2)
    p = Problem(mode, head, hq, hk, at, at, causal, seed=len(lengths), fused=fused, gap=5)
    p.forward(ctx)
    p.check()
    p.backward(ctx)
    p.check(gradients=True)
    p.backward(ctx, accumulate=True, start=0.5)
    inside = torch.zeros(p.rows_q, dtype=torch.bool, device="cuda")
    for first, n in at:
        inside[first:first + n] = True
    assert (p.gq[~inside] == 0.5).all() and (p.gk[~inside] == 0.5).all() and (p.gv[~inside] == 0.5).all()
    p.check(gradients=True, start=0.5)


@pytest.mark.parametrize("mode", ["fp16", "3xtf32", "3xfp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq, lk", [(5, 200), (200, 5), (1, 1), (130, 257), (64, 0), (257, 128), (3, 3)])
def test_different_numbers_of_queries_and_keys(ctx, mode, causal, lq, lk):
    """More keys than queries, and the other way round, where causal rows see nothing; a sequence without any key."""
    q_at, k_at = packed([lq, 7, lq]), packed([lk, 9, lk], first=1, gap=1)
    p = Problem(mode, 64, 4, 2, q_at, k_at, causal, seed=lq + lk, gap=3)
    p.forward(ctx)
    p.check()
    p.backward(ctx)
    p.check(gradients=True)


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("head, hq, hk", [(128, 32, 8), (64, 8, 1), (128, 4, 4), (80, 12, 2), (256, 4, 2), (40, 64, 2), (33, 3, 1)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_tokens_against_a_cache(ctx, mode, head, hq, hk, tokens):
    """Each sequence's cache has room for 700 keys, holds fewer, and NaN behind them."""
    lens = [700, 1, 64, 129, 3, 500]
    lens = [max(n, tokens) for n in lens]
    q_at, k_at = packed([tokens] * len(lens)), [(700 * i, n) for i, n in enumerate(lens)]
    p = Problem(mode, head, hq, hk, q_at, k_at, True, seed=tokens)
    p.forward(ctx)
    p.check()
    y = p.y.clone()
    p.y.fill_(7.0)
    p.forward(ctx, lse=False)
    assert torch.equal(y, p.y)


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
def test_a_long_cache(ctx, mode):
    p = Problem(mode, 128, 8, 2, packed([1, 1, 2]), packed([20011, 5, 4097]), True, seed=5)
    p.forward(ctx)
    p.check()


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
def test_large_scores(ctx, mode):
    """Softmax over scores of some hundreds: one key takes nearly all of a row, and exp of the score itself would overflow."""
    at = packed([190])
    p = Problem(mode, 64, 2, 1, at, at, True, seed=6, size=12.0, scale=0.25)
    p.forward(ctx)
    p.check()
    p.backward(ctx)
    p.check(gradients=True)


@pytest.mark.parametrize("gy_size", [1e-5, 1e4])
def test_gradients_of_any_size(ctx, gy_size):
    """Gradients far from one: gy of 1e-5 over 900 keys makes a ds far below the smallest half."""
    at = packed([900])
    p = Problem("fp16", 64, 2, 2, at, at, False, seed=7, gy_size=gy_size, size=0.3)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("shift", [1, 4])
def test_addresses_off_16_bytes(ctx, mode, shift):
    at = packed([150, 20])
    p = Problem(mode, 64, 4, 2, at, at, True, seed=8, shift=shift)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
def test_a_minibatch_needs_no_starts(ctx, mode):
    batch, t = 5, 75
    at = [(i * t, t) for i in range(batch)]
    p = Problem(mode, 64, 4, 4, at, at, False, seed=9)
    none = dict(q_starts=None, q_lens=None, k_starts=None, k_lens=None, max_q=0, max_k=0)
    p.forward(ctx, p.plan(**none))
    p.backward(ctx, p.plan(**none))
    p.check(gradients=True)
    # padded: lengths alone
    lens = [75, 0, 1, 33, 74]
    at = [(i * t, n) for i, n in enumerate(lens)]
    p = Problem(mode, 64, 4, 4, at, at, True, seed=10)
    rows = batch * t
    pad = {n: torch.full((rows,) + x.shape[1:], fill, device="cuda", dtype=p.dtype) for n, x, fill in
           (("q", p.q, NAN), ("k", p.k, NAN), ("v", p.v, NAN), ("gy", p.gy, NAN), ("y", p.y, 7.0))}
    for n, x in pad.items():
        x[:p.rows_q] = getattr(p, n)
        setattr(p, n, x)
    p.lse = torch.full((p.hq, rows), 7.0, device="cuda")
    p.rows_q = p.rows_k = rows
    none = dict(q_starts=None, k_starts=None, max_q=0, max_k=0)
    p.forward(ctx, p.plan(**none))
    p.backward(ctx, p.plan(**none))
    p.check(gradients=True)


def test_more_sequences_than_a_step_of_the_search(ctx):
    lengths = [(i * 37) % 90 for i in range(150)]
    at = packed(lengths, gap=1)
    p = Problem("fp16", 64, 2, 1, at, at, True, seed=11)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)
    q_at = packed([1] * 150)
    p = Problem("fp16", 64, 2, 1, q_at, packed([n + 1 for n in lengths]), True, seed=12)
    p.forward(ctx)
    p.check()


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("longest", [70, 300])
def test_thousands_of_sequences(ctx, mode, longest):
    """One long sequence among 3000 short ones: tiles are numbered through all of them, or apart for each."""
    lengths = [(i * 7) % 4 for i in range(3000)]
    lengths[1234] = longest
    at = packed(lengths)
    p = Problem(mode, 64, 2, 1, at, at, True, seed=25)
    p.forward(ctx)
    p.backward(ctx)
    # a few of them: each is compared on its own
    some = [0, 1, 2, 3, 1233, 1234, 1235, 2998, 2999]
    group = Problem(mode, 64, 2, 1, packed([1]), packed([1]), True, seed=26)
    for n in ("q", "k", "v", "gy"):
        setattr(group, n, torch.cat([getattr(p, n)[at[i][0]:at[i][0] + at[i][1]] for i in some]))
    group.q_at = group.k_at = packed([at[i][1] for i in some])
    group.rows_q = group.rows_k = group.q.shape[0]
    group.y = torch.cat([p.y[at[i][0]:at[i][0] + at[i][1]] for i in some])
    group.lse = torch.cat([p.lse[:, at[i][0]:at[i][0] + at[i][1]] for i in some], 1)
    for n in ("gq", "gk", "gv"):
        setattr(group, n, torch.cat([getattr(p, n)[at[i][0]:at[i][0] + at[i][1]] for i in some]))
    group.check(gradients=True)
    assert not any(g.isnan().any() for g in (p.y, p.gq, p.gk, p.gv))


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("tokens", [1, 130])
def test_scales_that_are_not_positive(ctx, mode, scale, tokens):
    q_at = packed([tokens, tokens])
    p = Problem(mode, 64, 4, 2, q_at, packed([140, 150]), True, seed=27, scale=scale)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)


def test_starts_beyond_the_rows_are_cut(ctx):
    """Numbers that a faulty program could hold: nothing outside the arrays is read or written."""
    at = [(0, 40), (40, 24)]
    p = Problem("fp16", 64, 2, 2, at, at, True, seed=13)
    starts, lens = i32([0, 40, 1 << 30]), i32([1 << 30, 1 << 30])
    p.forward(ctx, p.plan(q_starts=starts.data_ptr(), k_starts=starts.data_ptr(), q_lens=lens.data_ptr(), k_lens=lens.data_ptr(), max_q=0, max_k=0))
    p.check()
    down = i32([50, 10, 5])
    p.y.fill_(7.0)
    p.forward(ctx, p.plan(q_starts=down.data_ptr(), k_starts=down.data_ptr(), q_lens=None, k_lens=None, max_q=0, max_k=0))
    assert (p.y == 7.0).all()


def test_max_q_cuts(ctx):
    at = packed([100, 100])
    p = Problem("fp16", 64, 2, 2, at, at, True, seed=14)
    p.forward(ctx, p.plan(max_q=64, max_k=64))
    p.q_at = p.k_at = [(0, 64), (100, 64)]
    p.check()


def test_gradient_against_differences(ctx):
    q_at, k_at = packed([37, 20]), packed([50, 20])
    p = Problem("3xtf32", 32, 4, 2, q_at, k_at, True, seed=15)
    p.forward(ctx)
    p.backward(ctx)
    gen = torch.Generator(device="cuda").manual_seed(16)
    d = {n: torch.randn(getattr(p, n).shape, device="cuda", generator=gen, dtype=torch.float64) for n in "qkv"}

    def loss(step):
        total = 0.0
        for (q0, lq), (k0, lk) in zip(p.q_at, p.k_at):
            for h in range(p.hq):
                a = {n: getattr(p, n).double() + step * d[n] for n in "qkv"}
                val, _ = attention(a["q"][q0:q0 + lq, h], a["k"][k0:k0 + lk, h // 2], a["v"][k0:k0 + lk, h // 2], p.scale, True, mode="3xtf32")
                total = total + (val["y"] * p.gy[q0:q0 + lq, h].double()).sum()
        return total
    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    parts = [(g.double() * d[n]) for n, g in (("q", p.gq), ("k", p.gk), ("v", p.gv))]
    size = sum(abs(x).sum() for x in parts)
    # the kernel's gradient is good to 2^-16 of its terms at these lengths, the difference to 1e-9
    assert abs(slope - sum(x.sum() for x in parts)) <= 2.0 ** -16 * size


def test_the_same_bits_every_time_and_in_a_graph(ctx):
    at = packed([300, 41, 128])
    for p in (Problem("fp16", 128, 8, 2, at, at, True, seed=17), Problem("3xtf32", 64, 4, 4, at, at, False, seed=18)):
        plan = p.plan()
        p.forward(ctx, plan)
        p.backward(ctx, plan)
        first = [t.clone() for t in (p.y, p.lse, p.gq, p.gk, p.gv)]
        side = torch.cuda.Stream()
        outs = [torch.full_like(t, 3.0) for t in first]
        torch.cuda.synchronize()

        def both(stream):
            ctx.attention_fw(p.mode, plan, p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), outs[0].data_ptr(), outs[1].data_ptr(), stream=stream)
            ctx.attention_bw(p.mode, plan, p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), outs[0].data_ptr(), outs[1].data_ptr(), p.gy.data_ptr(),
                             outs[2].data_ptr(), outs[3].data_ptr(), outs[4].data_ptr(), p.scratch.data_ptr(), accumulate=False, stream=stream)
        with torch.cuda.stream(side):
            both(side.cuda_stream)
            side.synchronize()
            inside = torch.zeros(p.rows_q, dtype=torch.bool, device="cuda")
            for a, n in at:
                inside[a:a + n] = True
            assert all(torch.equal(a[inside], b[inside]) for a, b in zip(outs[:1] + outs[2:], first[:1] + first[2:]))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                both(torch.cuda.current_stream().cuda_stream)
            for o in outs:
                o.fill_(3.0)
            graph.replay()
            side.synchronize()
        assert all(torch.equal(a[inside], b[inside]) for a, b in zip(outs[:1] + outs[2:], first[:1] + first[2:]))
        assert torch.equal(outs[1][:, inside], first[1][:, inside])


def test_a_captured_step_of_generation_follows_its_lengths(ctx):
    """A graph captured once; between replays the cache grows and the lengths, which are on the device, with it."""
    room, seqs = 256, 3
    lens = [10, 200, 100]
    q_at, k_at = packed([1] * seqs), [(room * i, n) for i, n in enumerate(lens)]
    p = Problem("fp16", 64, 8, 2, q_at, k_at, True, seed=19)
    full = Problem("fp16", 64, 8, 2, q_at, [(room * i, room) for i in range(seqs)], True, seed=20)
    p.k, p.v, p.rows_k = full.k, full.v, full.rows_k
    on_device = i32(lens)
    plan = p.plan(k_lens=on_device.data_ptr(), max_k=room)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p.forward(ctx, plan, stream=torch.cuda.current_stream().cuda_stream)
    for grown in ([10, 200, 100], [11, 201, 101], [256, 1, 129]):
        on_device.copy_(i32(grown))
        graph.replay()
        torch.cuda.synchronize()
        p.k_at = [(room * i, n) for i, n in enumerate(grown)]
        p.check()


def test_a_layer_between_two_products(ctx):
    """The operators together, as a layer uses them: one product makes queries, keys and values side by side, norms and rotation turn
    them in place, attention reads them where they lie, and the gradients come back the same way into the product's."""
    t, model, hq, hk, d = 150, 96, 4, 2, 32
    lengths = [70, 80]
    wide = (hq + 2 * hk) * d
    gen = torch.Generator(device="cuda").manual_seed(21)
    x = torch.randn(t, model, device="cuda", generator=gen) / 8
    w = torch.randn(model, wide, device="cuda", generator=gen) / 8       # {wide, model} of the library
    gy = torch.randn(t, hq, d, device="cuda", generator=gen)
    gain = 1 + 0.2 * torch.randn(2, d, device="cuda", generator=gen)
    freqs = torch.tensor(pb.rotary_frequencies(d)[0], device="cuda", dtype=torch.float64)
    positions = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in lengths])
    starts = i32([0, 70, 150])
    qkv, turned = torch.empty(t, wide, device="cuda"), torch.empty(t, wide, device="cuda")
    ctx.matmul_fw(0, w.data_ptr(), x.data_ptr(), qkv.data_ptr(), wide, model, t, 1, 1)
    turned.copy_(qkv)
    at = (d, hq, hk, t, wide, wide)
    ctx.norm_rotary_fw(0, qkv.data_ptr(), gain[0].data_ptr(), gain[1].data_ptr(), turned.data_ptr(), *at, d, 1, freqs.data_ptr(), 1.0,
                       positions.data_ptr())
    es, k_at, v_at = 4, hq * d, (hq + hk) * d
    plan = pb.Attention(head=d, heads_q=hq, heads_k=hk, rows_q=t, rows_k=t, seqs=2, max_q=80, max_k=80, q_ld=wide, k_ld=wide, v_ld=wide,
                        q_starts=starts.data_ptr(), k_starts=starts.data_ptr(), causal=1, scale=d ** -0.5)
    y, lse, g = torch.empty(t, hq, d, device="cuda"), torch.empty(hq, t, device="cuda"), torch.empty(t, wide, device="cuda")
    base, gb = turned.data_ptr(), g.data_ptr()
    ctx.attention_fw(0, plan, base, base + k_at * es, base + v_at * es, y.data_ptr(), lse.data_ptr())
    scratch = torch.empty(max(plan.bw_scratch_floats(), pb.NORM_ROTARY_SCRATCH), device="cuda")
    ctx.attention_bw(0, plan, base, base + k_at * es, base + v_at * es, y.data_ptr(), lse.data_ptr(), gy.data_ptr(), gb, gb + k_at * es,
                     gb + v_at * es, scratch.data_ptr(), accumulate=False)
    ggain, gx, gw = torch.empty_like(gain), torch.zeros_like(x), torch.zeros_like(w)
    ctx.norm_rotary_bw(0, qkv.data_ptr(), gain[0].data_ptr(), gain[1].data_ptr(), gb, gb, ggain[0].data_ptr(), ggain[1].data_ptr(),
                       scratch.data_ptr(), d, hq, hk, t, wide, wide, wide, d, 1, freqs.data_ptr(), 1.0, positions.data_ptr(), accumulate_x=False,
                       accumulate_gain=False)
    ctx.matmul_bw(0, w.data_ptr(), x.data_ptr(), gb, gw.data_ptr(), gx.data_ptr(), wide, model, t, 1, 1)

    def layer(x, w, gain):
        from attention_lib import rotary
        out = (x @ w).view(t, hq + 2 * hk, d)
        n = out[:, :hq + hk]
        n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + 1e-6) * torch.stack([gain[0]] * hq + [gain[1]] * hk)
        n = rotary(n, positions.double()[:, None] * freqs, 1.0, d, 1)
        ys = []
        for a, b in ((0, 70), (70, 150)):
            k, v = (z.repeat_interleave(hq // hk, 1) for z in (n[a:b, hq:], out[a:b, hq + hk:]))
            s = torch.einsum("ihd,jhd->hij", n[a:b, :hq], k) * d ** -0.5
            p = torch.softmax(s.masked_fill(~torch.ones_like(s[0], dtype=torch.bool).tril(), -math.inf), -1)
            ys.append(torch.einsum("hij,jhd->ihd", p, v))
        return torch.cat(ys)
    args = [z.double().requires_grad_(True) for z in (x, w, gain)]
    want = layer(*args)
    grads = torch.autograd.grad(want, args, gy.double())
    # five fp32-grade steps, each good to 1e-5 of its largest values (the products' own bound)
    for got, exact in zip((y, gx, gw, ggain), (want.detach(),) + grads):
        assert abs(got.double() - exact).max() <= 5e-5 * abs(exact).max()


def test_refusals(ctx):
    at = packed([8])
    p = Problem("fp16", 64, 2, 2, at, at, True)
    a = [t.data_ptr() for t in (p.q, p.k, p.v, p.y, p.lse)]
    for at_null in range(4):
        with pytest.raises(pb.B200Error) as e:
            ctx.attention_fw(2, p.plan(), *[None if i == at_null else v for i, v in enumerate(a)])
        assert e.value.code == 1001
    for mode in (-1, 4):
        with pytest.raises(pb.B200Error):
            ctx.attention_fw(mode, p.plan(), *a)
    g = [t.data_ptr() for t in (p.gy, p.q, p.k, p.v, p.lse)]
    for at_null in range(10):
        with pytest.raises(pb.B200Error) as e:
            ctx.attention_bw(2, p.plan(), *[None if i == at_null else v for i, v in enumerate(a + g)])
        assert e.value.code == 1001
    for more, code in ((dict(head=300), 1006), (dict(heads_q=3), 1001), (dict(q_ld=100), 1001), (dict(scale=NAN), 1001)):
        with pytest.raises(pb.B200Error) as e:
            ctx.attention_fw(2, p.plan(**more), *a)
        assert e.value.code == code
    ctx.attention_fw(2, p.plan(seqs=0), *a)
    assert (p.y == 7.0).all()
    ctx.attention_fw(2, p.plan(rows_q=0), None, *a[1:3], None)
    # no keys at all: rows of zeros
    ctx.attention_fw(2, p.plan(rows_k=0, k_starts=None, k_lens=None), a[0], None, None, a[3], a[4])
    assert (p.y == 0.0).all() and (p.lse == -math.inf).all()


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
@pytest.mark.parametrize("rows", [200, 1])
def test_nans_are_not_lost(ctx, mode, rows):
    """A NaN in a key reaches the queries that see that key, all of them and in y no others; one in a query reaches that query's y alone."""
    for column in list(range(0, 16)) + [77, 130]:
        at = packed([200])
        p = Problem(mode, 64, 2, 1, at if rows > 1 else [(0, 1)], at, True, seed=23)
        p.k[column, 0, 5] = NAN
        p.forward(ctx)
        hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
        hit[column if rows > 1 else 0:] = True
        assert torch.equal(p.y[:rows].isnan().all(2).all(1), hit) and torch.equal(p.y[:rows].isnan().any(2).any(1), hit)
        if rows > 1:
            p.backward(ctx)
            assert p.gq[hit].isnan().all() and p.gk[0, 0].isnan().all() and p.gv[0].isnan().all()
            p = Problem(mode, 64, 2, 1, at, at, True, seed=24)
            p.q[column, 1, 3] = NAN
            p.forward(ctx)
            assert p.y[column, 1].isnan().all() and not p.y[column, 0].isnan().any()
            assert not p.y[torch.arange(200, device="cuda") != column].isnan().any()
            p.backward(ctx)
            assert p.gq[column, 1].isnan().all() and not p.gq[:, 0].isnan().any() and p.gv[:column + 1].isnan().all()


@pytest.mark.parametrize("head", [8, 16, 24, 48, 104, 120])
def test_halves_of_short_heads(ctx, head):
    at = packed([150, 66], first=1)
    p = Problem("fp16", head, 4, 2, at, at, True, seed=head)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)


@pytest.mark.parametrize("head", [64, 17])
@pytest.mark.parametrize("queries", [1, 130])
def test_offsets_that_pass_32_bits(ctx, head, queries):
    """Keys, values and their gradients in rows of a megabyte and more: the same bits as from rows of their own."""
    ld, at = (1 << 20) + 8, packed([100, 4300])
    p = Problem("fp16", head, 2, 2, packed([queries, queries]), at, True, seed=41)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)
    want = [t.clone() for t in (p.y, p.lse, p.gq, p.gk, p.gv)]
    far = [torch.empty(p.rows_k * ld, device="cuda", dtype=p.dtype) for _ in range(2)]
    assert far[0].numel() > 1 << 32
    k, v, gk, gv = (f[2 * head * i:].as_strided((p.rows_k, 2, head), (ld, head, 1)) for f in far for i in range(2))
    k.copy_(p.k), v.copy_(p.v), gk.fill_(NAN), gv.fill_(NAN)
    p.k, p.v = k, v
    p.y.fill_(7.0), p.lse.fill_(7.0), p.gq.fill_(NAN)
    plan = p.plan()
    p.forward(ctx, plan)
    ctx.attention_bw(p.mode, plan, p.q.data_ptr(), k.data_ptr(), v.data_ptr(), p.y.data_ptr(), p.lse.data_ptr(), p.gy.data_ptr(), p.gq.data_ptr(),
                     gk.data_ptr(), gv.data_ptr(), p.scratch.data_ptr(), accumulate=False)
    assert all(torch.equal(a, b) for a, b in zip((p.y, p.lse, p.gq, gk, gv), want))


@pytest.mark.parametrize("mode", ["fp16", "3xtf32"])
def test_two_calls_at_once(ctx, mode):
    """On two streams, each with its own outputs and scratch: the bits that either call gives alone."""
    problems = [Problem(mode, 64, 4, 2, packed(n), packed(n), True, seed=len(n)) for n in ([700, 90, 300], [1, 555, 40, 260])]
    plans, want = [p.plan() for p in problems], []
    for p, plan in zip(problems, plans):
        p.forward(ctx, plan)
        p.backward(ctx, plan)
        want.append([t.clone() for t in (p.y, p.lse, p.gq, p.gk, p.gv)])
    streams = [torch.cuda.Stream() for _ in problems]
    for p in problems:
        for t in (p.y, p.lse, p.gq, p.gk, p.gv):
            t.fill_(NAN)
    torch.cuda.synchronize()
    for _ in range(3):
        for p, plan, s in zip(problems, plans, streams):
            p.forward(ctx, plan, stream=s.cuda_stream)
            ctx.attention_bw(p.mode, plan, p.q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), p.y.data_ptr(), p.lse.data_ptr(), p.gy.data_ptr(),
                             p.gq.data_ptr(), p.gk.data_ptr(), p.gv.data_ptr(), p.scratch.data_ptr(), accumulate=False, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for p, w in zip(problems, want):
        assert all(torch.equal(a, b) for a, b in zip((p.y, p.lse, p.gq, p.gk, p.gv), w))


# kernels of a forward pass: (head, queries, keys); a few queries, mma.sync with one block to a tile and with a cluster, tcgen05
WAYS = [(64, 1, 100), (64, 3, 700), (40, 50, 90), (40, 50, 900), (33, 200, 900), (64, 200, 200), (128, 300, 520), (256, 1, 60), (256, 90, 90)]


@pytest.mark.parametrize("mode", ["fp16", "3xtf32", "tf32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("head, lq, lk", WAYS)
def test_rows_without_a_finite_score(ctx, mode, causal, head, lq, lk):
    """A query with a NaN has y and lse of NaN; one whose scores are all -infinity has weights of 0 / 0, and a sum of zeros in lse; one with a score
    of +infinity has infinity / infinity.  No other row is touched, and all three reach their gradients."""
    p = Problem(mode, head, 4, 2, packed([lq]), packed([lk]), causal, seed=61)
    p.k[:, :, 0] = abs(p.k[:, :, 0]) + 0.125      # so q = -inf here makes every score -inf
    rows = sorted({0, lq // 2, lq - 1})
    bad = {(r, h): (NAN, -math.inf, math.inf)[(i + h) % 3] for i, r in enumerate(rows) for h in (1, 2, 3)}
    clean = p.q.clone()
    for (r, h), v in bad.items():
        p.q[r, h, 0] = v
    p.forward(ctx)
    hit = torch.zeros(lq, 4, dtype=torch.bool, device="cuda")
    for (r, h), v in bad.items():
        hit[r, h] = True
        assert p.y[r, h].isnan().all(), (r, h, v)
        lse = p.lse[h, r].item()
        # (+infinity less itself is a NaN, and so is an infinity split into two parts of TF32)
        assert math.isnan(lse) or lse == v and v < 0, (r, h, v, lse)
        assert v != -math.inf or mode == "3xtf32" or lse == v, (r, h, v, lse)
    y, lse = p.y.clone(), p.lse.clone()
    assert not y[~hit].isnan().any() and lse.t()[~hit].isfinite().all()
    p.backward(ctx)
    assert p.gq[hit].isnan().all() and not p.gq[:, 0].isnan().any()
    for (r, h), v in bad.items():
        seen = r + lk - lq + 1 if causal else lk
        assert p.gk[:seen, h // 2].isnan().all() and p.gv[:seen, h // 2].isnan().all()
    p.q.copy_(clean)
    p.forward(ctx)
    assert torch.equal(p.y[~hit], y[~hit]) and torch.equal(p.lse.t()[~hit], lse.t()[~hit])
    p.check()


@pytest.mark.parametrize("mode", ["fp16", "3xtf32", "tf32"])
@pytest.mark.parametrize("bad", [NAN, math.inf])
@pytest.mark.parametrize("head, lq, lk", [(64, 4, 2), (40, 60, 20), (40, 1200, 700), (256, 90, 30), (64, 300, 200), (128, 200, 90), (128, 400, 130)])
def test_queries_that_see_no_key_are_zero_whatever_stands_in_the_keys(ctx, mode, bad, head, lq, lk):
    """A causal sequence with more queries than keys: the first see nothing, whatever their q and gy, or any k and v of the sequence, hold."""
    p = Problem(mode, head, 4, 2, packed([lq, lq]), packed([lk, lk]), True, seed=62)
    none = torch.zeros(p.rows_q, dtype=torch.bool, device="cuda")
    for first, n in p.q_at:
        none[first:first + n - lk] = True
    for t in (p.q, p.gy):
        t[none] = bad
    p.forward(ctx)
    p.backward(ctx)
    assert (p.y[none] == 0).all() and (p.lse[:, none] == -math.inf).all() and (p.gq[none] == 0).all()
    clean = [t.clone() for t in (p.y, p.lse, p.gq, p.gk, p.gv)]
    assert not any(t.isnan().any() for t in clean)
    for t in (p.k, p.v):
        t[::3] = bad
    p.forward(ctx)
    assert (p.y[none] == 0).all() and (p.lse[:, none] == -math.inf).all()
    p.backward(ctx)
    assert (p.gq[none] == 0).all()
    # with zeros in those rows instead: the same bits everywhere
    p = Problem(mode, head, 4, 2, packed([lq, lq]), packed([lk, lk]), True, seed=62)
    for t in (p.q, p.gy):
        t[none] = 0.0
    p.forward(ctx)
    p.backward(ctx)
    assert all(torch.equal(a, b) for a, b in zip(clean, (p.y, p.lse, p.gq, p.gk, p.gv)))


@pytest.mark.parametrize("head", [128, 40, 33, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("big", [3e4, math.inf])
def test_a_query_beside_one_with_a_huge_gradient(ctx, head, causal, big):
    """Gradients of queries do not mix: rows whose gy is 2^-14 keep their bits in a tile with rows of 3e4, or of infinities."""
    at = packed([700])
    p = Problem("fp16", head, 2, 1, at, at, causal, seed=63, gy_size=2.0 ** -14)
    loud = torch.zeros(700, dtype=torch.bool, device="cuda")
    loud[[3, 64, 130, 131, 400, 699]] = True
    p.gy[loud] = math.copysign(1.0, big) * big
    p.forward(ctx)
    p.backward(ctx)
    for h in range(2):
        gy = p.gy[:, h].double()
        gy[loud] = 0.0          # what the others' gradients may lose is counted from their own gy
        val, tol = attention(p.q[:, h].double(), p.k[:, 0].double(), p.v[:, 0].double(), p.scale, causal, gy, "fp16")
        off = abs(p.gq[:, h].double() - val["gq"]) - tol["gq"]
        assert not (off[~loud] > 0).any() and not p.gq[~loud, h].isnan().any(), off[~loud].max().item()


def test_fp32_gradients_leave_the_scratch_of_halves_alone(ctx):
    """Squares' sums are for the scales of halves: other modes neither read all of v for them nor store any."""
    at = packed([130, 40], gap=2)
    p = Problem("3xtf32", 64, 4, 2, at, at, True, seed=65, gap=3)
    p.forward(ctx)
    p.backward(ctx)
    p.check(gradients=True)
    used = p.rows_q * p.hq
    assert p.scratch[used:].isnan().all() and not p.scratch[:used].view(p.hq, p.rows_q)[:, :130].isnan().any()
