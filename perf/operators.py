"""The operators of attention layers as they are measured: rotary positions, head norms with the
rotation in one pass, and attention over packed sequences.

`run` computes one pass through one operator on what `prepare` made: in elementary torch operations where
`own` is false, with this library's kernels where it is true.  Layouts are the library's: a tensor of heads
is Shape({head, heads, tokens}), column-major, which torch sees as [tokens, heads, head].
"""
import math

import numpy as np
import torch

own = False

_DTYPE = {"fp16": torch.float16, "fp32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------------

def _rotary(name, direction, dtype, tokens, heads, head, rot, layout, scaling="plain", far=0, fused=False):
    return dict(name=name, op="rotary", direction=direction, dtype=dtype, tokens=tokens, heads=heads, head=head, rot=rot,
                layout=layout, scaling=scaling, far=far, fused=fused)


def _norm_rotary(name, direction, dtype, tokens, heads_q, heads_k, head, rot, layout, far=0, fused=True):
    return dict(name=name, op="norm_rotary", direction=direction, dtype=dtype, tokens=tokens, heads_q=heads_q, heads_k=heads_k,
                head=head, rot=rot, layout=layout, far=far, fused=fused)


def _attention(name, direction, dtype, seqs, longest_q, longest_k, spread, heads_q, heads_k, head, causal=True, fused=False):
    return dict(name=name, op="attention", direction=direction, dtype=dtype, seqs=seqs, longest_q=longest_q, longest_k=longest_k,
                spread=spread, heads_q=heads_q, heads_k=heads_k, head=head, causal=causal, fused=fused)


def listed():
    return [
        # one new token for each of 48 running sequences, a quarter of each head rotated, far into their contexts
        _rotary("rotary_tokens", "fw", "fp32", 48, 40, 128, 32, "pairs", far=100000),
        # queries and keys of a long prompt, out of the fused product of queries, keys and values
        _rotary("rotary_prompt", "fw", "fp16", 16384, 40, 128, 128, "halves", scaling="by_parts", fused=True),
        # gradient of a training batch with an odd number of tokens
        _rotary("rotary_gradient", "bw", "fp32", 4099, 24, 64, 64, "pairs"),
        # one new token for each of a few sequences: latency
        _norm_rotary("norm_rotary_tokens", "fw", "fp16", 7, 32, 8, 128, 128, "halves", far=30000),
        # a training batch, forward
        _norm_rotary("norm_rotary_batch", "fw", "fp16", 16384, 32, 8, 128, 128, "halves"),
        # the same batch's gradients, gains among them
        _norm_rotary("norm_rotary_gradient", "bw", "fp16", 16384, 32, 8, 128, 128, "halves"),
        # one new token against a long cache: latency, and keys read by many processors
        _attention("attention_one_token", "fw", "fp16", 1, 1, 32768, "even", 32, 8, 128),
        # a batch of running sequences of every length, one token each
        _attention("attention_tokens", "fw", "fp16", 64, 1, 8192, "ragged", 32, 8, 128),
        # prompts of very different lengths, packed one behind the other
        _attention("attention_prompts", "fw", "fp16", 12, 4096, 0, "ragged", 32, 8, 128, fused=True),
        # one long prompt
        _attention("attention_long", "fw", "fp16", 1, 16384, 0, "even", 32, 8, 128),
        # a training step on packed sequences: forward and all gradients
        _attention("attention_step", "step", "fp16", 6, 4096, 0, "ragged", 16, 4, 128),
        # a small model's training step in the default numeric mode, heads of 64, no mask
        _attention("attention_step_fp32", "step", "fp32", 8, 509, 0, "even", 8, 8, 64, causal=False),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "norm_rotary", "attention", "attention"])
    dtype = rng.choice(["fp16", "fp16", "fp32"])
    if op != "attention":
        head = rng.choice([48, 64, 80, 96, 128, 128, 192, 256])
        rot = rng.choice([head, head, head // 2, head // 4])
        layout = rng.choice(["pairs", "halves"])
        heads_k = rng.randint(1, 8)
        heads_q = heads_k * rng.choice([1, 2, 4, 7])
        most = 16384 * 40 * 128 // ((heads_q + heads_k) * head * (1 if dtype == "fp16" else 2))
        tokens = _between(rng, 1, max(1, most))
        if op == "rotary":
            return dict(op=op, direction=rng.choice(["fw", "bw"]), dtype=dtype, tokens=tokens, heads=heads_q + heads_k, head=head, rot=rot,
                        layout=layout, scaling=rng.choice(["plain", "linear", "by_parts"]), far=_between(rng, 1, 1000000),
                        fused=rng.random() < 0.5)
        return dict(op=op, direction=rng.choice(["fw", "bw"]), dtype=dtype, tokens=tokens, heads_q=heads_q, heads_k=heads_k, head=head,
                    rot=rot, layout=layout, far=_between(rng, 1, 1000000), fused=rng.random() < 0.5)
    head = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    heads_k = rng.choice([1, 2, 4, 8])
    heads_q = heads_k * rng.choice([1, 2, 4, 8])
    kind = rng.choice(["tokens", "prompt", "prompt", "step", "step"])
    c = dict(op=op, dtype=dtype, heads_q=heads_q, heads_k=heads_k, head=head, spread=rng.choice(["even", "ragged"]),
             causal=rng.random() < 0.75, fused=False)
    if kind == "tokens":
        c.update(direction="fw", seqs=_between(rng, 1, 64), longest_q=rng.choice([1, 1, 1, 2, 4]), longest_k=_between(rng, 8, 32768))
        while c["seqs"] * c["longest_k"] * heads_k * head > 64 * 8192 * 8 * 128:
            c["seqs"] = (c["seqs"] + 1) // 2
    else:
        c.update(direction="fw" if kind == "prompt" else "step", seqs=_between(rng, 1, 24), longest_q=_between(rng, 24, 8192), longest_k=0,
                 fused=rng.random() < 0.5)
        # against the largest listed case of its kind, with fp32 at an eighth of the rate
        most = (1.0 if kind == "prompt" else 0.05) * (1.0 if dtype == "fp16" else 0.02) * 32 * 16384.0 ** 2 * 128 / 2
        while heads_q * head * c["seqs"] * float(c["longest_q"]) ** 2 > most:
            if c["seqs"] > 1:
                c["seqs"] -= 1
            else:
                c["longest_q"] = c["longest_q"] * 3 // 4
    return c


def _lengths(seqs, longest, spread):
    """The lengths of a batch: all the longest, or spread from one up to it by a fixed rule."""
    if spread == "even":
        return [longest] * seqs
    return [longest if i == 0 else 1 + (i * 2654435761 % 4294967296) % longest for i in range(seqs)]


def _sequences(c):
    """(first row and length of each sequence's queries, the same of its keys, rows of q, rows of k)."""
    if c["longest_k"]:  # against a cache: room for the longest, each sequence filled as far as it has come
        lk = [max(n, c["longest_q"]) for n in _lengths(c["seqs"], c["longest_k"], c["spread"])]
        room = max(lk)
        q = [(i * c["longest_q"], c["longest_q"]) for i in range(c["seqs"])]
        k = [(i * room, n) for i, n in enumerate(lk)]
        return q, k, c["seqs"] * c["longest_q"], c["seqs"] * room
    n = _lengths(c["seqs"], c["longest_q"], c["spread"])
    at = [sum(n[:i]) for i in range(len(n))]
    q = list(zip(at, n))
    return q, q, sum(n), sum(n)


def work(c):
    es = 2 if c["dtype"] == "fp16" else 4
    if c["op"] == "attention":
        q, k, rows_q, _ = _sequences(c)
        keys = sum(n for _, n in k)
        pairs = 0
        for (_, lq), (_, lk) in zip(q, k):
            pairs += lq * lk - (lq * (lq - 1) // 2 if c["causal"] else 0)
        at_q, at_k = rows_q * c["heads_q"] * c["head"] * es, keys * c["heads_k"] * c["head"] * es
        flops = 4 * c["head"] * c["heads_q"] * pairs
        if c["direction"] == "fw":
            return {"bytes": 2 * at_q + 2 * at_k, "flops": flops}
        return {"bytes": 4 * at_q + 4 * at_k, "flops": flops * 7 // 2}
    heads = c["heads"] if c["op"] == "rotary" else c["heads_q"] + c["heads_k"]
    n = c["tokens"] * heads * c["head"]
    if c["op"] == "rotary":
        return {"bytes": 2 * n * es, "flops": 3 * c["tokens"] * heads * c["rot"]}
    passes, flops = (2, 7) if c["direction"] == "fw" else (3, 14)
    return {"bytes": passes * n * es, "flops": flops * n}


# ---- what a program has in hand before the call ----------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, scale, generator=gen).to(dtype)


def _frequencies(rot, scaling, base=10000.0, factor=8.0, original=4096.0):
    """Radians a position for each pair, and the factor on the rotated values."""
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "by_parts":
        # pairs that turn fewer than once over the original length are interpolated, those that turn more than 32
        # times are kept, and between the two it goes over linearly in the number of the pair
        def pair(turns):
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot // 2 - 1)
        keep = 1.0 - np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f / factor * (1.0 - keep) + f * keep, 0.1 * math.log(factor) + 1.0
    return f, 1.0


class _State:
    pass


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = _State()
    s.case, c = dict(case), case
    dtype = _DTYPE[c["dtype"]]
    if own:
        import primitiv_b200 as pb
        s.ctx = _context(pb)
        s.mode = pb.MODE_FP16 if c["dtype"] == "fp16" else pb.MODE_FP32_3XTF32
    if c["op"] == "attention":
        _prepare_attention(s, c, gen, dtype)
    else:
        _prepare_rotary(s, c, gen, dtype)
    torch.cuda.synchronize()
    return s


_CTX = []


def _context(pb):
    """The library's context: a program has one for its life."""
    if not _CTX:
        _CTX.append(pb.Context(torch.cuda.current_device()))
    return _CTX[0]


def _prepare_rotary(s, c, gen, dtype):
    t, d = c["tokens"], c["head"]
    heads = c["heads"] if c["op"] == "rotary" else c["heads_q"] + c["heads_k"]
    # where the heads come out of one fused product, as many values stand behind them for each token
    row = heads + (max(1, heads // 5) if c["fused"] else 0)
    s.heads = heads
    s.x = _normal(gen, (t, row, d), dtype)[:, :heads]
    if c["far"] and t <= 4096:  # tokens of running sequences, each at a place of its own
        s.positions = torch.randint(0, c["far"], (t,), device="cuda", generator=gen, dtype=torch.int64).to(torch.int32)
    else:  # whole sequences, one behind the other
        s.positions = torch.arange(t, device="cuda", dtype=torch.int32) % max(1, min(t, 8192)) + int(c["far"])
    freqs, s.amplitude = _frequencies(c["rot"], c.get("scaling", "plain"))
    s.freqs = torch.from_numpy(freqs).cuda()
    s.y = torch.empty((t, heads, d), device="cuda", dtype=dtype)
    if c["op"] == "norm_rotary":
        s.eps = 1e-6
        s.gain_q = _normal(gen, (d,), torch.float32, 0.2).add_(1.0).to(dtype)
        s.gain_k = _normal(gen, (d,), torch.float32, 0.2).add_(1.0).to(dtype)
        if c["direction"] == "bw":
            s.gy = _normal(gen, (t, heads, d), dtype, 0.05)
            s.ggain_q, s.ggain_k = torch.empty_like(s.gain_q), torch.empty_like(s.gain_k)
            if own:
                import primitiv_b200 as pb
                s.scratch = torch.empty(pb.NORM_ROTARY_SCRATCH, device="cuda", dtype=torch.float32)


def _prepare_attention(s, c, gen, dtype):
    d, hq, hk = c["head"], c["heads_q"], c["heads_k"]
    s.q_at, s.k_at, rows_q, rows_k = _sequences(c)
    if c["fused"]:  # one product's output holds the queries, keys and values of a token side by side
        qkv = _normal(gen, (rows_q, hq + 2 * hk, d), dtype)
        s.q, s.k, s.v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        s.q, s.k, s.v = (_normal(gen, (r, h, d), dtype) for r, h in ((rows_q, hq), (rows_k, hk), (rows_k, hk)))
    s.scale = 1.0 / math.sqrt(d)
    s.y = torch.empty((rows_q, hq, d), device="cuda", dtype=dtype)
    if c["direction"] == "step":
        s.gy = _normal(gen, (rows_q, hq, d), dtype, 0.05)
        s.lse = torch.empty((hq, rows_q), device="cuda", dtype=torch.float32)
    if own:
        import primitiv_b200 as pb

        def on_gpu(values):
            return torch.tensor(values, dtype=torch.int32, device="cuda")
        s.q_starts = on_gpu([at for at, _ in s.q_at] + [rows_q])
        s.k_starts = on_gpu([at for at, _ in s.k_at] + [rows_k])
        s.k_lens = on_gpu([n for _, n in s.k_at])
        s.plan = pb.Attention(head=d, heads_q=hq, heads_k=hk, rows_q=rows_q, rows_k=rows_k, q_ld=s.q.stride(0), k_ld=s.k.stride(0),
                              v_ld=s.v.stride(0), y_ld=s.y.stride(0), seqs=c["seqs"], max_q=max(n for _, n in s.q_at),
                              max_k=max(n for _, n in s.k_at), q_starts=s.q_starts.data_ptr(), k_starts=s.k_starts.data_ptr(),
                              k_lens=s.k_lens.data_ptr(), causal=int(c["causal"]), scale=s.scale)
        if c["direction"] == "step":
            s.scratch = torch.empty(s.plan.bw_scratch_floats(), device="cuda", dtype=torch.float32)
            if c["fused"]:  # the gradients go where the product's backward pass wants them
                gqkv = torch.empty((rows_q, hq + 2 * hk, d), device="cuda", dtype=dtype)
                s.gq, s.gk, s.gv = gqkv[:, :hq], gqkv[:, hq:hq + hk], gqkv[:, hq + hk:]
            else:
                s.gq, s.gk, s.gv = (torch.empty_like(t) for t in (s.q, s.k, s.v))


# ---- one pass ------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _RUN_OWN[s.case["op"]](s)
    return _RUN_PLAIN[s.case["op"]](s)


def _rotary_own(s):
    c, at = s.case, torch.cuda.current_stream().cuda_stream
    layout = 0 if c["layout"] == "pairs" else 1
    if c["direction"] == "fw":
        s.ctx.rotary_fw(s.mode, s.x.data_ptr(), s.y.data_ptr(), c["head"], s.heads, c["tokens"], s.x.stride(0), s.y.stride(0), c["rot"],
                        layout, s.freqs.data_ptr(), s.amplitude, s.positions.data_ptr(), stream=at)
    else:
        s.ctx.rotary_bw(s.mode, s.x.data_ptr(), s.y.data_ptr(), c["head"], s.heads, c["tokens"], s.x.stride(0), s.y.stride(0), c["rot"],
                        layout, s.freqs.data_ptr(), s.amplitude, s.positions.data_ptr(), accumulate=False, stream=at)
    return s.y


def _norm_rotary_own(s):
    c, at = s.case, torch.cuda.current_stream().cuda_stream
    layout = 0 if c["layout"] == "pairs" else 1
    if c["direction"] == "fw":
        s.ctx.norm_rotary_fw(s.mode, s.x.data_ptr(), s.gain_q.data_ptr(), s.gain_k.data_ptr(), s.y.data_ptr(), c["head"], c["heads_q"],
                             c["heads_k"], c["tokens"], s.x.stride(0), s.y.stride(0), c["rot"], layout, s.freqs.data_ptr(), s.amplitude,
                             s.positions.data_ptr(), s.eps, stream=at)
        return s.y
    s.ctx.norm_rotary_bw(s.mode, s.x.data_ptr(), s.gain_q.data_ptr(), s.gain_k.data_ptr(), s.gy.data_ptr(), s.y.data_ptr(),
                         s.ggain_q.data_ptr(), s.ggain_k.data_ptr(), s.scratch.data_ptr(), c["head"], c["heads_q"], c["heads_k"],
                         c["tokens"], s.x.stride(0), s.gy.stride(0), s.y.stride(0), c["rot"], layout, s.freqs.data_ptr(), s.amplitude,
                         s.positions.data_ptr(), s.eps, accumulate_x=False, accumulate_gain=False, stream=at)
    return s.y, s.ggain_q, s.ggain_k


def _attention_own(s):
    at = torch.cuda.current_stream().cuda_stream
    if s.case["direction"] == "fw":
        s.ctx.attention_fw(s.mode, s.plan, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.y.data_ptr(), stream=at)
        return s.y
    s.ctx.attention_fw(s.mode, s.plan, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.y.data_ptr(), s.lse.data_ptr(), stream=at)
    s.ctx.attention_bw(s.mode, s.plan, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.y.data_ptr(), s.lse.data_ptr(), s.gy.data_ptr(),
                       s.gq.data_ptr(), s.gk.data_ptr(), s.gv.data_ptr(), s.scratch.data_ptr(), accumulate=False, stream=at)
    return s.y, s.gq, s.gk, s.gv


_RUN_OWN = {"rotary": _rotary_own, "norm_rotary": _norm_rotary_own, "attention": _attention_own}


def _angles(s):
    """cos and sin of each token's angles, [tokens, 1, rot / 2], in 32 bits from angles in 64."""
    a = s.positions.to(torch.float64)[:, None, None] * s.freqs
    return (torch.cos(a) * s.amplitude).float(), (torch.sin(a) * s.amplitude).float()


def _rotate(x, cos, sin, rot, layout):
    """x in 32 bits, [tokens, heads, head]; sin negated turns back."""
    if layout == "pairs":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), -1).flatten(-2) if layout == "pairs" else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _rotary_plain(s):
    c = s.case
    cos, sin = _angles(s)
    return _rotate(s.x.float(), cos, sin if c["direction"] == "fw" else -sin, c["rot"], c["layout"]).to(s.x.dtype)


def _norm_rotary_plain(s):
    c, hq = s.case, s.case["heads_q"]
    cos, sin = _angles(s)
    x = s.x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + s.eps)
    gain = torch.cat((s.gain_q.float().expand(hq, -1), s.gain_k.float().expand(c["heads_k"], -1)))
    if c["direction"] == "fw":
        return _rotate(x * r * gain, cos, sin, c["rot"], c["layout"]).to(s.x.dtype)
    g = _rotate(s.gy.float(), cos, -sin, c["rot"], c["layout"])
    n = x * r
    per_head = (g * n).sum(0)
    g = g * gain
    gx = r * (g - n * (g * n).mean(-1, keepdim=True))
    return gx.to(s.x.dtype), per_head[:hq].sum(0).to(s.x.dtype), per_head[hq:].sum(0).to(s.x.dtype)


def _attention_plain(s):
    c = s.case
    step = c["direction"] == "step"
    group = c["heads_q"] // c["heads_k"]
    y = s.y
    if step:
        gq, gk, gv = (torch.empty_like(t) for t in (s.q, s.k, s.v))
    for (q0, lq), (k0, lk) in zip(s.q_at, s.k_at):
        later = None
        if c["causal"] and lq > 1:
            row, col = torch.arange(lq, device="cuda")[:, None], torch.arange(lk, device="cuda")
            later = col > row + (lk - lq)
        heads = max(1, min(c["heads_k"], (1 << 28) // (group * lq * lk)))  # as many at a time as a few GB hold
        for h in range(0, c["heads_k"], heads):
            e = min(h + heads, c["heads_k"])
            # [heads of k, heads of q for each, rows, head]
            q = s.q[q0:q0 + lq, h * group:e * group].float().view(lq, e - h, group, -1).permute(1, 2, 0, 3)
            k = s.k[k0:k0 + lk, h:e].float().permute(1, 0, 2)[:, None]
            v = s.v[k0:k0 + lk, h:e].float().permute(1, 0, 2)[:, None]
            p = (q @ k.transpose(-1, -2)).mul_(s.scale)
            if later is not None:
                p.masked_fill_(later, -math.inf)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True))
            y[q0:q0 + lq, h * group:e * group] = (p @ v).permute(2, 0, 1, 3).reshape(lq, (e - h) * group, -1).to(y.dtype)
            if step:
                g = s.gy[q0:q0 + lq, h * group:e * group].float().view(lq, e - h, group, -1).permute(1, 2, 0, 3)
                gv[k0:k0 + lk, h:e] = (p.transpose(-1, -2) @ g).sum(1).permute(1, 0, 2).to(y.dtype)
                gs = g @ v.transpose(-1, -2)
                gs = gs.sub_((p * gs).sum(-1, keepdim=True)).mul_(p).mul_(s.scale)
                gq[q0:q0 + lq, h * group:e * group] = (gs @ k).permute(2, 0, 1, 3).reshape(lq, (e - h) * group, -1).to(y.dtype)
                gk[k0:k0 + lk, h:e] = (gs.transpose(-1, -2) @ q).sum(1).permute(1, 0, 2).to(y.dtype)
    return (y, gq, gk, gv) if step else y


_RUN_PLAIN = {"rotary": _rotary_plain, "norm_rotary": _norm_rotary_plain, "attention": _attention_plain}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _rotary_exact, "norm_rotary": _norm_rotary_exact, "attention": _attention_exact}[case["op"]](s)


def _turn(x, s, c, back=False):
    """Each pair as a complex number times amplitude * exp(i angle); `back`: the transposed map."""
    rot = c["rot"]
    angle = s.positions.double()[:, None] * s.freqs
    unit = torch.polar(torch.full_like(angle, s.amplitude), -angle if back else angle)[:, None, :]
    y = x.clone()
    if c["layout"] == "pairs":
        y[..., :rot] = torch.view_as_real(torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * unit).flatten(-2)
    else:
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * unit
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def _rotary_exact(s):
    return _turn(s.x.double(), s, s.case, back=s.case["direction"] == "bw")


def _norm_rotary_exact(s):
    c, hq = s.case, s.case["heads_q"]
    fw = c["direction"] == "fw"
    at = 2048  # tokens at a time
    ys, gxs, ggq, ggk = [], [], 0.0, 0.0
    for t in range(0, c["tokens"], at):
        part = _State()
        part.positions, part.freqs, part.amplitude = s.positions[t:t + at], s.freqs, s.amplitude
        x = s.x[t:t + at].double()
        size = torch.sqrt(x.square().sum(-1, keepdim=True) / c["head"] + s.eps)
        gain = torch.stack([s.gain_q.double()] * hq + [s.gain_k.double()] * c["heads_k"])
        if fw:
            ys.append(_turn(x / size * gain, part, c))
            continue
        with torch.enable_grad():
            x.requires_grad_(True)
            gain.requires_grad_(True)
            n = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["head"] + s.eps) * gain
            gx, gg = torch.autograd.grad(n, (x, gain), _turn(s.gy[t:t + at].double(), part, c, back=True))
        gxs.append(gx)
        ggq, ggk = ggq + gg[:hq].sum(0), ggk + gg[hq:].sum(0)
    return torch.cat(ys) if fw else (torch.cat(gxs), ggq, ggk)


def _attention_exact(s):
    c = s.case
    group, step = c["heads_q"] // c["heads_k"], c["direction"] == "step"
    y = torch.zeros(s.y.shape, dtype=torch.float64, device="cuda")
    if step:
        gq, gk, gv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (s.q, s.k, s.v))
    for (q0, lq), (k0, lk) in zip(s.q_at, s.k_at):
        seen = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = seen.tril(lk - lq)
        for h in range(c["heads_q"]):
            kh = h // group
            q, k, v = (t.double() for t in (s.q[q0:q0 + lq, h], s.k[k0:k0 + lk, kh], s.v[k0:k0 + lk, kh]))
            with torch.set_grad_enabled(step):
                if step:
                    q.requires_grad_(True), k.requires_grad_(True), v.requires_grad_(True)
                weights = torch.einsum("id,jd->ij", q * s.scale, k).masked_fill(~seen, -math.inf)
                out = torch.einsum("ij,jd->id", torch.exp(weights - torch.logsumexp(weights, 1)[:, None]), v)
                if step:
                    a, b, e = torch.autograd.grad(out, (q, k, v), s.gy[q0:q0 + lq, h].double())
                    gq[q0:q0 + lq, h] = a
                    gk[k0:k0 + lk, kh] += b
                    gv[k0:k0 + lk, kh] += e
            y[q0:q0 + lq, h] = out.detach()
    return (y, gq, gk, gv) if step else y
