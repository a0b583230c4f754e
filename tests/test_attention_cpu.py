"""The attention layer's operators without a GPU: frequencies, the scratch a plan asks for, and what a plan is refused for."""
import ctypes
import math

import pytest

import primitiv_b200 as pb


def test_plain_frequencies():
    freqs, amplitude = pb.rotary_frequencies(8, 10000.0)
    assert amplitude == 1.0
    assert freqs == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)


def test_scaled_frequencies():
    plain, _ = pb.rotary_frequencies(64, 10000.0)
    linear, amplitude = pb.rotary_frequencies(64, 10000.0, "linear", 4.0)
    assert amplitude == 1.0 and linear == pytest.approx([f / 4 for f in plain], rel=1e-15)
    based, amplitude = pb.rotary_frequencies(64, 10000.0, "base", 4.0)
    assert amplitude == 1.0 and based[0] == 1.0
    assert based[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)          # the slowest pair is interpolated by the factor
    assert all(a >= b >= a / 4 * (1 - 1e-12) for a, b in zip(plain, based))
    parts, amplitude = pb.rotary_frequencies(64, 10000.0, "by_parts", 4.0, 4096.0)
    assert amplitude == pytest.approx(1 + 0.1 * math.log(4.0), rel=1e-15)
    turns = [4096.0 * f / (2 * math.pi) for f in plain]
    for f, g, n in zip(plain, parts, turns):
        if n > 40:
            assert g == pytest.approx(f, rel=1e-15)
        elif n < 0.7:
            assert g == pytest.approx(f / 4, rel=1e-15)
        else:
            assert f / 4 * (1 - 1e-12) <= g <= f * (1 + 1e-12)


def blend(rot, base, factor, original):
    """By the definition: floor and ceiling of the pairs that turn 32 times and once, wherever those lie."""
    at = [rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    first, last = math.floor(at[0]), math.ceil(at[1])
    freqs = []
    for p in range(rot // 2):
        slow = min(max((p - first) / (last - first), 0.0), 1.0)
        freqs.append(base ** (-2 * p / rot) * (1 - slow + slow / factor))
    return freqs


@pytest.mark.parametrize("rot, base, factor, original", [
    (8, 1e4, 4.0, 8192.0), (128, 1e4, 4.0, 65536.0), (128, 1e4, 4.0, 131072.0), (64, 1e4, 8.0, 1e6), (2, 1e4, 4.0, 4096.0), (12, 5e5, 2.0, 1e9),
    (64, 1e4, 4.0, 64.0), (64, 1e4, 4.0, 5.0), (128, 1e4, 8.0, 4096.0), (6, 10.0, 3.0, 1.0), (256, 1.5, 3.0, 1e30),
])
def test_blended_frequencies(rot, base, factor, original):
    """The blend's ends may lie before the first pair and behind the last: pairs of long contexts all turn more than once."""
    freqs, amplitude = pb.rotary_frequencies(rot, base, "by_parts", factor, original)
    assert amplitude == pytest.approx(1 + 0.1 * math.log(factor), rel=1e-15)
    assert freqs == pytest.approx(blend(rot, base, factor, original), rel=1e-14)
    for p, f in enumerate(freqs):
        plain = base ** (-2 * p / rot)
        turns = original * plain / (2 * math.pi)
        if turns < 1 - 1e-9:
            assert f == pytest.approx(plain / factor, rel=1e-14)
        elif turns > 32 + 1e-9:
            assert f == pytest.approx(plain, rel=1e-14)


def test_a_last_pair_that_turns_more_than_once_is_half_blended():
    """8 elements, base 10000, 8192 positions: the last pair turns 1.3 times; the blend runs from pair 1 to pair 4."""
    freqs, _ = pb.rotary_frequencies(8, 1e4, "by_parts", 4.0, 8192.0)
    assert freqs == pytest.approx([1.0, 0.1, 0.01 * 0.75, 0.001 * 0.5], rel=1e-12)


@pytest.mark.parametrize("args", [(0,), (7,), (8, 1.0), (8, math.nan), (8, 1e4, "linear", 0.5), (8, 1e4, "by_parts", 2.0, 0.0),
                                  (8, 1e4, "base", math.inf)])
def test_refused_frequencies(args):
    with pytest.raises(pb.B200Error) as e:
        pb.rotary_frequencies(*args)
    assert e.value.code == 1001


def test_unknown_scaling():
    with pytest.raises(ValueError):
        pb.rotary_frequencies(8, 1e4, "cubic", 2.0)


def plan(**more):
    fields = dict(head=64, heads_q=8, heads_k=2, rows_q=100, rows_k=70, seqs=3, causal=1, scale=0.125)
    fields.update(more)
    return pb.Attention(**fields)


def test_scratch():
    assert plan().bw_scratch_floats() == 2 * 100 * 8 + 70 * 2
    assert plan(rows_q=0, rows_k=0).bw_scratch_floats() == 0
    assert plan(rows_q=1 << 24, heads_q=64, heads_k=64, rows_k=1 << 24).bw_scratch_floats() == 3 << 30


@pytest.mark.parametrize("code, more", [
    (1001, dict(head=0)), (1006, dict(head=257)), (1001, dict(heads_q=0)), (1001, dict(heads_k=0)), (1001, dict(heads_q=7)),
    (1001, dict(scale=math.nan)), (1001, dict(scale=math.inf)), (1001, dict(q_ld=511)), (1001, dict(y_ld=1)), (1001, dict(k_ld=127)),
    (1001, dict(v_ld=127)), (1006, dict(rows_q=1 << 30)), (1006, dict(rows_k=1 << 31)), (1006, dict(seqs=1 << 30)),
    (1006, dict(heads_q=65536, heads_k=65536)),
])
def test_refused_plans(code, more):
    with pytest.raises(pb.B200Error) as e:
        plan(**more).bw_scratch_floats()
    assert e.value.code == code


@pytest.mark.parametrize("more", [dict(rows_k=(1 << 31) - 1, heads_k=1, head=1), dict(rows_q=(1 << 31) - 1, heads_q=1, heads_k=1, head=1),
                                  dict(rows_q=1, heads_q=1 << 24, heads_k=1, head=256)])
def test_sizes_whose_indexes_would_wrap_are_refused(more):
    """A tile that ends behind the last row, and the elements of a token, are counted in 32 bits."""
    with pytest.raises(pb.B200Error) as e:
        plan(**more).bw_scratch_floats()
    assert e.value.code == 1006


def test_the_largest_sizes_are_taken():
    assert plan(rows_k=(1 << 31) - (1 << 16), heads_k=1, head=1).bw_scratch_floats() == 2 * 100 * 8 + (1 << 31) - (1 << 16)
    assert plan(rows_q=1, heads_q=1 << 22, heads_k=1, head=256).bw_scratch_floats() == (2 << 22) + 70


def test_entry_points_refuse_a_null_context_and_plan():
    lib, n = pb.lib(), ctypes.c_uint64()
    p = ctypes.addressof(plan())
    assert lib.b200_attention_bw_scratch(None, ctypes.addressof(n)) == 1001
    assert lib.b200_attention_bw_scratch(p, None) == 1001
    assert lib.b200_attention_fw(None, 2, p, 1, 1, 1, 1, 0, None) == 1001
    assert lib.b200_attention_bw(None, 2, p, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 0, None) == 1001
    assert lib.b200_rotary_fw(None, 2, 1, 1, 64, 1, 1, 0, 0, 64, 0, 1, 1.0, None, None) == 1001
    assert lib.b200_rotary_bw(None, 2, 1, 1, 64, 1, 1, 0, 0, 64, 0, 1, 1.0, None, 0, None) == 1001
    assert lib.b200_norm_rotary_fw(None, 2, 1, 1, 1, 1, 64, 1, 1, 1, 0, 0, 64, 0, 1, 1.0, None, 1e-6, None) == 1001
    assert lib.b200_norm_rotary_bw(None, 2, 1, 1, 1, 1, 1, 1, 1, 1, 64, 1, 1, 1, 0, 0, 0, 64, 0, 1, 1.0, None, 1e-6, 0, 0, None) == 1001
