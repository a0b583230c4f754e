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
