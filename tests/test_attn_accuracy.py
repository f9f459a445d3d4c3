"""The bound that the cache attention's f32 and f16 rows are held to lets two f16 terms pass and nothing less."""
import pytest

from attn_accuracy import TOKENS, case, formula, tolerance, with_terms


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_one_term_less_is_seen(dt, n, hd, fmt):
    q, k, v, ks, vs = case(fmt, dt, n, 8, hd, n + hd)
    o, a, s = formula(q, k, v, ks, vs)
    tol = tolerance(o, a, s, vs, dt)
    worst = lambda q_terms, w_terms: float((abs(with_terms(q, k, v, ks, vs, dt, q_terms, w_terms) - o) / tol).max())      # noqa: E731
    assert worst(2, 2) < 1.0
    assert worst(2, 1) > 1.0
    if dt == "f32":
        assert worst(1, 2) > 1.0 and worst(1, 1) > 1.0
