"""Causal attention over packed prompts against the formula in 64 bits; the bounds are derived in attn_reference.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attn_reference import HALF_STEP, attend, tolerance  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def be():
    from tensorpencil_b200.backend import Backend
    b = Backend(0)
    yield b
    b.close()


def make(total, heads, kv, hd, dt, seed, scale_q=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn((total, h * hd), generator=g) for h in (heads, kv, kv))
    return [(t * s).to(DT[dt]).cuda() for t, s in ((q, scale_q), (k, 1.0), (v, 1.0))]


def offsets(lens, first=0):
    return torch.tensor(np.cumsum([first] + list(lens)), dtype=torch.int32).cuda()


def check(out, q, k, v, lens, heads, kv, hd, dt, first=0, scale=None, rows_at_most=60):
    """Every head; the sequences' rows, at most `rows_at_most` of each (the first, the last and others)."""
    group = heads // kv
    scale = hd ** -0.5 if scale is None else scale
    got, q, k, v = (t.double().cpu().numpy() for t in (out, q, k, v))
    rng = np.random.default_rng(5)
    at = first
    for n in lens:
        rows = np.arange(n) if n <= rows_at_most else np.unique(np.concatenate([[0, 1, 127, 128, n - 2, n - 1], rng.choice(n, rows_at_most - 6)]) % n)
        for h in range(heads):
            mine, of = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
            o, a, e = attend(q[at + rows][:, mine], k[at:at + n, of], v[at:at + n, of], rows, scale)
            tol = tolerance(o, a, e, hd, HALF_STEP[dt], HALF_STEP[dt])
            err = np.abs(got[at + rows][:, mine] - o)
            assert (err <= tol).all(), (n, h, float((err / tol).max()))
        at += n


CASES = [([1], 2, 1, 128), ([13], 8, 2, 128), ([128], 4, 4, 64), ([129, 1, 0, 255], 4, 2, 128), ([300, 77, 512], 7, 1, 64),
         ([64, 65, 31], 14, 2, 128), ([1, 1, 1, 1, 1, 2], 3, 3, 64), ([700], 5, 1, 128), ([5, 40], 128, 1, 64), ([257], 64, 1, 128),
         ([1100, 3], 12, 4, 128), ([0, 0, 9], 6, 2, 64), ([400, 130], 33, 1, 64)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("lens,heads,kv,hd", CASES)
def test_matches_the_formula(be, lens, heads, kv, hd, dt):
    total = sum(lens)
    q, k, v = make(total, heads, kv, hd, dt, total + heads)
    out = be.attentionPacked(q, k, v, offsets(lens), heads, kv, hd)
    be.status_poll()
    check(out, q, k, v, lens, heads, kv, hd, dt)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_scores_of_a_wide_range(be, dt):
    """Scores of several hundred: the running maximum moves far, and most weights vanish."""
    lens = [500, 333]
    q, k, v = make(sum(lens), 4, 2, 128, dt, 3, scale_q=60.0)
    q[:, 0] = 30.0
    k[::37, 0] = 40.0                                     # maxima that come late
    out = be.attentionPacked(q, k, v, offsets(lens), 4, 2)
    check(out, q, k, v, lens, 4, 2, 128, dt)


@pytest.mark.parametrize("scale", [0.0, 0.01, 1.0])
def test_scale(be, scale):
    q, k, v = make(200, 2, 1, 64, "f16", 4)
    check(be.attentionPacked(q, k, v, offsets([200]), 2, 1, 64, scale=scale), q, k, v, [200], 2, 1, 64, "f16", scale=scale)


@pytest.mark.parametrize("hd", [64, 128])
def test_parts_of_a_fused_projection_and_an_output_of_its_own_stride(be, hd):
    heads, kv, lens = 6, 2, [150, 90]
    total = sum(lens)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn((total, (heads + 2 * kv) * hd + 24), generator=g).bfloat16().cuda()
    q, k, v = fused[:, :heads * hd], fused[:, heads * hd:(heads + kv) * hd], fused[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
    wide = torch.full((total, heads * hd + 40), 7.0, dtype=torch.bfloat16).cuda()
    out = be.attentionPacked(q, k, v, offsets(lens), heads, kv, hd, out=wide[:, 8:8 + heads * hd])
    check(out, q, k, v, lens, heads, kv, hd, "bf16")
    assert (wide[:, :8] == 7.0).all() and (wide[:, 8 + heads * hd:] == 7.0).all()
    same = be.attentionPacked(q.reshape(total, heads, hd), k.reshape(total, kv, hd), v.reshape(total, kv, hd), offsets(lens), heads, kv, hd)
    assert torch.equal(same, out)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_is_no_part_of_it(be, bad):
    """NaN and infinities in rows of no sequence (in front, behind), in another sequence and in later tokens of the same one."""
    heads, kv, hd, lens, first = 4, 2, 128, [200, 70, 130], 11
    total = first + sum(lens) + 9
    q, k, v = make(total, heads, kv, hd, "bf16", 9)
    clean = be.attentionPacked(q, k, v, offsets(lens, first), heads, kv, hd)
    for t in (k, v):
        t[:first] = bad
        t[first + sum(lens):] = bad
        t[first + 200:first + 270] = bad                   # the whole second sequence
        t[first + 270 + 100, :hd] = bad                    # one token of the third, one head
    out = torch.full((total, heads * hd), 3.0, dtype=torch.bfloat16).cuda()
    be.attentionPacked(q, k, v, offsets(lens, first), heads, kv, hd, out=out)
    be.status_poll()
    assert (out[:first] == 3.0).all() and (out[first + sum(lens):] == 3.0).all()
    third = first + 270
    assert torch.equal(out[first:first + 200], clean[first:first + 200])
    assert torch.equal(out[third:third + 100], clean[third:third + 100])
    assert torch.equal(out[third + 100:third + 130, 2 * hd:], clean[third + 100:third + 130, 2 * hd:])     # the other kv head
    assert torch.isnan(out[third + 100:third + 130, :2 * hd]).all()        # bad keys: no finite row behind them
    assert torch.isnan(out[first + 200:first + 270]).all()


def test_an_infinite_or_nan_value_reaches_the_rows_that_see_it(be):
    heads, kv, hd, n = 2, 1, 64, 300
    q, k, v = make(n, heads, kv, hd, "f16", 12)
    clean = be.attentionPacked(q, k, v, offsets([n]), heads, kv, hd)
    v[130, 3], v[200, 5], v[40, 7], v[260, 7] = float("inf"), float("nan"), float("inf"), -float("inf")
    out = be.attentionPacked(q, k, v, offsets([n]), heads, kv, hd).view(n, heads, hd)
    clean = clean.view(n, heads, hd)
    assert torch.equal(out[:130, :, 3], clean[:130, :, 3]) and (out[130:, :, 3] == float("inf")).all()
    assert torch.equal(out[:200, :, 5], clean[:200, :, 5]) and torch.isnan(out[200:, :, 5]).all()
    assert torch.equal(out[:40, :, 7], clean[:40, :, 7]) and (out[40:260, :, 7] == float("inf")).all() and torch.isnan(out[260:, :, 7]).all()
    rest = [c for c in range(hd) if c not in (3, 5, 7)]
    assert torch.equal(out[:, :, rest], clean[:, :, rest])


def test_offsets_out_of_range_are_clamped(be):
    heads, kv, hd = 2, 1, 64
    q, k, v = make(100, heads, kv, hd, "bf16", 2)
    cu = torch.tensor([-5, 40, 1000], dtype=torch.int32).cuda()
    out = be.attentionPacked(q, k, v, cu, heads, kv, hd)
    check(out, q, k, v, [40, 60], heads, kv, hd, "bf16")


def test_many_sequences(be):
    """More sequences than one step of the search looks at, and empty ones among them."""
    rng = np.random.default_rng(0)
    lens = [int(n) for n in rng.integers(0, 6, 1500)]
    q, k, v = make(sum(lens), 4, 1, 64, "f16", 8)
    out = be.attentionPacked(q, k, v, offsets(lens), 4, 1, 64)
    check(out, q, k, v, lens[:150], 4, 1, 64, "f16")
    o2 = be.attentionPacked(q[-500:], k[-500:], v[-500:], offsets(lens)[-100:] - (sum(lens) - 500), 4, 1, 64)
    at = int(offsets(lens)[-100]) - (sum(lens) - 500)
    assert torch.equal(o2[at:], out[-(500 - at):])


def test_captured_and_replayed_with_other_lengths(be):
    heads, kv, hd = 8, 2, 128
    q, k, v = make(300, heads, kv, hd, "bf16", 6)
    cu = offsets([100, 200])
    out = torch.zeros((300, heads * hd), dtype=torch.bfloat16).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        be.attentionPacked(q, k, v, cu, heads, kv, hd, out=out)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.attentionPacked(q, k, v, cu, heads, kv, hd, out=out)
    for lens in ([100, 200], [299, 1], [0, 300]):
        cu.copy_(offsets(lens))
        g.replay()
        torch.cuda.synchronize()
        check(out, q, k, v, lens, heads, kv, hd, "bf16", rows_at_most=20)


def test_runs_on_the_callers_stream_and_gives_the_same_bits_again(be):
    lens = [777, 129, 1]
    q, k, v = make(sum(lens), 8, 2, 128, "bf16", 10)
    a = be.attentionPacked(q, k, v, offsets(lens), 8, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = torch.zeros_like(q)
        x.copy_(q)
        b = be.attentionPacked(x, k, v, offsets(lens), 8, 2)
    s.synchronize()
    assert torch.equal(a, b)


def test_no_tokens_and_no_sequences(be):
    q, k, v = make(0, 4, 2, 64, "bf16", 0)
    assert be.attentionPacked(q, k, v, offsets([0, 0]), 4, 2, 64).shape == (0, 256)
    q, k, v = make(5, 4, 2, 64, "bf16", 0)
    out = torch.full((5, 256), 2.0, dtype=torch.bfloat16).cuda()
    be.attentionPacked(q, k, v, offsets([]), 4, 2, 64, out=out)
    assert (out == 2.0).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_more_pairs_of_tiles_than_the_gpu_has_sms(be, hd):
    """Pairs of tiles that follow one another in one block: each sequence's rows come out as they do alone, with and without NaN and infinities that
    some of its rows see, whatever the pair before it saw."""
    rng = np.random.default_rng(hd)
    heads, kv = 16, 8
    lens = [int(n) for n in rng.choice([1, 60, 129, 300, 411], 90)]
    q, k, v = make(sum(lens), heads, kv, hd, "bf16", 21)
    starts = np.cumsum([0] + lens)
    for i in range(0, 90, 3):
        v[starts[i] + int(rng.integers(0, lens[i])), int(rng.integers(0, kv * hd))] = (float("nan"), float("inf"), -float("inf"))[i // 3 % 3]
    out = be.attentionPacked(q, k, v, offsets(lens), heads, kv, hd)
    be.status_poll()
    for i, n in enumerate(lens):
        rows = slice(int(starts[i]), int(starts[i]) + n)
        alone = be.attentionPacked(q[rows], k[rows], v[rows], offsets([n]), heads, kv, hd)
        assert torch.equal(torch.isnan(out[rows]), torch.isnan(alone))
        assert torch.equal(torch.nan_to_num(out[rows]), torch.nan_to_num(alone)), (i, n)
    assert torch.isnan(out).any() and torch.isinf(out).any()


def test_tens_of_thousands_of_sequences_without_tokens(be):
    """More of them than a block passes over on its way to work."""
    heads, kv, hd = 8, 8, 64
    lens = [150] + [0] * 30000 + [70] + [0] * 30000 + [129, 300]
    q, k, v = make(sum(lens), heads, kv, hd, "f16", 22)
    out = be.attentionPacked(q, k, v, offsets(lens), heads, kv, hd)
    be.status_poll()
    check(out, q, k, v, [n for n in lens if n], heads, kv, hd, "f16", rows_at_most=30)


@pytest.mark.parametrize("lens,heads,kv,hd,dt", [([900, 129, 1, 0, 255, 700, 64], 16, 8, 128, "f16"), ([333, 700, 18, 19, 512], 14, 2, 64, "f16"),
                                                ([1500, 2, 1030], 12, 4, 128, "bf16"), ([260] * 9, 33, 3, 64, "bf16"), ([130] * 12, 8, 8, 64, "f16")])
def test_large_batches_give_the_bits_of_small_ones(be, lens, heads, kv, hd, dt):
    """Two tiles of queries a block, or one where the batch is small: the same rows either way, and the formula's."""
    times = 6
    q, k, v = make(sum(lens) * times, heads, kv, hd, dt, sum(lens))
    out = be.attentionPacked(q, k, v, offsets(lens * times), heads, kv, hd)
    be.status_poll()
    at = 0
    for n in lens * times:
        rows = slice(at, at + n)
        assert torch.equal(out[rows], be.attentionPacked(q[rows], k[rows], v[rows], offsets([n]), heads, kv, hd)), n
        at += n
    check(out, q, k, v, lens, heads, kv, hd, dt, rows_at_most=20)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_up_to_the_documented_limit(be, hd, dt):
    """Single products up to 2^22, exact in f32 and 2^14 apart or equal: the row's largest has all the weight, or its equals share it.  What rounding the
    reference point loses is the same factor for weights and sum."""
    lens, heads, kv = [1, 5, 300], 2, 1
    total = sum(lens)
    g = torch.Generator().manual_seed(hd)
    q, k = torch.zeros((total, heads, hd)), torch.zeros((total, hd))
    q[:, 0, 0], q[:, 1, 3] = 2048.0, -2040.0
    k[:, 0], k[:, 3] = (1024.0 * (1.0 + torch.randint(0, 128, (total,), generator=g) / 128.0) * s for s in (1.0, -1.0))
    v = torch.randn((total, hd), generator=g)
    q, k, v = (t.reshape(total, -1).to(DT[dt]).cuda() for t in (q, k, v))
    out = be.attentionPacked(q, k, v, offsets(lens), heads, kv, hd, scale=1.0)
    be.status_poll()
    got, q, k, v = (t.double().cpu().numpy() for t in (out, q, k, v))
    at = 0
    for n in lens:
        for h in range(heads):
            mine = slice(h * hd, (h + 1) * hd)
            o, a, _ = attend(q[at:at + n, mine], k[at:at + n], v[at:at + n], np.arange(n), 1.0)
            tol = tolerance(o, a, np.zeros(n), hd, HALF_STEP[dt], HALF_STEP[dt])
            assert (np.abs(got[at:at + n, mine] - o) <= tol).all()
        at += n
