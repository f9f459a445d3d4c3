"""The 8-bit key / value cache on the GPU: page operations and quantising against a model in Python, bit for bit; attention against the
formula in 64 bits (bounds: attn_reference.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attn_reference import HALF_STEP, Model, attend, tolerance  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def be():
    from tensorpencil_b200.backend import Backend
    b = Backend(0)
    yield b
    b.close()


def i32(values):
    return torch.tensor(list(values), dtype=torch.int32).cuda()


def offsets(lens):
    return i32(np.cumsum([0] + list(lens)))


def both(be, n_pages=40, max_seqs=8, max_pages=12, page=16, kv=2, hd=64, fmt="s8", layers=1):
    from tensorpencil_b200.kv_cache import KvCache
    return (KvCache(be, layers, n_pages, kv, hd, max_seqs, max_pages, page, fmt), Model(n_pages, max_seqs, max_pages, page, kv, hd, fmt, layers))


def same_tables(c, m):
    assert c.table.tolist() == m.table
    assert c.lens.tolist() == m.lens and c.tail.tolist() == m.tail and c.refs.tolist() == m.refs
    r = c.result.tolist()
    assert r == m.result, (r, m.result)


def same_values(c, m, layer=0, dtype=torch.float32):
    seqs = [s for s in range(m.max_seqs) if m.lens[s]]
    if not seqs:
        return
    lens = [m.lens[s] for s in seqs]
    got = c.read(layer, i32(seqs), offsets(lens), sum(lens), dtype=dtype)
    for name, g in zip("kv", got):
        want = np.concatenate([m.read(layer, name, s) for s in seqs]).reshape(sum(lens), -1)
        g = g.double().cpu().numpy()
        if dtype != torch.float32:
            want = torch.from_numpy(want).to(dtype).double().numpy()
        assert np.array_equal(g, want, equal_nan=True), name


def values(rng, n, kv, hd, dt, big=1.0):
    x = rng.standard_normal((n, kv, hd)) * big * np.exp2(rng.integers(-3, 4, (n, kv, 1)))
    return torch.from_numpy(x).to(DT[dt]).cuda()


def append(c, m, seqs, xs, layer=0):
    """xs: one (k, v) a sequence, [n][kv][hd]."""
    k, v = (torch.cat([x[i] for x in xs]) for i in (0, 1))
    c.append(layer, k, v, i32(seqs), offsets([x[0].shape[0] for x in xs]))
    for s, x in zip(seqs, xs):
        for name, t in zip("kv", x):
            if t.shape[0]:
                m.append(layer, name, s, t.double().cpu().numpy())


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("page,hd,kv", [(16, 64, 2), (16, 128, 3), (32, 128, 1), (64, 64, 5), (64, 128, 2), (32, 64, 1)])
def test_append_and_read_bit_for_bit(be, page, hd, kv, dt, fmt):
    c, m = both(be, n_pages=60, page=page, hd=hd, kv=kv, fmt=fmt)
    rng = np.random.default_rng(page + hd + kv)
    for step, lens in enumerate([{0: 1, 3: 40, 5: 2 * page}, {0: 5, 3: 1, 5: 1}, {3: 1}, {0: page - 6, 1: 3, 3: page + 1, 5: 1}, {0: 1, 1: 1, 3: 1, 5: 1}]):
        seqs = list(lens)[::-1]
        n = [lens[s] for s in seqs]
        c.extend(i32(seqs), i32(n))
        m.extend(seqs, n)
        same_tables(c, m)
        append(c, m, seqs, [tuple(values(rng, k, kv, hd, dt, 2.0 ** step) for _ in range(2)) for k in n])     # scales grow with the steps
        same_values(c, m)
    assert c.check() == c.result.tolist()[1]
    assert np.array_equal(c.k_scale[0].cpu().numpy()[np.array(m.refs) > 0], m.scale["k"][0][np.array(m.refs) > 0].astype(np.float32))
    same_values(c, m, dtype=torch.bfloat16)
    same_values(c, m, dtype=torch.float16)


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
def test_blocks_at_the_edges_of_the_quantiser(be, fmt):
    """Zeros, the smallest and largest values, an amax at the limit times a power of two and next to it, ties, NaN and infinities."""
    c, m = both(be, fmt=fmt, kv=1, hd=64, n_pages=80)
    limit = {"s8": 127.0, "e4m3": 448.0}[fmt]
    near = lambda f, d: float(np.nextafter(np.float32(f), np.float32(d)))      # noqa: E731
    tops = [0.0, 1e-45, 1e-38, 1e-30, 3.0e38, 3.4028234e38, limit, near(limit, 0), near(limit, 1e9), limit * 2.0 ** -9, near(limit * 2.0 ** -9, 1e9),
            limit * 2.0 ** 40, 1.0, 2.0, near(1.0, 0)]
    seqs = [0, 1]
    per = [16 * 8, 16 * (len(tops) - 8)]
    c.extend(i32(seqs), i32(per))
    m.extend(seqs, per)
    rng = np.random.default_rng(0)
    xs = []
    for part in (tops[:8], tops[8:]):
        x = np.concatenate([np.clip(rng.integers(-255, 256, (16, 1, 64)) / 254.0, -1, 1) * t for t in part]).astype(np.float32)
        for i, t in enumerate(part):
            x[16 * i, 0, 0] = t
        xs.append((torch.from_numpy(x).cuda(), torch.from_numpy(-x[::-1].copy()).cuda()))
    append(c, m, seqs, xs)
    same_values(c, m)
    for s, bad in ((2, float("nan")), (3, float("inf")), (4, -float("inf"))):
        c.extend(i32([s]), i32([20]))
        m.extend([s], [20])
        k, v = values(rng, 20, 1, 64, "f32"), values(rng, 20, 1, 64, "f32")
        k[3, 0, 5] = bad
        append(c, m, [s], [(k, v)])
        c.extend(i32([s]), i32([1]))
        m.extend([s], [1])
        append(c, m, [s], [(values(rng, 1, 1, 64, "f32"), values(rng, 1, 1, 64, "f32"))])
    same_values(c, m)
    c.check()


def test_read_of_parts_and_behind_the_end(be):
    c, m = both(be, kv=2, hd=64)
    rng = np.random.default_rng(3)
    c.extend(i32([0, 1]), i32([37, 5]))
    m.extend([0, 1], [37, 5])
    append(c, m, [0, 1], [tuple(values(rng, n, 2, 64, "f32") for _ in range(2)) for n in (37, 5)])
    out = tuple(torch.full((30, 2 * 64 + 4), 9.0).cuda() for _ in range(2))
    c.read(0, i32([1, 0]), i32([2, 12, 25]), 30, start=i32([3, 30]), out=tuple(t[:, :128] for t in out))
    for name, t in zip("kv", out):
        t = t.cpu().numpy()
        want = np.full((30, 128), 9.0)
        want[2:12], want[12:25] = 0.0, 0.0
        want[2:4], want[12:19] = m.read(0, name, 1)[3:5].reshape(2, -1), m.read(0, name, 0)[30:].reshape(7, -1)
        assert np.array_equal(t[:, :128], want) and (t[:, 128:] == 9.0).all()


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
@pytest.mark.parametrize("seed", range(6))
def test_random_page_operations_follow_the_model(be, seed, fmt):
    """Extensions, appends, forks of both kinds, cuts, frees and compactions in any order, refused ones among them."""
    rng = np.random.default_rng(seed)
    page, kv, hd, layers = [16, 32, 64][seed % 3], 2, [64, 128][seed % 2], 2
    c, m = both(be, n_pages=26 if seed % 2 else 300, max_seqs=10, max_pages=9, page=page, kv=kv, hd=hd, fmt=fmt, layers=layers)
    for _ in range(60):
        op = rng.choice(["extend", "extend", "extend", "truncate", "free", "fork", "copy", "compact"])
        ids = [int(i) for i in rng.permutation(10)[:rng.integers(1, 5)]]
        if rng.random() < 0.05:
            ids.append(ids[0] if rng.random() < 0.5 else 10)
        if op == "extend":
            n = [int(rng.choice([0, 1, 3, page, 2 * page + 1])) for _ in ids]
            c.extend(i32(ids), i32(n))
            m.extend(ids, n)
            same_tables(c, m)
            if m.result[0] == 0:
                xs = [[tuple(values(rng, k, kv, hd, "f32") for _ in range(2)) for k in n] for _ in range(layers)]
                for layer in range(layers):
                    append(c, m, ids, xs[layer], layer)
        elif op == "truncate":
            n = [int(rng.integers(0, m.lens[i] + 1)) if 0 <= i < 10 else 0 for i in ids]
            if rng.random() < 0.05:
                n[0] += 1000
            c.truncate(i32(ids), i32(n))
            m.truncate(ids, n)
        elif op == "free":
            c.truncate(i32(ids))
            m.truncate(ids)
        elif op in ("fork", "copy"):
            free = [i for i in range(10) if m.lens[i] == 0]
            used = [i for i in range(10) if m.lens[i]]
            if not free or not used:
                continue
            dst = [int(d) for d in rng.permutation(free)[:rng.integers(1, 4)]]
            src = [int(rng.choice(used)) for _ in dst]
            if rng.random() < 0.1:
                dst[-1] = int(rng.choice(used))
            c.fork(i32(src), i32(dst), share=op == "fork")
            m.fork(src, dst, op == "fork")
        else:
            c.compact()
            m.compact()
        same_tables(c, m)
        for layer in range(layers):
            same_values(c, m, layer)
        assert all(0 <= p < m.n_pages for s in range(10) for p in m.table[s][:m.pages(m.lens[s])])
    be.status_poll()


def test_a_large_pool(be):
    """More pages than one step of the scans covers, a number that no vector load divides, and long lists."""
    n_pages, n = 70001, 600
    c, m = both(be, n_pages=n_pages, max_seqs=1300, max_pages=140, page=16, kv=1, hd=64)
    rng = np.random.default_rng(1)
    ids, lens = [int(i) for i in rng.permutation(600)], [int(x) for x in rng.integers(0, 2000, n)]
    for call in ("extend", "free", "fork", "compact", "cut"):
        if call == "extend":
            c.extend(i32(ids), i32(lens)), m.extend(ids, lens)
        elif call == "free":
            c.truncate(i32(ids[::3])), m.truncate(ids[::3])
        elif call == "fork":
            src, dst = ids[1::3], [600 + i for i in range(len(ids[1::3]))]
            c.fork(i32(src), i32(dst)), m.fork(src, dst, True)
        elif call == "compact":
            c.compact(), m.compact()
        else:
            live = [s for s in range(1300) if m.lens[s] > 50]
            to = [m.lens[s] - 33 for s in live]
            c.truncate(i32(live), i32(to)), m.truncate(live, to)
        same_tables(c, m)
    be.status_poll()


def test_long_lists_over_many_sequences(be):
    """Lists longer than a block has threads, more sequences than marks fit shared memory, and ids listed twice in them."""
    n, max_seqs = 2500, 40000
    c, m = both(be, n_pages=9000, max_seqs=max_seqs, max_pages=6, page=16, kv=1, hd=64)
    rng = np.random.default_rng(7)
    ids = [int(i) for i in rng.permutation(max_seqs)[:2 * n]]
    src, dst = ids[:n], ids[n:]
    lens = [int(x) for x in rng.integers(0, 50, n)]
    c.extend(i32(src), i32(lens)), m.extend(src, lens)
    same_tables(c, m)
    c.fork(i32(src), i32(dst)), m.fork(src, dst, True)
    same_tables(c, m)
    for bad in (src[:2000] + src[700:701], src[:2000] + [max_seqs]):
        c.truncate(i32(bad)), m.truncate(bad)
        same_tables(c, m)
    c.fork(i32(src[:1500] + src[:1]), i32(dst[:1501])), m.fork(src[:1500] + src[:1], dst[:1501], True)      # in use
    same_tables(c, m)
    to = [x // 2 for x in lens]
    c.truncate(i32(dst), i32(to)), m.truncate(dst, to)
    same_tables(c, m)
    c.truncate(i32(src)), m.truncate(src)
    same_tables(c, m)
    c.compact(), m.compact()
    same_tables(c, m)
    be.status_poll()


def test_refused_operations_change_nothing_and_say_why(be):
    from tensorpencil_b200 import _lib
    c, m = both(be, n_pages=5, max_seqs=4, max_pages=4, kv=1)
    for op, arg, status in ((c.extend, (i32([0]), i32([70])), _lib.TPB_ERR_INVALID_ARG),           # longer than a table row
                            (c.extend, (i32([0, 1]), i32([50, 40])), _lib.TPB_ERR_OOM),
                            (c.extend, (i32([0, 0]), i32([1, 1])), _lib.TPB_ERR_INVALID_ARG),
                            (c.extend, (i32([-1]), i32([1])), _lib.TPB_ERR_INVALID_ARG),
                            (c.extend, (i32([1]), i32([-1])), _lib.TPB_ERR_INVALID_ARG),
                            (c.truncate, (i32([0]), i32([1])), _lib.TPB_ERR_INVALID_ARG),
                            (c.truncate, (i32([4]),), _lib.TPB_ERR_INVALID_ARG),
                            (c.fork, (i32([0]), i32([0])), _lib.TPB_ERR_INVALID_ARG)):
        op(*arg)
        with pytest.raises(_lib.TpbError) as e:
            c.check()
        assert e.value.status == status
        m.result = c.result.tolist()
        same_tables(c, m)


def test_tokens_that_no_extension_made_room_for_are_not_written(be):
    from tensorpencil_b200 import _lib
    c, m = both(be, n_pages=2, kv=1)
    rng = np.random.default_rng(0)
    c.extend(i32([0]), i32([20]))
    m.extend([0], [20])
    append(c, m, [0], [tuple(values(rng, 20, 1, 64, "f32") for _ in range(2))])
    c.extend(i32([0]), i32([20]))                          # not enough pages: refused, and so is what follows
    x = values(rng, 20, 1, 64, "f32")
    c.append(0, x, x, i32([0]), i32([0, 20]))
    with pytest.raises(_lib.TpbError) as e:
        be.status_poll()
    assert e.value.status == _lib.TPB_ERR_STATE
    same_values(c, m)
    for seqs in ([7], [8], [-1]):                          # an empty sequence, and ids out of range
        c.append(0, x, x, i32(seqs), i32([0, 20]))
        with pytest.raises(_lib.TpbError) as e:
            be.status_poll()
        assert e.value.status == _lib.TPB_ERR_STATE
    same_values(c, m)


# -- attention -----------------------------------------------------------------------------


def filled(be, lens, fmt, page, kv, hd, seed, spare=6):
    """A cache whose sequences' pages lie out of order, with random contents."""
    n_pages = sum(-(-n // page) for n in lens) + spare
    c, m = both(be, n_pages=n_pages, max_seqs=len(lens) + 1, max_pages=max(1, max(-(-n // page) for n in lens)) + 1, page=page, kv=kv, hd=hd, fmt=fmt)
    rng = np.random.default_rng(seed)
    order = [int(p) for p in rng.permutation(n_pages)]
    lim = 127 if fmt == "s8" else 448
    for s, n in enumerate(lens):
        m.lens[s] = n
        for p in range(-(-n // page)):
            m.table[s][p] = order.pop()
            m.refs[m.table[s][p]] = 1
    for name, t, sc in (("k", c.k, c.k_scale), ("v", c.v, c.v_scale)):
        x = np.clip(rng.standard_normal(m.q[name].shape) * lim / 4, -lim, lim)
        q = torch.from_numpy(x)
        q = torch.round(q).to(torch.int8) if fmt == "s8" else q.to(torch.float8_e4m3fn)
        m.q[name] = q.double().numpy()
        m.scale[name] = np.exp2(rng.integers(-1, 2, m.scale[name].shape)) * 4.0 / lim * (1.0 + 0.25 * rng.random(m.scale[name].shape))
        m.scale[name] = m.scale[name].astype(np.float32).astype(np.float64)
        t.copy_(q.cuda())
        sc.copy_(torch.from_numpy(m.scale[name]).float())
    c.table.copy_(torch.tensor(m.table, dtype=torch.int32))
    c.lens.copy_(i32(m.lens))
    c.refs.copy_(i32(m.refs))
    return c, m


# What the weights lose before the second product.  f32 and f16 rows: two f16 terms, hi = rn(w) and lo = rn(w - hi), |w - hi - lo| <= 2^-11 |w - hi| <=
# 2^-22 w, or below the smallest f16 step relative to the reference (added apart).  bf16 rows: one f16 term, |w - rn(w)| <= 2^-11 w, an eighth of
# the half step of the bf16 result.
WEIGHTS = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": HALF_STEP["f16"]}


def check_attention(c, m, out, q, seqs, n_new, heads, dt, scale=None):
    kv, hd = c.kv_heads, c.head_dim
    scale = hd ** -0.5 if scale is None else scale
    got, q = out.double().cpu().numpy(), q.double().cpu().numpy()
    at = 0
    for s, n in zip(seqs, n_new):
        k, v = m.read(0, "k", s), m.read(0, "v", s)
        last = m.lens[s] - n + np.arange(n)
        for h in range(heads):
            mine, hk = slice(h * hd, (h + 1) * hd), h // (heads // kv)
            o, a, e = attend(q[at:at + n, mine], k[:, hk], v[:, hk], last, scale)
            # q in two f16 terms (bf16: exact in one): what is left of it is below 2^-21 of a row's largest
            tol = tolerance(o, a, e * (1 + 2.0 ** 4), hd, HALF_STEP[dt], WEIGHTS[dt]) + len(k) * 2.0 ** -33 * (np.abs(v).max() if len(k) else 0)
            err = np.abs(got[at:at + n, mine] - o)
            assert (err <= tol).all(), (s, n, h, float((err / tol).max()), float(err.max()))
        at += n


ATT = [([1], 1, 2, 1, 64, 16), ([16, 17, 15], 1, 4, 4, 128, 16), ([200, 1, 64, 63, 65], 1, 8, 2, 128, 32), ([777], 1, 7, 1, 64, 64),
       ([300, 5, 90], 4, 6, 2, 128, 16), ([130, 40], 5, 16, 1, 64, 32), ([2500], 2, 12, 4, 128, 16), ([3000, 2], 8, 8, 8, 64, 64),
       ([40, 500], 9, 5, 1, 128, 64), ([1000], 33, 4, 2, 64, 16), ([260], 1, 40, 1, 128, 32), ([9000], 1, 3, 1, 128, 32)]


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens,new,heads,kv,hd,page", ATT)
def test_attention_matches_the_formula(be, lens, new, heads, kv, hd, page, dt, fmt):
    c, m = filled(be, lens, fmt, page, kv, hd, sum(lens) + heads)
    seqs = list(range(len(lens)))[::-1]
    g = torch.Generator().manual_seed(1)
    q = torch.randn((new * len(seqs), heads * hd), generator=g).to(DT[dt]).cuda()
    out = c.attention(0, q, i32(seqs), offsets([new] * len(seqs)), heads)
    be.status_poll()
    check_attention(c, m, out, q, seqs, [new] * len(seqs), heads, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_different_numbers_of_queries_and_rows_that_see_nothing(be, dt):
    """0 to 20 queries a sequence, some of sequences that are shorter than that (their first rows see nothing: zeros), an empty one."""
    lens, new, heads, kv, hd = [90, 3, 0, 400, 18], [7, 5, 2, 0, 20], 6, 2, 64
    c, m = filled(be, lens, "s8", 16, kv, hd, 5)
    rows = sum(new)
    g = torch.Generator().manual_seed(2)
    wide_q = torch.randn((rows + 3, heads * hd + 8), generator=g).to(DT[dt]).cuda()
    wide = torch.full((rows + 3, heads * hd + 8), 5.0, dtype=DT[dt]).cuda()
    q, out = wide_q[:, :heads * hd], wide[:, :heads * hd]
    c.attention(0, q, i32(range(5)), offsets(new), heads, out=out)
    be.status_poll()
    check_attention(c, m, out[:rows], q[:rows], range(5), new, heads, dt)
    assert (out[7:9] == 0).all() and (out[12:14] == 0).all() and (out[14:16] == 0).all()
    assert (wide[rows:] == 5.0).all() and (wide[:, heads * hd:] == 5.0).all()


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
def test_stale_bytes_scales_and_tables_behind_the_end_are_not_part_of_it(be, fmt):
    """Whatever lies behind a sequence's last token -- NaN among it -- in its last page, in free pages and in the table."""
    lens, heads, kv, hd, page = [50, 129, 33], 4, 2, 64, 32
    c, m = filled(be, lens, fmt, page, kv, hd, 8)
    q = torch.randn((3, heads * hd), generator=torch.Generator().manual_seed(0)).cuda()
    clean = c.attention(0, q, i32([0, 1, 2]), offsets([1] * 3), heads)
    free = [p for p in range(m.n_pages) if m.refs[p] == 0]
    for t, sc in ((c.k, c.k_scale), (c.v, c.v_scale)):
        raw = t.view(torch.uint8)
        raw[:, free] = 0x7f                                # NaN in e4m3
        sc[:, free] = float("nan")
        for s, n in enumerate(lens):
            raw[0, m.table[s][n // page], :, n % page:] = 0x7f
    c.table[0, 2:] = 10 ** 9
    c.table[1, 5:] = -7
    out = c.attention(0, q, i32([0, 1, 2]), offsets([1] * 3), heads)
    be.status_poll()
    assert torch.equal(out, clean)


def test_a_block_with_a_nan_reaches_the_heads_that_see_it(be):
    lens, heads, kv, hd = [100, 40], 4, 2, 64
    c, m = filled(be, lens, "s8", 16, kv, hd, 8)
    q = torch.randn((2, heads * hd), generator=torch.Generator().manual_seed(0)).cuda()
    clean = c.attention(0, q, i32([0, 1]), offsets([1, 1]), heads)
    c.k_scale[0, m.table[0][3], 0] = float("nan")
    c.v_scale[0, m.table[0][1], 1] = float("nan")
    out = c.attention(0, q, i32([0, 1]), offsets([1, 1]), heads)
    assert torch.isnan(out[0]).all() and torch.equal(out[1], clean[1])


@pytest.mark.parametrize("fmt,dt", [("s8", "f32"), ("e4m3", "bf16"), ("s8", "f16")])
def test_scores_and_values_of_a_wide_range(be, fmt, dt):
    """Queries from tiny to large, maxima that come late, value scales that differ by 2^40 from page to page."""
    lens, heads, kv, hd, page = [700, 90], 8, 2, 128, 16
    c, m = filled(be, lens, fmt, page, kv, hd, 4)
    if dt != "f16":
        rng = np.random.default_rng(0)
        f = np.exp2(rng.integers(-20, 21, m.scale["v"].shape))
        m.scale["v"] = (m.scale["v"] * f).astype(np.float32).astype(np.float64)
        c.v_scale.copy_(torch.from_numpy(m.scale["v"]).float())
    q = torch.randn((2, heads * hd), generator=torch.Generator().manual_seed(3)) * torch.exp2(torch.arange(heads * hd) // hd * 1.0 - 4)
    q = q.to(DT[dt]).cuda()
    out = c.attention(0, q, i32([0, 1]), offsets([1, 1]), heads)
    # with values of very different sizes a weight's share of the largest product counts: all terms are below max |v| p
    kvs = c.kv_heads
    got = out.double().cpu().numpy()
    for r, s in enumerate([0, 1]):
        k, v = m.read(0, "k", s), m.read(0, "v", s)
        for h in range(heads):
            hk = h // (heads // kvs)
            qq = q[r:r + 1, h * hd:(h + 1) * hd].double().cpu().numpy()
            o, a, e = attend(qq, k[:, hk], v[:, hk], [lens[s] - 1], hd ** -0.5)
            p = np.exp((k[:, hk] @ qq[0]) * hd ** -0.5 - ((k[:, hk] @ qq[0]) * hd ** -0.5).max())
            biggest = (p / p.sum() * np.abs(v[:, hk]).max(1)).max()
            tol = tolerance(o, a, e * (1 + 2.0 ** 4), hd, HALF_STEP[dt], WEIGHTS[dt]) + len(k) * 2.0 ** -30 * biggest
            err = np.abs(got[r, h * hd:(h + 1) * hd] - o[0])
            assert (err <= tol).all(), (s, h, float((err / tol).max()))


def test_bad_entries_are_reported_and_skipped(be):
    from tensorpencil_b200 import _lib
    c, m = filled(be, [100, 40], "s8", 16, 1, 64, 3)
    q = torch.randn((2, 2 * 64)).cuda()
    c.attention(0, q, i32([0, 1]), offsets([1, 1]), 2)
    be.status_poll()
    for what, to in (("table", 10 ** 6), ("table", -1), ("lens", 10 ** 6), ("lens", -3), ("id", 3), ("id", -1)):
        seqs = i32([0, to if what == "id" else 1])
        old = (c.table.clone(), c.lens.clone())
        if what == "table":
            c.table[1, 1] = to
        if what == "lens":
            c.lens[1] = to
        out = c.attention(0, q, seqs, offsets([1, 1]), 2)
        with pytest.raises(_lib.TpbError) as e:
            be.status_poll()
        assert e.value.status == _lib.TPB_ERR_STATE
        check_attention(c, m, out[:1], q[:1], [0], [1], 2, "f32")
        c.table.copy_(old[0]), c.lens.copy_(old[1])


def test_max_len_is_a_hint(be):
    c, m = filled(be, [5000, 40, 1200], "e4m3", 16, 2, 128, 3)
    q = torch.randn((3, 8 * 128)).cuda()
    for hint in (0, 40, 200, 5000, 10 ** 9):
        check_attention(c, m, c.attention(0, q, i32([0, 1, 2]), offsets([1, 1, 1]), 8, max_len=hint), q, [0, 1, 2], [1] * 3, 8, "f32")


def test_many_sequences(be):
    rng = np.random.default_rng(2)
    lens = [int(n) for n in rng.integers(0, 60, 700)]
    lens[100], lens[650] = 900, 2000
    c, m = filled(be, lens, "s8", 16, 1, 64, 3)
    seqs = [int(s) for s in rng.permutation(700)]
    q = torch.randn((700, 2 * 64)).cuda()
    out = c.attention(0, q, i32(seqs), offsets([1] * 700), 2)
    be.status_poll()
    some = [i for i in range(700) if i % 13 == 0 or seqs[i] in (100, 650)]
    check_attention(c, m, out[some], q[some], [seqs[i] for i in some], [1] * len(some), 2, "f32")


def test_two_streams_and_the_same_bits_again(be):
    c, m = filled(be, [3000, 170, 1000], "s8", 32, 2, 128, 3)
    q = torch.randn((2, 3, 8 * 128)).cuda()
    want = [c.attention(0, q[i], i32([0, 1, 2]), offsets([1] * 3), 8) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ids, cu = i32([0, 1, 2]), offsets([1] * 3)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attention(0, q[i], ids, cu, 8))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_a_decode_loop_prompt_to_compaction(be):
    """Prompts through packed attention and into the cache, decoding with drafts that are cut back, beams, a freed sequence and a compaction, two
    layers: every step's attention against the formula on the cache's values."""
    kv, heads, hd, page, layers = 2, 6, 64, 16, 2
    c, m = both(be, n_pages=60, max_seqs=6, max_pages=20, page=page, kv=kv, hd=hd, fmt="e4m3", layers=layers)
    rng = np.random.default_rng(9)

    def step(seqs, n, dt="bf16"):
        c.extend(i32(seqs), i32(n))
        m.extend(seqs, n)
        same_tables(c, m)
        cu = offsets(n)
        for layer in range(layers):
            xs = [tuple(values(rng, k, kv, hd, dt) for _ in range(2)) for k in n]
            append(c, m, seqs, xs, layer)
            q = values(rng, sum(n), heads, hd, dt).reshape(sum(n), -1)
            out = c.attention(layer, q, i32(seqs), cu, heads)
            if layer == 0:
                check_attention(c, m, out, q, seqs, n, heads, dt)
        return xs

    prompts = [70, 33]
    step([0, 1], prompts)
    k, v = (torch.cat([values(rng, n, kv, hd, "bf16").reshape(n, -1) for n in prompts]) for _ in range(2))
    be.attentionPacked(values(rng, 103, heads, hd, "bf16").reshape(103, -1), k, v, offsets(prompts), heads, kv, hd)
    for _ in range(3):
        step([1, 0], [1, 1])
    step([0, 1], [5, 5], "f32")                             # five drafts each, some rejected
    to = [m.lens[0] - 3, m.lens[1] - 4]
    c.truncate(i32([0, 1]), i32(to)), m.truncate([0, 1], to)
    c.fork(i32([0, 0, 1]), i32([2, 3, 4])), m.fork([0, 0, 1], [2, 3, 4], True)
    same_tables(c, m)
    step([4, 2, 0, 3, 1], [1] * 5)
    c.truncate(i32([0, 1])), m.truncate([0, 1])
    c.compact(), m.compact()
    same_tables(c, m)
    step([2, 3, 4], [1, 2, 1], "f16")
    for layer in range(layers):
        same_values(c, m, layer)
    assert c.check() == m.result[1]


def test_a_captured_step_replays_while_the_lengths_grow(be):
    kv, heads, hd = 2, 8, 128
    c, m = both(be, n_pages=40, max_seqs=3, max_pages=12, page=16, kv=kv, hd=hd)
    rng = np.random.default_rng(4)
    seqs, one, cu = i32([2, 0]), i32([1, 1]), i32([0, 1, 2])
    c.extend(seqs, i32([30, 15]))
    m.extend([2, 0], [30, 15])
    append(c, m, [2, 0], [tuple(values(rng, n, kv, hd, "f32") for _ in range(2)) for n in (30, 15)])
    k, v, q = (torch.zeros((2, h * hd)).cuda() for h in (kv, kv, heads))
    out = torch.zeros((2, heads * hd)).cuda()

    def step():
        c.extend(seqs, one)
        c.append(0, k, v, seqs, cu)
        c.attention(0, q, seqs, cu, heads, out=out)

    graphs = []
    for _ in range(2):                                      # two graphs of the same step, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i in range(8):
        for t, h in ((k, kv), (v, kv), (q, heads)):
            t.copy_(values(rng, 2, h, hd, "f32").reshape(2, -1))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        m.extend([2, 0], [1, 1])
        for j, s in enumerate([2, 0]):
            m.append(0, "k", s, k[j:j + 1].view(1, kv, hd).double().cpu().numpy())
            m.append(0, "v", s, v[j:j + 1].view(1, kv, hd).double().cpu().numpy())
        same_tables(c, m)
        same_values(c, m)
        check_attention(c, m, out, q, [2, 0], [1, 1], heads, "f32")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("page,hd,total", [(16, 128, 4100), (16, 64, 4100), (32, 128, 3100), (64, 128, 8300), (64, 64, 4100)])
def test_long_prompts_are_cached_as_short_ones_are(be, page, hd, total, dt):
    """More pages than the GPU takes at once: the bytes and scales of a batch are those of its sequences one at a time, a page or two a call."""
    from tensorpencil_b200.kv_cache import KvCache
    kv, lens = 8, [total // 2, 5, total // 3, total - total // 2 - total // 3 - 5]
    rng = np.random.default_rng(total + hd)
    k, v = (values(rng, total, kv, hd, dt) for _ in "kv")
    seqs, cu = i32(range(4)), offsets(lens)
    made = []
    for whole in (True, False):
        c = KvCache(be, 1, total // page + 8, kv, hd, 4, total // page + 4, page, "s8")
        c.extend(seqs, i32([3, 1, 0, 7]))                  # the prompts begin inside a page
        c.append(0, k[:11], v[:11], seqs, offsets([3, 1, 0, 7]))
        if whole:
            c.extend(seqs, i32(lens))
            c.append(0, k, v, seqs, cu)
        else:
            at = 0
            for s, n in enumerate(lens):
                done, held = 0, [3, 1, 0, 7][s]
                while done < n:                            # up to the end of the page, so that every block is rounded the same number of times
                    part = min(n - done, 2 * page - (held + done) % page)
                    c.extend(i32([s]), i32([part]))
                    c.append(0, k[at + done:at + done + part], v[at + done:at + done + part], i32([s]), i32([0, part]))
                    done += part
                at += n
        c.check()
        made.append(c.read(0, seqs, offsets([a + b for a, b in zip(lens, [3, 1, 0, 7])]), total + 11, dtype=torch.float32))
    assert torch.equal(made[0][0], made[1][0]) and torch.equal(made[0][1], made[1][1])
    # the last to come to a block were rounded once: off by half a step, and a step is at most 2 amax / 127 (the first page's tokens before them are k's too)
    got, want = made[0][0].view(-1, kv, hd)[3:3 + lens[0]], k[:lens[0]].float()
    assert ((got - want).abs() <= want.abs().max() / 127 * 1.000001).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("new,heads,kv", [(4, 4, 1), (6, 8, 2), (8, 4, 1)])
def test_many_rows_over_a_long_cache(be, new, heads, kv, dt):
    """16 to 32 rows a kv head, joined from parts by two blocks."""
    test_attention_matches_the_formula(be, [5000, 700], new, heads, kv, 128, 64, dt, "s8")


@pytest.mark.parametrize("fmt,dt", [("s8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("page,hd", [(16, 64), (16, 128), (32, 64), (64, 128)])
@pytest.mark.parametrize("lead", [(0, 1), (1, 0), (2, 0), (7, 5)])
def test_rows_of_nobody_around_an_append(be, lead, page, hd, fmt, dt):
    """The batch's rows begin behind `lead` pages and tokens of somebody else's rows (NaN), and more of those follow: bytes, scales and tables of the
    whole pool are the model's, whether the batch's first sequence is the table's first, new, continued, or next to a row that is full."""
    kv, max_pages = 2, 4
    rng = np.random.default_rng(page + hd + 8 * lead[0] + lead[1])
    for order in ([0, 2], [2, 0], [2], [0], [3, 0, 2]):
        c, m = both(be, n_pages=24, max_seqs=4, max_pages=max_pages, page=page, kv=kv, hd=hd, fmt=fmt)
        c.extend(i32([1, 2]), i32([max_pages * page, page + 3])), m.extend([1, 2], [max_pages * page, page + 3])
        append(c, m, [1, 2], [tuple(values(rng, n, kv, hd, dt) for _ in range(2)) for n in (max_pages * page, page + 3)])
        new = {0: 1, 2: 2 * page, 3: page}
        n = [new[s] for s in order]
        c.extend(i32(order), i32(n)), m.extend(order, n)
        xs = [tuple(values(rng, k, kv, hd, dt, 4.0) for _ in range(2)) for k in n]
        front, behind = lead[0] * page + lead[1], page + 1
        k, v = (torch.cat([torch.full((front, kv, hd), float("nan"), dtype=DT[dt]).cuda()] + [x[i] for x in xs]
                          + [torch.full((behind, kv, hd), float("nan"), dtype=DT[dt]).cuda()]) for i in (0, 1))
        c.append(0, k, v, i32(order), i32(front + np.cumsum([0] + n)))
        for s, x in zip(order, xs):
            for name, t in zip("kv", x):
                m.append(0, name, s, t.double().cpu().numpy())
        same_tables(c, m)
        assert c.check() == m.result[1]
        for name, q, scale in (("k", c.k, c.k_scale), ("v", c.v, c.v_scale)):
            assert np.array_equal(q.float().cpu().numpy(), m.q[name]) and np.array_equal(scale.cpu().numpy(), m.scale[name])


def test_launches_are_the_kernels_of_a_captured_call(be):
    from graph_nodes import kernels
    c, m = filled(be, [300, 20], "s8", 16, 2, 64, 1)
    ids, cu, src, free, one = i32([0, 1]), i32([0, 1, 2]), i32([0]), i32([2]), i32([1, 1])
    x, q = torch.zeros((2, 128)).cuda(), torch.zeros((2, 256)).cuda()
    b = q.bfloat16()
    # a call without rows beside one that launches: an empty graph has no nodes to ask for
    for call in (lambda: c.extend(ids, one), lambda: c.append(0, x, x, ids, cu), lambda: (c.append(0, x[:0], x[:0], ids, cu), c.compact()),
                 lambda: c.read(0, ids, cu, 2), lambda: c.attention(0, q, ids, cu, 4), lambda: c.attention(0, q, ids, cu, 4, max_len=256),
                 lambda: c.attention(0, q, ids, cu, 4, max_len=400), lambda: (c.attention(0, q[:0], ids, cu, 4), c.compact()),
                 lambda: c.truncate(ids, one),
                 lambda: c.fork(src, free), lambda: c.compact(), lambda: c.truncate(free),
                 lambda: be.attentionPacked(b, b[:, :128], b[:, 128:], cu, 4, 2, 64)):
        before = be.launches
        made = kernels(call)
        assert len(made) == be.launches - before, [k.name for k in made]


def test_status_words_of_a_cache_and_of_a_wait(be):
    """Role 32 alone is a cache that does not fit (TPB_ERR_STATE); a wait that ran out is TPB_ERR_TIMEOUT, the peer barrier's with its 0xBA above 32."""
    import ctypes as C

    from tensorpencil_b200 import _lib

    def poll():
        word = C.c_uint32(0)
        return be.lib.tpb_status_poll(be.h, be._stream(), C.byref(word)), word.value

    c, m = filled(be, [40, 20], "s8", 16, 1, 64, 3)
    q, x = torch.zeros((1, 128)).cuda(), torch.zeros((1, 64)).cuda()
    assert poll() == (_lib.TPB_OK, 0)
    c.attention(0, q, i32([9]), i32([0, 1]), 2)
    assert poll() == (_lib.TPB_ERR_STATE, (32 << 24) | 1)
    c.append(0, x, x, i32([0]), i32([0, 1]))
    assert poll() == (_lib.TPB_ERR_STATE, (32 << 24) | 4)
    c.table[0, 1], c.lens[1] = -1, -5
    c.read(0, i32([0]), i32([0, 1]), 1, start=i32([17]))
    assert poll() == (_lib.TPB_ERR_STATE, (32 << 24) | 2)
    c.attention(0, q, i32([1]), i32([0, 1]), 2)
    assert poll() == (_lib.TPB_ERR_STATE, (32 << 24) | 3)
    flags = [torch.zeros(128, dtype=torch.int32, device="cuda") for _ in range(2)]
    both = (C.c_void_p * 2)(*[f.data_ptr() for f in flags])
    be._check(be.lib.tpb_peer_barrier(be.h, be._stream(), both, 2, 0, 1, 50))      # a rank that never comes: gives up after 50 ms
    status, word = poll()
    assert status == _lib.TPB_ERR_TIMEOUT and word >> 24 == 0xBA
    assert poll() == (_lib.TPB_OK, 0)


def test_a_workspace_that_is_too_small_is_refused(be):
    from tensorpencil_b200 import _lib
    c, m = filled(be, [200, 20], "s8", 16, 2, 64, 3)
    q, out, ids, cu = torch.randn((2, 256)).cuda(), torch.full((2, 256), 7.0).cuda(), i32([0, 1]), i32([0, 1, 2])
    need = be.lib.tpb_kv_attention_workspace_bytes(be.h, 64)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    call = lambda max_len, ws, n: be.lib.tpb_kv_attention(be.h, be._stream(), c._d, 0, out.data_ptr(), 256, q.data_ptr(), 256,      # noqa: E731
                                                          _lib.TPB_F32, ids.data_ptr(), cu.data_ptr(), 2, 2, 4, 0.125, max_len, ws, n)
    assert need > 0
    for max_len in (0, 257):
        for n in (0, need // 2, need - 1):
            assert call(max_len, work.data_ptr(), n) == _lib.TPB_ERR_INVALID_ARG
        assert call(max_len, None, need) == _lib.TPB_ERR_INVALID_ARG
    be.status_poll()
    assert (out == 7.0).all()
    for max_len, ws, n in ((0, work.data_ptr(), need), (257, work.data_ptr(), need), (256, None, 0)):
        out.fill_(7.0)
        assert call(max_len, ws, n) == _lib.TPB_OK
        be.status_poll()
        check_attention(c, m, out, q, [0, 1], [1, 1], 4, "f32")


def test_what_a_refused_operation_says_and_where(be):
    """`result` alone tells of a refusal, until the next page operation; what a kernel skips is in the handle's status word, whatever comes after it, and
    the operation that met it is done."""
    from tensorpencil_b200 import _lib
    c, m = both(be, n_pages=6, max_seqs=4, max_pages=4, kv=1)
    other, _ = both(be, n_pages=2, kv=1)
    c.extend(i32([0]), i32([40])), m.extend([0], [40])
    for refused, status in (((c.extend, (i32([1]), i32([64]))), _lib.TPB_ERR_OOM), ((c.fork, (i32([0, 0]), i32([1, 2]), False)), _lib.TPB_ERR_OOM),
                            ((c.fork, (i32([0]), i32([0]))), _lib.TPB_ERR_INVALID_ARG), ((c.truncate, (i32([0, 0]),)), _lib.TPB_ERR_INVALID_ARG)):
        refused[0](*refused[1])
        assert c.result.tolist()[0] == status
        be.status_poll()
        c.extend(i32([3]), i32([0]))
        assert c.check() == 3
    m.tail[1] = m.tail[3] = 0
    m.result = c.result.tolist()
    same_tables(c, m)
    page = int(c.table[0, 1])
    c.table[0, 1] = 99
    c.fork(i32([0]), i32([1]))                             # skips that entry, and is done
    c.extend(i32([3]), i32([0]))
    assert c.result.tolist()[0] == _lib.TPB_OK and c.lens.tolist() == [40, 40, 0, 0] and int(c.table[1, 0]) == int(c.table[0, 0])
    with pytest.raises(_lib.TpbError) as e:
        other.check()                                      # the word is the handle's
    assert e.value.status == _lib.TPB_ERR_STATE
    assert c.check() == 2
    c.table[0, 1] = page


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads", [1, 8, 16, 24, 32])
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_f32_and_f16_rows_keep_both_terms(be, dt, heads, hd, fmt):
    """Inputs and bounds that one f16 term of the queries or of the weights would not meet (attn_accuracy.py, test_attn_accuracy.py)."""
    import attn_accuracy as acc
    page = 64
    for n in acc.TOKENS:
        q, k, v, ks, vs = acc.case(fmt, dt, n, heads, hd, n + hd)
        c, _ = both(be, n_pages=3, max_seqs=1, max_pages=2, page=page, kv=1, hd=hd, fmt=fmt)
        for t, sc, x, f in ((c.k, c.k_scale, k, ks), (c.v, c.v_scale, v, vs)):
            x = torch.from_numpy(x)
            t[0, 2, 0, :n] = (x.to(torch.int8) if fmt == "s8" else x.float().to(torch.float8_e4m3fn)).cuda()
            sc[0, 2, 0] = f
        c.table[0, 0], c.lens[0], c.refs[2] = 2, n, 1
        o, a, s = acc.formula(q, k, v, ks, vs)
        tol = acc.tolerance(o, a, s, vs, dt)
        for max_len in (0, n):
            out = c.attention(0, torch.from_numpy(q.reshape(1, -1)).to(DT[dt]).cuda(), i32([0]), i32([0, 1]), heads, scale=acc.SCALE, max_len=max_len)
            be.status_poll()
            err = np.abs(out.double().cpu().numpy().reshape(heads, hd) - o)
            assert (err <= tol).all(), (n, max_len, float((err / tol).max()))


@pytest.mark.parametrize("fmt", ["s8", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_scores_up_to_the_documented_limit(be, dt, fmt):
    """Single products up to 2^22, far apart or equal: a row's largest has all the weight, or its equals (of one scale) share it.  Scales are append's, powers
    of two, whose logarithms the references of the weights hold exactly."""
    kv, heads, hd = 1, 4, 64
    lens = [1, 4, 30]
    c, m = both(be, n_pages=8, max_seqs=3, max_pages=4, kv=kv, hd=hd, fmt=fmt)
    rng = np.random.default_rng(3)
    c.extend(i32(range(3)), i32(lens)), m.extend(range(3), lens)
    xs = []
    for n in lens:
        k = np.zeros((n, kv, hd))
        k[:, 0, 5] = 1024.0 + 1024.0 * rng.permutation(60)[:n] / 64.0       # 16 apart: s8 holds multiples of 16 here
        if fmt == "e4m3":
            k[:, 0, 5] = 1024.0 * 2.0 ** -np.arange(n) if n < 5 else 1024.0 * (1.0 + np.arange(n) % 2 / 8.0 * 7.0)
        xs.append((torch.from_numpy(k).to(DT[dt]).cuda(), values(rng, n, kv, hd, dt)))
    append(c, m, range(3), xs)
    q = torch.zeros((3, heads, hd))
    q[:, :, 5] = torch.tensor([2048.0, 2047.0 if dt != "bf16" else 2040.0, 2000.0, 1500.0])
    q = q.reshape(3, -1).to(DT[dt]).cuda()
    out = c.attention(0, q, i32(range(3)), offsets([1] * 3), heads, scale=1.0)
    be.status_poll()
    got, q = out.double().cpu().numpy(), q.double().cpu().numpy()
    for s in range(3):
        k, v = m.read(0, "k", s)[:, 0], m.read(0, "v", s)[:, 0]
        o, a, _ = attend(q[s].reshape(heads, hd), k, v, [lens[s] - 1] * heads, 1.0)
        tol = tolerance(o, a, np.zeros(heads), hd, HALF_STEP[dt], WEIGHTS[dt])
        assert (np.abs(got[s].reshape(heads, hd) - o) <= tol).all()
