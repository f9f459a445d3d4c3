"""What the calls of packed attention and of the 8-bit key / value cache refuse before anything is launched.  No device: the C entry
points get a zeroed stand-in for a handle, which they only write their message to, and the Python methods CPU tensors.  Also the index
arithmetic that the kernels' launches rely on."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from tensorpencil_b200 import _lib  # noqa: E402
from tensorpencil_b200.backend import Backend  # noqa: E402
from tensorpencil_b200.kv_cache import KvCache  # noqa: E402

INVALID = _lib.TPB_ERR_INVALID_ARG


@pytest.fixture(scope="module")
def lib():
    from tensorpencil_b200 import build
    build.build()
    return _lib.load()


@pytest.fixture()
def handle():
    buf = C.create_string_buffer(1 << 20)
    at = (C.addressof(buf) + 255) & ~255
    yield at
    del buf


PACKED = dict(out=4096, ld_out=256, q=4096, ld_q=256, k=4096, ld_k=128, v=4096, ld_v=128, dtype=_lib.TPB_BF16, cu=4096, n_seqs=2, tokens=10,
              heads=4, kv_heads=2, head_dim=64, scale=0.1)


@pytest.mark.parametrize("change", [dict(dtype=_lib.TPB_F32), dict(dtype=_lib.TPB_S32), dict(head_dim=96), dict(head_dim=256, heads=1, kv_heads=1),
                                    dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(heads=258), dict(n_seqs=-1), dict(tokens=-1),
                                    dict(tokens=1 << 26), dict(out=0), dict(q=0), dict(k=0), dict(v=0), dict(cu=0), dict(q=4104), dict(out=4098),
                                    dict(cu=4097), dict(ld_q=248), dict(ld_out=252), dict(ld_k=127), dict(ld_k=64), dict(scale=-1.0),
                                    dict(scale=float("nan")), dict(scale=float("inf"))])
def test_attention_packed_refuses(lib, handle, change):
    a = {**PACKED, **change}
    assert lib.tpb_attention_packed(handle, None, *a.values()) == INVALID
    assert lib.tpb_attention_packed(None, None, *PACKED.values()) == INVALID


def test_nothing_to_do_is_no_error(lib, handle):
    for change in (dict(tokens=0), dict(n_seqs=0)):
        assert lib.tpb_attention_packed(handle, None, *{**PACKED, **change, "q": 0}.values()) == 0


def desc(**change):
    d = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, table=4096, lens=4096, tail=4096, refs=4096, result=4096, scratch=4096, n_pages=100,
             layers=2, kv_heads=2, page_tokens=16, head_dim=64, max_seqs=4, max_pages=10, format=0)
    d.update(change)
    return _lib.KvCacheDesc(**d)


def calls_on(lib, h, c):
    """Every call on a cache, with good arguments otherwise."""
    return [lib.tpb_kv_extend(h, None, c, 4096, 4096, 1), lib.tpb_kv_truncate(h, None, c, 4096, None, 1), lib.tpb_kv_fork(h, None, c, 4096, 4096, 1, 1),
            lib.tpb_kv_compact(h, None, c), lib.tpb_kv_append(h, None, c, 0, 4096, 128, 4096, 128, 0, 4096, 4096, 1, 1),
            lib.tpb_kv_read(h, None, c, 0, 4096, 128, 4096, 128, 0, 4096, None, 4096, 1, 1),
            lib.tpb_kv_attention(h, None, c, 0, 4096, 256, 4096, 256, 0, 4096, 4096, 1, 1, 4, 0.1, 0, 4096, 1 << 40)]


@pytest.mark.parametrize("change", [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(table=0), dict(lens=0), dict(tail=0), dict(refs=0),
                                    dict(result=0), dict(scratch=0), dict(k=4097), dict(v=4104), dict(table=4098), dict(n_pages=0),
                                    dict(n_pages=(1 << 24) + 1), dict(layers=0), dict(kv_heads=0), dict(kv_heads=65536, n_pages=1, layers=1),
                                    dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=128), dict(head_dim=32), dict(head_dim=256),
                                    dict(max_seqs=0), dict(max_pages=0), dict(format=2), dict(n_pages=1 << 24, layers=4),
                                    dict(max_pages=1 << 27), dict(max_seqs=1 << 20, max_pages=1 << 11)])
def test_every_call_refuses_a_bad_cache(lib, handle, change):
    assert calls_on(lib, handle, C.addressof(desc(**change))) == [INVALID] * 7
    assert calls_on(lib, handle, None) == [INVALID] * 7
    assert calls_on(lib, None, C.addressof(desc())) == [INVALID] * 7


def test_page_operations_refuse_bad_lists(lib, handle):
    c = C.addressof(desc())
    assert lib.tpb_kv_extend(handle, None, c, None, 4096, 1) == INVALID
    assert lib.tpb_kv_extend(handle, None, c, 4096, None, 1) == INVALID
    assert lib.tpb_kv_extend(handle, None, c, 4097, 4096, 1) == INVALID
    assert lib.tpb_kv_extend(handle, None, c, 4096, 4096, -1) == INVALID
    assert lib.tpb_kv_truncate(handle, None, c, None, None, 1) == INVALID
    assert lib.tpb_kv_fork(handle, None, c, 4096, None, 1, 0) == INVALID


ROWS = dict(layer=0, a=4096, ld_a=128, b=4096, ld_b=128, dtype=0, seqs=4096, cu=4096, n_seqs=1, rows=1)
BAD_ROWS = [dict(layer=2), dict(layer=-1), dict(a=0), dict(b=0), dict(a=4100), dict(ld_a=64), dict(ld_b=130), dict(dtype=3), dict(dtype=9),
            dict(dtype=1, ld_a=132), dict(seqs=0), dict(cu=0), dict(seqs=4097), dict(n_seqs=-1), dict(rows=-1), dict(rows=1 << 26)]


@pytest.mark.parametrize("change", BAD_ROWS)
def test_append_and_read_refuse(lib, handle, change):
    c = C.addressof(desc())
    a = {**ROWS, **change}
    assert lib.tpb_kv_append(handle, None, c, *a.values()) == INVALID
    r = list(a.values())
    assert lib.tpb_kv_read(handle, None, c, *r[:7], None, *r[7:]) == INVALID


@pytest.mark.parametrize("change", [dict(layer=2), dict(out=0), dict(q=0), dict(q=4100), dict(ld_out=128), dict(ld_q=250), dict(dtype=3), dict(seqs=0),
                                    dict(cu=0), dict(cu=4099), dict(n_seqs=-1), dict(rows=-1), dict(heads=3), dict(heads=0), dict(heads=65536),
                                    dict(scale=-0.5), dict(scale=float("nan")), dict(max_len=-1), dict(work=0), dict(work=4100)])
def test_attention_refuses(lib, handle, change):
    a = dict(layer=0, out=4096, ld_out=256, q=4096, ld_q=256, dtype=0, seqs=4096, cu=4096, n_seqs=1, rows=1, heads=4, scale=0.1, max_len=0, work=4096,
             nbytes=1 << 40)
    assert lib.tpb_kv_attention(handle, None, C.addressof(desc()), *{**a, **change}.values()) == INVALID


def test_a_small_workspace_is_refused(lib, handle):
    assert lib.tpb_kv_attention_workspace_bytes(None, 64) == 0 and lib.tpb_kv_attention_workspace_bytes(handle, 96) == 0
    C.c_int.from_address(handle)                           # the stand-in has no SMs: its workspace is empty, so ask the sizes alone
    assert lib.tpb_kv_scratch_bytes(100, 4) == 4 * (8 + 8 + 200)
    assert [lib.tpb_kv_scratch_bytes(*a) for a in ((0, 4), (100, 0), ((1 << 24) + 1, 4), (-1, 1))] == [0] * 4


def cpu_backend():
    be = Backend.__new__(Backend)                          # no device, no library behind it: the checks come first
    be.device, be._index = torch.device("cpu"), -1
    return be


def test_attention_packed_refuses_tensors():
    be = cpu_backend()
    q, k = torch.zeros(10, 256, dtype=torch.bfloat16), torch.zeros(10, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32)
    call = lambda q=q, k=k, v=k, cu=cu, heads=4, out=None: be.attentionPacked(q, k, v, cu, heads, 2, 64, out=out)      # noqa: E731
    for bad in (dict(q=q.float(), k=k.float(), v=k.float()), dict(k=k.half()), dict(cu=cu.long()), dict(out=q.float())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(q=q[:, :192]), dict(k=k[:9]), dict(v=k.t().contiguous().t()), dict(heads=8), dict(cu=cu.view(1, 2)), dict(out=q[:5]),
                dict(cu=torch.zeros(4, dtype=torch.int32)[::2]), dict(q=q.view(10, 2, 128))):
        with pytest.raises(ValueError):
            call(**bad)


def test_a_cache_refuses_tensors_that_do_not_fit():
    be = cpu_backend()
    shape = (1, 6, 2, 16, 64)
    good = dict(k=torch.zeros(shape, dtype=torch.int8), v=torch.zeros(shape, dtype=torch.int8), k_scale=torch.zeros(shape[:3]), v_scale=torch.zeros(shape[:3]),
                table=torch.zeros((3, 4), dtype=torch.int32), lens=torch.zeros(3, dtype=torch.int32), refs=torch.zeros(6, dtype=torch.int32),
                tail=torch.zeros(3, dtype=torch.int32))
    for name, t in (("k", good["k"].float()), ("v", good["v"].view(torch.uint8)), ("k_scale", good["k_scale"].half()), ("lens", good["lens"].long()),
                    ("table", good["table"].float())):
        with pytest.raises(TypeError):
            KvCache.wrap(be, **{**good, name: t})
    for name, t in (("k", good["k"][0]), ("v", good["v"][:, :5]), ("k_scale", good["k_scale"][:, :5]), ("lens", good["lens"][:2]),
                    ("table", good["table"][0]), ("refs", good["refs"][:3]), ("tail", torch.zeros(6, dtype=torch.int32)[::2]),
                    ("v_scale", good["v_scale"].to("meta"))):
        with pytest.raises(ValueError):
            KvCache.wrap(be, **{**good, name: t})
    with pytest.raises(TypeError):
        KvCache(be, 1, 4, 2, 64, 2, 2, dtype="int8")
    with pytest.raises(ValueError):
        KvCache(be, 1, 0, 2, 64, 2, 2)


def test_cache_methods_refuse_tensors():
    c = KvCache.__new__(KvCache)
    c.be, c.kv_heads, c.head_dim, c._index = cpu_backend(), 2, 64, -1
    x, ids, cu = torch.zeros(5, 128), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(k=x.double(), v=x.double()), dict(v=x.half()), dict(k=x.to(torch.int8))):
        with pytest.raises(TypeError):
            c.append(0, **{"k": x, "v": x, "seqs": ids, "cu": cu, **bad})
    for bad in (dict(k=x[:, :64]), dict(v=x[:4]), dict(v=x.t().contiguous().t())):
        with pytest.raises(ValueError):
            c.append(0, **{"k": x, "v": x, "seqs": ids, "cu": cu, **bad})
    with pytest.raises(TypeError):
        c._ints("seqs", ids.long(), 1)
    with pytest.raises(ValueError):
        c._ints("cu", cu, 3)
    with pytest.raises(ValueError):
        c._rows("q", torch.zeros(5, 256), 5, 8, torch.float32)
    c._index = 0                                           # tensors of another device than the cache's
    for call in (lambda: c._rows("q", torch.zeros(5, 128), 5, 2, torch.float32), lambda: c._ints("cu", cu, 2)):
        with pytest.raises(ValueError):
            call()
    be = cpu_backend()
    be._index = 0
    with pytest.raises(ValueError):
        be._packed_ld("q", torch.zeros(5, 128), 5, 2, 64)


def test_places_of_the_append_launch():
    """Sequence i's places cu[i] / page + 2 i .. cu[i + 1] / page + 2 (i + 1) - 1 are as many as the pages that its new tokens can touch,
    wherever they begin, and the launch has them all."""
    rnd = random.Random(3)
    for _ in range(400):
        page, n = rnd.choice([16, 32, 64]), rnd.randint(1, 9)
        new = [rnd.choice([0, 1, rnd.randint(0, 5 * page)]) for _ in range(n)]
        cu = [sum(new[:i]) for i in range(n + 1)]
        place = [cu[i] // page + 2 * i for i in range(n + 1)]
        assert place[n] <= cu[n] // page + 2 * n               # the launch's grid
        for i in range(n):
            first = rnd.randint(0, 10 * page)
            touched = (first + new[i] - 1) // page - first // page + 1 if new[i] else 0
            assert touched <= place[i + 1] - place[i]


def test_tables_of_a_scratch_hold_every_list():
    """marks and offsets a sequence, two lists a page, eight words in front: the order that the kernels cut the scratch in."""
    lib = _lib.load()
    for pages, seqs in ((1, 1), (17, 3), (70001, 1300)):
        assert lib.tpb_kv_scratch_bytes(pages, seqs) // 4 == 8 + seqs + seqs + pages + pages


@pytest.fixture(scope="module")
def page_at_place(tmp_path_factory):
    """The kernel's own arithmetic, compiled for the host."""
    gxx, cuda = shutil.which("g++"), "/usr/local/cuda/include"
    if gxx is None or not os.path.isdir(cuda):
        pytest.skip("no g++ / CUDA headers")
    root, at = os.path.dirname(os.path.dirname(os.path.abspath(__file__))), tmp_path_factory.mktemp("places")
    src, out = at / "places.cpp", at / "places.so"
    src.write_text('#include "kv_common.cuh"\n'
                   'extern "C" int at(int x, int i, int r0, int first, int len, int shift) { return tpb_kv::page_at_place(x, i, r0, first, len, shift); }\n')
    r = subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(root, "include"), "-I",
                        os.path.join(root, "tensorpencil_b200", "csrc"), "-I", cuda, str(src), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return C.CDLL(str(out)).at


def test_every_new_page_has_one_place_and_no_place_another_page(page_at_place):
    """Over the whole grid of an append, with rows of nobody ahead of the first sequence and behind the last: the pages that a sequence's new tokens touch
    come up once each, and nothing else does (no entry in front of the sequence's row of the table, none of an earlier page)."""
    rnd = random.Random(5)
    for trial in range(300):
        shift, n = rnd.choice([4, 5, 6]), rnd.randint(1, 6)
        page = 1 << shift
        lead = [0, 1, page - 1, page, 3 * page, 40 * page + 5][trial % 6]
        new = [rnd.choice([0, 1, rnd.randint(0, 5 * page)]) for _ in range(n)]
        cu = [lead + sum(new[:i]) for i in range(n + 1)]
        first = [rnd.choice([0, 0, rnd.randint(0, 10 * page)]) for _ in range(n)]
        rows = cu[n] + rnd.choice([0, 1, 2 * page])
        seen = [[] for _ in range(n)]
        for x in range(rows // page + 2 * n):
            i = max([0] + [j for j in range(n) if cu[j] // page + 2 * j <= x])      # the kernel's search: sequence 0 where there is none
            if new[i] == 0:
                continue
            pg = page_at_place(x, i, cu[i], first[i], first[i] + new[i], shift)
            if pg != -1:
                seen[i].append(pg)
        for i in range(n):
            assert seen[i] == (list(range(first[i] // page, (first[i] + new[i] - 1) // page + 1)) if new[i] else [])
    assert page_at_place(0, 0, 48, 0, 1, 4) == -1 and page_at_place(3, 0, 48, 0, 1, 4) == 0
    # offsets out of order, which a call may not have, lead nowhere else either
    for _ in range(2000):
        shift, first, n_new = rnd.choice([4, 5, 6]), rnd.randint(0, 1 << 29), rnd.randint(1, 1 << 20)
        pg = page_at_place(rnd.randint(0, 1 << 23), rnd.randint(0, 1 << 22), rnd.randint(0, 1 << 26), first, first + n_new, shift)
        assert pg == -1 or first >> shift <= pg <= (first + n_new - 1) >> shift


def test_launches_are_counted_as_they_are_made():
    """Backend.launches counts kernels: attention over the cache is two where a workspace joins parts, and a call with nothing to do is none."""
    class Calls:
        def __getattr__(self, name):
            return lambda *a: 0

    be = cpu_backend()
    be._hv, be._stream, be.launches, be._attn_calls = 0, lambda: 0, 0, Calls()
    c = KvCache.__new__(KvCache)
    c.be, c.kv_heads, c.head_dim, c._index, c._calls, c._d, c._like = be, 2, 64, -1, Calls(), 0, {}
    c._scale, c._no_workspace, c._scratch, c._workspace_bytes = 0.125, _lib.KV_SHORT, torch.empty(8, dtype=torch.uint8), 64
    ids, cu, none = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    zero = torch.zeros(1, dtype=torch.int32)
    x, q = torch.zeros(5, 128), torch.zeros(5, 256)
    b = q.bfloat16()
    for call, want in ((lambda: c.append(0, x, x, ids, cu), 1), (lambda: c.append(0, x[:0], x[:0], ids, cu), 0),
                       (lambda: c.append(0, x, x, none, zero), 0),
                       (lambda: c.read(0, ids, cu, 5), 1), (lambda: c.read(0, ids, cu, 0), 0), (lambda: c.read(0, none, zero, 5), 0),
                       (lambda: c.attention(0, q, ids, cu, 4), 2), (lambda: c.attention(0, q, ids, cu, 4, max_len=257), 2),
                       (lambda: c.attention(0, q, ids, cu, 4, max_len=256), 1), (lambda: c.attention(0, q[:0], ids, cu, 4), 0),
                       (lambda: c.attention(0, q, none, zero, 4), 0),
                       (lambda: be.attentionPacked(b, b[:, :128], b[:, :128], cu, 4, 2, 64), 1),
                       (lambda: be.attentionPacked(b, b[:, :128], b[:, :128], zero, 4, 2, 64), 0),
                       (lambda: be.attentionPacked(b[:0], b[:0, :128], b[:0, :128], cu, 4, 2, 64), 0)):
        before = be.launches
        call()
        assert be.launches - before == want


def test_workspaces_are_measured_before_anything_is_launched(lib):
    """A stand-in handle with SMs: every word of it is written with its own place until the library's answer tells where the number of SMs lies."""
    buf = (C.c_int32 * (1 << 18))(*range(1, (1 << 18) + 1))
    handle = (C.addressof(buf) + 255) & ~255
    word = lib.tpb_device_sm_count(handle)
    C.memset(buf, 0, C.sizeof(buf))
    buf[word - 1] = 148
    assert lib.tpb_device_sm_count(handle) == 148
    c = C.addressof(desc())
    need = lib.tpb_kv_attention_workspace_bytes(handle, 64)
    assert need >= 148 * 2 * 32 * (64 + 3) * 4
    for max_len in (0, 257, 1 << 20):
        for work, nbytes in ((4096, need - 1), (4096, need // 2), (4096, 0), (0, need)):
            assert lib.tpb_kv_attention(handle, None, c, 0, 4096, 256, 4096, 256, 0, 4096, 4096, 1, 1, 4, 0.1, max_len, work, nbytes) == INVALID
