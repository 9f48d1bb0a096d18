"""The paged key-value cache (include/kv_paged.h) against restatements on the
host: maps equal, appends to the rounding of each product, attention within
the bound of a 32-bit computation (tests/kv_paged_ref.py derives it)."""
import numpy as np
import pytest

import kv_paged_ref as ref
import pk_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch


def ints(torch, a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


# ---- map ----------------------------------------------------------------


def run_map(torch, kv, page, n_pages, length, start, end, table, free, max_rows, in_place=True, times=1):
    """A map call on lists: (error bits, table, free stack, rows, row0)."""
    n = len(length)
    d = [ints(torch, x) for x in (length, start, end)]
    tb = ints(torch, table)
    stack = torch.full((n_pages,), -5, dtype=torch.int32, device="cuda")
    stack[:len(free)] = ints(torch, free) if len(free) else stack[:0]
    nf = ints(torch, [len(free)])
    out = nf if in_place else ints(torch, [-9])
    rows = torch.full((3, max_rows), -77, dtype=torch.int32, device="cuda")
    row0 = torch.full((n + 1,), -77, dtype=torch.int32, device="cuda")
    step = 4 * max_rows
    for _ in range(times):
        kv.map(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), n, tb.data_ptr(), stack.data_ptr(), nf.data_ptr(),
               out.data_ptr(), max_rows, rows.data_ptr(), rows.data_ptr() + step, rows.data_ptr() + 2 * step,
               row0.data_ptr())
    code = kv.error()
    got = int(out[0])
    rows = rows.cpu().numpy()
    count = int(row0[-1])
    assert (rows[:, count:] == -1).all()
    return code, tb.cpu().tolist(), stack[:got].cpu().tolist(), [tuple(x) for x in rows[:, :count].T.tolist()], \
        row0.cpu().tolist()


def random_state(rng, n, page, blocks, n_pages):
    """Lengths whose pages are in the table, and the other pages on the stack."""
    ids = list(rng.permutation(n_pages))
    length, table = [], []
    for _ in range(n):
        a = int(rng.integers(0, blocks * page + 1))
        a = min(a, len(ids) * page)
        held = ref.pages_of(a, page)
        table.append([int(ids.pop()) for _ in range(held)] + [-3] * (blocks - held))
        length.append(a)
    return length, table, [int(x) for x in ids]


@pytest.mark.parametrize("n,page,blocks,n_pages", [(1, 1, 1, 1), (1, 16, 8, 9), (3, 7, 5, 12), (64, 16, 9, 400),
                                                   (257, 3, 6, 1100), (1000, 24, 4, 3000), (4096, 5, 3, 9000)])
@pytest.mark.parametrize("in_place", [True, False])
def test_map_random_steps(torch, n, page, blocks, n_pages, in_place):
    rng = np.random.default_rng(n + page)
    kv = pk_b200.KvPaged(1, 1, 8, pk_b200.F32, page, n_pages, n, blocks)
    length, table, free = random_state(rng, n, page, blocks, n_pages)
    for step in range(6):
        start = [int(rng.integers(0, a + 1)) if rng.random() < 0.4 else a for a in length]
        end = [int(rng.integers(s, blocks * page + 1)) if rng.random() < 0.5 else min(s + 1, blocks * page) for s in start]
        for i in range(n):
            if rng.random() < 0.2:
                start[i] = end[i] = 0
        want = ref.map_step(length, start, end, table, free, page, n_pages, 10 ** 9)
        max_rows = len(want[3]) + int(rng.integers(0, 9))
        want = ref.map_step(length, start, end, table, free, page, n_pages, max_rows)
        got = run_map(torch, kv, page, n_pages, length, start, end, table, free, max_rows, in_place,
                      times=1 if in_place else 3)
        assert got[0] == want[0]
        assert got[1] == want[1]
        assert got[2] == want[2]
        assert got[3] == want[3]
        assert got[4] == want[4]
        if want[0] == 0:
            length, table, free = end, want[1], want[2]
    kv.close()


def test_map_many_rows_over_several_ctas(torch):
    page, blocks, n_pages = 32, 300, 2000
    kv = pk_b200.KvPaged(1, 1, 8, pk_b200.F32, page, n_pages, 7, blocks)
    length, table = [0] * 7, [[-1] * blocks for _ in range(7)]
    free = [int(x) for x in np.random.default_rng(3).permutation(n_pages)]
    end = [9600, 1, 0, 31, 32, 33, 9599]
    for in_place in (True, False):
        for max_rows in (19296, 30001):
            want = ref.map_step(length, [0] * 7, end, table, free, page, n_pages, max_rows)
            assert run_map(torch, kv, page, n_pages, length, [0] * 7, end, table, free, max_rows, in_place) == want
    # a call that both gives pages back and takes those very pages again
    want = ref.map_step(length, [0] * 7, end, table, free, page, n_pages, 19296)
    code, table, free = want[:3]
    length, start, end = end, [0, 1, 0, 31, 0, 33, 9599], [0, 9600, 40, 64, 0, 33, 9600]
    assert len(free) < 1396
    want = ref.map_step(length, start, end, table, free, page, n_pages, 9700)
    assert want[0] == 0
    assert run_map(torch, kv, page, n_pages, length, start, end, table, free, 9700) == want
    kv.close()


@pytest.mark.parametrize("n,most,max_rows,off", [(50, 9000, 260001, 0), (50, 9000, 260001, 1), (1500, 400, 400003, 0),
                                                 (3, 100000, 299999, 3)])
def test_map_hundreds_of_thousands_of_rows(torch, n, most, max_rows, off):
    """More rows than threads: four of them a thread, stored in 16 bytes where
    the lists lie on 16 bytes (off 0) and singly where they do not."""
    page = 24
    rng = np.random.default_rng(n)
    blocks = -(-most // page)
    n_pages = n * blocks
    kv = pk_b200.KvPaged(1, 1, 8, pk_b200.F32, page, n_pages, n, blocks)
    start = rng.integers(0, 3, n) * (rng.random(n) < 0.3)
    end = np.maximum(start, np.minimum(rng.integers(0, most + 1, n), (max_rows - 5) // n))
    length = start + rng.integers(0, 2, n)
    length = np.minimum(length, most)
    table = np.full((n, blocks), -1)
    ids = rng.permutation(n_pages).tolist()
    for i in range(n):
        for b in range(ref.pages_of(int(length[i]), page)):
            table[i, b] = ids.pop()
    want = ref.map_step(length.tolist(), start.tolist(), end.tolist(), table.tolist(), ids, page, n_pages, max_rows)
    assert want[0] == 0 and max_rows > 148 * 1024
    d = [ints(torch, x) for x in (length, start, end)]
    tb, stack, nf = ints(torch, table), ints(torch, ids + [-5] * (n_pages - len(ids))), ints(torch, [len(ids)])
    rows = [torch.full((max_rows + 4,), -77, dtype=torch.int32, device="cuda") for _ in range(3)]
    row0 = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    kv.map(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), n, tb.data_ptr(), stack.data_ptr(), nf.data_ptr(),
           nf.data_ptr(), max_rows, *(r.data_ptr() + 4 * off for r in rows), row0.data_ptr())
    assert kv.error() == 0 and row0.cpu().tolist() == want[4] and tb.cpu().tolist() == want[1]
    assert stack[:int(nf[0])].cpu().tolist() == want[2]
    got = np.stack([r[off:off + max_rows].cpu().numpy() for r in rows], 1)
    count = len(want[3])
    assert np.array_equal(got[:count], np.asarray(want[3])) and (got[count:] == -1).all()
    for r in rows:  # nothing around the lists was written
        assert (r[:off] == -77).all() and (r[off + max_rows:] == -77).all()
    kv.close()


@pytest.mark.parametrize("change,code", [
    (dict(start=[3, 6, 0]), ref.BAD_LENGTH), (dict(start=[-1, 5, 0]), ref.BAD_LENGTH), (dict(end=[2, 6, 1]), ref.BAD_LENGTH),
    (dict(end=[3, 17, 1]), ref.BAD_LENGTH), (dict(length=[3, 2 ** 31 - 1, 0]), ref.BAD_LENGTH),
    (dict(end=[16, 16, 16]), ref.NO_PAGES), (dict(max_rows=1), ref.NO_ROWS),
    (dict(end=[16, 16, 16], max_rows=1), ref.NO_PAGES | ref.NO_ROWS),
])
def test_map_refuses_a_step_whole(torch, change, code):
    kv = pk_b200.KvPaged(1, 1, 8, pk_b200.F32, 4, 7, 3, 4)
    a = dict(length=[3, 5, 0], start=[3, 5, 0], end=[3, 6, 1], table=[[4, -1, -1, -1], [0, 6, -1, -1], [-1] * 4],
             free=[1, 2, 3, 5], max_rows=50)
    a.update(change)
    got = run_map(torch, kv, 4, 7, a["length"], a["start"], a["end"], a["table"], a["free"], a["max_rows"])
    assert got == (code, a["table"], a["free"], [], [0, 0, 0, 0])
    # the handle goes on working
    got = run_map(torch, kv, 4, 7, [3, 5, 0], [3, 5, 0], [3, 6, 1], a["table"], [1, 2, 3, 5], 50)
    assert got[0] == 0 and got[3] == [(1, 5, 25), (2, 0, 20)]
    kv.close()


def test_map_bad_pages_give_no_slot(torch):
    kv = pk_b200.KvPaged(1, 1, 8, pk_b200.F32, 4, 7, 3, 4)
    table = [[4, -1, -1, -1], [0, 7, -1, -1], [-1] * 4]
    got = run_map(torch, kv, 4, 7, [3, 5, 0], [2, 4, 0], [3, 6, 5], table, [1, 2, 99, 5], 9)
    want = ref.map_step([3, 5, 0], [2, 4, 0], [3, 6, 5], table, [1, 2, 99, 5], 4, 7, 9)
    assert want[0] == ref.BAD_PAGE and got == want
    kv.close()


# ---- append -------------------------------------------------------------

TYPES = {"f32": pk_b200.F32, "f16": pk_b200.F16}


def pool(torch, kind, shape, fill=3.5):
    return torch.full(shape, fill, device="cuda", dtype=torch.float16 if kind == "f16" else torch.float32)


def strides_of(layout, page, kvh, hs, n_pages):
    if layout == "token":
        return (0, 0, 0)
    if layout == "head":
        return (page * kvh * hs, hs, page * hs)
    return (page * (kvh * hs + 8) + 16, kvh * hs + 8, hs)  # "gaps": room between tokens and pages


def entries(layout, p, n_pages, page, kvh, hs):
    """The pool as numpy [page][token][head][channel]."""
    a = p.float().cpu().numpy().astype(np.float64)
    if layout == "token":
        return a.reshape(n_pages, page, kvh, hs)
    if layout == "head":
        return a.reshape(n_pages, kvh, page, hs).transpose(0, 2, 1, 3)
    ps, ts, _ = strides_of(layout, page, kvh, hs, n_pages)
    return np.lib.stride_tricks.as_strided(a, (n_pages, page, kvh, hs), (ps * 8, ts * 8, hs * 8, 8)).copy()


def pool_size(layout, n_pages, page, kvh, hs):
    ps = strides_of(layout, page, kvh, hs, n_pages)[0]
    return n_pages * (ps or page * kvh * hs)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("layout", ["token", "head", "gaps"])
@pytest.mark.parametrize("n,heads,kvh,hs,rope,page", [(1, 1, 1, 8, 8, 1), (5, 8, 2, 64, 64, 16), (33, 6, 3, 80, 42, 7),
                                                      (300, 4, 4, 128, 0, 24), (64, 32, 4, 64, 64, 32), (3, 5, 1, 256, 254, 5)])
def test_append(torch, kind, layout, n, heads, kvh, hs, rope, page):
    rng = np.random.default_rng(n * hs + rope)
    n_pages = n // page + 3
    kv = pk_b200.KvPaged(heads, kvh, hs, TYPES[kind], page, n_pages, 2, 4, strides=strides_of(layout, page, kvh, hs, n_pages))
    q = rng.standard_normal((n, heads, hs)).astype(np.float32)
    k = (3 * rng.standard_normal((n, kvh, hs))).astype(np.float32)
    v = rng.standard_normal((n, kvh, hs)).astype(np.float32)
    pos = rng.integers(0, 500, n)
    slot = rng.permutation(n_pages * page)[:n]
    skip = rng.random(n) < 0.2 if n > 1 else np.zeros(n, bool)
    slot[skip] = -1
    cs = ref.rope_table(500, rope)
    dq, dk, dv, dcs = (torch.from_numpy(x).cuda() for x in (q, k, v, cs))
    kp, vp = (pool(torch, kind, (pool_size(layout, n_pages, page, kvh, hs),)) for _ in range(2))
    qo = torch.full_like(dq, -7.0)
    rp, rs = ints(torch, pos), ints(torch, slot)
    kv.append(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), rp.data_ptr(), rs.data_ptr(), n, qo.data_ptr(), kp.data_ptr(),
              vp.data_ptr(), dcs.data_ptr() if rope else 0, rope, 500 if rope else 0)
    assert kv.error() == 0
    # the same rounding steps in 32 bits; so also within two roundings of the sizes in 64
    tq, tk = (ref.turn(x, cs, pos, rope, np.float32) if rope else x for x in (q, k))
    eq = ref.turn(q, cs, pos, rope, np.float64) if rope else q
    want_q = np.where(skip[:, None, None], np.float32(-7), tq)
    got_q = qo.cpu().numpy()
    assert np.array_equal(got_q, want_q)
    size = ref.turn(np.abs(q), np.abs(cs) * np.where(np.arange(max(rope, 1)) % 2, -1, 1)[:rope], pos, rope, np.float64) if rope else q
    even = np.abs(size[..., 0:rope:2]) if rope else 0
    if rope:
        err = np.abs(got_q - eq)[..., 0:rope:2][~skip]
        assert (err <= 2 * 2.0 ** -24 * even[~skip] * (1 + 2.0 ** -20)).all()
    store = np.float16 if kind == "f16" else np.float32
    for p, x in ((kp, tk), (vp, v)):
        want = np.full((n_pages, page, kvh, hs), 3.5)
        for r in range(n):
            if slot[r] >= 0:
                want[slot[r] // page, slot[r] % page] = x[r].astype(store)
        assert np.array_equal(entries(layout, p, n_pages, page, kvh, hs), want)
    if layout == "gaps":  # nothing between the entries was written
        assert int((kp == 3.5).sum()) >= kp.numel() - int((slot >= 0).sum()) * kvh * hs
    kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_append_fused_rows_in_place(torch, kind):
    """q, k and v as parts of one product's rows, q turned in place, and k and v alone."""
    rng = np.random.default_rng(5)
    n, heads, kvh, hs, page, n_pages = 9, 4, 2, 64, 4, 5
    kv = pk_b200.KvPaged(heads, kvh, hs, TYPES[kind], page, n_pages, 1, 5)
    wide = (heads + 2 * kvh) * hs
    x = rng.standard_normal((n, wide)).astype(np.float32)
    cs = ref.rope_table(50, hs)
    pos, slot = np.arange(n) + 30, rng.permutation(n_pages * page)[:n]
    d, dcs = torch.from_numpy(x).cuda(), torch.from_numpy(cs).cuda()
    kp, vp = (pool(torch, kind, (n_pages, page, kvh, hs)) for _ in range(2))
    rp, rs = ints(torch, pos), ints(torch, slot)
    at = d.data_ptr()
    kq, kk, kvv = at, at + heads * hs * 4, at + (heads + kvh) * hs * 4
    kv.append(kq, kk, kvv, rp.data_ptr(), rs.data_ptr(), n, kq, kp.data_ptr(), vp.data_ptr(), dcs.data_ptr(), hs, 50,
              q_stride=wide, kv_stride=wide)
    qk = ref.turn(x[:, :(heads + kvh) * hs].reshape(n, heads + kvh, hs), cs, pos, hs, np.float32)
    got = d.cpu().numpy()
    assert np.array_equal(got[:, :heads * hs].reshape(n, heads, hs), qk[:, :heads])
    assert np.array_equal(got[:, heads * hs:], x[:, heads * hs:])
    store = np.float16 if kind == "f16" else np.float32
    k1 = kp.cpu().numpy().reshape(-1, kvh, hs)[slot]
    assert np.array_equal(k1, qk[:, heads:].astype(store))
    kp2, vp2 = torch.zeros_like(kp), torch.zeros_like(vp)
    kv.append(0, kk, kvv, rp.data_ptr(), rs.data_ptr(), n, 0, kp2.data_ptr(), vp2.data_ptr(), dcs.data_ptr(), hs, 50,
              kv_stride=wide)
    assert np.array_equal(kp2.cpu().numpy().reshape(-1, kvh, hs)[slot], k1)
    assert kv.error() == 0
    kv.close()


def test_append_bad_rows_are_passed_over(torch):
    kvh, hs, page, n_pages = 1, 8, 4, 3
    kv = pk_b200.KvPaged(1, kvh, hs, pk_b200.F32, page, n_pages, 1, 3)
    k = torch.ones(5, hs, device="cuda")
    q, qo = torch.ones(5, hs, device="cuda"), torch.full((5, hs), -7.0, device="cuda")
    cs = torch.from_numpy(ref.rope_table(10, 8)).cuda()
    pos, slot = ints(torch, [0, 0, 10, -1, 0]), ints(torch, [3, 12, 4, 5, -9])
    guard = torch.zeros(n_pages * page + 8, hs, device="cuda")
    kv.append(q.data_ptr(), k.data_ptr(), k.data_ptr(), pos.data_ptr(), slot.data_ptr(), 5, qo.data_ptr(), guard.data_ptr(),
              guard.data_ptr(), cs.data_ptr(), 8, 10)
    assert kv.error() == ref.BAD_ROW and kv.error() == 0
    assert guard.sum(1).nonzero().flatten().tolist() == [3]
    assert (qo[1:] == -7).all() and (qo[0] == 1).all()
    kv.close()


# ---- attend -------------------------------------------------------------


class Setup:
    """Pools with random entries, tables of random pages, and rows."""

    def __init__(self, torch, kind, layout, heads, kvh, hs, page, lens, seed=0, q_scale=1.5, spare=2):
        rng = np.random.default_rng(seed + hs + page)
        self.torch, self.kind, self.layout = torch, kind, layout
        self.heads, self.kvh, self.hs, self.page = heads, kvh, hs, page
        self.lens = list(lens)
        n = len(self.lens)
        self.blocks = max(1, max(ref.pages_of(a, page) for a in self.lens))
        self.n_pages = sum(ref.pages_of(a, page) for a in self.lens) + spare
        ids = list(rng.permutation(self.n_pages))
        self.table = np.full((n, self.blocks), -1, dtype=np.int64)
        for i, a in enumerate(self.lens):
            for b in range(ref.pages_of(a, page)):
                self.table[i, b] = ids.pop()
        store = np.float16 if kind == "f16" else np.float32
        full = (self.n_pages, page, kvh, hs)
        self.k = rng.standard_normal(full).astype(store)
        self.v = rng.standard_normal(full).astype(store)
        self.q = (q_scale * rng.standard_normal((n, heads, hs))).astype(np.float32)
        self.req, self.pos = np.arange(n), np.asarray(self.lens) - 1
        self.scale = 1.0 / np.sqrt(hs)
        self.kv = pk_b200.KvPaged(heads, kvh, hs, TYPES[kind], page, self.n_pages, n, self.blocks,
                                  strides=strides_of(layout, page, kvh, hs, self.n_pages))

    def spoil(self, value):
        """Every entry that no row may use, in used pages too, holds `value`."""
        used = np.zeros((self.n_pages, self.page), bool)
        for r, i in enumerate(self.req):
            if i >= 0:
                for t in range(self.pos[r] + 1):
                    used[self.table[i, t // self.page], t % self.page] = True
        self.k[~used] = value
        self.v[~used] = value

    def device_pool(self, a):
        t, shape = self.torch, a.shape
        if self.layout == "head":
            a = a.transpose(0, 2, 1, 3)
        if self.layout == "gaps":
            ps, ts, _ = strides_of("gaps", self.page, self.kvh, self.hs, self.n_pages)
            buf = np.full(self.n_pages * ps, np.nan, a.dtype)
            z = a.dtype.itemsize
            np.lib.stride_tricks.as_strided(buf, shape, (ps * z, ts * z, self.hs * z, z))[:] = a
            a = buf
        return t.from_numpy(np.ascontiguousarray(a)).cuda()

    def run(self, stream=0):
        t = self.torch
        self.d = [t.from_numpy(self.q).cuda(), self.device_pool(self.k), self.device_pool(self.v), ints(t, self.table),
                  ints(t, self.req), ints(t, self.pos)]
        out = t.full((len(self.req), self.heads, self.hs), -7.0, device="cuda")
        t.cuda.synchronize()
        p = [x.data_ptr() for x in self.d]
        self.kv.attend(p[0], p[1], p[2], p[3], len(self.table), p[4], p[5], len(self.req), self.scale, out.data_ptr(),
                       stream=stream)
        t.cuda.synchronize()
        return out.cpu().numpy()

    def tokens(self, i, last):
        at = np.arange(last + 1)
        pages = self.table[i, at // self.page]
        return self.k[pages, at % self.page], self.v[pages, at % self.page]

    def check(self, out):
        for r, (i, last) in enumerate(zip(self.req, self.pos)):
            if i < 0:
                assert (out[r] == -7).all(), r
                continue
            k, v = self.tokens(i, last)
            want, weight, size = ref.attend(self.q[r], k, v, self.scale)
            tol = ref.attend_tolerance(weight, size, self.hs, last + 1)
            bad = np.abs(out[r] - want) > tol
            assert not bad.any(), (r, last, float(np.abs(out[r] - want).max()), float(tol.min()))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads,kvh,hs,page", [(1, 1, 8, 1), (8, 1, 64, 16), (32, 4, 64, 16), (4, 4, 128, 24),
                                               (12, 3, 128, 7), (24, 2, 80, 64), (5, 1, 256, 16), (9, 3, 72, 3),
                                               (16, 1, 200, 5), (6, 2, 16, 128), (28, 4, 112, 33)])
def test_attend_against_64_bits(torch, kind, heads, kvh, hs, page):
    lens = [1, 2, 3, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 200, 0]
    for layout in ("token", "head", "gaps"):
        s = Setup(torch, kind, layout, heads, kvh, hs, page, lens)
        s.check(s.run())
        assert s.kv.error() == 0
        s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hs,page", [(64, 16), (64, 7), (128, 8), (128, 64), (80, 24), (136, 32), (256, 5)])
def test_attend_never_uses_what_is_behind_a_row(torch, kind, value, hs, page):
    s = Setup(torch, kind, "token", 8, 2, hs, page, [1, 5, 16, 18, 47, 100, 0, 130])
    s.spoil(value)
    out = s.run()
    assert np.isfinite(out).all()
    assert (out[6] == 0).all()
    s.check(out)
    s.kv.close()


@pytest.mark.parametrize("heads,kvh", [(3, 3), (6, 3)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hs,page", [(32, 8), (64, 16), (64, 7), (72, 32), (128, 8), (128, 64), (160, 40), (256, 5),
                                     (256, 16)])
def test_attend_few_heads_never_use_what_is_behind_a_row(torch, heads, kvh, value, hs, page):
    s = Setup(torch, "f32", "token", heads, kvh, hs, page, [1, 5, 16, 18, 47, 100, 0, 130])
    s.spoil(value)
    out = s.run()
    assert np.isfinite(out).all()
    assert (out[6] == 0).all()
    s.check(out)
    s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_attend_rows_of_one_request_and_rows_passed_over(torch, kind):
    """Several rows of a request at different positions, in any order, rows
    without a request, and rows whose request is empty."""
    s = Setup(torch, kind, "token", 8, 4, 64, 16, [70, 3, 0, 40])
    s.req = np.array([0, 0, -1, 3, 1, 0, 2, -1, 3, 0])
    s.pos = np.array([69, 0, 5, 39, 2, 33, -1, -1, 7, 48])
    s.q = np.random.default_rng(1).standard_normal((10, 8, 64)).astype(np.float32)
    out = s.run()
    s.check(out)
    assert s.kv.error() == 0
    s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads,kvh,hs,page,lens", [(8, 1, 64, 16, [5000]), (32, 8, 128, 16, [4097, 1, 300]),
                                                    (2, 2, 128, 24, [9001, 8999]), (16, 1, 32, 1, [777] * 5)])
def test_attend_counts_every_token_once(torch, kind, heads, kvh, hs, page, lens):
    """Equal scores and small whole values: sums are exact in 32 bits, so a
    token that is missed or taken twice shows. One division (or a reciprocal
    and a product): two roundings."""
    s = Setup(torch, kind, "token", heads, kvh, hs, page, lens)
    s.q[:] = 0
    s.v = np.random.default_rng(2).integers(-8, 9, s.v.shape).astype(s.v.dtype)
    out = s.run()
    for r, a in enumerate(lens):
        _, v = s.tokens(r, a - 1)
        want = np.repeat(v.astype(np.float64).sum(0) / a, heads // kvh, axis=0)
        assert (np.abs(out[r] - want) <= 3 * 2.0 ** -24 * np.abs(want)).all()
    s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_attend_single_token_takes_all(torch, kind):
    """A score far above the others picks its token's values, wherever it lies."""
    lens = [300] * 12
    s = Setup(torch, kind, "head", 4, 2, 64, 16, lens)
    for r, t in enumerate((0, 1, 15, 16, 63, 64, 127, 128, 255, 256, 298, 299)):
        page = s.table[r, t // 16]
        s.k[page, t % 16] = 0
        s.k[page, t % 16, :, 0] = 1000.0
        s.q[r, :, 0] = 10.0
    out = s.run()
    for r, t in enumerate((0, 1, 15, 16, 63, 64, 127, 128, 255, 256, 298, 299)):
        v = s.v[s.table[r, t // 16], t % 16].astype(np.float64)
        want = np.repeat(v, 2, axis=0)
        assert (np.abs(out[r] - want) <= 2.0 ** -22 * np.abs(want)).all(), t
    s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("q_scale", [1e-30, 1e-4, 30.0, 3e4])
def test_attend_sizes_of_q(torch, kind, q_scale):
    """Queries from far below to far above the usual: the split of q and the running maximum hold."""
    s = Setup(torch, kind, "token", 8, 2, 64, 16, [1, 50, 129, 300], q_scale=q_scale)
    out = s.run()
    assert np.isfinite(out).all()
    s.check(out)
    s.kv.close()


@pytest.mark.parametrize("n,kind", [(127, "f32"), (129, "f16"), (1000, "f16"), (5000, "f32")])
def test_attend_many_rows(torch, n, kind):
    """More rows than a CTA has threads, some passed over, over few requests
    and pages."""
    rng = np.random.default_rng(n)
    s = Setup(torch, kind, "head", 4, 2, 64, 8, [60, 33, 90, 0, 7])
    s.req = rng.integers(-1, 5, n)
    s.pos = np.array([rng.integers(-1, max(1, s.lens[i])) if i >= 0 else 3 for i in s.req])
    s.pos[s.req == 3] = -1
    s.q = rng.standard_normal((n, 4, 64)).astype(np.float32)
    s.check(s.run())
    assert s.kv.error() == 0
    s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_attend_nan_stays_in_its_head(torch, kind):
    """A query or a value that is not a number spoils its own heads only."""
    s = Setup(torch, kind, "token", 8, 2, 64, 16, [300, 300, 40])
    good = s.run()
    s.q[0, 3, 5] = np.nan
    s.v[s.table[1, 2], 4, 1, 7] = np.nan  # request 1, KV head 1: query heads 4 .. 7, channel 7
    out = s.run()
    bad = np.isnan(out)
    assert bad[0, 3].all() and bad[1, 4:, 7].all() and bad.sum() == 64 + 4
    assert np.array_equal(out[~bad], good[~bad])
    s.kv.close()


def test_attend_refuses_too_much_work(torch):
    """2^31 chunks (a billion tokens for each of 256 KV heads) give an error
    bit and no output; the table is one page again and again."""
    page, blocks = 1 << 20, 1 << 10
    kv = pk_b200.KvPaged(256, 256, 8, pk_b200.F16, page, 1, 1, blocks)
    kp = torch.zeros(page * 256 * 8, device="cuda", dtype=torch.float16)
    q, out = torch.zeros(1, 256, 8, device="cuda"), torch.full((1, 256, 8), -7.0, device="cuda")
    tb, rr, rp = ints(torch, [[0] * blocks]), ints(torch, [0]), ints(torch, [(1 << 30) - 1])
    args = (q.data_ptr(), kp.data_ptr(), kp.data_ptr(), tb.data_ptr(), 1, rr.data_ptr(), rp.data_ptr(), 1, 1.0, out.data_ptr())
    kv.attend(*args)
    assert kv.error() == 32 and (out == -7).all()
    rp.fill_(1000)
    kv.attend(*args)
    assert kv.error() == 0 and (out == 0).all()
    kv.close()


def test_attend_bad_pages_and_rows(torch):
    s = Setup(torch, "f16", "token", 8, 2, 64, 16, [40, 64, 20])
    good = s.run()
    assert s.kv.error() == 0
    s.table[0, 1] = s.n_pages  # tokens 16..31 of request 0 are left out
    s.req[2] = 3
    out = s.run()
    assert s.kv.error() == ref.BAD_PAGE | ref.BAD_ROW
    assert np.array_equal(out[1], good[1]) and (out[2] == -7).all()
    at = np.r_[0:16, 32:40]
    pages = s.table[0, at // 16]
    want, weight, size = ref.attend(s.q[0], s.k[pages, at % 16], s.v[pages, at % 16], s.scale)
    assert (np.abs(out[0] - want) <= ref.attend_tolerance(weight, size, 64, 24)).all()
    s.table[0, :] = -1         # nothing is left of request 0
    s.req[2], s.pos[2] = 2, 64  # behind the table's end: the row's own last token is the end
    s.pos[1] = 2 ** 31 - 1
    out = s.run()
    assert s.kv.error() == ref.BAD_PAGE | ref.BAD_ROW
    assert (out[0] == 0).all() and np.array_equal(out[1], good[1])
    s.kv.close()


def test_attend_same_bits_again(torch):
    s = Setup(torch, "f16", "token", 32, 8, 128, 16, [3000, 1, 700, 64, 65])
    a = s.run()
    for _ in range(4):
        assert np.array_equal(a, s.run())
    s.kv.close()


def test_attend_far_pages(torch):
    """Page offsets past 2^31 entries: the pool's pages stand 2^27 entries apart."""
    page, kvh, hs, n_pages = 16, 1, 64, 20
    stride = 1 << 27
    kv = pk_b200.KvPaged(2, kvh, hs, pk_b200.F16, page, n_pages, 1, 3, strides=(stride, hs, hs))
    k = torch.empty(stride * (n_pages - 1) + page * hs, device="cuda", dtype=torch.float16)
    v = k  # one pool for both: 5 GB
    g = torch.Generator(device="cuda").manual_seed(1)
    table = [19, 2, 17]
    toks = torch.randn(3, page, hs, device="cuda", generator=g).half()
    for b, p in enumerate(table):
        k[p * stride:p * stride + page * hs] = toks[b].flatten()
    q = torch.randn(1, 2, hs, device="cuda", generator=g)
    out = torch.empty_like(q)
    tb, rr, rp = ints(torch, [table]), ints(torch, [0]), ints(torch, [40])
    kv.attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), tb.data_ptr(), 1, rr.data_ptr(), rp.data_ptr(), 1, 0.125,
              out.data_ptr())
    t = toks.cpu().numpy().reshape(48, 1, hs)[:41]
    want, weight, size = ref.attend(q[0].cpu().numpy(), t, t, 0.125)
    assert (np.abs(out[0].cpu().numpy() - want) <= ref.attend_tolerance(weight, size, hs, 41)).all()
    # and a row appended into the farthest page
    one = torch.ones(1, hs, device="cuda")
    rs = ints(torch, [19 * page + 15])
    kv.append(0, one.data_ptr(), one.data_ptr(), rp.data_ptr(), rs.data_ptr(), 1, 0, k.data_ptr(), v.data_ptr())
    assert (k[-hs:] == 1).all() and kv.error() == 0
    kv.close()


# ---- a step's calls together --------------------------------------------


class Server:
    """Requests that grow, are cut back and end, over steps of map, append and
    attend; the host keeps every request's keys and values without pages."""

    def __init__(self, torch, kind, heads=8, kvh=2, hs=64, page=16, n=5, blocks=8, n_pages=25, max_rows=40, seed=0):
        self.t, self.kind = torch, kind
        self.heads, self.kvh, self.hs, self.page, self.n = heads, kvh, hs, page, n
        self.blocks, self.n_pages, self.max_rows = blocks, n_pages, max_rows
        self.rng = np.random.default_rng(seed)
        self.kv = pk_b200.KvPaged(heads, kvh, hs, TYPES[kind], page, n_pages, n, blocks)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.dlen, self.dstart, self.dend = (torch.zeros(n, **i32) for _ in range(3))
        self.table = torch.full((n, blocks), -1, **i32)
        self.free = torch.arange(n_pages, **i32)
        self.n_free = torch.full((1,), n_pages, **i32)
        self.rows = [torch.empty(max_rows, **i32) for _ in range(3)]
        self.row0 = torch.empty(n + 1, **i32)
        shape = (n_pages, page, kvh, hs)
        self.kp, self.vp = (pool(torch, kind, shape, float("nan")) for _ in range(2))
        self.cs_h = ref.rope_table(blocks * page, hs)
        self.cs = torch.from_numpy(self.cs_h).cuda()
        self.q = torch.zeros(max_rows, heads, hs, device="cuda")
        self.k, self.v = (torch.zeros(max_rows, kvh, hs, device="cuda") for _ in range(2))
        self.out = torch.zeros_like(self.q)
        self.hk = [np.zeros((0, kvh, hs)) for _ in range(n)]
        self.hv = [np.zeros((0, kvh, hs)) for _ in range(n)]

    def calls(self, stream=0):
        r = [x.data_ptr() for x in self.rows]
        self.kv.map(self.dlen.data_ptr(), self.dstart.data_ptr(), self.dend.data_ptr(), self.n, self.table.data_ptr(),
                    self.free.data_ptr(), self.n_free.data_ptr(), self.n_free.data_ptr(), self.max_rows, *r,
                    self.row0.data_ptr(), stream=stream)
        self.kv.append(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), r[1], r[2], self.max_rows, self.q.data_ptr(),
                       self.kp.data_ptr(), self.vp.data_ptr(), self.cs.data_ptr(), self.hs, len(self.cs_h), stream=stream)
        self.kv.attend(self.q.data_ptr(), self.kp.data_ptr(), self.vp.data_ptr(), self.table.data_ptr(), self.n, r[0], r[1],
                       self.max_rows, 0.125, self.out.data_ptr(), stream=stream)

    def plan(self, start, end):
        self.start, self.end = start, end
        self.dlen.copy_(ints(self.t, [len(x) for x in self.hk]))
        self.dstart.copy_(ints(self.t, start))
        self.dend.copy_(ints(self.t, end))
        self.hq = self.rng.standard_normal(self.q.shape).astype(np.float32)
        self.hnk = self.rng.standard_normal(self.k.shape).astype(np.float32)
        self.hnv = self.rng.standard_normal(self.k.shape).astype(np.float32)
        for d, h in ((self.q, self.hq), (self.k, self.hnk), (self.v, self.hnv)):
            d.copy_(self.t.from_numpy(h))
        self.out.fill_(-7.0)
        self.t.cuda.synchronize()

    def check(self):
        assert self.kv.error() == 0
        out, store = self.out.cpu().numpy(), np.float16 if self.kind == "f16" else np.float32
        r = 0
        for i in range(self.n):
            s, e = self.start[i], self.end[i]
            pos = np.arange(s, e)
            turned = ref.turn(self.hnk[r:r + e - s], self.cs_h, pos, self.hs, np.float32).astype(store)
            self.hk[i] = np.concatenate([self.hk[i][:s], turned])
            self.hv[i] = np.concatenate([self.hv[i][:s], self.hnv[r:r + e - s].astype(store)])
            q = ref.turn(self.hq[r:r + e - s], self.cs_h, pos, self.hs, np.float32)
            for j, p in enumerate(pos):
                want, weight, size = ref.attend(q[j], self.hk[i][:p + 1], self.hv[i][:p + 1], 0.125)
                tol = ref.attend_tolerance(weight, size, self.hs, p + 1)
                assert (np.abs(out[r + j] - want) <= tol).all(), (i, p)
            r += e - s
        assert (out[r:] == -7).all()
        held = sum(ref.pages_of(len(x), self.page) for x in self.hk)
        assert int(self.n_free[0]) == self.n_pages - held
        pages = [int(self.table[i, b]) for i in range(self.n) for b in range(ref.pages_of(len(self.hk[i]), self.page))]
        pages += self.free[:int(self.n_free[0])].tolist()
        assert sorted(pages) == list(range(self.n_pages))

    STEPS = [([0, 0, 0, 0, 0], [17, 3, 0, 1, 16]),       # prompts
             ([17, 3, 0, 1, 16], [18, 4, 1, 2, 17]),     # a token each
             ([15, 4, 1, 0, 17], [20, 4, 30, 0, 18]),    # drafts taken back, a prompt, a request that ends
             ([20, 4, 30, 0, 18], [20, 4, 30, 0, 18]),   # nothing
             ([0, 4, 16, 0, 18], [0, 40, 17, 1, 19]),    # pages given back and taken again
             ([0, 40, 17, 1, 19], [1, 41, 18, 2, 20])]


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_steps_of_a_server(torch, kind):
    s = Server(torch, kind)
    for start, end in s.STEPS:
        s.plan(start, end)
        s.calls()
        s.check()
    s.kv.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_steps_captured_once_and_replayed(torch, kind):
    """One graph for max_rows rows serves every step, on a stream of its own;
    a step that is refused on the device leaves all outputs as they were."""
    s = Server(torch, kind, seed=4)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        s.calls(stream=torch.cuda.current_stream().cuda_stream)
    for start, end in s.STEPS:
        s.plan(start, end)
        g.replay()
        s.check()
    s.plan([1, 41, 18, 2, 20], [1, 128, 18, 2, 20])  # more rows than the graph has
    g.replay()
    assert s.kv.error() == ref.NO_ROWS
    assert (s.out == -7).all()
    s.kv.close()


def test_two_graphs_of_one_handle_in_turn(torch):
    """Two captured calls that share a handle's scratch, replayed one after
    the other on one stream, with lengths that change between replays."""
    s = Setup(torch, "f16", "token", 32, 8, 128, 16, [3000, 900, 1])
    s.run()
    st, graphs, outs = torch.cuda.Stream(), [], []
    p = [x.data_ptr() for x in s.d]
    for rows in (3, 2):
        out = torch.full((3, 32, 128), -7.0, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.kv.attend(p[0], p[1], p[2], p[3], 3, p[4], p[5], rows, s.scale, out.data_ptr(),
                        stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
        outs.append(out)
    for lens in ([3000, 900, 1], [1, 17, 0], [2049, 1, 1], [3000, 900, 1]):
        s.pos = np.asarray(lens) - 1
        s.d[5].copy_(ints(torch, s.pos))
        for g in graphs:
            g.replay()
        a, b = (o.cpu().numpy() for o in outs)
        s.check(a)
        assert np.array_equal(a[:2], b[:2]) and (b[2] == -7).all()
    assert s.kv.error() == 0
    s.kv.close()


def test_another_stream(torch):
    s = Setup(torch, "f16", "token", 8, 2, 64, 16, [300, 20])
    st = torch.cuda.Stream()
    s.check(s.run(stream=st.cuda_stream))
    s.kv.close()


def test_another_current_device(torch):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    s = Setup(torch, "f16", "token", 8, 2, 64, 16, [300, 20])
    with torch.cuda.device(1):
        out = s.run()
        assert torch.cuda.current_device() == 1
    s.check(out)
    s.kv.close()


def test_two_handles_side_by_side(torch):
    """Two handles over the same pools on two streams at once."""
    a = Setup(torch, "f16", "token", 32, 8, 128, 16, [2000, 900, 1])
    first = a.run()
    b = pk_b200.KvPaged(32, 8, 128, pk_b200.F16, 16, a.n_pages, 3, a.blocks)
    outs = [torch.full((3, 32, 128), -7.0, device="cuda") for _ in range(2)]
    sts = [torch.cuda.Stream() for _ in range(2)]
    p = [x.data_ptr() for x in a.d]
    torch.cuda.synchronize()
    for _ in range(20):
        for kv, o, st in zip((a.kv, b), outs, sts):
            kv.attend(p[0], p[1], p[2], p[3], 3, p[4], p[5], 3, a.scale, o.data_ptr(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.cpu().numpy(), first)
    a.kv.close()
    b.close()
