"""Batched decode over a pool of pages (engine_batch_open_paged) against the
oracle's single-sequence forward and against the contiguous batched state:
the same logits (1e-3 max-abs, as the other batched tests) and greedy tokens,
whatever pages the sequences get, share out and give back."""
import numpy as np
import pytest

import pk_b200

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-3


def feed(e, refs, rows, check=True):
    """One step of rows (token, position, sequence); every row's logits against
    its oracle. Returns the greedy tokens."""
    out = e.forward_batch([r[0] for r in rows], [r[1] for r in rows], [r[2] for r in rows], logits=True)
    assert out is not None, e.last_error()
    nxt, lg = out
    if check:
        # the oracle takes a sequence's rows in the order of their positions
        for i in sorted(range(len(rows)), key=lambda i: (rows[i][2], rows[i][1])):
            t, p, s = rows[i]
            want = np.asarray(refs[s].forward(int(t), int(p))).copy()
            assert float(np.max(np.abs(lg[i] - want))) <= LOGIT_TOL, rows[i]
            assert int(nxt[i]) == int(np.argmax(want)), rows[i]
    return nxt


@pytest.mark.parametrize("preset", ["tiny-q4km", "tiny-q5k", "tiny-legacy", "tiny-float", "tp-q4km"])
@pytest.mark.parametrize("page", [1, 7, 16])
def test_decode_matches_oracle(orc, synth_model, preset, page):
    """Prompts in chunks, then greedy decoding, sequences joining one by one,
    rows in any order."""
    path = synth_model(preset)
    e = pk_b200.Engine(path, 64, device=0)
    seqs = [3, 0, 4]
    e.batch_open_paged(5, page, 3 * (-(-40 // page)) + 1)
    total = e.batch_free_pages()
    rng = np.random.default_rng(page)
    refs = {s: orc.open(path, 64) for s in seqs}
    prompts = {s: list(rng.integers(0, e.vocab_size, size=int(rng.integers(3, 20)))) for s in seqs}
    length, last = {}, {}
    for step in range(10):
        rows = []
        for j, s in enumerate(seqs):
            if step == 2 * j:
                rows += [(t, p, s) for p, t in enumerate(prompts[s])]
            elif s in last:
                rows.append((last[s], length[s], s))
        rng.shuffle(rows)
        rows = [tuple(int(x) for x in r) for r in rows]
        nxt = feed(e, refs, rows)
        for s in {r[2] for r in rows}:
            i = max((p, k) for k, (_, p, q) in enumerate(rows) if q == s)[1]
            length[s], last[s] = rows[i][1] + 1, int(nxt[i])
        assert e.batch_free_pages() == total - sum(-(-n // page) for n in length.values())
    for r in refs.values():
        r.close()
    e.close()


def test_pages_are_shared_out_and_given_back(orc, synth_model):
    """Fewer pages than whole contexts: a call that needs more is refused and
    changes nothing, a release makes room, and a new text in the same place
    of the batch is right."""
    path = synth_model("tiny-q4km")
    e = pk_b200.Engine(path, 64, device=0)
    e.batch_open_paged(3, 4, 6)
    refs = {s: orc.open(path, 64) for s in range(3)}
    a = [(10 + i, i, 0) for i in range(13)]  # 4 pages
    b = [(50 + i, i, 1) for i in range(8)]   # 2 pages
    feed(e, refs, a + b)
    assert e.batch_free_pages() == 0
    assert e.forward_batch([1], [0], [2]) is None
    assert "Not enough free pages: 1 needed, 0 left" in e.last_error()
    assert e.forward_batch([7, 7], [13, 8], [0, 1]) is None  # sequence 1 would need a page
    feed(e, refs, [(7, 13, 0)])                               # sequence 0 alone does not
    assert e.batch_release(0) and e.batch_free_pages() == 4
    refs[0].close()
    refs[0] = orc.open(path, 64)
    feed(e, refs, [(90, 0, 0), (7, 8, 1), (33, 0, 2)])
    feed(e, refs, [(91, 1, 0), (8, 9, 1), (34, 1, 2)])
    assert e.batch_free_pages() == 1
    assert e.batch_release(2) and e.batch_release(2) and e.batch_free_pages() == 2
    assert not e.batch_release(3) and not e.batch_release(-1)
    for r in refs.values():
        r.close()
    e.close()


def test_positions_are_taken_back(orc, synth_model):
    """Rows at positions that were filled replace what was there and behind
    (rejected drafts), down to position 0."""
    path = synth_model("tiny-q4km")
    e = pk_b200.Engine(path, 64, device=0)
    e.batch_open_paged(2, 4, 8)
    refs = {s: orc.open(path, 64) for s in range(2)}
    feed(e, refs, [(t, p, 0) for p, t in enumerate(range(20, 31))] + [(5, 0, 1)])
    assert e.batch_free_pages() == 8 - 3 - 1
    feed(e, refs, [(100, 6, 0), (101, 7, 0)])  # positions 6 .. 10 are taken back
    assert e.batch_free_pages() == 8 - 2 - 1
    assert e.forward_batch([1], [9], [0]) is None and "no K/V" in e.last_error()
    feed(e, refs, [(102, 8, 0), (6, 1, 1)])
    feed(e, refs, [(60, 0, 0), (61, 1, 0)])    # a new text
    assert e.batch_free_pages() == 8 - 1 - 1
    assert e.forward_batch([1, 2], [2, 4], [0, 0]) is None    # a gap
    assert e.forward_batch([1, 2], [0, 2], [0, 0]) is None    # not consecutive, though both are filled or next
    assert "consecutive" in e.last_error()
    feed(e, refs, [(62, 2, 0)])
    for r in refs.values():
        r.close()
    e.close()


@pytest.mark.parametrize("half", [False, True])
def test_same_as_contiguous(synth_model, monkeypatch, half):
    """64 sequences over pages and over contiguous caches, float and half, with
    a context put in by engine_kv_write: logits within the bound, the same tokens."""
    if half:
        monkeypatch.setenv("POCKET_CUDA_KV", "f16")
    path = synth_model("tp-q4km")
    rng = np.random.default_rng(8)
    ctx, n, layers, kvd = 300, 64, 3, 256
    runs = []
    for paged in (False, True):
        e = pk_b200.Engine(path, 512, device=0)
        if paged:
            e.batch_open_paged(n, 16, 700)
        else:
            e.batch_open(n)
        rng = np.random.default_rng(8)
        for s in (0, 5, 63):
            for layer in range(layers):
                k, v = (rng.standard_normal((ctx, kvd)).astype(np.float32) for _ in range(2))
                e.kv_write(layer, 0, k, v, seq=s)
        pos = np.zeros(n, int)
        pos[[0, 5, 63]] = ctx
        toks = rng.integers(0, e.vocab_size, n)
        got = []
        for _ in range(4):
            nxt, lg = e.forward_batch(toks, pos, np.arange(n), logits=True)
            got.append((nxt.copy(), lg.copy()))
            toks, pos = nxt, pos + 1
        # later positions of a context are replaced: the map finds their pages again
        k, v = (rng.standard_normal((5, kvd)).astype(np.float32) for _ in range(2))
        for layer in range(layers):
            e.kv_write(layer, ctx - 10, k, v, seq=5)
        nxt, lg = e.forward_batch(toks, pos, np.arange(n), logits=True)
        got.append((nxt.copy(), lg.copy()))
        if paged:
            assert e.batch_free_pages() == 700 - 61 - 3 * 20
        runs.append(got)
        e.close()
    for (ta, la), (tb, lb) in zip(*runs):
        assert float(np.max(np.abs(la - lb))) <= LOGIT_TOL
        assert np.array_equal(ta, tb)


def test_kv_write_refuses_without_pages(synth_model):
    path = synth_model("tiny-q4km")
    e = pk_b200.Engine(path, 64, device=0)
    e.batch_open_paged(2, 4, 2)
    k = np.zeros((9, 64), np.float32)
    with pytest.raises(RuntimeError, match="Not enough free pages"):
        e.kv_write(0, 0, k, k, seq=1)
    e.kv_write(0, 0, k[:8], k[:8], seq=1)
    assert e.batch_free_pages() == 0
    with pytest.raises(RuntimeError, match="gap"):
        e.kv_write(0, 1, k[:1], k[:1], seq=0)
    e.close()


def test_open_refusals(synth_model):
    path = synth_model("tiny-q4km")
    e = pk_b200.Engine(path, 64, device=0)
    assert e.batch_free_pages() == -1 and not e.batch_release(0)
    for bad in ((0, 16, 4), (65, 16, 4), (2, 0, 4), (2, 16, 0), (2, 1 << 20, 1 << 20)):
        with pytest.raises(RuntimeError):
            e.batch_open_paged(*bad)
        assert e.forward_batch([1], [0], [0]) is None
    e.batch_open_paged(2, 16, 4)
    assert e.batch_free_pages() == 4
    e.batch_open(2)  # back to contiguous caches
    assert e.batch_free_pages() == -1 and e.batch_release(1)
    assert e.forward_batch([1, 2], [0, 0], [0, 1]) is not None
    # the single-sequence path is independent of the batched state
    assert e.forward(1, 0) is not None
    e.close()
