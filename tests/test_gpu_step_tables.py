"""GPU parity of step_tables (block tables, slot maps, page allocation) against its CPU restatement."""
import numpy as np
import pytest
import torch

from oracle import sparse as O

pytestmark = pytest.mark.gpu

# (requests, lengths lo..hi, new lo..hi, width, max_pages, rows beyond the new tokens)
CASES = [(1, 0, 0, 1, 1, 64, 1, 0), (1, 63, 64, 1, 2, 128, 2, 0), (3, 0, 130, 0, 3, 256, 5, 4),
         (5, 60, 70, 5, 9, 192, 3, 0), (33, 1, 900, 1, 4, 1024, 17, 1), (300, 0, 500, 0, 2, 576, 9, 0),
         (2, 100, 9000, 200, 700, 16384, 160, 3), (64, 4096, 16000, 2, 2, 16448, 257, 0)]


def _make(case, seed):
    b, lo, hi, nlo, nhi, width, mp, extra = case
    g = np.random.default_rng(seed)
    seq = g.integers(lo, hi + 1, b).astype(np.int32)
    new = np.minimum(g.integers(nlo, nhi + 1, b), min(width, mp * 64) - seq).astype(np.int32)
    need = int((-(-(seq + new) // 64) - -(-seq // 64)).sum())
    ids = g.permutation(2 * b * mp + need + 7).astype(np.int32)
    rp = ids[:2 * b * mp].reshape(2 * b, mp).copy()
    free = ids[2 * b * mp:].copy()
    return rp, g.permutation(2 * b)[:b].astype(np.int32), seq, new, free, int(new.sum()) + extra, width


def _call(hcu, dev, rp, idx, seq, new, free, head, rows, width):
    t = [torch.from_numpy(np.ascontiguousarray(x)).to(dev) for x in (rp, idx, seq, new, free)]
    h = torch.tensor([head], dtype=torch.int32, device=dev)
    out = hcu.step_tables(*t, h, rows, width)
    got = {k: v.cpu().numpy() for k, v in out._asdict().items()}
    got["req_pages"] = t[0].cpu().numpy()
    return got


@pytest.mark.parametrize("case", CASES, ids=[f"b{c[0]}-w{c[5]}" for c in CASES])
def test_matches_restatement(hcu, dev, case):
    rp, idx, seq, new, free, rows, width = _make(case, 11)
    for head in (0, 5):
        ref = O.step_tables(rp, idx, seq, new, free, head, rows, width)
        got = _call(hcu, dev, rp, idx, seq, new, free, head, rows, width)
        for k, v in ref.items():
            assert np.array_equal(got[k], v), k


def test_row_strided_pages_and_two_steps(hcu, dev):
    """req_pages as a view with a longer row stride; the second step continues from the first one's state."""
    rp, idx, seq, new, free, rows, width = _make((7, 50, 500, 1, 80, 1024, 16, 0), 3)
    big = torch.full((14, 40), -7, dtype=torch.int32, device=dev)
    big[:, 8:24] = torch.from_numpy(rp).to(dev)
    view = big[:, 8:24]
    t = [torch.from_numpy(x).to(dev) for x in (idx, seq, new, free)]
    head = torch.zeros(1, dtype=torch.int32, device=dev)
    free2 = np.concatenate([free, np.arange(10000, 10100, dtype=np.int32)])
    f2 = torch.from_numpy(free2).to(dev)
    a = hcu.step_tables(view, t[0], t[1], t[2], f2, head, rows, width)
    r1 = O.step_tables(rp, idx, seq, new, free2, 0, rows, width)
    b = hcu.step_tables(view, t[0], t[1] + t[2], torch.ones_like(t[2]), f2, a.free_head, 7, width)
    r2 = O.step_tables(r1["req_pages"], idx, seq + new, np.ones_like(new), free2, int(r1["free_head"][0]), 7, width)
    for k in ("block_table", "page_table_size_1", "loc", "free_head"):
        assert np.array_equal(getattr(a, k).cpu().numpy(), r1[k]), k
        assert np.array_equal(getattr(b, k).cpu().numpy(), r2[k]), k
    assert np.array_equal(view.cpu().numpy(), r2["req_pages"])
    assert (big[:, :8] == -7).all() and (big[:, 24:] == -7).all()


def test_exhausted_pages_and_bad_lengths_are_flagged(hcu, dev, request):
    request.node.allowed_status = 2
    rp = np.arange(8, dtype=np.int32).reshape(2, 4)
    one = np.array([1], np.int32)
    # one free page for a request that needs two: the second page and its tokens are -1
    got = _call(hcu, dev, rp, np.array([0], np.int32), np.array([60], np.int32), np.array([70], np.int32),
                np.array([99], np.int32), 0, 70, 256)
    assert hcu.read_device_status(clear=True) & 2
    assert got["block_table"][0].tolist() == [0, 99, -1, -1] and got["free_head"][0] == 2
    assert got["loc"][3] == 63 and got["loc"][4] == 99 * 64 and got["loc"][69] == -1
    assert got["page_table_size_1"][0, 127] == 99 * 64 + 63 and (got["page_table_size_1"][0, 128:] == -1).all()
    # a request row out of range, a negative length, more tokens than rows
    for idx, seq, new, rows in ((5, 3, 1, 1), (0, -4, 1, 1), (0, 3, 4, 2)):
        got = _call(hcu, dev, rp, np.array([idx], np.int32), np.array([seq], np.int32), np.array([new], np.int32),
                    one, 0, rows, 256)
        assert hcu.read_device_status(clear=True) & 2, (idx, seq, new)
        if idx == 5:
            assert (got["block_table"] == -1).all() and got["loc"][0] == -1
            assert np.array_equal(got["req_pages"], rp)
    # outgrown width: the tables are cut, the length too
    got = _call(hcu, dev, rp, np.array([1], np.int32), np.array([130], np.int32), one, one, 0, 1, 128)
    assert hcu.read_device_status(clear=True) & 2
    assert got["block_table"][0].tolist() == [4, 5] and got["lengths"][0] == 128 and got["loc"][0] == 6 * 64 + 2


def test_graph_replay_follows_the_lengths(hcu, dev):
    rp, idx, seq, new, free, rows, width = _make((9, 10, 700, 2, 2, 1024, 16, 0), 5)
    t = [torch.from_numpy(x).to(dev) for x in (rp, idx, seq, new, free)]
    head = torch.zeros(1, dtype=torch.int32, device=dev)
    hcu.step_tables(*t, head, rows, width)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = hcu.step_tables(*t, head, rows, width)
    seq2 = np.minimum(seq + 61, 1000).astype(np.int32)
    t[0].copy_(torch.from_numpy(rp))
    t[2].copy_(torch.from_numpy(seq2))
    g.replay()
    ref = O.step_tables(rp, idx, seq2, new, free, 0, rows, width)
    for k in ("block_table", "page_table_size_1", "lengths", "loc", "free_head"):
        assert np.array_equal(getattr(out, k).cpu().numpy(), ref[k]), k


def test_refusals(hcu, dev):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    ok = [i(2, 4), i(2), i(2), i(2), i(8), i(1), 2, 256]
    hcu.step_tables(*ok)
    for k, bad in ((0, i(2, 4).long()), (0, i(4, 2).t()), (1, i(3)), (2, i(2).long()), (4, i(2, 4)), (5, i(2)),
                   (6, -1), (7, 100), (7, 0), (3, i(4)[::2])):
        a = list(ok)
        a[k] = bad
        with pytest.raises(RuntimeError):
            hcu.step_tables(*a)
