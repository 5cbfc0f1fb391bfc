"""GPU parity of select_blocks (top-n 64-token blocks by the indexer's scores) against its CPU restatement."""
import numpy as np
import pytest
import torch

from oracle import sparse as O

pytestmark = pytest.mark.gpu


def _mask_words(bits):
    rows, width = bits.shape
    pad = np.zeros((rows, -(-width // 16) * 16), bool)
    pad[:, :width] = bits
    w = (pad.reshape(rows, -1, 16) * (1 << np.arange(16))).sum(-1)
    return w.astype(np.uint16).view(np.int16)


def _make(rows, width, lens, kind, seed):
    g = np.random.default_rng(seed)
    s = g.standard_normal((rows, width)).astype(np.float32)
    if kind == "ties":      # few distinct values: the threshold is a tie nearly everywhere
        s = np.round(s).astype(np.float32)
    elif kind == "negative":
        s = -np.abs(s)
    elif kind == "zeros":   # unset mask bits dominate
        s[g.random((rows, width)) < 0.999] = 0
    elif kind == "inf":
        s[g.random((rows, width)) < 0.002] = np.inf
        s[g.random((rows, width)) < 0.3] = -np.inf
    elif kind == "minus0":
        s = np.where(g.random((rows, width)) < 0.5, np.float32(-0.0), np.float32(-1)).astype(np.float32)
    bits = (s.view(np.int32) != 0) & (np.arange(width)[None] < np.asarray(lens)[:, None])
    return s, bits


SHAPES = [(1, 64, [1]), (2, 100, [0, 100]), (3, 4096, [4096, 1, 65]), (5, 5056, [5056, 5055, 4999, 640, 641]),
          (2, 131072, [131001, 70000]), (300, 2112, None), (40, 16384, None)]


@pytest.mark.parametrize("kind", ["normal", "ties", "negative", "zeros", "inf", "minus0"])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}" for s in SHAPES])
def test_matches_restatement(hcu, dev, shape, kind):
    rows, width, lens = shape
    if lens is None:
        lens = np.random.default_rng(1).integers(-3, width + 100, rows)
    lens = np.asarray(lens, np.int32)
    s, bits = _make(rows, width, lens, kind, 7)
    # values where the mask bit is clear are not defined: poison them
    d = np.where(bits, s, np.float32(np.nan))
    stride = -(-width // 4) * 4
    buf = torch.full((rows, stride + 4), float("inf"), device=dev)
    buf[:, :width] = torch.from_numpy(d).to(dev)
    mask = torch.from_numpy(_mask_words(bits)).to(dev)
    L = torch.from_numpy(lens).to(dev)
    for n, sink, local in ((1, 0, 0), (8, 1, 2), (31, 0, 0), (64, 2, 4), (128, 0, 1)):
        got = hcu.select_blocks(buf[:, :width], mask, L, n, n_sink=sink, n_local=local).cpu().numpy()
        some = range(rows) if rows <= 5 else range(0, rows, 13)
        for r in some:
            ref = O.select_blocks(s[r], bits[r], int(np.clip(lens[r], 0, width)), n, sink, local)
            assert np.array_equal(got[r], ref), (r, n, sink, local)


def test_reads_the_logits_of_the_indexer(hcu, dev):
    """Fed by mqa_logits itself, whose scores are written at set bits only."""
    from hcu_ops.workloads import make_decode

    w = make_decode(3, 2, [9000, 4100, 130], heads=64, seed=3)
    d = {k: (v.to(dev) if torch.is_tensor(v) else v) for k, v in w.items()}
    logits, mask = hcu.mqa_logits(d["q"], d["kv_cache"], d["weights"], d["context_lens"], d["block_table"],
                                  d["max_context_len"], d["group_size"])
    got = hcu.select_blocks(logits, mask, d["context_lens"], 32, n_sink=1, n_local=2).cpu().numpy()
    lg, mk = logits.cpu().numpy(), mask.cpu().numpy().view(np.uint16)
    bits = ((mk[:, :, None] >> np.arange(16)) & 1).reshape(lg.shape).astype(bool)
    for r in range(6):
        assert np.array_equal(got[r], O.select_blocks(lg[r], bits[r], int(w["context_lens"][r]), 32, 1, 2))


def test_graph_replay_and_side_stream(hcu, dev):
    rows, width = 4, 8192
    lens = np.array([8192, 5000, 64, 3], np.int32)
    s, bits = _make(rows, width, lens, "normal", 2)
    S, M, L = torch.from_numpy(s).to(dev), torch.from_numpy(_mask_words(bits)).to(dev), torch.from_numpy(lens).to(dev)
    hcu.select_blocks(S, M, L, 16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = hcu.select_blocks(S, M, L, 16)
    s2, bits2 = _make(rows, width, lens, "normal", 9)
    S.copy_(torch.from_numpy(s2))
    M.copy_(torch.from_numpy(_mask_words(bits2)))
    g.replay()
    got = out.cpu().numpy()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got2 = hcu.select_blocks(S, M, L, 16)
    side.synchronize()
    for r in range(rows):
        ref = O.select_blocks(s2[r], bits2[r], int(lens[r]), 16, 1, 1)
        assert np.array_equal(got[r], ref) and np.array_equal(got2[r].cpu().numpy(), ref)


def test_refusals_and_empty(hcu, dev):
    S = torch.zeros(2, 256, device=dev)
    M = torch.zeros(2, 16, dtype=torch.int16, device=dev)
    L = torch.full((2,), 256, dtype=torch.int32, device=dev)
    assert hcu.select_blocks(S[:0], M[:0], L[:0], 4).shape == (0, 4)
    for args in ((S.half(), M, L, 4), (S.t(), M, L, 4), (S, M[:, :8], L, 4), (S, M, L.long(), 4), (S, M, L[:1], 4),
                 (S, M, L, 0), (S, M, L, 4, 3, 2), (S, M, L, 4, -1, 0), (S[:, :250][:, 1:], M, L, 4)):
        with pytest.raises(RuntimeError):
            hcu.select_blocks(*args)
