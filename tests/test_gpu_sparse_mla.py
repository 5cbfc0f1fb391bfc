"""GPU parity of sparse_mla_attention / block_sparse_mla_attention against the 64-bit restatement
(``oracle/sparse.py``, whose ``attend`` derives the bounds): both slot formats, both forms, head
counts, lengths from nothing to long, strides, masked and poisoned places, streams and graphs."""
import numpy as np
import pytest
import torch

from oracle import sparse as O

pytestmark = pytest.mark.gpu

SCALE = 1.0 / 16.0
# relative error of a k operand (f16 of a group's scale ratio, then of the product); the 4-bit
# values are exact but for the rounding the bound allows in the accumulation
EPS = {"fp8": 2.0 ** -11, "kv4": 2.0 ** -14}
SLOT = {"fp8": 656, "kv4": 432}


def _pool(fmt, slots, seed, stride=None):
    """uint8 [slots, stride] of valid slots of mixed magnitudes."""
    g = torch.Generator().manual_seed(seed)
    lat = torch.randn(slots, 512, generator=g) * torch.exp2(torch.randint(-3, 3, (slots, 4), generator=g).float()
                                                             ).repeat_interleave(128, 1)
    lat, rope = lat.bfloat16(), torch.randn(slots, 64, generator=g).bfloat16()
    u = lambda t: t.contiguous().view(torch.int16).numpy().view(np.uint16)
    if fmt == "kv4":
        body = O.kv4_pack(u(lat), u(rope))
    else:
        x = lat.float().view(slots, 4, 128)
        sc = (x.abs().amax(-1).clamp_min(1e-6) / 448).float()
        q = (x / sc[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(slots, 512).view(torch.uint8).numpy()
        body = np.concatenate([q, sc.contiguous().view(torch.uint8).numpy().reshape(slots, 16),
                               u(rope).view(np.uint8).reshape(slots, 128)], 1)
    out = np.full((slots, stride or SLOT[fmt]), 0xFF, np.uint8)
    out[:, :SLOT[fmt]] = body
    return out


def _values(fmt, pool, slots):
    return (O.fp8_values if fmt == "fp8" else O.kv4_values)(pool[slots])


def _q(rows, heads, seed, gain=1.0):
    return (torch.randn(rows, heads, 576, generator=torch.Generator().manual_seed(seed)) * gain).bfloat16()


def _check(fmt, q, pool, lists, out, lse, scale=SCALE):
    """Every row of (out, lse) within its bounds; lists: per row the slots it attends to."""
    qd = q.double().numpy()
    o, z = out.float().cpu().double().numpy(), lse.cpu().double().numpy()
    worst = 0.0
    for r, sl in enumerate(lists):
        ro, rl, to, tl = O.attend(qd[r], _values(fmt, pool, np.asarray(sl, np.int64)), scale, EPS[fmt])
        if len(sl) == 0:
            assert (o[r] == 0).all() and np.isneginf(z[r]).all(), r
            continue
        e = np.abs(o[r] - ro) / to
        assert e.max() <= 1, (r, float(e.max()))
        assert (np.abs(z[r] - rl) <= tl).all(), (r, float((np.abs(z[r] - rl) / tl).max()))
        worst = max(worst, float(e.max()))
    return worst


CASES = [(1, 64, 1), (1, 64, 63), (2, 64, 64), (3, 64, 65), (1, 64, 2048), (4, 8, 130), (3, 1, 200), (2, 16, 1000),
         (2, 48, 129), (2, 128, 257), (5, 72, 66), (150, 64, 96), (300, 16, 33)]


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
@pytest.mark.parametrize("rows,heads,n", CASES)
def test_tokens(hcu, dev, fmt, rows, heads, n):
    pool = _pool(fmt, 3000, 1)
    g = np.random.default_rng(rows * 1000 + n)
    idx = g.integers(0, 3000, (rows, n)).astype(np.int32)
    idx[g.random((rows, n)) < 0.03] = -1
    if rows > 1:
        idx[1, n // 3:] = -1      # a short row
    if rows > 2:
        idx[2] = -1               # a row with nothing
    q = _q(rows, heads, 2)
    out, lse = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(pool).to(dev).view(3000, 1, -1),
                                        torch.from_numpy(idx).to(dev), SCALE)
    assert out.shape == (rows, heads, 512) and out.dtype == torch.bfloat16 and lse.dtype == torch.float32
    some = range(rows) if rows <= 5 else list(range(0, 5)) + list(range(5, rows, 29))
    _check(fmt, q[list(some)], pool, [idx[r][idx[r] >= 0] for r in some], out[list(some)], lse[list(some)])


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
@pytest.mark.parametrize("rows,heads,n", [(1, 64, 1), (3, 64, 7), (2, 16, 32), (6, 128, 5), (160, 64, 3)])
def test_blocks(hcu, dev, fmt, rows, heads, n):
    pool = _pool(fmt, 64 * 40, 3)
    g = np.random.default_rng(rows * 77 + n)
    pages = 36
    table = np.stack([g.permutation(40)[:pages] for _ in range(rows)]).astype(np.int32)
    lens = g.integers(1, pages * 64 + 1, rows).astype(np.int32)
    lens[0] = pages * 64 - 13
    if rows > 2:
        lens[1], lens[2] = 0, 70
    idx = np.full((rows, n), -1, np.int32)
    for r in range(rows):
        nb = -(-int(lens[r]) // 64)
        k = min(n, nb)
        # ascending, the last (partial) block among them
        c = np.sort(np.append(g.permutation(nb - 1)[:k - 1], nb - 1)) if k else np.zeros(0, np.int32)
        idx[r, :k] = c
    q = _q(rows, heads, 5)
    out, lse = hcu.block_sparse_mla_attention(q.to(dev), torch.from_numpy(pool).to(dev).view(-1, 1, SLOT[fmt]),
                                              torch.from_numpy(idx).to(dev), torch.from_numpy(table).to(dev),
                                              torch.from_numpy(lens).to(dev), SCALE)
    some = range(rows) if rows <= 6 else range(0, rows, 23)
    _check(fmt, q[list(some)], pool, [O.block_slots(idx[r], table[r], lens[r]) for r in some], out[list(some)],
           lse[list(some)])


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_every_token_counts_once(hcu, dev, fmt):
    """q = 0: all weights equal, so lse = log n to fp32 precision and out is the mean."""
    pool = _pool(fmt, 5000, 6)
    for n in (1, 2, 31, 64, 100, 127, 128, 129, 1023, 2048, 4097):
        idx = np.random.default_rng(n).permutation(5000)[:n].astype(np.int32)[None]
        q = torch.zeros(1, 64, 576, dtype=torch.bfloat16)
        out, lse = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(pool).to(dev), torch.from_numpy(idx).to(dev), SCALE)
        assert np.allclose(lse.cpu().numpy(), np.log(n), rtol=2e-6, atol=2e-6), n
        _check(fmt, q, pool, [idx[0]], out, lse)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_sharp_softmax_follows_one_token(hcu, dev, fmt):
    """A query aligned with one token by a wide margin returns that token's latent (bf16 rounding only), wherever
    the token stands in the list and however far the running maximum climbs before it."""
    pool = _pool(fmt, 700, 8)
    g = np.random.default_rng(0)
    idx = g.permutation(700)[:515].astype(np.int32)
    k = _values(fmt, pool, idx)
    rows = [0, 1, 63, 64, 200, 257, 511, 514]
    # s = q.k* grows with |k*|^2; climb: earlier tokens scaled copies are met on the way
    q = torch.from_numpy(np.stack([np.stack([k[t] * 40.0 / np.linalg.norm(k[t])] * 64) for t in rows])).bfloat16()
    out, lse = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(pool).to(dev),
                                        torch.from_numpy(np.tile(idx, (len(rows), 1))).to(dev), 4.0)
    _check(fmt, q, pool, [idx] * len(rows), out, lse, scale=4.0)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
@pytest.mark.parametrize("gain", [2.0 ** -60, 2.0 ** -14, 2.0 ** 10, 2.0 ** 40])
def test_query_magnitudes(hcu, dev, fmt, gain):
    """Queries far outside f16's range, the scale compensating."""
    pool = _pool(fmt, 400, 9)
    idx = np.arange(200, dtype=np.int32)[None].repeat(2, 0)
    q = _q(2, 64, 3, gain)
    out, lse = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(pool).to(dev), torch.from_numpy(idx).to(dev),
                                        SCALE / gain)
    _check(fmt, q, pool, [idx[0], idx[1]], out, lse, scale=SCALE / gain)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_cache_magnitudes(hcu, dev, fmt):
    """Latents from 2^-30 to 2^30 beside ropes of order 1, zero latents, zero ropes, in one list."""
    g = torch.Generator().manual_seed(12)
    n = 320
    lat = torch.randn(n, 512, generator=g)
    mag = torch.zeros(n)
    mag[:40], mag[40:80], mag[80:90] = -30, 12, 30
    lat = (lat * torch.exp2(mag)[:, None])
    lat[100:110] = 0
    rope = torch.randn(n, 64, generator=g)
    rope[105:120] = 0
    rope[120:125] *= 2.0 ** 14
    lat, rope = lat.bfloat16(), rope.bfloat16()
    u = lambda t: t.contiguous().view(torch.int16).numpy().view(np.uint16)
    if fmt == "kv4":
        pool = O.kv4_pack(u(lat), u(rope))
    else:
        x = lat.float().view(n, 4, 128)
        sc = (x.abs().amax(-1).clamp_min(1e-6) / 448).float()
        q8 = (x / sc[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(n, 512).view(torch.uint8).numpy()
        pool = np.concatenate([q8, sc.contiguous().view(torch.uint8).numpy().reshape(n, 16),
                               u(rope).view(np.uint8).reshape(n, 128)], 1)
    P = torch.from_numpy(pool).to(dev)
    for a, b in ((0, 40), (40, 80), (80, 90), (90, 320), (0, 80), (100, 110)):
        idx = np.arange(a, b, dtype=np.int32)[None]
        q = _q(1, 64, a)
        # keep the scores of large latents within a softmax's reach
        scale = SCALE * 2.0 ** -float(max(mag[a:b].max(), 0)) * (2.0 ** -14 if a <= 120 < b else 1)
        out, lse = hcu.sparse_mla_attention(q.to(dev), P, torch.from_numpy(idx).to(dev), scale)
        _check(fmt, q, pool, [idx[0]], out, lse, scale=scale)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_strides_and_views(hcu, dev, fmt):
    """q as the front end's view (rows and heads strided), a padded slot stride, strided index rows."""
    stride = 672 if fmt == "fp8" else 448
    pool = _pool(fmt, 1000, 4, stride)
    P = torch.from_numpy(pool).to(dev)[:, :SLOT[fmt]].unsqueeze(1)
    idx = np.random.default_rng(3).integers(0, 1000, (6, 150)).astype(np.int32)
    I = torch.full((6, 201), 123456789, dtype=torch.int32, device=dev)
    I[:, 7:157] = torch.from_numpy(idx).to(dev)
    q = _q(6, 24, 1)
    Q = torch.full((6, 30, 640), float("nan"), dtype=torch.bfloat16, device=dev)
    Q[:, 3:27, 8:584] = q.to(dev)
    out, lse = hcu.sparse_mla_attention(Q[:, 3:27, 8:584], P, I[:, 7:157], SCALE)
    _check(fmt, q, pool, list(idx), out, lse)
    # the rows of one query broadcast
    q1 = _q(1, 24, 9)
    out, lse = hcu.sparse_mla_attention(q1.to(dev).expand(6, 24, 576), P, I[:, 7:157], SCALE)
    _check(fmt, q1.expand(6, 24, 576), pool, list(idx), out, lse)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_poisoned_slots_outside_the_list(hcu, dev, fmt):
    """NaN and inf everywhere but in the selected slots, the tail of the last block included."""
    pool = _pool(fmt, 640, 2)
    keep = np.arange(128, 300)
    bad = np.setdiff1d(np.arange(640), keep)
    pool[bad] = 0xFF  # NaN codes, NaN scales, NaN ropes
    q = _q(2, 64, 2)
    idx = np.full((2, 200), -1, np.int32)
    idx[:, 5:5 + 172] = keep
    P = torch.from_numpy(pool).to(dev)
    out, lse = hcu.sparse_mla_attention(q.to(dev), P, torch.from_numpy(idx).to(dev), SCALE)
    _check(fmt, q, pool, [keep, keep], out, lse)
    table = np.array([[2, 3, 4]] * 2, np.int32)
    out, lse = hcu.block_sparse_mla_attention(q.to(dev), P, torch.tensor([[0, 1, 2, -1]] * 2, dtype=torch.int32, device=dev),
                                              torch.from_numpy(table).to(dev),
                                              torch.tensor([172, 100], dtype=torch.int32, device=dev), SCALE)
    _check(fmt, q, pool, [keep, keep[:100]], out, lse)


def test_offsets_past_32_bits(hcu, dev):
    """A cache of more than 2^32 bytes, rows at both ends."""
    slots = 7_000_000
    P = torch.empty(slots, 1, 656, dtype=torch.uint8, device=dev)
    base = _pool("fp8", 256, 5)
    where = np.concatenate([np.arange(64), np.arange(3_300_000, 3_300_064), np.arange(slots - 128, slots)])
    P[torch.from_numpy(where).to(dev), 0] = torch.from_numpy(base).to(dev)
    q = _q(1, 64, 4)
    out, lse = hcu.sparse_mla_attention(q.to(dev), P, torch.from_numpy(where.astype(np.int32))[None].to(dev), SCALE)
    _check("fp8", q, base, [np.arange(256)], out, lse)


@pytest.mark.parametrize("rows,n", [(1, 2048), (7, 500), (150, 130)])
def test_repeats_are_identical_and_graphs_replay(hcu, dev, rows, n):
    pool = _pool("fp8", 3000, 1)
    P = torch.from_numpy(pool).to(dev)
    idx = np.random.default_rng(n).integers(0, 3000, (rows, n)).astype(np.int32)
    q = _q(rows, 64, 2)
    Q, I = q.to(dev), torch.from_numpy(idx).to(dev)
    a = hcu.sparse_mla_attention(Q, P, I, SCALE)
    for _ in range(3):
        b = hcu.sparse_mla_attention(Q, P, I, SCALE)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = hcu.sparse_mla_attention(Q, P, I, SCALE)
    q2 = _q(rows, 64, 33)
    Q.copy_(q2.to(dev))
    idx2 = np.random.default_rng(n + 1).integers(-1, 3000, (rows, n)).astype(np.int32)
    I.copy_(torch.from_numpy(idx2))
    g.replay()
    some = list(range(min(rows, 4)))
    _check("fp8", q2[some], pool, [idx2[r][idx2[r] >= 0] for r in some], c[0][some], c[1][some])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d = hcu.sparse_mla_attention(Q, P, I, SCALE)
    side.synchronize()
    assert torch.equal(c[0], d[0]) and torch.equal(c[1], d[1])


def test_bad_slots_and_blocks_are_skipped_and_flagged(hcu, dev, request):
    request.node.allowed_status = 2
    pool = _pool("fp8", 640, 1)
    P = torch.from_numpy(pool).to(dev)
    q = _q(1, 64, 1)
    idx = np.array([[3, 640, 5, 2 ** 30, 7]], np.int32)
    out, lse = hcu.sparse_mla_attention(q.to(dev), P, torch.from_numpy(idx).to(dev), SCALE)
    assert hcu.read_device_status(clear=True) & 2
    _check("fp8", q, pool, [[3, 5, 7]], out, lse)
    table = torch.tensor([[1, 10, -1]], dtype=torch.int32, device=dev)  # page 10 lies outside, page -1 is none
    out, lse = hcu.block_sparse_mla_attention(q.to(dev), P, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=dev),
                                              table, torch.tensor([250], dtype=torch.int32, device=dev), SCALE)
    assert hcu.read_device_status(clear=True) & 2
    _check("fp8", q, pool, [np.arange(64, 128)], out, lse)


def test_empty_calls_and_refusals(hcu, dev):
    P = torch.from_numpy(_pool("fp8", 64, 1)).to(dev)
    q = _q(2, 8, 1).to(dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    out, lse = hcu.sparse_mla_attention(q, P, i32(2, 0), SCALE)
    assert (out == 0).all() and torch.isneginf(lse).all()
    out, lse = hcu.sparse_mla_attention(q[:0], P, i32(0, 5), SCALE)
    assert out.shape == (0, 8, 512) and lse.shape == (0, 8)
    for a in ((q.half(), P, i32(2, 4)), (q[..., :512], P, i32(2, 4)), (q, P[:, :640], i32(2, 4)), (q, P, i32(3, 4)),
              (q, P, i32(2, 4).long()), (q, P, i32(4, 2).t()), (q, P.cpu(), i32(2, 4)),
              (torch.zeros(2, 8, 577, dtype=torch.bfloat16, device=dev)[..., 1:], P, i32(2, 4))):
        with pytest.raises(RuntimeError):
            hcu.sparse_mla_attention(*a, SCALE)
    for t, l in ((i32(3, 4), i32(2)), (i32(2, 4), i32(3)), (i32(2, 4).long(), i32(2))):
        with pytest.raises(RuntimeError):
            hcu.block_sparse_mla_attention(q, P, i32(2, 4), t, l, SCALE)


@pytest.mark.parametrize("n", [1, 64])
def test_table_without_pages_is_still_the_block_form(hcu, dev, n):
    """A block table of width 0 holds no block: entries below the row's length are flagged, none is a slot."""
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    q = torch.randn(2, 16, 576, generator=g, device=dev).bfloat16()
    kv = torch.zeros(128, 1, 432, dtype=torch.uint8, device=dev)
    table = torch.empty(2, 0, dtype=torch.int32, device=dev)
    blocks = torch.zeros(2, n, dtype=torch.int32, device=dev)
    hcu.read_device_status()
    out, lse = hcu.block_sparse_mla_attention(q, kv, blocks, table, torch.full((2,), 64, dtype=torch.int32, device=dev), 0.1)
    assert (out == 0).all() and (lse == float("-inf")).all()
    assert hcu.read_device_status() == 2
    out, lse = hcu.block_sparse_mla_attention(q, kv, blocks, table, torch.zeros(2, dtype=torch.int32, device=dev), 0.1)
    assert (lse == float("-inf")).all() and hcu.read_device_status() == 0


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_many_rows_repeat_bit_for_bit(hcu, dev, fmt):
    """Every SM busy over many tiles: the tile buffers' hand-overs under load.  No atomics, so runs are equal."""
    rows, pool = 2048, 16384
    g = torch.Generator(device=dev)
    g.manual_seed(11)
    host = _pool(fmt, pool, 11)
    kv = torch.from_numpy(host).to(dev)
    q = torch.randn(rows, 64, 576, generator=g, device=dev).bfloat16()
    idx = torch.randint(0, pool, (rows, 2048), generator=g, device=dev, dtype=torch.int32)
    out, lse = hcu.sparse_mla_attention(q, kv, idx, SCALE)
    for _ in range(8):
        o, z = hcu.sparse_mla_attention(q, kv, idx, SCALE)
        assert torch.equal(o, out) and torch.equal(z, lse)
    some = list(range(0, rows, 97))
    lists = idx[some].cpu().numpy()
    _check(fmt, q[some].cpu(), host, list(lists), out[some], lse[some])


@pytest.mark.parametrize("form", ["tokens", "blocks"])
@pytest.mark.parametrize("n", [1, 33, 96, 97, 200, 500])
def test_lse_of_short_fp8_rows(hcu, dev, form, n):
    """lse of few tokens, whose scores' errors do not average out.  Per head: the rope is the one operand that is
    rounded, to 11 bits (2^-12 of |q k| each); 2^-17 of all |q k| and 2e-6 for the fp32 sums and exponentials.
    From 33 tokens on 2e-5 of itself (2-norm) as well."""
    pool = _pool("fp8", 1024, 21)
    rng = np.random.default_rng(n)
    q = _q(24, 64, 22)
    P, Q = torch.from_numpy(pool).to(dev), q.to(dev)
    if form == "tokens":
        lists = [rng.permutation(1024)[:n] for _ in range(24)]
        _, lse = hcu.sparse_mla_attention(Q, P, torch.from_numpy(np.stack(lists).astype(np.int32)).to(dev), SCALE)
    else:
        nb = -(-n // 64)
        table = np.stack([rng.permutation(16)[:nb] for _ in range(24)]).astype(np.int32)
        lists = [(table[r].astype(np.int64)[:, None] * 64 + np.arange(64)).reshape(-1)[:n] for r in range(24)]
        blocks = np.tile(np.arange(nb, dtype=np.int32), (24, 1))
        _, lse = hcu.block_sparse_mla_attention(Q, P, torch.from_numpy(blocks).to(dev), torch.from_numpy(table).to(dev),
                                                torch.full((24,), n, dtype=torch.int32, device=dev), SCALE)
    z, qd = lse.double().cpu().numpy(), q.double().numpy()
    ref, tol = [], []
    for r in range(24):
        v = _values("fp8", pool, lists[r])
        s = qd[r] @ v.T * SCALE
        every = np.abs(qd[r]) @ np.abs(v).T * SCALE
        rope = np.abs(qd[r][:, 512:]) @ np.abs(v[:, 512:]).T * SCALE
        tol.append((2.0 ** -12 * rope + 2.0 ** -17 * every).max(1) + 2e-6)
        m = s.max(1, keepdims=True)
        ref.append(m[:, 0] + np.log(np.exp(s - m).sum(1)))
    ref = np.stack(ref)
    assert (np.abs(z - ref) <= np.stack(tol)).all()
    assert n < 33 or np.linalg.norm(z - ref) <= 2e-5 * np.linalg.norm(ref)
