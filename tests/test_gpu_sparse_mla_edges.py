"""Edges of sparse_mla_attention / block_sparse_mla_attention: lists that end in whole tiles of padding,
non-finite values and zero bytes in selected slots; and bounds tight enough to see a factor left out of one 128-value
group."""
import numpy as np
import pytest
import torch

from oracle import sparse as O
from test_gpu_sparse_mla import SCALE, SLOT, _check, _pool, _q, _values

pytestmark = pytest.mark.gpu

TILE = 48  # candidates per tile of the kernel


def _short_lists(rows, tiles, empty, pool, seed):
    """int32 [rows, TILE * tiles]: random slots, the last `empty` tiles of every row and a few entries before them -1."""
    g = np.random.default_rng(seed)
    idx = g.integers(0, pool, (rows, TILE * tiles)).astype(np.int32)
    valid = TILE * (tiles - empty) - g.integers(0, TILE, rows)
    valid[::3] = TILE * (tiles - empty)  # a full last tile
    idx[np.arange(TILE * tiles)[None] >= valid[:, None]] = -1
    return idx


@pytest.mark.parametrize("empty", [1, 2, 3])
@pytest.mark.parametrize("heads", [64, 16])
@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_whole_rows_that_end_in_empty_tiles(hcu, dev, fmt, heads, empty):
    """Rows handled whole by one CTA: the result is bit for bit that of the list cut before the empty tiles, as
    the tiles that hold tokens are the same.  Every SM has several rows, and every run gives the same bits."""
    rows, tiles = 4 * torch.cuda.get_device_properties(dev).multi_processor_count, 7
    host = _pool(fmt, 4000, 31)
    P, q = torch.from_numpy(host).to(dev), _q(rows, heads, 32)
    Q, idx = q.to(dev), _short_lists(rows, tiles, empty, 4000, 33 + empty)
    full = torch.from_numpy(idx).to(dev)
    cut = torch.from_numpy(np.ascontiguousarray(idx[:, :TILE * (tiles - empty)])).to(dev)
    out, lse = hcu.sparse_mla_attention(Q, P, cut, SCALE)
    some = list(range(0, rows, 83))
    _check(fmt, q[some], host, [idx[r][idx[r] >= 0] for r in some], out[some], lse[some])
    for _ in range(20):
        o, z = hcu.sparse_mla_attention(Q, P, full, SCALE)
        assert torch.equal(o, out) and torch.equal(z, lse)


@pytest.mark.parametrize("empty", [1, 2, 13])
@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_split_rows_that_end_in_empty_tiles(hcu, dev, fmt, empty):
    """Rows shared by several CTAs, whose shares end in empty tiles or hold nothing else."""
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    for rows, tiles in ((sms * 2 // 3, 40), (1, 43)):
        host = _pool(fmt, 4000, 41)
        P, q = torch.from_numpy(host).to(dev), _q(rows, 64, 42)
        Q, idx = q.to(dev), _short_lists(rows, tiles, empty, 4000, 43 + empty)
        full = torch.from_numpy(idx).to(dev)
        out, lse = hcu.sparse_mla_attention(Q, P, full, SCALE)
        for _ in range(20):
            o, z = hcu.sparse_mla_attention(Q, P, full, SCALE)
            assert torch.equal(o, out) and torch.equal(z, lse)
        some = list(range(0, rows, 7))
        _check(fmt, q[some], host, [idx[r][idx[r] >= 0] for r in some], out[some], lse[some])


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_short_block_rows_end_in_empty_tiles(hcu, dev, fmt):
    """Block form, rows shorter than the selection: visible tokens end one to three tiles before the list's end."""
    rows, nb = 2 * torch.cuda.get_device_properties(dev).multi_processor_count, 6
    host = _pool(fmt, 64 * 50, 51)
    P, q = torch.from_numpy(host).to(dev), _q(rows, 64, 52)
    g = np.random.default_rng(53)
    table = np.stack([g.permutation(50)[:nb] for _ in range(rows)]).astype(np.int32)
    lens = (64 * nb - TILE * g.integers(1, 4, rows) - g.integers(0, TILE, rows) * (np.arange(rows) % 2)).astype(np.int32)
    blocks = np.tile(np.arange(nb, dtype=np.int32), (rows, 1))
    args = [torch.from_numpy(x).to(dev) for x in (blocks, table, lens)]
    out, lse = hcu.block_sparse_mla_attention(q.to(dev), P, *args, SCALE)
    for _ in range(20):
        o, z = hcu.block_sparse_mla_attention(q.to(dev), P, *args, SCALE)
        assert torch.equal(o, out) and torch.equal(z, lse)
    some = list(range(0, rows, 17))
    lists = [(table[r].astype(np.int64)[:, None] * 64 + np.arange(64)).reshape(-1)[:lens[r]] for r in some]
    _check(fmt, q[some], host, lists, out[some], lse[some])


def _poison(fmt, slot, kind):
    """Puts a non-finite value into one slot (uint8 [slot bytes]) in place."""
    nan, inf = np.float32(np.nan), np.float32(np.inf)
    put = lambda at, v: slot.__setitem__(slice(at, at + v.nbytes), np.frombuffer(v.tobytes(), np.uint8))
    if kind == "rope":
        put((304 if fmt == "kv4" else 528) + 14, np.uint16(0x7FC0))
    elif fmt == "fp8":
        if kind == "code":
            slot[300] = 0x7F
        else:
            put(512 + 4 * int(kind[-1]), nan if kind.startswith("nan") else inf)
    elif kind == "code":
        slot[256 + 9] = 0x7F  # a group's scale
    else:
        put(288, nan if kind.startswith("nan") else inf)


@pytest.mark.parametrize("fmt,kind", [("fp8", k) for k in ("nan0", "nan1", "nan2", "nan3", "inf0", "inf3", "code", "rope")] +
                         [("kv4", k) for k in ("nan", "inf", "code", "rope")])
def test_non_finite_slots_are_seen(hcu, dev, fmt, kind):
    """A NaN or infinity in a selected slot makes the row's out and lse NaN, as the definition does; rows that do
    not select the slot keep their bits."""
    host = _pool(fmt, 1000, 61)
    q = _q(12, 64, 62)
    g = np.random.default_rng(63)
    idx = g.integers(1, 1000, (12, 200)).astype(np.int32)
    idx[4, 150:] = -1
    clean = torch.from_numpy(host.copy()).to(dev)
    _poison(fmt, host[0], kind)
    P, Q = torch.from_numpy(host).to(dev), q.to(dev)
    want, lse0 = hcu.sparse_mla_attention(Q, clean, torch.from_numpy(idx).to(dev), SCALE)
    idx[2, 0] = idx[4, 149] = idx[7, 77] = idx[11, 199] = 0
    out, lse = hcu.sparse_mla_attention(Q, P, torch.from_numpy(idx).to(dev), SCALE)
    bad = [2, 4, 7, 11]
    rest = [r for r in range(12) if r not in bad]
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(out[rest], want[rest]) and torch.equal(lse[rest], lse0[rest])


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_infinite_rope(hcu, dev, fmt):
    """An infinite rope element scores +inf in heads whose query element is positive, which gives NaN, and -inf where it
    is negative: there the slot has no weight, and the result is that of the list without it."""
    host = _pool(fmt, 300, 68)
    at = (304 if fmt == "kv4" else 528) + 14
    host[0, at:at + 2] = np.frombuffer(np.uint16(0x7F80).tobytes(), np.uint8)
    q = _q(3, 64, 69)
    idx = np.random.default_rng(70).integers(1, 300, (3, 130)).astype(np.int32)
    idx[:, 60] = 0
    out, lse = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(host).to(dev), torch.from_numpy(idx).to(dev), SCALE)
    for r in range(3):
        up = q[r, :, 512 + 7] > 0
        assert torch.isnan(out[r, up.to(dev)]).all() and torch.isnan(lse[r, up.to(dev)]).all()
        rest = (~up).to(dev)
        _check(fmt, q[r:r + 1, ~up], host, [idx[r][idx[r] > 0]], out[r:r + 1, rest], lse[r:r + 1, rest])


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_non_finite_slot_in_a_row_of_one_part(hcu, dev, fmt):
    """A row split over many CTAs all of whose tokens lie in one share: the join keeps that share's NaN though every
    other share is empty."""
    host = _pool(fmt, 100, 64)
    _poison(fmt, host[0], "code")
    idx = np.full((1, 2048), -1, np.int32)
    idx[0, 5] = 0
    q = _q(1, 64, 65).to(dev)
    out, lse = hcu.sparse_mla_attention(q, torch.from_numpy(host).to(dev), torch.from_numpy(idx).to(dev), SCALE)
    assert torch.isnan(out).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_long_lists_of_zero_slots(hcu, dev, fmt):
    """More than 2^20 slots of zero bytes per row (a cache that has not been written): every score is 0, so lse is
    log n and out 0."""
    rows, n = torch.cuda.get_device_properties(dev).multi_processor_count, 16400
    kv = torch.zeros(64, 1, SLOT[fmt], dtype=torch.uint8, device=dev)
    table = torch.zeros(1, n, dtype=torch.int32, device=dev).expand(rows, n)
    blocks = torch.arange(n, dtype=torch.int32, device=dev).expand(rows, n)
    lens = torch.full((rows,), 64 * n, dtype=torch.int32, device=dev)
    out, lse = hcu.block_sparse_mla_attention(_q(rows, 8, 3).to(dev), kv, blocks, table, lens, SCALE)
    assert (out == 0).all()
    assert np.allclose(lse.cpu().numpy(), np.log(64.0 * n), rtol=2e-6)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_zero_slots_beside_large_latents(hcu, dev, fmt):
    """Slots of zero bytes in a list with latents of order 2^48, whose scores the scale brings to order 1: the zero
    slots' score of 0 has its full weight."""
    host = _pool(fmt, 200, 66)
    host[::2] = 0
    f32 = lambda at, n: np.ascontiguousarray(host[1::2, at:at + 4 * n]).view(np.float32)
    at, n = (512, 4) if fmt == "fp8" else (288, 1)
    host[1::2, at:at + 4 * n] = (f32(at, n) * np.float32(2.0 ** 48)).view(np.uint8)
    idx = np.arange(200, dtype=np.int32)[None]
    q = _q(1, 64, 67)
    out, lse = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(host).to(dev), torch.from_numpy(idx).to(dev),
                                        SCALE * 2.0 ** -48)
    _check(fmt, q, host, [idx[0]], out, lse, scale=SCALE * 2.0 ** -48)


def test_empty_cache(hcu, dev):
    """A cache without slots: a list of -1 gives the empty row, any other entry is skipped and flagged."""
    for w in (656, 432):
        kv = torch.empty(0, 1, w, dtype=torch.uint8, device=dev)
        q = _q(2, 8, 1).to(dev)
        out, lse = hcu.sparse_mla_attention(q, kv, torch.full((2, 50), -1, dtype=torch.int32, device=dev), SCALE)
        assert (out == 0).all() and torch.isneginf(lse).all() and hcu.read_device_status() == 0


def _bf16_step(x):
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 1e-30))) - 7)


@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_one_token_rows_give_the_token(hcu, dev, fmt):
    """A row of one token returns its latent.  Its one weight is exact but for P's rounding to f16 (2^-11 at most,
    with an fp8 group's remainder, up to 2^-7, in it), and the result is rounded to bf16 (half a step).  A
    remainder left out of any one group breaks the bound at some of the 96 tokens."""
    host = _pool(fmt, 96, 71)
    q = _q(96, 64, 72)
    idx = torch.arange(96, dtype=torch.int32, device=dev).view(96, 1)
    out, _ = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(host).to(dev), idx, SCALE)
    o = out.double().cpu().numpy()
    v = _values(fmt, host, np.arange(96))[:, None, :512]
    assert (np.abs(o - v) <= 0.5 * _bf16_step(v) * 1.02 + (2.0 ** -11 + 2.0 ** -16) * np.abs(v)).all()


@pytest.mark.parametrize("n", [33, 200, 2048])
@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_out_of_each_group(hcu, dev, fmt, n):
    """2-norm of out's error over all heads, per row and 128-value group, relative to out's own.  The rounding to bf16
    is 2^-7 / sqrt(12) at most where all values are just above a power of two; weights are off by 2^-11 (P in f16) and
    by their scores' errors, for which six deviations (2^-11 / sqrt(3) of each of 64 rope products, 1/16 x 8 in all)
    are allowed.  The two are independent."""
    host = _pool(fmt, 4096, 81)
    g = np.random.default_rng(82 + n)
    idx = np.stack([g.permutation(4096)[:n] for _ in range(12)]).astype(np.int32)
    q = _q(12, 64, 83)
    out, _ = hcu.sparse_mla_attention(q.to(dev), torch.from_numpy(host).to(dev), torch.from_numpy(idx).to(dev), SCALE)
    o, qd = out.double().cpu().numpy(), q.double().numpy()
    bound = ((2.0 ** -7 / 12 ** 0.5) ** 2 + (2.0 ** -11 + 6 * 2.0 ** -11 / 3 ** 0.5 * 0.5) ** 2) ** 0.5
    for r in range(12):
        v = _values(fmt, host, idx[r])
        s = qd[r] @ v.T * SCALE
        w = np.exp(s - s.max(1, keepdims=True))
        ref = (w / w.sum(1, keepdims=True)) @ v[:, :512]
        for k in range(4):
            a, b = o[r][:, 128 * k:128 * k + 128], ref[:, 128 * k:128 * k + 128]
            assert np.linalg.norm(a - b) <= bound * np.linalg.norm(b), (r, k)


@pytest.mark.parametrize("form", ["tokens", "blocks"])
@pytest.mark.parametrize("n", [33, 50, 100, 200, 500, 2048])
@pytest.mark.parametrize("fmt", ["fp8", "kv4"])
def test_lse_is_that_of_32_bit_products(hcu, dev, fmt, n, form):
    """No operand of the scores is rounded by more than 2^-18 (a rope of an fp8 slot goes in as two f16 terms), so lse is
    off by what 40 steps of 32-bit accumulation leave, 2^-23 of the running sum each: for scores up to 8 about
    sqrt(40) 2^-23 8 = 6e-6 a score, over at least five tokens of weight 2.7e-6, of an lse of 4 or more 7e-7.  1e-6 of
    itself is allowed (2-norm)."""
    rows, heads = 24, 64
    g = torch.Generator().manual_seed(91)
    lat, rope = torch.randn(2048, 512, generator=g).bfloat16(), torch.randn(2048, 64, generator=g).bfloat16()
    u = lambda t: t.contiguous().view(torch.int16).numpy().view(np.uint16)
    if fmt == "kv4":
        host = O.kv4_pack(u(lat), u(rope))
    else:
        x = lat.float().view(2048, 4, 128)
        sc = (x.abs().amax(-1) / 448).float()
        codes = (x / sc[..., None]).to(torch.float8_e4m3fn).view(2048, 512).view(torch.uint8).numpy()
        host = np.concatenate([codes, sc.contiguous().view(torch.uint8).numpy().reshape(2048, 16),
                               u(rope).view(np.uint8).reshape(2048, 128)], 1)
    rng = np.random.default_rng(92 + n)
    q = _q(rows, heads, 93)
    P, Q = torch.from_numpy(host).to(dev), q.to(dev)
    if form == "tokens":
        lists = [rng.permutation(2048)[:n] for _ in range(rows)]
        _, lse = hcu.sparse_mla_attention(Q, P, torch.from_numpy(np.stack(lists).astype(np.int32)).to(dev), SCALE)
    else:
        nb = -(-n // 64)
        table = np.stack([rng.permutation(32)[:nb] for _ in range(rows)]).astype(np.int32)
        lists = [(table[r].astype(np.int64)[:, None] * 64 + np.arange(64)).reshape(-1)[:n] for r in range(rows)]
        blocks = np.tile(np.arange(nb, dtype=np.int32), (rows, 1))
        _, lse = hcu.block_sparse_mla_attention(Q, P, torch.from_numpy(blocks).to(dev), torch.from_numpy(table).to(dev),
                                                torch.full((rows,), n, dtype=torch.int32, device=dev), SCALE)
    z, qd = lse.double().cpu().numpy(), q.double().numpy()
    ref = []
    for r in range(rows):
        s = qd[r] @ _values(fmt, host, lists[r]).T * SCALE
        m = s.max(1, keepdims=True)
        ref.append(m[:, 0] + np.log(np.exp(s - m).sum(1)))
    ref = np.stack(ref)
    assert np.linalg.norm(z - ref) <= 1e-6 * np.linalg.norm(ref)
