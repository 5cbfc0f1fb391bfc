"""GPU parity of the 4-bit MLA slot: the writer byte for byte against its CPU restatement (zeros may
carry either sign), the paged read exactly."""
import numpy as np
import pytest
import torch

from oracle import sparse as O

pytestmark = pytest.mark.gpu


def _latents(n, seed):
    """bf16 rows of every kind: normal, tiny, huge, zero, one outlier, values on the e2m1 midpoints of
    their group's scale."""
    g = np.random.default_rng(seed)
    x = g.standard_normal((n, 512)).astype(np.float32) * np.exp2(g.integers(-6, 7, (n, 1))).astype(np.float32)
    if n > 8:
        x[1] = 0
        x[2] *= np.float32(2.0 ** -120)
        x[3] *= np.float32(2.0 ** 110)
        x[4, 17] = 3e4
        x[5, :256] = 0
        mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)
        for r, m in ((6, 8), (7, 13), (8, 15)):  # group amax = 6 s with s of significand m / 8: codes tie exactly
            s = np.exp2(g.integers(-4, 1, 32)).astype(np.float32) * np.float32(m / 8)
            v = g.choice(mids, (32, 16)) * g.choice(np.array([-1, 1], np.float32), (32, 16))
            v[:, 0] = 6
            x[r] = (v * s[:, None]).reshape(-1)
    return torch.from_numpy(x).bfloat16()


def _u16(t):
    return t.contiguous().view(torch.int16).numpy().view(np.uint16)


def _canon(b):
    """Code bytes with the sign of zero codes cleared."""
    c = b.copy()
    lo, hi = c[:, :256] & 15, c[:, :256] >> 4
    c[:, :256] = np.where(lo == 8, 0, lo) | (np.where(hi == 8, 0, hi) << 4)
    return c


@pytest.mark.parametrize("n,packed,odd_rope", [(1, False, False), (9, True, False), (70, False, True), (1000, True, False)])
def test_store_and_read_back(hcu, dev, n, packed, odd_rope):
    lat = _latents(n, n)
    rope = torch.randn(n, 64, generator=torch.Generator().manual_seed(n)).bfloat16()
    slots = n + 50
    loc = torch.randperm(slots, generator=torch.Generator().manual_seed(1))[:n]
    if packed:  # views into one [T, 2048 + 576] latent, as the front end hands them over
        P = torch.zeros(n, 2624, dtype=torch.bfloat16)
        P[:, 2048:2560], P[:, 2560:] = lat, rope
        P = P.to(dev)
        kv_c, k_pe = P[:, 2048:2560], P[:, 2560:].unsqueeze(1)
    else:
        kv_c, k_pe = lat.to(dev), rope.to(dev)
    if odd_rope:  # rows that are not 16-byte aligned
        R = torch.zeros(n, 67, dtype=torch.bfloat16, device=dev)
        R[:, 3:] = rope.to(dev)
        k_pe = R[:, 3:]
    buf = torch.full((slots, 1, 448), 0xAB, dtype=torch.uint8, device=dev)
    kv = buf[..., :432]  # a longer slot stride
    hcu.store_mla_kv4(kv_c, k_pe, loc.to(dev), kv)
    b = buf.cpu().numpy().reshape(slots, 448)
    ref = O.kv4_pack(_u16(lat), _u16(rope))
    assert np.array_equal(_canon(b[loc.numpy()][:, :432]), ref)
    rest = np.setdiff1d(np.arange(slots), loc.numpy())
    assert (b[rest] == 0xAB).all() and (b[:, 432:] == 0xAB).all()
    got = hcu.dequantize_mla_kv4_paged(kv, loc.int().to(dev)).float().cpu().numpy().reshape(n, 576)
    assert np.array_equal(got.astype(np.float64), O.kv4_values(b[loc.numpy()]))


def test_e2m1_steps_of_the_result(hcu, dev):
    """Quality of the format: a group's largest error is half a step of its scale (2^-4 of e4m3 on top)."""
    lat = torch.randn(256, 512, generator=torch.Generator().manual_seed(4)).bfloat16()
    buf = torch.zeros(256, 1, 432, dtype=torch.uint8, device=dev)
    loc = torch.arange(256, device=dev)
    hcu.store_mla_kv4(lat.to(dev), torch.zeros(256, 64, dtype=torch.bfloat16, device=dev), loc, buf)
    got = hcu.dequantize_mla_kv4_paged(buf, loc.int()).float().cpu()[:, 0, :512].view(256, 32, 16)
    x = lat.float().view(256, 32, 16)
    amax = x.abs().amax(-1, keepdim=True)
    # the widest half step is 1 (4 to 6) of a scale amax / 6 (1 + 2^-4); a scale rounded down saturates by 6 * 2^-4
    assert ((got - x).abs() <= amax / 6 * (1 + 2.0 ** -4)).all()


def test_bad_slots_are_skipped_and_flagged(hcu, dev, request):
    request.node.allowed_status = 2
    lat, rope = _latents(4, 4).to(dev), torch.ones(4, 64, dtype=torch.bfloat16, device=dev)
    buf = torch.zeros(6, 1, 432, dtype=torch.uint8, device=dev)
    hcu.store_mla_kv4(lat, rope, torch.tensor([2, -1, 6], device=dev), buf)  # the fourth token is not stored
    assert hcu.read_device_status(clear=True) & 2
    assert (buf[2] != 0).any() and (buf[[0, 1, 3, 4, 5]] == 0).all()
    hcu.dequantize_mla_kv4_paged(buf, torch.tensor([6, 2], dtype=torch.int32, device=dev))
    assert hcu.read_device_status(clear=True) & 2


def test_refusals_and_empty(hcu, dev):
    bf = torch.bfloat16
    lat, rope = torch.zeros(2, 512, dtype=bf, device=dev), torch.zeros(2, 64, dtype=bf, device=dev)
    loc, buf = torch.zeros(1, dtype=torch.int64, device=dev), torch.zeros(4, 1, 432, dtype=torch.uint8, device=dev)
    hcu.store_mla_kv4(lat, rope, loc[:0], buf)
    assert hcu.dequantize_mla_kv4_paged(buf, loc[:0].int()).shape == (0, 1, 576)
    for a in ((lat.float(), rope, loc, buf), (lat[:, :510], rope, loc, buf), (lat, rope[:1], loc, buf),
              (lat, rope, loc.int(), buf), (lat, rope, torch.zeros(3, dtype=torch.int64, device=dev), buf),
              (lat, rope, loc, torch.zeros(4, 1, 656, dtype=torch.uint8, device=dev)),
              (torch.zeros(2, 513, dtype=bf, device=dev)[:, 1:], rope, loc, buf)):
        with pytest.raises(RuntimeError):
            hcu.store_mla_kv4(*a)
    with pytest.raises(RuntimeError):
        hcu.dequantize_mla_kv4_paged(buf, loc)
