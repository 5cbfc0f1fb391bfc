"""The example decode step (examples/sparse_decode.py) as an MLA step: the latent normed, ropes rotated in both slot
formats; the step repeats itself, eager and in a graph; the new token takes part with its own weight."""
import numpy as np
import pytest
import torch

from oracle import mla as M
from oracle import sparse as O
from test_gpu_sparse_step import example  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def _u16(t):
    return t.contiguous().cpu().view(torch.int16).numpy().view(np.uint16)


@pytest.mark.parametrize("slots", ["fp8", "kv4"])
def test_latent_is_normed_and_ropes_are_rotated(hcu, dev, example, slots):  # noqa: F811
    st = example.make_state(3, 700, 2, slots)
    t, *_ = example.decode_step(st, "tokens")
    q, kv, pe = (_u16(st[k + "_in"]) for k in ("q_cat", "kv_c", "k_pe"))
    qr, kvr, per, _ = M.rope_qout_kv_store(t.positions.cpu().numpy(), q[..., 512:], kv, _u16(st["kv_weight"]), 1e-6, pe,
                                           _u16(st["cos_sin"]), False, np.zeros((1, 656), np.uint8), np.zeros(0, np.int64))
    got_q = _u16(st["q_cat"])
    assert np.array_equal(got_q[..., 512:], qr.reshape(got_q[..., 512:].shape))
    assert np.array_equal(got_q[..., :512], q[..., :512])
    assert not np.array_equal(qr.reshape(-1), q[..., 512:].reshape(-1))
    normed = _u16(st["kv_c"])
    assert np.abs(normed.astype(np.int32) - kvr.astype(np.int32)).max() <= 1  # rsqrtf: one bf16 step
    rows = st["kv"].cpu().numpy().reshape(st["kv"].shape[0], -1)[t.loc.cpu().numpy()]
    at = 528 if slots == "fp8" else 304
    assert np.array_equal(np.ascontiguousarray(rows[:, at:at + 128]).view(np.uint16), per.reshape(-1, 64))
    if slots == "kv4":
        want = O.kv4_values(O.kv4_pack(normed, per.reshape(-1, 64)))
        assert np.array_equal(O.kv4_values(rows), want)


@pytest.mark.parametrize("slots", ["fp8", "kv4"])
@pytest.mark.parametrize("form", ["tokens", "blocks"])
def test_step_repeats_itself(hcu, dev, example, slots, form):  # noqa: F811
    st = example.make_state(2, 3000, 2, slots)
    _, sel, out, lse = (x.clone() if torch.is_tensor(x) else x for x in example.decode_step(st, form))
    for _ in range(2):
        _, sel2, out2, lse2 = example.decode_step(st, form)
        assert torch.equal(sel, sel2) and torch.equal(out, out2) and torch.equal(lse, lse2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, sel2, out2, lse2 = example.decode_step(st, form)
    for _ in range(3):
        g.replay()
        assert torch.equal(sel, sel2) and torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("slots", ["fp8", "kv4"])
def test_new_token_has_its_own_weight(hcu, dev, example, slots):  # noqa: F811
    """exp(lse) with the new token less exp(lse) without it is its own exp(score), within the bound of the two lse."""
    st = example.make_state(1, 100, 1, slots)
    t, sel, _, lse = example.decode_step(st, "tokens")
    less = sel.clone()
    assert sel[0, 100].item() == t.loc[0].item()
    less[0, 100] = -1
    _, without = hcu.sparse_mla_attention(st["q_cat"], st["kv"], less, example.SM_SCALE)
    kv = st["kv"].cpu().numpy().reshape(st["kv"].shape[0], -1)
    values = O.fp8_values if slots == "fp8" else O.kv4_values
    q = st["q_cat"].double().cpu().numpy()[0]
    s = example.SM_SCALE * (q @ values(kv[[t.loc[0].item()]])[0])
    a, b = lse.double().cpu().numpy()[0], without.double().cpu().numpy()[0]
    # each lse within 2^-12 of the ropes' |q k| and 2^-17 of every |q k|
    k = np.abs(values(kv[sel[0, :101].cpu().numpy()]))
    d = (2.0 ** -12 * (np.abs(q[:, 512:]) @ k[:, 512:].T) + 2.0 ** -17 * (np.abs(q) @ k.T)).max(1) * example.SM_SCALE + 2e-6
    assert (np.abs((np.exp(a) - np.exp(b)) - np.exp(s)) <= np.expm1(d) * (np.exp(a) + np.exp(b))).all()
    assert (np.exp(s) > 10 * np.expm1(d) * (np.exp(a) + np.exp(b))).any()  # a head where dropping it would show
