"""The example decode step (examples/sparse_decode.py): tables, cache writes, logits, selection and
attention run together, in both slot formats and both forms, each stage against its restatement on the
previous stage's own outputs, and a graph replay equal to the eager step."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import sparse as O

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang0.5.18-opt_b200", "examples",
                    "sparse_decode.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("sparse_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("slots", ["fp8", "kv4"])
@pytest.mark.parametrize("form", ["tokens", "blocks"])
@pytest.mark.parametrize("requests,context,new", [(3, 5000, 2), (1, 700, 1)])
def test_step(hcu, dev, example, slots, form, requests, context, new):
    st = example.make_state(requests, context, new, slots)
    rp = st["req_pages"].cpu().numpy().copy()
    t, sel, out, lse = example.decode_step(st, form)
    ref = O.step_tables(rp, np.arange(requests), [context] * requests, [new] * requests, st["free_pages"].cpu().numpy(), 0,
                        st["rows"], st["width"])
    for k in ("block_table", "page_table_size_1", "lengths", "positions", "loc"):
        assert np.array_equal(getattr(t, k).cpu().numpy(), ref[k]), k
    q = st["q_cat"].double().cpu().numpy()
    kv = st["kv"].cpu().numpy().reshape(st["kv"].shape[0], -1)
    o, z = out.double().cpu().numpy(), lse.double().cpu().numpy()
    s = sel.cpu().numpy()
    for r in range(st["rows"]):
        if form == "tokens":
            slot = s[r][s[r] >= 0]
            assert len(slot) == min(2048, ref["lengths"][r])
        else:
            assert (s[r] >= 0).sum() == min(32, -(-ref["lengths"][r] // 64))
            slot = O.block_slots(s[r], ref["block_table"][r], ref["lengths"][r])
        v = (O.fp8_values if slots == "fp8" else O.kv4_values)(kv[slot])
        ro, rl, to, tl = O.attend(q[r], v, example.SM_SCALE, 2.0 ** -11 if slots == "fp8" else 2.0 ** -14)
        assert (np.abs(o[r] - ro) <= to).all() and (np.abs(z[r] - rl) <= tl).all(), r


def test_new_token_is_seen_by_its_own_row(hcu, dev, example):
    """The newest token's latent, written in the step, takes part in the step's attention: with a context that
    fits the selection, dropping it changes the row's lse by its own weight."""
    st = example.make_state(1, 100, 1, "kv4")
    t, sel, out, lse = example.decode_step(st, "tokens")
    slot = sel[0, 100].item()
    assert slot == t.loc[0].item()
    kv = st["kv"].cpu().numpy().reshape(st["kv"].shape[0], -1)
    v = O.kv4_values(kv[[slot]])
    assert np.array_equal(v[0, 512:].astype(np.float32), st["k_pe"][0].float().cpu().numpy())


def test_graph_replay_equals_the_eager_step(hcu, dev, example):
    st = example.make_state(2, 3000, 2, "kv4")
    example.decode_step(st, "tokens")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, sel, out, lse = example.decode_step(st, "tokens")
    g.replay()
    torch.cuda.synchronize()
    keep = [x.clone() for x in (sel, out, lse)]
    _, sel2, out2, lse2 = example.decode_step(st, "tokens")
    assert torch.equal(keep[0], sel2) and torch.equal(keep[1], out2) and torch.equal(keep[2], lse2)


def test_every_request_takes_a_page(hcu, dev, example):
    """A context that ends on a page's edge: each request's new token opens a page from the free list."""
    st = example.make_state(5, 640, 1, "kv4")
    hcu.read_device_status()
    t, *_ = example.decode_step(st, "tokens")
    assert t.free_head.item() == 5 and hcu.read_device_status() == 0
    assert sorted(t.block_table[:, 10].tolist()) == sorted(st["free_pages"][:5].tolist())
