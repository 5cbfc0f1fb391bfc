"""A decode step around the indexer, from the requests' lengths to the attention output.

    python sglang0.5.18-opt_b200/examples/sparse_decode.py [--requests 8] [--context 6000] [--slots fp8|kv4]

One layer's step for a batch of requests that bring one or two tokens each:

1. ``step_tables``: pages for the new tokens, block table, slot table, lengths, slots;
2. the new tokens' rows go into the caches: ``quant_store_index_k`` (indexer K), and the latent through
   ``rope_qout_kv_store``, which norms it, rotates its rope and the queries' and writes the 656-byte fp8 slot;
   for 432-byte 4-bit slots it is given no slot, and ``store_mla_kv4`` writes what it has normed and rotated;
3. ``mqa_logits`` scores the context;
4. token form: ``sparse_mask_topk_transform`` and ``sparse_mla_attention`` over the 2048 best tokens;
   block form: ``select_blocks`` and ``block_sparse_mla_attention`` over the 32 best 64-token blocks.

Everything is enqueued on the current stream without a read on the host, so the step can be captured in a
CUDA graph.  Weights, queries and caches are random; only the shapes are a model's.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hcu_ops  # noqa: E402

HEADS, LATENT, ROPE, INDEX_HEADS, INDEX_DIM = 64, 512, 64, 64, 128
SM_SCALE = 1.0 / 16.0  # 1 / sqrt(192 + 64)


def make_state(requests, context, new_tokens, slots, seed=0, device="cuda"):
    """Caches filled with `context` tokens per request and one step's activations."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    bf = torch.bfloat16

    def randn(*s):
        return torch.randn(*s, generator=g, device=device)

    width = (context + new_tokens + 63) // 64 * 64 + 64
    per = width // 64
    pages = requests * (per + (new_tokens + 63) // 64)  # no request takes more new pages in a step
    ids = torch.randperm(pages, generator=g, device=device).int()
    rows = requests * new_tokens
    st = dict(slots=slots, width=width, rows=rows, new_tokens=new_tokens,
              req_pages=ids[:requests * per].view(requests, per).contiguous(), free_pages=ids[requests * per:],
              free_head=torch.zeros(1, dtype=torch.int32, device=device),
              req_idx=torch.arange(requests, dtype=torch.int32, device=device),
              seq_lens=torch.full((requests,), context, dtype=torch.int32, device=device),
              new_lens=torch.full((requests,), new_tokens, dtype=torch.int32, device=device),
              cu=torch.arange(rows + 1, dtype=torch.int32, device=device))
    # caches: every slot of the pool filled through the framework's own writers
    every = torch.arange(pages * 64, device=device)
    st["index_cache"] = torch.zeros(pages, 64, 1, INDEX_DIM + 4, dtype=torch.uint8, device=device)
    hcu_ops.quant_store_index_k(randn(pages * 64, INDEX_DIM), every.int(), st["index_cache"])
    st["kv_weight"] = torch.ones(LATENT, dtype=bf, device=device)
    ang = torch.arange(width, device=device)[:, None] * (10000.0 ** (-torch.arange(32, device=device) / 32))
    st["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).to(bf).contiguous()
    st["kv"] = torch.zeros(pages * 64, 1, 656 if slots == "fp8" else 432, dtype=torch.uint8, device=device)
    for a in range(0, pages * 64, 8192):
        loc = every[a:a + 8192].contiguous()
        lat, pe = randn(loc.numel(), LATENT).to(bf), randn(loc.numel(), ROPE).to(bf)
        q_pe = torch.zeros(loc.numel(), 1, ROPE, dtype=bf, device=device)
        write_slots(st, torch.zeros(loc.numel(), dtype=torch.int32, device=device), lat, pe, q_pe, loc)
    # the step's activations, and the buffers that the front end norms and rotates in place
    st["kv_c_in"], st["k_pe_in"] = randn(rows, LATENT).to(bf), randn(rows, ROPE).to(bf)
    st["q_cat_in"] = randn(rows, HEADS, LATENT + ROPE).to(bf)
    for k in ("kv_c", "k_pe", "q_cat"):
        st[k] = torch.empty_like(st[k + "_in"])
    qi = randn(rows, INDEX_HEADS * INDEX_DIM)
    qs = qi.abs().amax(1) / 448
    st["index_q"] = (qi / qs[:, None]).to(torch.float8_e4m3fn).view(rows, 1, INDEX_HEADS, INDEX_DIM)
    st["index_w"] = (randn(rows, INDEX_HEADS) / 8 * qs[:, None]).contiguous()
    st["index_k"] = randn(rows, INDEX_DIM).to(bf)
    return st


def write_slots(st, positions, kv_c, k_pe, q_pe, loc):
    """Norms the latents, rotates k_pe and q_pe (all in place) and writes the latents' slots."""
    fp8 = st["slots"] == "fp8"
    # without slots (an empty loc) the front end writes none; its slot buffer is a stand-in then
    buf, where = (st["kv"], loc) if fp8 else (kv_c.new_empty(1, 1, 656, dtype=torch.uint8), loc[:0])
    hcu_ops.rope_qout_kv_store(positions, q_pe, q_pe, kv_c, st["kv_weight"], 1e-6, k_pe.unsqueeze(1), st["cos_sin"],
                               False, buf, where)
    if not fp8:
        hcu_ops.store_mla_kv4(kv_c, k_pe, loc, st["kv"])


def decode_step(st, form="tokens", n_blocks=32):
    """One step: returns the tables, the selection and (out, lse).  The activations are copied to the buffers that the
    front end works on, so the state stays as it is and a replay is the same step again; the next one would take
    ``t.free_head`` and lengths raised by the new tokens."""
    for k in ("kv_c", "k_pe", "q_cat"):
        st[k].copy_(st[k + "_in"])
    t = hcu_ops.step_tables(st["req_pages"], st["req_idx"], st["seq_lens"], st["new_lens"], st["free_pages"],
                            st["free_head"], st["rows"], st["width"])
    hcu_ops.quant_store_index_k(st["index_k"], t.token_loc, st["index_cache"])
    write_slots(st, t.positions, st["kv_c"], st["k_pe"], st["q_cat"][..., LATENT:], t.loc)
    logits, mask = hcu_ops.mqa_logits(st["index_q"], st["index_cache"], st["index_w"], t.lengths, t.block_table,
                                      st["width"], st["new_tokens"])
    if form == "tokens":
        sel = hcu_ops.sparse_mask_topk_transform(logits, mask, t.lengths, t.page_table_size_1, st["cu"], 2048)
        out, lse = hcu_ops.sparse_mla_attention(st["q_cat"], st["kv"], sel, SM_SCALE)
    else:
        sel = hcu_ops.select_blocks(logits, mask, t.lengths, n_blocks, n_sink=1, n_local=2)
        out, lse = hcu_ops.block_sparse_mla_attention(st["q_cat"], st["kv"], sel, t.block_table, t.lengths, SM_SCALE)
    return t, sel, out, lse


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--context", type=int, default=6000)
    ap.add_argument("--new-tokens", type=int, default=2)
    ap.add_argument("--slots", choices=["fp8", "kv4"], default="fp8")
    a = ap.parse_args()
    st = make_state(a.requests, a.context, a.new_tokens, a.slots)
    for form in ("tokens", "blocks"):
        decode_step(st, form)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, sel, out, lse = decode_step(st, form)
        graph.replay()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(20):
            graph.replay()
        end.record()
        torch.cuda.synchronize()
        print(f"{form}: {st['rows']} rows, selection {tuple(sel.shape)}, out {tuple(out.shape)}, "
              f"{begin.elapsed_time(end) * 50:.1f} us a step")
    print("device status", hcu_ops.read_device_status())


if __name__ == "__main__":
    main()
