"""Workloads of the sparse-attention operators: inputs, plain forms, 64-bit forms and floors.

The operators are what a decode or prefill step of the indexer's user calls around the top-k:

* ``tables``   block tables, slot maps and page allocation of a step, from the requests' lengths;
* ``blocks``   the 64-token blocks a row attends to, chosen by the indexer's scores;
* ``attend``   latent (MLA) attention over selected tokens or blocks, from 656-byte fp8 slots or
               432-byte 4-bit slots;
* ``kv4``      the writer of the 4-bit slots and the read of what was written.

``run`` computes an operator in its plain form (elementary torch operations in float32) or, with
``own`` set, through ``hcu_ops``.  Latents and queries are N(0, 1) like normed activations; the
softmax scale is 1 / sqrt(192 + 64), the un-absorbed head size.
"""
import math
import os
import sys

import torch

own = False

PAGE = 64
LATENT, ROPE = 512, 64
QK = LATENT + ROPE
SM_SCALE = 1.0 / 16.0
FP8_SLOT, KV4_SLOT = 656, 432
FP8_MAX, FP4_MAX = 448.0, 6.0
FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang0.5.18-opt_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import hcu_ops

    return hcu_ops


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One request decoding one token at an 8192-token context: the step's bookkeeping is all latency.
        dict(name="tables_one", op="tables", reqs=1, new=1, lo=8192, hi=8192, width=8256, ragged=False),
        # 64 requests verifying two tokens each, contexts of 4096..65536 tokens: the batch decode step.
        dict(name="tables_mtp64", op="tables", reqs=64, new=2, lo=4096, hi=65536, width=65600, ragged=False),
        # The batch decode step: 128 rows, 2048 tokens' worth of blocks each.
        dict(name="blocks_decode", op="blocks", rows=128, lo=4096, hi=65536, n=32, sink=1, local=2),
        # A prefill chunk over a 65536-token prefix: many rows, a stream of scores.
        dict(name="blocks_prefill", op="blocks", rows=4096, lo=65537, hi=69632, n=64, sink=1, local=4),
        # One row of a lone request: the attention of a single token, split over the GPU.
        dict(name="attend_one", op="attend", fmt="fp8", form="tokens", rows=1, heads=64, k=2048, lo=8192, hi=8192,
             pool=16384),
        # 64 requests x 2 rows over their 2048 selected tokens: the batch decode step.
        dict(name="attend_decode", op="attend", fmt="fp8", form="tokens", rows=128, heads=64, k=2048, lo=4096,
             hi=65536, pool=393216),
        # Part of a prefill chunk, whose rows share one context: the compute-bound end.
        dict(name="attend_prefill", op="attend", fmt="fp8", form="tokens", rows=2048, heads=64, k=2048, lo=65537,
             hi=67584, pool=69632),
        # The batch decode step over whole blocks, some rows shorter than the selection.
        dict(name="attend_blocks", op="attend", fmt="fp8", form="blocks", rows=128, heads=64, k=32, lo=1000, hi=65536,
             pool=393216),
        # 4-bit slots: the decode step of a larger batch, and an odd one of 37 rows with 16 heads
        # (tensor parallel over four GPUs) where several rows see fewer tokens than the selection holds.
        dict(name="attend_kv4", op="attend", fmt="kv4", form="tokens", rows=192, heads=64, k=2048, lo=4096, hi=65536,
             pool=393216),
        dict(name="attend_kv4_odd", op="attend", fmt="kv4", form="blocks", rows=37, heads=16, k=21, lo=700, hi=9001,
             pool=65536),
        # 4-bit slot writer and read-back: a decode step's 128 new tokens, and a long prompt of odd length.
        dict(name="kv4_step", op="kv4", tokens=128, pool=65536),
        dict(name="kv4_prompt", op="kv4", tokens=70001, pool=131072),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "blocks", "blocks", "attend", "attend", "attend", "attend", "kv4"])
    if op == "tables":
        hi = _log_int(rng, 70, 65536)
        width = -(-(hi + 300) // PAGE) * PAGE
        new = rng.choice([1, 1, 2, 3, 4, 5])
        reqs = _log_int(rng, 1, max(1, min(128, int(8.6e6) // (width * new))))
        return dict(op=op, reqs=reqs, new=new, lo=_log_int(rng, 1, hi), hi=hi, width=width,
                    ragged=rng.random() < 0.5)
    if op == "blocks":
        hi = _log_int(rng, 500, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, int(2.8e8) // hi)))
        sink, local = rng.choice([0, 1, 2]), rng.choice([0, 1, 2, 4])
        return dict(op=op, rows=rows, lo=_log_int(rng, 1, hi), hi=hi, n=_log_int(rng, 8, 128), sink=sink, local=local)
    if op == "kv4":
        n = _log_int(rng, 1, 70001)
        return dict(op=op, tokens=n, pool=n + rng.randrange(1, 60000))
    fmt, form = rng.choice(["fp8", "kv4"]), rng.choice(["tokens", "tokens", "blocks"])
    heads = rng.choice([8, 16, 32, 64, 64, 128])
    k = _log_int(rng, 4, 64) if form == "blocks" else _log_int(rng, 33, 2048)
    toks = k * PAGE if form == "blocks" else k
    rows = _log_int(rng, 1, max(1, min(1024, int(2.0e8) // (toks * heads))))
    hi = _log_int(rng, max(64, toks // 2), 65536)
    return dict(op="attend", fmt=fmt, form=form, rows=rows, heads=heads, k=k, lo=_log_int(rng, 1, hi), hi=hi,
                pool=-(-rng.randrange(hi, 200000) // PAGE) * PAGE + PAGE)


# ----------------------------------------------------------------------------------------- inputs
def _lengths(case, n, gen):
    return torch.randint(case["lo"], case["hi"] + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)


def _pack_fp8(latent, rope):
    """656-byte slots: 512 fp8 in four groups, 4 fp32 scales (amax / 448), 64 bf16."""
    n = latent.shape[0]
    x = latent.float().view(n, 4, 128)
    scale = x.abs().amax(-1).clamp_min(1e-6) / FP8_MAX
    q = (x / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return torch.cat([q.view(torch.uint8).view(n, LATENT), scale.contiguous().view(torch.uint8).view(n, 16),
                      rope.contiguous().view(torch.uint8).view(n, 2 * ROPE)], 1)


def _pack_kv4(latent, rope):
    """432-byte slots: 512 e2m1 codes (element 2j in the low half of byte j), 32 e4m3 scales of 16
    elements, one fp32 power of two, 12 zero bytes, 64 bf16."""
    n = latent.shape[0]
    x = latent.float().view(n, 32, 16)
    amax = x.abs().amax(-1)
    _, e = torch.frexp(amax.amax(-1))
    e = torch.where(amax.amax(-1) > 0, e - 11, -100).clamp_min(-100).int()
    t = ((e + 127) << 23).view(torch.float32)  # 2^e; pow and ldexp are not exact on the GPU
    sg = (amax / (FP4_MAX * t)[:, None]).clamp_max(FP8_MAX).to(torch.float8_e4m3fn)
    s = sg.float() * t[:, None]
    a = torch.where(s[..., None] > 0, x.abs() / s[..., None], torch.zeros_like(x))
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * torch.signbit(x)).to(torch.uint8).view(n, LATENT // 2, 2)
    return torch.cat([code[..., 0] + code[..., 1] * 16, sg.view(torch.uint8), t.view(n, 1).view(torch.uint8),
                      torch.zeros(n, 12, dtype=torch.uint8, device=x.device),
                      rope.contiguous().view(torch.uint8).view(n, 2 * ROPE)], 1)


def _cache(fmt, pool, gen):
    out = torch.empty(pool, 1, FP8_SLOT if fmt == "fp8" else KV4_SLOT, dtype=torch.uint8, device="cuda")
    for a in range(0, pool, 65536):
        n = min(65536, pool - a)
        lat = torch.randn(n, LATENT, generator=gen, device="cuda").bfloat16()
        rope = torch.randn(n, ROPE, generator=gen, device="cuda").bfloat16()
        out[a:a + n, 0] = (_pack_fp8 if fmt == "fp8" else _pack_kv4)(lat, rope)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    if op == "tables":
        b, width = case["reqs"], case["width"]
        new = torch.full((b,), case["new"], dtype=torch.int32, device="cuda")
        if case["ragged"]:  # some requests are idle, some take a few tokens more
            new = torch.randint(0, case["new"] + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        seq = torch.minimum(_lengths(case, b, gen), width - new)
        mp = width // PAGE
        ids = torch.randperm((2 * b + 1) * mp, generator=gen, device="cuda").int()
        req_pages = ids[:2 * b * mp].view(2 * b, mp).contiguous()
        return dict(case=case, req_pages=req_pages, seq_lens=seq, new_lens=new, free_pages=ids[2 * b * mp:].contiguous(),
                    req_idx=torch.randperm(2 * b, generator=gen, device="cuda")[:b].int().contiguous(),
                    free_head=torch.zeros(1, dtype=torch.int32, device="cuda"), n_rows=b * case["new"])
    if op == "blocks":
        rows, width = case["rows"], -(-case["hi"] // PAGE) * PAGE
        lens = _lengths(case, rows, gen)
        score = torch.randn(rows, width, generator=gen, device="cuda")
        mask = torch.empty(rows, width // 16, dtype=torch.int16, device="cuda")
        bit = (1 << torch.arange(16, device="cuda", dtype=torch.int32))
        tok = torch.arange(width, device="cuda")
        for a in range(0, rows, 256):  # a set bit: a visible token whose score is not +0 (here all but 1 in 64)
            s = score[a:a + 256]
            on = (tok[None] < lens[a:a + 256, None]) & ((s.view(torch.int32) & 63) != 0)
            w = (on.view(-1, width // 16, 16).int() * bit).sum(-1)
            mask[a:a + 256] = torch.where(w > 32767, w - 65536, w).to(torch.int16)
        return dict(case=case, score=score, mask=mask, lengths=lens)
    if op == "kv4":
        n, pool = case["tokens"], case["pool"]
        loc = torch.randperm(pool, generator=gen, device="cuda")[:n].contiguous()
        gain = torch.exp2(torch.randint(-3, 4, (n, 1), generator=gen, device="cuda").float())
        return dict(case=case, kv_c=(torch.randn(n, LATENT, generator=gen, device="cuda") * gain).bfloat16(),
                    k_pe=torch.randn(n, ROPE, generator=gen, device="cuda").bfloat16(), loc=loc, loc32=loc.int(),
                    buf=torch.zeros(pool, 1, KV4_SLOT, dtype=torch.uint8, device="cuda"))
    rows, pool, k = case["rows"], case["pool"], case["k"]
    st = dict(case=case, kv=_cache(case["fmt"], pool, gen),
              q=torch.randn(rows, case["heads"], QK, generator=gen, device="cuda").bfloat16())
    lens = _lengths(case, rows, gen)
    pages = pool // PAGE
    need = -(-case["hi"] // PAGE)
    # rows walk the pool's shuffled pages from their own offset, as requests that share the pool do
    perm = torch.randperm(pages, generator=gen, device="cuda").int()
    first = torch.randint(0, pages, (rows, 1), generator=gen, device="cuda")
    table = perm[(first + torch.arange(need, device="cuda")[None]) % pages].contiguous()

    def choose(n, m):  # m of the first n[r] in ascending order, all of them and -1 where there are fewer
        j = torch.arange(m, device="cuda")
        u = torch.rand(n.shape[0], m, generator=gen, device="cuda")
        gap = n[:, None] / m
        spread = (j[None] * gap + u * (gap - 1.0)).long()
        return torch.where(n[:, None] > m, torch.minimum(spread, n[:, None].long() - 1),
                           torch.where(j[None] < n[:, None], j[None], -1))

    if case["form"] == "blocks":
        st.update(table=table, lengths=lens, idx=choose((lens + PAGE - 1) // PAGE, k).int().contiguous())
    else:
        pos = choose(lens, k)
        slot = torch.gather(table, 1, pos.clamp_min(0) // PAGE) * PAGE + (pos % PAGE)
        st["idx"] = torch.where(pos >= 0, slot, -1).int().contiguous()
    return st


# ------------------------------------------------------------------------------------ plain forms
def _plain_tables(st):
    case, width = st["case"], st["case"]["width"]
    seq, new, rp, ridx = st["seq_lens"].long(), st["new_lens"].long(), st["req_pages"], st["req_idx"].long()
    rows, mp = st["n_rows"], rp.shape[1]
    have, total = (seq + PAGE - 1) // PAGE, (seq + new + PAGE - 1) // PAGE
    take = total - have
    before = torch.cumsum(take, 0) - take + st["free_head"].long()
    p = torch.arange(mp, device="cuda")[None]
    fresh = (p >= have[:, None]) & (p < total[:, None])
    src = (before[:, None] + p - have[:, None]).clamp(0, st["free_pages"].shape[0] - 1)
    pages = torch.where(fresh, st["free_pages"][src], rp[ridx])
    rp[ridx] = pages
    end = torch.cumsum(new, 0)
    r = torch.arange(rows, device="cuda")
    req = torch.searchsorted(end, r, right=True)
    live = req < seq.shape[0]
    req = req.clamp_max(seq.shape[0] - 1)
    pos = torch.where(live, seq[req] + r - (end - new)[req], 0)
    bt = torch.where(live[:, None] & (p < total[req][:, None]), pages[req], -1)
    off = torch.arange(PAGE, device="cuda", dtype=torch.int32)
    pt = (bt[:, :, None] * PAGE + off).view(rows, mp * PAGE)
    tok = torch.arange(width, device="cuda")[None]
    pt = torch.where(live[:, None] & (tok < (seq + new)[req][:, None]), pt[:, :width], -1)
    loc = torch.where(live, torch.gather(pt, 1, pos[:, None])[:, 0], -1)
    lens = torch.where(live, pos + 1, 0)
    return dict(block_table=bt.int(), page_table=pt.int(), lengths=lens.int(), positions=pos.int(), token_loc=loc.int(),
                loc=loc.long(), free_head=(st["free_head"] + take.sum()).int(), req_pages=rp)


def _plain_blocks(st):
    case = st["case"]
    out = []
    width = st["score"].shape[1]
    nb = width // PAGE
    tok = torch.arange(width, device="cuda")
    blk = torch.arange(nb, device="cuda")[None]
    for a in range(0, case["rows"], 512):
        s, lens = st["score"][a:a + 512], st["lengths"][a:a + 512, None].long()
        bits = (st["mask"][a:a + 512, :, None].int() >> torch.arange(16, device="cuda", dtype=torch.int32)) & 1
        s = torch.where(bits.view(s.shape) != 0, s, 0.0)
        s = torch.where(tok[None] < lens, s, -math.inf)
        m = s.view(-1, nb, PAGE).amax(-1)
        have = (lens + PAGE - 1) // PAGE
        seen = blk < have
        forced = seen & ((blk < case["sink"]) | (blk >= have - case["local"]))
        m = torch.where(seen, torch.where(forced, math.inf, m), -math.inf)
        n = min(case["n"], nb)
        top = torch.sort(m, dim=1, descending=True, stable=True).indices[:, :n]
        top = torch.sort(torch.where(torch.arange(n, device="cuda")[None] < have, top, nb), 1).values
        top = torch.where(top < nb, top, -1)
        out.append(torch.nn.functional.pad(top, (0, case["n"] - n), value=-1).int())
    return torch.cat(out)


def _unpack(slots, fmt):
    """[n, slot] uint8 -> [n, 576] float32."""
    n = slots.shape[0]
    if fmt == "fp8":
        v = slots[:, :LATENT].contiguous().view(torch.float8_e4m3fn).float().view(n, 4, 128)
        v = v * slots[:, LATENT:LATENT + 16].contiguous().view(torch.float32)[..., None]
        rope = slots[:, LATENT + 16:FP8_SLOT]
    else:
        b = slots[:, :LATENT // 2]
        code = torch.stack([b & 15, b >> 4], -1).view(n, 32, 16).long()
        lut = torch.tensor(FP4_VALUES + tuple(-x for x in FP4_VALUES), device=slots.device)
        s = slots[:, 256:288].contiguous().view(torch.float8_e4m3fn).float()
        v = lut[code] * (s * slots[:, 288:292].contiguous().view(torch.float32))[..., None]
        rope = slots[:, 304:KV4_SLOT]
    return torch.cat([v.reshape(n, LATENT), rope.contiguous().view(torch.bfloat16).float()], 1)


def _slots(st, a, b):
    """Slot numbers [b - a, tokens] of the selected tokens of rows a..b, -1 where there is none."""
    idx = st["idx"][a:b].long()
    if st["case"]["form"] == "tokens":
        return idx
    off = torch.arange(PAGE, device="cuda")
    pos = idx[..., None] * PAGE + off
    page = torch.gather(st["table"][a:b].long(), 1, idx.clamp_min(0))
    on = (idx >= 0)[..., None] & (pos < st["lengths"][a:b, None, None])
    return torch.where(on, page[..., None] * PAGE + off, -1).view(b - a, -1)


def _plain_attend(st):
    case = st["case"]
    rows, h = case["rows"], case["heads"]
    kv = st["kv"].view(st["kv"].shape[0], -1)
    toks = case["k"] * (PAGE if case["form"] == "blocks" else 1)
    step = max(1, (1 << 18) // toks)
    outs, lses = [], []
    for a in range(0, rows, step):
        b = min(rows, a + step)
        slot = _slots(st, a, b)
        k = _unpack(kv[slot.clamp_min(0).view(-1)], case["fmt"]).view(b - a, toks, QK)
        s = torch.bmm(st["q"][a:b].float(), k.transpose(1, 2)) * SM_SCALE
        s = torch.where((slot >= 0)[:, None], s, -math.inf)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        o = torch.bmm(p, k[..., :LATENT])
        outs.append(torch.where(z > 0, o / z, 0.0).bfloat16())
        lses.append((m + torch.log(z))[..., 0])
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _plain_kv4(st):
    st["buf"][st["loc"], 0] = _pack_kv4(st["kv_c"], st["k_pe"])
    return _unpack(st["buf"][st["loc32"].long(), 0], "kv4").bfloat16().view(-1, 1, QK)


def run(state):
    op = state["case"]["op"]
    if not own:
        return dict(tables=_plain_tables, blocks=_plain_blocks, attend=_plain_attend, kv4=_plain_kv4)[op](state)
    ops = _ops()
    case = state["case"]
    if op == "tables":
        t = ops.step_tables(state["req_pages"], state["req_idx"], state["seq_lens"], state["new_lens"],
                            state["free_pages"], state["free_head"], state["n_rows"], case["width"])
        return dict(block_table=t.block_table, page_table=t.page_table_size_1, lengths=t.lengths, positions=t.positions,
                    token_loc=t.token_loc, loc=t.loc, free_head=t.free_head, req_pages=state["req_pages"])
    if op == "blocks":
        return ops.select_blocks(state["score"], state["mask"], state["lengths"], case["n"], n_sink=case["sink"],
                                 n_local=case["local"])
    if op == "kv4":
        ops.store_mla_kv4(state["kv_c"], state["k_pe"], state["loc"], state["buf"])
        return ops.dequantize_mla_kv4_paged(state["buf"], state["loc32"])
    if case["form"] == "blocks":
        out, lse = ops.block_sparse_mla_attention(state["q"], state["kv"], state["idx"], state["table"],
                                                  state["lengths"], SM_SCALE)
    else:
        out, lse = ops.sparse_mla_attention(state["q"], state["kv"], state["idx"], SM_SCALE)
    return dict(out=out, lse=lse)


# ---------------------------------------------------------------------------- 64-bit forms, floors
def _exact_attend(st):
    """Row by row from the definition: softmax(scale q k^T) v, values read from the slots in float64."""
    case = st["case"]
    kv = st["kv"].view(st["kv"].shape[0], -1)
    e2m1 = torch.tensor([(-1) ** (c >> 3) * (((c & 1) + 2 * ((c >> 1 & 3) > 0)) * 2.0 ** (max(c >> 1 & 3, 1) - 2))
                         for c in range(16)], dtype=torch.float64, device="cuda")
    out = torch.zeros(case["rows"], case["heads"], LATENT, dtype=torch.float64, device="cuda")
    lse = torch.full((case["rows"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for r in range(case["rows"]):
        if case["form"] == "tokens":
            sl = st["idx"][r]
            sl = sl[sl >= 0].long()
        else:
            b = st["idx"][r]
            pos = (b[b >= 0].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")).view(-1)
            pos = pos[pos < st["lengths"][r]]
            sl = st["table"][r].long()[pos // PAGE] * PAGE + pos % PAGE
        if sl.numel() == 0:
            continue
        raw = kv[sl]
        if case["fmt"] == "fp8":
            sc = raw[:, 512:528].contiguous().view(torch.float32).double()
            v = raw[:, :512].contiguous().view(torch.float8_e4m3fn).double() * sc.repeat_interleave(128, 1)
            rope = raw[:, 528:656]
        else:
            sc = raw[:, 256:288].contiguous().view(torch.float8_e4m3fn).double()
            sc = sc * raw[:, 288:292].contiguous().view(torch.float32).double()
            v = torch.empty(sl.numel(), 512, dtype=torch.float64, device="cuda")
            v[:, 0::2] = e2m1[(raw[:, :256] % 16).long()]
            v[:, 1::2] = e2m1[(raw[:, :256] // 16).long()]
            v = v * sc.repeat_interleave(16, 1)
            rope = raw[:, 304:432]
        k = torch.cat([v, rope.contiguous().view(torch.bfloat16).double()], 1)
        s = st["q"][r].double() @ k.T * SM_SCALE
        lse[r] = torch.logsumexp(s, -1)
        out[r] = torch.softmax(s, -1) @ v
    return dict(out=out, lse=lse)


def _pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_kv4(st):
    """The stored values from the format's definition: nearest e2m1 multiple of the group's scale."""
    x = st["kv_c"].double().view(-1, 32, 16)
    amax = x.abs().amax(-1)
    top = amax.amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 11, -100).clamp_min(-100)
    t = _pow2(e)
    sg = torch.clamp(amax / t[:, None] / 6.0, max=448.0)
    # nearest e4m3: steps of 2^(exponent - 3), 2^-9 below the normals; torch.round ties to even
    step = _pow2((torch.frexp(sg)[1] - 4).clamp_min(-9))
    s = torch.round(sg / step) * step * t[:, None]
    a = x.abs() / torch.where(s > 0, s, 1.0)[..., None] * (s > 0)[..., None]
    step = torch.where(a >= 4.0, 2.0, torch.where(a >= 2.0, 1.0, 0.5)).double()
    q = (torch.round(a / step) * step).clamp_max(6.0)
    v = torch.sign(x) * q * s[..., None]
    return torch.cat([v.view(-1, 1, LATENT), st["k_pe"].double().view(-1, 1, ROPE)], -1)


def exact(case, seed):
    if case["op"] in ("tables", "blocks"):
        return None  # whole numbers
    st = prepare(case, seed)
    if case["op"] == "kv4":
        return _exact_kv4(st)
    toks = case["k"] * (PAGE if case["form"] == "blocks" else 1)
    if case["rows"] * toks * case["heads"] > 1.3e8:  # the 64-bit products would take too long
        return None
    return _exact_attend(st)


def work(case):
    op = case["op"]
    if op == "tables":
        rows, pages = case["reqs"] * case["new"], case["width"] // PAGE
        mean = (case["lo"] + case["hi"]) // 2
        return dict(bytes=rows * (case["width"] * 4 + pages * 4 + 24) + case["reqs"] * (mean // PAGE * 4 + 12), flops=0)
    if op == "blocks":
        mean = (case["lo"] + case["hi"]) / 2
        return dict(bytes=int(case["rows"] * (mean * 4.125 + 4 + case["n"] * 4)), flops=int(case["rows"] * mean))
    if op == "kv4":
        return dict(bytes=case["tokens"] * (2 * QK + 8 + KV4_SLOT + KV4_SLOT + 4 + 2 * QK),
                    flops=case["tokens"] * LATENT * 4)
    toks = case["k"] * (PAGE if case["form"] == "blocks" else 1)
    rows, h = case["rows"], case["heads"]
    # tokens a row attends to, over lengths spread evenly from lo to hi
    lo, hi = case["lo"], case["hi"]
    part = min(max((toks - lo) / max(hi - lo, 1), 0.0), 1.0)
    mean = part * (lo + min(hi, toks)) / 2 + (1 - part) * toks if lo < toks else toks
    read = min(case["pool"], rows * mean) * (FP8_SLOT if case["fmt"] == "fp8" else KV4_SLOT)
    return dict(bytes=int(read + rows * (case["k"] * 4 + h * (2 * QK + 2 * LATENT + 4))),
                flops=int(2 * rows * mean * h * (QK + LATENT)))
