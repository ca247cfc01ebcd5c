"""What a serving step does next to the KV cache, as measurable cases.

Four operators around the paged cache: block tables and slot maps from request
lengths (``build_slot_mapping``), rotary positions of fresh rows with K and V
written to their pages (``rotary_embedding_and_cache``), attention of a batch
over a prefix that all its requests share (``shared_prefix_attention``), and
CacheBlend's attention of rows at given positions over all keys
(``position_attention``).  ``run`` computes each in plain PyTorch, or through
the framework's own entry points where ``own`` is true.  Geometry comes from
the model shapes of ``lmcache_ascend_b200.models`` (Llama-3-8B: 32/8 heads of
128; Qwen3-32B: 64/8; its TP4 shard: 16/2) and the block sizes the tests and
benchmarks use (16, 64, 128).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a few requests: only the launch counts
        dict(name="slots_decode", op="slots", batch=7, ctx_min=1, ctx_max=4096, new_min=1, new_max=1,
             block=16, layout=1),
        # admission of whole prompts next to running decodes, int64 slots of ~0.6 M tokens
        dict(name="slots_ingest", op="slots", batch=1000, ctx_min=0, ctx_max=512, new_min=1,
             new_max=2048, block=16, layout=2),
        # decode batch of Qwen3-32B: one fresh row per request
        dict(name="rope_decode", op="rope", tokens=64, heads=64, kv_heads=8, dim=128, rot=128,
             neox=True, dtype="bf16", block=16, scaling="none", layout=3),
        # a 16k-token prompt of Qwen3-32B (one token more, an odd length)
        dict(name="rope_prefill", op="rope", tokens=16385, heads=64, kv_heads=8, dim=128,
             rot=128, neox=True, dtype="bf16", block=128, scaling="none", layout=4),
        # half of each head rotated, pairs interleaved, positions scaled for long contexts
        dict(name="rope_partial", op="rope", tokens=5001, heads=32, kv_heads=8, dim=128, rot=64,
             neox=False, dtype="fp16", block=64, scaling="yarn", layout=5),
        # four requests on a short system prompt: latency
        dict(name="prefix_small", op="prefix", batch=4, q_len=1, prefix=500, own_min=1,
             own_max=64, heads=32, kv_heads=8, dim=128, dtype="bf16", block=16, softcap=0.0,
             alibi=False, layout=6),
        # decode of 64 requests of Qwen3-32B on a 16k-token prefix (the prefix-hit workload)
        dict(name="prefix_serving", op="prefix", batch=64, q_len=1, prefix=16384,
             own_min=64, own_max=1024, heads=64, kv_heads=8, dim=128, dtype="bf16", block=16,
             softcap=0.0, alibi=False, layout=7),
        # four drafted tokens each of 33 requests over 100k shared tokens, TP4 shard, capped
        # scores
        dict(name="prefix_verify", op="prefix", batch=33, q_len=4, prefix=100003, own_min=4,
             own_max=500, heads=16, kv_heads=2, dim=128, dtype="fp16", block=64, softcap=30.0,
             alibi=False, layout=8),
        # CacheBlend of a short request: a few rows recomputed
        dict(name="blend_small", op="blend", q_tokens=38, k_tokens=257, docs=1, heads=32,
             kv_heads=8, dim=128, dtype="bf16", softcap=0.0, alibi=False, prefix=0, layout=9),
        # CacheBlend of a 16k-token prompt of Llama-3-8B at the default ratio (15 % of the rows)
        dict(name="blend_recompute", op="blend", q_tokens=2457, k_tokens=16384, docs=1, heads=32,
             kv_heads=8, dim=128, dtype="bf16", softcap=0.0, alibi=False, prefix=0, layout=10),
        # 24 documents of ragged lengths packed, each seeing the start of itself whole, capped
        # scores, distance bias, heads of 64
        dict(name="blend_documents", op="blend", q_tokens=8191, k_tokens=8191, docs=24, heads=32,
             kv_heads=8, dim=64, dtype="fp16", softcap=50.0, alibi=True, prefix=100, layout=11),
        # every row of a 16k-token prompt of Qwen3-32B
        dict(name="blend_full", op="blend", q_tokens=16384, k_tokens=16384, docs=1, heads=64,
             kv_heads=8, dim=128, dtype="bf16", softcap=0.0, alibi=False, prefix=0, layout=12),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "rope", "prefix", "blend"])
    layout = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 7, 8])
    block = rng.choice([16, 32, 64, 128])
    if op == "slots":
        batch = _logint(rng, 1, 1000)
        hi = _logint(rng, 1, max(1, min(8192, 1000000 // batch)))
        return dict(op=op, batch=batch, ctx_min=0, ctx_max=_logint(rng, 1, 8192),
                    new_min=0 if batch > 4 else 1, new_max=hi, block=block, layout=layout)
    if op == "rope":
        tokens = _logint(rng, 1, 16385 * 80 // (heads + 2 * kv))
        rot = rng.choice([dim, dim // 2, dim // 4])
        return dict(op=op, tokens=min(tokens, 65536), heads=heads, kv_heads=kv, dim=dim, rot=rot,
                    neox=rng.random() < 0.5, dtype=dtype, block=block,
                    scaling=rng.choice(["none", "linear", "yarn"]), layout=layout)
    softcap = rng.choice([0.0, 0.0, 30.0, 50.0])
    alibi = rng.random() < 0.3
    if op == "prefix":
        q_len = rng.choice([1, 1, 1, 2, 4, 5])
        batch = _logint(rng, 1, 96)
        rows = batch * q_len * heads
        prefix = _logint(rng, 1, min(131072, max(2000, 33 * 4 * 16 * 100003 // rows)))
        return dict(op=op, batch=batch, q_len=q_len, prefix=prefix,
                    own_min=q_len, own_max=q_len + _logint(rng, 1, 1024), heads=heads,
                    kv_heads=kv, dim=dim, dtype=dtype, block=block, softcap=softcap,
                    alibi=alibi, layout=layout)
    k_tokens = _logint(rng, 1, 16384)
    docs = rng.choice([1, 1, 2, 5, 24])
    full = rng.random() < 0.3
    q_tokens = k_tokens if full else max(1, _logint(rng, 1, k_tokens + 1) - 1)
    return dict(op=op, q_tokens=min(q_tokens, k_tokens), k_tokens=k_tokens,
                docs=min(docs, k_tokens), heads=heads, kv_heads=kv, dim=dim, dtype=dtype,
                softcap=softcap, alibi=alibi, prefix=rng.choice([0, 0, 100]), layout=layout)


# ------------------------------------------------------------------ layouts
# Lengths, tables and positions of a case; drawn from the case alone.
def _lens(r, case, what):
    return [r.randint(case[what + "_min"], case[what + "_max"]) for _ in range(case["batch"])]


def _slot_lens(case):
    r = random.Random(case["layout"])
    return _lens(r, case, "ctx"), _lens(r, case, "new")


def _own_lens(case):
    return _lens(random.Random(case["layout"]), case, "own")


def _doc_lens(case):
    r = random.Random(case["layout"])
    n, k = case["k_tokens"], case["docs"]
    cuts = sorted(r.sample(range(1, n), k - 1)) if k > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [n])]


def _blend_layout(case):
    """Key positions and documents, and the recomputed rows, as numpy arrays."""
    lens = _doc_lens(case)
    kp = np.concatenate([np.arange(n) for n in lens])
    kd = np.repeat(np.arange(len(lens)), lens)
    r = np.random.default_rng(case["layout"])
    if case["q_tokens"] == case["k_tokens"]:
        rows = np.arange(case["k_tokens"])
    else:
        rows = np.sort(r.choice(case["k_tokens"], case["q_tokens"], replace=False))
    return kp, kd, rows


def _blend_pairs(case):
    lens = _doc_lens(case)
    kp, kd, rows = _blend_layout(case)
    limit = np.maximum(kp[rows] + 1, case["prefix"])
    return int(np.minimum(limit, np.asarray(lens)[kd[rows]]).sum())


def _slopes(heads):
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


# ------------------------------------------------------------------ prepare
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _int(x, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype, device=DEV)


def _prep_slots(case, seed):
    ctx, new = _slot_lens(case)
    bs = case["block"]
    have = [-(-c // bs) for c in ctx]
    need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    width = max(1, max(need)) + 2
    total = sum(need) + 5
    ids = torch.randperm(total, device=DEV, generator=_gen(seed)).to(torch.int32)
    h = _int(have, torch.int64)
    col = torch.arange(width, device=DEV)
    first = torch.cumsum(h, 0) - h
    idx = (first[:, None] + col[None, :]).clamp(max=total - 1)
    tables = torch.where(col[None, :] < h[:, None], ids[idx], ids.new_full((), -1))
    return dict(ctx=_int(ctx), new=_int(new), tables=tables.contiguous(),
                free=ids[sum(have):].contiguous(), tokens=sum(new), blocks=total)


def _scaling(case):
    s = case["scaling"]
    if s == "linear":
        return {"rope_type": "linear", "factor": 4.0}
    if s == "yarn":
        return {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 8192}
    return None


def _angles(case, positions):
    """Rotation table rows (cos | sin), angles in 64 bits."""
    rot, base, s = case["rot"], 1000000.0, _scaling(case)
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    gain = 1.0
    if s and s["rope_type"] == "linear":
        inv = inv / s["factor"]
    elif s:
        orig, f = s["original_max_position_embeddings"], s["factor"]

        def dim_of(turns):
            return rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), rot - 1)
        i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        inv = inv / f * ramp + inv * (1 - ramp)
        gain = 0.1 * math.log(f) + 1.0
    a = positions.to(torch.float64)[:, None] * inv[None, :]
    return (torch.cat([a.cos(), a.sin()], 1) * gain).to(torch.float32)


def _prep_rope(case, seed):
    g = _gen(seed)
    dt, T, D, bs = DTYPES[case["dtype"]], case["tokens"], case["dim"], case["block"]
    H, KH = case["heads"], case["kv_heads"]
    # q, k and v are slices of one projection's rows
    qkv = torch.randn(T, (H + 2 * KH) * D, device=DEV, generator=g).to(dt)
    nb = -(-T // bs) + 3
    kc = torch.randn(nb, bs, KH, D, device=DEV, generator=g).to(dt)
    vc = torch.randn(nb, bs, KH, D, device=DEV, generator=g).to(dt)
    blocks = torch.randperm(nb, device=DEV, generator=g)
    t = torch.arange(T, device=DEV)
    slots = blocks[t // bs] * bs + t % bs
    max_pos = 40960 if T <= 40960 else T
    start = random.Random(case["layout"]).randrange(max_pos - T + 1)
    if T <= 64:  # a decode batch: every request somewhere else
        pos = torch.randint(0, max_pos, (T,), device=DEV, generator=g)
    else:
        pos = t + start
    table = _angles(case, torch.arange(max_pos, device=DEV))
    q, k, v = qkv.split([H * D, KH * D, KH * D], dim=1)
    return dict(q=q, k=k, v=v, kc=kc, vc=vc, slots=slots, pos=pos, table=table)


def _prep_prefix(case, seed):
    g = _gen(seed)
    dt, D, bs, B, P = (DTYPES[case["dtype"]], case["dim"], case["block"], case["batch"],
                       case["prefix"])
    H, KH, Tq = case["heads"], case["kv_heads"], case["q_len"]
    lens = _own_lens(case)
    npb = -(-P // bs)
    nob = [-(-n // bs) for n in lens]
    nb = npb + sum(nob) + 2
    kc = torch.randn(nb, bs, KH, D, device=DEV, generator=g).to(dt)
    vc = torch.randn(nb, bs, KH, D, device=DEV, generator=g).to(dt)
    ids = torch.randperm(nb, device=DEV, generator=g).to(torch.int32)
    width = max(nob) + 1
    tables = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    at = npb
    for b, n in enumerate(nob):
        tables[b, :n] = ids[at:at + n]
        at += n
    # queries wide enough that the softmax is not flat
    q = (torch.randn(B, Tq, H, D, device=DEV, generator=g) * 2).to(dt)
    slopes = torch.tensor(_slopes(H), device=DEV) if case["alibi"] else None
    return dict(q=q, kc=kc, vc=vc, prefix=ids[:npb].contiguous(), tables=tables,
                lens=_int(lens), slopes=slopes)


def _prep_blend(case, seed):
    g = _gen(seed)
    dt, D, H, KH = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    kp, kd, rows = _blend_layout(case)
    k = torch.randn(case["k_tokens"], KH, D, device=DEV, generator=g).to(dt)
    v = torch.randn(case["k_tokens"], KH, D, device=DEV, generator=g).to(dt)
    q = (torch.randn(case["q_tokens"], H, D, device=DEV, generator=g) * 2).to(dt)
    packed = case["docs"] > 1
    prefix = _int(np.full(len(rows), case["prefix"])) if case["prefix"] else None
    slopes = torch.tensor(_slopes(H), device=DEV) if case["alibi"] else None
    return dict(q=q, k=k, v=v, qp=_int(kp[rows], torch.int64), kp=_int(kp, torch.int64),
                qd=_int(kd[rows]) if packed else None, kd=_int(kd) if packed else None,
                prefix=prefix, slopes=slopes)


def prepare(case, seed):
    made = {"slots": _prep_slots, "rope": _prep_rope, "prefix": _prep_prefix,
            "blend": _prep_blend}[case["op"]](case, seed)
    made["case"] = case
    return made


# ---------------------------------------------------------------------- run
def _plain_slots(s):
    case = s["case"]
    bs, n = case["block"], s["tokens"]
    ctx, new, tables = s["ctx"].long(), s["new"].long(), s["tables"]
    have, need = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    taken = torch.cumsum(need - have, 0)
    zero = taken.new_zeros(1)
    off = torch.cat([zero, taken])
    col = torch.arange(tables.shape[1], device=DEV)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    src = (off[:-1, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    tables.copy_(torch.where(fresh, s["free"][src], tables))
    start = torch.cat([zero, torch.cumsum(new, 0)])
    t = torch.arange(n, device=DEV)
    req = torch.searchsorted(start[1:].contiguous(), t, right=True)
    pos = ctx[req] + t - start[req]
    slot = tables[req, pos // bs].long() * bs + pos % bs
    return (slot, pos, req.int(), start.int(), (ctx + new).int(), off.int(), tables)


def _own_slots(s):
    from lmcache_ascend_b200.ops import api

    m = api.build_slot_mapping(s["ctx"], s["new"], s["tables"], s["case"]["block"], s["tokens"],
                               free_blocks=s["free"], num_blocks=s["blocks"])
    return (m.slot_mapping, m.positions, m.request_ids, m.query_start_loc, m.seq_lens, m.taken,
            s["tables"])


def _rotate(x, cs, rot, neox):
    """x [T, heads, D] in 32 bits, cs [T, rot]."""
    half = rot // 2
    c, sn = cs[:, None, :half], cs[:, None, half:]
    y = x.clone()
    if neox:
        a, b = x[..., :half], x[..., half:rot]
        y[..., :half], y[..., half:rot] = a * c - b * sn, b * c + a * sn
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * sn, b * c + a * sn
    return y


def _plain_rope(s):
    case = s["case"]
    D, T = case["dim"], case["tokens"]
    cs = s["table"][s["pos"]]
    q = _rotate(s["q"].float().view(T, -1, D), cs, case["rot"], case["neox"])
    k = _rotate(s["k"].float().view(T, -1, D), cs, case["rot"], case["neox"])
    dt = s["q"].dtype
    kf, vf = s["kc"].view(-1, k.shape[1], D), s["vc"].view(-1, k.shape[1], D)
    kf[s["slots"]] = k.to(dt)
    vf[s["slots"]] = s["v"].reshape(T, -1, D)
    return q.to(dt).view(T, -1), s["kc"], s["vc"]


def _own_rope(s):
    from lmcache_ascend_b200.ops import api

    q = api.rotary_embedding_and_cache(s["pos"], s["q"], s["k"], s["v"], s["kc"], s["vc"],
                                       s["slots"], s["case"]["dim"], s["table"],
                                       s["case"]["neox"])
    return q, s["kc"], s["vc"]


def _shape_scores(x, case, distance, slopes):
    cap = case["softcap"]
    if cap:
        x = cap * torch.tanh(x / cap)
    if slopes is not None:
        x = x - slopes * distance
    return x


def _plain_prefix(s):
    case = s["case"]
    q = s["q"].float()
    B, Tq, H, D = q.shape
    KH, P, bs = case["kv_heads"], case["prefix"], case["block"]
    G = H // KH
    kf, vf = s["kc"].view(-1, KH, D), s["vc"].view(-1, KH, D)
    t = torch.arange(P, device=DEV)
    pslot = s["prefix"].long()[t // bs] * bs + t % bs
    lens = s["lens"].long()
    n = case["own_max"]
    j = torch.arange(n, device=DEV)
    oslot = s["tables"].long()[:, (j // bs).clamp(max=s["tables"].shape[1] - 1)] * bs + j % bs
    seen = j[None, None, :] <= (lens[:, None] - Tq + torch.arange(Tq, device=DEV))[:, :, None]
    qpos = P + lens[:, None] - Tq + torch.arange(Tq, device=DEV)
    dist_p = (qpos[:, :, None] - t).abs().float()[:, :, None, :]
    dist_o = (qpos[:, :, None] - P - j).abs().float()[:, :, None, :]
    out = torch.empty(B, Tq, H, D, device=DEV)
    lse = torch.empty(B, Tq, H, device=DEV)
    for h in range(KH):
        qh = q[:, :, h * G:(h + 1) * G] * D ** -0.5
        sl = None if s["slopes"] is None else s["slopes"][h * G:(h + 1) * G][:, None]
        kp, vp = kf[pslot, h].float(), vf[pslot, h].float()
        ko, vo = kf[oslot, h].float(), vf[oslot, h].float()
        a = _shape_scores(qh @ kp.T, case, dist_p, sl)
        o = (qh.reshape(B, Tq * G, D) @ ko.transpose(1, 2)).view(B, Tq, G, n)
        o = _shape_scores(o, case, dist_o, sl).masked_fill(~seen[:, :, None, :], -math.inf)
        m = torch.maximum(a.amax(-1), o.amax(-1))[..., None]
        ea, eo = torch.exp(a - m), torch.exp(o - m)
        l = ea.sum(-1) + eo.sum(-1)
        y = ea @ vp + (eo.view(B, Tq * G, n) @ vo).view(B, Tq, G, D)
        out[:, :, h * G:(h + 1) * G] = y / l[..., None]
        lse[:, :, h * G:(h + 1) * G] = m[..., 0] + torch.log(l)
    return out.to(s["q"].dtype), lse


def _own_prefix(s):
    from lmcache_ascend_b200.ops import api

    return api.shared_prefix_attention(
        s["q"], s["kc"], s["vc"], s["prefix"], s["case"]["prefix"], s["tables"], s["lens"],
        softcap=s["case"]["softcap"], alibi_slopes=s["slopes"], return_lse=True)


def _plain_blend(s):
    case = s["case"]
    q, k, v = s["q"], s["k"].float(), s["v"].float()
    Tq, H, D = q.shape
    KH = k.shape[1]
    G = H // KH
    out = torch.empty(Tq, H, D, device=DEV)
    lse = torch.empty(Tq, H, device=DEV)
    for a in range(0, Tq, 1024):
        b = min(Tq, a + 1024)
        limit = s["qp"][a:b] + 1
        if s["prefix"] is not None:
            limit = torch.maximum(limit, s["prefix"][a:b].long())
        seen = s["kp"][None, :] < limit[:, None]
        if s["qd"] is not None:
            seen &= s["qd"][a:b, None] == s["kd"][None, :]
        dist = (s["qp"][a:b, None] - s["kp"][None, :]).abs().float()
        for h in range(KH):
            qh = q[a:b, h * G:(h + 1) * G].float().transpose(0, 1) * D ** -0.5
            sl = None if s["slopes"] is None else s["slopes"][h * G:(h + 1) * G][:, None, None]
            x = _shape_scores(qh @ k[:, h].T, case, dist, sl)
            x = x.masked_fill(~seen, -math.inf)
            m = x.amax(-1, keepdim=True)
            e = torch.exp(x - m)
            l = e.sum(-1, keepdim=True)
            out[a:b, h * G:(h + 1) * G] = (e @ v[:, h] / l).transpose(0, 1)
            lse[a:b, h * G:(h + 1) * G] = (m + torch.log(l))[..., 0].T
    return out.to(s["q"].dtype), lse


def _own_blend(s):
    from lmcache_ascend_b200.ops import api

    return api.position_attention(
        s["q"], s["k"], s["v"], s["qp"], s["kp"], softcap=s["case"]["softcap"],
        alibi_slopes=s["slopes"], q_documents=s["qd"], k_documents=s["kd"],
        q_prefix_lens=s["prefix"], return_lse=True)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"slots": _own_slots, "rope": _own_rope, "prefix": _own_prefix,
                "blend": _own_blend}[op](state)
    return {"slots": _plain_slots, "rope": _plain_rope, "prefix": _plain_prefix,
            "blend": _plain_blend}[op](state)


# -------------------------------------------------------------------- exact
def _exact_slots(s):
    case = s["case"]
    bs = case["block"]
    ctx, new = s["ctx"].cpu().numpy(), s["new"].cpu().numpy()
    tables, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy()
    slots, pos, req, start, off = [], [], [], [0], [0]
    for b, (c, n) in enumerate(zip(ctx.tolist(), new.tolist())):
        have, need = -(-c // bs), -(-(c + n) // bs)
        tables[b, have:need] = free[off[-1]:off[-1] + need - have]
        off.append(off[-1] + need - have)
        start.append(start[-1] + n)
        p = np.arange(c, c + n, dtype=np.int64)
        slots.append(tables[b, p // bs].astype(np.int64) * bs + p % bs)
        pos.append(p)
        req.append(np.full(n, b, dtype=np.int32))
    return (torch.from_numpy(np.concatenate(slots)), torch.from_numpy(np.concatenate(pos)),
            torch.from_numpy(np.concatenate(req)), torch.tensor(start, dtype=torch.int32),
            torch.from_numpy(ctx + new), torch.tensor(off, dtype=torch.int32),
            torch.from_numpy(tables))


def _exact_rope(s):
    case = s["case"]
    T, D, rot = case["tokens"], case["dim"], case["rot"]
    cs = s["table"].double()[s["pos"]]
    # the pair (first, second) as one complex number times cos + i sin
    w = torch.complex(cs[:, :rot // 2], cs[:, rot // 2:])[:, None, :]
    first = torch.arange(rot // 2, device=DEV) * (1 if case["neox"] else 2)
    second = first + (rot // 2 if case["neox"] else 1)

    def turn(x):
        x = x.double().reshape(T, -1, D).clone()
        z = torch.complex(x[..., first], x[..., second]) * w
        x[..., first], x[..., second] = z.real, z.imag
        return x

    kc, vc = s["kc"].double(), s["vc"].double()
    bs = case["block"]
    kc[s["slots"] // bs, s["slots"] % bs] = turn(s["k"])
    vc[s["slots"] // bs, s["slots"] % bs] = s["v"].double().reshape(T, -1, D)
    return turn(s["q"]).reshape(T, -1), kc, vc


def _exact_attend(q, k, v, visible, distance, case, slopes):
    """q [R, D] over k, v [N, D] in 64 bits; visible and distance [R, N] or None."""
    x = (q @ k.T) / math.sqrt(q.shape[1])
    if case["softcap"]:
        x = torch.tanh(x / case["softcap"]) * case["softcap"]
    if slopes is not None:
        x -= slopes * distance
    if visible is not None:
        x[~visible] = -math.inf
    lse = torch.logsumexp(x, dim=1)
    return torch.exp(x - lse[:, None]) @ v, lse


def _exact_prefix(s):
    case = s["case"]
    B, Tq, H, D = s["q"].shape
    KH, P, bs = case["kv_heads"], case["prefix"], case["block"]
    G = H // KH
    if 4 * B * Tq * H * D * P > 4e12:
        return None
    out = torch.empty(B, Tq, H, D, dtype=torch.float64, device=DEV)
    lse = torch.empty(B, Tq, H, dtype=torch.float64, device=DEV)
    flat = [c.flatten(0, 1) for c in (s["kc"], s["vc"])]
    row = torch.arange(bs, device=DEV)
    pages = (s["prefix"].long()[:, None] * bs + row).flatten()[:P]
    shared = [f[pages].double() for f in flat]
    for b, n in enumerate(s["lens"].tolist()):
        own_rows = (s["tables"][b].long()[:, None] * bs + row).flatten()[:n]
        k, v = (torch.cat([p, f[own_rows].double()]) for p, f in zip(shared, flat))
        at = torch.arange(P + n, device=DEV)
        for i in range(Tq):
            p = P + n - Tq + i
            for h in range(KH):
                sl = None
                if s["slopes"] is not None:
                    sl = s["slopes"][h * G:(h + 1) * G].double()[:, None]
                o, e = _exact_attend(s["q"][b, i, h * G:(h + 1) * G].double(), k[:p + 1, h],
                                     v[:p + 1, h], None, (p - at[:p + 1]).double()[None], case,
                                     sl)
                out[b, i, h * G:(h + 1) * G], lse[b, i, h * G:(h + 1) * G] = o, e
    return out, lse


def _exact_blend(s):
    case = s["case"]
    Tq, H, D = s["q"].shape
    Tk, KH, _ = s["k"].shape
    if H * Tq * Tk > 2e10:
        return None
    qp, kp = s["qp"], s["kp"]
    out = torch.empty(Tq, H, D, dtype=torch.float64, device=DEV)
    lse = torch.empty(Tq, H, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // Tk)
    for a in range(0, Tq, step):
        r = slice(a, min(Tq, a + step))
        gap = qp[r, None] - kp[None, :]
        visible = gap >= 0
        if s["prefix"] is not None:
            visible |= kp[None, :] < s["prefix"][r, None]
        if s["qd"] is not None:
            visible &= s["qd"][r, None] == s["kd"][None, :]
        gap = gap.abs().double()
        for h in range(H):
            sl = None if s["slopes"] is None else s["slopes"][h].double()
            out[r, h], lse[r, h] = _exact_attend(
                s["q"][r, h].double(), s["k"][:, h * KH // H].double(),
                s["v"][:, h * KH // H].double(), visible, gap, case, sl)
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    return {"slots": _exact_slots, "rope": _exact_rope, "prefix": _exact_prefix,
            "blend": _exact_blend}[case["op"]](s)


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "slots":
        ctx, new = _slot_lens(case)
        bs, B, T = case["block"], case["batch"], sum(new)
        fresh = sum(-(-(c + n) // bs) + (-c // bs) for c, n in zip(ctx, new))
        # lengths in, free blocks in and out, two int64 and one int32 per token
        return {"bytes": 8 * B + 8 * fresh + 20 * T + 12 * B + 8, "flops": 4 * T}
    H, KH, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        T, rot = case["tokens"], case["rot"]
        return {"bytes": T * (2 * 2 * D * (H + 2 * KH) + 4 * rot + 16),
                "flops": 3 * T * (H + KH) * rot}
    if case["op"] == "prefix":
        lens, P, Tq = _own_lens(case), case["prefix"], case["q_len"]
        pairs = sum(Tq * P + sum(n - Tq + 1 + i for i in range(Tq)) for n in lens)
        rows = len(lens) * Tq * H
        return {"bytes": 4 * KH * D * (P + sum(lens)) + 4 * rows * D + 4 * rows,
                "flops": 4 * D * H * pairs}
    Tq, Tk = case["q_tokens"], case["k_tokens"]
    return {"bytes": 4 * Tk * KH * D + 4 * Tq * H * D + 4 * Tq * H + 8 * (Tq + Tk),
            "flops": 4 * D * H * _blend_pairs(case)}
