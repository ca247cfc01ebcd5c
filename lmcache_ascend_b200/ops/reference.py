"""PyTorch / NumPy oracles of the native kernels.

Used (a) as the numerics reference of the GPU tests and (b) as the CPU
implementation when tensors live on the host (CPU-only deployments and the
CPU test tier).  They implement the same formats as the CUDA kernels:

* CacheGen (``cachegen_kernels.cu``): aligned power-of-two CDF with the code
  length in the low 4 bits of each entry, MSB-first prefix codes, decode
  from an inclusive prefix sum of stream lengths;
* RoPE delta re-rotation (``pos_kernels.cu``);
* slot maps from request lengths, rotary positions with cache writes, and the
  attention operators (``slot_kernels.cu``, ``rope_cache_kernels.cu``,
  ``prefix_attention.cu``, ``position_attention.cu``).
"""

from __future__ import annotations

import math
from typing import Any, Dict, List, Optional, Tuple

import numpy as np
import torch

MAX_BINS = 256


# ---------------------------------------------------------------------------
# CacheGen
# ---------------------------------------------------------------------------
def cdf_assign(counts: List[int]) -> List[int]:
    """Aligned CDF of one channel (exact mirror of ``cdf_assign`` in C++).

    Returns bins + 1 uint16 entries: ``(start & 0xFFF0) | code_len``; the
    last entry (0) stands for 0x10000.
    """
    bins = len(counts)
    if bins == 1:
        return [0, 0]
    total = sum(int(c) for c in counts)
    den = 2 * total + bins
    out = [0] * (bins + 1)
    pos = 0
    for s in range(bins):
        k = bins - s
        R = 65536 - pos
        if k == 1:
            w = R
        else:
            x = (2 * int(counts[s]) + 1) * 65536
            wd = 16
            while wd < 32768 and den * (2 * wd) <= x:
                wd <<= 1
            if wd < 32768 and 2 * x >= 3 * den * wd:
                wd <<= 1
            ed = wd.bit_length() - 1
            maxw = 32768 if pos == 0 else (pos & -pos)
            best_e, best_d = -1, 1 << 30
            e = 4
            while (1 << e) <= maxw:
                cand = 1 << e
                if cand >= R:
                    break
                rem = R - cand
                if bin(rem).count("1") <= k - 1 and (k - 1) <= rem // 16:
                    d = abs(e - ed)
                    if d < best_d or (d == best_d and e > best_e):
                        best_d, best_e = d, e
                e += 1
            w = (1 << best_e) if best_e >= 0 else 16
        length = 16 - (w.bit_length() - 1)
        out[s] = (pos & 0xFFF0) | length
        pos += w
    out[bins] = 0
    return out


def calculate_cdf_ref(symbols: torch.Tensor, n_bins: int) -> torch.Tensor:
    """symbols [L, T, C] uint8 -> int16 [L, C, n_bins + 1]."""
    s = symbols.detach().cpu().numpy().astype(np.int64)
    L, T, C = s.shape
    s = np.minimum(s, n_bins - 1)
    out = np.zeros((L, C, n_bins + 1), dtype=np.uint16)
    for l in range(L):
        for c in range(C):
            counts = np.bincount(s[l, :, c], minlength=n_bins)[:n_bins]
            out[l, c] = cdf_assign(counts.tolist())
    return torch.from_numpy(out.view(np.int16).copy())


def _code_tables(cdf_row: np.ndarray) -> Tuple[List[int], List[int]]:
    bins = len(cdf_row) - 1
    starts = [int(v) & 0xFFF0 for v in cdf_row[:bins]] + [65536]
    codes, lens = [], []
    for s in range(bins):
        w = starts[s + 1] - starts[s]
        if w <= 0:
            codes.append(0)
            lens.append(-1)
            continue
        e = w.bit_length() - 1
        ln = 16 - e
        lens.append(ln)
        codes.append(0 if ln == 0 else starts[s] >> (16 - ln))
    return codes, lens


def encode_ref(cdf: torch.Tensor, symbols: torch.Tensor, cap: int
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (bytes [L, C, cap] uint8, lengths [L, C] int32)."""
    c = cdf.detach().cpu().numpy().view(np.uint16) if cdf.dtype == torch.int16 else \
        cdf.detach().cpu().numpy().astype(np.int64).astype(np.uint16)
    s = symbols.detach().cpu().numpy().astype(np.int64)
    L, T, C = s.shape
    bins = c.shape[2] - 1
    out = np.zeros((L, C, cap), dtype=np.uint8)
    lens = np.zeros((L, C), dtype=np.int32)
    for l in range(L):
        for ch in range(C):
            codes, cl = _code_tables(c[l, ch])
            acc, nb, buf = 0, 0, bytearray()
            for t in range(T):
                sym = min(int(s[l, t, ch]), bins - 1)
                ln = cl[sym]
                if ln < 0:
                    raise ValueError(f"symbol {sym} has zero width in the CDF")
                acc = (acc << ln) | codes[sym]
                nb += ln
                while nb >= 8:
                    buf.append((acc >> (nb - 8)) & 0xFF)
                    nb -= 8
                    acc &= (1 << nb) - 1
            if nb:
                buf.append((acc << (8 - nb)) & 0xFF)
            n = min(len(buf), cap)
            out[l, ch, :n] = np.frombuffer(bytes(buf[:n]), dtype=np.uint8)
            lens[l, ch] = n
    return torch.from_numpy(out), torch.from_numpy(lens)


def decode_ref(cdf: torch.Tensor, bytestream: torch.Tensor, cum_lengths: torch.Tensor,
               num_tokens: int) -> torch.Tensor:
    """Inverse of ``encode_ref`` with concatenated streams -> [L, T, C] uint8."""
    c = cdf.detach().cpu().numpy().view(np.uint16) if cdf.dtype == torch.int16 else \
        cdf.detach().cpu().numpy().astype(np.int64).astype(np.uint16)
    b = bytestream.detach().cpu().numpy().astype(np.uint8).tobytes()
    cl = cum_lengths.detach().cpu().numpy().astype(np.int64).reshape(-1)
    L, C, bp1 = c.shape
    bins = bp1 - 1
    out = np.zeros((L, num_tokens, C), dtype=np.uint8)
    for l in range(L):
        for ch in range(C):
            idx = l * C + ch
            b0 = 0 if idx == 0 else int(cl[idx - 1])
            stream = b[b0:int(cl[idx])]
            starts = [int(v) & 0xFFF0 for v in c[l, ch, :bins]]
            lens = [int(v) & 0xF for v in c[l, ch, :bins]]
            bits = int.from_bytes(stream, "big") if stream else 0
            nbits = 8 * len(stream)
            pos = 0
            for t in range(num_tokens):
                # next 16 bits (zero padded)
                if pos >= nbits:
                    v = 0
                else:
                    sh = nbits - pos - 16
                    v = (bits >> sh) & 0xFFFF if sh >= 0 else (bits << -sh) & 0xFFFF
                lo, hi = 0, bins - 1
                while lo < hi:
                    mid = (lo + hi + 1) >> 1
                    if starts[mid] <= v:
                        lo = mid
                    else:
                        hi = mid - 1
                out[l, t, ch] = lo
                pos += lens[lo]
    return torch.from_numpy(out)


# ---------------------------------------------------------------------------
# RoPE delta re-rotation
# ---------------------------------------------------------------------------
def rope_delta_ref(old_pos: torch.Tensor, new_pos: torch.Tensor, key: torch.Tensor,
                   head_size: int, cos_sin_cache: torch.Tensor, is_neox: bool
                   ) -> torch.Tensor:
    """fp32 reference: rotate K from ``old_pos`` to ``new_pos`` (returns a copy)."""
    T = key.shape[0]
    k = key.reshape(T, -1, head_size).float().clone()
    rot = cos_sin_cache.shape[1]
    half = rot // 2
    cs = cos_sin_cache.float()
    cn, sn = cs[new_pos.long(), :half], cs[new_pos.long(), half:]
    co, so = cs[old_pos.long(), :half], cs[old_pos.long(), half:]
    cd = (cn * co + sn * so)[:, None, :]
    sd = (sn * co - cn * so)[:, None, :]
    if is_neox:
        x1, x2 = k[..., :half].clone(), k[..., half:rot].clone()
        k[..., :half] = x1 * cd - x2 * sd
        k[..., half:rot] = x2 * cd + x1 * sd
    else:
        x1, x2 = k[..., 0:rot:2].clone(), k[..., 1:rot:2].clone()
        k[..., 0:rot:2] = x1 * cd - x2 * sd
        k[..., 1:rot:2] = x2 * cd + x1 * sd
    return k.reshape(key.shape)


def rope_apply_ref(pos: torch.Tensor, key: torch.Tensor, head_size: int,
                   cos_sin_cache: torch.Tensor, is_neox: bool) -> torch.Tensor:
    """Plain RoPE at ``pos`` (fp32): rotation from position 0."""
    zero = torch.zeros_like(pos)
    return rope_delta_ref(zero, pos, key, head_size, cos_sin_cache, is_neox)


def make_cos_sin_cache(max_pos: int, rot_dim: int, base: float = 10000.0,
                       dtype=torch.float32) -> torch.Tensor:
    """vLLM layout: [max_pos, rot_dim], first half cos, second half sin."""
    inv = 1.0 / (base ** (torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim))
    t = torch.arange(max_pos, dtype=torch.float64)
    f = torch.outer(t, inv)
    return torch.cat([f.cos(), f.sin()], dim=-1).to(dtype)


_ROPE_KEYS = {
    "default": {"factor", "original_max_position_embeddings"},  # of no effect
    "linear": {"factor", "original_max_position_embeddings"},
    "dynamic": {"factor", "original_max_position_embeddings"},
    "llama3": {"factor", "original_max_position_embeddings", "low_freq_factor",
               "high_freq_factor"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate",
             "attention_factor", "mscale", "mscale_all_dim"},
}


def make_scaled_cos_sin_cache(max_pos: int, rot_dim: int, base: float = 10000.0,
                              scaling: Optional[Dict[str, Any]] = None,
                              dtype=torch.float32) -> torch.Tensor:
    """``make_cos_sin_cache`` with the frequencies scaled for long contexts;
    angles in 64 bits.  ``scaling`` is a ``rope_scaling`` dict:

    * ``linear``: every frequency divided by ``factor``;
    * ``dynamic``: the base grown so that ``max_pos`` positions keep the slowest
      turn of ``original_max_position_embeddings`` (``factor`` times as many);
    * ``llama3``: frequencies of more than ``high_freq_factor`` turns over the
      original context kept, of fewer than ``low_freq_factor`` divided by
      ``factor``, a ramp between;
    * ``yarn``: a ramp over the dimensions between ``beta_fast`` and ``beta_slow``
      turns (rounded outwards unless ``truncate`` is false), and a gain on the
      cosines and sines: ``attention_factor``, or with ``mscale`` and
      ``mscale_all_dim`` the quotient of 0.1 m ln(factor) + 1 for each, or that for
      m = 1.

    A key that would change the table and is not known here is refused.
    """
    scaling = dict(scaling or {})
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    unknown = {k for k, v in scaling.items() if v is not None} - _ROPE_KEYS.get(kind, set()) \
        - {"rope_type", "type", "rope_theta"}
    if kind in _ROPE_KEYS and unknown:
        raise ValueError(f"{kind} rope scaling does not know {sorted(unknown)}")
    if float(scaling.get("rope_theta") or base) != float(base):
        raise ValueError(f"rope_theta {scaling['rope_theta']} is not the base {base}")
    dims = torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim
    gain = 1.0
    if kind == "default":
        inv = 1.0 / base ** dims
    elif kind == "linear":
        inv = base ** -dims / float(scaling["factor"])
    elif kind == "dynamic":
        f, orig = float(scaling["factor"]), int(scaling["original_max_position_embeddings"])
        if rot_dim <= 2:
            raise ValueError("dynamic rope scaling needs a rotated part of more than one pair")
        grown = base * max(1.0, f * max_pos / orig - (f - 1)) ** (rot_dim / (rot_dim - 2))
        inv = grown ** -dims
    elif kind == "llama3":
        f, orig = float(scaling["factor"]), int(scaling["original_max_position_embeddings"])
        lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        inv = base ** -dims
        turns = orig * inv / (2 * math.pi)
        ramp = ((turns - lo) / (hi - lo)).clamp(0, 1) if hi > lo else (turns >= hi).double()
        inv = inv / f * (1 - ramp) + inv * ramp
    elif kind == "yarn":
        f, orig = float(scaling["factor"]), int(scaling["original_max_position_embeddings"])

        def dim_of(turns: float) -> float:
            return rot_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = dim_of(float(scaling.get("beta_fast") or 32.0))
        hi = dim_of(float(scaling.get("beta_slow") or 1.0))
        if scaling.get("truncate") in (None, True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rot_dim - 1)
        ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo)
                / max(hi - lo, 0.001)).clamp(0, 1)
        inv = base ** -dims
        inv = inv / f * ramp + inv * (1 - ramp)

        def gain_of(m: float) -> float:
            return 0.1 * m * math.log(f) + 1.0 if f > 1 else 1.0

        m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        if scaling.get("attention_factor") is not None:
            gain = float(scaling["attention_factor"])
        elif m and m_all:
            gain = gain_of(float(m)) / gain_of(float(m_all))
        else:
            gain = gain_of(1.0)
    else:
        raise ValueError(f"unknown rope scaling {kind!r}")
    a = torch.outer(torch.arange(max_pos, dtype=torch.float64), inv)
    return (torch.cat([a.cos(), a.sin()], dim=-1) * gain).to(dtype)


# ---------------------------------------------------------------------------
# Serving operators next to the cache
# ---------------------------------------------------------------------------
def build_slot_mapping_ref(context_lens, new_lens, block_tables, block_size, num_tokens,
                           free_blocks=None, num_blocks=None, dtype=torch.int64):
    """One request after the other; grows ``block_tables`` in place.  Returns
    (slots, positions, request ids, query_start_loc, seq_lens, taken)."""
    ctx = [max(0, int(c)) for c in context_lens]
    new = [max(0, int(n)) for n in new_lens]
    free = None if free_blocks is None else [int(x) for x in free_blocks]
    limit = (1 << 31) - 1 if num_blocks is None else num_blocks
    width = block_tables.shape[1]
    slots = torch.full((num_tokens,), -1, dtype=dtype)
    positions = torch.zeros(num_tokens, dtype=dtype)
    ids = torch.full((num_tokens,), -1, dtype=torch.int32)
    start, taken = [0], [0]
    for b, (c, n) in enumerate(zip(ctx, new)):
        have, need = -(-c // block_size), -(-(c + n) // block_size)
        got = 0
        if free is not None:
            for j in range(need - have):
                at = taken[-1] + j
                if have + j < width:
                    block_tables[b, have + j] = free[at] if at < len(free) else -1
            got = need - have
        for i in range(n):
            t = start[-1] + i
            if t >= num_tokens:
                break
            p = c + i
            col = p // block_size
            page = int(block_tables[b, col]) if col < width else -1
            if 0 <= page < limit:
                slots[t] = page * block_size + p % block_size
            positions[t] = p
            ids[t] = b
        start.append(start[-1] + n)
        taken.append(taken[-1] + got)
    i32 = torch.int32
    return (slots, positions, ids, torch.tensor(start, dtype=i32),
            torch.tensor([c + n for c, n in zip(ctx, new)], dtype=i32),
            torch.tensor(taken, dtype=i32))


def rotary_embedding_ref(positions, x, head_size, cos_sin_cache, is_neox, compute=torch.float32):
    """Rows x [T, heads * D] or [T, heads, D] rotated by the table rows of
    ``positions``; rows whose position is outside the table are zero.  In
    ``compute``, not rounded."""
    T, rot = positions.numel(), cos_sin_cache.shape[1]
    half = rot // 2
    ok = (positions >= 0) & (positions < cos_sin_cache.shape[0])
    cs = cos_sin_cache.to(compute)[positions.long() * ok]
    c, s = cs[:, None, :half], cs[:, None, half:]
    y = x.reshape(T, -1, head_size).to(compute).clone()
    first = slice(0, half) if is_neox else slice(0, rot, 2)
    second = slice(half, rot) if is_neox else slice(1, rot, 2)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    y[~ok] = 0
    return y.reshape(x.shape)


def write_cache_ref(positions, rows, cache, slot_mapping, max_pos):
    """Rows [T, KH, D] to their slots of a [NB, BS, KH, D] cache; rows of slot
    -1 or of a position outside the table stay out."""
    bs = cache.shape[1]
    sm = slot_mapping.long()
    keep = (sm >= 0) & (sm < cache.shape[0] * bs) & (positions >= 0) & (positions < max_pos)
    cache[sm[keep] // bs, sm[keep] % bs] = rows.reshape(
        rows.shape[0], cache.shape[2], cache.shape[3])[keep].to(cache.dtype)


def attend_ref(q, k, v, visible, distance, scale, softcap, slopes):
    """q [H, R, D] over k, v [KH, N, D] (already in the type to compute in);
    ``visible`` and ``distance`` [R, N].  Keys that a row does not see take no
    part.  Returns (o [H, R, D], lse [H, R]); a row without keys is 0, -inf."""
    H, R, D = q.shape
    rep = H // k.shape[0]
    o = torch.zeros_like(q)
    lse = torch.full((H, R), -math.inf, dtype=q.dtype)
    for h in range(H):
        x = (q[h] @ k[h // rep].T) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        if slopes is not None:
            x = x - slopes[h].to(q.dtype) * distance.to(q.dtype)
        x = torch.where(visible, x, torch.full_like(x, -math.inf))
        some = visible.any(dim=1)
        m = x.amax(dim=1, keepdim=True) if x.shape[1] else x.new_full((R, 1), -math.inf)
        w = torch.exp(x - torch.where(some[:, None], m, torch.zeros_like(m)))
        total = w.sum(dim=1)
        y = w @ v[h // rep]
        for r in torch.nonzero(~torch.isfinite(y).all(dim=1)).flatten().tolist():
            sel = visible[r]  # a key it does not see holds an inf or NaN
            y[r] = w[r, sel] @ v[h // rep][sel]
        o[h] = torch.where(some[:, None], y / total[:, None], torch.zeros_like(y))
        lse[h] = torch.where(some, m[:, 0] + torch.log(total), lse[h])
    return o, lse


def shared_prefix_attention_ref(query, key_cache, value_cache, prefix_blocks, prefix_len,
                                block_tables, seq_lens, scale, softcap=0.0, alibi_slopes=None,
                                compute=torch.float32):
    """Oracle of ``api.shared_prefix_attention`` in ``compute``, not rounded."""
    q4 = query.unsqueeze(1) if query.dim() == 3 else query
    B, Tq, H, D = q4.shape
    NB, bs = key_cache.shape[0], key_cache.shape[1]
    out = torch.zeros(B, Tq, H, D, dtype=compute)
    lse = torch.full((B, Tq, H), -math.inf, dtype=compute)
    for b in range(B):
        n = max(0, int(seq_lens[b]))
        cols = min(-(-n // bs), block_tables.shape[1])
        page = torch.cat([prefix_blocks[:-(-prefix_len // bs)].long().repeat_interleave(bs)[
            :prefix_len], block_tables[b, :cols].long().repeat_interleave(bs)[:n]])
        off = torch.cat([torch.arange(prefix_len) % bs, torch.arange(min(n, cols * bs)) % bs])
        ok = (page >= 0) & (page < NB)
        k = key_cache[page * ok, off].to(compute).transpose(0, 1)
        v = value_cache[page * ok, off].to(compute).transpose(0, 1)
        at = torch.arange(page.numel())
        i = torch.arange(Tq)[:, None]
        visible = ok[None] & ((at < prefix_len) | (at - prefix_len <= n - Tq + i))
        distance = (prefix_len + n - Tq + i - at).abs()
        o, e = attend_ref(q4[b].to(compute).transpose(0, 1), k, v, visible, distance, scale,
                          softcap, alibi_slopes)
        out[b], lse[b] = o.transpose(0, 1), e.T
    return out.reshape(query.shape), lse.reshape(query.shape[:-1])


def position_attention_ref(query, key, value, q_positions, k_positions, scale, softcap=0.0,
                           alibi_slopes=None, q_documents=None, k_documents=None,
                           q_prefix_lens=None, causal=True, compute=torch.float32):
    """Oracle of ``api.position_attention`` in ``compute``, not rounded."""
    qp = q_positions.long()
    kp = torch.arange(key.shape[0]) if k_positions is None else k_positions.long()
    limit = qp + 1 if causal else torch.full_like(qp, 1 << 40)  # no row is that far
    if q_prefix_lens is not None:
        limit = torch.maximum(limit, q_prefix_lens.long())
    visible = kp[None] < limit[:, None]
    if q_documents is not None:
        visible &= (q_documents[:, None] == k_documents[None]) & (q_documents[:, None] >= 0)
    o, e = attend_ref(query.to(compute).transpose(0, 1), key.to(compute).transpose(0, 1),
                      value.to(compute).transpose(0, 1), visible,
                      (qp[:, None] - kp[None]).abs(), scale, softcap, alibi_slopes)
    return o.transpose(0, 1), e.T
