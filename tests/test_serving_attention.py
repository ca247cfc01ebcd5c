"""Attention next to the cache: the oracles against a row at a time, the
kernels against the oracles in 64 bits.

Tolerance of an output element, for weights p (sum 1) and values v, with
e = eps / 2 of the type (half a step):

* the weights are rounded to the type before the product: e * sum p|v|;
* the scores are fp32 sums of exact products: off by at most
  dx = D 2^-23 * scale * max sum_d |q_d k_d| (plus 2^-22 of the largest shaped
  score, and 2^-20 of the cap or, below it, the largest score), which scales a weight and the sum: 2 dx sum p|v|;
* exponentials, fp32 sums and joins of partial results: 2^-16 sum p|v|;
* float16 weights below the normal range: 2^-25 per key, times max|v|;
* the result's own rounding: e |o| (and 2^-25 below float16's normal range).

The log of the sum is off by at most dx + 2^-18 (1 + |lse|).
"""

import math

import pytest
import torch

from lmcache_ascend_b200 import ops
from lmcache_ascend_b200.ops import api
from lmcache_ascend_b200.ops import reference as R

BF, FP = torch.bfloat16, torch.float16


def _bounds(ref, q, k, v, dtype, scale, softcap, slopes, reach):
    """(o, lse, tolerance of o, of lse); ``ref(q, k, v)`` is the oracle."""
    o, lse = ref(q, k, v)
    a, _ = ref(q, k, v.abs())
    fin = lambda x: torch.nan_to_num(x.double(), 0.0, 0.0, 0.0).abs()
    D = q.shape[-1]
    reachable = scale * float((fin(q).amax(dim=tuple(range(q.dim() - 1)))
                               * fin(k).amax(dim=tuple(range(k.dim() - 1)))).sum())
    top = min(reachable, softcap or reachable)
    if slopes is not None:
        top += float(slopes.abs().max()) * reach
    dx = D * 2.0 ** -23 * reachable + 2.0 ** -22 * top + 2.0 ** -20 * min(softcap, reachable)
    e = torch.finfo(dtype).eps / 2
    n_keys = reach + 1
    tol = (e + 2 * dx + 2.0 ** -16) * a + e * o.abs() + 1e-30
    if dtype == FP:
        tol = tol + n_keys * 2.0 ** -25 * float(fin(v).max()) + 2.0 ** -25
    return o, lse, tol, dx + 2.0 ** -18 * (1 + torch.nan_to_num(lse, 0.0, 0.0, 0.0).abs())


def _check(got, got_lse, o, lse, tol, tol_lse):
    g = got.cpu().double()
    assert bool(torch.isfinite(g).all())
    err = (g - o).abs()
    assert bool((err <= tol).all()), f"off by {float((err - tol).max())} over the tolerance"
    gl = got_lse.cpu().double()
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(gl) & (gl < 0), empty)
    assert bool(((gl - lse).abs()[~empty] <= tol_lse[~empty]).all())
    assert bool((g[empty] == 0).all())


def _slopes(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)])


# ------------------------------------------------------------------ oracles
def test_prefix_oracle_is_plain_attention_over_the_joined_keys():
    B, Tq, H, KH, D, bs, P = 3, 2, 4, 2, 8, 4, 6
    g = torch.Generator().manual_seed(0)
    kc, vc = torch.randn(2, 20, bs, KH, D, generator=g, dtype=torch.float64)
    q = torch.randn(B, Tq, H, D, generator=g, dtype=torch.float64)
    prefix = torch.tensor([3, 9], dtype=torch.int32)
    tables = torch.tensor([[0, 1], [2, 4], [5, 6]], dtype=torch.int32)
    lens = [2, 7, 5]
    o, lse = R.shared_prefix_attention_ref(q, kc, vc, prefix, P, tables, lens, 0.3, 5.0,
                                           _slopes(H), torch.float64)
    for b, n in enumerate(lens):
        rows = [(int(prefix[t // bs]), t % bs) for t in range(P)]
        rows += [(int(tables[b, t // bs]), t % bs) for t in range(n)]
        for i in range(Tq):
            p = P + n - Tq + i
            for h in range(H):
                x = []
                for j, (pg, off) in enumerate(rows[:p + 1]):
                    s = 0.3 * float(q[b, i, h] @ kc[pg, off, h // 2])
                    x.append(5 * math.tanh(s / 5) - float(_slopes(H)[h]) * (p - j))
                w = torch.tensor(x, dtype=torch.float64).softmax(0)
                want = sum(w[j] * vc[pg, off, h // 2] for j, (pg, off) in enumerate(rows[:p + 1]))
                assert torch.allclose(o[b, i, h], want)
                assert abs(float(lse[b, i, h])
                           - float(torch.logsumexp(torch.tensor(x, dtype=torch.float64), 0))) < 1e-9


def test_position_oracle_masks():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(5, 2, 8, generator=g, dtype=torch.float64) for _ in range(3))
    pos = torch.tensor([0, 1, 0, 1, 2])
    doc = torch.tensor([0, 0, 1, 1, -1], dtype=torch.int32)
    v[4] = math.nan
    o, lse = R.position_attention_ref(q, k, v, pos, pos, 0.5, q_documents=doc, k_documents=doc,
                                      compute=torch.float64)
    assert torch.allclose(o[0], v[0]) and torch.allclose(o[2], v[2])
    w = torch.stack([(0.5 * q[3, 0] @ k[j, 0]) for j in (2, 3)]).softmax(0)
    assert torch.allclose(o[3, 0], w[0] * v[2, 0] + w[1] * v[3, 0])
    assert bool((o[4] == 0).all()) and bool(torch.isinf(lse[4]).all())
    o2, _ = R.position_attention_ref(q[:4], k[:4], v[:4], pos[:4], pos[:4], 0.5,
                                     q_prefix_lens=torch.tensor([2, 0, 0, 0], dtype=torch.int32),
                                     compute=torch.float64)
    w = (0.5 * k[:4, 0] @ q[0, 0]).softmax(0)
    assert torch.allclose(o2[0, 0], w @ v[:4, 0])


def test_cpu_forms_and_refusals():
    q, kc = torch.randn(2, 4, 8), torch.randn(3, 4, 2, 8)
    one = torch.zeros(1, dtype=torch.int32)
    t, n = torch.tensor([[1], [2]], dtype=torch.int32), torch.tensor([1, 3], dtype=torch.int32)
    out, lse = api.shared_prefix_attention(q, kc, kc, one, 4, t, n, return_lse=True)
    assert out.shape == q.shape and lse.shape == (2, 4) and out.dtype == q.dtype
    for bad in (dict(scale=0.0), dict(softcap=-1.0), dict(prefix_len=5), dict(prefix_len=-1), dict(query=q[0]), dict(query=q[:, :3])):
        kw = dict(query=q, key_cache=kc, value_cache=kc, prefix_blocks=one, prefix_len=4,
                  block_tables=t, seq_lens=n)
        with pytest.raises(ValueError):
            api.shared_prefix_attention(**{**kw, **bad})
    k = torch.randn(5, 2, 8)
    assert api.position_attention(q, k, k, torch.tensor([0, 4])).shape == q.shape
    with pytest.raises(ValueError):
        api.position_attention(q, k, k, torch.tensor([0, 4]), q_documents=one)
    with pytest.raises(ValueError):
        api.position_attention(q[0], k, k, torch.tensor([0, 4]))


@pytest.mark.skipif(not ops.native_available(), reason="native module not built")
def test_part_whose_wait_ran_out_is_not_taken_for_an_empty_one():
    """A join leaves parts of -inf out; a NaN makes it compute the row again."""
    log = ops.native().log2_of_sum
    assert log(True, -math.inf, 0.0) == -math.inf
    assert log(True, 3.0, 0.25) == 1.0
    assert math.isnan(log(True, -math.inf, 0.25))  # scores of -inf only
    for m, l in ((-math.inf, 0.0), (3.0, 0.25), (3.0, 0.0)):
        assert math.isnan(log(False, m, l))


def test_cpu_forms_refuse_marks_that_do_not_fit():
    """What would be broadcast, or compared as a fraction."""
    q, k = torch.randn(2, 4, 8), torch.randn(5, 2, 8)
    p = torch.tensor([0, 4])
    for bad in (dict(q_positions=p.float()), dict(q_positions=p[:1]),
                dict(k_positions=torch.tensor([3])), dict(k_positions=torch.arange(5) / 2),
                dict(q_prefix_lens=torch.tensor([1])), dict(alibi_slopes=torch.ones(6)),
                dict(q_documents=p[:1].int(), k_documents=torch.zeros(5, dtype=torch.int32))):
        with pytest.raises(ValueError):
            api.position_attention(**{**dict(query=q, key=k, value=k, q_positions=p), **bad})
    kc, one = torch.randn(3, 4, 2, 8), torch.zeros(1, dtype=torch.int32)
    kw = dict(query=q, key_cache=kc, value_cache=kc, prefix_blocks=one, prefix_len=4,
              block_tables=torch.tensor([[1], [2]], dtype=torch.int32),
              seq_lens=torch.tensor([1, 3], dtype=torch.int32))
    for bad in (dict(seq_lens=torch.tensor([1, 3, 2])), dict(block_tables=kw["block_tables"][:1]),
                dict(alibi_slopes=torch.ones(5))):
        with pytest.raises(ValueError):
            api.shared_prefix_attention(**{**kw, **bad})


# Scales and caps that fp32 does not hold: infinite, or zero and so no cap at all.
OUT_OF_FP32 = [dict(scale=1e300), dict(scale=1e39), dict(scale=1e-50), dict(softcap=1e39),
               dict(softcap=1e-50), dict(softcap=math.inf), dict(softcap=math.nan),
               dict(scale=1e20, softcap=1e-20)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_scores_outside_of_fp32_are_refused(device):
    q, k, v, qp, kp, _ = (x.to(device) if isinstance(x, torch.Tensor) else x
                          for x in _position_case(8, 30, 4, 2, 64, BF, "subset"))
    p = [x.to(device) for x in _prefix_case(2, 1, 4, 2, 64, 16, 32, [3, 4], BF)]
    for kw in OUT_OF_FP32:
        with pytest.raises((ValueError, RuntimeError)):
            api.position_attention(q, k, v, qp, kp, **kw)
        with pytest.raises((ValueError, RuntimeError)):
            api.shared_prefix_attention(p[0], p[1], p[2], p[3], 32, p[4], p[5], **kw)
    # at the borders: a cap far below the scores is a mean of the values seen
    for kw in (dict(softcap=1e-20), dict(scale=1e-37), dict(scale=1.0, softcap=1e38)):
        want = R.position_attention_ref(q.cpu(), k.cpu(), v.cpu(), qp.cpu(), kp.cpu(),
                                        kw.get("scale", 0.125), kw.get("softcap", 0.0),
                                        compute=torch.float64)[0]
        got = api.position_attention(q, k, v, qp, kp, **kw).cpu().double()
        # weights and result rounded to 8 bits, |v| below 5
        assert bool(((got - want).abs() <= 2 * 2.0 ** -8 * 5).all())


# ------------------------------------------------------------ shared prefix
def _prefix_case(B, Tq, H, KH, D, bs, P, own, dtype, seed=0, layout="plain", junk=math.nan):
    """A paged batch whose unused slots hold ``junk``."""
    g = torch.Generator().manual_seed(seed)
    npb = -(-P // bs)
    nob = [-(-max(0, n) // bs) for n in own]
    nb = npb + sum(nob) + 2
    kc = torch.full((nb, bs, KH, D), junk, dtype=dtype)
    vc = torch.full((nb, bs, KH, D), junk, dtype=dtype)
    ids = torch.randperm(nb, generator=g).int()
    tables = torch.full((B, max([1] + nob) + 1), -7, dtype=torch.int32)

    def fill(pages, n):
        if n <= 0:
            return
        t = torch.arange(n)
        for c in (kc, vc):
            c[pages.long()[t // bs], t % bs] = torch.randn(n, KH, D, generator=g).to(dtype)

    fill(ids[:npb], P)
    at = npb
    for b, n in enumerate(own):
        tables[b, :nob[b]] = ids[at:at + nob[b]]
        fill(ids[at:at + nob[b]], n)
        at += nob[b]
    q = (torch.randn(B, Tq, H, D, generator=g) * 2).to(dtype)
    if Tq == 1:
        q = q[:, 0]
    return q, kc, vc, ids[:npb].contiguous(), tables, torch.tensor(own, dtype=torch.int32)


def _on_device(kc, vc, layout):
    if layout == "plain":
        return kc.cuda(), vc.cuda()
    if layout == "merged":  # [2, NB, BS, KH, D] and [NB, 2, BS, KH, D]
        m = torch.stack([kc, vc], 1).cuda()
        return m[:, 0], m[:, 1]
    h = torch.stack([kc.transpose(1, 2), vc.transpose(1, 2)]).contiguous().cuda()  # head-major
    return h[0].transpose(1, 2), h[1].transpose(1, 2)


PREFIX = [
    # B, Tq, H, KH, D, bs, P, own, dtype, softcap, slopes, layout
    (1, 1, 8, 2, 128, 16, 0, [1], BF, 0.0, False, "plain"),
    (3, 1, 4, 4, 64, 16, 0, [0, 5, 33], FP, 0.0, False, "plain"),
    (2, 1, 8, 1, 128, 16, 1, [0, 0], BF, 0.0, False, "plain"),
    (4, 1, 32, 8, 128, 16, 500, [1, 64, 17, 30], BF, 0.0, False, "plain"),
    (5, 3, 10, 2, 64, 32, 129, [3, 1, 40, 2, 77], FP, 0.0, True, "merged"),
    (7, 1, 7, 1, 128, 64, 255, [64, 1, 200, 0, 5, 130, 63], BF, 30.0, False, "heads"),
    (3, 5, 14, 2, 128, 128, 384, [5, 6, 300], FP, 50.0, True, "plain"),
    (2, 1, 4, 2, 64, 1, 37, [3, 9], BF, 0.0, False, "plain"),
    (2, 2, 4, 2, 128, 24, 100, [30, 2], FP, 20.0, False, "plain"),
    (33, 4, 16, 2, 128, 64, 1000, [4 + 7 * i for i in range(33)], FP, 30.0, False, "plain"),
    (64, 1, 32, 4, 128, 16, 2049, [1 + 5 * i for i in range(64)], BF, 0.0, False, "plain"),
    (70, 2, 8, 1, 64, 32, 1500, [2 + i % 9 for i in range(70)], BF, 0.0, True, "heads"),
    (40, 1, 56, 8, 64, 128, 700, [1 + i for i in range(40)], FP, 0.0, False, "merged"),
    (130, 1, 8, 8, 128, 256, 1111, [1 + i % 3 for i in range(130)], BF, 0.0, False, "plain"),
    (50, 1, 20, 2, 128, 8, 640, [i for i in range(50)], BF, 10.0, True, "plain"),
    (1, 1, 8, 2, 128, 16, 20, [9000], BF, 0.0, False, "plain"),
    # many heads on one KV head, not a multiple of the row tiles
    (3, 2, 96, 1, 64, 16, 200, [5, 6, 7], BF, 0.0, False, "plain"),
    (20, 1, 96, 1, 128, 64, 1500, [1 + i for i in range(20)], FP, 0.0, True, "heads"),
    # caps far above the scores, and below them
    (3, 1, 8, 2, 64, 16, 40, [7, 8, 9], FP, 1e6, False, "plain"),
    (80, 1, 16, 1, 64, 16, 3057, [3] * 80, FP, 1e5, False, "plain"),
    (80, 1, 16, 1, 128, 16, 2000, [3] * 80, FP, 1.0, True, "plain"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PREFIX, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_prefix_kernel(case):
    B, Tq, H, KH, D, bs, P, own, dtype, cap, bias, layout = case
    q, kc, vc, prefix, tables, lens = _prefix_case(B, Tq, H, KH, D, bs, P, own, dtype)
    slopes = _slopes(H) if bias else None
    scale = D ** -0.5

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, scale, cap,
                                             slopes, torch.float64)

    want = _bounds(ref, q, kc, vc, dtype, scale, cap, slopes, P + max(own))
    dk, dv = _on_device(kc, vc, layout)
    st = ops.DeviceStatus("cuda")
    args = (prefix.cuda(), P, tables.cuda(), lens.cuda())
    kw = dict(softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda())
    got, lse = api.shared_prefix_attention(q.cuda(), dk, dv, *args, return_lse=True,
                                           status=st.tensor, **kw)
    assert got.shape == q.shape and got.dtype == dtype
    _check(got, lse, *want)
    st.check()
    again = api.shared_prefix_attention(q.cuda(), dk, dv, *args, **kw)
    assert torch.equal(again, got)  # no order of atomics in the result


@pytest.mark.gpu
@pytest.mark.parametrize("B,P", [(3, 300), (80, 1200)])
def test_prefix_kernel_bad_pages_are_left_out_and_reported(B, P):
    H, KH, D, bs = 8, 1, 128, 16
    own = [20 + i % 30 for i in range(B)]
    q, kc, vc, prefix, tables, lens = _prefix_case(B, 1, H, KH, D, bs, P, own, BF)
    prefix[3], prefix[7] = -1, 1 << 30
    tables[1, 0] = kc.shape[0]
    lens[2] = 10 ** 6  # past the end of its table row
    tables[2] = int(prefix[0])  # every column a block that holds keys

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, 0.1,
                                             compute=torch.float64)

    want = _bounds(ref, q, kc, vc, BF, 0.1, 0.0, None, P + 100)
    st = ops.DeviceStatus("cuda")
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), P,
                                           tables.cuda(), lens.cuda(), scale=0.1, return_lse=True,
                                           status=st.tensor)
    _check(got, lse, *want)
    assert st.read()["name"] in ("bad_slot", "bad_index")


@pytest.mark.gpu
def test_inputs_that_ask_for_gradients_are_refused():
    q, k, v, qp, kp, _ = _position_case(8, 30, 4, 2, 64, BF, "subset")
    d = [x.cuda() for x in (q, k, v, qp, kp)]
    for i in range(3):
        g = list(d)
        g[i] = d[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="forward only"):
            api.position_attention(*g)
        with torch.no_grad():
            api.position_attention(*g)


@pytest.mark.gpu
def test_no_gradient_is_lost_without_a_word():
    """Slopes and caches that ask for gradients, and forward tangents of any input."""
    q, k, v, qp, kp, _ = _position_case(8, 30, 4, 2, 64, BF, "subset")
    d = [x.cuda() for x in (q, k, v, qp, kp)]
    slopes = _slopes(4).cuda()
    p = [x.cuda() for x in _prefix_case(2, 1, 4, 2, 64, 16, 32, [3, 4], BF)]

    def dense(q_=d[0], k_=d[1], v_=d[2], s_=slopes):
        return api.position_attention(q_, k_, v_, d[3], d[4], alibi_slopes=s_)

    def paged(q_=p[0], k_=p[1], v_=p[2], s_=slopes):
        return api.shared_prefix_attention(q_, k_, v_, p[3], 32, p[4], p[5], alibi_slopes=s_)

    for call, tensors in ((dense, d[:3]), (paged, p[:3])):
        want = call()
        for name, t in zip(("q_", "k_", "v_", "s_"), tensors + [slopes]):
            leaf = t.clone().requires_grad_()
            with pytest.raises(RuntimeError, match="forward only"):
                call(**{name: leaf})
            with torch.no_grad():
                assert torch.equal(call(**{name: leaf}), want)
            with torch.autograd.forward_ad.dual_level():
                dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
                with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                    call(**{name: dual})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,value", [(BF, torch.finfo(BF).min), (FP, torch.finfo(FP).min),
                                         (BF, math.inf)])
def test_prefix_kernel_unused_slots_hold_anything(dtype, value):
    q, kc, vc, prefix, tables, lens = _prefix_case(40, 2, 8, 1, 64, 16, 1000,
                                                   [2 + i for i in range(40)], dtype, junk=value)

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, 1000, tables, lens, 0.125,
                                             compute=torch.float64)

    o, e, tol, tl = _bounds(ref, q, torch.where(kc.float().abs() > 100, torch.zeros_like(kc), kc),
                            torch.where(vc.float().abs() > 100, torch.zeros_like(vc), vc), dtype,
                            0.125, 0.0, None, 1100)
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), 1000,
                                           tables.cuda(), lens.cuda(), scale=0.125,
                                           return_lse=True)
    _check(got, lse, o, e, tol, tl)


@pytest.mark.gpu
def test_prefix_kernel_large_scores_and_nan_keys_stay_in_their_rows():
    # scores far above and below others: no overflow; a NaN key of one request
    # stays in that request
    q, kc, vc, prefix, tables, lens = _prefix_case(48, 1, 8, 1, 128, 16, 600, [40] * 48, BF)
    kc[prefix.long()[2]] *= 100
    bad = int(tables[5, 0])
    kc[bad, 3] = math.nan

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, 600, tables, lens, 1.0,
                                             compute=torch.float64)

    clean = kc.clone()
    clean[bad, 3] = 0
    o, e, tol, tl = _bounds(ref, q, clean, vc, BF, 1.0, 0.0, None, 640)
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), 600,
                                           tables.cuda(), lens.cuda(), scale=1.0, return_lse=True)
    assert bool(torch.isnan(got[5]).all())
    keep = [b for b in range(48) if b != 5]
    _check(got[keep], lse[keep], o[keep], e[keep], tol[keep], tl[keep])


@pytest.mark.gpu
def test_prefix_kernel_refusals():
    q, kc, vc, prefix, tables, lens = (x.cuda() for x in _prefix_case(
        2, 1, 4, 2, 64, 16, 32, [3, 4], BF))
    good = dict(query=q, key_cache=kc, value_cache=vc, prefix_blocks=prefix, prefix_len=32,
                block_tables=tables, seq_lens=lens)
    api.shared_prefix_attention(**good)
    assert api.shared_prefix_attention(**{**good, "query": q[:0], "seq_lens": lens[:0]}).numel() == 0
    for bad in (dict(query=q.float(), key_cache=kc.float(), value_cache=vc.float()),
                dict(query=q[..., :32], key_cache=kc[..., :32], value_cache=vc[..., :32]),
                dict(query=q[:, :3]), dict(query=q.half()), dict(query=q[0, 0]),
                dict(key_cache=kc.cpu()), dict(value_cache=vc[:, :8]),
                dict(value_cache=vc.transpose(2, 3).contiguous().transpose(2, 3)),
                dict(prefix_len=33), dict(prefix_len=-1), dict(prefix_blocks=prefix.long()),
                dict(block_tables=tables[:1]), dict(block_tables=tables.long()),
                dict(seq_lens=lens[:1]), dict(seq_lens=lens.long()), dict(softcap=-1.0),
                dict(softcap=math.nan), dict(scale=math.inf), dict(scale=0.0), dict(scale=-1.0),
                dict(alibi_slopes=torch.zeros(3, device="cuda")),
                dict(alibi_slopes=torch.zeros(4, device="cuda").half()),
                dict(status=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises((RuntimeError, TypeError)):
            api.shared_prefix_attention(**{**good, **bad})
    flat = torch.zeros(kc.numel() + 1, dtype=BF, device="cuda")[1:].view(kc.shape)
    with pytest.raises(RuntimeError):
        api.shared_prefix_attention(**{**good, "key_cache": flat})


@pytest.mark.gpu
def test_prefix_kernel_captured_twice_replayed_with_other_lengths():
    B, P, own = 66, 777, [30] * 66
    q, kc, vc, prefix, tables, lens = _prefix_case(B, 1, 8, 2, 64, 16, P, own, BF, junk=0.0)
    d = [x.cuda() for x in (q, kc, vc, prefix, tables, lens)]

    def call():
        return api.shared_prefix_attention(d[0], d[1], d[2], d[3], P, d[4], d[5], return_lse=True)

    want = call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):  # both at once
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    d[5].copy_(torch.arange(B) % 31)
    want = call()
    torch.cuda.synchronize()
    for g, out in graphs:
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


# ---------------------------------------------------------------- positions
def _rand(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype)


POSITION = [
    # Tq, Tk, H, KH, D, dtype, softcap, slopes, kind
    (1, 1, 1, 1, 64, BF, 0.0, False, "causal"),
    (1, 0, 2, 1, 128, BF, 0.0, False, "causal"),
    (38, 257, 32, 8, 128, BF, 0.0, False, "subset"),
    (129, 129, 4, 4, 128, FP, 0.0, False, "causal"),
    (200, 700, 6, 2, 64, BF, 30.0, True, "subset"),
    (300, 300, 10, 2, 128, FP, 50.0, False, "documents"),
    (513, 513, 4, 2, 64, FP, 0.0, True, "documents"),
    (257, 640, 3, 1, 128, BF, 0.0, False, "shuffled"),
    (150, 385, 4, 1, 64, FP, 15.0, True, "shuffled"),
    (260, 260, 2, 2, 128, BF, 0.0, False, "prefix"),
    (140, 500, 4, 2, 128, FP, 0.0, True, "all"),
    (333, 333, 8, 8, 64, BF, 0.0, False, "padded"),
    (640, 1500, 5, 1, 128, BF, 20.0, False, "interleaved"),
    (1000, 1000, 2, 1, 128, FP, 0.0, False, "causal"),
    (5, 2993, 2, 2, 64, BF, 0.0, False, "subset"),
    (40, 300, 96, 1, 64, BF, 0.0, False, "subset"),
    (130, 700, 96, 1, 128, FP, 0.0, False, "shuffled"),
    # the same kinds again above the split kernel's sizes
    (1200, 2500, 8, 2, 64, BF, 0.0, True, "subset"),
    (2000, 2000, 6, 1, 128, FP, 30.0, True, "documents"),
    (1500, 1500, 7, 1, 64, BF, 0.0, False, "padded"),
    (1300, 1700, 8, 1, 128, FP, 5.0, True, "shuffled"),
    (1600, 1600, 8, 2, 128, BF, 0.0, True, "prefix"),
    (1100, 1900, 8, 4, 64, FP, 1e5, True, "all"),
]


def _position_case(Tq, Tk, H, KH, D, dtype, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = _rand(g, Tq, H, D, dtype=dtype) * 2
    k, v = _rand(g, Tk, KH, D, dtype=dtype), _rand(g, Tk, KH, D, dtype=dtype)
    kp, kw = torch.arange(Tk), {}
    rows = torch.arange(Tq) if Tq == Tk else torch.randperm(max(Tk, Tq), generator=g)[:Tq].sort()[0]
    kd = None
    if kind in ("documents", "padded", "prefix"):
        cuts = sorted(torch.randperm(Tk - 1, generator=g)[:6].add(1).tolist())
        lens = [b - a for a, b in zip([0] + cuts, cuts + [Tk])]
        kp = torch.cat([torch.arange(n) for n in lens])
        kd = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).int()
        if kind == "padded":
            kd[kd == len(lens) - 1] = -1
            kd[3] = -1
        if kind == "prefix":
            kw["q_prefix_lens"] = torch.full((Tq,), 20, dtype=torch.int32)
    if kind == "interleaved":
        kd = (torch.arange(Tk) % 3).int()
    qp = kp[rows.clamp(max=max(0, Tk - 1))] if Tk else rows
    qd = None if kd is None else kd[rows]
    if kind == "shuffled":
        perm = torch.randperm(Tk, generator=g)
        kp, k, v = kp[perm], k[perm], v[perm]
        qperm = torch.randperm(Tq, generator=g)
        qp = qp[qperm] - 3  # some rows before every key
    if kind == "all":
        kw["causal"] = False
    if kd is not None:
        kw.update(q_documents=qd, k_documents=kd)
    return q, k, v, qp, kp, kw


def _run_position(q, k, v, qp, kp, kw, dtype, cap, slopes, **more):
    to = {a: b.cuda() if isinstance(b, torch.Tensor) else b for a, b in kw.items()}
    return api.position_attention(q.cuda(), k.cuda(), v.cuda(), qp.cuda(),
                                  None if kp is None else kp.cuda(), softcap=cap,
                                  alibi_slopes=None if slopes is None else slopes.cuda(),
                                  return_lse=True, **to, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("case", POSITION, ids=lambda c: "-".join(str(x) for x in c[:5]) + c[8])
def test_position_kernel(case):
    Tq, Tk, H, KH, D, dtype, cap, bias, kind = case
    q, k, v, qp, kp, kw = _position_case(Tq, Tk, H, KH, D, dtype, kind)
    slopes = _slopes(H) if bias else None

    def ref(q_, k_, v_):
        return R.position_attention_ref(q_, k_, v_, qp, kp, D ** -0.5, cap, slopes,
                                        compute=torch.float64, **kw)

    want = _bounds(ref, q, k, v, dtype, D ** -0.5, cap, slopes, Tk + 3) if Tk else \
        (*ref(q, k, v), torch.zeros(Tq, H, D), torch.zeros(Tq, H))
    got, lse = _run_position(q, k, v, qp, kp, kw, dtype, cap, slopes)
    _check(got, lse, *want)
    # int32 positions, and rows that are slices of one projection: the same bits
    w = torch.zeros(max(Tq, Tk), (H + 2 * KH) * D + 8, dtype=dtype, device="cuda")
    w[:Tq, :H * D] = q.flatten(1).cuda()
    w[:Tk, H * D:(H + KH) * D] = k.flatten(1).cuda()
    w[:Tk, (H + KH) * D:(H + 2 * KH) * D] = v.flatten(1).cuda()
    s = [w[:n, a * D:b * D].unflatten(1, (-1, D)) for n, a, b in (
        (Tq, 0, H), (Tk, H, H + KH), (Tk, H + KH, H + 2 * KH))]
    got2, lse2 = _run_position(*s, qp.int(), kp.int(), kw, dtype, cap, slopes)
    assert torch.equal(got2, got) and torch.equal(lse2, lse)
    if kind == "causal":
        got3, _ = _run_position(q, k, v, qp, None, kw, dtype, cap, slopes)
        assert torch.equal(got3, got)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Tq,H,D,T", [(300, 2, 64, 300), (20, 4, 128, 300),
                                      (2200, 8, 64, 2200), (1000, 8, 128, 2200)])
def test_position_kernel_masked_keys_hold_anything(value, Tq, H, D, T):
    """A key or value of NaN or infinity reaches the rows that see it, no other."""
    q, k, v, qp, kp, kw = _position_case(Tq, T, H, 1, D, BF, "documents")
    clean_k, clean_v = k.clone(), v.clone()
    hit_k, hit_v = 77, 210
    k[hit_k] = math.nan
    v[hit_v, 0, 5] = value

    def ref(q_, k_, v_):
        return R.position_attention_ref(q_, k_, v_, qp, kp, D ** -0.5, compute=torch.float64, **kw)

    o, e, tol, tl = _bounds(ref, q, clean_k, clean_v, BF, D ** -0.5, 0.0, None, T)
    got, lse = _run_position(q, k, v, qp, kp, kw, BF, 0.0, None)
    qd, kd = kw["q_documents"], kw["k_documents"]
    sees = lambda j: (qd == kd[j]) & (kp[j] <= qp)
    a, b = sees(hit_k), sees(hit_v)
    assert bool(torch.isnan(got[a.cuda()]).all())
    if bool(b.any()):
        assert not bool(torch.isfinite(got[(b & ~a).cuda()][..., 5]).any())
        other = [d for d in range(D) if d != 5]
        r = b & ~a
        g = got.cpu().double()[r][..., other]
        assert bool(((g - o[r][..., other]).abs() <= tol[r][..., other]).all())
    keep = ~(a | b)
    _check(got[keep.cuda()], lse[keep.cuda()], o[keep], e[keep], tol[keep], tl[keep])


# Dense calls of every form: one part, parts joined in a cluster and in memory, the
# tensor-core kernel whole and in slices.
FORMS = [(20, 200, 8, 2, 64), (20, 300, 4, 2, 128), (1, 6000, 4, 2, 64), (400, 700, 16, 2, 128),
         (500, 850, 16, 2, 64), (300, 3000, 16, 2, 64)]
# ... and paged: B, Tq, H, KH, D, P
PAGED_FORMS = [(3, 1, 8, 2, 64, 20), (2, 1, 8, 2, 64, 500), (1, 1, 8, 2, 128, 6000),
               (30, 1, 32, 2, 128, 1000), (40, 1, 32, 2, 64, 1700), (40, 1, 32, 2, 128, 1200)]


def _check_with_nan(got, lse, want):
    """NaN exactly where the oracle has it, the others within the tolerance."""
    o, e, tol, tl = want
    hit = torch.isnan(e)
    assert torch.equal(torch.isnan(lse.cpu()), hit)
    assert bool(torch.isnan(got.cpu()[hit]).all())
    _check(got.cpu()[~hit], lse.cpu()[~hit], o[~hit], e[~hit], tol[~hit], tl[~hit])
    return hit


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["query", "first key"])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_position_kernel_nan_scores_reach_their_rows(form, where):
    Tq, Tk, H, KH, D = form
    q, k, v, qp, kp, kw = _position_case(Tq, Tk, H, KH, D, BF, "subset")
    if where == "query":
        q[Tq // 2, 1, 5] = math.nan
    else:
        k[0, 0, 7] = math.nan  # every row sees key 0

    def ref(q_, k_, v_):
        return R.position_attention_ref(q_, k_, v_, qp, kp, D ** -0.5, compute=torch.float64)

    want = _bounds(ref, q, k, v, BF, D ** -0.5, 0.0, None, Tk)
    hit = _check_with_nan(*_run_position(q, k, v, qp, kp, kw, BF, 0.0, None), want)
    assert int(hit.sum()) == (1 if where == "query" else Tq * H // KH)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["query", "first key", "first own key"])
@pytest.mark.parametrize("form", PAGED_FORMS, ids=str)
def test_prefix_kernel_nan_scores_reach_their_rows(form, where):
    B, Tq, H, KH, D, P = form
    q, kc, vc, prefix, tables, lens = _prefix_case(B, Tq, H, KH, D, 16, P, [20] * B, FP)
    if where == "query":
        q[B // 2, 1, 5] = math.nan
    else:
        page = prefix[0] if where == "first key" else tables[B - 1, 0]
        kc[int(page), 0, 0, 7] = math.nan

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, D ** -0.5,
                                             compute=torch.float64)

    want = _bounds(ref, q, kc, vc, FP, D ** -0.5, 0.0, None, P + 20)
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), P,
                                           tables.cuda(), lens.cuda(), return_lse=True)
    hit = _check_with_nan(got, lse, want)
    assert int(hit.sum()) == (1 if where == "query" else
                              (B if where == "first key" else 1) * H // KH)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_position_kernel_scores_of_minus_infinity(form):
    """They take no part beside a finite score; a row that sees nothing else has
    no weights: NaN, unlike a row that sees no key."""
    Tq, Tk, H, KH, D = form
    q, k, v, qp, kp, kw = _position_case(Tq, Tk, H, KH, D, BF, "subset")
    q[..., 0] = 1.0
    k[:Tk // 2, 0, 0] = -math.inf
    qp[0] = Tk // 2 - 1
    if Tq > 1:
        qp[-1] = -1

    def ref(q_, k_, v_):
        return R.position_attention_ref(q_, k_, v_, qp, kp, D ** -0.5, compute=torch.float64)

    want = _bounds(ref, q, k, v, BF, D ** -0.5, 0.0, None, Tk)
    hit = _check_with_nan(*_run_position(q, k, v, qp, kp, kw, BF, 0.0, None), want)
    sees = (qp >= 0) & (qp < Tk // 2)
    assert int(hit.sum()) == int(sees.sum()) * H // KH


@pytest.mark.gpu
@pytest.mark.parametrize("form", PAGED_FORMS, ids=str)
def test_prefix_kernel_scores_of_minus_infinity(form):
    B, Tq, H, KH, D, P = form
    own = [20 + b % 9 for b in range(B)]
    q, kc, vc, prefix, tables, lens = _prefix_case(B, Tq, H, KH, D, 16, P, own, BF)
    q[..., 0] = 1.0
    kc[prefix.long(), :, 0, 0] = -math.inf
    kc[tables[B - 1, :2].long(), :, 0, 0] = -math.inf

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, D ** -0.5,
                                             compute=torch.float64)

    want = _bounds(ref, q, kc, vc, BF, D ** -0.5, 0.0, None, P + 30)
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), P,
                                           tables.cuda(), lens.cuda(), return_lse=True)
    hit = _check_with_nan(got, lse, want)
    assert int(hit.sum()) == H // KH


@pytest.mark.gpu
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_rows_computed_again_have_the_same_scores(form, paged):
    """An infinity in the first value: every row is computed a second time, with cap
    and distance bias, and only that column shows it."""
    if paged:
        B, Tq, H, KH, D, P = PAGED_FORMS[form]
        q, kc, vc, prefix, tables, lens = _prefix_case(B, Tq, H, KH, D, 16, P, [20] * B, BF)
        reach, slopes = P + 20, _slopes(H)
        k, v = kc, vc
        hit = (int(prefix[0]), 0, 0, 5)

        def ref(q_, k_, v_):
            return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, D ** -0.5,
                                                 20.0, slopes, torch.float64)

        def run(v_):
            return api.shared_prefix_attention(
                q.cuda(), kc.cuda(), v_.cuda(), prefix.cuda(), P, tables.cuda(), lens.cuda(),
                softcap=20.0, alibi_slopes=slopes.cuda(), return_lse=True)
    else:
        Tq, Tk, H, KH, D = FORMS[form]
        q, k, v, qp, kp, kw = _position_case(Tq, Tk, H, KH, D, BF, "subset")
        reach, slopes = Tk, _slopes(H)
        hit = (0, 0, 5)

        def ref(q_, k_, v_):
            return R.position_attention_ref(q_, k_, v_, qp, kp, D ** -0.5, 20.0, slopes,
                                            compute=torch.float64)

        def run(v_):
            return _run_position(q, k, v_, qp, kp, {}, BF, 20.0, slopes)

    o, e, tol, tl = _bounds(ref, q, k, v, BF, D ** -0.5, 20.0, slopes, reach)
    bad = v.clone()
    bad[hit] = math.inf
    got, lse = run(bad)
    rows = got.cpu().reshape(-1, H, D)[:, :H // KH]
    assert bool((rows[..., 5] == math.inf).all())
    mended = got.cpu().clone()
    mended.reshape(-1, H, D)[:, :H // KH, 5] = o.reshape(-1, H, D)[:, :H // KH, 5].to(BF)
    _check(mended, lse, o, e, tol, tl)


def _tail(n, D, bits):
    """One key whose weight is 2^bits times each of n others and whose value is
    zero: the result is the others' share."""
    q = torch.zeros(1, 1, D, dtype=FP)
    q[0, 0, 0] = 8.0
    k = torch.zeros(n + 1, 1, D, dtype=FP)
    k[n // 3, 0, 0] = bits * math.log(2) / 8
    v = torch.rand(n + 1, 1, D, generator=torch.Generator().manual_seed(n)).to(FP) + 1
    v[n // 3] = 0
    return q, k, v


# Weights pass through float16 times 2^7: below its normal range they are off by at
# most 2^-25 of that, 2^-32 of the largest weight, each.
def _tail_tolerance(o, v, n):
    return (2.0 ** -10 + 2.0 ** -14) * o.abs() + n * 2.0 ** -32 * float(v.max()) + 2.0 ** -25


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [20.3, 24.7, 25.4, 27.0])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_position_kernel_float16_keeps_the_tail_of_a_row(form, bits):
    Tq, Tk, H, KH, D = form
    q, k, v = _tail(Tk - 1, D, bits)
    o, lse = R.position_attention_ref(q, k, v, torch.tensor([Tk]), None, 1.0,
                                      compute=torch.float64)
    got, gl = api.position_attention(
        q.cuda().expand(Tq, H, D), k.cuda().expand(Tk, KH, D), v.cuda().expand(Tk, KH, D),
        torch.full((Tq,), Tk, device="cuda"), scale=1.0, return_lse=True)
    err = (got.cpu().double() - o).abs()
    assert bool((err <= _tail_tolerance(o, v, Tk)).all())
    assert bool(((gl.cpu().double() - lse).abs() <= 2.0 ** -18 * (1 + lse.abs())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [20.3, 24.7, 25.4, 27.0])
@pytest.mark.parametrize("form", PAGED_FORMS, ids=str)
def test_prefix_kernel_float16_keeps_the_tail_of_a_row(form, bits):
    B, Tq, H, KH, D, P = form
    q, k, v = _tail(P, D, bits)
    _, kc, vc, prefix, tables, lens = _prefix_case(B, Tq, H, KH, D, 16, P, [1] * B, FP, junk=0.0)
    at = torch.arange(P)
    for c, x in ((kc, k), (vc, v)):
        c[prefix.long()[at // 16], at % 16] = x[:P].expand(P, KH, D)
        c[tables[:, 0].long(), 0] = x[P].expand(B, KH, D)
    o, lse = R.position_attention_ref(q, k, v, torch.tensor([P]), None, 1.0,
                                      compute=torch.float64)
    got, gl = api.shared_prefix_attention(
        q.cuda().expand(B, H, D), kc.cuda(), vc.cuda(), prefix.cuda(), P, tables.cuda(),
        lens.cuda(), scale=1.0, return_lse=True)
    err = (got.cpu().double() - o).abs()
    assert bool((err <= _tail_tolerance(o, v, P + 1)).all())
    assert bool(((gl.cpu().double() - lse).abs() <= 2.0 ** -18 * (1 + lse.abs())).all())


# The tensor-core pass over the prefix: parts of large pages and many small ones, every
# layout, several KV heads, and a last page that ends inside a tile.
PREFIX_TC = [
    (40, 1, 32, 2, 64, 8, 1700, [1 + i for i in range(40)], BF, 0.0, False, "merged"),
    (40, 1, 32, 2, 128, 16, 1705, [1 + i % 5 for i in range(40)], FP, 0.0, False, "heads"),
    (40, 1, 32, 2, 128, 32, 1705, [3 * i for i in range(40)], FP, 30.0, True, "heads"),
    (40, 1, 32, 2, 128, 128, 1790, [1 + i for i in range(40)], BF, 0.0, True, "merged"),
    (44, 1, 32, 2, 64, 256, 1801, [1 + i for i in range(44)], FP, 0.0, False, "heads"),
    (33, 4, 16, 2, 64, 384, 1000, [4 + i for i in range(33)], BF, 20.0, False, "merged"),
    (30, 2, 64, 4, 128, 64, 700, [2 + i for i in range(30)], BF, 0.0, False, "plain"),
]
# Dense calls on the tensor cores whose blocks write their rows themselves.
POSITION_WHOLE = [
    (700, 700, 16, 2, 64, FP, 50.0, True, "documents"),
    (700, 700, 16, 2, 128, FP, 0.0, False, "documents"),
    (650, 650, 16, 2, 128, BF, 0.0, False, "padded"),
    (800, 800, 8, 2, 64, BF, 0.0, True, "prefix"),
    (600, 850, 16, 2, 128, FP, 15.0, True, "shuffled"),
    (640, 895, 10, 2, 128, BF, 20.0, False, "interleaved"),
    (500, 600, 16, 1, 64, FP, 0.0, True, "all"),
    (700, 700, 8, 1, 64, BF, 0.0, False, "causal"),
    (1000, 1300, 40, 4, 128, BF, 0.0, False, "subset"),
    (1000, 1000, 40, 4, 64, FP, 0.0, True, "documents"),
]


@pytest.mark.skipif(not ops.native_available(), reason="native module not built")
def test_shapes_reach_the_kernels_they_are_there_for():
    dense = lambda c: ops.native().position_attention_passes(*c[:4])
    tc, split = zip(*(dense(c) for c in FORMS))
    assert tc[:3] == (0, 0, 0) and split[0] == 1 and 2 <= split[1] <= 8 < split[2]
    assert split[3:] == (0, 0, 0) and tc[3:5] == (1, 1) and tc[5] > 1
    for c in POSITION_WHOLE:
        assert dense(c) == (1, 0), c
    for T in (700, 850):
        assert dense((T, T, 16, 1)) == (1, 0)

    def paged(B, Tq, H, KH, D, P, bs=16, own=20):
        return ops.native().shared_prefix_attention_passes(B, Tq, H, KH, bs, P, -(-own // bs) + 1)

    got = [paged(*c) for c in PAGED_FORMS]
    assert got[0] == (0, 0, 1) and got[1][:2] == (0, 0) and 2 <= got[1][2] <= 8
    assert got[2][:2] == (0, 0) and got[2][2] > 8
    assert got[3][:2] == (0, 0) and got[4][0] > 1 and got[4][1] == 0
    assert got[5][0] == 0 and got[5][1] > 1
    for B, Tq, H, KH, D, bs, P, own in (c[:8] for c in PREFIX_TC):
        assert paged(B, Tq, H, KH, D, P, bs, max(own))[0] > 1
    for bs in (8, 16, 64, 256):
        assert paged(40, 1, 32, 2, 128, 1700, bs, 50)[0] > 1


@pytest.mark.gpu
@pytest.mark.parametrize("case", PREFIX_TC, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_prefix_kernel_on_the_tensor_cores(case):
    test_prefix_kernel(case)


@pytest.mark.gpu
@pytest.mark.parametrize("case", POSITION_WHOLE,
                         ids=lambda c: "-".join(str(x) for x in c[:5]) + c[8])
def test_position_kernel_whole_rows_on_the_tensor_cores(case):
    test_position_kernel(case)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,T", [(64, 700), (128, 850)])
def test_position_kernel_masked_keys_hold_anything_whole_rows(value, D, T):
    test_position_kernel_masked_keys_hold_anything(value, T, 16, D, T)


@pytest.mark.gpu
@pytest.mark.parametrize("bs,bad", [(8, (3, 17, 40)), (16, (0, 30)), (64, (2, 5, 6)), (256, (1, 3)),
                                    (16, tuple(range(8))), (64, tuple(range(27)))])
def test_prefix_kernel_bad_pages_on_the_tensor_cores(bs, bad):
    """Single pages, the first whole tile, every page of the prefix."""
    B, H, KH, D, P = 40, 32, 2, 128, 1700
    own = [20 + i % 30 for i in range(B)]
    q, kc, vc, prefix, tables, lens = _prefix_case(B, 1, H, KH, D, bs, P, own, BF)
    for i, page in enumerate(bad):
        prefix[page] = (-1, kc.shape[0], 1 << 30, -(1 << 31))[i % 4]

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, 0.1,
                                             compute=torch.float64)

    want = _bounds(ref, q, kc, vc, BF, 0.1, 0.0, None, P + 50)
    st = ops.DeviceStatus("cuda")
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), P,
                                           tables.cuda(), lens.cuda(), scale=0.1, return_lse=True,
                                           status=st.tensor)
    _check(got, lse, *want)
    assert st.read()["name"] == "bad_slot"


@pytest.mark.gpu
def test_prefix_kernel_large_scores_on_the_tensor_cores():
    B, H, KH, D, P = 40, 32, 2, 64, 1700
    q, kc, vc, prefix, tables, lens = _prefix_case(B, 1, H, KH, D, 16, P, [40] * B, BF)
    kc[prefix.long()[2]] *= 100
    kc[prefix.long()[70]] *= 200

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, 1.0,
                                             compute=torch.float64)

    want = _bounds(ref, q, kc, vc, BF, 1.0, 0.0, None, P + 40)
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), P,
                                           tables.cuda(), lens.cuda(), scale=1.0, return_lse=True)
    _check(got, lse, *want)


@pytest.mark.gpu
def test_prefix_kernel_on_the_tensor_cores_captured_twice():
    B, P = 40, 1700
    q, kc, vc, prefix, tables, lens = _prefix_case(B, 1, 32, 2, 64, 16, P, [30] * B, BF, junk=0.0)
    d = [x.cuda() for x in (q, kc, vc, prefix, tables, lens)]

    def call():
        return api.shared_prefix_attention(d[0], d[1], d[2], d[3], P, d[4], d[5], return_lse=True)

    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for shift in (0, 1):
        d[5].copy_(torch.arange(B) % 30 + shift)
        want = call()
        torch.cuda.synchronize()
        for _ in range(5):  # both at once
            for (g, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


# Chunks of a prompt on a shared prefix: split and tensor-core prefix, more rows than
# a tile, requests with fewer own tokens than queries.
CHUNKS = [(2, 300, 8, 2, 64, 16, 100, [300, 700], BF, 0.0, False, "plain"),
          (3, 129, 16, 2, 128, 32, 700, [40, 129, 500], FP, 30.0, True, "heads"),
          (1, 1024, 4, 1, 64, 64, 300, [1024], FP, 0.0, True, "merged")]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_prefix_kernel_many_query_tokens(case):
    test_prefix_kernel(case)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [3, 20, 600, 4096])
@pytest.mark.parametrize("form", PAGED_FORMS, ids=str)
def test_prefix_kernel_tables_wider_than_the_requests(form, width):
    """Most parts of a row are empty where a table has room for long requests."""
    B, Tq, H, KH, D, P = form
    q, kc, vc, prefix, tables, lens = _prefix_case(B, Tq, H, KH, D, 16, P, [20] * B, BF)
    wide = torch.full((B, width), -1, dtype=torch.int32)
    wide[:, :tables.shape[1]] = tables

    def ref(q_, k_, v_):
        return R.shared_prefix_attention_ref(q_, k_, v_, prefix, P, tables, lens, D ** -0.5,
                                             compute=torch.float64)

    want = _bounds(ref, q, kc, vc, BF, D ** -0.5, 0.0, None, P + 20)
    st = ops.DeviceStatus("cuda")
    got, lse = api.shared_prefix_attention(q.cuda(), kc.cuda(), vc.cuda(), prefix.cuda(), P,
                                           wide.cuda(), lens.cuda(), return_lse=True,
                                           status=st.tensor)
    _check(got, lse, *want)
    st.check()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_position_kernel_keys_and_values_of_other_strides(form):
    """K as a slice of wider rows, V and Q head by head."""
    Tq, Tk, H, KH, D = form
    q, k, v, qp, kp, kw = _position_case(Tq, Tk, H, KH, D, BF, "subset")
    want = _run_position(q, k, v, qp, kp, {}, BF, 0.0, None)
    wide = torch.zeros(Tk, (KH + 3) * D, dtype=BF, device="cuda")
    wide[:, 2 * D:(KH + 2) * D] = k.flatten(1).cuda()
    dk = wide[:, 2 * D:(KH + 2) * D].unflatten(1, (KH, D))
    dv = v.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    dq = q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    got, lse = api.position_attention(dq, dk, dv, qp.cuda(), kp.cuda(), return_lse=True)
    assert torch.equal(got, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
def test_prefix_kernel_caches_of_other_strides():
    for form in PAGED_FORMS:
        B, Tq, H, KH, D, P = form
        q, kc, vc, *rest = _prefix_case(B, Tq, H, KH, D, 16, P, [20] * B, BF)
        rest = [x.cuda() for x in rest]
        a = (rest[0], P, rest[1], rest[2])
        want = api.shared_prefix_attention(q.cuda(), *_on_device(kc, vc, "plain"), *a)
        dk = _on_device(kc, vc, "merged")[0]
        dv = _on_device(kc, vc, "heads")[1]
        assert torch.equal(api.shared_prefix_attention(q.cuda(), dk, dv, *a), want)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    cases = [_position_case(Tq, Tk, H, KH, D, BF, "subset") for Tq, Tk, H, KH, D in FORMS[2:]]
    dev = [[x.cuda() for x in c[:5]] for c in cases]
    want = [api.position_attention(*d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for i, d in enumerate(dev):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append((i, api.position_attention(*d)))
    torch.cuda.synchronize()
    for i, g in got:
        assert torch.equal(g, want[i])


@pytest.mark.gpu
@pytest.mark.parametrize("form", [PAGED_FORMS[i] for i in (1, 2, 4, 5)], ids=str)
def test_offsets_of_a_long_cache_pass_32_bits(form):
    """The same pages at the end of caches of 2^31 elements and more."""
    from lmcache_ascend_b200.ops.reference import make_cos_sin_cache

    B, Tq, H, KH, D, P = form
    q, kc, vc, prefix, tables, lens = (x.cuda() for x in _prefix_case(
        B, Tq, H, KH, D, 16, P, [20] * B, BF, junk=0.0))
    want = api.shared_prefix_attention(q, kc, vc, prefix, P, tables, lens)
    first = (1 << 31) // (16 * KH * D) + 7
    long_k, long_v = (torch.empty(first + c.shape[0], 16, KH, D, dtype=BF, device="cuda")
                      for c in (kc, vc))
    long_k[first:], long_v[first:] = kc, vc
    got = api.shared_prefix_attention(q, long_k, long_v, prefix + first, P, tables + first, lens)
    assert torch.equal(got, want)
    # rows written there, by the slots of a slot map
    st = ops.DeviceStatus("cuda")
    new = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    small, far = (api.build_slot_mapping(lens, new, t, 16, 3 * B, num_blocks=nb, status=st.tensor)
                  for t, nb in ((tables, kc.shape[0]), (tables + first, long_k.shape[0])))
    st.check()
    assert torch.equal(far.slot_mapping, small.slot_mapping + first * 16)
    x = torch.randn(3 * B, KH * D, device="cuda").to(BF)
    table = make_cos_sin_cache(64, D).cuda()
    args = (small.positions, x, x, x)
    api.rotary_embedding_and_cache(*args, kc, vc, small.slot_mapping, D, table)
    api.rotary_embedding_and_cache(*args, long_k, long_v, far.slot_mapping, D, table)
    assert torch.equal(long_k[first:], kc) and torch.equal(long_v[first:], vc)


@pytest.mark.gpu
def test_position_kernel_unaligned_rows_and_far_positions():
    q, k, v, qp, kp, kw = _position_case(100, 300, 4, 2, 64, BF, "subset")
    want = _run_position(q, k, v, qp, kp, kw, BF, 0.0, None)
    flat = torch.zeros(k.numel() + 1, dtype=BF, device="cuda")
    flat[1:] = k.flatten().cuda()
    got = api.position_attention(q.cuda(), flat[1:].view(k.shape), v.cuda(), qp.cuda(), kp.cuda())
    assert torch.equal(got, want[0])
    # the same differences of positions near the end of the 32-bit range
    base = 2 ** 31 - 1000
    got = _run_position(q, k, v, qp + base, kp + base, kw, BF, 0.0, _slopes(4))
    want = _run_position(q, k, v, qp, kp, kw, BF, 0.0, _slopes(4))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_position_kernel_refusals():
    q, k, v, qp, kp, kw = _position_case(8, 30, 4, 2, 64, BF, "interleaved")
    d = {a: b.cuda() for a, b in dict(query=q, key=k, value=v, q_positions=qp, k_positions=kp,
                                      **kw).items()}
    api.position_attention(**d)
    assert api.position_attention(d["query"][:0], d["key"], d["value"], d["q_positions"][:0],
                                  d["k_positions"]).numel() == 0
    for bad in (dict(query=q.cuda().float(), key=k.cuda().float(), value=v.cuda().float()),
                dict(query=q[..., :32].cuda(), key=k[..., :32].cuda(), value=v[..., :32].cuda()),
                dict(query=q.cuda()[:, :3]), dict(key=k.cuda().half()), dict(key=k),
                dict(value=v.cuda()[:4]), dict(q_positions=qp.cuda()[:3]),
                dict(q_positions=qp.cuda().float()), dict(k_positions=kp.cuda()[:3]),
                dict(q_documents=None), dict(q_documents=kw["q_documents"].cuda().long()),
                dict(k_documents=kw["k_documents"].cuda()[:3]),
                dict(q_prefix_lens=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(softcap=-2.0), dict(scale=math.nan),
                dict(alibi_slopes=torch.zeros(2, device="cuda"))):
        with pytest.raises((RuntimeError, TypeError)):
            api.position_attention(**{**d, **bad})


@pytest.mark.gpu
def test_position_kernel_captured_on_a_side_stream():
    q, k, v, qp, kp, kw = _position_case(200, 600, 4, 2, 128, BF, "subset")
    d = [x.cuda() for x in (q, k, v, qp, kp)]
    want = api.position_attention(*d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        got = api.position_attention(*d)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    d[0].normal_()
    d[3].copy_(d[3].flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, api.position_attention(*d))
