"""Rotary positions of fresh rows with K/V written to their pages: scaled
tables against the formulas, the kernel against the 64-bit oracle."""

import math

import pytest
import torch

from lmcache_ascend_b200 import ops
from lmcache_ascend_b200.ops import api
from lmcache_ascend_b200.ops import reference as R

SCALINGS = [None, {"rope_type": "linear", "factor": 4.0},
            {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 512},
            {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
             "high_freq_factor": 4.0, "original_max_position_embeddings": 512},
            {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512}]


@pytest.mark.parametrize("scaling", SCALINGS)
def test_scaled_tables_one_angle_at_a_time(scaling):
    n, rot, base = 2048, 64, 10000.0
    table = R.make_scaled_cos_sin_cache(n, rot, base, scaling, torch.float64)
    kind = (scaling or {}).get("rope_type", "default")
    f = (scaling or {}).get("factor", 1.0)
    for i in (0, 1, 9, 17, 31):
        w = base ** (-2 * i / rot)
        gain = 1.0
        if kind == "linear":
            w /= f
        elif kind == "dynamic":
            w = (base * (f * n / 512 - (f - 1)) ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif kind == "llama3":
            turns = 512 * w / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            w = keep * w + (1 - keep) * w / f
        elif kind == "yarn":
            at = [rot * math.log(512 / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32, 1)]
            lo, hi = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
            mix = min(1.0, max(0.0, (i - lo) / (hi - lo)))
            w = mix * w / f + (1 - mix) * w
            gain = 0.1 * math.log(f) + 1
        for p in (0, 1, 777, 2047):
            assert abs(float(table[p, i]) - gain * math.cos(p * w)) < 1e-9
            assert abs(float(table[p, rot // 2 + i]) - gain * math.sin(p * w)) < 1e-9
    if kind == "default":
        assert torch.equal(table, R.make_cos_sin_cache(n, rot, base, torch.float64))


def test_unknown_scaling_is_refused():
    with pytest.raises(ValueError):
        R.make_scaled_cos_sin_cache(16, 8, scaling={"rope_type": "other", "factor": 2.0})


def test_yarn_gains_and_untruncated_ramp():
    n, rot, base, f, orig = 64, 64, 10000.0, 40.0, 4096
    yarn = {"rope_type": "yarn", "factor": f, "original_max_position_embeddings": orig}
    gain = lambda m: 0.1 * m * math.log(f) + 1

    def first(**more):  # cosine of angle 0: the gain
        return float(R.make_scaled_cos_sin_cache(n, rot, base, {**yarn, **more},
                                                 torch.float64)[0, 0])

    assert abs(first() - gain(1)) < 1e-12
    assert abs(first(mscale=1.0, mscale_all_dim=1.0) - 1) < 1e-12
    assert abs(first(mscale=0.707, mscale_all_dim=1.5) - gain(0.707) / gain(1.5)) < 1e-12
    assert abs(first(attention_factor=1.25, mscale=1.0, mscale_all_dim=1.0) - 1.25) < 1e-12
    lo, hi = (rot * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (16, 2))
    table = R.make_scaled_cos_sin_cache(n, rot, base, {**yarn, "beta_fast": 16, "beta_slow": 2,
                                                       "truncate": False,
                                                       "attention_factor": 1.0}, torch.float64)
    for i in range(rot // 2):
        w = base ** (-2 * i / rot)
        mix = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        w = mix * w / f + (1 - mix) * w
        assert abs(float(table[63, rot // 2 + i]) - math.sin(63 * w)) < 1e-9


def test_scaling_keys_that_are_not_known_are_refused():
    for bad in ({"rope_type": "linear", "factor": 2.0, "mscale": 1.0},
                {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 64,
                 "partial_rotary_factor": 0.5},
                {"rope_type": "llama3", "factor": 8.0, "rope_theta": 500000.0}):
        with pytest.raises(ValueError):
            R.make_scaled_cos_sin_cache(16, 8, 10000.0, bad)
    same = {"rope_type": "default", "rope_theta": 10000.0, "mscale": None}
    assert torch.equal(R.make_scaled_cos_sin_cache(16, 8, 10000.0, same),
                       R.make_cos_sin_cache(16, 8))


def test_oracle_is_a_rotation_and_undone_by_the_opposite():
    T, H, D, rot = 9, 3, 32, 16
    x = torch.randn(T, H * D, dtype=torch.float64)
    pos = torch.arange(T) * 11
    table = R.make_cos_sin_cache(128, rot, dtype=torch.float64)
    for neox in (True, False):
        y = R.rotary_embedding_ref(pos, x, D, table, neox, torch.float64)
        assert torch.allclose(y.view(T, H, D).norm(dim=-1), x.view(T, H, D).norm(dim=-1))
        back = table.clone()
        back[:, rot // 2:] *= -1
        assert torch.allclose(R.rotary_embedding_ref(pos, y, D, back, neox, torch.float64), x)


def test_cpu_form_writes_pages():
    T, KH, D = 6, 2, 8
    q, k, v = torch.randn(T, 4 * D), torch.randn(T, KH * D), torch.randn(T, KH * D)
    kc, vc = torch.randn(3, 4, KH, D), torch.randn(3, 4, KH, D)
    k0 = kc.clone()
    slots = torch.tensor([5, -1, 0, 11, 7, 99])
    pos = torch.tensor([0, 1, 2, 3, 400, 5])
    table = R.make_cos_sin_cache(16, D)
    out = api.rotary_embedding_and_cache(pos, q, k, v, kc, vc, slots, D, table)
    want = R.rotary_embedding_ref(pos, k, D, table, True).view(T, KH, D)
    assert torch.equal(kc.view(12, KH, D)[[5, 0, 11]], want[[0, 2, 3]])
    assert torch.equal(vc.view(12, KH, D)[5], v.view(T, KH, D)[0])
    rest = [s for s in range(12) if s not in (5, 0, 11)]
    assert torch.equal(kc.view(12, KH, D)[rest], k0.view(12, KH, D)[rest])
    assert bool((out[4] == 0).all())


# Half a step of the result's type on |y|, plus two fp32 products and one sum:
# |x1 cos| + |x2 sin| <= 2 max|x| gain, each off by 2^-24 relative, times 3.
def _tolerance(want, x, table):
    size = float(x.abs().max()) * float(table.abs().max())
    return want.abs() * torch.finfo(x.dtype).eps / 2 + 6 * size * 2.0 ** -24


def _rows(T, H, KH, D, dtype, g, fused=True, pad=0):
    w = torch.randn(T, (H + 2 * KH) * D + pad, generator=g).to(dtype)
    return w[:, pad:].split([H * D, KH * D, KH * D], dim=1) if fused else w


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,KH,D,rot,bs", [
    (1, 8, 2, 128, 128, 16), (3, 32, 8, 64, 64, 16), (257, 5, 1, 128, 64, 64),
    (700, 14, 2, 64, 32, 128), (65, 4, 4, 96, 32, 16), (33, 3, 1, 80, 20, 7), (5, 2, 2, 7, 6, 3)])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype,tdt", [(torch.bfloat16, torch.float32),
                                       (torch.float16, torch.float32),
                                       (torch.float32, torch.float32),
                                       (torch.bfloat16, torch.bfloat16),
                                       (torch.float32, torch.float16)])
@pytest.mark.parametrize("pad", [0, 1])
def test_kernel_against_oracle(T, H, KH, D, rot, bs, neox, dtype, tdt, pad):
    g = torch.Generator().manual_seed(T * 31 + D)
    q, k, v = _rows(T, H, KH, D, dtype, g, pad=pad)
    table = R.make_scaled_cos_sin_cache(4096, rot, 10000.0, SCALINGS[4], tdt)
    pos = torch.randint(0, 4096, (T,), generator=g)
    nb = -(-T // bs) + 2
    slots = torch.randperm(nb * bs, generator=g)[:T]
    slots[::5] = -1
    cache = torch.randn(2, nb, bs, KH, D, generator=g).to(dtype)
    base = torch.zeros(T, q.shape[1] + 2 * k.shape[1] + pad, dtype=dtype, device="cuda")
    base[:, pad:] = torch.cat([q, k, v], 1).cuda()
    dq, dk, dv = base[:, pad:].split([H * D, KH * D, KH * D], dim=1)
    dc = cache.cuda()
    kout = torch.zeros(T, KH, D, dtype=dtype, device="cuda")
    st = ops.DeviceStatus("cuda")
    out = api.rotary_embedding_and_cache(pos.cuda(), dq, dk, dv, dc[0], dc[1],
                                         slots.int().cuda(), D, table.cuda(), neox, key_out=kout,
                                         status=st.tensor)
    st.check()
    wq = R.rotary_embedding_ref(pos, q, D, table, neox, torch.float64)
    wk = R.rotary_embedding_ref(pos, k, D, table, neox, torch.float64)
    assert bool(((out.cpu().double() - wq).abs() <= _tolerance(wq, q, table)).all())
    assert bool(((kout.cpu().view(T, -1).double() - wk).abs() <= _tolerance(wk, k, table)).all())
    want = cache.clone()
    R.write_cache_ref(pos, kout.cpu(), want[0], slots, 4096)
    R.write_cache_ref(pos, v, want[1], slots, 4096)
    assert torch.equal(dc.cpu(), want)  # rows of other slots untouched
    # without pages, and in place: the same bits
    q2, k2 = api.rotary_embedding(pos.cuda(), dq, dk, D, table.cuda(), neox, query_out=dq)
    assert q2.data_ptr() == dq.data_ptr() and torch.equal(q2, out)
    assert torch.equal(k2.reshape(T, -1), kout.view(T, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 40])
def test_kernel_strided_pages_and_positions_outside_the_table(D):
    T, H, KH, bs, nb = 50, 4, 2, 16, 6
    g = torch.Generator().manual_seed(2)
    q, k, v = (x.contiguous() for x in _rows(T, H, KH, D, torch.bfloat16, g))
    table = R.make_cos_sin_cache(256, D)
    pos = torch.randint(0, 256, (T,), generator=g)
    pos[7], pos[8] = -1, 256
    slots = torch.randperm(nb * bs, generator=g)[:T]
    slots[9] = nb * bs
    # heads apart from tokens: [NB, 2, KH, BS, D] storage
    store = torch.randn(nb, 2, KH, bs, D, generator=g).to(torch.bfloat16)
    dev = store.cuda()
    kc, vc = dev[:, 0].transpose(1, 2), dev[:, 1].transpose(1, 2)
    st = ops.DeviceStatus("cuda")
    out = api.rotary_embedding_and_cache(pos.int().cuda(), q.cuda(), k.cuda(), v.cuda(), kc, vc,
                                         slots.cuda(), D, table.cuda(), status=st.tensor)
    assert st.read()["name"] in ("bad_index", "bad_slot")
    assert bool((out[7:9] == 0).all())
    ref = store.clone()
    wk = R.rotary_embedding_ref(pos, k, D, table, True).to(torch.bfloat16)
    R.write_cache_ref(pos, wk, ref[:, 0].transpose(1, 2), slots, 256)
    R.write_cache_ref(pos, v, ref[:, 1].transpose(1, 2), slots, 256)
    assert torch.equal(dev[:, 1].cpu(), ref[:, 1])
    got, want = dev[:, 0].cpu().double(), ref[:, 0].double()
    assert bool(((got - want).abs() <= want.abs() * 2.0 ** -7 + 1e-6).all())
    same = torch.ones(nb, KH, bs, D, dtype=torch.bool)
    keep = (slots >= 0) & (slots < nb * bs) & (pos >= 0) & (pos < 256)
    same.transpose(1, 2)[slots[keep] // bs, slots[keep] % bs] = False
    assert torch.equal(got[same], store[:, 0].double()[same])


@pytest.mark.gpu
def test_kernel_no_rows_and_refusals():
    D, table = 64, R.make_cos_sin_cache(64, 64).cuda()
    q = torch.zeros(4, 2 * D, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(4, D, device="cuda", dtype=torch.bfloat16)
    c = torch.zeros(2, 4, 1, D, device="cuda", dtype=torch.bfloat16)
    p = torch.arange(4, device="cuda")
    empty = api.rotary_embedding_and_cache(p[:0], q[:0], k[:0], k[:0], c, c.clone(), p[:0], D,
                                           table)
    assert empty.shape == (0, 2 * D)
    good = dict(positions=p, query=q, key=k, value=k, key_cache=c, value_cache=c.clone(),
                slot_mapping=p, head_size=D, cos_sin_cache=table)
    api.rotary_embedding_and_cache(**good)
    for bad in (dict(positions=p.float()), dict(positions=p[:3]), dict(positions=p.cpu()),
                dict(key=k.float()), dict(value=k.cpu()), dict(head_size=48), dict(head_size=0),
                dict(key_cache=c[..., :32]), dict(value_cache=c.half()), dict(value_cache=c[:1]),
                dict(slot_mapping=p.double()), dict(slot_mapping=p[:2]),
                dict(cos_sin_cache=table.double()), dict(cos_sin_cache=table[:, ::2]),
                dict(cos_sin_cache=R.make_cos_sin_cache(64, 128).cuda()),
                dict(query_out=q[:2]), dict(query_out=q.t().contiguous().t()),
                dict(value=torch.cat([k, k], 1)), dict(slot_mapping=None)):
        with pytest.raises((RuntimeError, TypeError)):
            api.rotary_embedding_and_cache(**{**good, **bad})


@pytest.mark.gpu
def test_no_gradient_is_lost_without_a_word():
    D, table = 64, R.make_cos_sin_cache(64, 64).cuda()
    q = torch.randn(4, 2 * D, device="cuda")
    k, v = torch.randn(4, D, device="cuda"), torch.randn(4, D, device="cuda")
    kc, vc = torch.zeros(2, 4, 1, D, device="cuda"), torch.zeros(2, 4, 1, D, device="cuda")
    p = torch.arange(4, device="cuda")
    kw = dict(query=q, key=k, value=v, key_cache=kc, value_cache=vc, cos_sin_cache=table,
              query_out=torch.zeros_like(q), key_out=torch.zeros_like(k))

    def call(**more):
        return api.rotary_embedding_and_cache(positions=p, slot_mapping=p, head_size=D,
                                              **{**kw, **more})

    call()
    for name, t in kw.items():
        with pytest.raises(RuntimeError, match="forward only"):
            call(**{name: t.clone().requires_grad_()})
        with torch.no_grad():
            call(**{name: t.clone().requires_grad_()})
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="tangent"):
                call(**{name: dual})


@pytest.mark.gpu
def test_kernel_on_a_side_stream_captured():
    T, H, D = 40, 8, 128
    q = torch.randn(T, H * D, device="cuda").bfloat16()
    k = torch.randn(T, 2 * D, device="cuda").bfloat16()
    table = R.make_cos_sin_cache(512, D).cuda()
    pos = torch.arange(T, device="cuda")
    want, kwant = api.rotary_embedding(pos, q, k, D, table)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got, kgot = api.rotary_embedding(pos, q, k, D, table)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(kgot, kwant)
    pos += 100
    q.normal_()
    g.replay()
    torch.cuda.synchronize()
    want, kwant = api.rotary_embedding(pos, q, k, D, table)
    assert torch.equal(got, want) and torch.equal(kgot, kwant)
