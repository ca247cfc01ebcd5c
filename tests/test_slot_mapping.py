"""Block tables and slot maps from request lengths: the oracle against the
formula one token at a time, the kernel against the oracle (equal integers)."""

import pytest
import torch

from lmcache_ascend_b200 import ops
from lmcache_ascend_b200.ops import api
from lmcache_ascend_b200.ops import reference as R


def _case(ctx, new, bs, extra=3, seed=0, width=None):
    have = [-(-c // bs) for c in ctx]
    need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    total = sum(need) + extra
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    w = max([1] + need) + 2 if width is None else width
    tables = torch.full((len(ctx), w), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(have):
        tables[b, :min(h, w)] = ids[at:at + min(h, w)]
        at += h
    return tables, ids[at:].contiguous(), total


CASES = [([5], [1], 4), ([0], [1], 16), ([0, 0, 0], [0, 0, 0], 16), ([16, 15, 17], [1, 1, 1], 16),
         ([3, 0, 700, 64], [0, 130, 1, 5], 64), ([0] * 40, list(range(40)), 1),
         ([7, 9], [2100, 2049], 3)]


@pytest.mark.parametrize("ctx,new,bs", CASES)
def test_oracle_follows_the_formula(ctx, new, bs):
    tables, free, total = _case(ctx, new, bs)
    n = sum(new)
    m = api.build_slot_mapping(torch.tensor(ctx), torch.tensor(new), tables, bs, n + 2, free, total)
    t = 0
    for b, (c, k) in enumerate(zip(ctx, new)):
        assert int(m.query_start_loc[b]) == t
        for p in range(c, c + k):
            assert int(m.slot_mapping[t]) == int(tables[b, p // bs]) * bs + p % bs
            assert int(m.positions[t]) == p and int(m.request_ids[t]) == b
            t += 1
    used = m.slot_mapping[:n]
    assert used.unique().numel() == n and bool((used >= 0).all())
    assert m.slot_mapping[n:].tolist() == [-1, -1] and m.request_ids[n:].tolist() == [-1, -1]
    assert int(m.taken[-1]) == sum(-(-(c + k) // bs) - -(-c // bs) for c, k in zip(ctx, new))


def test_oracle_missing_blocks():
    tables, free, total = _case([4, 4], [8, 8], 4, extra=0)
    m = api.build_slot_mapping(torch.tensor([4, 4]), torch.tensor([8, 8]), tables, 4, 16, free[:3],
                               total)
    assert int((m.slot_mapping == -1).sum()) == 4 and int(tables[1, 2]) == -1
    assert int(m.taken[-1]) == 4


def test_cpu_refusals():
    z = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 2, dtype=torch.int32)
    for bad in (dict(dtype=torch.int16), dict(num_tokens=-1), dict(block_size=0),
                dict(block_tables=t[:1]), dict(new_lens=z[:1])):
        kw = dict(context_lens=z, new_lens=z, block_tables=t, block_size=4, num_tokens=2)
        kw.update(bad)
        with pytest.raises(ValueError):
            api.build_slot_mapping(**kw)


def test_block_size_of_zero_is_refused_for_both_slot_types():
    z, t = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    for dtype in (torch.int32, torch.int64):
        with pytest.raises(ValueError):
            api.build_slot_mapping(z, z, t, 0, 2, dtype=dtype)


def _compare(got, want, tables, tables_ref):
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
    assert torch.equal(tables.cpu(), tables_ref)


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new,bs", CASES + [
    ([i * 7 % 90 for i in range(1500)], [i * 5 % 13 for i in range(1500)], 16),
    ([0, 3, 0], [30000, 1, 7001], 128)])
@pytest.mark.parametrize("lens,slots", [(torch.int32, torch.int64), (torch.int64, torch.int32)])
@pytest.mark.parametrize("grow", [True, False])
def test_kernel_equals_oracle(ctx, new, bs, lens, slots, grow):
    tables, free, total = _case(ctx, new, bs)
    if not grow:  # the tables hold every block already
        api.build_slot_mapping(torch.tensor(ctx), torch.tensor(new), tables, bs, 0, free, total)
    dev = tables.cuda()
    c, n = torch.tensor(ctx, dtype=lens), torch.tensor(new, dtype=lens)
    rows = sum(new) + 5
    st = ops.DeviceStatus("cuda")
    got = api.build_slot_mapping(c.cuda(), n.cuda(), dev, bs, rows, free.cuda() if grow else None,
                                 total, slots, st.tensor)
    want = api.build_slot_mapping(c, n, tables, bs, rows, free if grow else None, total, slots)
    _compare(got, want, dev, tables)
    st.check()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["free", "width", "page", "negative", "total"])
def test_kernel_bad_input_is_reported_and_leaves_no_slot(what):
    ctx, new, bs = [4, 9, 2], [8, 8, 30], 4
    tables, free, total = _case(ctx, new, bs, width=5 if what == "width" else None)
    rows = sum(new)
    if what == "free":
        free = free[:4]
    if what == "page":
        tables[1, 2] = 1 << 30
    if what == "negative":
        ctx, new = [4, -9, 2], [8, 8, -30]
    if what == "total":
        rows -= 7
    dev = tables.cuda()
    st = ops.DeviceStatus("cuda")
    c, n = torch.tensor(ctx), torch.tensor(new)
    got = api.build_slot_mapping(c.cuda(), n.cuda(), dev, bs, rows, free.cuda(), total,
                                 status=st.tensor)
    want = api.build_slot_mapping(c, n, tables, bs, rows, free, total)
    _compare(got, want, dev, tables)
    assert st.read()["name"] in ("bad_index", "bad_slot")


@pytest.mark.gpu
def test_kernel_empty_batch_and_no_tokens():
    t = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    m = api.build_slot_mapping(z, z, t, 16, 3, z, 0)
    assert m.slot_mapping.tolist() == [-1] * 3 and m.query_start_loc.tolist() == [0]
    assert m.taken.tolist() == [0] and m.seq_lens.numel() == 0
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    m = api.build_slot_mapping(one, one * 0, t.new_zeros(2, 1), 16, 0)
    assert m.slot_mapping.numel() == 0 and m.seq_lens.tolist() == [1, 1]


@pytest.mark.gpu
def test_kernel_refusals():
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    t = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    good = dict(context_lens=z, new_lens=z, block_tables=t, block_size=4, num_tokens=2)
    api.build_slot_mapping(**good)
    for bad in (dict(context_lens=z.cpu()), dict(new_lens=z.long()), dict(new_lens=z[:1]),
                dict(context_lens=z.float(), new_lens=z.float()), dict(block_tables=t.long()),
                dict(block_tables=t[:1]), dict(block_tables=t.t()[:, :2].expand(2, 2).t()[:, ::2]),
                dict(block_size=0), dict(num_tokens=-1), dict(num_tokens=1 << 31),
                dict(free_blocks=z.long()), dict(free_blocks=z.cpu()), dict(num_blocks=-1),
                dict(num_blocks=1 << 30, dtype=torch.int32),
                dict(status=torch.zeros(1, dtype=torch.int64, device="cuda"))):
        if "block_tables" in bad and bad["block_tables"].shape == (2, 1):
            continue  # one column has no stride
        with pytest.raises((RuntimeError, ValueError)):
            api.build_slot_mapping(**{**good, **bad})


@pytest.mark.gpu
def test_kernel_captured_and_replayed_with_other_lengths():
    ctx, new, bs = [5, 0, 31], [1, 1, 1], 16
    tables, free, total = _case(ctx, new, bs)
    c, n = torch.tensor(ctx).cuda(), torch.tensor(new).cuda()
    dev, f = tables.cuda(), free.cuda()
    api.build_slot_mapping(c, n, dev, bs, 8, f, total)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = api.build_slot_mapping(c, n, dev, bs, 8, f, total)
    for new2 in ([1, 2, 5], [0, 0, 1], [2, 3, 1]):
        n.copy_(torch.tensor(new2))
        dev.copy_(tables)
        g.replay()
        torch.cuda.synchronize()
        ref = tables.clone()
        want = R.build_slot_mapping_ref(ctx, new2, ref, bs, 8, free, total)
        _compare(got, want, dev, ref)
