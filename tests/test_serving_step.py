"""The serving operators together: a batch decoded step by step on a shared
prefix, and a blend whose attention is ``position_attention``."""

import pytest
import torch

from lmcache_ascend_b200 import ops
from lmcache_ascend_b200.models.llama import LlamaConfig, LlamaForBlend
from lmcache_ascend_b200.v1.blend.vllm_model import LMCVLLMModel

NB, BS, B, P, STEPS = 64, 8, 5, 21, 11


def _config(head_dim):
    return LlamaConfig.tiny(vocab_size=300, hidden_size=128, num_layers=2, num_heads=4,
                            num_kv_heads=2, head_dim=head_dim, intermediate_size=256,
                            max_position=512)


def _pages(c, device, dtype):
    return [tuple(torch.zeros(NB, BS, c.num_kv_heads, c.head_dim, device=device, dtype=dtype)
                  for _ in range(2)) for _ in range(c.num_layers)]


def _decode(model, seqs, device, dtype):
    """Hidden state of each new token of every request, one step at a time."""
    c = model.config
    kv = _pages(c, device, dtype)
    ids = torch.randperm(NB, generator=torch.Generator().manual_seed(3)).int()
    npb = -(-P // BS)
    prefix = ids[:npb].to(device)
    slots = (ids[:npb].long()[torch.arange(P) // BS] * BS + torch.arange(P) % BS).to(device)
    model.prefill(seqs[0, :P], kv, slots)
    tables = torch.full((B, -(-STEPS // BS)), -1, dtype=torch.int32, device=device)
    free = ids[npb:].to(device)
    own = torch.zeros(B, dtype=torch.int32, device=device)
    status = ops.DeviceStatus(device) if device != "cpu" else None
    out = []
    for s in range(STEPS):
        h, step = model.decode_batch(seqs[:, P + s].to(device), own, kv, tables, free, prefix, P,
                                     status=status.tensor if status else None)
        out.append(h)
        own = step.seq_lens
        free = free[int(step.taken[-1]):]
    if status:
        status.check()
    return torch.stack(out, 1), tables


def _sequences():
    g = torch.Generator().manual_seed(5)
    seqs = torch.randint(0, 300, (B, P + STEPS), generator=g)
    seqs[:, :P] = seqs[0, :P]
    return seqs


def test_batch_on_a_shared_prefix_equals_whole_prefills():
    c = _config(32)
    model = LlamaForBlend(c, seed=2)
    seqs = _sequences()
    got, tables = _decode(model, seqs, "cpu", torch.float32)
    assert tables.unique().numel() == tables.numel() and int(tables.min()) >= 0
    for b in range(B):
        kv = _pages(c, "cpu", torch.float32)
        want = model.prefill(seqs[b], kv, torch.arange(P + STEPS))[P:]
        assert torch.allclose(got[b], want, atol=1e-4, rtol=1e-4)


def test_native_attention_of_the_model_on_the_cpu():
    c = _config(32)
    plain, native = LlamaForBlend(c, seed=2), LlamaForBlend(c, seed=2, native_attention=True)
    tokens = _sequences()[0]
    outs = [m.prefill(tokens, _pages(c, "cpu", torch.float32), torch.arange(tokens.numel()))
            for m in (plain, native)]
    assert torch.allclose(outs[0], outs[1], atol=1e-4, rtol=1e-4)


# A hidden state went through about 16 roundings to float16 a layer (projections,
# norms, rotary, weights and results of attention, sums), 2 layers and the final
# norm: 40 x 2^-11 relative, in the norm of a row.
_TOLERANCE = 40 * 2.0 ** -11


def _close(got, want):
    err = (got.cpu().double() - want.double()).norm(dim=-1) / want.double().norm(dim=-1)
    assert float(err.max()) <= _TOLERANCE, float(err.max())


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_decode_batch_on_the_gpu(head_dim):
    c = _config(head_dim)
    half = LlamaForBlend(c, "cpu", torch.float16, seed=4)
    full = LlamaForBlend(c, "cpu", torch.float32)
    full.load_state_dict(half.state_dict())
    seqs = _sequences()
    want, _ = _decode(full, seqs, "cpu", torch.float32)
    gpu = LlamaForBlend(c, "cuda", torch.float16, native_attention=True)
    gpu.load_state_dict(half.state_dict())
    got, tables = _decode(gpu, seqs, "cuda", torch.float16)
    _close(got, want)
    assert tables.unique().numel() == tables.numel()


@pytest.mark.gpu
def test_decode_step_captured():
    c = _config(64)
    model = LlamaForBlend(c, "cuda", torch.float16, seed=4, native_attention=True)
    kv = _pages(c, "cuda", torch.float16)
    for layer in kv:
        for t in layer:
            t.normal_()
    prefix = torch.arange(4, device="cuda", dtype=torch.int32)
    tables = torch.arange(4, 4 + 2 * B, device="cuda", dtype=torch.int32).view(B, 2).contiguous()
    free = torch.arange(30, 40, device="cuda", dtype=torch.int32)
    own = torch.tensor([0, 3, 7, 8, 12], device="cuda", dtype=torch.int32)
    tokens = torch.arange(B, device="cuda")

    def step():
        return model.decode_batch(tokens, own, kv, tables, free, prefix, 27)[0]

    step()  # cuBLAS workspaces
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for shift in (0, 1):
        own.add_(shift)
        tokens.add_(shift)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 700])
def test_blend_attention_against_sdpa(rows):
    """The blender's two attention paths on the same rows."""
    c = _config(64)
    model = LlamaForBlend(c, "cuda", torch.float16, seed=1)
    g = torch.Generator().manual_seed(rows)
    T = 1500
    q = torch.randn(rows, 4, 64, generator=g).half().cuda()
    k, v = (torch.randn(T, 2, 64, generator=g).half().cuda() for _ in range(2))
    qp = torch.randperm(T, generator=g)[:rows].sort().values.cuda()
    kp = torch.arange(T, device="cuda")
    want = model.attend(q, k, v, qp, kp)
    model.native_attention = True
    got = model.attend(q, k, v, qp, kp)
    wrapper = LMCVLLMModel.__new__(LMCVLLMModel)
    wrapper.native_attention, wrapper.config = True, c

    class _Layer:
        self_attn = None

    wrapper.layers = [_Layer()]
    assert torch.equal(wrapper.attend(q, k, v, qp, kp), got)
    # each path rounds weights and result (2^-11 each) of sums over values of N(0, 1)
    err = (got.double() - want.double()).norm(dim=-1) / want.double().norm(dim=-1)
    assert float(err.max()) <= 4 * 2.0 ** -11 * 4
